// field_gated.h - what the gated projections' kernels share, and the ways that
// field_gated.hip chooses from.
#pragma once

#include <algorithm>

#include "field.h"

#include "field_act.h"
#include "field_device.h"
#include "field_tiles.h"

namespace gs {

constexpr int kShortDim = 128;
size_t gated_short_ws(const GatedArgs& a, bool grad);
hipError_t gated_short_f32(const GatedArgs& a, bool grad, hipStream_t st);
hipError_t gated_short_bf16(const GatedArgs& a, bool grad, hipStream_t st);

// 8 values of a row from column c, zeros past `cols`.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t cols, float* v) {
    if (c + 8 <= cols) {
        load_any<8>(row + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? to_float(row[c + k]) : 0.0f;
    }
}
// VEC values at any address of a T, past the caches.
template <int VEC, typename T>
__device__ __forceinline__ void store_past(T* p, const float* in) {
    T u[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[j] = from_float<T>(in[j]);
    typedef __attribute__((ext_vector_type(4))) uint32_t words;
    typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t words_any;
    static_assert(sizeof(u) % 16 == 0, "whole quads");
#pragma unroll
    for (int q = 0; q < (int)(sizeof(u) / 16); ++q) {
        words w;
        __builtin_memcpy(&w, reinterpret_cast<const char*>(u) + q * 16, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<words_any*>(p) + q);
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t cols, const float* v) {
    if (c + VEC <= cols) {
        store_any<VEC>(row + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (c + k < cols) row[c + k] = from_float<T>(v[k]);
    }
}

// 8 values as they lie in memory, at any address; zeros from column `cols` on.
template <typename T>
struct Raw {
    quad q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols) {
        T v[8];
        if (c + 8 <= cols) {
            __builtin_memcpy(v, row + c, sizeof(v));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? row[c + e] : (T)0.0f;
        }
        __builtin_memcpy(q, v, sizeof(v));
    }
    __device__ __forceinline__ float operator[](int k) const {
        if constexpr (sizeof(T) == 2)
            return __uint_as_float(k & 1 ? q[0][k / 2] & 0xFFFF0000u : q[0][k / 2] << 16);
        else
            return __uint_as_float(q[k / 4][k % 4]);
    }
};

}  // namespace gs
