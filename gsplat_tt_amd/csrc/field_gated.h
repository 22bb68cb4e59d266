// field_gated.h - what the gated projections' kernels share, and the ways that
// field_gated.hip chooses from.
#pragma once

#include <algorithm>

#include "field.h"

#include "field_act.h"
#include "field_device.h"
#include "field_tiles.h"

namespace gs {

// Rows of up to 128 stay in registers (field_gated_short.h); against tiles, h and a training
// pass: 100000 x 128 to 512 bf16 50 and 249 us, in tiles 78 and 333; 30000 x 128 to 512 fp32
// 56 and 288, in tiles 62 and 298.
constexpr int kShortDim = 128;
size_t gated_short_ws(const GatedArgs& a, bool grad);
hipError_t gated_short_f32(const GatedArgs& a, bool grad, hipStream_t st);
hipError_t gated_short_bf16(const GatedArgs& a, bool grad, hipStream_t st);
// dx's rows n0 .. + n as sums of `shares` parts (rows, ld).
hipError_t gated_dx_join(const GatedArgs& a, const float* part, int shares, int64_t rows, int ld,
                         int64_t n0, int64_t n, hipStream_t st);

// Workgroups of the kernels that join sums, 64 quads each and walking over the rest.
inline unsigned sum_blocks(int64_t quads) {
    return (unsigned)std::min<int64_t>((quads + 63) / 64, (int64_t)1 << 20);
}

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

// N values of a row from column c as they lie in memory, at any address. load() has no
// branch that lanes could part at: one would hold the program up until the values are there, and
// they are loaded a step ahead. Past the row's end it reads values that are there; finish(),
// when they are needed, moves the row's last ones to their places and puts zeros behind.
template <typename T, int N = 8>
struct Raw {
    quad q[N * sizeof(T) / 16];
    __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols) {
        if (cols >= N) {
            __builtin_memcpy(q, row + min(c, cols - N), sizeof(q));
        } else {  // a short row, the same for all
            T v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = row[min((int64_t)e, cols - 1)];
            __builtin_memcpy(q, v, sizeof(q));
        }
    }
    // Both at once.
    __device__ __forceinline__ void load_finished(const T* row, int64_t c, int64_t cols) {
        T v[N];
        if (c + N <= cols) {
            __builtin_memcpy(v, row + c, sizeof(v));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = c + e < cols ? row[c + e] : (T)0.0f;
        }
        __builtin_memcpy(q, v, sizeof(q));
    }
    __device__ __forceinline__ void finish(int64_t c, int64_t cols, bool on) {
        if (on && c + N <= cols) return;
        T v[N];
        __builtin_memcpy(v, q, sizeof(q));
        const int left = on && c < cols ? (int)(cols - c) : 0;  // below N
        const int by = cols >= N ? N - left : 0;
#pragma unroll
        for (int o = N / 2; o > 0; o /= 2)
#pragma unroll
            for (int e = 0; e + o < N; ++e) v[e] = by & o ? v[e + o] : v[e];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = e < left ? v[e] : (T)0.0f;
        __builtin_memcpy(q, v, sizeof(q));
    }
    // As operands.
    template <int NP>
    __device__ __forceinline__ void parts(quad (&out)[NP]) const {
        if constexpr (NP == 1) {
            out[0] = q[0];
        } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = plain_input<NP>((*this)[e]);
            split8_input<NP>(v, out);
        }
    }
    __device__ __forceinline__ float operator[](int k) const {
        if constexpr (sizeof(T) == 2)
            return __uint_as_float(k & 1 ? q[0][k / 2] & 0xFFFF0000u : q[0][k / 2] << 16);
        else
            return __uint_as_float(q[k / 4][k % 4]);
    }
};

}  // namespace gs
