// field_device.h - device helpers of the feature operators: element types, vector
// loads and stores, checked ids, workgroup scans, workspace layout.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "field.h"

namespace gs {

using bf16 = __bf16;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return (float)v; }
// to bf16: round to nearest even, NaN kept
template <typename T>
__device__ __forceinline__ T from_float(float v) { return (T)v; }

// VEC elements at an address aligned to VEC * sizeof(T) bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) VecOf {
    T v[VEC];
};
template <int VEC, typename T>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
    const VecOf<T, VEC> u = *reinterpret_cast<const VecOf<T, VEC>*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = to_float(u.v[j]);
}
// The same at any address of a T.
template <int VEC, typename T>
__device__ __forceinline__ void load_any(const T* p, float* out) {
    T u[VEC];
    __builtin_memcpy(u, p, sizeof(u));
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = to_float(u[j]);
}
template <int VEC, typename T>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
    VecOf<T, VEC> u;
#pragma unroll
    for (int j = 0; j < VEC; ++j) u.v[j] = from_float<T>(in[j]);
    *reinterpret_cast<VecOf<T, VEC>*>(p) = u;
}

template <int VEC, typename T>
__device__ __forceinline__ void store_any(T* p, const float* in) {
    T u[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[j] = from_float<T>(in[j]);
    __builtin_memcpy(p, u, sizeof(u));
}
// The same past the caches, for outputs that are not read again soon.
template <int VEC, typename T>
__device__ __forceinline__ void store_nt(T* p, const float* in) {
    VecOf<T, VEC> u;
#pragma unroll
    for (int j = 0; j < VEC; ++j) u.v[j] = from_float<T>(in[j]);
    if constexpr (sizeof(u) % 4 == 0) {
        typedef __attribute__((ext_vector_type(sizeof(u) / 4))) uint32_t words;
        __builtin_nontemporal_store(__builtin_bit_cast(words, u), reinterpret_cast<words*>(p));
    } else {
        *reinterpret_cast<VecOf<T, VEC>*>(p) = u;
    }
}

// Whether rows at `stride` elements apart can be read VEC elements at a time.
template <typename T>
inline bool aligned_rows(const void* p, int64_t stride, int vec) {
    return reinterpret_cast<uintptr_t>(p) % (sizeof(T) * vec) == 0 && stride % vec == 0;
}

// Id i, or -1 where it is masked (below 0) or past the table; the latter is
// reported in *flags.
__device__ __forceinline__ int32_t load_id(const void* ids, int ids64, int64_t i, int64_t rows,
                                           uint32_t* flags) {
    const int64_t v = ids64 ? static_cast<const int64_t*>(ids)[i]
                            : (int64_t) static_cast<const int32_t*>(ids)[i];
    if (v >= rows) {
        if (flags != nullptr) atomicOr(flags, kFlagIdRange);
        return -1;
    }
    return v < 0 ? -1 : (int32_t)v;
}

// Exclusive prefix of one value per thread over the workgroup, and the total; lds:
// a word per wave.
template <int THREADS>
__device__ __forceinline__ uint32_t block_excl_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
    const int t = threadIdx.x, lane = t & 63;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(s, o, 64);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 63) lds[t >> 6] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < THREADS / 64; ++k) {
        if (k == (t >> 6)) before = all;
        all += lds[k];
    }
    *total = all;
    return before + s - v;
}

// Most blocks of a grid that its kernel walks over with: a launch takes fewer than 2^32
// threads a dimension, 2^24 blocks of 256 (2^24 were refused, two more ran as two).
constexpr int64_t kMostBlocks = (int64_t)1 << 22;
inline unsigned blocks_of(int64_t items, int64_t per_block) {
    const int64_t b = (items + per_block - 1) / per_block;
    return (unsigned)(b < kMostBlocks ? b : kMostBlocks);
}

// Returns a launch's error, so that nothing runs on what it would have written.
#define GS_LAUNCHED()                               \
    do {                                            \
        const hipError_t e_ = hipGetLastError();    \
        if (e_ != hipSuccess) return e_;            \
    } while (0)

// Consecutive 256-byte aligned arrays of a workspace; a null base only counts.
struct Carve {
    uintptr_t base;
    size_t at = 0;
    explicit Carve(void* p) : base(reinterpret_cast<uintptr_t>(p)) {}
    template <typename T>
    T* take(size_t n) {
        T* p = reinterpret_cast<T*>(base + at);
        at += (n * sizeof(T) + 255) & ~size_t(255);
        return p;
    }
    size_t bytes() const { return at; }
};

}  // namespace gs
