// field_grads.hip - the global norm of many tensors' gradients, and their scaling down to
// a limit.
//
//   norm = sqrt(sum of x^2), or max |x|;  out = x min(1, limit / (norm + 1e-6))
//
// Squares are formed and summed in 64 bits: those of fp32 values are exact there, and
// neither overflow nor vanish. Sizes are compared as bit patterns, in which NaN is the
// largest. A launch takes the list's tensors as its arguments, some hundred at a time, cut
// into chunks of equal length, a workgroup each; the chunks' sums are joined in order by
// one workgroup. Bound by the values' bytes: 59 M fp32 values in 62 us, 3.8 TB/s (51 at
// best), and scaled into other buffers in 73, 6.5 TB/s; 43 M bf16 in 18. Short lists are
// bound by the host, 0.4 us a tensor.
#include <algorithm>

#include "field.h"

#include "field_device.h"

namespace gs {

namespace {

constexpr int kThreads = 256;
constexpr int kVec = 4;
constexpr int kAhead = 4;  // vectors that a thread loads before it uses them
constexpr int64_t kChunk = 2 * kThreads * kVec * kAhead;  // whole rounds of either type
constexpr int64_t kMostChunks = 4096;  // of the whole list, about

struct Entry {
    const void* in;
    void* out;
    int64_t n;  // values
    uint32_t first;  // the tensor's first chunk among the launch's
    uint16_t in_type, out_type;
    // of rows at a distance
    int64_t cols, in_stride, out_stride;
};
// ROWS false: the entries' last three are not kept.
template <bool ROWS>
struct List;
template <>
struct List<true> {
    static constexpr int kMost = 64;
    Entry e[kMost];
    int count;
    int64_t chunk;
    __host__ __device__ uint32_t first(int k) const { return e[k].first; }
    __host__ __device__ Entry entry(int k) const { return e[k]; }
    void set(int k, const Entry& v) { e[k] = v; }
};
template <>
struct List<false> {
    static constexpr int kMost = 120;
    struct Flat {
        const void* in;
        void* out;
        int64_t n;
        uint32_t first;
        uint16_t in_type, out_type;
    } e[kMost];
    int count;
    int64_t chunk;
    __host__ __device__ uint32_t first(int k) const { return e[k].first; }
    __host__ __device__ Entry entry(int k) const {
        return {e[k].in, e[k].out, e[k].n, e[k].first, e[k].in_type, e[k].out_type, 0, 0, 0};
    }
    void set(int k, const Entry& v) { e[k] = {v.in, v.out, v.n, v.first, v.in_type, v.out_type}; }
};
static_assert(sizeof(List<true>) <= 4000 && sizeof(List<false>) <= 4000, "a launch's arguments");

// Place of value i of a tensor of rows.
struct RowWalk {
    int64_t r0, cols;
    uint64_t c0;
    __device__ __forceinline__ RowWalk(int64_t i0, int64_t n_cols) : r0(i0 / n_cols), cols(n_cols) {
        c0 = (uint64_t)(i0 - r0 * n_cols);
    }
    __device__ __forceinline__ void at(int64_t l, int64_t* r, int64_t* c) const {
        const uint64_t v = c0 + (uint64_t)l;
        const uint64_t d = v >> 32 ? v / (uint64_t)cols
                           : cols >> 32 ? 0 : (uint64_t)((uint32_t)v / (uint32_t)cols);
        *r = r0 + (int64_t)d;
        *c = (int64_t)(v - d * (uint64_t)cols);
    }
};

// The launch's tensor that holds chunk b.
template <bool ROWS>
__device__ __forceinline__ int tensor_of(const List<ROWS>& list, uint32_t b) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.first(mid) <= b) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// A sum of squares, or the largest size as a bit pattern.
template <int KIND>
struct Total;
template <>
struct Total<kNormL2> {
    double v;
    __device__ __forceinline__ void add(float x) { v = fma((double)x, (double)x, v); }
    __device__ __forceinline__ void join(const Total& o) { v += o.v; }
    __device__ __forceinline__ float norm() const { return (float)sqrt(v); }
};
template <>
struct Total<kNormMax> {
    uint32_t v, unused;
    __device__ __forceinline__ void add(float x) { v = max(v, __float_as_uint(x) & 0x7FFFFFFFu); }
    __device__ __forceinline__ void join(const Total& o) { v = max(v, o.v); }
    __device__ __forceinline__ float norm() const { return __uint_as_float(v); }
};
template <int KIND>
__device__ __forceinline__ Total<KIND> other_lane(const Total<KIND>& t, int o) {
    Total<KIND> r = {};
    if constexpr (KIND == kNormL2) r.v = __shfl_xor(t.v, o, 64);
    else r.v = (uint32_t)__shfl_xor((int)t.v, o, 64);
    return r;
}
// Over the workgroup, for thread 0.
template <int KIND, int THREADS>
__device__ __forceinline__ Total<KIND> block_total(Total<KIND> t) {
    __shared__ Total<KIND> lds[THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t.join(other_lane(t, o));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = t;
    __syncthreads();
    t = lds[0];
#pragma unroll
    for (int k = 1; k < THREADS / 64; ++k) t.join(lds[k]);
    return t;
}

template <typename T, int KIND>
__device__ __forceinline__ void add_run(const T* p, int64_t n, Total<KIND>& t) {
    constexpr int V = 16 / sizeof(T);
    int64_t i = (int64_t)threadIdx.x * V;
    const int64_t step = (int64_t)kThreads * V;
    for (; i + (kAhead - 1) * step + V <= n; i += kAhead * step) {
        float v[kAhead][V];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load_any<V>(p + i + k * step, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) t.add(v[k][j]);
    }
    for (; i + V <= n; i += step) {
        float v[V];
        load_any<V>(p + i, v);
#pragma unroll
        for (int j = 0; j < V; ++j) t.add(v[j]);
    }
    for (; i < n; ++i) t.add(to_float(p[i]));  // one thread's, fewer than V
}
template <typename T, int KIND>
__device__ __forceinline__ void add_rows(const Entry& e, int64_t i0, int64_t n, Total<KIND>& t) {
    const T* p = static_cast<const T*>(e.in);
    const RowWalk walk(i0, e.cols);
    for (int64_t l = threadIdx.x; l < n; l += kThreads) {
        int64_t r, c;
        walk.at(l, &r, &c);
        t.add(to_float(p[r * e.in_stride + c]));
    }
}

template <int KIND, bool ROWS>
__global__ __launch_bounds__(kThreads) void k_norm_chunks(List<ROWS> list, Total<KIND>* part) {
    const Entry e = list.entry(tensor_of(list, blockIdx.x));
    const int64_t i0 = (int64_t)(blockIdx.x - e.first) * list.chunk;
    const int64_t n = min(list.chunk, e.n - i0);
    Total<KIND> t = {};
    if (!ROWS || e.cols == 0) {
        if (e.in_type == 0) add_run(static_cast<const float*>(e.in) + i0, n, t);
        else add_run(static_cast<const bf16*>(e.in) + i0, n, t);
    } else {
        if (e.in_type == 0) add_rows<float>(e, i0, n, t);
        else add_rows<bf16>(e, i0, n, t);
    }
    t = block_total<KIND, kThreads>(t);
    if (threadIdx.x == 0) part[blockIdx.x] = t;
}

template <int KIND>
__global__ __launch_bounds__(1024) void k_norm_join(const Total<KIND>* part, int64_t count,
                                                    float* norm) {
    Total<KIND> t = {};
    for (int64_t i = threadIdx.x; i < count; i += 1024) t.join(part[i]);
    t = block_total<KIND, 1024>(t);
    if (threadIdx.x == 0) *norm = t.norm();
}

// The factor of a norm; NaN stays NaN.
__device__ __forceinline__ float factor_of(float norm, double max_norm) {
    const double most = max_norm / ((double)norm + 1e-6);
    return most >= 1.0 ? 1.0f : (float)most;
}

template <typename TI, typename TO>
__device__ __forceinline__ void scale_run(const TI* in, TO* out, int64_t n, float f) {
    constexpr int V = 16 / sizeof(TI);
    int64_t i = (int64_t)threadIdx.x * V;
    const int64_t step = (int64_t)kThreads * V;
    for (; i + (kAhead - 1) * step + V <= n; i += kAhead * step) {
        float v[kAhead][V];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load_any<V>(in + i + k * step, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] *= f;
            store_any<V>(out + i + k * step, v[k]);
        }
    }
    for (; i + V <= n; i += step) {
        float v[V];
        load_any<V>(in + i, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= f;
        store_any<V>(out + i, v);
    }
    for (; i < n; ++i) out[i] = from_float<TO>(to_float(in[i]) * f);  // one thread's
}
template <typename TI, typename TO>
__device__ __forceinline__ void scale_part(const Entry& e, int64_t i0, int64_t n, float f) {
    const TI* in = static_cast<const TI*>(e.in);
    TO* out = static_cast<TO*>(e.out);
    if (e.cols == 0) {
        scale_run(in + i0, out + i0, n, f);
        return;
    }
    const RowWalk walk(i0, e.cols);
    for (int64_t l = threadIdx.x; l < n; l += kThreads) {
        int64_t r, c;
        walk.at(l, &r, &c);
        out[r * e.out_stride + c] = from_float<TO>(to_float(in[r * e.in_stride + c]) * f);
    }
}

// Last chunks first: the norm's pass has read them last, and caches may still hold them.
template <bool ROWS>
__global__ __launch_bounds__(kThreads) void k_clip(List<ROWS> list, const float* norm,
                                                   double max_norm) {
    const uint32_t b = gridDim.x - 1 - blockIdx.x;
    const Entry e = list.entry(tensor_of(list, b));
    const float f = factor_of(*norm, max_norm);
    if (f == 1.0f && e.in == e.out) return;
    const int64_t i0 = (int64_t)(b - e.first) * list.chunk;
    const int64_t n = min(list.chunk, e.n - i0);
    if (e.in_type == 0) {
        if (e.out_type == 0) scale_part<float, float>(e, i0, n, f);
        else scale_part<float, bf16>(e, i0, n, f);
    } else {
        if (e.out_type == 0) scale_part<bf16, float>(e, i0, n, f);
        else scale_part<bf16, bf16>(e, i0, n, f);
    }
}

// ---------------------------------------------------------------- small lists
// Few values in all (a head's parameters): one workgroup, one launch, which keeps them in
// registers until the factor is known. `first` counts units of 4 values here.
constexpr int kSmallThreads = 1024, kSmallUnits = 8;  // of a thread

template <int KIND, bool CLIP>
__global__ __launch_bounds__(kSmallThreads) void k_grad_small(List<false> list, uint32_t units,
                                                              float* norm, double max_norm) {
    __shared__ uint32_t first[List<false>::kMost];
    if ((int)threadIdx.x < list.count) first[threadIdx.x] = list.first(threadIdx.x);
    __syncthreads();
    auto entry_of = [&](uint32_t u) {
        int lo = 0, hi = list.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= u) lo = mid; else hi = mid - 1;
        }
        return list.entry(lo);
    };
    float v[kSmallUnits][kVec];
    Total<KIND> t = {};
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
        const uint32_t u = k * kSmallThreads + threadIdx.x;
        if (u >= units) break;
        const Entry e = entry_of(u);
        const int i = (int)(u - e.first) * kVec, n = min(kVec, (int)e.n - i);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            v[k][j] = j >= n ? 0.0f
                      : e.in_type == 0 ? static_cast<const float*>(e.in)[i + j]
                                       : to_float(static_cast<const bf16*>(e.in)[i + j]);
            t.add(v[k][j]);
        }
    }
    t = block_total<KIND, kSmallThreads>(t);
    const float total = t.norm();
    if (threadIdx.x == 0) *norm = total;
    if (!CLIP) return;
    const float f = factor_of(total, max_norm);
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
        const uint32_t u = k * kSmallThreads + threadIdx.x;
        if (u >= units) break;
        const Entry e = entry_of(u);
        if (f == 1.0f && e.in == e.out) continue;
        const int i = (int)(u - e.first) * kVec, n = min(kVec, (int)e.n - i);
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            if (j < n) {
                if (e.out_type == 0) static_cast<float*>(e.out)[i + j] = v[k][j] * f;
                else static_cast<bf16*>(e.out)[i + j] = from_float<bf16>(v[k][j] * f);
            }
    }
}

// Whether one workgroup takes a list, and then the list.
bool small_list(const TensorRef* in, const TensorRef* out, int64_t count, List<false>* list,
                uint32_t* units) {
    if (count > List<false>::kMost) return false;
    *units = 0;
    list->count = (int)count;
    list->chunk = 0;
    for (int64_t k = 0; k < count; ++k) {
        const TensorRef &i = in[k], &o = out != nullptr ? out[k] : in[k];
        const int64_t n = i.rows * i.cols;
        if (i.rows > 1 || o.rows > 1 || n > kSmallThreads * kSmallUnits * kVec) return false;
        list->set((int)k, Entry{i.data, o.data, n, *units, (uint16_t)i.dtype, (uint16_t)o.dtype,
                                0, 0, 0});
        *units += (uint32_t)((n + kVec - 1) / kVec);
        if (*units > kSmallThreads * kSmallUnits) return false;
    }
    return true;
}

// ---------------------------------------------------------------- launches
int64_t chunk_of(const TensorRef* t, int64_t count) {
    int64_t total = 0;
    for (int64_t k = 0; k < count; ++k) total += t[k].rows * t[k].cols;
    const int64_t per = (total + kMostChunks - 1) / kMostChunks;
    return std::max(kChunk, (per + kChunk - 1) / kChunk * kChunk);
}
int64_t chunks_of(const TensorRef& t, int64_t chunk) {
    return (t.rows * t.cols + chunk - 1) / chunk;
}

// Runs of the list that a launch takes, tensors of rows and others apart, given to
// `launch(list, blocks)`; the chunks in order.
template <bool ROWS, class Launch>
hipError_t each_list(const TensorRef* in, const TensorRef* out, int64_t count, int64_t chunk,
                     Launch launch) {
    List<ROWS> list;
    list.chunk = chunk;
    int64_t k = 0;
    while (k < count) {
        list.count = 0;
        uint32_t blocks = 0;
        for (; k < count && list.count < List<ROWS>::kMost; ++k) {
            const TensorRef &i = in[k], &o = out != nullptr ? out[k] : in[k];
            const bool rows = i.rows > 1 || o.rows > 1;
            if (rows != ROWS) continue;
            // one of the two may be one run of values where the other has rows
            const int64_t cols = i.rows > 1 ? i.cols : o.cols;
            list.set(list.count++, Entry{i.data, o.data, i.rows * i.cols, blocks, (uint16_t)i.dtype,
                                         (uint16_t)o.dtype, cols, i.rows > 1 ? i.stride : cols,
                                         o.rows > 1 ? o.stride : cols});
            blocks += (uint32_t)chunks_of(i, chunk);
        }
        if (list.count == 0) break;
        const hipError_t e = launch(list, blocks);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int KIND>
hipError_t norm_run(const TensorRef* t, int64_t count, float* norm, void* ws, hipStream_t st) {
    const int64_t chunk = chunk_of(t, count);
    Total<KIND>* part = static_cast<Total<KIND>*>(ws);
    int64_t done = 0;
    auto launch = [&](const auto& list, uint32_t blocks) {
        k_norm_chunks<KIND><<<blocks, kThreads, 0, st>>>(list, part + done);
        done += blocks;
        return hipGetLastError();
    };
    hipError_t e = each_list<false>(t, nullptr, count, chunk, launch);
    if (e == hipSuccess) e = each_list<true>(t, nullptr, count, chunk, launch);
    if (e != hipSuccess) return e;
    k_norm_join<KIND><<<1, 1024, 0, st>>>(part, done, norm);
    return hipGetLastError();
}

}  // namespace

size_t grad_norm_ws(const TensorRef* t, int64_t count) {
    const int64_t chunk = chunk_of(t, count);
    size_t chunks = 0;
    for (int64_t k = 0; k < count; ++k) chunks += (size_t)chunks_of(t[k], chunk);
    return chunks * sizeof(Total<kNormL2>);
}

hipError_t launch_grad_norm(const TensorRef* t, int64_t count, int kind, float* norm, void* ws,
                            hipStream_t st) {
    List<false> small;
    uint32_t units;
    if (small_list(t, nullptr, count, &small, &units)) {
        if (kind == kNormMax)
            k_grad_small<kNormMax, false><<<1, kSmallThreads, 0, st>>>(small, units, norm, 0.0);
        else
            k_grad_small<kNormL2, false><<<1, kSmallThreads, 0, st>>>(small, units, norm, 0.0);
        return hipGetLastError();
    }
    return kind == kNormMax ? norm_run<kNormMax>(t, count, norm, ws, st)
                            : norm_run<kNormL2>(t, count, norm, ws, st);
}

hipError_t launch_grad_clip(const TensorRef* in, const TensorRef* out, int64_t count, int kind,
                            float* norm, double max_norm, void* ws, hipStream_t st) {
    if (kind != kNormGiven) {
        List<false> small;
        uint32_t units;
        if (small_list(in, out, count, &small, &units)) {
            if (kind == kNormMax)
                k_grad_small<kNormMax, true><<<1, kSmallThreads, 0, st>>>(small, units, norm,
                                                                          max_norm);
            else
                k_grad_small<kNormL2, true><<<1, kSmallThreads, 0, st>>>(small, units, norm,
                                                                         max_norm);
            return hipGetLastError();
        }
        const hipError_t e = launch_grad_norm(in, count, kind, norm, ws, st);
        if (e != hipSuccess) return e;
    }
    const int64_t chunk = chunk_of(in, count);
    auto launch = [&](const auto& list, uint32_t blocks) {
        k_clip<<<blocks, kThreads, 0, st>>>(list, norm, max_norm);
        return hipGetLastError();
    };
    const hipError_t e = each_list<true>(in, out, count, chunk, launch);
    return e != hipSuccess ? e : each_list<false>(in, out, count, chunk, launch);
}

}  // namespace gs
