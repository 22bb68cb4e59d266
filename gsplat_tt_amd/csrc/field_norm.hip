// field_norm.hip - group norm with an activation over channels-last images.
//
//   mean, var over a group's channels and all pixels; rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd;  z = xh weight + bias;  y = act(z)
// and, from dy: dz = dy act'(z), dbias = sum dz, dweight = sum dz xh,
//   dx = rstd (weight dz - m1 - xh m2), m1, m2 the group's means of weight dz
//   and of weight dz xh.
//
// All arithmetic is fp32. A thread keeps VEC channels and walks over pixels, so
// every per-channel value stays in registers.
#include "field.h"

#include "field_device.h"

namespace gs {

namespace {

constexpr int kThreads = 256;
enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

template <int ACT>
__device__ __forceinline__ float act(float z) {
    if (ACT == kActRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (ACT == kActSilu) return z / (1.0f + __expf(-z));
    if (ACT == kActGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if (ACT == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == kActSilu) {
        const float s = 1.0f / (1.0f + __expf(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    if (ACT == kActGelu)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
               z * 0.39894228040143268f * __expf(-0.5f * z * z);
    return 1.0f;
}

// Count, mean and sum of squared distances from the mean, joined pairwise, so
// that a mean far from 0 costs no digits.
struct Moments {
    float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
    if (b.n == 0.0f) return a;
    if (a.n == 0.0f) return b;
    const float n = a.n + b.n, d = b.mean - a.mean, f = b.n / n;
    return {n, a.mean + d * f, a.m2 + b.m2 + d * d * a.n * f};
}

// A workgroup's place: image b, chunk of pixels, channel vectors from cv0; a
// thread's channels and its first pixel.
struct Place {
    int64_t b, p0, p1;
    int64_t part;  // the chunk's place among (batch, chunks)
    int cols, slots, slot, c;  // channel vectors of the workgroup, pixels at a time
    bool on;
};
template <int VEC>
__device__ __forceinline__ Place place_of(int64_t pixels, int channels, int chunks) {
    Place p;
    const int all = (channels + VEC - 1) / VEC, cv0 = blockIdx.y * kThreads;
    p.cols = min(kThreads, all - cv0);
    p.slots = kThreads / p.cols;
    p.slot = threadIdx.x / p.cols;
    p.c = (cv0 + (int)threadIdx.x % p.cols) * VEC;
    p.on = p.slot < p.slots;
    p.b = blockIdx.x / (unsigned)chunks;
    p.part = blockIdx.x;
    const int64_t per = (pixels + chunks - 1) / chunks;
    p.p0 = min(pixels, per * (blockIdx.x % (unsigned)chunks));
    p.p1 = min(pixels, p.p0 + per);
    return p;
}

// ---------------------------------------------------------------- statistics
// Partials (batch, chunks, channels) of a chunk's mean and squared distances.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void k_norm_stats(NormArgs a, int chunks, float2* part) {
    __shared__ Moments lds[kThreads * VEC];
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    Moments m[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) m[j] = {0.0f, 0.0f, 0.0f};
    if (p.on) {
        for (int64_t q = p.p0 + p.slot; q < p.p1; q += p.slots) {
            float v[VEC];
            load_vec<VEC>(x + q * a.x_pixel, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) m[j] = join(m[j], {1.0f, v[j], 0.0f});
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) lds[threadIdx.x * VEC + j] = m[j];
    __syncthreads();
    if (p.slot == 0) {
        for (int j = 0; j < VEC; ++j) {
            Moments s = m[j];
            for (int k = 1; k < p.slots; ++k) s = join(s, lds[(threadIdx.x + k * p.cols) * VEC + j]);
            part[p.part * a.channels + p.c + j] = make_float2(s.mean, s.m2);
        }
    }
}

// One workgroup per (image, group): joins its channels' chunks.
__global__ __launch_bounds__(kThreads) void k_norm_finish(NormArgs a, int chunks,
                                                          const float2* part) {
    __shared__ Moments lds[kThreads];
    const int64_t b = blockIdx.x / a.groups;
    const int g = blockIdx.x % a.groups, per_group = a.channels / a.groups;
    const int64_t per = (a.pixels + chunks - 1) / chunks;
    Moments m = {0.0f, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < chunks * per_group; i += kThreads) {
        const int k = i / per_group, c = g * per_group + i % per_group;
        const int64_t p0 = min(a.pixels, per * k), p1 = min(a.pixels, p0 + per);
        const float2 v = part[(b * chunks + k) * a.channels + c];
        m = join(m, {(float)(p1 - p0), v.x, v.y});
    }
    lds[threadIdx.x] = m;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) lds[threadIdx.x] = join(lds[threadIdx.x], lds[threadIdx.x + o]);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float count = (float)a.pixels * (float)per_group;
        a.mean[blockIdx.x] = lds[0].mean;
        a.rstd[blockIdx.x] = 1.0f / sqrtf(lds[0].m2 / count + a.eps);
    }
}

// ---------------------------------------------------------------- forward
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_apply(NormArgs a, int chunks) {
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    if (!p.on) return;
    const int per_group = a.channels / a.groups;
    float mean[VEC], k[VEC], bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int64_t g = p.b * a.groups + (p.c + j) / per_group;
        mean[j] = a.mean[g];
        k[j] = a.rstd[g] * (a.weight != nullptr ? a.weight[p.c + j] : 1.0f);
        bias[j] = a.bias != nullptr ? a.bias[p.c + j] : 0.0f;
    }
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    T* y = static_cast<T*>(a.y) + p.b * a.y_batch + p.c;
    for (int64_t q = p.p0 + p.slot; q < p.p1; q += p.slots) {
        float v[VEC];
        load_vec<VEC>(x + q * a.x_pixel, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = act<ACT>(fmaf(v[j] - mean[j], k[j], bias[j]));
        store_vec<VEC>(y + q * a.y_pixel, v);
    }
}

// ---------------------------------------------------------------- gradient
// Partials (batch, chunks, channels) of sum dz and sum dz xh.
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_grad_sums(NormArgs a, int chunks, float2* part) {
    __shared__ float2 lds[kThreads * VEC];
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    const int per_group = a.channels / a.groups;
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
    if (p.on) {
        float mean[VEC], rstd[VEC], w[VEC], bias[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int64_t g = p.b * a.groups + (p.c + j) / per_group;
            mean[j] = a.mean[g];
            rstd[j] = a.rstd[g];
            w[j] = a.weight != nullptr ? a.weight[p.c + j] : 1.0f;
            bias[j] = a.bias != nullptr ? a.bias[p.c + j] : 0.0f;
        }
        const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
        const T* dy = static_cast<const T*>(a.dy) + p.b * a.dy_batch + p.c;
        for (int64_t q = p.p0 + p.slot; q < p.p1; q += p.slots) {
            float v[VEC], d[VEC];
            load_vec<VEC>(x + q * a.x_pixel, v);
            load_vec<VEC>(dy + q * a.dy_pixel, d);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float xh = (v[j] - mean[j]) * rstd[j];
                const float dz = d[j] * act_slope<ACT>(fmaf(xh, w[j], bias[j]));
                s1[j] += dz;
                s2[j] = fmaf(dz, xh, s2[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) lds[threadIdx.x * VEC + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    if (p.slot == 0) {
        for (int j = 0; j < VEC; ++j) {
            for (int k = 1; k < p.slots; ++k) {
                const float2 u = lds[(threadIdx.x + k * p.cols) * VEC + j];
                s1[j] += u.x;
                s2[j] += u.y;
            }
            part[p.part * a.channels + p.c + j] = make_float2(s1[j], s2[j]);
        }
    }
}

// One workgroup per (image, group): the group's channel sums over the chunks, and m1, m2.
__global__ __launch_bounds__(kThreads) void k_norm_grad_finish(NormArgs a, int chunks,
                                                               const float2* part, float2* sums,
                                                               float2* means) {
    __shared__ float2 lds[kThreads];
    const int64_t b = blockIdx.x / a.groups;
    const int g = blockIdx.x % a.groups, per_group = a.channels / a.groups;
    float m1 = 0.0f, m2 = 0.0f;
    for (int c = g * per_group; c < (g + 1) * per_group; ++c) {
        float2 s = make_float2(0.0f, 0.0f);
        for (int k = threadIdx.x; k < chunks; k += kThreads) {
            const float2 v = part[(b * chunks + k) * a.channels + c];
            s.x += v.x;
            s.y += v.y;
        }
        __syncthreads();
        lds[threadIdx.x] = s;
        __syncthreads();
        for (int o = kThreads / 2; o > 0; o >>= 1) {
            if ((int)threadIdx.x < o) {
                lds[threadIdx.x].x += lds[threadIdx.x + o].x;
                lds[threadIdx.x].y += lds[threadIdx.x + o].y;
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            const float w = a.weight != nullptr ? a.weight[c] : 1.0f;
            sums[b * a.channels + c] = lds[0];
            m1 += w * lds[0].x;
            m2 += w * lds[0].y;
        }
    }
    if (threadIdx.x == 0) {
        const float count = (float)a.pixels * (float)per_group;
        means[blockIdx.x] = make_float2(m1 / count, m2 / count);
    }
}

__global__ __launch_bounds__(kThreads) void k_norm_grad_params(NormArgs a, const float2* sums) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.channels) return;
    float db = 0.0f, dw = 0.0f;
    for (int64_t b = 0; b < a.batch; ++b) {
        const float2 s = sums[b * a.channels + c];
        db += s.x;
        dw += s.y;
    }
    if (a.dbias != nullptr) a.dbias[c] = db;
    if (a.dweight != nullptr) a.dweight[c] = dw;
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_grad_apply(NormArgs a, int chunks,
                                                              const float2* means) {
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    if (!p.on) return;
    const int per_group = a.channels / a.groups;
    float mean[VEC], rstd[VEC], w[VEC], bias[VEC], m1[VEC], m2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int64_t g = p.b * a.groups + (p.c + j) / per_group;
        mean[j] = a.mean[g];
        rstd[j] = a.rstd[g];
        w[j] = a.weight != nullptr ? a.weight[p.c + j] : 1.0f;
        bias[j] = a.bias != nullptr ? a.bias[p.c + j] : 0.0f;
        const float2 m = means[g];
        m1[j] = m.x;
        m2[j] = m.y;
    }
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    const T* dy = static_cast<const T*>(a.dy) + p.b * a.dy_batch + p.c;
    T* dx = static_cast<T*>(a.dx) + p.b * a.dx_batch + p.c;
    for (int64_t q = p.p0 + p.slot; q < p.p1; q += p.slots) {
        float v[VEC], d[VEC];
        load_vec<VEC>(x + q * a.x_pixel, v);
        load_vec<VEC>(dy + q * a.dy_pixel, d);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float xh = (v[j] - mean[j]) * rstd[j];
            const float dz = d[j] * act_slope<ACT>(fmaf(xh, w[j], bias[j]));
            v[j] = rstd[j] * (fmaf(w[j], dz, -m1[j]) - xh * m2[j]);
        }
        store_vec<VEC>(dx + q * a.dx_pixel, v);
    }
}

// Chunks of an image's pixels: enough workgroups for the chip, at least 64
// pixels each.
int chunks_of(int64_t batch, int64_t pixels) {
    int64_t k = batch < 1 ? 1 : (2048 + batch - 1) / batch;
    if (k > (pixels + 63) / 64) k = (pixels + 63) / 64;
    return k < 1 ? 1 : (int)k;
}

struct NormWs {
    float2 *part, *sums, *means;
    size_t bytes;
    NormWs(void* base, int64_t batch, int64_t pixels, int channels) {
        Carve c(base);
        part = c.take<float2>((size_t)batch * chunks_of(batch, pixels) * channels);
        sums = c.take<float2>((size_t)batch * channels);
        means = c.take<float2>((size_t)batch * channels);
        bytes = c.bytes();
    }
};

template <typename T, int VEC, int ACT>
hipError_t norm_run(const NormArgs& a, bool grad, hipStream_t st) {
    const NormWs w(a.ws, a.batch, a.pixels, a.channels);
    const int chunks = chunks_of(a.batch, a.pixels);
    const int cols = (a.channels + VEC - 1) / VEC;
    const dim3 grid((unsigned)(chunks * a.batch), (unsigned)((cols + kThreads - 1) / kThreads));
    const unsigned groups = (unsigned)(a.batch * a.groups);
    if (!grad) {
        k_norm_stats<T, VEC><<<grid, kThreads, 0, st>>>(a, chunks, w.part);
        k_norm_finish<<<groups, kThreads, 0, st>>>(a, chunks, w.part);
        k_norm_apply<T, VEC, ACT><<<grid, kThreads, 0, st>>>(a, chunks);
    } else {
        k_norm_grad_sums<T, VEC, ACT><<<grid, kThreads, 0, st>>>(a, chunks, w.part);
        k_norm_grad_finish<<<groups, kThreads, 0, st>>>(a, chunks, w.part, w.sums, w.means);
        k_norm_grad_params<<<(unsigned)((a.channels + kThreads - 1) / kThreads), kThreads, 0, st>>>(
            a, w.sums);
        k_norm_grad_apply<T, VEC, ACT><<<grid, kThreads, 0, st>>>(a, chunks, w.means);
    }
    return hipGetLastError();
}

template <typename T, int VEC>
hipError_t norm_act(const NormArgs& a, bool grad, hipStream_t st) {
    switch (a.act) {
        case kActRelu: return norm_run<T, VEC, kActRelu>(a, grad, st);
        case kActSilu: return norm_run<T, VEC, kActSilu>(a, grad, st);
        case kActGelu: return norm_run<T, VEC, kActGelu>(a, grad, st);
        default: return norm_run<T, VEC, kActNone>(a, grad, st);
    }
}

template <typename T>
hipError_t norm_typed(const NormArgs& a, bool grad, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    auto rows_ok = [&](const void* p, int64_t batch, int64_t pixel) {
        return p == nullptr || (aligned_rows<T>(p, pixel, VEC) && batch % VEC == 0);
    };
    const bool vec = a.channels % VEC == 0 && rows_ok(a.x, a.x_batch, a.x_pixel) &&
                     rows_ok(a.y, a.y_batch, a.y_pixel) && rows_ok(a.dy, a.dy_batch, a.dy_pixel) &&
                     rows_ok(a.dx, a.dx_batch, a.dx_pixel);
    return vec ? norm_act<T, VEC>(a, grad, st) : norm_act<T, 1>(a, grad, st);
}

}  // namespace

size_t group_norm_ws(int64_t batch, int64_t pixels, int channels) {
    return NormWs(nullptr, batch, pixels, channels).bytes;
}

hipError_t launch_group_norm(const NormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.pixels == 0) return hipSuccess;
    return a.dtype == 0 ? norm_typed<float>(a, false, st) : norm_typed<bf16>(a, false, st);
}

hipError_t launch_group_norm_grad(const NormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.pixels == 0) {
        NormArgs e = a;  // no pixels: the parameters' gradients are 0
        e.batch = 0;
        k_norm_grad_params<<<(unsigned)((a.channels + kThreads - 1) / kThreads), kThreads, 0, st>>>(
            e, nullptr);
        return hipGetLastError();
    }
    return a.dtype == 0 ? norm_typed<float>(a, true, st) : norm_typed<bf16>(a, true, st);
}

}  // namespace gs
