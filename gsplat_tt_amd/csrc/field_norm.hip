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

#include "field_act.h"
#include "field_device.h"

namespace gs {

namespace {

constexpr int kThreads = 256;

// Count, mean and sum of squared distances from the mean. Pieces are joined by
// their means' difference, so that a mean far from 0 costs no digits. An empty piece
// (count and mean 0) joins as nothing: the other's mean stays as it is, and the square of
// the difference, infinite for means past 1.8e19, is not formed before its factor 0.
struct Moments {
    float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
    const float n = a.n + b.n, d = b.mean - a.mean;
    const float f = a.n > 0.0f ? b.n * __builtin_amdgcn_rcpf(n) : 1.0f;
    return {n, fmaf(d, f, a.mean), a.m2 + fmaf(d * (a.n * f), d, b.m2)};
}

// A wave's and then the workgroup's sum, the same order every time.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* lds) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = lds[0];
#pragma unroll
    for (int k = 1; k < THREADS / 64; ++k) s += lds[k];
    return s;
}

// What VEC channels from c of image b need: xh = (x - m) r, z = xh w + bias. The mean is
// subtracted first: folded into one multiply-add, x r - m r, the product's rounding
// stays as a share of m r, which a mean far from 0 makes larger than xh.
template <int VEC>
struct Channels {
    float m[VEC], r[VEC], w[VEC], bias[VEC];
    __device__ __forceinline__ Channels(const NormArgs& a, int64_t b, int c) {
        const int per_group = a.channels / a.groups;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int64_t g = b * a.groups + (c + j) / per_group;
            m[j] = a.mean[g];
            r[j] = a.rstd[g];
            w[j] = a.weight != nullptr ? a.weight[c + j] : 1.0f;
            bias[j] = a.bias != nullptr ? a.bias[c + j] : 0.0f;
        }
    }
    __device__ __forceinline__ float xh(float x, int j) const { return (x - m[j]) * r[j]; }
    __device__ __forceinline__ float z(float h, int j) const { return fmaf(h, w[j], bias[j]); }
};

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

// Pixels that a thread loads before it uses them.
constexpr int kAhead = 4;

// ---------------------------------------------------------------- statistics
// Partials (batch, chunks, channels) of a chunk's mean and squared distances.
// Four pixels at a time get a mean of their own, then their distances from it:
// 3 operations a value, against 10 for a running mean; their sum in pairs, which for four
// equal values is exact. Bound by x's bytes: 921600 x 64
// bf16 (118 MB) 23 us, 5.2 TB/s.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void k_norm_stats(NormArgs a, int chunks, float2* part) {
    __shared__ Moments lds[kThreads * VEC];
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    float n = 0.0f, mean[VEC], m2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) mean[j] = m2[j] = 0.0f;
    if (p.on) {
        int64_t q = p.p0 + p.slot;
        for (; q + (kAhead - 1) * p.slots < p.p1; q += kAhead * p.slots) {
            float v[kAhead][VEC];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) load_vec<VEC>(x + (q + k * p.slots) * a.x_pixel, v[k]);
            const float total = n + kAhead, f = kAhead * __builtin_amdgcn_rcpf(total), nf = n * f;
            n = total;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                static_assert(kAhead == 4, "two pairs");
                const float s = ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j])) * 0.25f;
                float d2 = 0.0f;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) d2 = fmaf(v[k][j] - s, v[k][j] - s, d2);
                const float d = s - mean[j];
                mean[j] = fmaf(d, f, mean[j]);
                m2[j] += fmaf(d * nf, d, d2);
            }
        }
        for (; q < p.p1; q += p.slots) {
            float v[VEC];
            load_vec<VEC>(x + q * a.x_pixel, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Moments m = join({n, mean[j], m2[j]}, {1.0f, v[j], 0.0f});
                mean[j] = m.mean;
                m2[j] = m.m2;
            }
            n += 1.0f;
        }
    }
    const int at = threadIdx.x;
#pragma unroll
    for (int j = 0; j < VEC; ++j) lds[j * kThreads + at] = {n, mean[j], m2[j]};
    // halve the slots until one is left
    for (int len = p.slots; len > 1;) {
        const int half = (len + 1) / 2;
        __syncthreads();
        if (p.slot < len - half)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                lds[j * kThreads + at] =
                    join(lds[j * kThreads + at], lds[j * kThreads + at + half * p.cols]);
        len = half;
    }
    if (p.slot == 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            part[p.part * a.channels + p.c + j] =
                make_float2(lds[j * kThreads + at].mean, lds[j * kThreads + at].m2);
}

// A workgroup an (image, group), or several one after the other: joins its channels'
// chunks. Bound by latency, 5 to 7 us.
__global__ __launch_bounds__(kThreads) void k_norm_finish(NormArgs a, int chunks,
                                                          const float2* part) {
    __shared__ Moments lds[kThreads];
    const int per_group = a.channels / a.groups;
    const int64_t per = (a.pixels + chunks - 1) / chunks;
    for (int64_t at = blockIdx.x; at < a.batch * a.groups; at += gridDim.x) {
        const int64_t b = at / a.groups;
        const float2* from = part + b * chunks * a.channels + (at - b * a.groups) * per_group;
        Moments m = {0.0f, 0.0f, 0.0f};
        const int all = chunks * per_group;
        for (int i0 = threadIdx.x; i0 < all; i0 += kThreads * 8) {
            float2 v[8];
            float n[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = min(i0 + u * kThreads, all - 1);
                const int k = i / per_group, c = i - k * per_group;
                const bool on = i0 + u * kThreads < all;
                v[u] = from[(int64_t)k * a.channels + c];
                if (!on) v[u] = make_float2(0.0f, 0.0f);
                const int64_t p0 = min(a.pixels, per * k);
                n[u] = on ? (float)(min(a.pixels, p0 + per) - p0) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) m = join(m, {n[u], v[u].x, v[u].y});
        }
        lds[threadIdx.x] = m;
        __syncthreads();
        for (int o = kThreads / 2; o > 0; o >>= 1) {
            if ((int)threadIdx.x < o)
                lds[threadIdx.x] = join(lds[threadIdx.x], lds[threadIdx.x + o]);
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            const float count = (float)a.pixels * (float)per_group;
            a.mean[at] = lds[0].mean;
            a.rstd[at] = 1.0f / sqrtf(lds[0].m2 / count + a.eps);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- forward
// y, from x once more: where x fits the cache behind the L2s the second read comes from
// there. Stored past the caches. Bound by bytes: 921600 x 64 bf16 40 us, 5.9 TB/s read
// and written.
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_apply(NormArgs a, int chunks) {
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    if (!p.on) return;
    Channels<VEC> ch(a, p.b, p.c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) ch.w[j] *= ch.r[j];  // xh is not needed
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    T* y = static_cast<T*>(a.y) + p.b * a.y_batch + p.c;
    auto one = [&](float* v) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = act<ACT>(ch.z(v[j] - ch.m[j], j));
    };
    int64_t q = p.p0 + p.slot;
    for (; q + (kAhead - 1) * p.slots < p.p1; q += kAhead * p.slots) {
        float v[kAhead][VEC];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) load_vec<VEC>(x + (q + k * p.slots) * a.x_pixel, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            one(v[k]);
            store_nt<VEC>(y + (q + k * p.slots) * a.y_pixel, v[k]);
        }
    }
    for (; q < p.p1; q += p.slots) {
        float v[VEC];
        load_vec<VEC>(x + q * a.x_pixel, v);
        one(v);
        store_vec<VEC>(y + q * a.y_pixel, v);
    }
}

// ---------------------------------------------------------------- gradient
// Adds the slots' channel sums, halving; slot 0 ends with the total.
template <int VEC, int THREADS>
__device__ __forceinline__ void slots_sum(float2* lds, int at, int slot, int slots, int cols,
                                          float* s1, float* s2) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) lds[j * THREADS + at] = make_float2(s1[j], s2[j]);
    for (int len = slots; len > 1;) {
        const int half = (len + 1) / 2;
        __syncthreads();
        if (slot < len - half)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float2 u = lds[j * THREADS + at + half * cols];
                s1[j] += u.x;
                s2[j] += u.y;
                lds[j * THREADS + at] = make_float2(s1[j], s2[j]);
            }
        len = half;
    }
}

// Partials (batch, chunks, channels) of sum dz and sum dz xh. Bound by the bytes of dy
// and x, with gelu as much by its arithmetic: 333666 x 48 fp32 relu (128 MB) 22 us, 5.8
// TB/s; 614400 x 128 bf16 gelu (315 MB) 80 us, 3.9 TB/s, with the vector units busy 72 %
// of the time.
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_grad_sums(NormArgs a, int chunks, float2* part) {
    __shared__ float2 lds[kThreads * VEC];
    constexpr int AHEAD = kAhead / 2;  // of x and of dy
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.0f;
    if (p.on) {
        const Channels<VEC> ch(a, p.b, p.c);
        const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
        const T* dy = static_cast<const T*>(a.dy) + p.b * a.dy_batch + p.c;
        auto one = [&](const float* v, const float* d) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float xh = ch.xh(v[j], j);
                const float dz = d[j] * act_slope<ACT>(ch.z(xh, j));
                s1[j] += dz;
                s2[j] = fmaf(dz, xh, s2[j]);
            }
        };
        int64_t q = p.p0 + p.slot;
        for (; q + (AHEAD - 1) * p.slots < p.p1; q += AHEAD * p.slots) {
            float v[AHEAD][VEC], d[AHEAD][VEC];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                load_vec<VEC>(x + (q + k * p.slots) * a.x_pixel, v[k]);
                load_vec<VEC>(dy + (q + k * p.slots) * a.dy_pixel, d[k]);
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) one(v[k], d[k]);
        }
        for (; q < p.p1; q += p.slots) {
            float v[VEC], d[VEC];
            load_vec<VEC>(x + q * a.x_pixel, v);
            load_vec<VEC>(dy + q * a.dy_pixel, d);
            one(v, d);
        }
    }
    slots_sum<VEC, kThreads>(lds, threadIdx.x, p.slot, p.slots, p.cols, s1, s2);
    if (p.slot == 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            part[p.part * a.channels + p.c + j] = make_float2(s1[j], s2[j]);
}

// A workgroup an (image, group), or several one after the other: the group's channel
// sums over the chunks, and m1, m2. Threads of one channel stand `per_group` apart (or
// walk over channels when a group has more than the workgroup has threads).
__global__ __launch_bounds__(kThreads) void k_norm_grad_finish(NormArgs a, int chunks,
                                                               const float2* part, float2* sums,
                                                               float2* means) {
    __shared__ float2 lds[kThreads];
    __shared__ float red[kThreads / 64];
    const int per_group = a.channels / a.groups;
    const int cols = min(per_group, kThreads), rows = kThreads / cols;
    const int row = threadIdx.x / cols, col = threadIdx.x % cols;
    for (int64_t at = blockIdx.x; at < a.batch * a.groups; at += gridDim.x) {
        const int64_t b = at / a.groups;
        const int g = (int)(at - b * a.groups);
        float m1 = 0.0f, m2 = 0.0f;
        for (int c0 = 0; c0 < per_group; c0 += cols) {
            const bool on = row < rows && c0 + col < per_group;
            const int c = g * per_group + c0 + col;
            float s1[1] = {0.0f}, s2[1] = {0.0f};
            if (on) {
                const float2* from = part + b * chunks * a.channels + c;
                for (int k0 = row; k0 < chunks; k0 += rows * 8) {
                    float2 v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int k = k0 + u * rows;
                        v[u] = from[(int64_t)min(k, chunks - 1) * a.channels];
                        if (k >= chunks) v[u] = make_float2(0.0f, 0.0f);
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        s1[0] += v[u].x;
                        s2[0] += v[u].y;
                    }
                }
            }
            __syncthreads();
            slots_sum<1, kThreads>(lds, threadIdx.x, row, rows, cols, s1, s2);
            if (on && row == 0) {
                const float w = a.weight != nullptr ? a.weight[c] : 1.0f;
                sums[b * a.channels + c] = make_float2(s1[0], s2[0]);
                m1 = fmaf(w, s1[0], m1);
                m2 = fmaf(w, s2[0], m2);
            }
        }
        m1 = block_sum<kThreads>(m1, red);
        m2 = block_sum<kThreads>(m2, red);
        if (threadIdx.x == 0) {
            const float count = (float)a.pixels * (float)per_group;
            means[at] = make_float2(m1 / count, m2 / count);
        }
    }
}

// dweight and dbias of channel c: its sums over a few images.
__device__ __forceinline__ void grad_params(const NormArgs& a, const float2* sums, int c) {
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
// The same of many: a share of the images a workgroup, whose slots take 8 at a time; sums
// in a tree, so that their error does not grow with the images. Into out (shares,
// channels) for a second such launch, or (null) to the gradients.
__global__ __launch_bounds__(kThreads) void k_norm_grad_params(NormArgs a, const float2* sums,
                                                               int64_t images, int64_t share,
                                                               float2* out) {
    __shared__ float2 lds[kThreads];
    constexpr int U = 8;
    const int c0 = blockIdx.y * kThreads, cols = min(kThreads, a.channels - c0);
    const int slots = kThreads / cols, slot = threadIdx.x / cols;
    const int c = c0 + (int)threadIdx.x % cols;
    const int64_t b0 = blockIdx.x * share, b1 = min(images, b0 + share);
    float s1[1] = {0.0f}, s2[1] = {0.0f};
    if (slot < slots)
        for (int64_t b = b0 + slot; b < b1; b += U * slots) {
            float2 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u] = b + u * slots < b1 ? sums[(b + u * slots) * a.channels + c]
                                          : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int o = U / 2; o > 0; o /= 2)
#pragma unroll
                for (int u = 0; u < o; ++u) {
                    v[u].x += v[u + o].x;
                    v[u].y += v[u + o].y;
                }
            s1[0] += v[0].x;
            s2[0] += v[0].y;
        }
    slots_sum<1, kThreads>(lds, threadIdx.x, slot, slots, cols, s1, s2);
    if (slot != 0) return;
    if (out != nullptr) {
        out[(int64_t)blockIdx.x * a.channels + c] = make_float2(s1[0], s2[0]);
        return;
    }
    if (a.dbias != nullptr) a.dbias[c] = s1[0];
    if (a.dweight != nullptr) a.dweight[c] = s2[0];
}
// One launch for some hundred images; two, with 32 images a share or 1024 shares, past
// that. `part` holds (1024, channels). The gradient of 100000 images of one pixel and 512
// channels takes 5.2 ms, 44.5 with one thread a channel.
hipError_t launch_grad_params(const NormArgs& a, const float2* sums, int64_t images, float2* part,
                              hipStream_t st) {
    const unsigned cols = (unsigned)((a.channels + kThreads - 1) / kThreads);
    if (images > 256) {
        const int64_t share = (images + 1023) / 1024 > 32 ? (images + 1023) / 1024 : 32;
        const int64_t shares = (images + share - 1) / share;
        k_norm_grad_params<<<dim3((unsigned)shares, cols), kThreads, 0, st>>>(a, sums, images,
                                                                              share, part);
        GS_LAUNCHED();
        sums = part;
        images = shares;
    }
    k_norm_grad_params<<<dim3(1, cols), kThreads, 0, st>>>(a, sums, images, images, nullptr);
    return hipGetLastError();
}

// dx = rstd w dz - rstd m1 - xh rstd m2. Bound as the sums are: 333666 x 48 fp32 relu
// 31 us, 6.1 TB/s read and written; 614400 x 128 bf16 gelu 83 us, 5.7 TB/s, vector units
// busy 74 %.
template <int ACT, int VEC>
__device__ __forceinline__ void grad_of(const Channels<VEC>& ch, const float* rw, const float* m1,
                                        const float* m2, float* v, const float* d) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float xh = ch.xh(v[j], j);
        const float dz = d[j] * act_slope<ACT>(ch.z(xh, j));
        v[j] = fmaf(-xh, m2[j], fmaf(rw[j], dz, -m1[j]));
    }
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void k_norm_grad_apply(NormArgs a, int chunks,
                                                              const float2* means,
                                                              const float2* sums) {
    constexpr int AHEAD = kAhead / 2;
    // with few images the parameters' gradients need no launch of their own
    if (sums != nullptr && blockIdx.y == 0)
        for (int c = blockIdx.x * kThreads + threadIdx.x; c < a.channels; c += gridDim.x * kThreads)
            grad_params(a, sums, c);
    const Place p = place_of<VEC>(a.pixels, a.channels, chunks);
    if (!p.on) return;
    const Channels<VEC> ch(a, p.b, p.c);
    float rw[VEC], m1[VEC], m2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float2 m = means[p.b * a.groups + (p.c + j) / (a.channels / a.groups)];
        rw[j] = ch.r[j] * ch.w[j];
        m1[j] = ch.r[j] * m.x;
        m2[j] = ch.r[j] * m.y;
    }
    const T* x = static_cast<const T*>(a.x) + p.b * a.x_batch + p.c;
    const T* dy = static_cast<const T*>(a.dy) + p.b * a.dy_batch + p.c;
    T* dx = static_cast<T*>(a.dx) + p.b * a.dx_batch + p.c;
    int64_t q = p.p0 + p.slot;
    for (; q + (AHEAD - 1) * p.slots < p.p1; q += AHEAD * p.slots) {
        float v[AHEAD][VEC], d[AHEAD][VEC];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            load_vec<VEC>(x + (q + k * p.slots) * a.x_pixel, v[k]);
            load_vec<VEC>(dy + (q + k * p.slots) * a.dy_pixel, d[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            grad_of<ACT, VEC>(ch, rw, m1, m2, v[k], d[k]);
            store_nt<VEC>(dx + (q + k * p.slots) * a.dx_pixel, v[k]);
        }
    }
    for (; q < p.p1; q += p.slots) {
        float v[VEC], d[VEC];
        load_vec<VEC>(x + q * a.x_pixel, v);
        load_vec<VEC>(dy + q * a.dy_pixel, d);
        grad_of<ACT, VEC>(ch, rw, m1, m2, v, d);
        store_vec<VEC>(dx + q * a.dx_pixel, v);
    }
}

// ---------------------------------------------------------------- small groups
// A group of an image that fits one workgroup's registers: one workgroup per (image,
// group) reads it once, in one launch. Bound by latency: 4800 x 32 fp32 in 8 groups 9
// us, 15 with the call; by the three launches above 20.
constexpr int kSmallThreads = 1024;
// Vectors of a thread: 32 values, or 4 single ones where a group's channels do
// not make vectors.
template <int VEC>
constexpr int kSmallVectors = VEC > 1 ? 32 / VEC : 4;

struct SmallPlace {
    int cols, slots, slot, c;
    bool on;
};
template <int VEC>
__device__ __forceinline__ SmallPlace small_place(int per_group) {
    SmallPlace p;
    p.cols = per_group / VEC;
    p.slots = kSmallThreads / p.cols;
    p.slot = threadIdx.x / p.cols;
    p.c = (blockIdx.x * p.cols + (int)threadIdx.x % p.cols) * VEC;
    p.on = p.slot < p.slots;
    return p;
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kSmallThreads) void k_norm_small(NormArgs a) {
    constexpr int K = kSmallVectors<VEC>;
    __shared__ float red[kSmallThreads / 64];
    const int per_group = a.channels / a.groups;
    const SmallPlace p = small_place<VEC>(per_group);
    const int64_t b = blockIdx.y;
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch + p.c;
    const int pixels = (int)a.pixels;
    float v[K][VEC], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int q = p.slot + k * p.slots;
        if (p.on && q < pixels) load_vec<VEC>(x + q * a.x_pixel, v[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (p.on && p.slot + k * p.slots < pixels)
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum += v[k][j];
    const float count = (float)pixels * (float)per_group;
    const float mean = block_sum<kSmallThreads>(sum, red) / count;
    float m2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (p.on && p.slot + k * p.slots < pixels)
#pragma unroll
            for (int j = 0; j < VEC; ++j) m2 = fmaf(v[k][j] - mean, v[k][j] - mean, m2);
    const float rstd = 1.0f / sqrtf(block_sum<kSmallThreads>(m2, red) / count + a.eps);
    if (threadIdx.x == 0) {
        a.mean[b * a.groups + blockIdx.x] = mean;
        a.rstd[b * a.groups + blockIdx.x] = rstd;
    }
    if (!p.on) return;
    float w[VEC], bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        w[j] = a.weight != nullptr ? a.weight[p.c + j] : 1.0f;
        bias[j] = a.bias != nullptr ? a.bias[p.c + j] : 0.0f;
    }
    T* y = static_cast<T*>(a.y) + b * a.y_batch + p.c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int q = p.slot + k * p.slots;
        if (q < pixels) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                v[k][j] = act<ACT>(fmaf((v[k][j] - mean) * rstd, w[j], bias[j]));
            store_vec<VEC>(y + q * a.y_pixel, v[k]);
        }
    }
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kSmallThreads) void k_norm_small_grad(NormArgs a, float2* sums) {
    constexpr int K = kSmallVectors<VEC>;
    __shared__ float2 lds[kSmallThreads * VEC];
    __shared__ float red[kSmallThreads / 64];
    const int per_group = a.channels / a.groups;
    const SmallPlace p = small_place<VEC>(per_group);
    const int64_t b = blockIdx.y;
    const int pixels = (int)a.pixels;
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch + p.c;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch + p.c;
    float v[K][VEC], d[K][VEC], s1[VEC], s2[VEC], w[VEC], bias[VEC];
    const float mean = a.mean[b * a.groups + blockIdx.x], rstd = a.rstd[b * a.groups + blockIdx.x];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        s1[j] = s2[j] = 0.0f;
        w[j] = a.weight != nullptr && p.on ? a.weight[p.c + j] : 1.0f;
        bias[j] = a.bias != nullptr && p.on ? a.bias[p.c + j] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int q = p.slot + k * p.slots;
        if (p.on && q < pixels) {
            load_vec<VEC>(x + q * a.x_pixel, v[k]);
            load_vec<VEC>(dy + q * a.dy_pixel, d[k]);
        }
    }
    // v and d become xh and dz
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (p.on && p.slot + k * p.slots < pixels)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[k][j] = (v[k][j] - mean) * rstd;
                d[k][j] *= act_slope<ACT>(fmaf(v[k][j], w[j], bias[j]));
                s1[j] += d[k][j];
                s2[j] = fmaf(d[k][j], v[k][j], s2[j]);
            }
    slots_sum<VEC, kSmallThreads>(lds, threadIdx.x, p.slot, p.slots, p.cols, s1, s2);
    float m1 = 0.0f, m2 = 0.0f;
    if (p.slot == 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            m1 = fmaf(w[j], s1[j], m1);
            m2 = fmaf(w[j], s2[j], m2);
            if (a.batch > 1) {
                sums[b * a.channels + p.c + j] = make_float2(s1[j], s2[j]);
            } else {
                if (a.dbias != nullptr) a.dbias[p.c + j] = s1[j];
                if (a.dweight != nullptr) a.dweight[p.c + j] = s2[j];
            }
        }
    const float count = (float)pixels * (float)per_group;
    m1 = block_sum<kSmallThreads>(m1, red) / count;
    m2 = block_sum<kSmallThreads>(m2, red) / count;
    if (!p.on) return;
    T* dx = static_cast<T*>(a.dx) + b * a.dx_batch + p.c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int q = p.slot + k * p.slots;
        if (q < pixels) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                v[k][j] = rstd * (fmaf(w[j], d[k][j], -m1) - v[k][j] * m2);
            store_vec<VEC>(dx + q * a.dx_pixel, v[k]);
        }
    }
}

// Chunks of an image's pixels: four workgroups a compute unit, at least 64 pixels each.
constexpr int kGroups = 1024;
int chunks_of(int64_t batch, int64_t pixels) {
    int64_t k = (kGroups + batch - 1) / batch;
    if (k > (pixels + 63) / 64) k = (pixels + 63) / 64;
    return k < 1 ? 1 : (int)k;
}

// Images whose sums k_norm_grad_apply adds in passing; of more launch_grad_params does,
// with launches of its own (2 images of 166833 x 48: 106 against 104 us for both passes, 8 of
// 76800 x 128 257 against 254).
constexpr int64_t kFewImages = 16;

struct NormWs {
    float2 *part, *sums, *means;
    size_t bytes;
    NormWs(void* base, int64_t batch, int channels) {
        Carve c(base);
        part = c.take<float2>((size_t)(kGroups + batch) * channels);  // at least batch * chunks
        sums = c.take<float2>((size_t)batch * channels);
        means = c.take<float2>((size_t)batch * channels);
        bytes = c.bytes();
    }
};

// Whether a group is one workgroup's work: it fits the registers in whole vectors
// (or is so small that reading by single values costs nothing).
template <int VEC>
bool small_group(const NormArgs& a) {
    const int per_group = a.channels / a.groups;
    if (a.batch > 65535 || per_group % VEC != 0 || per_group / VEC > kSmallThreads) return false;
    return a.pixels <= kSmallThreads / (per_group / VEC) * kSmallVectors<VEC>;
}

template <typename T, int VEC, int ACT>
hipError_t norm_run(const NormArgs& a, bool grad, hipStream_t st) {
    const NormWs w(a.ws, a.batch, a.channels);
    const int chunks = chunks_of(a.batch, a.pixels);
    const int cols = (a.channels + VEC - 1) / VEC;
    if (small_group<VEC>(a)) {
        const dim3 small((unsigned)a.groups, (unsigned)a.batch);
        if (!grad) {
            k_norm_small<T, VEC, ACT><<<small, kSmallThreads, 0, st>>>(a);
        } else {
            k_norm_small_grad<T, VEC, ACT><<<small, kSmallThreads, 0, st>>>(a, w.sums);
            GS_LAUNCHED();
            if (a.batch > 1) return launch_grad_params(a, w.sums, a.batch, w.part, st);
        }
        return hipGetLastError();
    }
    const dim3 grid((unsigned)(chunks * a.batch), (unsigned)((cols + kThreads - 1) / kThreads));
    const unsigned groups = blocks_of(a.batch * a.groups, 1);
    if (!grad) {
        k_norm_stats<T, VEC><<<grid, kThreads, 0, st>>>(a, chunks, w.part);
        GS_LAUNCHED();
        k_norm_finish<<<groups, kThreads, 0, st>>>(a, chunks, w.part);
        GS_LAUNCHED();
        k_norm_apply<T, VEC, ACT><<<grid, kThreads, 0, st>>>(a, chunks);
    } else {
        k_norm_grad_sums<T, VEC, ACT><<<grid, kThreads, 0, st>>>(a, chunks, w.part);
        GS_LAUNCHED();
        k_norm_grad_finish<<<groups, kThreads, 0, st>>>(a, chunks, w.part, w.sums, w.means);
        GS_LAUNCHED();
        if (a.batch > kFewImages) {
            const hipError_t e = launch_grad_params(a, w.sums, a.batch, w.part, st);
            if (e != hipSuccess) return e;
        }
        k_norm_grad_apply<T, VEC, ACT><<<grid, kThreads, 0, st>>>(
            a, chunks, w.means, a.batch > kFewImages ? nullptr : w.sums);
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
    // groups that make no vectors, but are small enough, still go in one launch
    if (vec && (small_group<VEC>(a) || !small_group<1>(a))) return norm_act<T, VEC>(a, grad, st);
    return norm_act<T, 1>(a, grad, st);
}

}  // namespace

size_t group_norm_ws(int64_t batch, int channels) {
    return NormWs(nullptr, batch, channels).bytes;
}

hipError_t launch_group_norm(const NormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.pixels == 0) return hipSuccess;
    return a.dtype == 0 ? norm_typed<float>(a, false, st) : norm_typed<bf16>(a, false, st);
}

hipError_t launch_group_norm_grad(const NormArgs& a, hipStream_t st) {
    if (a.batch == 0 || a.pixels == 0) {
        // no pixels: the parameters' gradients are 0
        return launch_grad_params(a, nullptr, 0, nullptr, st);
    }
    return a.dtype == 0 ? norm_typed<float>(a, true, st) : norm_typed<bf16>(a, true, st);
}

}  // namespace gs
