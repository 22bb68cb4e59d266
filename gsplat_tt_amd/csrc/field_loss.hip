// field_loss.hip - softmax cross entropy of features against a table of labels,
// with its gradients, without ever holding the (n, rows) scores.
//
//   l_iv = scale <feat_i, table_v>;  lse_i = log sum_v exp l_iv
//   loss_i = lse_i - l_i,label(i)      (0 for a masked row, label < 0)
//   G_iv = weight_i scale (exp(l_iv - lse_i) - [v = label(i)])
//   dfeat = G table;  dtable = G^T feat
//
// All products run on the matrix cores with bf16 operands and fp32 sums. fp32
// inputs are cut into three bf16 parts of 8 bits each (exact: 24 bits) and the
// six products whose weight is above 2^-24 are added up, which keeps fp32's
// precision at 6/16 of the cost of the fp32 matrix instructions.
//
// Operands are first laid out with the summed index contiguous and padded to
// the tiles, rows that a mask leaves out zeroed. The gradients go in pieces of
// rows and of the table, G of one piece at a time in the workspace.
#include <algorithm>

#include "field.h"

#include "field_device.h"

namespace gs {

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int kThreads = 256;
constexpr int kTile = 128;  // rows and columns of a workgroup's tile
constexpr int kStep = 64;   // summed index per step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Part p of a value: the leading 8 significant bits, the next 8, the rest.
// Cutting off (not rounding) leaves exact remainders; a value that is not
// finite stays whole in part 0.
__device__ __forceinline__ float cut_bf16(float v) {
    return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
}
template <int NP>
__device__ __forceinline__ void split(float v, bf16* out) {
    if (NP == 1) {
        out[0] = (bf16)v;
    } else {
        const float a = cut_bf16(v);
        float r = v - a;
        if (!(fabsf(v) <= 3.402823466e38f)) r = 0.0f;
        const float b = cut_bf16(r), c = cut_bf16(r - b);
        out[0] = (v != v) ? (bf16)v : (bf16)a;
        out[1] = (bf16)b;
        out[2] = (bf16)c;
    }
}
// The products of parts: (0,0) for one part; for three, all with p + q <= 2.
template <int NP>
struct Products;
template <>
struct Products<1> {
    static constexpr int kCount = 1;
    __device__ static int a(int) { return 0; }
    __device__ static int b(int) { return 0; }
};
template <>
struct Products<3> {
    static constexpr int kCount = 6;
    // (2,0) (1,1) (0,2) (1,0) (0,1) (0,0): the small ones first
    __device__ static int a(int i) { return (0x001012 >> (4 * i)) & 3; }
    __device__ static int b(int i) { return (0x010210 >> (4 * i)) & 3; }
};

// ---------------------------------------------------------------- layout
// Labels as 32-bit (-1: masked) with their weights; rows past n are masked.
__global__ __launch_bounds__(kThreads) void k_loss_rows(LossArgs a, int64_t padded, int32_t* label,
                                                        float* weight) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= padded) return;
    const int32_t l = i < a.n ? load_id(a.labels, a.labels64, i, a.rows, a.flags) : -1;
    label[i] = l;
    if (weight != nullptr)
        weight[i] = l < 0 ? 0.0f : a.scale * (a.row_weight != nullptr ? a.row_weight[i] : 1.0f);
}

// Parts of (rows, dim) as (padded, kd), zeros in the padding and masked rows.
template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void k_parts(const T* src, int64_t rows, int64_t stride,
                                                    int dim, const int32_t* label, int64_t padded,
                                                    int kd, bf16* out) {
    const int64_t total = padded * kd;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t r = e / kd;
        const int c = (int)(e - r * kd);
        float v = 0.0f;
        if (r < rows && c < dim && (label == nullptr || label[r] >= 0))
            v = to_float(src[r * stride + c]);
        bf16 part[NP];
        split<NP>(v, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) out[p * total + e] = part[p];
    }
}

// The same transposed: (dq, padded), dq >= dim a multiple of the tile.
template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void k_parts_t(const T* src, int64_t rows, int64_t stride,
                                                      int dim, const int32_t* label, int64_t padded,
                                                      int dq, bf16* out) {
    __shared__ float tile[32][33];
    const int64_t r0 = (int64_t)blockIdx.x * 32;
    const int c0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int k = ty; k < 32; k += 8) {
        const int64_t r = r0 + k;
        const int c = c0 + tx;
        float v = 0.0f;
        if (r < rows && c < dim && (label == nullptr || label[r] >= 0))
            v = to_float(src[r * stride + c]);
        tile[k][tx] = v;
    }
    __syncthreads();
    for (int k = ty; k < 32; k += 8) {
        bf16 part[NP];
        split<NP>(tile[tx][k], part);
#pragma unroll
        for (int p = 0; p < NP; ++p)
            out[(size_t)p * dq * padded + (size_t)(c0 + k) * padded + r0 + tx] = part[p];
    }
}

// ---------------------------------------------------------------- products
struct Mat {
    const bf16* p;
    int64_t ld, plane;  // elements between rows and between parts
};

// acc += A[m0.., k0..k1) B[n0.., k0..k1)^T for a 128 x 128 tile, 4 waves of
// 64 x 64. Rows of 64 bf16 (128 bytes) in LDS; a row's 16-byte pieces are
// placed by (piece ^ row % 8), so that 8 lanes reading one column of pieces
// touch all banks once.
template <int NP>
__device__ __forceinline__ void tile_product(const Mat& A, const Mat& B, int64_t m0, int64_t n0,
                                             int64_t k0, int64_t k1, uint4 (*lds)[2][kTile * 8],
                                             f32x4 acc[4][4]) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const int steps_k = (int)((k1 - k0) / kStep);
    const int steps = steps_k * Products<NP>::kCount;
    uint4 ra[4], rb[4];
    auto fetch = [&](int s) {
        const int q = s / steps_k;
        const int64_t k = k0 + (int64_t)(s - q * steps_k) * kStep;
        const bf16* pa = A.p + Products<NP>::a(q) * A.plane + m0 * A.ld + k;
        const bf16* pb = B.p + Products<NP>::b(q) * B.plane + n0 * B.ld + k;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = t + j * kThreads, r = e >> 3, c = e & 7;
            ra[j] = *reinterpret_cast<const uint4*>(pa + r * A.ld + c * 8);
            rb[j] = *reinterpret_cast<const uint4*>(pb + r * B.ld + c * 8);
        }
    };
    auto keep = [&](int buf) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = t + j * kThreads, r = e >> 3, c = e & 7;
            lds[buf][0][r * 8 + (c ^ (r & 7))] = ra[j];
            lds[buf][1][r * 8 + (c ^ (r & 7))] = rb[j];
        }
    };
    if (steps == 0) return;
    fetch(0);
    keep(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        if (s + 1 < steps) fetch(s + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = h * 4 + (lane >> 4);
                const int r = wm + i * 16 + (lane & 15), n = wn + i * 16 + (lane & 15);
                fa[i] = lds[buf][0][r * 8 + (c ^ (r & 7))];
                fb[i] = lds[buf][1][n * 8 + (c ^ (n & 7))];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, fa[i]), __builtin_bit_cast(bf16x8, fb[j]),
                        acc[i][j], 0, 0, 0);
        }
        if (s + 1 < steps) keep(buf ^ 1);
        __syncthreads();
    }
}

#define GS_TILE_LDS __shared__ uint4 lds[2][2][kTile * 8]
#define GS_TILE_ACC                    \
    f32x4 acc[4][4];                   \
    for (int i = 0; i < 4; ++i)        \
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}

// Per (64 columns, row): largest score and sum of exp2(score - largest), scores
// in log2 units; and the label's own score. A largest that is not finite is
// taken as 0, so that infinite scores give infinite sums.
template <int NP>
__global__ __launch_bounds__(kThreads) void k_loss_scores(Mat F, Mat T, int kd, int64_t rows,
                                                          float scale2, const int32_t* label,
                                                          int64_t padded, float2* part,
                                                          float* label_score) {
    GS_TILE_LDS;
    GS_TILE_ACC;
    const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
    tile_product<NP>(F, T, m0, n0, 0, kd, lds, acc);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = m0 + wm + i * 16 + (lane >> 4) * 4 + j;
            const int32_t y = label[r];
            float s[4], m = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t v = n0 + wn + k * 16 + (lane & 15);
                s[k] = v < rows ? acc[i][k][j] * scale2 : -INFINITY;
                if (v == y) label_score[r] = s[k];
                m = fmaxf(m, s[k]);
            }
            for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            const float base = fabsf(m) < INFINITY ? m : 0.0f;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += exp2f(s[k] - base);
            for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o, 64);
            if ((lane & 15) == 0)
                part[((int64_t)blockIdx.y * 2 + (w & 1)) * padded + r] = make_float2(m, sum);
        }
}

// Joins a row's partials; lse2 is kept in log2 units for the gradients.
__global__ __launch_bounds__(kThreads) void k_loss_join(LossArgs a, const float2* part, int parts,
                                                        int64_t padded, const int32_t* label,
                                                        const float* label_score, float* lse2) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= padded) return;
    float m = -INFINITY;
    for (int k = 0; k < parts; ++k) m = fmaxf(m, part[k * padded + i].x);
    const float base = fabsf(m) < INFINITY ? m : 0.0f;
    float sum = 0.0f;
    for (int k = 0; k < parts; ++k) {
        const float2 p = part[k * padded + i];
        sum += p.y * exp2f((fabsf(p.x) < INFINITY ? p.x : 0.0f) - base);
    }
    const float l = base + log2f(sum);
    const bool on = label[i] >= 0;
    if (lse2 != nullptr) lse2[i] = on ? l : 0.0f;
    if (i < a.n) {
        if (a.loss != nullptr) a.loss[i] = on ? (l - label_score[i]) * kLn2 : 0.0f;
        if (a.lse != nullptr) a.lse[i] = on ? l * kLn2 : 0.0f;
    }
}

// G of one piece (rows r0.., table rows v0..) and its transpose, in parts.
template <int NP>
__global__ __launch_bounds__(kThreads) void k_loss_g(Mat F, Mat T, int kd, int64_t rows,
                                                     float scale2, const int32_t* label,
                                                     const float* weight, const float* lse2,
                                                     int64_t r0, int64_t v0, int64_t rc, int64_t vc,
                                                     bf16* G, bf16* GT) {
    GS_TILE_LDS;
    GS_TILE_ACC;
    const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
    tile_product<NP>(F, T, r0 + m0, v0 + n0, 0, kd, lds, acc);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t rl = m0 + wm + i * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t vl = n0 + wn + k * 16 + (lane & 15);
            bf16 g[4][NP];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t r = r0 + rl + j;
                const int32_t y = label[r];
                float v = 0.0f;
                if (y >= 0 && v0 + vl < rows)
                    v = weight[r] * (exp2f(acc[i][k][j] * scale2 - lse2[r]) -
                                     (v0 + vl == y ? 1.0f : 0.0f));
                split<NP>(v, g[j]);
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                VecOf<bf16, 4> u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u.v[j] = g[j][p];
                    G[p * rc * vc + (rl + j) * vc + vl] = g[j][p];
                }
                *reinterpret_cast<VecOf<bf16, 4>*>(GT + p * rc * vc + vl * rc + rl) = u;
            }
        }
    }
}

// slices[z] (m, dq) = A B^T over the z-th share of the summed index.
template <int NP>
__global__ __launch_bounds__(kThreads) void k_loss_sum(Mat A, Mat B, int64_t k, int64_t share,
                                                       int64_t m, int dq, float* slices) {
    GS_TILE_LDS;
    GS_TILE_ACC;
    const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
    const int64_t k0 = min(k, share * blockIdx.z), k1 = min(k, k0 + share);
    tile_product<NP>(A, B, m0, n0, k0, k1, lds, acc);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    float* out = slices + (size_t)blockIdx.z * m * dq;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                out[(m0 + wm + i * 16 + (lane >> 4) * 4 + j) * dq + n0 + wn + n * 16 + (lane & 15)] =
                    acc[i][n][j];
}

// Adds the slices in order (and the earlier pieces' sum), and rounds the last
// sum into the caller's rows; masked rows get zeros.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_loss_fold(const float* slices, int nz, int64_t m,
                                                        int dq, float* sum, int first, int last,
                                                        T* out, int64_t rows, int64_t stride,
                                                        int dim, const int32_t* label) {
    const int64_t total = m * dq;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        float s = first ? 0.0f : sum[e];
        for (int z = 0; z < nz; ++z) s += slices[(size_t)z * total + e];
        if (!last) {
            sum[e] = s;
            continue;
        }
        const int64_t r = e / dq;
        const int c = (int)(e - r * dq);
        if (r < rows && c < dim)
            out[r * stride + c] = from_float<T>(label != nullptr && label[r] < 0 ? 0.0f : s);
    }
}

// ---------------------------------------------------------------- pieces
int64_t pad_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Pieces of G: up to 8192 table rows by as many rows as make 2^26 values
// (128 MB and as much for the transpose), which the cache behind the L2s holds.
struct LossPlan {
    int np, kd, dq;
    int64_t np_rows, vp, rc, vc;
    int zf, zt;  // shares of the summed index: for dfeat and for dtable
    int64_t share_f, share_t;
    bf16 *F, *T, *FT, *TT, *G, *GT;
    float2* part;
    float *score, *lse2, *weight, *slices, *sum_f, *sum_t;
    int32_t* label;
    size_t bytes;

    static void shares(int64_t tiles, int64_t k, int* z, int64_t* share) {
        int64_t want = tiles >= 512 ? 1 : (512 + tiles - 1) / tiles;
        want = std::min<int64_t>(want, std::max<int64_t>(1, k / 512));
        *share = pad_to((k + want - 1) / want, kStep);
        *z = (int)((k + *share - 1) / *share);
    }
    LossPlan(void* base, int64_t n, int64_t rows, int dim, int dtype, bool grad) {
        np = dtype == 0 ? 3 : 1;
        kd = (int)pad_to(dim, kStep);
        dq = (int)pad_to(dim, kTile);
        np_rows = pad_to(n, kTile);
        vp = pad_to(rows, kTile);
        vc = std::min<int64_t>(vp, 8192);
        rc = std::min<int64_t>(np_rows, std::max<int64_t>(kTile, ((1 << 26) / np / vc) / kTile * kTile));
        shares(rc / kTile * (dq / kTile), vc, &zf, &share_f);
        shares(vc / kTile * (dq / kTile), rc, &zt, &share_t);
        Carve c(base);
        F = c.take<bf16>((size_t)np * np_rows * kd);
        T = c.take<bf16>((size_t)np * vp * kd);
        part = c.take<float2>((size_t)(vp / 64) * np_rows);
        score = c.take<float>((size_t)np_rows);
        label = c.take<int32_t>((size_t)np_rows);
        FT = TT = G = GT = nullptr;
        lse2 = weight = slices = sum_f = sum_t = nullptr;
        if (grad) {
            FT = c.take<bf16>((size_t)np * np_rows * dq);
            TT = c.take<bf16>((size_t)np * vp * dq);
            lse2 = c.take<float>((size_t)np_rows);
            weight = c.take<float>((size_t)np_rows);
            G = c.take<bf16>((size_t)np * rc * vc);
            GT = c.take<bf16>((size_t)np * rc * vc);
            slices = c.take<float>(std::max((size_t)zf * rc * dq, (size_t)zt * vc * dq));
            sum_f = c.take<float>((size_t)rc * dq);
            sum_t = c.take<float>((size_t)vp * dq);
        }
        bytes = c.bytes();
    }
};

unsigned blocks_for(int64_t items) {
    const int64_t b = (items + kThreads - 1) / kThreads;
    return (unsigned)(b < 65536 ? b : 65536);
}

template <typename T, int NP>
hipError_t loss_run(const LossArgs& a, bool grad, hipStream_t st) {
    const LossPlan w(a.ws, a.n, a.rows, a.dim, a.dtype, grad);
    const int64_t nr = w.np_rows;
    const T* feat = static_cast<const T*>(a.feat);
    const T* table = static_cast<const T*>(a.table);
    const float scale2 = a.scale * kLog2e;
    k_loss_rows<<<(unsigned)((nr + kThreads - 1) / kThreads), kThreads, 0, st>>>(a, nr, w.label,
                                                                                 w.weight);
    k_parts<T, NP><<<blocks_for(nr * w.kd), kThreads, 0, st>>>(feat, a.n, a.feat_stride, a.dim,
                                                               w.label, nr, w.kd, w.F);
    k_parts<T, NP><<<blocks_for(w.vp * w.kd), kThreads, 0, st>>>(
        table, a.rows, a.table_stride, a.dim, nullptr, w.vp, w.kd, w.T);
    const Mat F{w.F, w.kd, nr * w.kd}, Tm{w.T, w.kd, w.vp * w.kd};
    const dim3 grid((unsigned)(nr / kTile), (unsigned)(w.vp / kTile));
    k_loss_scores<NP><<<grid, kThreads, 0, st>>>(F, Tm, w.kd, a.rows, scale2, w.label, nr, w.part,
                                                 w.score);
    k_loss_join<<<(unsigned)((nr + kThreads - 1) / kThreads), kThreads, 0, st>>>(
        a, w.part, (int)(w.vp / 64), nr, w.label, w.score, w.lse2);
    if (!grad) return hipGetLastError();
    k_parts_t<T, NP><<<dim3((unsigned)(nr / 32), (unsigned)(w.dq / 32)), kThreads, 0, st>>>(
        feat, a.n, a.feat_stride, a.dim, w.label, nr, w.dq, w.FT);
    k_parts_t<T, NP><<<dim3((unsigned)(w.vp / 32), (unsigned)(w.dq / 32)), kThreads, 0, st>>>(
        table, a.rows, a.table_stride, a.dim, nullptr, w.vp, w.dq, w.TT);
    for (int64_t r0 = 0; r0 < nr; r0 += w.rc) {
        const int64_t rc = std::min(w.rc, nr - r0);
        for (int64_t v0 = 0; v0 < w.vp; v0 += w.vc) {
            const int64_t vc = std::min(w.vc, w.vp - v0);
            k_loss_g<NP><<<dim3((unsigned)(rc / kTile), (unsigned)(vc / kTile)), kThreads, 0, st>>>(
                F, Tm, w.kd, a.rows, scale2, w.label, w.weight, w.lse2, r0, v0, rc, vc, w.G, w.GT);
            const int zf = (int)((vc + w.share_f - 1) / w.share_f);
            k_loss_sum<NP><<<dim3((unsigned)(rc / kTile), (unsigned)(w.dq / kTile), zf), kThreads,
                             0, st>>>({w.G, vc, rc * vc}, {w.TT + v0, w.vp, w.dq * w.vp}, vc,
                                      w.share_f, rc, w.dq, w.slices);
            k_loss_fold<T><<<blocks_for(rc * w.dq), kThreads, 0, st>>>(
                w.slices, zf, rc, w.dq, w.sum_f, v0 == 0, v0 + vc >= w.vp,
                static_cast<T*>(a.dfeat) + r0 * a.dfeat_stride, a.n - r0, a.dfeat_stride, a.dim,
                w.label + r0);
            const int zt = (int)((rc + w.share_t - 1) / w.share_t);
            k_loss_sum<NP><<<dim3((unsigned)(vc / kTile), (unsigned)(w.dq / kTile), zt), kThreads,
                             0, st>>>({w.GT, rc, rc * vc}, {w.FT + r0, nr, w.dq * nr}, rc,
                                      w.share_t, vc, w.dq, w.slices);
            k_loss_fold<T><<<blocks_for(vc * w.dq), kThreads, 0, st>>>(
                w.slices, zt, vc, w.dq, w.sum_t + v0 * w.dq, r0 == 0, r0 + rc >= nr,
                static_cast<T*>(a.dtable) + v0 * a.dtable_stride, a.rows - v0, a.dtable_stride,
                a.dim, nullptr);
        }
    }
    return hipGetLastError();
}

}  // namespace

size_t label_loss_ws(int64_t n, int64_t rows, int dim, int dtype, bool grad) {
    return LossPlan(nullptr, n, rows, dim, dtype, grad).bytes;
}

hipError_t launch_label_loss(const LossArgs& a, bool grad, hipStream_t st) {
    if (a.n == 0) {  // no rows: the table's gradient is 0
        if (!grad) return hipSuccess;
        const unsigned b = blocks_for(a.rows * a.dim);
        if (a.dtype == 0)
            k_loss_fold<float><<<b, kThreads, 0, st>>>(nullptr, 0, a.rows, a.dim, nullptr, 1, 1,
                                                       static_cast<float*>(a.dtable), a.rows,
                                                       a.dtable_stride, a.dim, nullptr);
        else
            k_loss_fold<bf16><<<b, kThreads, 0, st>>>(nullptr, 0, a.rows, a.dim, nullptr, 1, 1,
                                                      static_cast<bf16*>(a.dtable), a.rows,
                                                      a.dtable_stride, a.dim, nullptr);
        return hipGetLastError();
    }
    return a.dtype == 0 ? loss_run<float, 3>(a, grad, st) : loss_run<bf16, 1>(a, grad, st);
}

}  // namespace gs
