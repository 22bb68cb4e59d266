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
typedef __attribute__((ext_vector_type(4))) uint32_t quad;  // 16 bytes: one lane's operand

constexpr int kThreads = 256;
constexpr int kTile = 128;  // rows and columns of a workgroup's tile
constexpr int kStep = 64;   // summed index per step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Part p of a value: the leading 8 significant bits, the next 8, the rest.
// Cutting off (not rounding) leaves exact remainders.
__device__ __forceinline__ float cut_bf16(float v) {
    return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
}
// An input is made canonical first: one that is not finite has parts that are not.
template <int NP>
__device__ __forceinline__ float plain_input(float v) {
    if (NP > 1 && v != v) return __uint_as_float(0x7FC00000u);
    return v;
}
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
// Parts of two values, each pair in one word.
template <int NP>
__device__ __forceinline__ void split2(float v0, float v1, uint32_t* out) {
    if (NP == 1) {
        out[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v0, v1}, bf16x2));
    } else {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            // the high halves of both
            out[p] = __builtin_amdgcn_perm(__float_as_uint(v1), __float_as_uint(v0), 0x07060302u);
            v0 -= cut_bf16(v0);
            v1 -= cut_bf16(v1);
        }
    }
}
// Parts of eight values, as operands.
template <int NP>
__device__ __forceinline__ void split8(const float* v, quad* out) {
    uint32_t w[4][NP];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2<NP>(v[2 * k], v[2 * k + 1], w[k]);
#pragma unroll
    for (int p = 0; p < NP; ++p) out[p] = quad{w[0][p], w[1][p], w[2][p], w[3][p]};
}
template <int NP>
__device__ __forceinline__ void split(float v, bf16* out) {
    uint32_t w[NP];
    split2<NP>(v, 0.0f, w);
#pragma unroll
    for (int p = 0; p < NP; ++p) out[p] = __builtin_bit_cast(bf16x2, w[p])[0];
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
            v = plain_input<NP>(to_float(src[r * stride + c]));
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
            v = plain_input<NP>(to_float(src[r * stride + c]));
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
                                             int64_t k0, int64_t k1, quad (*lds)[2][kTile * 8],
                                             f32x4 acc[4][4]) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const int steps_k = (int)((k1 - k0) / kStep);
    const int steps = steps_k * Products<NP>::kCount;
    quad ra[4], rb[4];
    auto fetch = [&](int s) {
        const int q = s / steps_k;
        const int64_t k = k0 + (int64_t)(s - q * steps_k) * kStep;
        const bf16* pa = A.p + Products<NP>::a(q) * A.plane + m0 * A.ld + k;
        const bf16* pb = B.p + Products<NP>::b(q) * B.plane + n0 * B.ld + k;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = t + j * kThreads, r = e >> 3, c = e & 7;
            ra[j] = *reinterpret_cast<const quad*>(pa + r * A.ld + c * 8);
            rb[j] = *reinterpret_cast<const quad*>(pb + r * B.ld + c * 8);
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
            quad fa[4], fb[4];
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

#define GS_TILE_LDS __shared__ quad lds[2][2][kTile * 8]
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

// ---------------------------------------------------------------- streaming
// For rows short enough that a wave keeps its own in registers: a workgroup
// holds 4 x 64 "queries", the other side's rows ("keys") stream through LDS, 32
// a tile, and neither scores nor G ever leave the registers.
//
// The scores of a tile are made transposed, keys by queries: a lane then holds
// 16 keys' scores of one query, the sums over keys need no other lane until the
// end, and the same registers, as they are, are the left operand of the second
// product (queries by keys times keys by dim). The keys' order within that
// product is the lane's own: slot (h, e) of a half tile f is key
// 16 f + 4 h + e (e < 4) or 16 f + 4 h + 4 + e (e >= 4), h = lane / 32.
//
// Keys are laid out once as whole matrix-instruction operands (1 KB each, 16
// bytes a lane), so that LDS is filled and read in order: per tile the operands
// of the scores, [part][dim / 16], then those of the second product,
// [part][dim / 32][f].
typedef __attribute__((ext_vector_type(16))) float f32x16;

enum { kScores = 0, kGradFeat = 1, kGradTable = 2 };

struct StreamArgs {
    const void* q;  // queries (nq, dim)
    int64_t nq, q_stride;
    const quad* keys;  // tiles of 32 keys
    int64_t nk;         // keys that are there
    int tiles, share;   // tiles in all, and of a share
    int tile_stride;    // quad from tile to tile
    int dim;
    float scale2;  // scale * log2(e)
    // of the samples, whichever side they are: label, weight * scale, lse in log2 units
    const int32_t* label;
    const float *weight, *lse2;
    // kScores
    const void* labels;
    int labels64;
    float2* part;
    float *label_score, *loss, *lse, *lse2_out;
    uint32_t* flags;
    int64_t table_rows;
    // gradients: into out where there is one share, else into (share, padded, KD) sums
    void* out;
    int64_t out_stride;
    float* sums;
    int64_t padded;
};

// exp2 of a gradient's exponent. The bare instruction gives 0 below 2^-126, which
// fp32 gradients, times weight * scale, would show; for bf16 ones it is left so.
template <int NP>
__device__ __forceinline__ float grad_exp2(float x) {
    return NP == 1 ? __builtin_amdgcn_exp2f(x) : exp2f(x);
}

// Key of register r of a lane in half h.
__device__ __forceinline__ constexpr int key_of(int r) { return (r & 3) + 8 * (r >> 2); }

// A row's 8 values from column c, cut into parts; zeros past the row.
template <typename T, int NP>
__device__ __forceinline__ void load_parts(const T* row, int dim, int c, bool on, quad* out) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = on && c + e < dim ? plain_input<NP>(to_float(row[c + e])) : 0.0f;
    split8<NP>(v, out);
}

// (rows, dim) as tiles of operands, one workgroup a tile; of samples (label) the
// masked ones are zeros, and label and weight are written for the gradients.
template <typename T, int NP, int KD, bool SECOND>
__global__ __launch_bounds__(kThreads) void k_operands(const T* src, int64_t rows, int64_t stride,
                                                       int dim, LossArgs a, int32_t* label,
                                                       float* weight, float* lse2, quad* out) {
    __shared__ float tile[32][KD + 1];
    __shared__ int32_t lab[32];
    const int64_t r0 = (int64_t)blockIdx.x * 32;
    if (threadIdx.x < 32) {
        int32_t l = 0;
        if (label != nullptr) {
            const int64_t i = r0 + threadIdx.x;
            l = i < rows ? load_id(a.labels, a.labels64, i, a.rows, nullptr) : -1;
            label[i] = l;
            weight[i] = l < 0 ? 0.0f : a.scale * (a.row_weight != nullptr ? a.row_weight[i] : 1.0f);
            if (i >= rows) lse2[i] = 0.0f;  // the others' come from the scores
        }
        lab[threadIdx.x] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * KD; e += kThreads) {
        const int r = e / KD, c = e % KD;
        float v = 0.0f;
        if (r0 + r < rows && c < dim && lab[r] >= 0) v = plain_input<NP>(to_float(src[(r0 + r) * stride + c]));
        tile[r][c] = v;
    }
    __syncthreads();
    constexpr int kFirst = KD / 16 * 64, kSecond = SECOND ? KD / 32 * 2 * 64 : 0;
    quad* to = out + (size_t)blockIdx.x * NP * (kFirst + kSecond);
    for (int e = threadIdx.x; e < kFirst + kSecond; e += kThreads) {
        const int lane = e & 63, h = lane >> 5;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (e < kFirst) {
                v[k] = tile[lane & 31][(e >> 6) * 16 + 8 * h + k];
            } else {
                const int b = (e - kFirst) >> 6;  // dim / 32, f
                v[k] = tile[16 * (b & 1) + 4 * h + k + (k < 4 ? 0 : 4)][(b >> 1) * 32 + (lane & 31)];
            }
        }
        quad piece[NP];
        split8<NP>(v, piece);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const size_t at = e < kFirst ? p * kFirst + e : NP * kFirst + p * kSecond + (e - kFirst);
            to[at] = piece[p];
        }
    }
}

template <typename T, int NP, int KD, int ROLE>
struct StreamShape {
    static constexpr int kPieces = NP * KD / 16 * 64 * (ROLE == kScores ? 1 : 2);  // quad a tile
    // tiles per step: about 16 KB
    static constexpr int kTiles = kPieces * 16 >= 16384 ? 1 : (kPieces * 16 >= 8192 ? 2 : 4);
    static constexpr int kStage = kPieces * kTiles;
    static constexpr size_t kLds = 2 * kStage * 16 + (ROLE == kGradTable ? 2 * kTiles * 32 * 12 : 0);
};

template <typename T, int NP, int KD, int ROLE>
__global__ __launch_bounds__(kThreads, (NP * KD >= (ROLE == kScores ? 256 : 128) ? 1 : 2)) void k_stream(StreamArgs a) {
    using Shape = StreamShape<T, NP, KD, ROLE>;
    constexpr int KJ = KD / 16, DB = KD / 32, TS = Shape::kTiles, STAGE = Shape::kStage;
    constexpr int PER = STAGE / kThreads;
    static_assert(STAGE % kThreads == 0, "a stage is whole rounds of loads");
    extern __shared__ quad lds[];
    float* info = reinterpret_cast<float*>(lds + 2 * STAGE);  // kGradTable: lse2, weight, label
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5, col = lane & 31;
    const int64_t q0 = ((int64_t)blockIdx.x * 4 + (t >> 6)) * 64;

    // the wave's own queries, as right operands of the scores
    quad q[2][KJ][NP];
    int32_t y[2];
    float lse2[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int64_t i = q0 + b * 32 + col;
        bool on = i < a.nq;
        y[b] = -1;
        lse2[b] = 0.0f;
        if (ROLE == kScores) {
            if (on) y[b] = load_id(a.labels, a.labels64, i, a.table_rows,
                                   blockIdx.y == 0 && h == 0 ? a.flags : nullptr);
            on = y[b] >= 0;
        }
        if (ROLE == kGradFeat) {
            if (on) {
                y[b] = a.label[i];
                lse2[b] = a.lse2[i];
            }
            on = y[b] >= 0;
        }
        if (ROLE == kGradTable) y[b] = (int32_t)min(i, (int64_t)0x7FFFFFFF);
        const T* row = static_cast<const T*>(a.q) + i * a.q_stride;
#pragma unroll
        for (int j = 0; j < KJ; ++j) load_parts<T, NP>(row, a.dim, 16 * j + 8 * h, on, q[b][j]);
    }

    f32x16 acc[2][ROLE == kScores ? 1 : DB];
    float m[2], sum[2], own[2];
    if (ROLE == kScores) {
        m[0] = m[1] = -1e30f;
        sum[0] = sum[1] = own[0] = own[1] = 0.0f;
    } else {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[b][d][r] = 0.0f;
    }

    const int t0 = blockIdx.y * a.share, t1 = min(a.tiles, t0 + a.share);
    const int steps = (t1 - t0 + TS - 1) / TS;
    quad pre[PER];
    // a step past the last tile reads on into the padding behind the tiles
    auto fetch = [&](int s) {
        const quad* from = a.keys + ((size_t)t0 + (size_t)s * TS) * a.tile_stride;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int e = k * kThreads + t;
            pre[k] = from[(size_t)(e / Shape::kPieces) * a.tile_stride + e % Shape::kPieces];
        }
    };
    auto keep = [&](int s) {
        quad* to = lds + (s & 1) * STAGE + t;
#pragma unroll
        for (int k = 0; k < PER; ++k) to[k * kThreads] = pre[k];
        if (ROLE == kGradTable) {
            float* f = info + (s & 1) * TS * 96;
            for (int k = t; k < TS * 32; k += kThreads) {
                const int64_t i = ((int64_t)t0 + (int64_t)s * TS) * 32 + k;
                f[k] = a.lse2[i];
                f[TS * 32 + k] = a.weight[i];
                f[2 * TS * 32 + k] = __int_as_float(a.label[i]);
            }
        }
    };
    fetch(0);
    keep(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) fetch(s + 1);
        const quad* stage = lds + (s & 1) * STAGE;
#pragma unroll 1
        for (int u = 0; u < TS; ++u) {
            const int tile = t0 + s * TS + u;
            if (tile >= t1) break;
            const quad* kf = stage + u * Shape::kPieces + lane;
            f32x16 sc[2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[b][r] = 0.0f;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                bf16x8 k[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    k[p] = __builtin_bit_cast(bf16x8, kf[(p * KJ + j) * 64]);
#pragma unroll
                for (int i = 0; i < Products<NP>::kCount; ++i)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            k[Products<NP>::a(i)],
                            __builtin_bit_cast(bf16x8, q[b][j][Products<NP>::b(i)]), sc[b], 0, 0, 0);
            }
            const int64_t k0 = (int64_t)tile * 32;
            if (ROLE == kScores) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[b][r] *= a.scale2;
                    if (k0 + 32 > a.nk) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (k0 + key_of(r) + 4 * h >= a.nk) sc[b][r] = -INFINITY;
                    }
                    const int64_t yl = y[b] - k0;
                    if (__any(yl >= 0 && yl < 32)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (yl == key_of(r) + 4 * h) own[b] = sc[b][r];
                    }
                    float mt = m[b];
#pragma unroll
                    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[b][r]);
                    // an infinite largest counts as 0: the sum is infinite too then
                    const float base = mt < INFINITY ? mt : 0.0f;
                    const float was = m[b] < INFINITY ? m[b] : 0.0f;
                    float add = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        add += __builtin_amdgcn_exp2f(sc[b][r] - base);
                    sum[b] = sum[b] * __builtin_amdgcn_exp2f(was - base) + add;
                    m[b] = mt;
                }
                continue;
            }
            quad g[2][2][NP];
            const float* f = info + (s & 1) * TS * 96 + u * 32;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float v[16];
                if (ROLE == kGradFeat) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        v[r] = grad_exp2<NP>(fmaf(sc[b][r], a.scale2, -lse2[b]));
                    const int64_t yl = y[b] - k0;
                    if (__any(yl >= 0 && yl < 32)) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (yl == key_of(r) + 4 * h) v[r] -= 1.0f;
                    }
                } else {
                    const int yk = __float_as_int(f[2 * TS * 32 + col]);
                    const bool any = __any(yk >= q0 + b * 32 && yk < q0 + b * 32 + 32);
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const float4 l4 = *reinterpret_cast<const float4*>(f + g4 * 8 + 4 * h);
                        const float4 w4 =
                            *reinterpret_cast<const float4*>(f + TS * 32 + g4 * 8 + 4 * h);
                        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[g4 * 4 + e] =
                                grad_exp2<NP>(fmaf(sc[b][g4 * 4 + e], a.scale2, -l[e]));
                        if (any) {
                            const float4 y4 = *reinterpret_cast<const float4*>(
                                f + 2 * TS * 32 + g4 * 8 + 4 * h);
                            const float yy[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (__float_as_int(yy[e]) == y[b]) v[g4 * 4 + e] -= 1.0f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[g4 * 4 + e] *= w[e];
                    }
                }
                split8<NP>(v, g[b][0]);
                split8<NP>(v + 8, g[b][1]);
            }
            const quad* kt = kf + NP * KJ * 64;
#pragma unroll
            for (int d = 0; d < (ROLE == kScores ? 1 : DB); ++d)
#pragma unroll
                for (int f2 = 0; f2 < 2; ++f2) {
                    bf16x8 k[NP];
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        k[p] = __builtin_bit_cast(bf16x8, kt[(p * DB * 2 + d * 2 + f2) * 64]);
#pragma unroll
                    for (int i = 0; i < Products<NP>::kCount; ++i)
#pragma unroll
                        for (int b = 0; b < 2; ++b)
                            acc[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                __builtin_bit_cast(bf16x8, g[b][f2][Products<NP>::a(i)]),
                                k[Products<NP>::b(i)], acc[b][d], 0, 0, 0);
                }
        }
        if (s + 1 < steps) keep(s + 1);
        __syncthreads();
    }

    if (ROLE == kScores) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t i = q0 + b * 32 + col;
            const float m2 = __shfl_xor(m[b], 32, 64), s2 = __shfl_xor(sum[b], 32, 64);
            const float mm = fmaxf(m[b], m2), base = mm < INFINITY ? mm : 0.0f;
            const float total =
                sum[b] * __builtin_amdgcn_exp2f((m[b] < INFINITY ? m[b] : 0.0f) - base) +
                s2 * __builtin_amdgcn_exp2f((m2 < INFINITY ? m2 : 0.0f) - base);
            // the half that holds the label's score gives it to the other
            const bool here = y[b] >= 0 && ((y[b] >> 2) & 1) == h;
            const float o2 = __shfl_xor(own[b], 32, 64);
            const float mine = here ? own[b] : o2;
            if (h != 0 || i >= a.nq) continue;
            if (gridDim.y == 1) {
                const float l = base + log2f(total);
                const bool on = y[b] >= 0;
                if (a.loss != nullptr) a.loss[i] = on ? (l - mine) * kLn2 : 0.0f;
                if (a.lse != nullptr) a.lse[i] = on ? l * kLn2 : 0.0f;
                if (a.lse2_out != nullptr) a.lse2_out[i] = on ? l : 0.0f;
            } else {
                a.part[blockIdx.y * a.padded + i] = make_float2(mm, total);
                if (y[b] >= (int64_t)t0 * 32 && y[b] < (int64_t)t1 * 32) a.label_score[i] = mine;
            }
        }
        return;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t i = q0 + b * 32 + key_of(r) + 4 * h;
            if (i >= a.nq) continue;
            float w = 1.0f;
            bool on = true;
            if (ROLE == kGradFeat) {
                on = a.label[i] >= 0;
                w = a.weight[i];
            }
#pragma unroll
            for (int d = 0; d < (ROLE == kScores ? 1 : DB); ++d) {
                const int c = d * 32 + col;
                const float v = on ? acc[b][d][r] * w : 0.0f;
                if (gridDim.y > 1)
                    a.sums[((size_t)blockIdx.y * a.padded + i) * KD + c] = v;
                else if (c < a.dim)
                    static_cast<T*>(a.out)[i * a.out_stride + c] = from_float<T>(v);
            }
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

// Joins the shares' partials of a row's scores.
__global__ __launch_bounds__(kThreads) void k_stream_join(StreamArgs a, int shares) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.nq) return;
    const bool on = load_id(a.labels, a.labels64, i, a.table_rows, nullptr) >= 0;
    float m = -INFINITY;
    for (int k = 0; k < shares; ++k) m = fmaxf(m, a.part[k * a.padded + i].x);
    const float base = m < INFINITY ? m : 0.0f;
    float sum = 0.0f;
    for (int k = 0; k < shares; ++k) {
        const float2 p = a.part[k * a.padded + i];
        sum += p.y * __builtin_amdgcn_exp2f((p.x < INFINITY ? p.x : 0.0f) - base);
    }
    const float l = base + log2f(sum);
    if (a.loss != nullptr) a.loss[i] = on ? (l - a.label_score[i]) * kLn2 : 0.0f;
    if (a.lse != nullptr) a.lse[i] = on ? l * kLn2 : 0.0f;
    if (a.lse2_out != nullptr) a.lse2_out[i] = on ? l : 0.0f;
}

// Shares of the streamed side: enough workgroups for the chip (two a compute
// unit), at least `least` tiles each, at most `most` of them.
struct Shares {
    int count, tiles;
    Shares(int64_t queries, int64_t tiles_all, int least, int64_t most) {
        const int64_t groups = (queries + 255) / 256;
        int64_t want = groups >= 512 ? 1 : (512 + groups - 1) / std::max<int64_t>(groups, 1);
        want = std::min(want, std::max<int64_t>(1, tiles_all / least));
        want = std::max<int64_t>(1, std::min(want, most));
        tiles = (int)((tiles_all + want - 1) / want);
        count = (int)((tiles_all + tiles - 1) / tiles);
    }
};

// Workspace of the streaming kernels.
struct StreamPlan {
    int64_t tf, tt;  // tiles of the samples and of the table
    Shares scores, by_feat, by_table;
    quad *F, *T;
    int32_t* label;
    float *weight, *lse2, *score, *sums;
    float2* part;
    size_t bytes;
    // partial sums of the gradients: at most 64 MB a side
    static int64_t most(int64_t rows, int kd) {
        return std::max<int64_t>(1, ((int64_t)1 << 24) / std::max<int64_t>(1, rows * kd));
    }
    StreamPlan(void* base, int64_t n, int64_t rows, int np, int kd, bool grad)
        : tf((n + 31) / 32), tt((rows + 31) / 32), scores(n, tt, 4, 512),
          by_feat(n, tt, 8, most(n, kd)), by_table(rows, tf, 8, most(rows, kd)) {
        Carve c(base);
        const size_t first = (size_t)np * kd / 16 * 64, tile = grad ? 2 * first : first;
        T = c.take<quad>((tt + 4) * tile);
        part = c.take<float2>(scores.count > 1 ? (size_t)scores.count * n : 0);
        score = c.take<float>(scores.count > 1 ? (size_t)n : 0);
        F = nullptr;
        label = nullptr;
        weight = lse2 = sums = nullptr;
        if (grad) {
            F = c.take<quad>((tf + 4) * tile);
            label = c.take<int32_t>((tf + 4) * 32);
            weight = c.take<float>((tf + 4) * 32);
            lse2 = c.take<float>((tf + 4) * 32);
            const size_t sf = by_feat.count > 1 ? (size_t)by_feat.count * n * kd : 0;
            const size_t sr = by_table.count > 1 ? (size_t)by_table.count * rows * kd : 0;
            sums = c.take<float>(std::max(sf, sr));
        }
        bytes = c.bytes();
    }
};

template <typename T, int NP, int KD, int ROLE>
hipError_t launch_stream(const StreamArgs& a, const Shares& sh, hipStream_t st) {
    constexpr size_t lds = StreamShape<T, NP, KD, ROLE>::kLds;
    if (lds > 65536) {  // above the default limit of a launch
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void*>(&k_stream<T, NP, KD, ROLE>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    k_stream<T, NP, KD, ROLE>
        <<<dim3((unsigned)((a.nq + 255) / 256), (unsigned)sh.count), kThreads, lds, st>>>(a);
    return hipGetLastError();
}

template <typename T, int NP, int KD>
hipError_t stream_run(const LossArgs& a, bool grad, hipStream_t st) {
    const StreamPlan w(a.ws, a.n, a.rows, NP, KD, grad);
    const T* feat = static_cast<const T*>(a.feat);
    const T* table = static_cast<const T*>(a.table);
    if (grad)
        k_operands<T, NP, KD, true><<<(unsigned)w.tt, kThreads, 0, st>>>(
            table, a.rows, a.table_stride, a.dim, a, nullptr, nullptr, nullptr, w.T);
    else
        k_operands<T, NP, KD, false><<<(unsigned)w.tt, kThreads, 0, st>>>(
            table, a.rows, a.table_stride, a.dim, a, nullptr, nullptr, nullptr, w.T);
    StreamArgs s{};
    s.q = feat;
    s.nq = a.n;
    s.q_stride = a.feat_stride;
    s.keys = w.T;
    s.nk = a.rows;
    s.tiles = (int)w.tt;
    s.dim = a.dim;
    s.scale2 = a.scale * kLog2e;
    s.labels = a.labels;
    s.labels64 = a.labels64;
    s.flags = a.flags;
    s.table_rows = a.rows;
    s.label = w.label;
    s.weight = w.weight;
    s.lse2 = w.lse2;
    s.share = w.scores.tiles;
    s.part = w.part;
    s.label_score = w.score;
    s.loss = a.loss;
    s.lse = a.lse;
    s.lse2_out = w.lse2;
    s.padded = a.n;
    hipError_t e;
    // the gradients' tiles hold both products' operands, the scores take the first
    constexpr int kFirst = NP * KD / 16 * 64;
    s.tile_stride = grad ? 2 * kFirst : kFirst;
    e = launch_stream<T, NP, KD, kScores>(s, w.scores, st);
    if (e != hipSuccess) return e;
    if (w.scores.count > 1)
        k_stream_join<<<(unsigned)((a.n + kThreads - 1) / kThreads), kThreads, 0, st>>>(
            s, w.scores.count);
    if (!grad) return hipGetLastError();
    k_operands<T, NP, KD, true><<<(unsigned)w.tf, kThreads, 0, st>>>(
        feat, a.n, a.feat_stride, a.dim, a, w.label, w.weight, w.lse2, w.F);
    s.share = w.by_feat.tiles;
    s.out = a.dfeat;
    s.out_stride = a.dfeat_stride;
    s.sums = w.sums;
    e = launch_stream<T, NP, KD, kGradFeat>(s, w.by_feat, st);
    if (e != hipSuccess) return e;
    if (w.by_feat.count > 1)
        k_loss_fold<T><<<blocks_for(a.n * KD), kThreads, 0, st>>>(
            w.sums, w.by_feat.count, a.n, KD, nullptr, 1, 1, static_cast<T*>(a.dfeat), a.n,
            a.dfeat_stride, a.dim, w.label);
    s.q = table;
    s.nq = a.rows;
    s.q_stride = a.table_stride;
    s.keys = w.F;
    s.nk = a.n;
    s.tiles = (int)w.tf;
    s.share = w.by_table.tiles;
    s.out = a.dtable;
    s.out_stride = a.dtable_stride;
    s.padded = a.rows;
    e = launch_stream<T, NP, KD, kGradTable>(s, w.by_table, st);
    if (e != hipSuccess) return e;
    if (w.by_table.count > 1)
        k_loss_fold<T><<<blocks_for(a.rows * KD), kThreads, 0, st>>>(
            w.sums, w.by_table.count, a.rows, KD, nullptr, 1, 1, static_cast<T*>(a.dtable), a.rows,
            a.dtable_stride, a.dim, nullptr);
    return hipGetLastError();
}

// Padded row length that the streaming kernels take, 0: none. Past it a wave's
// own rows and sums no longer fit its registers.
int stream_kd(int dim, int dtype) {
    for (int kd : {32, 64, 128, 256})
        if (dim <= kd) return dtype == 0 && kd > 128 ? 0 : kd;
    return 0;
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
    const int kd = stream_kd(dim, dtype);
    if (kd != 0) return StreamPlan(nullptr, n, rows, dtype == 0 ? 3 : 1, kd, grad).bytes;
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
    const bool f = a.dtype == 0;
    switch (stream_kd(a.dim, a.dtype)) {
        case 32: return f ? stream_run<float, 3, 32>(a, grad, st) : stream_run<bf16, 1, 32>(a, grad, st);
        case 64: return f ? stream_run<float, 3, 64>(a, grad, st) : stream_run<bf16, 1, 64>(a, grad, st);
        case 128:
            return f ? stream_run<float, 3, 128>(a, grad, st) : stream_run<bf16, 1, 128>(a, grad, st);
        case 256: return stream_run<bf16, 1, 256>(a, grad, st);
        default: return f ? loss_run<float, 3>(a, grad, st) : loss_run<bf16, 1>(a, grad, st);
    }
}

}  // namespace gs
