// field_loss.hip - softmax cross entropy of features against a table of labels,
// with its gradients, without ever holding the (n, rows) scores.
//
//   l_iv = scale <feat_i, table_v>;  lse_i = log sum_v exp l_iv
//   loss_i = lse_i - l_i,label(i)      (0 for a masked row, label < 0)
//   G_iv = weight_i scale (exp(l_iv - lse_i) - [v = label(i)])
//   dfeat = G table;  dtable = G^T feat
//
// All products run on the matrix cores with bf16 operands and fp32 sums. fp32
// inputs are cut into three bf16 parts of 8 bits each (exact: 24 bits; for infinite
// values see split8_input) and the six products whose weight is above 2^-24 are added up, which keeps fp32's
// precision at 6/16 of the cost of the fp32 matrix instructions. Bf16 inputs are
// the operands as they are; their G is rounded to bf16, as their gradients are in
// the end, since parts of G would double the products that it enters: 30011 x 32003 of
// 512 the gradients are 0.0023 off (2-norm, relative), where rounding them alone gives
// 0.0017.
//
// Three ways, by size:
//   few        up to 8 samples, losses alone: one read of the table, no layout.
//   streaming  rows of at most 128: scores and G stay in registers, the other
//              side streams through LDS (k_stream), in 2 passes that each make the
//              scores and one of the gradients.
//   pieces     longer rows: 128 x 128 tiles, G of one piece at a time in the
//              workspace; the scores are made twice here too, once for lse.
// All sums are made in an order that depends on the sizes alone.
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
// Where a running maximum begins: finite, so that differences of two are numbers.
constexpr float kLowest = -3.402823466e38f;

// Part p of a value: the leading 8 significant bits, the next 8, the rest.
// Cutting off (not rounding) leaves exact remainders.
__device__ __forceinline__ float cut_bf16(float v) {
    return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
}
// A NaN is made canonical first, so that its parts are NaN.
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
// The same of inputs. An infinite value has the parts (1, 0, inf) with its sign: its last
// part meets the other value's first part alone, which is 0 only where that value is, so
// the product is what arithmetic gives, also of two infinite values.
template <int NP>
__device__ __forceinline__ void split8_input(const float* v, quad* out) {
    if constexpr (NP == 1) {
        split8<NP>(v, out);
    } else {
        float u[8];
        bool any = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool inf = fabsf(v[k]) == INFINITY;
            u[k] = inf ? copysignf(1.0f, v[k]) : v[k];
            any |= inf;
        }
        split8<NP>(u, out);
        if (!any) return;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (fabsf(v[k]) == INFINITY)
                out[NP - 1][k / 2] |= (__float_as_uint(v[k]) >> 16) << (k & 1) * 16;
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
// A row's 8 values from column c, cut into parts; zeros past the row.
template <typename T, int NP>
__device__ __forceinline__ void load_parts(const T* row, int dim, int c, bool on, quad* out) {
    if constexpr (NP == 1 && sizeof(T) == 2) {
        if (c + 8 <= dim) {  // as they are
            quad u = {0u, 0u, 0u, 0u};
            if (on) __builtin_memcpy(&u, row + c, sizeof(u));
            out[0] = u;
            return;
        }
    }
    float v[8];
    if (on && c + 8 <= dim) {
        load_any<8>(row + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = plain_input<NP>(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = on && c + e < dim ? plain_input<NP>(to_float(row[c + e])) : 0.0f;
    }
    split8_input<NP>(v, out);
}

// Parts of the samples as (nr, ld) and of the table as (vp, ld), zeros in the padding
// and in masked samples; labels as 32-bit (-1: masked), with their weights where the
// gradients need them.
template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void k_parts(LossArgs a, int64_t nr, int64_t vp, int ld,
                                                    int32_t* label, float* weight, quad* F,
                                                    quad* table) {
    const int units = ld / 8;
    const int64_t samples = nr * units, total = samples + vp * units;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const bool of_table = e >= samples;
        const int64_t u = of_table ? e - samples : e, r = u / units;
        const int c = (int)(u - r * units) * 8;
        quad part[NP];
        if (of_table) {
            load_parts<T, NP>(static_cast<const T*>(a.table) + r * a.table_stride, a.dim, c,
                              r < a.rows, part);
        } else {
            const int32_t l = r < a.n ? load_id(a.labels, a.labels64, r, a.rows,
                                                c == 0 ? a.flags : nullptr)
                                      : -1;
            if (c == 0) {
                label[r] = l;
                if (weight != nullptr)
                    weight[r] =
                        l < 0 ? 0.0f
                              : a.scale * (a.row_weight != nullptr ? a.row_weight[r] : 1.0f);
            }
            load_parts<T, NP>(static_cast<const T*>(a.feat) + r * a.feat_stride, a.dim, c, l >= 0,
                              part);
        }
        quad* out = of_table ? table : F;
        const int64_t plane = of_table ? total - samples : samples;
#pragma unroll
        for (int p = 0; p < NP; ++p) out[p * plane + u] = part[p];
    }
}

// ---------------------------------------------------------------- products
struct Mat {
    const bf16* p;
    int64_t ld, plane;  // elements between rows and between parts
};

// The wave's number, known to be the same in all its lanes.
__device__ __forceinline__ int wave_id() {
    return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
}

// One operand's 128 x 64 tile in LDS (1024 quads). K: rows of the matrix hold the
// summed index, and the tile's 128 rows of 64 are placed by (piece ^ row % 8), so
// that 8 lanes reading one column of pieces touch all banks once. Not K: the
// matrix's rows are the summed index; 64 rows of 128, 32-byte pieces placed by
// (piece ^ the row's bits 0, 1 and 2 ^ 3), read through the transposing LDS load: in a
// group of 16 lanes, lane s reads 4 values of row s / 4 at column 4 (s % 4), and lane
// g gets column g of the 4 rows; two groups touch all banks once. Addresses are a base common to the wave and one lane
// offset: with one 64-bit address a load, the registers do not last.
//
// PAIRS (with K): block i of 16 rows takes rows 32 (i / 2) + 8 (s / 4) + 4 (i % 2) +
// s % 4 instead of 16 i + s, so that a lane's sums of two blocks are 8 rows in a row.
template <bool K, bool PAIRS = false>
struct Side {
    __device__ __forceinline__ static uint32_t place(uint32_t row) {
        if (!K) return (row & 3) | ((row ^ (row >> 1)) & 4);
        return PAIRS ? (row & 3) | ((row >> 1) & 4) : row & 7;
    }
    uint32_t from;  // the lane's byte offset in memory
    int64_t ld;
    __device__ __forceinline__ explicit Side(const Mat& m) : ld(m.ld) {
        const uint32_t t = threadIdx.x, row = K ? t >> 3 : t >> 4;
        const uint32_t c = K ? (t & 7) ^ place(row) : (t & 15) ^ (place(row) << 1);
        from = (row * (uint32_t)m.ld + c * 8) * 2;
    }
    // Straight into LDS: a wave's 64 quads lie there in lane order.
    __device__ __forceinline__ void fetch(const Mat& m, int part, int64_t row0, int64_t k,
                                          quad* lds) const {
        typedef const __attribute__((address_space(1))) void* from_t;
        typedef __attribute__((address_space(3))) void* to_t;
        const char* p = reinterpret_cast<const char*>(m.p + part * m.plane +
                                                      (K ? row0 * ld + k : k * ld + row0));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            __builtin_amdgcn_global_load_lds(
                (from_t)(p + (int64_t)j * (K ? 64 : 32) * ld + from),
                (to_t)(lds + j * 256 + wave_id() * 64), 16, 0, 0);
    }
    // the operand of rows b + 16 i .. + 15 (b 0 or 64, the same in the wave), summed
    // index 32 h .. 32 h + 31
    __device__ __forceinline__ static bf16x8 operand(const quad* lds, int b, int i, int h) {
        const int lane = threadIdx.x & 63, g = lane >> 4, s = lane & 15;
        if (K) {
            const uint32_t row = PAIRS ? (s >> 2) * 8 + (s & 3) : s;
            const quad* at = lds + row * 8 + ((g ^ place(row)) ^ (h * 4));
            return __builtin_bit_cast(
                bf16x8, at[(b + (PAIRS ? (i >> 1) * 32 + (i & 1) * 4 : i * 16)) * 8]);
        }
        typedef __attribute__((ext_vector_type(4))) short s16x4;
        typedef __attribute__((address_space(3))) s16x4* lds4;
        // row r = 32 h + 8 g + 4 u + s / 4: its piece b / 16 + i lies at
        // 4 (b / 64 ^ u ^ g % 2) + (i ^ s / 4)
        const char* at = reinterpret_cast<const char*>(lds) + (g * 8 + (s >> 2)) * 256 +
                         (s & 3) * 8 + (i ^ (s >> 2)) * 32;
        s16x4 half[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds4)(at + h * 8192 + u * 1024 + ((b >> 6) ^ u ^ (g & 1)) * 128));
        return __builtin_bit_cast(
            bf16x8, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// Tiles of A B^T one after the other for one workgroup: 4 waves of 64 x 64, 64 of
// the summed index a step, the next step's operands on their way from memory
// straight into the other half of LDS while this one's are multiplied, also across
// tiles. `rows(tile)` gives the tile's first rows of A and B; `done(tile, acc)`
// takes its 128 x 128 sums. All of a step's operands are read from LDS before the
// next loads are started: the compiler cannot tell the halves apart, and would have
// a read after them wait for all of them.
//
// 30011 x 32003 of 512 bf16: scores 1010 TFLOP/s, G 800, dfeat 810, dtable 930. The
// matrix cores are busy 37 to 48 % of the time, LDS 18 to 24 %: bound by the wait
// for the next step's loads, a step's products ahead of their use, and G and its sums
// by their bytes. Two steps ahead would need LDS reads that the compiler does not hold
// up for loads in flight. Through registers a step took 5 to 10 % longer. Tiles of 256
// x 128 in steps of 32 move a quarter less, but G's epilogue spilled: 5.45 against 5.20
// ms, though sums alone gained a seventh.
#define GS_TILE_LDS __shared__ quad lds[4 * kTile * 8]
template <int NP, bool AK, bool BK, bool PAIRS = false, class Rows, class Done>
__device__ __forceinline__ void tile_products(const Mat& A, const Mat& B, int64_t k0, int64_t k1,
                                              int tiles, quad* lds, Rows rows,
                                              Done done) {
    const int w = wave_id(), wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const int steps_k = (int)((k1 - k0) / kStep), per_tile = steps_k * Products<NP>::kCount;
    using SideA = Side<AK, PAIRS>;
    SideA a(A);
    Side<BK> b(B);
    int tile_f = 0, q_f = 0, k_f = 0;  // the next step to fetch
    auto fetch = [&](quad* to) {
        const auto at = rows(tile_f);
        const int64_t k = k0 + (int64_t)k_f * kStep;
        a.fetch(A, Products<NP>::a(q_f), at.m, k, to);
        b.fetch(B, Products<NP>::b(q_f), at.n, k, to + kTile * 8);
        if (++k_f == steps_k) {
            k_f = 0;
            if (++q_f == Products<NP>::kCount) {
                q_f = 0;
                ++tile_f;
            }
        }
    };
    f32x4 acc[4][4];
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    const int steps = per_tile * tiles;
    if (steps > 0) fetch(lds);
    int left = per_tile, tile = 0;
    for (int s = 0; s < steps; ++s) {
        const quad* la = lds + (s & 1) * (2 * kTile * 8);
        const quad* lb = la + kTile * 8;
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part has arrived
        __syncthreads();
        bf16x8 fa[2][4], fb[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fa[h][i] = SideA::operand(la, wm, i, h);
                fb[h][i] = Side<BK>::operand(lb, wn, i, h);
            }
        if (s + 1 < steps) fetch(lds + ((s + 1) & 1) * (2 * kTile * 8));
        if (left == 0) {  // here the tile's stores have a step's time until loads wait for them
            done(tile++, acc);
            clear();
            left = per_tile;
        }
        --left;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[h][i], fb[h][j],
                                                                        acc[i][j], 0, 0, 0);
    }
    done(tile, acc);
}

// A value for a block that few tiles reach: what depends on it stays in the block,
// and takes no registers outside. 400000 x 1000 of 16 bf16 without gradients took 101
// us, 93 so; k_stream's gradients took up to 2 % longer with it and go without.
__device__ __forceinline__ int rare(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

struct TileRows {
    int64_t m, n;
};

// Work (x, y) of a workgroup, x < nx and, if it has any, y < ny: every eighth
// workgroup runs on the same XCD, and there `gy` values of y follow each other with
// one x, so that its L2 serves what belongs to x to all of them, and the y's parts
// to the x's that run beside. With x first in plain order, samples came from beyond
// the L2 for every tile of scores and G once per 128 columns of the sums: 30011 x
// 32003 of 512 bf16 took 5.23 ms, so 4.87.
struct Spot {
    int x, y;
};
__device__ __forceinline__ Spot spot(int nx, int gy) {
    const int k = blockIdx.x >> 3, e = k / gy * 8 + (blockIdx.x & 7);
    return {e % nx, e / nx * gy + k % gy};
}
constexpr int kSpot = 8;  // y's of the scores and of G: 4 took 5.00 ms of the above
struct SpotGrid {
    int gy;
    unsigned blocks;
    SpotGrid(int64_t nx, int64_t ny, int64_t most) {
        const int64_t groups = (ny + most - 1) / most;
        gy = (int)((ny + groups - 1) / groups);
        blocks = (unsigned)((nx * groups + 7) / 8 * 8 * gy);
    }
};

// Largest score and sum of exp2(score - largest) of two sets of scores, into the
// first. A largest that is infinite counts as 0 there, so that the sum is infinite.
__device__ __forceinline__ void join_sums(float& m, float& sum, float m2, float s2) {
    const float mm = fmaxf(m, m2), base = mm < INFINITY ? mm : 0.0f;
    sum = sum * __builtin_amdgcn_exp2f((m < INFINITY ? m : 0.0f) - base) +
          s2 * __builtin_amdgcn_exp2f((m2 < INFINITY ? m2 : 0.0f) - base);
    m = mm;
}

// Scores of one tile of samples (columns) against a share of the table's tiles: a
// lane keeps the largest and the sum of exp2(score - largest) of its 4 samples,
// scores in log2 units, and joins the other lanes' at the end. A largest that is
// infinite is taken as 0, so that infinite scores give infinite sums.
template <int NP>
__global__ __launch_bounds__(kThreads, 2) void k_loss_scores(Mat F, Mat T, int kd, int64_t rows,
                                                          float scale2, const int32_t* label,
                                                          int64_t padded, int tiles, int share,
                                                          int gy, float2* part,
                                                          float* label_score) {
    GS_TILE_LDS;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const Spot at = spot((int)(padded / kTile), gy);
    const int64_t n0 = (int64_t)at.x * kTile;
    const int t0 = at.y * share, t1 = min(tiles, t0 + share);
    if (t0 >= tiles) return;
    float m[4], sum[4];
    int32_t y[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        m[n] = kLowest;
        sum[n] = 0.0f;
        y[n] = label[n0 + wn + n * 16 + (lane & 15)];
    }
    tile_products<NP, true, true>(
        T, F, 0, kd, t1 - t0, lds,
        [&](int t) { return TileRows{(int64_t)(t0 + t) * kTile, n0}; },
        [&](int t, f32x4(&acc)[4][4]) {
            const int64_t v0 = (int64_t)(t0 + t) * kTile + wm + (lane >> 4) * 4;
            const int64_t v_wave = (int64_t)(t0 + t) * kTile + wm;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][n] *= scale2;
                if (v_wave + 64 > rows) {
                    const int left = rare((int)(rows - v0));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[i][n][j] = i * 16 + j < left ? acc[i][n][j] : -INFINITY;
                }
                if (__any(y[n] >= v_wave && y[n] < v_wave + 64)) {
                    const int own = rare(y[n] - (int)v0);
                    float score = 0.0f;
                    bool here = false;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            score = own == i * 16 + j ? acc[i][n][j] : score;
                            here |= own == i * 16 + j;
                        }
                    if (here) label_score[n0 + wn + n * 16 + (lane & 15)] = score;
                }
                float mt = m[n];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mt = fmaxf(mt, acc[i][n][j]);
                const float base = mt < INFINITY ? mt : 0.0f;
                const float was = m[n] < INFINITY ? m[n] : 0.0f;
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        add += __builtin_amdgcn_exp2f(acc[i][n][j] - base);
                sum[n] = sum[n] * __builtin_amdgcn_exp2f(was - base) + add;
                m[n] = mt;
            }
        });
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[n], o, 64), s2 = __shfl_xor(sum[n], o, 64);
            join_sums(m[n], sum[n], m2, s2);
        }
        if (lane < 16)
            part[((int64_t)at.y * 2 + (w >> 1)) * padded + n0 + wn + n * 16 + lane] =
                make_float2(m[n], sum[n]);
    }
}

// Joins the partials (parts, padded) of a row's scores: 8 threads a row. lse2, for
// the gradients, is in log2 units.
__global__ __launch_bounds__(kThreads) void k_loss_join(LossArgs a, const float2* part, int parts,
                                                        int64_t padded, const float* label_score,
                                                        float* lse2) {
    const int sub = threadIdx.x >> 5;  // of the workgroup's 32 rows
    __shared__ float2 lds[8][32];
    for (int64_t i0 = (int64_t)blockIdx.x * 32; i0 < padded; i0 += (int64_t)gridDim.x * 32) {
        const int64_t i = i0 + (threadIdx.x & 31);
        float m = kLowest, sum = 0.0f;
        if (i < padded)
            for (int k0 = sub; k0 < parts; k0 += 8 * 8) {
                float2 p[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    p[u] = k0 + u * 8 < parts ? part[(int64_t)(k0 + u * 8) * padded + i]
                                              : make_float2(kLowest, 0.0f);
#pragma unroll
                for (int u = 0; u < 8; ++u) join_sums(m, sum, p[u].x, p[u].y);
            }
        __syncthreads();
        lds[sub][threadIdx.x & 31] = make_float2(m, sum);
        __syncthreads();
        if (sub != 0 || i >= padded) continue;
        for (int k = 1; k < 8; ++k) {
            const float2 p = lds[k][threadIdx.x & 31];
            join_sums(m, sum, p.x, p.y);
        }
        const float l = (m < INFINITY ? m : 0.0f) + log2f(sum);
        const bool on = i < a.n && load_id(a.labels, a.labels64, i, a.rows, nullptr) >= 0;
        if (lse2 != nullptr) lse2[i] = on ? l : 0.0f;
        if (i < a.n) {
            if (a.loss != nullptr) a.loss[i] = on ? (l - label_score[i]) * kLn2 : 0.0f;
            if (a.lse != nullptr) a.lse[i] = on ? l * kLn2 : 0.0f;
        }
    }
}

// The exponential of a gradient, exp2(x) from kHalf x: the square of exp2(x / 2) in
// fp32, since the bare instruction gives 0 below 2^-126, which gradients, times
// weight * scale, would show; halves are exact. For bf16 gradients it is left so.
template <int NP>
constexpr float kHalf = NP == 1 ? 1.0f : 0.5f;
template <int NP>
__device__ __forceinline__ float grad_exp2(float x) {
    const float e = __builtin_amdgcn_exp2f(x);
    return NP == 1 ? e : e * e;
}

// G of one piece (samples r0.., table rows v0..) in parts, (rc, vc) each.
template <int NP>
__global__ __launch_bounds__(kThreads, 2) void k_loss_g(Mat F, Mat T, int kd, int64_t rows,
                                                     float scale2, const int32_t* label,
                                                     const float* weight, const float* lse2,
                                                     int64_t r0, int64_t v0, int64_t rc, int64_t vc,
                                                     int share, int gy, bf16* G) {
    GS_TILE_LDS;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const Spot place = spot((int)(rc / kTile), gy);
    const int64_t n0 = (int64_t)place.x * kTile;
    const int t0 = place.y * share, t1 = min((int)(vc / kTile), t0 + share);
    if (t0 >= t1) return;
    int32_t y[4];
    float wt[4], l2[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int64_t i = r0 + n0 + wn + n * 16 + (lane & 15);
        y[n] = label[i];
        wt[n] = weight[i];
        l2[n] = lse2[i] * kHalf<NP>;
    }
    tile_products<NP, true, true, true>(
        T, F, 0, kd, t1 - t0, lds,
        [&](int t) { return TileRows{v0 + (int64_t)(t0 + t) * kTile, r0 + n0}; },
        [&](int t, f32x4(&acc)[4][4]) {
            const int64_t tile = (int64_t)(t0 + t) * kTile + wm;  // within the piece
            const int64_t at = tile + (lane >> 4) * 8;
            const bool in = v0 + tile + 64 <= rows;  // else some rows are padding
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const bool any = __any(y[n] >= v0 + tile && y[n] < v0 + tile + 64);
                bf16* row = G + (n0 + wn + n * 16 + (lane & 15)) * vc + at;
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // 8 values of blocks 2 i and 2 i + 1
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[j] = grad_exp2<NP>(
                            fmaf(acc[2 * i + (j >> 2)][n][j & 3], scale2 * kHalf<NP>, -l2[n]));
                    const int first = (int)(v0 + at) + i * 32;
                    if (any) {
                        const int own = rare(y[n] - first);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] -= j == own ? 1.0f : 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = v[j] * wt[n];
                        v[j] = y[n] >= 0 ? x : 0.0f;
                    }
                    if (!in) {
                        const int left = rare((int)rows - first);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = j < left ? v[j] : 0.0f;
                    }
                    quad part[NP];
                    split8<NP>(v, part);
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        *reinterpret_cast<quad*>(row + p * rc * vc + i * 32) = part[p];
                }
            }
        });
}

// Where a product's sums go: with one share of the summed index onto the earlier
// pieces' (`sum`), and with the last piece, rounded, into the caller's rows, masked
// rows as zeros; with several shares each into its slice, for k_loss_fold.
template <typename T>
struct SumOut {
    float* slices;
    float* sum;
    int first, last;
    int64_t m;
    int dq;
    T* out;
    int64_t rows, stride;
    int dim;
    const int32_t* label;
    // 4 values from column c of row r
    __device__ __forceinline__ void put(int64_t r, int c, f32x4 v) const {
        f32x4* to = reinterpret_cast<f32x4*>(sum + r * dq + c);
        if (!first) v += *to;
        if (!last) {
            *to = v;
            return;
        }
        if (r >= rows || c >= dim) return;
        if (label != nullptr && label[r] < 0) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const float x[4] = {v[0], v[1], v[2], v[3]};
        T* row = out + r * stride + c;
        if (c + 4 <= dim) {
            store_any<4>(row, x);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < dim) row[j] = from_float<T>(x[j]);
        }
    }
};

// Share z of A B over the summed index, for 128 x 128 sums. A: G, by
// samples (AK) or transposed; B's rows are the summed index. The sums leave through
// LDS, half of the columns at a time, as rows of whole vectors: straight from the
// registers the 64 addresses of a lane spilled.
template <typename T, int NP, bool AK>
__global__ __launch_bounds__(kThreads, 2) void k_loss_sum(Mat A, Mat B, int64_t k, int64_t share,
                                                          int nz, SumOut<T> o) {
    constexpr int kRow = 68;  // floats of a row of 64, so that rows 4 apart use other banks
    __shared__ quad buf[4 * kTile * 8];
    static_assert(kTile * kRow / 4 <= 4 * kTile * 8, "half of the sums fits");
    const int nm = (int)(o.m / kTile);
    const Spot at = spot(nm * nz, o.dq / kTile);
    const int z = at.x / nm;
    if (at.y >= o.dq / kTile) return;
    const int64_t m0 = (int64_t)(at.x % nm) * kTile, n0 = (int64_t)at.y * kTile;
    const int64_t k0 = min(k, share * z), k1 = min(k, k0 + share);
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    tile_products<NP, AK, false>(
        A, B, k0, k1, 1, buf,
        [&](int) { return TileRows{m0, n0}; },
        [&](int, f32x4(&acc)[4][4]) {
            float* f = reinterpret_cast<float*>(buf);
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                __syncthreads();
                if (wn == half * 64) {
                    float* at = f + (wm + (lane >> 4) * 4) * kRow + (lane & 15);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                at[(i * 16 + j) * kRow + n * 16] = acc[i][n][j];
                }
                __syncthreads();
#pragma unroll 2
                for (int e = threadIdx.x; e < kTile * 16; e += kThreads) {
                    const int r = e >> 4, c = (e & 15) * 4;
                    const f32x4 v = *reinterpret_cast<const f32x4*>(f + r * kRow + c);
                    const int64_t row = m0 + r;
                    const int column = (int)n0 + half * 64 + c;
                    if (nz > 1)
                        *reinterpret_cast<f32x4*>(
                            o.slices + ((int64_t)z * o.m + row) * o.dq + column) = v;
                    else
                        o.put(row, column, v);
                }
            }
        });
}

// Adds nz slices (m, dq) in order: 4 columns a thread, the slices over Z threads.
// Bound by latency and the slices' bytes: 8 of 8192 x 64 in 5 us.
template <typename T, int Z>
__global__ __launch_bounds__(kThreads) void k_loss_fold(SumOut<T> o, int nz) {
    __shared__ f32x4 lds[Z > 1 ? kThreads : 1];
    constexpr int kItems = kThreads / Z;
    const int64_t total = o.m * (o.dq / 4);
    const int z0 = threadIdx.x / kItems;
    for (int64_t e0 = (int64_t)blockIdx.x * kItems; e0 < total; e0 += (int64_t)gridDim.x * kItems) {
        const int64_t e = e0 + threadIdx.x % kItems;
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e < total)
            for (int z = z0; z < nz; z += Z * 4) {
                f32x4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    v[u] = z + u * Z < nz ? reinterpret_cast<const f32x4*>(
                                                o.slices)[(int64_t)(z + u * Z) * total + e]
                                          : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 4; ++u) s += v[u];
            }
        if (Z > 1) {
            __syncthreads();
            lds[threadIdx.x] = s;
            __syncthreads();
            if (z0 != 0) continue;
            for (int z = 1; z < Z; ++z) s += lds[z * kItems + threadIdx.x];
        }
        if (e >= total) continue;
        const int64_t r = e / (o.dq / 4);
        const int c = (int)(e - r * (o.dq / 4)) * 4;
        o.put(r, c, s);
    }
}

unsigned blocks_for(int64_t items) { return std::min(65536u, blocks_of(items, kThreads)); }

template <typename T>
hipError_t fold(const SumOut<T>& o, int nz, hipStream_t st) {
    const int64_t items = o.m * (o.dq / 4);
    if (nz <= 8)
        k_loss_fold<T, 1><<<blocks_for(items), kThreads, 0, st>>>(o, nz);
    else
        k_loss_fold<T, 16><<<blocks_for(items * 16), kThreads, 0, st>>>(o, nz);
    return hipGetLastError();
}

// ---------------------------------------------------------------- streaming
// For rows short enough that a wave keeps its own in registers: each of a
// workgroup's 4 waves holds 32 QB "queries", the other side's rows ("keys") stream
// through LDS, 32 a tile, and neither scores nor G ever leave the registers.
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
//
// kScores: losses alone. kGradFeat: losses and dfeat in one pass over the table: the
// sums of e_v table_v, e_v = exp2(score_v - m), go along with the sum of e_v, both
// scaled down when a query's largest score has grown past m by more than kSlack
// (at a query's first tile, then hardly ever). The label's row stays out of the
// rounded products: dfeat = weight (sums / sum + (e_label / sum - 1) table_label),
// its factor in fp32, so that a label with almost all of its row's probability
// costs no digits. kGradTable: the table's gradient, with the losses known.
//
// Bound by the matrix cores and, in fp32, as much by cutting the exponentials into
// parts (88 of about 440 vector instructions a tile beside 42 products of 16 cycles).
// 10007 x 8192 of 48 fp32: losses and dfeat 111 us, dtable 104, at six bf16 products
// for each one 0.85 and 0.91 PFLOP/s. 307200 x 150 of 32 bf16, losses alone: 17 us, where
// the 46 million exponentials take 5 at the transcendental rate and the bytes 5; the
// vector units are busy half of the time.
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float kSlack = 8.0f;
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
    // kScores, kGradFeat
    const void* labels;
    int labels64;
    float2* part;
    float *label_score, *loss, *lse, *lse2_out;
    uint32_t* flags;
    int64_t table_rows;
    // kGradFeat
    const void* table;
    int64_t table_stride;
    const float* row_weight;
    float scale;
    // gradients: into out where there is one share, else into (share, padded, row) sums
    void* out;
    int64_t out_stride;
    float* sums;
    int64_t padded;
};

// The larger of lane l's and lane l ^ 32's value.
__device__ __forceinline__ float max_of_halves(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// Key of register r of a lane in half h.
__device__ __forceinline__ constexpr int key_of(int r) { return (r & 3) + 8 * (r >> 2); }

// Row length of the second product, whose operands are 32 columns wide.
constexpr int padded_dim(int ks) { return (ks + 31) / 32 * 32; }
// Blocks of 32 queries a wave. A key's operand read from LDS serves QB products of
// each part: with one part two blocks are needed to feed the matrix cores, with
// three one does, and two waves a unit fit.
template <int NP>
constexpr int kBlocks = NP == 1 ? 2 : 1;

// (rows, dim) as tiles of operands, a workgroup a tile (or several); of samples (label) the
// masked ones are zeros, and label and weight are written for the gradients. Bound by
// latency: 10007 x 48 fp32 7 us.
template <typename T, int NP, int KS, bool SECOND>
__global__ __launch_bounds__(kThreads) void k_operands(const T* src, int64_t rows, int64_t stride,
                                                       int dim, LossArgs a, int32_t* label,
                                                       float* weight, float* lse2, quad* out) {
    constexpr int DD = padded_dim(KS);
    __shared__ float tile[32][DD + 1];
    __shared__ int32_t lab[32];
    constexpr int kFirst = KS / 16 * 64, kSecond = SECOND ? DD / 32 * 2 * 64 : 0;
    for (int64_t r0 = (int64_t)blockIdx.x * 32; r0 < rows; r0 += (int64_t)gridDim.x * 32) {
        __syncthreads();
        if (threadIdx.x < 32) {
            int32_t l = 0;
            if (label != nullptr) {
                const int64_t i = r0 + threadIdx.x;
                l = i < rows ? load_id(a.labels, a.labels64, i, a.rows, nullptr) : -1;
                label[i] = l;
                weight[i] =
                    l < 0 ? 0.0f : a.scale * (a.row_weight != nullptr ? a.row_weight[i] : 1.0f);
                if (i >= rows) lse2[i] = 0.0f;  // the others' come from the scores
            }
            lab[threadIdx.x] = l;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 32 * DD; e += kThreads) {
            const int r = e / DD, c = e % DD;
            float v = 0.0f;
            if (r0 + r < rows && c < dim && lab[r] >= 0)
                v = plain_input<NP>(to_float(src[(r0 + r) * stride + c]));
            tile[r][c] = v;
        }
        __syncthreads();
        quad* to = out + (size_t)(r0 / 32) * NP * (kFirst + kSecond);
        for (int e = threadIdx.x; e < kFirst + kSecond; e += kThreads) {
            const int lane = e & 63, h = lane >> 5;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (e < kFirst) {
                    v[k] = tile[lane & 31][(e >> 6) * 16 + 8 * h + k];
                } else {
                    const int b = (e - kFirst) >> 6;  // dim / 32, f
                    v[k] =
                        tile[16 * (b & 1) + 4 * h + k + (k < 4 ? 0 : 4)][(b >> 1) * 32 + (lane & 31)];
                }
            }
            quad piece[NP];
            split8_input<NP>(v, piece);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const size_t at =
                    e < kFirst ? p * kFirst + e : NP * kFirst + p * kSecond + (e - kFirst);
                to[at] = piece[p];
            }
        }
    }
}

// Whether a kernel's registers leave it one wave a unit (two with spills were
// slower: 20000 x 5000 of 128 fp32 with gradients 1137 against 811 us).
constexpr bool one_a_unit(int ks, int role) { return role != kScores && ks >= 128; }

template <typename T, int NP, int KS, int ROLE>
struct StreamShape {
    static constexpr int kPieces =  // quads of a tile
        NP * 64 * (KS / 16 + (ROLE == kScores ? 0 : padded_dim(KS) / 16));
    // tiles per step: 8 to 24 KB (more takes registers on the way to LDS)
    static constexpr int kTiles = kPieces * 16 >= 16384 ? 1 : (kPieces * 16 >= 6144 ? 2 : 4);
    static constexpr int kStage = kPieces * kTiles;
    static constexpr size_t kLds = 2 * kStage * 16 + (ROLE == kGradTable ? 2 * kTiles * 32 * 12 : 0);
};

template <typename T, int NP, int KS, int ROLE>
__global__ __launch_bounds__(kThreads, one_a_unit(KS, ROLE) ? 1 : 2) void k_stream(StreamArgs a) {
    using Shape = StreamShape<T, NP, KS, ROLE>;
    constexpr int QB = kBlocks<NP>, KJ = KS / 16, DD = padded_dim(KS), DB = DD / 32;
    constexpr int TS = Shape::kTiles, STAGE = Shape::kStage;
    constexpr int PER = (STAGE + kThreads - 1) / kThreads;
    extern __shared__ quad lds[];
    float* info = reinterpret_cast<float*>(lds + 2 * STAGE);  // kGradTable: lse2, weight, label
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5, col = lane & 31;
    const int64_t q0 = ((int64_t)blockIdx.x * 4 + (t >> 6)) * (32 * QB);

    // the wave's own queries, as right operands of the scores
    quad q[QB][KJ][NP];
    int32_t y[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int64_t i = q0 + b * 32 + col;
        bool on = i < a.nq;
        y[b] = -1;
        if (ROLE != kGradTable) {
            if (on) y[b] = load_id(a.labels, a.labels64, i, a.table_rows,
                                   blockIdx.y == 0 && h == 0 ? a.flags : nullptr);
            on = y[b] >= 0;
        }
        if (ROLE == kGradTable) y[b] = (int32_t)min(i, (int64_t)0x7FFFFFFF);
        const T* row = static_cast<const T*>(a.q) + i * a.q_stride;
#pragma unroll
        for (int j = 0; j < KJ; ++j) load_parts<T, NP>(row, a.dim, 16 * j + 8 * h, on, q[b][j]);
    }
    // kGradTable: whether a table row of the wave's holds infinities or NaN (its last part
    // does then), whose products with masked samples, zeros, are NaN
    bool odd = false;
    if (ROLE == kGradTable) {
#pragma unroll
        for (int b = 0; b < QB; ++b)
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = q[b][j][NP - 1][e];
                    odd |= (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
                }
        odd = __any(odd);
    }

    f32x16 acc[QB][ROLE == kScores ? 1 : DB];
    float m[QB], sum[QB], own[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        m[b] = kLowest;
        sum[b] = own[b] = 0.0f;
    }
    if (ROLE != kScores) {
#pragma unroll
        for (int b = 0; b < QB; ++b)
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
            if (STAGE % kThreads == 0 || e < STAGE)
                pre[k] = from[(size_t)(e / Shape::kPieces) * a.tile_stride + e % Shape::kPieces];
        }
    };
    auto keep = [&](int s) {
        quad* to = lds + (s & 1) * STAGE + t;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (STAGE % kThreads == 0 || k * kThreads + t < STAGE) to[k * kThreads] = pre[k];
        if (ROLE == kGradTable) {
            float* f = info + (s & 1) * TS * 96;
            for (int k = t; k < TS * 32; k += kThreads) {
                const int64_t i = ((int64_t)t0 + (int64_t)s * TS) * 32 + k;
                f[k] = a.lse2[i] * kHalf<NP>;
                f[TS * 32 + k] = a.weight[i];
                f[2 * TS * 32 + k] = __int_as_float(a.label[i]);
            }
        }
    };
    const float scale_half = a.scale2 * kHalf<NP>;
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
            f32x16 sc[QB];
#pragma unroll
            for (int b = 0; b < QB; ++b)
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
                    for (int b = 0; b < QB; ++b)
                        sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            k[Products<NP>::a(i)],
                            __builtin_bit_cast(bf16x8, q[b][j][Products<NP>::b(i)]), sc[b], 0, 0, 0);
            }
            const int k0 = tile * 32;
            if (ROLE != kGradTable) {
#pragma unroll
                for (int b = 0; b < QB; ++b) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[b][r] *= a.scale2;
                    if (tile + 1 == a.tiles) {
                        const int last = (int)(a.nk - k0) - 4 * h;
                        const int left = ROLE == kScores ? rare(last) : last;
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            sc[b][r] = key_of(r) < left ? sc[b][r] : -INFINITY;
                    }
                    const int yl = y[b] - k0;
                    if (__any((unsigned)yl < 32u)) {
                        const int at = ROLE == kScores ? rare(yl - 4 * h) : yl - 4 * h;
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            own[b] = at == key_of(r) ? sc[b][r] : own[b];
                    }
                    float mt = m[b];
#pragma unroll
                    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[b][r]);
                    if (ROLE == kGradFeat) {
                        // both halves' keys enter the same sums
                        mt = max_of_halves(mt);
                        if (__any(mt > m[b] + kSlack)) {
                            mt = mt > m[b] + kSlack ? mt : m[b];
                            const float down = __builtin_amdgcn_exp2f(
                                (m[b] < INFINITY ? m[b] : 0.0f) - (mt < INFINITY ? mt : 0.0f));
                            sum[b] *= down;
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const float f = __shfl(down, key_of(r) + 4 * h, 64);
#pragma unroll
                                for (int d = 0; d < DB; ++d) acc[b][d][r] *= f;
                            }
                            m[b] = mt;
                        }
                        continue;  // the exponentials follow with the second product
                    }
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
                if (ROLE == kScores) continue;
            }
            quad g[QB][2][NP];
            const float* f = info + (s & 1) * TS * 96 + u * 32;
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                float v[16];
                if (ROLE == kGradFeat) {
                    const float base = m[b] < INFINITY ? m[b] : 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        v[r] = __builtin_amdgcn_exp2f(sc[b][r] - base);
                        sum[b] += v[r];
                    }
                    const int yl = y[b] - k0;
                    if (__any((unsigned)yl < 32u)) {
                        const int at = yl - 4 * h;
#pragma unroll
                        for (int r = 0; r < 16; ++r) v[r] = at == key_of(r) ? 0.0f : v[r];
                    }
                } else {
                    const int yk = __float_as_int(f[2 * TS * 32 + col]);
                    const bool any = __any((unsigned)(yk - (int)q0 - b * 32) < 32u);
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
                                grad_exp2<NP>(fmaf(sc[b][g4 * 4 + e], scale_half, -l[e]));
                        if (any) {
                            const float4 y4 = *reinterpret_cast<const float4*>(
                                f + 2 * TS * 32 + g4 * 8 + 4 * h);
                            const float yy[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[g4 * 4 + e] -=
                                    __float_as_int(yy[e]) == y[b] ? 1.0f : 0.0f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[g4 * 4 + e] *= w[e];
                        if (odd) {  // masked samples and padding have no gradient
                            const int4 y4 = *reinterpret_cast<const int4*>(
                                f + 2 * TS * 32 + g4 * 8 + 4 * h);
                            const int yy[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[g4 * 4 + e] = yy[e] < 0 ? 0.0f : v[g4 * 4 + e];
                        }
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
                        for (int b = 0; b < QB; ++b)
                            acc[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                __builtin_bit_cast(bf16x8, g[b][f2][Products<NP>::a(i)]),
                                k[Products<NP>::b(i)], acc[b][d], 0, 0, 0);
                }
        }
        if (s + 1 < steps) keep(s + 1);
        __syncthreads();
    }

    float w[QB], label_f[QB];  // kGradFeat: weight * scale, and the label row's factor
    if (ROLE != kGradTable) {
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int64_t i = q0 + b * 32 + col;
            const float m2 = __shfl_xor(m[b], 32, 64), s2 = __shfl_xor(sum[b], 32, 64);
            join_sums(m[b], sum[b], m2, s2);
            // the half that holds the label's score gives it to the other
            const bool here = y[b] >= 0 && ((y[b] >> 2) & 1) == h;
            const float o2 = __shfl_xor(own[b], 32, 64);
            const float mine = here ? own[b] : o2;
            w[b] = 0.0f;
            label_f[b] =
                __builtin_amdgcn_exp2f(mine - (m[b] < INFINITY ? m[b] : 0.0f)) / sum[b] - 1.0f;
            if (i >= a.nq) continue;
            if (ROLE == kGradFeat && y[b] >= 0)
                w[b] = a.scale * (a.row_weight != nullptr ? a.row_weight[i] : 1.0f);
            if (h != 0) continue;
            if (gridDim.y == 1) {
                const float l = (m[b] < INFINITY ? m[b] : 0.0f) + log2f(sum[b]);
                const bool on = y[b] >= 0;
                if (a.loss != nullptr) a.loss[i] = on ? (l - mine) * kLn2 : 0.0f;
                if (a.lse != nullptr) a.lse[i] = on ? l * kLn2 : 0.0f;
                if (a.lse2_out != nullptr) a.lse2_out[i] = on ? l : 0.0f;
            } else {
                a.part[blockIdx.y * a.padded + i] = make_float2(m[b], sum[b]);
                if (y[b] >= (int64_t)t0 * 32 && y[b] < (int64_t)t1 * 32) a.label_score[i] = mine;
            }
        }
        if (ROLE == kScores) return;
    }
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = key_of(r) + 4 * h;  // whose lane holds what belongs to it
            const int64_t i = q0 + b * 32 + row;
            int32_t label = 0;
            float over = 1.0f, weight = 1.0f, factor = 0.0f;
            if (ROLE == kGradFeat && gridDim.y == 1) {
                label = __shfl(y[b], row, 64);
                over = 1.0f / __shfl(sum[b], row, 64);
                weight = __shfl(w[b], row, 64);
                factor = __shfl(label_f[b], row, 64);
            }
            if (i >= a.nq) continue;
            const T* own_row = static_cast<const T*>(a.table) + (int64_t)max(label, 0) * a.table_stride;
#pragma unroll
            for (int d = 0; d < (ROLE == kScores ? 1 : DB); ++d) {
                const int c = d * 32 + col;
                float v = acc[b][d][r];
                if (gridDim.y > 1) {
                    a.sums[((size_t)blockIdx.y * a.padded + i) * DD + c] = v;
                } else if (c < a.dim) {
                    if (ROLE == kGradFeat)
                        v = label >= 0 ? weight * fmaf(v, over, factor * to_float(own_row[c])) : 0.0f;
                    static_cast<T*>(a.out)[i * a.out_stride + c] = from_float<T>(v);
                }
            }
        }
}

// Losses and dfeat from the shares of kGradFeat: DD / 4 threads a row and 4 columns
// each, Z times as many with every Z-th share each. Bound by the shares' bytes: 6 of
// 10007 x 64 (15 MB) 8 us.
template <typename T, int DD, int Z>
__global__ __launch_bounds__(kThreads) void k_feat_join(StreamArgs a, int shares) {
    constexpr int kLanes = DD / 4, kRows = kThreads / (kLanes * Z);
    __shared__ f32x4 sums[Z > 1 ? kThreads : 1];
    __shared__ float2 stats[Z > 1 ? kThreads : 1];
    const int at = threadIdx.x / kLanes, row = at % kRows, z = at / kRows;
    const int64_t i = (int64_t)blockIdx.x * kRows + row;
    const int c = threadIdx.x % kLanes * 4;
    float m = kLowest, sum = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float m2, float s2, f32x4 v2) {
        const float mm = fmaxf(m, m2), base = mm < INFINITY ? mm : 0.0f;
        const float f = __builtin_amdgcn_exp2f((m < INFINITY ? m : 0.0f) - base);
        const float f2 = __builtin_amdgcn_exp2f((m2 < INFINITY ? m2 : 0.0f) - base);
        sum = sum * f + s2 * f2;
        v = v * f + v2 * f2;
        m = mm;
    };
    if (i < a.nq)
        for (int s0 = z; s0 < shares; s0 += 4 * Z) {
            float2 p[4];
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s0 + u * Z < shares) {
                    const int64_t from = (int64_t)(s0 + u * Z) * a.padded + i;
                    p[u] = a.part[from];
                    x[u] = *reinterpret_cast<const f32x4*>(a.sums + from * DD + c);
                }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s0 + u * Z < shares) add(p[u].x, p[u].y, x[u]);
        }
    if (Z > 1) {
        sums[threadIdx.x] = v;
        stats[threadIdx.x] = make_float2(m, sum);
        __syncthreads();
        if (z != 0) return;
        for (int k = 1; k < Z; ++k) {
            const int from = threadIdx.x + k * kRows * kLanes;
            add(stats[from].x, stats[from].y, sums[from]);
        }
    }
    if (i >= a.nq) return;
    const int32_t y = load_id(a.labels, a.labels64, i, a.table_rows, nullptr);
    if (c == 0) {
        const float l = (m < INFINITY ? m : 0.0f) + log2f(sum);
        if (a.loss != nullptr) a.loss[i] = y >= 0 ? (l - a.label_score[i]) * kLn2 : 0.0f;
        if (a.lse != nullptr) a.lse[i] = y >= 0 ? l * kLn2 : 0.0f;
        a.lse2_out[i] = y >= 0 ? l : 0.0f;
    }
    const T* own_row = static_cast<const T*>(a.table) + (int64_t)max(y, 0) * a.table_stride;
    const float over = 1.0f / sum;
    const float factor =
        y >= 0 ? __builtin_amdgcn_exp2f(a.label_score[i] - (m < INFINITY ? m : 0.0f)) * over - 1.0f
               : 0.0f;
    const float w = a.scale * (a.row_weight != nullptr ? a.row_weight[i] : 1.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < a.dim)
            static_cast<T*>(a.out)[i * a.out_stride + c + j] = from_float<T>(
                y >= 0 ? w * fmaf(v[j], over, factor * to_float(own_row[c + j])) : 0.0f);
}

template <typename T, int DD, int Z>
hipError_t feat_join(const StreamArgs& a, int shares, hipStream_t st) {
    constexpr int kRows = kThreads / (DD / 4 * Z);
    k_feat_join<T, DD, Z><<<(unsigned)((a.nq + kRows - 1) / kRows), kThreads, 0, st>>>(a, shares);
    return hipGetLastError();
}

// ---------------------------------------------------------------- pieces
int64_t pad_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Pieces of G: up to 16384 table rows by as many samples as make 1 GB of bf16 parts,
// more table rows where there are few samples; all pieces of one size, so that
// none leaves the chip half empty. Of 256 MB, which the cache behind the L2s holds,
// the pieces were too many: 30011 x 32003 of 512 bf16 4.81 against 4.64 ms, 20000 x
// 50257 of 384 4.43 against 4.02 (512 MB: 4.75, 4.06).
constexpr int64_t kPieceValues = (int64_t)1 << 29;
constexpr int kAtOnce = 512;  // workgroups that the chip holds
struct LossPlan {
    int np, kd, dq;
    int64_t np_rows, vp, rc, vc;
    int shares, share;    // of the table's tiles, for the scores
    int zf, zt;           // of the summed index: for dfeat and for dtable
    int64_t share_f, share_t;
    bf16 *F, *T, *G;
    float2* part;
    float *score, *lse2, *weight, *slices, *sum_f, *sum_t;
    int32_t* label;
    size_t bytes;

    // Shares of the summed index for `tiles` tiles of sums: the fewest that leave at
    // most a tenth of the chip's rounds of workgroups empty, or come nearest (576
    // tiles in one share took 1020 us, 448 of the same length 554), and are worth the
    // slices: 4 steps, in three parts 12. With shares of 512 at least, and 16 at
    // most, 45 samples by 12078 rows of 512 fp32 took 180 us, so 137; with 128 in one
    // part 1000 x 1200 of 512 bf16 69 us, so 60.
    void split_k(int64_t tiles, int64_t k, int* z, int64_t* share) const {
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(64, k / (np == 1 ? 256 : 128)));
        int64_t best = 1;
        double best_full = 0.0;
        for (int64_t want = 1; want <= most && best_full < 0.9; ++want) {
            const int64_t all = tiles * want;
            const double full = (double)all / (double)((all + kAtOnce - 1) / kAtOnce * kAtOnce);
            if (full > best_full + 1e-9) {
                best = want;
                best_full = full;
            }
        }
        *share = pad_to((k + best - 1) / best, kStep);
        *z = *share == 0 ? 1 : (int)((k + *share - 1) / *share);
    }
    // `all` in equal pieces of at most `most`
    static int64_t piece(int64_t all, int64_t most) {
        const int64_t pieces = std::max<int64_t>(1, (all + most - 1) / most);
        return pad_to((all + pieces - 1) / pieces, kTile);
    }
    LossPlan(void* base, int64_t n, int64_t rows, int dim, int dtype, bool grad) {
        np = dtype == 0 ? 3 : 1;
        kd = (int)pad_to(dim, kStep);
        dq = (int)pad_to(dim, kTile);
        np_rows = pad_to(n, kTile);
        vp = pad_to(rows, kTile);
        const int64_t area = kPieceValues / np;
        vc = piece(vp, 16384);
        rc = piece(np_rows, std::max<int64_t>(kTile, area / std::max(vc, (int64_t)kTile)));
        vc = piece(vp, std::max(vc, area / std::max(rc, (int64_t)kTile)));
        split_k(rc / kTile * (dq / kTile), vc, &zf, &share_f);
        split_k(vc / kTile * (dq / kTile), rc, &zt, &share_t);
        // scores: about 4096 workgroups, where that leaves 8 tiles each
        const int64_t tiles = vp / kTile, groups = np_rows / kTile;
        const int64_t want = std::max<int64_t>(
            1, std::min(tiles / (groups < 64 ? 1 : 8), (4096 + groups - 1) / std::max<int64_t>(groups, 1)));
        share = (int)((tiles + want - 1) / want);
        shares = (int)((tiles + share - 1) / share);
        Carve c(base);
        F = c.take<bf16>((size_t)np * np_rows * dq);
        T = c.take<bf16>((size_t)np * vp * dq);
        part = c.take<float2>((size_t)shares * 2 * np_rows);
        score = c.take<float>((size_t)np_rows);
        label = c.take<int32_t>((size_t)np_rows);
        G = nullptr;
        lse2 = weight = slices = sum_f = sum_t = nullptr;
        if (grad) {
            lse2 = c.take<float>((size_t)np_rows);
            weight = c.take<float>((size_t)np_rows);
            G = c.take<bf16>((size_t)np * rc * vc);
            slices = c.take<float>(std::max((size_t)(zf > 1 ? zf : 0) * rc * dq,
                                            (size_t)(zt > 1 ? zt : 0) * vc * dq));
            sum_f = c.take<float>(vp > vc ? (size_t)rc * dq : 0);
            sum_t = c.take<float>(np_rows > rc ? (size_t)vp * dq : 0);
        }
        bytes = c.bytes();
    }
};

template <typename T, int NP>
hipError_t loss_run(const LossArgs& a, bool grad, hipStream_t st) {
    const LossPlan w(a.ws, a.n, a.rows, a.dim, a.dtype, grad);
    const int64_t nr = w.np_rows;
    const float scale2 = a.scale * kLog2e;
    k_parts<T, NP><<<blocks_for((nr + w.vp) * w.dq / 8), kThreads, 0, st>>>(
        a, nr, w.vp, w.dq, w.label, w.weight, reinterpret_cast<quad*>(w.F),
        reinterpret_cast<quad*>(w.T));
    GS_LAUNCHED();
    const Mat F{w.F, w.dq, nr * w.dq}, Tm{w.T, w.dq, w.vp * w.dq};
    const SpotGrid gs(nr / kTile, w.shares, kSpot);
    k_loss_scores<NP><<<gs.blocks, kThreads, 0, st>>>(F, Tm, w.kd, a.rows, scale2, w.label, nr,
                                                      (int)(w.vp / kTile), w.share, gs.gy, w.part,
                                                      w.score);
    GS_LAUNCHED();
    k_loss_join<<<blocks_of(nr, 32), kThreads, 0, st>>>(a, w.part, w.shares * 2, nr, w.score,
                                                        w.lse2);
    hipError_t e = hipGetLastError();
    if (!grad || e != hipSuccess) return e;
    for (int64_t r0 = 0; r0 < nr; r0 += w.rc) {
        const int64_t rc = std::min(w.rc, nr - r0);
        for (int64_t v0 = 0; v0 < w.vp; v0 += w.vc) {
            const int64_t vc = std::min(w.vc, w.vp - v0);
            // 8 tiles a workgroup where that leaves two workgroups a compute unit
            const int share = (int)std::max<int64_t>(
                1, std::min<int64_t>(8, rc / kTile * (vc / kTile) / 512));
            const SpotGrid gg(rc / kTile, (vc / kTile + share - 1) / share, kSpot);
            k_loss_g<NP><<<gg.blocks, kThreads, 0, st>>>(F, Tm, w.kd, a.rows, scale2, w.label,
                                                         w.weight, w.lse2, r0, v0, rc, vc, share,
                                                         gg.gy, w.G);
            GS_LAUNCHED();
            const Mat G{w.G, vc, rc * vc};
            const int zf = (int)((vc + w.share_f - 1) / w.share_f);
            const SumOut<T> of{w.slices, w.sum_f, v0 == 0, v0 + vc >= w.vp, rc, w.dq,
                               static_cast<T*>(a.dfeat) + r0 * a.dfeat_stride, a.n - r0,
                               a.dfeat_stride, a.dim, w.label + r0};
            k_loss_sum<T, NP, true>
                <<<SpotGrid(rc / kTile * zf, w.dq / kTile, w.dq).blocks, kThreads, 0, st>>>(
                    G, {w.T + v0 * w.dq, w.dq, w.vp * w.dq}, vc, w.share_f, zf, of);
            GS_LAUNCHED();
            if (zf > 1 && (e = fold(of, zf, st)) != hipSuccess) return e;
            const int zt = (int)((rc + w.share_t - 1) / w.share_t);
            const SumOut<T> ot{w.slices, w.sum_t + (w.sum_t != nullptr ? v0 * w.dq : 0), r0 == 0,
                               r0 + rc >= nr, vc, w.dq,
                               static_cast<T*>(a.dtable) + v0 * a.dtable_stride, a.rows - v0,
                               a.dtable_stride, a.dim, nullptr};
            k_loss_sum<T, NP, false>
                <<<SpotGrid(vc / kTile * zt, w.dq / kTile, w.dq).blocks, kThreads, 0, st>>>(
                    G, {w.F + r0 * w.dq, w.dq, nr * w.dq}, rc, w.share_t, zt, ot);
            GS_LAUNCHED();
            if (zt > 1 && (e = fold(ot, zt, st)) != hipSuccess) return e;
        }
    }
    return hipGetLastError();
}

// Shares of the streamed side: whole rounds of workgroups on the chip, `at_once` of
// which it holds, with at least `least` tiles a share and at most `most` shares.
struct Shares {
    int count, tiles;
    Shares(int64_t queries, int per, int64_t tiles_all, int at_once, int least, int64_t most) {
        const int64_t groups = std::max<int64_t>(1, (queries + per - 1) / per);
        const int64_t cap =
            std::max<int64_t>(1, std::min(most, std::max<int64_t>(1, tiles_all / least)));
        // the fewest shares that leave at most a tenth of the last round empty, of those
        // that make no more than four rounds
        int64_t best = 1;
        double best_full = 0.0;
        for (int64_t want = 1; want <= cap && (want == 1 || groups * want <= 4 * at_once); ++want) {
            const int64_t all = groups * want;
            const double full = (double)all / (double)((all + at_once - 1) / at_once * at_once);
            if (full > best_full + 1e-9) {
                best = want;
                best_full = full;
            }
            if (full >= 0.9) break;
        }
        tiles = (int)((tiles_all + best - 1) / best);
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
    // workgroups that the chip holds
    static int at_once(int ks, int role) { return one_a_unit(ks, role) ? 256 : 512; }
    // partial sums of the gradients: at most 64 MB a side
    static int64_t most(int64_t rows, int kd) {
        return std::max<int64_t>(1, ((int64_t)1 << 24) / std::max<int64_t>(1, rows * kd));
    }
    StreamPlan(void* base, int64_t n, int64_t rows, int np, int ks, bool grad)
        : tf((n + 31) / 32), tt((rows + 31) / 32),
          scores(n, np == 1 ? 256 : 128, tt, at_once(ks, kScores), 4, 512),
          by_feat(n, np == 1 ? 256 : 128, tt, at_once(ks, kGradFeat), 4,
                  most(n, padded_dim(ks))),
          by_table(rows, np == 1 ? 256 : 128, tf, at_once(ks, kGradTable), 4,
                   most(rows, padded_dim(ks))) {
        Carve c(base);
        const int kd = padded_dim(ks);
        const size_t first = (size_t)np * ks / 16 * 64;
        const size_t tile = first + (grad ? (size_t)np * kd / 16 * 64 : 0);
        T = c.take<quad>((tt + 4) * tile);
        const int shares = grad ? by_feat.count : scores.count;
        part = c.take<float2>(shares > 1 ? (size_t)shares * n : 0);
        score = c.take<float>(shares > 1 ? (size_t)n : 0);
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

template <typename T, int NP, int KS, int ROLE>
hipError_t launch_stream(const StreamArgs& a, const Shares& sh, hipStream_t st) {
    constexpr size_t lds = StreamShape<T, NP, KS, ROLE>::kLds;
    if (lds > 65536) {  // above the default limit of a launch
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void*>(&k_stream<T, NP, KS, ROLE>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    constexpr int kQueries = 128 * kBlocks<NP>;
    k_stream<T, NP, KS, ROLE><<<dim3((unsigned)((a.nq + kQueries - 1) / kQueries),
                                     (unsigned)sh.count), kThreads, lds, st>>>(a);
    return hipGetLastError();
}

template <typename T, int NP, int KS>
hipError_t stream_run(const LossArgs& a, bool grad, hipStream_t st) {
    const StreamPlan w(a.ws, a.n, a.rows, NP, KS, grad);
    const T* feat = static_cast<const T*>(a.feat);
    const T* table = static_cast<const T*>(a.table);
    if (grad)
        k_operands<T, NP, KS, true><<<blocks_of(w.tt, 1), kThreads, 0, st>>>(
            table, a.rows, a.table_stride, a.dim, a, nullptr, nullptr, nullptr, w.T);
    else
        k_operands<T, NP, KS, false><<<blocks_of(w.tt, 1), kThreads, 0, st>>>(
            table, a.rows, a.table_stride, a.dim, a, nullptr, nullptr, nullptr, w.T);
    GS_LAUNCHED();
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
    s.part = w.part;
    s.label_score = w.score;
    s.loss = a.loss;
    s.lse = a.lse;
    s.lse2_out = w.lse2;
    s.padded = a.n;
    hipError_t e;
    constexpr int DD = padded_dim(KS), kFirst = NP * KS / 16 * 64;
    if (!grad) {
        s.tile_stride = kFirst;
        s.share = w.scores.tiles;
        e = launch_stream<T, NP, KS, kScores>(s, w.scores, st);
        if (e == hipSuccess && w.scores.count > 1) {
            k_loss_join<<<blocks_of(a.n, 32), kThreads, 0, st>>>(a, w.part, w.scores.count, a.n,
                                                                 w.score, nullptr);
            e = hipGetLastError();
        }
        return e;
    }
    s.tile_stride = kFirst + NP * DD / 16 * 64;
    s.table = table;
    s.table_stride = a.table_stride;
    s.row_weight = a.row_weight;
    s.scale = a.scale;
    s.share = w.by_feat.tiles;
    s.out = a.dfeat;
    s.out_stride = a.dfeat_stride;
    s.sums = w.sums;
    e = launch_stream<T, NP, KS, kGradFeat>(s, w.by_feat, st);
    if (e != hipSuccess) return e;
    if (w.by_feat.count > 1)
        e = w.by_feat.count > 16 ? feat_join<T, DD, 8>(s, w.by_feat.count, st)
                                 : feat_join<T, DD, 1>(s, w.by_feat.count, st);
    if (e != hipSuccess) return e;
    k_operands<T, NP, KS, true><<<blocks_of(w.tf, 1), kThreads, 0, st>>>(
        feat, a.n, a.feat_stride, a.dim, a, w.label, w.weight, w.lse2, w.F);
    GS_LAUNCHED();
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
    e = launch_stream<T, NP, KS, kGradTable>(s, w.by_table, st);
    if (e != hipSuccess) return e;
    if (w.by_table.count > 1)
        return fold(SumOut<T>{w.sums, nullptr, 1, 1, a.rows, DD, static_cast<T*>(a.dtable), a.rows,
                       a.dtable_stride, a.dim, nullptr},
             w.by_table.count, st);
    return hipGetLastError();
}

// Padded row length that the streaming kernels take, 0: none. Past 128 a wave's own
// rows and sums leave it alone on its unit: 20000 x 8000 of 256 bf16 with gradients
// took 1073 us so, in pieces 511. Of 128 with gradients 361 against 344, fp32 (20000
// x 5000) 665 against 1019; losses alone (50000 x 20000) 319 against 390.
int stream_ks(int dim) {
    for (int ks : {16, 32, 48, 64, 128})
        if (dim <= ks) return ks;
    return 0;
}

// ---------------------------------------------------------------- few samples
// Losses of up to kFew samples, a picked pixel or a handful: the table is read once
// and nothing is laid out. `lpr` lanes take kFewRows table rows at a time, whose dot
// products with all samples, held in LDS in fp32, share one read of them; a
// workgroup's slots keep each sample's largest score and sum, and k_loss_join adds
// the workgroups up. Bound by the table's bytes in fp32 (or, below about 1 MB, by the two
// launches, 15 us with the call): 1 by 100000 of 512 fp32 45 us, 4.6 TB/s; a row at a
// time 114. Of bf16, half the bytes, 45 too: bound by the sums over lanes. 8 by 100000 of 64 fp32 30 us, by streaming 34; one 19 and 37.
constexpr int kFew = 8;
constexpr int kFewValues = 12288;  // samples * dim in LDS: 48 KB
constexpr int kFewRows = 4;

template <typename T, int VEC, int NQ>
__global__ __launch_bounds__(kThreads) void k_loss_few(LossArgs a, int lpr, float scale2,
                                                       float2* part, float* label_score) {
    __shared__ float f[kFewValues];
    __shared__ float2 lds[kThreads / 64][NQ];
    const int n = (int)a.n, dim = a.dim;
    const T* feat = static_cast<const T*>(a.feat);
    const T* table = static_cast<const T*>(a.table);
    for (int e = threadIdx.x; e < n * dim; e += kThreads)
        f[e] = to_float(feat[(int64_t)(e / dim) * a.feat_stride + e % dim]);
    int32_t y[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
        y[q] = q < n ? load_id(a.labels, a.labels64, q, a.rows,
                               blockIdx.x == 0 && threadIdx.x == 0 ? a.flags : nullptr)
                     : -1;
    __syncthreads();
    const int slots = kThreads / lpr, slot = threadIdx.x / lpr, lane = threadIdx.x % lpr;
    const int64_t step = (int64_t)gridDim.x * slots;
    float m[NQ], sum[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q] = kLowest;
        sum[q] = 0.0f;
    }
    for (int64_t v0 = (int64_t)blockIdx.x * slots + slot; v0 < a.rows; v0 += kFewRows * step) {
        float dot[kFewRows][NQ];
#pragma unroll
        for (int u = 0; u < kFewRows; ++u)
#pragma unroll
            for (int q = 0; q < NQ; ++q) dot[u][q] = 0.0f;
        for (int c = lane * VEC; c < dim; c += lpr * VEC) {
            float t[kFewRows][VEC];
            const int w = min(VEC, dim - c);
#pragma unroll
            for (int u = 0; u < kFewRows; ++u) {
                // past the table: the first of the rows again, the products unused
                const int64_t v = v0 + u * step < a.rows ? v0 + u * step : v0;
                const T* row = table + v * a.table_stride + c;
                if (w == VEC) {
                    load_any<VEC>(row, t[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) t[u][j] = j < w ? to_float(row[j]) : 0.0f;
                }
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                if (q >= n) break;
                float x[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[j] = j < w ? f[q * dim + c + j] : 0.0f;
#pragma unroll
                for (int u = 0; u < kFewRows; ++u)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dot[u][q] = fmaf(t[u][j], x[j], dot[u][q]);
            }
        }
        for (int o = 1; o < lpr; o <<= 1)
#pragma unroll
            for (int u = 0; u < kFewRows; ++u)
#pragma unroll
                for (int q = 0; q < NQ; ++q) dot[u][q] += __shfl_xor(dot[u][q], o, 64);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            if (q >= n) break;
            float mm = m[q];
#pragma unroll
            for (int u = 0; u < kFewRows; ++u) {
                const int64_t v = v0 + u * step;
                dot[u][q] = v < a.rows ? dot[u][q] * scale2 : -INFINITY;
                if (v == y[q] && lane == 0) label_score[q] = dot[u][q];
                mm = fmaxf(mm, dot[u][q]);
            }
            const float base = mm < INFINITY ? mm : 0.0f;
            sum[q] *= __builtin_amdgcn_exp2f((m[q] < INFINITY ? m[q] : 0.0f) - base);
#pragma unroll
            for (int u = 0; u < kFewRows; ++u) sum[q] += __builtin_amdgcn_exp2f(dot[u][q] - base);
            m[q] = mm;
        }
    }
    // over the slots: within the wave, then the waves (the lanes of a slot agree)
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        if (q >= n) break;
        for (int o = lpr; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[q], o, 64), s2 = __shfl_xor(sum[q], o, 64);
            join_sums(m[q], sum[q], m2, s2);
        }
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][q] = make_float2(m[q], sum[q]);
    }
    __syncthreads();
    if (threadIdx.x < n) {
        float2 r = lds[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < kThreads / 64; ++k)
            join_sums(r.x, r.y, lds[k][threadIdx.x].x, lds[k][threadIdx.x].y);
        part[(int64_t)blockIdx.x * n + threadIdx.x] = r;
    }
}

// Of several samples the dot products' sums over lanes weigh with long bf16 rows, and
// their scores are left to the pieces: 2 by 100000 of 512 95 us so, 78 in pieces (8:
// 135 and 78), one 54 and 78. In fp32 8 took 111 and 232.
bool is_few(int64_t n, int dim, int dtype, bool grad) {
    return !grad && n <= kFew && n * dim <= kFewValues && (n == 1 || dtype == 0 || dim <= 128);
}

struct FewPlan {
    int lpr, blocks;
    float2* part;
    float* score;
    size_t bytes;
    FewPlan(void* base, int64_t n, int64_t rows, int dim, int dtype) {
        const int vec = dtype == 0 ? 4 : 8;
        lpr = 1;
        while (lpr < 64 && lpr * vec < dim) lpr *= 2;
        const int64_t slots = kThreads / lpr;
        blocks = (int)std::min<int64_t>(512, (rows + slots - 1) / slots);
        Carve c(base);
        part = c.take<float2>((size_t)blocks * n);
        score = c.take<float>((size_t)n);
        bytes = c.bytes();
    }
};

template <typename T>
hipError_t few_run(const LossArgs& a, hipStream_t st) {
    const FewPlan w(a.ws, a.n, a.rows, a.dim, a.dtype);
    constexpr int VEC = 16 / sizeof(T);
    const float scale2 = a.scale * kLog2e;
    if (a.n == 1)
        k_loss_few<T, VEC, 1><<<w.blocks, kThreads, 0, st>>>(a, w.lpr, scale2, w.part, w.score);
    else
        k_loss_few<T, VEC, kFew><<<w.blocks, kThreads, 0, st>>>(a, w.lpr, scale2, w.part, w.score);
    GS_LAUNCHED();
    k_loss_join<<<1, kThreads, 0, st>>>(a, w.part, w.blocks, a.n, w.score, nullptr);
    return hipGetLastError();
}

}  // namespace

size_t label_loss_ws(int64_t n, int64_t rows, int dim, int dtype, bool grad) {
    if (is_few(n, dim, dtype, grad)) return FewPlan(nullptr, n, rows, dim, dtype).bytes;
    const int ks = stream_ks(dim);
    if (ks != 0) return StreamPlan(nullptr, n, rows, dtype == 0 ? 3 : 1, ks, grad).bytes;
    return LossPlan(nullptr, n, rows, dim, dtype, grad).bytes;
}

hipError_t launch_label_loss(const LossArgs& a, bool grad, hipStream_t st) {
    if (a.n == 0) {  // no rows: the table's gradient is 0
        if (!grad) return hipSuccess;
        const int dq = (int)pad_to(a.dim, 4);
        if (a.dtype == 0)
            return fold(SumOut<float>{nullptr, nullptr, 1, 1, a.rows, dq,
                                      static_cast<float*>(a.dtable), a.rows, a.dtable_stride, a.dim,
                                      nullptr}, 0, st);
        return fold(SumOut<bf16>{nullptr, nullptr, 1, 1, a.rows, dq, static_cast<bf16*>(a.dtable),
                                 a.rows, a.dtable_stride, a.dim, nullptr}, 0, st);
    }
    const bool f = a.dtype == 0;
    if (is_few(a.n, a.dim, a.dtype, grad)) return f ? few_run<float>(a, st) : few_run<bf16>(a, st);
    switch (stream_ks(a.dim)) {
        case 16: return f ? stream_run<float, 3, 16>(a, grad, st) : stream_run<bf16, 1, 16>(a, grad, st);
        case 32: return f ? stream_run<float, 3, 32>(a, grad, st) : stream_run<bf16, 1, 32>(a, grad, st);
        case 48: return f ? stream_run<float, 3, 48>(a, grad, st) : stream_run<bf16, 1, 48>(a, grad, st);
        case 64: return f ? stream_run<float, 3, 64>(a, grad, st) : stream_run<bf16, 1, 64>(a, grad, st);
        case 128:
            return f ? stream_run<float, 3, 128>(a, grad, st) : stream_run<bf16, 1, 128>(a, grad, st);
        default: return f ? loss_run<float, 3>(a, grad, st) : loss_run<bf16, 1>(a, grad, st);
    }
}

}  // namespace gs
