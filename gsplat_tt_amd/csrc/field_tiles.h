// field_tiles.h - matrix products of the feature operators on the matrix cores: values
// cut into bf16 parts, 128 x 128 tiles that come from memory straight into LDS, and the
// order of workgroups over tiles.
#pragma once

#include "field_device.h"

namespace gs {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t quad;  // 16 bytes: one lane's operand

constexpr int kTileThreads = 256;
constexpr int kTile = 128;  // rows and columns of a workgroup's tile
constexpr int kStep = 64;   // summed index per step

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
// the product is what arithmetic gives, also of two infinite values. Bits of an fp32 value
// below bf16's least, 2^-133, are in no part (the matrix cores take subnormal operands as
// they are): values above 2^-110 have none, and one below 2^-133 counts as 0, here too.
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
// The products of parts: (0,0) for one part; for three, all with p + q <= 2. A value's second
// part is below 2^-7 of it and its third below 2^-15, so that the products left out are below
// 2^-21 of the values' product together, and of its sign (the parts are cut off, not rounded);
// 0.7 x 2^-24 of it on average over normally distributed values.
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

}  // namespace gs
