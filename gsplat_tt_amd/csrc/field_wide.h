// field_wide.h - large matrix products of the feature operators: tiles of 256 x 256 (bf16, a
// workgroup of 8 waves a CU) or 128 x 128 (fp32 in three parts, two of 4 waves).
//
// What bounds such a product is the way of the operands and the power that the matrix cores
// draw. 4096 x 512 over 100096 bf16, 420 GFLOP: the products alone take 283 us (from registers;
// 174 at the clock that a lighter load runs at), the way from memory into LDS 253 (342 with
// tiles of 128 x 256: the caches give some 13 TB/s to all CUs), the reads of LDS 163, all
// together 398, since a workgroup's waves read and multiply at the same time. Not faster:
// waves that take turns (400), steps of 32 with four in LDS (409), operands read a step
// ahead (they do not fit the registers: 883), tiles of 128 x 256 with two workgroups (410).
//
// The loads into LDS are written as assembly, which the compiler does not count: with its
// builtin every read of LDS would wait for all of them. They have no output registers, and
// a step waits for them itself.
#pragma once

#include "field_tiles.h"

namespace gs {

// An operand: rows of ld elements; a row past `rows` and a column past `cols` is read as
// zeros, from `zero` (16 bytes). Both are multiples of 8 in the direction of the rows'
// values, and so are all offsets.
struct WideMat {
    const bf16* p;
    int64_t ld, plane;
    int64_t rows, cols;
    const void* zero;
};

// m0 is a reserved register to the compiler, which says so; it keeps nothing in it here.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    // an SGPR that a vector instruction has written needs 5 wait states before the load
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds),
                 "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(const void* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds),
                 "v"(at)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// This wave's loads have arrived and its reads of LDS are done, then the others'.
__device__ __forceinline__ void step_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// This wave's reads of LDS are done, then the others'.
__device__ __forceinline__ void read_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const quad* p) {
    typedef const __attribute__((address_space(3))) quad* lds_t;
    return (uint32_t)(uintptr_t)(lds_t)p;
}

// 128 rows and 32 H of the summed index of one operand in LDS (512 H quads). K: the matrix's
// rows hold the summed index, 4 H quads a row, placed so that the 8 lanes that read one
// column of rows r .. r + 3, or r .. and r + 16 .. (SPREAD), touch all banks once. Not K: the
// matrix's rows are the summed index, as in Side.
template <bool K, int H, bool SPREAD, int THREADS>
struct Face {
    static constexpr int kQuads = 512 * H;
    __device__ __forceinline__ static uint32_t place(uint32_t row) {
        if (!K) return (row & 3) | ((row ^ (row >> 1)) & 4);
        if (H == 1) return SPREAD ? ((row >> 1) & 1) | ((row >> 3) & 2) : (row >> 1) & 3;
        return SPREAD ? (row & 3) | ((row >> 2) & 4) : row & 7;
    }
    // The thread's quad of a sweep of THREADS: row and column (in elements) within the face
    __device__ __forceinline__ static uint32_t row_of() {
        return K ? threadIdx.x / (4 * H) : threadIdx.x >> 4;
    }
    __device__ __forceinline__ static uint32_t col_of() {
        const uint32_t r = row_of();
        return (K ? (threadIdx.x & (4 * H - 1)) ^ place(r) : (threadIdx.x & 15) ^ (place(r) << 1)) * 8;
    }
    static constexpr int kSweepRows = K ? THREADS / (4 * H) : THREADS / 16, kSweeps = kQuads / THREADS;

    // Into LDS at `to`, from the lane's offset past p, all of it in the matrix.
    __device__ __forceinline__ static void fetch(const char* p, int64_t sweep, uint32_t offset,
                                                 uint32_t to) {
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) load_to_lds(p + j * sweep, offset, to + j * THREADS * 16);
    }
    // The same at the matrix's edges: row r0, column c0 of it, zeros past them.
    __device__ __forceinline__ static void fetch_edge(const WideMat& m, int part, int64_t r0,
                                                      int64_t c0, uint32_t to) {
        const bf16* p = m.p + part * m.plane + r0 * m.ld + c0;
#pragma unroll
        for (int j = 0; j < kSweeps; ++j) {
            const uint32_t r = j * kSweepRows + row_of();
            const bool in = r0 + r < m.rows && c0 + col_of() < m.cols;
            load_to_lds(in ? static_cast<const void*>(p + r * m.ld + col_of()) : m.zero,
                        to + j * THREADS * 16);
        }
    }
    // The operand of block i of 16 rows from row b, summed index 32 h .. + 31. SPREAD:
    // of 64 rows from b, block i has the rows 16 (s / 4) + 4 i + s % 4.
    __device__ __forceinline__ static bf16x8 operand(const quad* lds, int b, int i, int h) {
        const uint32_t lane = threadIdx.x & 63, g = lane >> 4, s = lane & 15;
        if (K) {
            const uint32_t row = SPREAD ? (s >> 2) * 16 + (s & 3) : s;
            const quad* at = lds + row * (4 * H) + ((g ^ place(row)) ^ (h * 4));
            return __builtin_bit_cast(bf16x8, at[(b + (SPREAD ? i * 4 : i * 16)) * (4 * H)]);
        }
        typedef __attribute__((ext_vector_type(4))) short s16x4;
        typedef __attribute__((address_space(3))) s16x4* lds4;
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

// One side's faces of a workgroup, U of 128 rows, fetched step by step along the summed
// index: what changes from step to step is one address, since a step's scalar instructions
// come before its products in every wave.
template <class F, bool K, int H, int U, int NP>
struct Feed {
    const WideMat& m;
    const char* p;      // the next step's
    int64_t row0, k;    // the tile's first row; the next step's summed index
    int64_t step, sweep;  // bytes
    int whole;          // steps left that lie in the matrix as a whole
    uint32_t off[U];
    __device__ __forceinline__ explicit Feed(const WideMat& mat) : m(mat) {
        step = (K ? 32 * H : 32 * H * m.ld) * 2;
        sweep = F::kSweepRows * m.ld * 2;
#pragma unroll
        for (int u = 0; u < U; ++u)
            off[u] = (F::row_of() * (uint32_t)m.ld + F::col_of() +
                      u * 128 * (K ? (uint32_t)m.ld : 1u)) * 2;
    }
    __device__ __forceinline__ void start(int64_t row, int64_t k0, int steps) {
        row0 = row;
        k = k0;
        p = reinterpret_cast<const char*>(m.p + (K ? row * m.ld + k0 : k0 * m.ld + row));
        const int64_t last = K ? m.rows : m.cols, along = K ? m.cols : m.rows;
        whole = row + 128 * U <= last ? (int)min((int64_t)steps, (along - k0) / (32 * H)) : 0;
    }
    __device__ __forceinline__ void fetch(uint32_t to) {
        if (whole > 0) {
#pragma unroll
            for (int part = 0; part < NP; ++part)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    F::fetch(p + part * m.plane * 2, sweep, off[u], to + (part * U + u) * F::kQuads * 16);
        } else {
#pragma unroll
            for (int part = 0; part < NP; ++part)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t row = row0 + u * 128;
                    F::fetch_edge(m, part, K ? row : k, K ? k : row,
                                  to + (part * U + u) * F::kQuads * 16);
                }
        }
        --whole;
        p += step;
        k += 32 * H;
    }
};

// NP: parts of a value. WA x WB waves of AB x BB blocks of 16 rows; steps of 32 H of the
// summed index, S of them in LDS. fp32's parts fill LDS with one: its operands go into
// registers before the next step's are fetched.
template <int NP, int AB>
struct WideShape {
    static constexpr int WA = 2, WB = NP == 1 ? 4 : 2, BB = 4, H = NP == 1 ? 2 : 1, S = NP == 1 ? 2 : 1;
    static constexpr int kThreads = 64 * WA * WB;
    static constexpr int kRows = WA * AB * 16, kCols = WB * BB * 16;  // a tile's rows of A and B
    static constexpr int kQuads = S * NP * (kRows + kCols) / 128 * 512 * H;  // of LDS
    // the wave's first row of either
    __device__ __forceinline__ static int row() { return wave_id() / WB * (AB * 16); }
    __device__ __forceinline__ static int col() { return wave_id() % WB * (BB * 16); }
};

// Tiles of A B^T one after the other for one workgroup. `rows(tile)` gives the tile's first
// rows; `ahead(tile)` is called a step before the tile's last products, `done(tile, acc)` takes
// the wave's sums (rows of A in 64s, SPREAD as above).
template <int NP, int AB, bool AK, bool BK, bool SPREAD, class Rows, class Ahead, class Done>
__device__ __forceinline__ void wide_products(const WideMat& A, const WideMat& B, int64_t k0,
                                              int64_t k1, int tiles, quad* lds, Rows rows,
                                              Ahead ahead, Done done) {
    using Shape = WideShape<NP, AB>;
    constexpr int BB = Shape::BB, H = Shape::H, S = Shape::S, T = Shape::kThreads;
    constexpr int AU = Shape::kRows / 128, BU = Shape::kCols / 128;
    using FaceA = Face<AK, H, SPREAD, T>;
    using FaceB = Face<BK, H, false, T>;
    constexpr int Q = FaceA::kQuads, STAGE = NP * (AU + BU) * Q;
    const int wa = Shape::row(), wb = Shape::col();
    const uint32_t base = lds_address(lds) + wave_id() * 1024;
    const int per_tile = (int)((k1 - k0) / (32 * H)), steps = per_tile * tiles;
    Feed<FaceA, AK, H, AU, NP> feed_a(A);
    Feed<FaceB, BK, H, BU, NP> feed_b(B);
    int tile_f = 0, left_f = 0;  // of the next step to fetch
    auto fetch = [&](int stage) {
        if (left_f == 0) {
            const auto at = rows(tile_f++);
            feed_a.start(at.m, k0, per_tile);
            feed_b.start(at.n, k0, per_tile);
            left_f = per_tile;
        }
        --left_f;
        const uint32_t to = base + stage * (STAGE * 16);
        feed_a.fetch(to);
        feed_b.fetch(to + NP * AU * Q * 16);
    };
    f32x4 acc[AB][BB];
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < AB; ++i)
#pragma unroll
            for (int j = 0; j < BB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    if (steps > 0) fetch(0);
    int left = per_tile, tile = 0;
    for (int s = 0; s < steps; ++s) {
        step_barrier();
        // into the stage that the step before has read
        if (S == 2 && s + 1 < steps) fetch((s + 1) & 1);
        if (left == 0) {  // the tile before
            done(tile++, acc);
            clear();
            left = per_tile;
        }
        if (left == 1) ahead(tile);
        --left;
        const quad* at = lds + (S == 2 ? s & 1 : 0) * STAGE;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            bf16x8 fa[NP][AB], fb[NP][BB];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const quad* la = at + (p * AU + (wa >> 7)) * Q;
                const quad* lb = at + (NP * AU + p * BU + (wb >> 7)) * Q;
#pragma unroll
                for (int j = 0; j < BB; ++j) fb[p][j] = FaceB::operand(lb, wb & 64, j, h);
#pragma unroll
                for (int i = 0; i < AB; ++i)
                    fa[p][i] = FaceA::operand(la, (wa & 64) + i / 4 * 64, i % 4, h);
            }
            if (S == 1) {
                read_barrier();
                if (s + 1 < steps) fetch(0);
            }
#pragma unroll
            for (int q = 0; q < Products<NP>::kCount; ++q)
#pragma unroll
                for (int i = 0; i < AB; ++i)
#pragma unroll
                    for (int j = 0; j < BB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            fa[Products<NP>::a(q)][i], fb[Products<NP>::b(q)][j], acc[i][j], 0, 0, 0);
        }
    }
    done(tile, acc);
}

}  // namespace gs
