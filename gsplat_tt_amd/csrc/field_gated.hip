// field_gated.hip - gated projections of features, forward and backward.
//
//   gate = x Wg^T + bg;  up = x Wu^T + bu;  h = act(gate) up
// and, from dh:
//   dgate = dh up act'(gate);  dup = dh act(gate);
//   dx = dgate Wg + dup Wu;  dWg = dgate^T x;  dWu = dup^T x;  db = column sums.
//
// The backward pass makes gate and up again: keeping them would cost 2 n hidden values
// written and read against 4 n dim hidden operations (in fp32 50021 x 256 to 1024 820 MB, 160
// us at a copy's rate, against 276 of products; such a form was not built).
//
// All products run on the matrix cores with bf16 operands and fp32 sums; fp32 values are
// cut into three bf16 parts, whose six largest products are added up (field_tiles.h).
// For bf16 inputs dgate and dup are rounded to bf16 as operands of the next products, as they
// are where gate and up are bf16 tensors with gradients of their own: 100003 x 512 to 2048 the
// gradients are 0.0024 off (2-norm, relative), where rounding them alone gives 0.0017. A
// second part of them would take that away for twice the products of dx and dW, 840 of 1950
// us there, and twice the bytes of [dgate, dup]. The biases' gradients sum what was not
// rounded, in fp32.
//
// Four ways, by size:
//   few     up to 64 rows: one launch, operands straight from memory (with gradients of long
//           rows, their first part).
//   short   rows of up to 128 (field_gated_short.h): rows in registers, weights through LDS; dx
//           in a pass over the weights, the weights' gradients in one over the rows, and
//           [dgate, dup] made in both, which costs 8 n dim hidden operations but not 12 bytes
//           a value.
//   wide    longer rows, many tiles: 256 x 256 (fp32 128 x 128), [dgate, dup] of one piece of the
//           rows at a time in the workspace.
//   tiles   what is between: 128 x 128, all operands laid out before.
// All sums are made in an order that depends on the sizes alone.
#include <type_traits>

#include "field_gated.h"
#include "field_wide.h"

namespace gs {

namespace {

constexpr int kThreads = kTileThreads;

int64_t pad_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Both weights as one matrix of rows r: 64 of them hold 32 gate rows, then the same 32 up
// rows, so that a wave's 64 x 64 tile has both projections of a hidden unit. Within 32,
// block i of 16 takes the units 8 (s / 4) + 4 i + s % 4: a lane's sums of two blocks are
// 8 units in a row.
struct UnitOf {
    int64_t unit;
    bool up;
};
__device__ __forceinline__ UnitOf unit_of(int64_t r) {
    const int t = (int)(r & 63), s = t & 15;
    return {(r >> 6) * 32 + (s >> 2) * 8 + ((t >> 4) & 1) * 4 + (s & 3), t >= 32};
}

// The gate row of a unit that is a multiple of 4; its up row is 32 on.
__device__ __forceinline__ int64_t row_of_unit(int64_t u) {
    return (u >> 5) * 64 + ((u >> 2) & 1) * 16 + ((u >> 3) & 3) * 4;
}

// Parts of x's rows from n0 as (nr, ld), or of the weights in the order above; zeros in
// the padding.
template <typename T, int NP, bool WEIGHTS>
__global__ __launch_bounds__(kThreads) void k_gated_parts(GatedArgs a, int64_t n0, int64_t nr,
                                                          int ld, quad* out) {
    const int units = ld / 8;
    const int64_t total = nr * units;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t r = e / units;
        const int c = (int)(e - r * units) * 8;
        quad part[NP];
        if (WEIGHTS) {
            const UnitOf u = unit_of(r);
            const bool on = u.unit < a.hidden;
            const T* w = static_cast<const T*>(u.up ? a.w_up : a.w_gate);
            load_parts<T, NP>(w + (on ? u.unit : 0) * (u.up ? a.up_stride : a.gate_stride), a.dim,
                              c, on, part);
        } else {
            const bool on = n0 + r < a.n;
            load_parts<T, NP>(static_cast<const T*>(a.x) + (on ? n0 + r : 0) * a.x_stride, a.dim,
                              c, on, part);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) out[p * total + e] = part[p];
    }
}

// The projections of one tile and what follows from them: h, or with GRAD the operand
// rows [dgate, dup] (in the weights' order) of the samples and the biases' sums over each
// wave's 64 samples.
template <typename T, int NP, int ACT, bool GRAD>
__global__ __launch_bounds__(kThreads, 2) void k_gated(GatedArgs a, Mat X, Mat W, int kd,
                                                       int64_t n0, int64_t nr, int64_t wr, int gy,
                                                       bf16* dz, float* db) {
    GS_TILE_LDS;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64, g = lane >> 4, s = lane & 15;
    const Spot at = spot((int)(nr / kTile), gy);
    const int64_t r0 = (int64_t)at.y * kTile, s0 = (int64_t)at.x * kTile;
    if (r0 >= wr) return;
    tile_products<NP, true, true>(
        W, X, 0, kd, 1, lds, [&](int) { return TileRows{r0, s0}; },
        [&](int, f32x4(&acc)[4][4]) {
            const int64_t u0 = (r0 + wm) / 2 + g * 8;  // the lane's first hidden unit
            float bg[8], bu[8], sg[8], su[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool on = u0 + k < a.hidden;
                bg[k] = on && a.b_gate != nullptr ? a.b_gate[u0 + k] : 0.0f;
                bu[k] = on && a.b_up != nullptr ? a.b_up[u0 + k] : 0.0f;
                sg[k] = su[k] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t row = s0 + wn + j * 16 + s, i = n0 + row;
                float zg[8], zu[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    zg[k] = acc[k / 4][j][k % 4] + bg[k];
                    zu[k] = acc[2 + k / 4][j][k % 4] + bu[k];
                }
                if (!GRAD) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) zg[k] = act<ACT>(zg[k]) * zu[k];
                    if (i < a.n) store_cols<8>(static_cast<T*>(a.h) + i * a.h_stride, u0, a.hidden, zg);
                } else {
                    float d[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) d[k] = 0.0f;
                    if (i < a.n)
                        load8(static_cast<const T*>(a.dh) + i * a.dh_stride, u0, a.hidden, d);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const bool on = i < a.n && u0 + k < a.hidden;
                        const float z = zg[k], u = zu[k];
                        zg[k] = on ? d[k] * u * act_slope<ACT>(z) : 0.0f;
                        zu[k] = on ? d[k] * act<ACT>(z) : 0.0f;
                        sg[k] += zg[k];
                        su[k] += zu[k];
                    }
                    // 4 units of block 0, 4 of block 1, for either
                    quad pg[NP], pu[NP];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        zg[k] = plain_input<NP>(zg[k]);
                        zu[k] = plain_input<NP>(zu[k]);
                    }
                    split8_input<NP>(zg, pg);
                    split8_input<NP>(zu, pu);
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        uint2* to = reinterpret_cast<uint2*>(dz + (p * nr + row) * wr + r0 + wm + g * 4);
                        to[0] = make_uint2(pg[p][0], pg[p][1]);
                        to[4] = make_uint2(pg[p][2], pg[p][3]);
                        to[8] = make_uint2(pu[p][0], pu[p][1]);
                        to[12] = make_uint2(pu[p][2], pu[p][3]);
                    }
                }
            }
            if (GRAD && db != nullptr) {
#pragma unroll
                for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        sg[k] += __shfl_xor(sg[k], o, 64);
                        su[k] += __shfl_xor(su[k], o, 64);
                    }
                if (s == 0) {
                    float* to = db + ((s0 + wn) / 64) * wr + r0 + wm + g * 4;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        to[(k / 4) * 16 + k % 4] = sg[k];
                        to[32 + (k / 4) * 16 + k % 4] = su[k];
                    }
                }
            }
        });
}

// dx of one tile: the weights' columns against the samples' [dgate, dup]; of several shares of
// these (blockIdx.y) each leaves its sums in `part` (share, samples, ld).
template <typename T, int NP>
__global__ __launch_bounds__(kThreads, 2) void k_gated_dx(GatedArgs a, Mat W, Mat Z, int64_t n0,
                                                          int64_t nr, int ld, int64_t wr, int gy,
                                                          int64_t per_share, float* part) {
    GS_TILE_LDS;
    const int64_t k0 = min(wr, blockIdx.y * per_share), k1 = min(wr, k0 + per_share);
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const Spot at = spot((int)(nr / kTile), gy);
    const int64_t c0 = (int64_t)at.y * kTile, s0 = (int64_t)at.x * kTile;
    if (c0 >= ld) return;
    tile_products<NP, false, true>(
        W, Z, k0, k1, 1, lds, [&](int) { return TileRows{c0, s0}; },
        [&](int, f32x4(&acc)[4][4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t r = s0 + wn + j * 16 + (lane & 15), i = n0 + r;
                if (gridDim.y > 1) {
                    f32x4* to = reinterpret_cast<f32x4*>(part + (blockIdx.y * nr + r) * ld + c0 + wm);
#pragma unroll
                    for (int k = 0; k < 4; ++k) to[k * 4 + (lane >> 4)] = acc[k][j];
                    continue;
                }
                if (i >= a.n) continue;
                T* row = static_cast<T*>(a.dx) + i * a.dx_stride;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float v[4] = {acc[k][j][0], acc[k][j][1], acc[k][j][2], acc[k][j][3]};
                    store_cols<4>(row, c0 + wm + k * 16 + (lane >> 4) * 4, a.dim, v);
                }
            }
        });
}

// 4 columns of dx a thread, summed over the parts in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_gated_dx_join(GatedArgs a, const float* part,
                                                            int shares, int64_t rows, int ld,
                                                            int64_t n0, int64_t n) {
    const int units = (a.dim + 3) / 4;
    const int64_t total = n * units;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t i = e / units;
        const int c = (int)(e - i * units) * 4;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int k = 0; k < shares; ++k)
            v += *reinterpret_cast<const f32x4*>(part + (k * rows + i) * ld + c);
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_cols<4>(static_cast<T*>(a.dx) + (n0 + i) * a.dx_stride, c, a.dim, o);
    }
}

// One tile of the weights' gradients, over a share of the samples; with `add` onto what an
// earlier piece left.
template <int NP>
__global__ __launch_bounds__(kThreads, 2) void k_gated_dw(Mat X, Mat Z, int64_t nr, int ld,
                                                          int64_t wr, int64_t per_share, int add,
                                                          float* part) {
    GS_TILE_LDS;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const int cols = ld / kTile;
    const int64_t c0 = (int64_t)(blockIdx.x % cols) * kTile;
    const int64_t r0 = (int64_t)(blockIdx.x / cols) * kTile;
    const int64_t k0 = min(nr, blockIdx.y * per_share), k1 = min(nr, k0 + per_share);
    tile_products<NP, false, false>(
        X, Z, k0, k1, 1, lds, [&](int) { return TileRows{c0, r0}; },
        [&](int, f32x4(&acc)[4][4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t r = r0 + wn + j * 16 + (lane & 15);
                f32x4* to = reinterpret_cast<f32x4*>(part + (blockIdx.y * wr + r) * ld + c0 + wm);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f32x4 v = acc[k][j];
                    if (add) v += to[k * 4 + (lane >> 4)];
                    to[k * 4 + (lane >> 4)] = v;
                }
            }
        });
}

// The shares' sums as the weights' gradients, and the sums over blocks of samples as the
// biases' (onto what an earlier piece left with `add`): 64 quads of columns a workgroup, 16
// runs that are joined in order. WIDE: the weights' rows in the wide tiles' order.
template <typename T, bool WIDE, bool BIASES>
__global__ __launch_bounds__(1024) void k_gated_sum(GatedArgs a, const float* part, int shares,
                                                    int64_t wr, int ld, int add) {
    __shared__ f32x4 lds[16][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t quads = BIASES ? wr / 4 : wr * (ld / 4);
    const int per = (shares + 15) / 16, b0 = min(shares, run * per), b1 = min(shares, b0 + per);
    for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < quads; e0 += (int64_t)gridDim.x * 64) {
        const int64_t e = e0 + lane;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e < quads) {
            const f32x4* from = reinterpret_cast<const f32x4*>(part) + e;
#pragma unroll 8
            for (int b = b0; b < b1; ++b) v += from[b * quads];
        }
        __syncthreads();  // what was there has been read
        lds[run][lane] = v;
        __syncthreads();
        if (run != 0 || e >= quads) continue;
#pragma unroll
        for (int k = 1; k < 16; ++k) v += lds[k][lane];
        const int64_t r = BIASES ? e * 4 : e / (ld / 4);
        // a quad of rows has 4 units in a row, all gate or all up, in either order
        const UnitOf u = WIDE ? UnitOf{(r >> 4) * 8 + (r & 7), (r & 8) != 0} : unit_of(r);
        if (u.unit >= a.hidden) continue;
        if (BIASES) {
            float* out = u.up ? a.db_up : a.db_gate;
            if (out == nullptr) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (u.unit + k < a.hidden) out[u.unit + k] = add ? out[u.unit + k] + v[k] : v[k];
        } else {
            T* row = static_cast<T*>(u.up ? a.dw_up : a.dw_gate) +
                     u.unit * (u.up ? a.dup_stride : a.dgate_stride);
            const float o[4] = {v[0], v[1], v[2], v[3]};
            store_cols<4>(row, (e - r * (ld / 4)) * 4, a.dim, o);
        }
    }
}

// ---------------------------------------------------------------- wide tiles
// The same products in the tiles of field_wide.h, where there are enough of them to
// fill the chip. The weights' rows lie in groups of 16, 8 gate and the same 8 up rows, so
// that with spread blocks a lane's sums are 8 units in a row of both, and its dgate and dup
// 32 bytes in a row. bf16 rows of x that are aligned are read where they are.
//
// 100003 x 512 to 2048 bf16, 420 GFLOP each: h 487 us (the library's plain product, without
// activation, 613), dgate and dup 603, dx 472 (483), dW 370 (741); the matrix cores are
// busy 30 to 50 % of the time at 2.2 GHz. 50021 x 256 to 1024 fp32, 52 GFLOP in six products:
// 276 (509), 392, 310 (487), 227 (618); busy 35 to 69 %. What bounds them: field_wide.h; h,
// dgate and dup also by the activation, which a CU's only workgroup does between its
// products.
template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void k_wide_weights(GatedArgs a, int64_t wr, int ld,
                                                           quad* out, quad* zero) {
    const int units = ld / 8;
    const int64_t total = wr * units;
    if (blockIdx.x == 0 && threadIdx.x == 0) *zero = quad{0u, 0u, 0u, 0u};
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t r = e / units, unit = (r >> 4) * 8 + (r & 7);
        const bool on = unit < a.hidden, up = (r & 8) != 0;
        const T* w = static_cast<const T*>(up ? a.w_up : a.w_gate);
        quad part[NP];
        load_parts<T, NP>(w + (on ? unit : 0) * (up ? a.up_stride : a.gate_stride), a.dim,
                          (int)(e - r * units) * 8, on, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) out[p * total + e] = part[p];
    }
}

template <int NP>
constexpr int kWideBlocks = NP == 1 ? 8 : 4;  // of 16 rows of A, of a wave

template <typename T, int NP, int ACT, bool GRAD>
__global__ __launch_bounds__((WideShape<NP, 8>::kThreads), 2) void k_gated_wide(GatedArgs a, WideMat W, WideMat X,
                                                                int kd, int64_t n0, int64_t nr,
                                                                int tiles_w, int share, int gy,
                                                                bf16* dz, float* db) {
    constexpr int AB = kWideBlocks<NP>;
    using Shape = WideShape<NP, AB>;
    __shared__ quad lds[Shape::kQuads];
    const int lane = threadIdx.x & 63, g = lane >> 4, s = lane & 15;
    const Spot at = spot((int)(nr / Shape::kCols), gy);
    const int64_t s0 = (int64_t)at.x * Shape::kCols + Shape::col();
    const int t0 = at.y * share, t1 = min(tiles_w, t0 + share);
    if (t0 >= t1) return;
    const int64_t wr = W.rows;
    Raw<T> d[AB / 4][GRAD ? 4 : 1];
    auto row_of = [&](int t) { return (int64_t)(t0 + t) * Shape::kRows + Shape::row(); };
    wide_products<NP, AB, true, true, true>(
        W, X, 0, kd, t1 - t0, lds,
        [&](int t) { return TileRows{(int64_t)(t0 + t) * Shape::kRows, (int64_t)at.x * Shape::kCols}; },
        [&](int t) {
            if (!GRAD) return;
#pragma unroll
            for (int v = 0; v < AB / 4; ++v)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t i = n0 + s0 + j * 16 + s;
                    d[v][j].load_finished(
                        static_cast<const T*>(a.dh) + (i < a.n ? i : 0) * a.dh_stride,
                        (row_of(t) + v * 64) / 2 + g * 8, i < a.n ? a.hidden : 0);
                }
        },
        [&](int t, f32x4(&acc)[AB][Shape::BB]) {
#pragma unroll
            for (int v = 0; v < AB / 4; ++v) {
                const int64_t r0 = row_of(t) + v * 64, u0 = r0 / 2 + g * 8;
                const bool whole = r0 / 2 + 32 <= a.hidden;
                float bg[8], bu[8], sg[8], su[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bool on = u0 + k < a.hidden;
                    bg[k] = on && a.b_gate != nullptr ? a.b_gate[u0 + k] : 0.0f;
                    bu[k] = on && a.b_up != nullptr ? a.b_up[u0 + k] : 0.0f;
                    sg[k] = su[k] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t row = s0 + j * 16 + s, i = n0 + row;
                    float dg[8], du[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float zg = acc[v * 4 + k / 4][j][k % 4] + bg[k];
                        const float zu = acc[v * 4 + 2 + k / 4][j][k % 4] + bu[k];
                        if (!GRAD) {
                            dg[k] = act<ACT>(zg) * zu;
                        } else {
                            dg[k] = plain_input<NP>(d[v][j][k] * zu * act_slope<ACT>(zg));
                            du[k] = plain_input<NP>(d[v][j][k] * act<ACT>(zg));
                        }
                    }
                    if (!GRAD) {
                        if (i >= a.n) continue;
                        T* to = static_cast<T*>(a.h) + i * a.h_stride;
                        store_cols<8>(to, u0, a.hidden, dg);
                        continue;
                    }
                    if (!whole || i >= a.n) {  // what is infinite times a dh of 0 is NaN
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (i >= a.n || u0 + k >= a.hidden) dg[k] = du[k] = 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        sg[k] += dg[k];
                        su[k] += du[k];
                    }
                    quad pg[NP], pu[NP];
                    split8_input<NP>(dg, pg);
                    split8_input<NP>(du, pu);
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        quad* to = reinterpret_cast<quad*>(dz + (p * nr + row) * wr + r0 + g * 16);
                        to[0] = pg[p];
                        to[1] = pu[p];
                    }
                }
                if (GRAD && db != nullptr) {
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            sg[k] += __shfl_xor(sg[k], o, 64);
                            su[k] += __shfl_xor(su[k], o, 64);
                        }
                    if (s == 0) {
                        float* to = db + (s0 / 64) * wr + r0 + g * 16;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            to[k] = sg[k];
                            to[8 + k] = su[k];
                        }
                    }
                }
            }
        });
}

template <typename T, int NP, int AB>
__global__ __launch_bounds__((WideShape<NP, AB>::kThreads), 2) void k_wide_dx(GatedArgs a, WideMat W, WideMat Z,
                                                             int64_t n0, int64_t nr, int tiles_c,
                                                             int gy) {
    using Shape = WideShape<NP, AB>;
    __shared__ quad lds[Shape::kQuads];
    const int lane = threadIdx.x & 63;
    const Spot at = spot((int)(nr / Shape::kCols), gy);
    if (at.y >= tiles_c) return;
    const int64_t c0 = (int64_t)at.y * Shape::kRows, s0 = (int64_t)at.x * Shape::kCols;
    wide_products<NP, AB, false, true, false>(
        W, Z, 0, W.rows, 1, lds, [&](int) { return TileRows{c0, s0}; }, [](int) {},
        [&](int, f32x4(&acc)[AB][Shape::BB]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t i = n0 + s0 + Shape::col() + j * 16 + (lane & 15);
                if (i >= a.n) continue;
                T* row = static_cast<T*>(a.dx) + i * a.dx_stride;
#pragma unroll
                for (int k = 0; k < AB; ++k) {
                    const float v[4] = {acc[k][j][0], acc[k][j][1], acc[k][j][2], acc[k][j][3]};
                    store_cols<4>(row, c0 + Shape::row() + k * 16 + (lane >> 4) * 4, a.dim, v);
                }
            }
        });
}

template <int NP, int AB>
__global__ __launch_bounds__((WideShape<NP, AB>::kThreads), 2) void k_wide_dw(WideMat X, WideMat Z, int64_t nr,
                                                             int cols, int ldp, int spread,
                                                             int64_t per_share,
                                                             int add, float* part) {
    using Shape = WideShape<NP, AB>;
    __shared__ quad lds[Shape::kQuads];
    const int lane = threadIdx.x & 63;
    // with `spread` 8 a share's tiles run on one XCD, whose L2 gives them its rows of x and dz
    const int tiles = (int)(Z.cols / Shape::kCols) * cols;
    const int k = (int)blockIdx.x / spread, tile = k % tiles;
    const int64_t share = k / tiles * spread + (int)blockIdx.x % spread;
    const int64_t c0 = (int64_t)(tile % cols) * Shape::kRows, r0 = (int64_t)(tile / cols) * Shape::kCols;
    const int64_t k0 = min(nr, share * per_share), k1 = min(nr, k0 + per_share);
    wide_products<NP, AB, false, false, false>(
        X, Z, k0, k1, 1, lds, [&](int) { return TileRows{c0, r0}; }, [](int) {},
        [&](int, f32x4(&acc)[AB][Shape::BB]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t r = r0 + Shape::col() + j * 16 + (lane & 15);
                f32x4* to = reinterpret_cast<f32x4*>(part + (share * Z.cols + r) * ldp + c0 +
                                                     Shape::row());
#pragma unroll
                for (int k = 0; k < AB; ++k) {
                    f32x4 v = acc[k][j];
                    if (add) v += to[k * 4 + (lane >> 4)];
                    to[k * 4 + (lane >> 4)] = v;
                }
            }
        });
}

// ---------------------------------------------------------------- few rows
// Up to 64 rows: every workgroup makes 16 hidden units of all rows, its waves sharing the
// summed index; the operands come from memory as the matrix cores take them, 8 values of a
// row a lane, so that nothing is laid out before. 64 rows of 512 to 1024 bf16 take 13.5 us
// a call so and 39 in tiles, with their gradients 58 and 173; 40 of fp32 13.6 and 56, 96
// and 236. One row of 64 to 256 fp32 is a kernel of 4.1 us, 33 of 512 to 2048 bf16 of 5.9:
// the way to memory and back, once.
constexpr int kFewRows = 64;

// With GRAD the rows [dgate, dup] as operands of the tiles below, 128 rows with zeros behind, and
// the biases' sums over each block of 16 rows.
template <typename T, int NP, int ACT, int J, bool GRAD>
__global__ __launch_bounds__(kThreads) void k_gated_few(GatedArgs a, bf16* dz, float* db,
                                                        int64_t wr) {
    __shared__ f32x4 lds[kThreads / 64][2 * J][64];
    const int lane = threadIdx.x & 63, w = wave_id(), g = lane >> 4, s = lane & 15;
    const int64_t u0 = (int64_t)blockIdx.x * 16;
    const bool on = u0 + s < a.hidden;
    const int64_t unit = on ? u0 + s : 0;
    const T* gate = static_cast<const T*>(a.w_gate) + unit * a.gate_stride;
    const T* up = static_cast<const T*>(a.w_up) + unit * a.up_stride;
    f32x4 acc[2][J];
#pragma unroll
    for (int j = 0; j < J; ++j) acc[0][j] = acc[1][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = w * 32; k < a.dim; k += kThreads / 64 * 32) {
        quad wp[2][NP], xp[J][NP];
        const int c = k + g * 8;
        load_parts<T, NP>(gate, a.dim, c, on, wp[0]);
        load_parts<T, NP>(up, a.dim, c, on, wp[1]);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int64_t i = j * 16 + s;
            load_parts<T, NP>(static_cast<const T*>(a.x) + (i < a.n ? i : 0) * a.x_stride, a.dim,
                              c, i < a.n, xp[j]);
        }
#pragma unroll
        for (int q = 0; q < Products<NP>::kCount; ++q)
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, wp[t][Products<NP>::a(q)]),
                        __builtin_bit_cast(bf16x8, xp[j][Products<NP>::b(q)]), acc[t][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) lds[w][t * J + j][lane] = acc[t][j];
    __syncthreads();
    // wave w joins every fourth block of 16 rows: the lane's row is i, its units u0 + 4 g ..
    for (int j = w; j < J; j += kThreads / 64) {
        f32x4 z[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            z[t] = lds[0][t * J + j][lane];
#pragma unroll
            for (int v = 1; v < kThreads / 64; ++v) z[t] += lds[v][t * J + j][lane];
        }
        const int64_t i = j * 16 + s, u = u0 + g * 4;
        if (!GRAD && i >= a.n) continue;
        float h[4], d[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = u + k < a.hidden;
            const float bg = in && a.b_gate != nullptr ? a.b_gate[u + k] : 0.0f;
            const float bu = in && a.b_up != nullptr ? a.b_up[u + k] : 0.0f;
            const float zg = z[0][k] + bg, zu = z[1][k] + bu;
            if (!GRAD) {
                h[k] = act<ACT>(zg) * zu;
            } else {
                const bool on = in && i < a.n;
                const float v = on ? to_float(static_cast<const T*>(a.dh)[i * a.dh_stride + u + k])
                                   : 0.0f;
                d[k] = on ? plain_input<NP>(v * zu * act_slope<ACT>(zg)) : 0.0f;
                d[4 + k] = on ? plain_input<NP>(v * act<ACT>(zg)) : 0.0f;
            }
        }
        if (!GRAD) {
            store_cols<4>(static_cast<T*>(a.h) + i * a.h_stride, u, a.hidden, h);
            continue;
        }
        // 4 units in a row are 4 rows of the weights in a row, gate and 32 on up
        const int64_t r = row_of_unit(u);
        quad q[NP];
        split8_input<NP>(d, q);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            uint2* to = reinterpret_cast<uint2*>(dz + (p * kTile + i) * wr + r);
            to[0] = make_uint2(q[p][0], q[p][1]);
            to[8] = make_uint2(q[p][2], q[p][3]);
        }
        if (db != nullptr) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                for (int k = 0; k < 8; ++k) d[k] += __shfl_xor(d[k], o, 64);
            if (s == 0) {
#pragma unroll
                for (int k = 0; k < 8; ++k) db[j * wr + r + (k / 4) * 32 + k % 4] = d[k];
            }
        }
    }
    if (!GRAD) return;
    // the rows behind: 4 units a thread and row
    const int64_t r = row_of_unit(u0 + (threadIdx.x & 3) * 4);
    for (int i = 16 * J + (int)(threadIdx.x >> 2); i < kTile; i += kThreads / 4)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            uint2* to = reinterpret_cast<uint2*>(dz + (p * kTile + i) * wr + r);
            to[0] = to[8] = make_uint2(0u, 0u);
        }
}

bool is_few(const GatedArgs& a, bool grad) { return !grad && a.n <= kFewRows; }

template <typename T, int NP, int ACT>
hipError_t few_run(const GatedArgs& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.hidden + 15) / 16);
    if (a.n <= 16) k_gated_few<T, NP, ACT, 1, false><<<blocks, kThreads, 0, st>>>(a, nullptr, nullptr, 0);
    else if (a.n <= 32) k_gated_few<T, NP, ACT, 2, false><<<blocks, kThreads, 0, st>>>(a, nullptr, nullptr, 0);
    else k_gated_few<T, NP, ACT, 4, false><<<blocks, kThreads, 0, st>>>(a, nullptr, nullptr, 0);
    return hipGetLastError();
}
// Every unit of the padded weights has its place in dz.
template <typename T, int NP, int ACT>
hipError_t few_grad(const GatedArgs& a, bf16* dz, float* db, int64_t wr, hipStream_t st) {
    const unsigned blocks = (unsigned)(wr / 32);
    if (a.n <= 16) k_gated_few<T, NP, ACT, 1, true><<<blocks, kThreads, 0, st>>>(a, dz, db, wr);
    else if (a.n <= 32) k_gated_few<T, NP, ACT, 2, true><<<blocks, kThreads, 0, st>>>(a, dz, db, wr);
    else k_gated_few<T, NP, ACT, 4, true><<<blocks, kThreads, 0, st>>>(a, dz, db, wr);
    return hipGetLastError();
}

// ---------------------------------------------------------------- plans
// Bytes of x's parts and of [dgate, dup] in the workspace at most, about.
constexpr int64_t kPieceBytes = (int64_t)1 << 30;

struct GatedPlan {
    int ld;            // padded dim
    int64_t wr, piece, shares;  // weight rows, samples of a piece, shares of the weights' sums
    int64_t dx_shares = 1, dx_per = 0;  // shares of the weights' rows in dx
    bf16 *w = nullptr, *x = nullptr, *dz = nullptr;
    float *part = nullptr, *db = nullptr, *dx = nullptr;
    size_t bytes;
    GatedPlan(void* base, int64_t n, int64_t hidden, int dim, int np, bool grad) {
        ld = (int)pad_to(dim, kTile);
        wr = pad_to(2 * hidden, kTile);
        const int64_t row = (int64_t)np * 2 * (ld + (grad ? wr : 0));
        const int64_t all = pad_to(n, kTile);
        // a launch takes fewer than 2^32 threads
        const int64_t most = std::min(kPieceBytes / row, ((int64_t)1 << 30) / (wr / kTile));
        piece = std::min(all, std::max<int64_t>(kTile, most / kTile * kTile));
        const int64_t tiles = (wr / kTile) * (ld / kTile);
        shares = std::max<int64_t>(1, std::min((512 + tiles - 1) / tiles, piece / 512));
        Carve c(base);
        w = c.take<bf16>((size_t)(wr * ld) * np);
        x = c.take<bf16>((size_t)(piece * ld) * np);
        if (grad) {
            dz = c.take<bf16>((size_t)(piece * wr) * np);
            part = c.take<float>((size_t)(shares * wr * ld));
            db = c.take<float>((size_t)(std::max<int64_t>(4, piece / 64) * wr));
            // one step of the summed index at least, and as many workgroups as run at a time
            const int64_t of_dx = std::max<int64_t>(1, piece / kTile * (ld / kTile));
            const int64_t want = std::max<int64_t>(1, std::min(wr / kStep, 512 / of_dx));
            dx_per = pad_to((wr + want - 1) / want, kStep);
            dx_shares = (wr + dx_per - 1) / dx_per;
            dx = dx_shares > 1 ? c.take<float>((size_t)(dx_shares * piece * ld)) : nullptr;
        }
        bytes = c.bytes();
    }
};

// Wide tiles pay from about 448 of them. h and a training pass in tiles, then in wide ones, us:
//   bf16 512 to 1024, 12000 rows (376 tiles): 44 and 203, 42 and 210; 15000 (472): 52 and
//   246, 43 and 222; 256 to 512, 20000 (316): 30 and 134, 28 and 144; 30000 (472): 38 and 181,
//   30 and 154; fp32 512 to 1024, 3000 (384): 54 and 252, 63 and 273; 4000 (512): 59 and 297,
//   65 and 287; 6000 (752): 95 and 455, 86 and 352; 256 to 512, 8000 (504): 39 and 195, 44
//   and 179; 12000 (752): 55 and 290, 54 and 214.
// Of wider weights a training pass needs more of them: bf16 1024 to 4096, 4000 rows (512): 83
// and 518, 77 and 643; 7000 (896): 134 and 753, 128 and 805; fp32 1200 (640): 188 and 982, 163
// and 924.
constexpr int kWideLeast = 448;
bool is_wide(const GatedArgs& a) {
    const int64_t tile = a.dtype == 0 ? 128 : 256;
    return a.dim > kShortDim &&
           ((2 * a.hidden + tile - 1) / tile) * ((a.n + tile - 1) / tile) >= kWideLeast;
}

struct WidePlan {
    int ld, ldp = 0, ab = 4;  // the weights' columns, the partial sums', blocks of A for the gradients
    int spread = 8;  // XCDs that the shares of the weights' sums go over
    int64_t wr, piece, shares = 0, per_share = 0;
    bool direct;  // x is read where it is
    quad* zero;
    bf16 *w, *x = nullptr, *dz = nullptr;
    float *part = nullptr, *db = nullptr;
    size_t bytes;
    WidePlan(void* base, const GatedArgs& a, int np, bool grad) {
        ld = (int)pad_to(a.dim, kStep);
        wr = pad_to(2 * a.hidden, 256);
        direct = np == 1 && a.dim % 8 == 0 && a.x_stride % 8 == 0 &&
                 reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                 a.x_stride < ((int64_t)1 << 22);  // 256 rows within a lane's 32-bit offset
        const int64_t row = (int64_t)np * 2 * ((direct ? 0 : ld) + (grad ? wr : 0));
        const int cols = np == 1 ? 256 : 128;  // rows of a tile
        const int64_t all = pad_to(a.n, cols);
        // a launch takes fewer than 2^32 threads
        const int64_t most = std::min(row == 0 ? all : kPieceBytes / row,
                                      ((int64_t)1 << 30) / (wr / 128 * (1 + ld / 1024)));
        piece = std::min(all, std::max<int64_t>(cols, most / cols * cols));
        Carve c(base);
        zero = c.take<quad>(1);
        w = c.take<bf16>((size_t)(wr * ld) * np);
        if (!direct) x = c.take<bf16>((size_t)(piece * ld) * np);
        if (grad) {
            // tiles of 256 or 128 columns of x for the gradients: what wastes less
            ab = np == 1 && (a.dim + 127) / 128 % 2 == 0 ? 8 : 4;  // 256 or 128 columns of x
            ldp = (int)pad_to(a.dim, 32 * ab);
            const int64_t tiles = (wr / cols) * (ldp / (32 * ab));
            // of weights whose tiles alone fill the chip, one
            spread = tiles >= 256 ? 1 : 8;
            shares = spread * std::max<int64_t>(1, (np == 1 ? 32 : 64) / tiles);
            per_share = pad_to((piece + shares - 1) / shares, kStep);
            dz = c.take<bf16>((size_t)(piece * wr) * np);
            part = c.take<float>((size_t)(shares * wr * ldp));
            db = c.take<float>((size_t)(piece / 64 * wr));
        }
        bytes = c.bytes();
    }
};

template <typename T, int NP, int ACT>
hipError_t wide_run(const GatedArgs& a, bool grad, hipStream_t st) {
    const WidePlan w(a.ws, a, NP, grad);
    using Shape = WideShape<NP, kWideBlocks<NP>>;
    constexpr int COLS = Shape::kCols, THREADS = Shape::kThreads;
    k_wide_weights<T, NP><<<blocks_of(w.wr * (w.ld / 8), kThreads), kThreads, 0, st>>>(
        a, w.wr, w.ld, reinterpret_cast<quad*>(w.w), w.zero);
    GS_LAUNCHED();
    const WideMat W{w.w, w.ld, w.wr * w.ld, w.wr, w.ld, w.zero};
    const bool biases = a.db_gate != nullptr || a.db_up != nullptr;
    for (int64_t n0 = 0; n0 < a.n; n0 += w.piece) {
        const int64_t nr = std::min(w.piece, pad_to(a.n - n0, COLS));
        WideMat X{w.x, w.ld, nr * w.ld, nr, w.ld, w.zero};
        if (w.direct) {
            X = WideMat{static_cast<const bf16*>(a.x) + n0 * a.x_stride, a.x_stride, 0, a.n - n0,
                        a.dim, w.zero};
        } else {
            k_gated_parts<T, NP, false><<<blocks_of(nr * (w.ld / 8), kThreads), kThreads, 0, st>>>(
                a, n0, nr, w.ld, reinterpret_cast<quad*>(w.x));
            GS_LAUNCHED();
        }
        const int tiles_w = (int)(w.wr / Shape::kRows), share = 2;
        const SpotGrid sg(nr / COLS, (tiles_w + share - 1) / share, kSpot);
        if (!grad) {
            k_gated_wide<T, NP, ACT, false><<<sg.blocks, THREADS, 0, st>>>(
                a, W, X, w.ld, n0, nr, tiles_w, share, sg.gy, nullptr, nullptr);
            GS_LAUNCHED();
            continue;
        }
        k_gated_wide<T, NP, ACT, true><<<sg.blocks, THREADS, 0, st>>>(
            a, W, X, w.ld, n0, nr, tiles_w, share, sg.gy, w.dz, biases ? w.db : nullptr);
        GS_LAUNCHED();
        if (biases) {
            k_gated_sum<T, true, true><<<sum_blocks(w.wr / 4), 1024, 0, st>>>(
                a, w.db, (int)(nr / 64), w.wr, 4, n0 > 0);
            GS_LAUNCHED();
        }
        const WideMat Z{w.dz, w.wr, nr * w.wr, nr, w.wr, w.zero};
        const int tiles_c = w.ldp / (32 * w.ab);
        const SpotGrid xg(nr / COLS, tiles_c, kSpot);
        const unsigned wg = (unsigned)(w.wr / COLS * tiles_c * w.shares);
        auto sums = [&](auto ab) {
            constexpr int AB = decltype(ab)::value;
            k_wide_dx<T, NP, AB><<<xg.blocks, THREADS, 0, st>>>(a, W, Z, n0, nr, tiles_c, xg.gy);
            GS_LAUNCHED();
            k_wide_dw<NP, AB><<<wg, THREADS, 0, st>>>(X, Z, nr, tiles_c, w.ldp, w.spread, w.per_share,
                                                      n0 > 0, w.part);
            return hipGetLastError();
        };
        hipError_t e;
        if constexpr (NP == 1) {
            e = w.ab == 8 ? sums(std::integral_constant<int, 8>())
                          : sums(std::integral_constant<int, 4>());
        } else {
            e = sums(std::integral_constant<int, 4>());
        }
        if (e != hipSuccess) return e;
    }
    if (!grad) return hipSuccess;
    k_gated_sum<T, true, false><<<sum_blocks(w.wr * (w.ldp / 4)), 1024, 0, st>>>(
        a, w.part, (int)w.shares, w.wr, w.ldp, 0);
    return hipGetLastError();
}

template <typename T, int NP, int ACT>
hipError_t gated_run(const GatedArgs& a, bool grad, hipStream_t st) {
    if (is_few(a, grad)) return few_run<T, NP, ACT>(a, st);
    if (is_wide(a)) return wide_run<T, NP, ACT>(a, grad, st);
    const GatedPlan w(a.ws, a.n, a.hidden, a.dim, NP, grad);
    const int kd = (int)pad_to(a.dim, kStep);
    const int64_t wu = w.wr * (w.ld / 8);
    if (a.n > 0) {
        k_gated_parts<T, NP, true><<<blocks_of(wu, kThreads), kThreads, 0, st>>>(
            a, 0, w.wr, w.ld, reinterpret_cast<quad*>(w.w));
        GS_LAUNCHED();
    }
    const Mat W{w.w, w.ld, w.wr * w.ld};
    const bool biases = a.db_gate != nullptr || a.db_up != nullptr;
    for (int64_t n0 = 0; n0 < a.n; n0 += w.piece) {
        const int64_t nr = std::min(w.piece, pad_to(a.n - n0, kTile));
        const Mat X{w.x, w.ld, nr * w.ld}, Z{w.dz, w.wr, nr * w.wr};
        k_gated_parts<T, NP, false><<<blocks_of(nr * (w.ld / 8), kThreads), kThreads, 0, st>>>(
            a, n0, nr, w.ld, reinterpret_cast<quad*>(w.x));
        GS_LAUNCHED();
        const SpotGrid sg(nr / kTile, w.wr / kTile, kSpot);
        if (!grad) {
            k_gated<T, NP, ACT, false><<<sg.blocks, kThreads, 0, st>>>(
                a, X, W, kd, n0, nr, w.wr, sg.gy, nullptr, nullptr);
            GS_LAUNCHED();
            continue;
        }
        const bool few = a.n <= kFewRows;
        if (few) {
            const hipError_t e = few_grad<T, NP, ACT>(a, w.dz, biases ? w.db : nullptr, w.wr, st);
            if (e != hipSuccess) return e;
        } else {
            k_gated<T, NP, ACT, true><<<sg.blocks, kThreads, 0, st>>>(
                a, X, W, kd, n0, nr, w.wr, sg.gy, w.dz, biases ? w.db : nullptr);
            GS_LAUNCHED();
        }
        if (biases) {
            const int64_t blocks = few ? (a.n <= 32 ? (a.n + 15) / 16 : 4) : nr / 64;
            k_gated_sum<T, false, true><<<sum_blocks(w.wr / 4), 1024, 0, st>>>(
                a, w.db, (int)blocks, w.wr, 4, n0 > 0);
            GS_LAUNCHED();
        }
        const SpotGrid xg(nr / kTile, w.ld / kTile, kSpot);
        k_gated_dx<T, NP><<<dim3(xg.blocks, (unsigned)w.dx_shares), kThreads, 0, st>>>(
            a, W, Z, n0, nr, w.ld, w.wr, xg.gy, w.dx_per, w.dx);
        GS_LAUNCHED();
        if (w.dx_shares > 1) {
            const hipError_t e = gated_dx_join(a, w.dx, (int)w.dx_shares, nr, w.ld, n0,
                                               std::min(w.piece, a.n - n0), st);
            if (e != hipSuccess) return e;
        }
        const int64_t per = pad_to((nr + w.shares - 1) / w.shares, kStep);
        const dim3 grid((unsigned)(w.wr / kTile * (w.ld / kTile)), (unsigned)w.shares);
        k_gated_dw<NP><<<grid, kThreads, 0, st>>>(X, Z, nr, w.ld, w.wr, per, n0 > 0, w.part);
        GS_LAUNCHED();
    }
    if (!grad) return hipSuccess;
    if (a.n == 0 && biases) {
        k_gated_sum<T, false, true><<<sum_blocks(w.wr / 4), 1024, 0, st>>>(a, nullptr, 0, w.wr, 4, 0);
        GS_LAUNCHED();
    }
    k_gated_sum<T, false, false><<<sum_blocks(w.wr * (w.ld / 4)), 1024, 0, st>>>(
        a, w.part, a.n > 0 ? (int)w.shares : 0, w.wr, w.ld, 0);
    return hipGetLastError();
}

template <typename T, int NP>
hipError_t gated_act(const GatedArgs& a, bool grad, hipStream_t st) {
    switch (a.act) {
        case kActRelu: return gated_run<T, NP, kActRelu>(a, grad, st);
        case kActSilu: return gated_run<T, NP, kActSilu>(a, grad, st);
        case kActGelu: return gated_run<T, NP, kActGelu>(a, grad, st);
        default: return gated_run<T, NP, kActNone>(a, grad, st);
    }
}

}  // namespace

hipError_t gated_dx_join(const GatedArgs& a, const float* part, int shares, int64_t rows, int ld,
                         int64_t n0, int64_t n, hipStream_t st) {
    const unsigned blocks = blocks_of(n * ((a.dim + 3) / 4), kThreads);
    if (a.dtype == 0)
        k_gated_dx_join<float><<<blocks, kThreads, 0, st>>>(a, part, shares, rows, ld, n0, n);
    else
        k_gated_dx_join<bf16><<<blocks, kThreads, 0, st>>>(a, part, shares, rows, ld, n0, n);
    return hipGetLastError();
}

size_t gated_linear_ws(const GatedArgs& a, bool grad) {
    if (a.n == 0 || is_few(a, grad)) return 0;
    if (a.dim <= kShortDim) return gated_short_ws(a, grad);
    if (is_wide(a)) return WidePlan(nullptr, a, a.dtype == 0 ? 3 : 1, grad).bytes;
    return GatedPlan(nullptr, a.n, a.hidden, a.dim, a.dtype == 0 ? 3 : 1, grad).bytes;
}

hipError_t launch_gated_linear(const GatedArgs& a, bool grad, hipStream_t st) {
    if (a.n == 0 && !grad) return hipSuccess;
    if (a.n > 0 && a.dim <= kShortDim && !is_few(a, grad))
        return a.dtype == 0 ? gated_short_f32(a, grad, st) : gated_short_bf16(a, grad, st);
    return a.dtype == 0 ? gated_act<float, 3>(a, grad, st) : gated_act<bf16, 1>(a, grad, st);
}

}  // namespace gs
