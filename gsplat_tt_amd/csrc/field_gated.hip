// field_gated.hip - gated projections of features, forward and backward.
//
//   gate = x Wg^T + bg;  up = x Wu^T + bu;  h = act(gate) up
// and, from dh:
//   dgate = dh up act'(gate);  dup = dh act(gate);
//   dx = dgate Wg + dup Wu;  dWg = dgate^T x;  dWu = dup^T x;  db = column sums.
//
// The backward pass makes gate and up again: keeping them would cost 2 n hidden values
// written and read against 4 n dim hidden operations.
//
// All products run on the matrix cores with bf16 operands and fp32 sums; fp32 values are
// cut into three bf16 parts, whose six products above 2^-24 are added up (field_tiles.h).
// For bf16 inputs dgate and dup are rounded to bf16 as operands of the next products; the
// biases' gradients sum them in fp32.
#include "field_gated.h"

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

// dx of one tile: the weights' columns against the samples' [dgate, dup].
template <typename T, int NP>
__global__ __launch_bounds__(kThreads, 2) void k_gated_dx(GatedArgs a, Mat W, Mat Z, int64_t n0,
                                                          int64_t nr, int ld, int64_t wr, int gy) {
    GS_TILE_LDS;
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const Spot at = spot((int)(nr / kTile), gy);
    const int64_t c0 = (int64_t)at.y * kTile, s0 = (int64_t)at.x * kTile;
    if (c0 >= ld) return;
    tile_products<NP, false, true>(
        W, Z, 0, wr, 1, lds, [&](int) { return TileRows{c0, s0}; },
        [&](int, f32x4(&acc)[4][4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t i = n0 + s0 + wn + j * 16 + (lane & 15);
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

// The shares' sums as the weights' gradients: 4 columns a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_gated_dw_sum(GatedArgs a, const float* part,
                                                           int shares, int64_t wr, int ld) {
    const int units = ld / 4;
    const int64_t total = wr * units;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t r = e / units;
        const int c = (int)(e - r * units) * 4;
        const UnitOf u = unit_of(r);
        if (u.unit >= a.hidden || c >= a.dim) continue;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < shares; ++k)
            v += *reinterpret_cast<const f32x4*>(part + (k * wr + r) * ld + c);
        T* row = static_cast<T*>(u.up ? a.dw_up : a.dw_gate) +
                 u.unit * (u.up ? a.dup_stride : a.dgate_stride);
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_cols<4>(row, c, a.dim, o);
    }
}

// The biases' gradients: sums over the blocks of 64 samples, in 16 runs a row that are
// joined in order; with `add` onto what an earlier piece left.
__global__ __launch_bounds__(kThreads) void k_gated_db(GatedArgs a, const float* db,
                                                       int64_t blocks, int64_t wr, int add) {
    __shared__ float lds[16][16];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t r = (int64_t)blockIdx.x * 16 + c;
    const int64_t per = (blocks + 15) / 16, b1 = min(blocks, (k + 1) * per);
    float v = 0.0f;
    for (int64_t b = k * per; b < b1; ++b) v += db[b * wr + r];
    lds[k][c] = v;
    __syncthreads();
    if (k != 0) return;
    v = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) v += lds[j][c];
    const UnitOf u = unit_of(r);
    float* out = u.up ? a.db_up : a.db_gate;
    if (out == nullptr || u.unit >= a.hidden) return;
    out[u.unit] = add ? out[u.unit] + v : v;
}

// ---------------------------------------------------------------- few rows
// Up to 64 rows, without their gradients: every workgroup makes 16 hidden units of all
// rows, its waves sharing the summed index; the operands come from memory as the matrix
// cores take them, 8 values of a row a lane, so that nothing is laid out before.
constexpr int kFewRows = 64;

template <typename T, int NP, int ACT, int J>
__global__ __launch_bounds__(kThreads) void k_gated_few(GatedArgs a) {
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
        if (i >= a.n) continue;
        float h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = u + k < a.hidden;
            const float bg = in && a.b_gate != nullptr ? a.b_gate[u + k] : 0.0f;
            const float bu = in && a.b_up != nullptr ? a.b_up[u + k] : 0.0f;
            h[k] = act<ACT>(z[0][k] + bg) * (z[1][k] + bu);
        }
        store_cols<4>(static_cast<T*>(a.h) + i * a.h_stride, u, a.hidden, h);
    }
}

bool is_few(const GatedArgs& a, bool grad) { return !grad && a.n <= kFewRows; }

template <typename T, int NP, int ACT>
hipError_t few_run(const GatedArgs& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.hidden + 15) / 16);
    if (a.n <= 16) k_gated_few<T, NP, ACT, 1><<<blocks, kThreads, 0, st>>>(a);
    else if (a.n <= 32) k_gated_few<T, NP, ACT, 2><<<blocks, kThreads, 0, st>>>(a);
    else k_gated_few<T, NP, ACT, 4><<<blocks, kThreads, 0, st>>>(a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- plans
// Bytes of x's parts and of [dgate, dup] in the workspace at most, about.
constexpr int64_t kPieceBytes = (int64_t)1 << 30;

struct GatedPlan {
    int ld;            // padded dim
    int64_t wr, piece, shares;  // weight rows, samples of a piece, shares of the weights' sums
    bf16 *w, *x, *dz;
    float *part, *db;
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
            db = c.take<float>((size_t)(piece / 64 * wr));
        }
        bytes = c.bytes();
    }
};

template <typename T, int NP, int ACT>
hipError_t gated_run(const GatedArgs& a, bool grad, hipStream_t st) {
    if (is_few(a, grad)) return few_run<T, NP, ACT>(a, st);
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
        k_gated<T, NP, ACT, true><<<sg.blocks, kThreads, 0, st>>>(
            a, X, W, kd, n0, nr, w.wr, sg.gy, w.dz, biases ? w.db : nullptr);
        GS_LAUNCHED();
        if (biases) {
            k_gated_db<<<(unsigned)(w.wr / 16), kThreads, 0, st>>>(a, w.db, nr / 64, w.wr, n0 > 0);
            GS_LAUNCHED();
        }
        const SpotGrid xg(nr / kTile, w.ld / kTile, kSpot);
        k_gated_dx<T, NP><<<xg.blocks, kThreads, 0, st>>>(a, W, Z, n0, nr, w.ld, w.wr, xg.gy);
        GS_LAUNCHED();
        const int64_t per = pad_to((nr + w.shares - 1) / w.shares, kStep);
        const dim3 grid((unsigned)(w.wr / kTile * (w.ld / kTile)), (unsigned)w.shares);
        k_gated_dw<NP><<<grid, kThreads, 0, st>>>(X, Z, nr, w.ld, w.wr, per, n0 > 0, w.part);
        GS_LAUNCHED();
    }
    if (!grad) return hipSuccess;
    if (a.n == 0 && biases) {
        k_gated_db<<<(unsigned)(w.wr / 16), kThreads, 0, st>>>(a, nullptr, 0, w.wr, 0);
        GS_LAUNCHED();
    }
    k_gated_dw_sum<T><<<blocks_of(w.wr * (w.ld / 4), kThreads), kThreads, 0, st>>>(
        a, w.part, a.n > 0 ? (int)w.shares : 0, w.wr, w.ld);
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

size_t gated_linear_ws(const GatedArgs& a, bool grad) {
    if (a.n == 0 || is_few(a, grad)) return 0;
    if (a.dim <= kShortDim) return gated_short_ws(a, grad);
    return GatedPlan(nullptr, a.n, a.hidden, a.dim, a.dtype == 0 ? 3 : 1, grad).bytes;
}

hipError_t launch_gated_linear(const GatedArgs& a, bool grad, hipStream_t st) {
    if (a.n == 0 && !grad) return hipSuccess;
    if (a.n > 0 && a.dim <= kShortDim && !is_few(a, grad))
        return a.dtype == 0 ? gated_short_f32(a, grad, st) : gated_short_bf16(a, grad, st);
    return a.dtype == 0 ? gated_act<float, 3>(a, grad, st) : gated_act<bf16, 1>(a, grad, st);
}

}  // namespace gs
