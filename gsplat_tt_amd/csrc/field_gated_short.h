// field_gated_short.h - gated projections of rows of up to 128 values (field_gated.hip
// says what they are). A source file each for fp32 and bf16, which compile side by side.
#pragma once

#include "field_gated.h"

namespace gs {

namespace {

constexpr int kThreads = kTileThreads;

// Rows of up to 128 values. Both kernels keep tiles of operands in LDS in the order in
// which the matrix cores take them: block (16 rows), step of 32 of the row, lane; a lane's
// quad is row lane % 16, values 8 (lane / 16) .. + 7. The last two quarters' rows are placed
// by (row ^ 8), so that the transposing loads, which take 4 rows of 4 x 4 values for 16
// lanes, touch all banks once for two such groups.

__device__ __forceinline__ uint32_t quad_place(uint32_t row, uint32_t quarter) {
    return (row ^ ((quarter >> 1) << 3)) + 16 * quarter;
}
// The operand of 16 rows and 32 values as it lies in LDS.
__device__ __forceinline__ bf16x8 operand_of(const quad* at) {
    const uint32_t lane = threadIdx.x & 63;
    return __builtin_bit_cast(bf16x8, at[quad_place(lane & 15, lane >> 4)]);
}
// The transposed operand of 16 of the 32 values and the 32 rows of two blocks, `step` quads
// apart: rows 4 (lane / 16) .. + 3 of the first, then of the second. Of quarter q, half b ^
// (q & 1): a lane's sums of b = 0 and 1 are 8 values in a row, in turned order where the
// lane's quarter is odd.
__device__ __forceinline__ bf16x8 operand_across(const quad* at, int step, int b) {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const uint32_t lane = threadIdx.x & 63, s = lane & 15, q = s & 3;
    const char* p = reinterpret_cast<const char*>(at + quad_place((lane >> 4) * 4 + (s >> 2), q)) +
                    ((b ^ q) & 1) * 8;
    s16x4 half[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + u * step * 16));
    return __builtin_bit_cast(bf16x8,
                              __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
}
// acc(m, n) += a[m] b[n]; neighbouring products go to different sums, which spares the wait
// of one for the other.
template <int NP, int M, int N, class Acc>
__device__ __forceinline__ void multiply(const bf16x8 (&a)[M][NP], const bf16x8 (&b)[N][NP],
                                         Acc acc) {
#pragma unroll
    for (int q = 0; q < Products<NP>::kCount; ++q)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4& c = acc(m, n);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m][Products<NP>::a(q)],
                                                            b[n][Products<NP>::b(q)], c, 0, 0, 0);
            }
}

// A chunk of the weights, 32 units, as 4 blocks of 16 rows: gate, gate, up, up; block i of
// two has the units 8 (s / 4) + 4 i + s % 4, so that a lane's sums are 8 units in a row.
__device__ __forceinline__ int64_t weight_unit(int64_t u0, int i, int s) {
    return u0 + (s >> 2) * 8 + (i & 1) * 4 + (s & 3);
}
template <typename T>
__device__ __forceinline__ const T* weight_row(const GatedArgs& a, int64_t u0, int i, int s) {
    const int64_t unit = weight_unit(u0, i, s);
    return static_cast<const T*>(i >= 2 ? a.w_up : a.w_gate) +
           (unit < a.hidden ? unit : 0) * (i >= 2 ? a.up_stride : a.gate_stride);
}
// The chunks' parts laid out as LDS takes them, so that fp32 weights are cut once.
template <typename T, int NP, int KS>
__global__ __launch_bounds__(kThreads) void k_gated_chunks(GatedArgs a, int64_t chunks,
                                                           quad* out) {
    const int64_t total = chunks * (256 * KS);
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
         e += (int64_t)gridDim.x * kThreads) {
        const int64_t chunk = e / (256 * KS);
        const int q = (int)(e - chunk * (256 * KS)), lane = q & 63, b = q >> 6;
        quad part[NP];
        load_parts<T, NP>(weight_row<T>(a, chunk * 32, b / KS, lane & 15), a.dim,
                          (b % KS) * 32 + (lane >> 4) * 8,
                          weight_unit(chunk * 32, b / KS, lane & 15) < a.hidden, part);
#pragma unroll
        for (int p = 0; p < NP; ++p)
            out[(chunk * NP + p) * (256 * KS) + b * 64 + quad_place(lane & 15, lane >> 4)] = part[p];
    }
}

// Rows stay with their wave, 16 J of them in registers, and the weights pass through LDS
// chunk by chunk: h, or with GRAD dx, whose sums stay in registers too. The gradients of
// gate and up leave the sums in the layout that the next product takes them in. LAID: the
// chunks' parts come from k_gated_chunks (cutting them in the kernel took dx of 10007 x 75 to
// 201 from 26 to 38 us). bf16 rows are 64 a wave, with gradients 32; fp32 rows 32, with
// gradients of more than 64 values 16: 16 took as long, 128 do not fit the registers. 307200 x
// 64 to 256 bf16: 45 us a call, 197 MB at 4.4 TB/s, bound by them; to 128 with gradients 52,
// 157 MB, the vector units busy half of the time with silu and its slope. 921600 x 128 to 128
// fp32: 365 a call (355 to 416 in kernel traces), the matrix cores busy 48 % and the vector
// units 38 % of the time, at a clock that has come down to 2 GHz. Shares of the chunks
// (blockIdx.y) leave sums of dx of their own in `part` (share, rows, 32 KS), where there are
// several.
template <typename T, int NP, int ACT, int KS, int J, bool GRAD, bool LAID>
__global__ __launch_bounds__(kThreads, NP == 1 || J * KS < 8 ? 2 : 1) void k_gated_rows(
    GatedArgs a, const quad* laid, int64_t block0, int64_t chunks, int64_t per_share, float* part) {
    __shared__ quad lds[NP * 256 * KS];
    __shared__ float bias[64];
    const int lane = threadIdx.x & 63, w = wave_id(), g = lane >> 4, s = lane & 15;
    const int64_t i0 = ((block0 + blockIdx.x) * (kThreads / 64) + w) * (16 * J);
    const int64_t c0 = blockIdx.y * per_share, c1 = min(chunks, c0 + per_share);
    quad next[KS][LAID ? NP : 1];
    Raw<T> next_w[LAID ? 1 : KS];
    Raw<T> next_d[J];
    float next_bias = 0.0f;
    auto fetch = [&](int64_t chunk) {
        if (GRAD) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int64_t i = i0 + j * 16 + s;
                next_d[j].load(static_cast<const T*>(a.dh) + (i < a.n ? i : 0) * a.dh_stride,
                               chunk * 32 + g * 8, a.hidden);
            }
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if constexpr (LAID) {
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    next[k][p] = laid[(chunk * NP + p) * (256 * KS) + k * 256 + threadIdx.x];
            } else {
                const int blk = k * 4 + w;
                next_w[k].load(weight_row<T>(a, chunk * 32, blk / KS, s), (blk % KS) * 32 + g * 8,
                               a.dim);
            }
        }
        if (w == 0) {
            const int i = g;
            const int64_t unit = weight_unit(chunk * 32, i, s);
            const float* from = i >= 2 ? a.b_up : a.b_gate;
            next_bias = from != nullptr && unit < a.hidden ? from[unit] : 0.0f;
        }
    };
    if (c0 < c1) fetch(c0);
    bf16x8 x[KS][J][NP];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int64_t i = i0 + j * 16 + s;
        const T* row = static_cast<const T*>(a.x) + (i < a.n ? i : 0) * a.x_stride;
        Raw<T> raw[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) raw[k].load(row, k * 32 + g * 8, a.dim);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            raw[k].finish(k * 32 + g * 8, a.dim, i < a.n);
            quad part[NP];
            raw[k].parts(part);
#pragma unroll
            for (int p = 0; p < NP; ++p) x[k][j][p] = __builtin_bit_cast(bf16x8, part[p]);
        }
    }
    constexpr int DB = GRAD ? 2 * KS : 1;
    f32x4 dx[DB][J];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < J; ++j) dx[d][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t chunk = c0; chunk < c1; ++chunk) {
        __syncthreads();  // the last chunk has been read
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if constexpr (LAID) {
#pragma unroll
                for (int p = 0; p < NP; ++p) lds[p * (256 * KS) + k * 256 + threadIdx.x] = next[k][p];
            } else {
                const int blk = k * 4 + w;
                next_w[k].finish((blk % KS) * 32 + g * 8, a.dim,
                                 weight_unit(chunk * 32, blk / KS, s) < a.hidden);
                quad q[NP];
                next_w[k].parts(q);
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    lds[p * (256 * KS) + (k * 4 + w) * 64 + quad_place(s, g)] = q[p];
            }
        }
        if (w == 0) bias[lane] = next_bias;
        Raw<T> d[J];
        if (GRAD) {
#pragma unroll
            for (int j = 0; j < J; ++j) d[j] = next_d[j];
            if (chunk * 32 + 32 > a.hidden || i0 + J * 16 > a.n) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    d[j].finish(chunk * 32 + g * 8, a.hidden, i0 + j * 16 + s < a.n);
            }
        }
        __syncthreads();
        if (chunk + 1 < c1) fetch(chunk + 1);
        const int64_t u0 = chunk * 32 + g * 8;
        f32x4 z[4][J];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(bias + i * 16 + g * 4);
#pragma unroll
            for (int j = 0; j < J; ++j) z[i][j] = b;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                bf16x8 f[2][NP];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        f[m][p] = operand_of(lds + p * (256 * KS) + ((i + m) * KS + k) * 64);
                multiply<NP>(f, x[k], [&](int m, int j) -> f32x4& { return z[i + m][j]; });
            }
        if (!GRAD) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int64_t i = i0 + j * 16 + s;
                float h[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    h[k] = act<ACT>(z[k / 4][j][k % 4]) * z[2 + k / 4][j][k % 4];
                if (i < a.n) {
                    T* row = static_cast<T*>(a.h) + i * a.h_stride;
                    if (u0 + 8 <= a.hidden) store_past<8>(row + u0, h);
                    else store_cols<8>(row, u0, a.hidden, h);
                }
            }
            continue;
        }
        bf16x8 dz[2][J][NP];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float dg[8], du[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float zg = z[k / 4][j][k % 4], zu = z[2 + k / 4][j][k % 4];
                dg[k] = plain_input<NP>(d[j][k] * zu * act_slope<ACT>(zg));
                du[k] = plain_input<NP>(d[j][k] * act<ACT>(zg));
            }
            if (chunk * 32 + 32 > a.hidden) {  // an infinite x against no weights is NaN
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (u0 + k >= a.hidden) dg[k] = du[k] = 0.0f;
            }
            quad part[NP];
            split8_input<NP>(dg, part);
#pragma unroll
            for (int p = 0; p < NP; ++p) dz[0][j][p] = __builtin_bit_cast(bf16x8, part[p]);
            split8_input<NP>(du, part);
#pragma unroll
            for (int p = 0; p < NP; ++p) dz[1][j][p] = __builtin_bit_cast(bf16x8, part[p]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                bf16x8 f[2][NP];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        f[m][p] = operand_across(
                            lds + p * (256 * KS) + u * (2 * KS * 64) + k * 64, KS * 64, m);
                multiply<NP>(f, dz[u], [&](int m, int j) -> f32x4& { return dx[2 * k + m][j]; });
            }
    }
    if (!GRAD) return;
    if (gridDim.y > 1) {
        const int64_t rows = (int64_t)gridDim.x * (kThreads / 64 * 16 * J);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            f32x4* to = reinterpret_cast<f32x4*>(
                part + (blockIdx.y * rows + i0 + j * 16 + s) * (32 * KS));
#pragma unroll
            for (int c = 0; c < DB; ++c) to[c / 2 * 8 + g * 2 + ((c ^ g) & 1)] = dx[c][j];
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int64_t i = i0 + j * 16 + s;
        if (i >= a.n) continue;
        T* row = static_cast<T*>(a.dx) + i * a.dx_stride;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int c = k * 32 + g * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = (g & 1) != e / 4 ? dx[2 * k + 1][j][e % 4] : dx[2 * k][j][e % 4];
            if (c + 8 <= a.dim) store_past<8>(row + c, v);
            else store_cols<8>(row, c, a.dim, v);
        }
    }
}

// The weights' gradients: the weights stay with their wave, 16 VB units in registers, and
// the rows pass through LDS, 64 at a time. Here the sums come out with the unit in the lane,
// so that they are the next product's operand over the rows as they are; dh turns on its
// way through LDS, in a part of its own for each wave. WU waves have units of their own;
// the others share the tile's rows, and leave sums of their own. 307200 x 64 to 128 bf16: 48
// us, 118 MB, the vector units busy 48 % of the time, two waves a SIMD (registers); dh
// loaded value by value took 100.
template <typename T>
constexpr int kUnitBlocks = sizeof(T) == 2 ? 2 : 1;  // 64 bytes of a row of dh

template <typename T, int NP, int ACT, int KS, int WU>
__global__ __launch_bounds__(kThreads, KS <= 2 ? 2 : 1) void k_gated_units(
    GatedArgs a, int64_t tiles, int64_t per_share, int64_t wr, float* part, float* db) {
    constexpr int WS = kThreads / 64 / WU, VB = kUnitBlocks<T>;
    constexpr int DQ = 4 / WS;  // quads of dh of a lane
    __shared__ quad lds[NP * 256 * KS];
    __shared__ quad dh_lds[4][64 * DQ];
    const int lane = threadIdx.x & 63, w = wave_id(), g = lane >> 4, s = lane & 15;
    const int wu = w / WS, ws = w % WS;
    const int64_t u0 = ((int64_t)blockIdx.x * WU + wu) * (16 * VB);
    const int64_t t0 = blockIdx.y * per_share, t1 = min(tiles, t0 + per_share);
    const int64_t slot = (int64_t)blockIdx.y * WS + ws;
    bf16x8 wt[KS][VB][2][NP];  // gate, up
    float b[VB][2], sum[VB][2];
    f32x4 dw[VB][2][2 * KS];
#pragma unroll
    for (int v = 0; v < VB; ++v)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t unit = u0 + v * 16 + s;
            const bool on = unit < a.hidden;
            const float* bias = t ? a.b_up : a.b_gate;
            const T* row = static_cast<const T*>(t ? a.w_up : a.w_gate) +
                           (on ? unit : 0) * (t ? a.up_stride : a.gate_stride);
            b[v][t] = bias != nullptr && on ? bias[unit] : 0.0f;
            sum[v][t] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                Raw<T> raw;
                raw.load(row, k * 32 + g * 8, a.dim);
                raw.finish(k * 32 + g * 8, a.dim, on);
                quad q[NP];
                raw.parts(q);
#pragma unroll
                for (int p = 0; p < NP; ++p) wt[k][v][t][p] = __builtin_bit_cast(bf16x8, q[p]);
            }
#pragma unroll
            for (int c = 0; c < 2 * KS; ++c) dw[v][t][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    // the next tile's x and dh, cut when they are stored
    Raw<T> next[KS];
    constexpr int V = 16 / sizeof(T);
    Raw<T, V> next_d[DQ];
    auto fetch = [&](int64_t tile) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int blk = k * 4 + w;
            const int64_t i = tile * 64 + (blk / KS) * 16 + s;
            next[k].load(static_cast<const T*>(a.x) + (i < a.n ? i : 0) * a.x_stride,
                         (blk % KS) * 32 + g * 8, a.dim);
        }
#pragma unroll
        for (int k = 0; k < DQ; ++k) {
            const int64_t i = tile * 64 + ws * (64 / WS) + k * 16 + (lane >> 2);
            next_d[k].load(static_cast<const T*>(a.dh) + (i < a.n ? i : 0) * a.dh_stride,
                           u0 + (lane & 3) * V, a.hidden);
        }
    };
    if (t0 < t1) fetch(t0);
    for (int64_t tile = t0; tile < t1; ++tile) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            quad q[NP];
            next[k].finish(((k * 4 + w) % KS) * 32 + g * 8, a.dim,
                           tile * 64 + ((k * 4 + w) / KS) * 16 + s < a.n);
            next[k].parts(q);
#pragma unroll
            for (int p = 0; p < NP; ++p)
                lds[p * (256 * KS) + (k * 4 + w) * 64 + quad_place(s, g)] = q[p];
        }
        // a row's 64 bytes: bf16's 32-byte halves change places every fourth row, fp32's
        // rows within 4, so that rows 4 apart lie in other banks
#pragma unroll
        for (int k = 0; k < DQ; ++k) {
            const int r = k * 16 + (lane >> 2), q = lane & 3;
            if (u0 + 16 * VB > a.hidden || tile * 64 + 64 > a.n)
                next_d[k].finish(u0 + q * V, a.hidden, tile * 64 + ws * (64 / WS) + r < a.n);
            dh_lds[w][sizeof(T) == 2 ? r * 4 + (q ^ ((r >> 2 & 1) << 1))
                                     : (r ^ (r >> 2 & 3)) * 4 + q] = next_d[k].q[0];
        }
        __syncthreads();
        if (tile + 1 < t1) fetch(tile + 1);
#pragma unroll 1
        for (int half = ws; half < 2; half += WS) {  // 32 rows at a time
            const quad* at = lds + half * (2 * KS * 64);
            const int64_t left = a.n - (tile * 64 + half * 32);
            bf16x8 dz[VB][2][NP];
#pragma unroll
            for (int v = 0; v < VB; ++v) {  // one block at a time: the registers do not last for more
                f32x4 z[2][2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) z[t][j] = f32x4{b[v][t], b[v][t], b[v][t], b[v][t]};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    bf16x8 f[2][NP];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int p = 0; p < NP; ++p)
                            f[j][p] = operand_of(at + p * (256 * KS) + (j * KS + k) * 64);
                    multiply<NP>(f, wt[k][v], [&](int j, int t) -> f32x4& { return z[t][j]; });
                }
                // units u0 + 16 v + s, rows 16 j + 4 g + r of the 32
                float d[8];
                const char* from = reinterpret_cast<const char*>(dh_lds[w] + (half - ws) * 128);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (sizeof(T) == 2) {
                        typedef __attribute__((ext_vector_type(4))) short s16x4;
                        typedef __attribute__((address_space(3))) s16x4* lds4;
                        const int r = j * 16 + g * 4 + (s >> 2);
                        const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds4)(from + r * 64 + ((v ^ (g & 1)) * 32) + (s & 3) * 8));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            d[j * 4 + e] = __uint_as_float((uint32_t)(uint16_t)q[e] << 16);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = j * 16 + g * 4 + (e ^ g);
                            d[j * 4 + e] = *reinterpret_cast<const float*>(from + r * 64 + s * 4);
                        }
                    }
                }
                float dg[8], du[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float zg = z[0][e / 4][e % 4], zu = z[1][e / 4][e % 4];
                    dg[e] = plain_input<NP>(d[e] * zu * act_slope<ACT>(zg));
                    du[e] = plain_input<NP>(d[e] * act<ACT>(zg));
                }
                if (left < 32) {  // an infinite bias against a dh of 0 is NaN
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((e / 4) * 16 + g * 4 + e % 4 >= left) dg[e] = du[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum[v][0] += dg[e];
                    sum[v][1] += du[e];
                }
                quad q[NP];
                split8_input<NP>(dg, q);
#pragma unroll
                for (int p = 0; p < NP; ++p) dz[v][0][p] = __builtin_bit_cast(bf16x8, q[p]);
                split8_input<NP>(du, q);
#pragma unroll
                for (int p = 0; p < NP; ++p) dz[v][1][p] = __builtin_bit_cast(bf16x8, q[p]);
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                bf16x8 f[2][NP];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        f[m][p] = operand_across(at + p * (256 * KS) + k * 64, KS * 64, m);
#pragma unroll
                for (int v = 0; v < VB; ++v)
                    multiply<NP>(f, dz[v], [&](int m, int t) -> f32x4& { return dw[v][t][2 * k + m]; });
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * VB; ++i) {
        const int64_t r = u0 * 2 + i * 16 + s;
        f32x4* to = reinterpret_cast<f32x4*>(part + (slot * wr + r) * (32 * KS));
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m)
                to[k * 8 + g * 2 + (m ^ (g & 1))] = dw[i % VB][i / VB][2 * k + m];
        float v = sum[i % VB][i / VB];
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
        if (g == 0) db[slot * wr + r] = v;
    }
}

// The slots' sums as the weights' and biases' gradients: 64 quads of columns a workgroup,
// 16 runs of slots that are joined in order. The rows are 16 VB gate rows and the same units' up
// rows by turns.
template <typename T>
__global__ __launch_bounds__(1024) void k_gated_join(GatedArgs a, const float* part,
                                                     const float* db, int slots, int64_t wr, int ld) {
    constexpr int U = 16 * kUnitBlocks<T>;
    __shared__ f32x4 lds[16][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t quads = wr * (ld / 4), all = quads + wr / 4;
    const int per = (slots + 15) / 16, b0 = min(slots, run * per), b1 = min(slots, b0 + per);
    for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < all; e0 += (int64_t)gridDim.x * 64) {
        const int64_t e = e0 + lane;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e < all) {
            const f32x4* from = reinterpret_cast<const f32x4*>(e < quads ? part : db);
            const int64_t at = e < quads ? e : e - quads, step = e < quads ? quads : wr / 4;
#pragma unroll 8
            for (int b = b0; b < b1; ++b) v += from[b * step + at];
        }
        __syncthreads();  // what was there has been read
        lds[run][lane] = v;
        __syncthreads();
        if (run != 0 || e >= all) continue;
#pragma unroll
        for (int k = 1; k < 16; ++k) v += lds[k][lane];
        if (e < quads) {
            const int64_t r = e / (ld / 4), unit = r / (2 * U) * U + r % U;
            const bool up = (r & U) != 0;
            if (unit >= a.hidden) continue;
            T* row = static_cast<T*>(up ? a.dw_up : a.dw_gate) +
                     unit * (up ? a.dup_stride : a.dgate_stride);
            const float o[4] = {v[0], v[1], v[2], v[3]};
            store_cols<4>(row, (int)(e - r * (ld / 4)) * 4, a.dim, o);
        } else {
            const int64_t r = (e - quads) * 4, unit = r / (2 * U) * U + r % U;
            float* out = (r & U) != 0 ? a.db_up : a.db_gate;
            if (out == nullptr) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (unit + k < a.hidden) out[unit + k] = v[k];
        }
    }
}

// Up to so many rows the kernels do not fill the chip: 16 rows a wave, chunks in shares, and
// for h alone no launch to cut the weights before. h and a training pass so, then as more rows
// do, us: 16000 x 64 to 128 fp32 15 and 53, 18 and 59; 75 to 201 17 and 86, 24 and 96; 128 to
// 512 37 and 179, 54 and 209, bf16 15 and 76, 35 and 105. 24000 x 75 to 201 fp32 26 and 119,
// 25 and 118; 128 to 512 64 and 274, 54 and 263; bf16 of long rows goes over later (24000 24
// and 97, 35 and 118). bf16 x 64 to 128 does not gain: 16000 15 and 48, 14 and 44, by the
// launch that joins dx.
constexpr int64_t kFewerRows = 16384;

struct ShortPlan {
    int64_t chunks, tiles = 0, wr = 0;
    int ks, wu = 4;
    unsigned unit_blocks = 0, shares = 0;
    int64_t per_share = 0;
    int slots = 0;
    int64_t row_blocks, row_shares;  // of k_gated_rows with few rows
    quad* laid;
    float *part = nullptr, *db = nullptr, *dx = nullptr;
    size_t bytes;
    ShortPlan(void* base, int64_t n, int64_t hidden, int dim, int np, bool grad) {
        ks = (dim + 31) / 32;
        chunks = (hidden + 31) / 32;
        // with gradients each share's sums of dx are written and read: at least 2 chunks each
        row_blocks = (n + 63) / 64;
        row_shares = 1;
        if (n <= kFewerRows) {
            const int64_t want = std::max<int64_t>(1, std::min((grad ? chunks / 2 : chunks),
                                                               512 / std::max<int64_t>(1, row_blocks)));
            const int64_t per = (chunks + want - 1) / want;
            row_shares = (chunks + per - 1) / per;
        }
        Carve c(base);
        laid = np > 1 && (grad || n > kFewerRows) ? c.take<quad>((size_t)(chunks * np * 256 * ks))
                                                  : nullptr;
        if (grad) {
            const int64_t units = np > 1 ? 16 : 32;  // of a wave
            wu = hidden > 2 * units ? 4 : 2;
            unit_blocks = (unsigned)((hidden + wu * units - 1) / (wu * units));
            wr = (int64_t)unit_blocks * wu * 2 * units;
            tiles = (n + 63) / 64;
            // workgroups that run at a time: two a CU, of longer rows one
            const int64_t want = std::max<int64_t>(1, (ks <= 2 ? 512 : 256) / unit_blocks);
            per_share = std::max<int64_t>((tiles + want - 1) / want, 1);
            shares = (unsigned)std::max<int64_t>(1, (tiles + per_share - 1) / per_share);
            slots = (int)shares * (4 / wu);
            part = c.take<float>((size_t)slots * wr * 32 * ks);
            db = c.take<float>((size_t)slots * wr);
            dx = row_shares > 1 ? c.take<float>((size_t)(row_shares * row_blocks * 64 * 32 * ks))
                                : nullptr;
        }
        bytes = c.bytes();
    }
};

template <typename T, int NP, int ACT, int KS, int J, bool GRAD, bool LAID>
hipError_t rows_run(const GatedArgs& a, const ShortPlan& w, hipStream_t st) {
    const int64_t blocks = (a.n + 64 * J - 1) / (64 * J);
    const int64_t per = (w.chunks + w.row_shares - 1) / w.row_shares;
    for (int64_t at = 0; at < blocks; at += kMostBlocks) {
        const dim3 grid((unsigned)std::min(blocks - at, kMostBlocks), (unsigned)w.row_shares);
        k_gated_rows<T, NP, ACT, KS, J, GRAD, LAID>
            <<<grid, kThreads, 0, st>>>(a, w.laid, at, w.chunks, per, w.dx);
        GS_LAUNCHED();
    }
    return hipSuccess;
}

template <typename T, int NP, int ACT, int KS>
hipError_t short_run(const GatedArgs& a, bool grad, hipStream_t st) {
    const ShortPlan w(a.ws, a.n, a.hidden, a.dim, NP, grad);
    constexpr bool CUT = NP > 1;
    if (w.laid != nullptr) {
        k_gated_chunks<T, NP, KS><<<blocks_of(w.chunks * 256 * KS, kThreads), kThreads, 0, st>>>(
            a, w.chunks, w.laid);
        GS_LAUNCHED();
    }
    constexpr int kMost = NP == 1 ? 4 : 2, kMostGrad = NP == 1 ? 2 : (KS <= 2 ? 2 : 1);
    if (!grad)
        return a.n <= kFewerRows ? rows_run<T, NP, ACT, KS, 1, false, false>(a, w, st)
                                 : rows_run<T, NP, ACT, KS, kMost, false, CUT>(a, w, st);
    hipError_t e = a.n <= kFewerRows ? rows_run<T, NP, ACT, KS, 1, true, CUT>(a, w, st)
                                     : rows_run<T, NP, ACT, KS, kMostGrad, true, CUT>(a, w, st);
    if (e != hipSuccess) return e;
    if (w.row_shares > 1) {
        e = gated_dx_join(a, w.dx, (int)w.row_shares, w.row_blocks * 64, 32 * KS, 0, a.n, st);
        if (e != hipSuccess) return e;
    }
    const dim3 grid(w.unit_blocks, w.shares);
    if (w.wu == 4)
        k_gated_units<T, NP, ACT, KS, 4><<<grid, kThreads, 0, st>>>(a, w.tiles, w.per_share, w.wr,
                                                                   w.part, w.db);
    else
        k_gated_units<T, NP, ACT, KS, 2><<<grid, kThreads, 0, st>>>(a, w.tiles, w.per_share, w.wr,
                                                                   w.part, w.db);
    GS_LAUNCHED();
    const int64_t quads = w.wr * (32 * KS / 4) + w.wr / 4;
    k_gated_join<T><<<sum_blocks(quads), 1024, 0, st>>>(a, w.part, w.db, w.slots, w.wr,
                                                                    32 * KS);
    return hipGetLastError();
}

template <typename T, int NP, int ACT>
hipError_t short_steps(const GatedArgs& a, bool grad, hipStream_t st) {
    switch ((a.dim + 31) / 32) {
        case 1: return short_run<T, NP, ACT, 1>(a, grad, st);
        case 2: return short_run<T, NP, ACT, 2>(a, grad, st);
        case 3: return short_run<T, NP, ACT, 3>(a, grad, st);
        default: return short_run<T, NP, ACT, 4>(a, grad, st);
    }
}
template <typename T, int NP>
hipError_t short_act(const GatedArgs& a, bool grad, hipStream_t st) {
    switch (a.act) {
        case kActRelu: return short_steps<T, NP, kActRelu>(a, grad, st);
        case kActSilu: return short_steps<T, NP, kActSilu>(a, grad, st);
        case kActGelu: return short_steps<T, NP, kActGelu>(a, grad, st);
        default: return short_steps<T, NP, kActNone>(a, grad, st);
    }
}

}  // namespace

}  // namespace gs
