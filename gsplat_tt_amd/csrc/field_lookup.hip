// field_lookup.hip - rows of a feature table by id, and the table's gradient.
//
//   out[i]    = scale * table[ids[i]]            (zeros for an id outside [0, rows))
//   dtable[v] = scale * sum over ids[i] = v of dout[i]
//
// The gradient is by sorted ids: a stable radix sort of (id, position), then
// each id's run of rows is summed in position order, so the result does not
// depend on timing. Sums are held in fp32.
#include <type_traits>

#include "field.h"

#include "field_device.h"

namespace gs {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- lookup
// A workgroup takes R consecutive ids, stages where their rows begin in LDS and
// writes the rows in memory order, a unit of VEC values a lane, so that reads
// and writes of a wave are contiguous whatever the row length. A thread's next
// unit lies kThreads further: its row and column follow by addition, where a
// division a unit took longer than the memory.
//
// FLAT: the output has no gaps, so a unit is 16 aligned bytes of it whatever the
// row length, read in one (unaligned) load; only the units that hold a row's end
// are read value by value. Else a unit is a divisor of a row. Outputs are stored
// past the caches, which are left to the table.
constexpr int kLookupRows = 1024;  // most ids of a workgroup
constexpr int kLookupUnits = 4;    // units that a thread loads before it stores

template <typename TT, typename TO, int VEC, bool FLAT>
__global__ __launch_bounds__(kThreads) void k_lookup(LookupArgs a, int R) {
    __shared__ int64_t start[kLookupRows];
    const TT* table = static_cast<const TT*>(a.table);
    TO* out = static_cast<TO*>(a.out);
    const uint32_t dim = (uint32_t)a.dim;
    const uint32_t step_r = kThreads * VEC / dim, step_c = kThreads * VEC % dim;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.n; r0 += (int64_t)gridDim.x * R) {
        const int nr = (int)min((int64_t)R, a.n - r0);
        __syncthreads();
        for (int i = threadIdx.x; i < nr; i += kThreads) {
            const int32_t t = load_id(a.ids, a.ids64, r0 + i, a.rows, a.flags);
            start[i] = t >= 0 ? t * a.table_stride : -1;
        }
        __syncthreads();
        uint32_t r = threadIdx.x * VEC / dim, c = threadIdx.x * VEC % dim;
        const uint32_t total = (uint32_t)nr * dim;
        TO* to = out + r0 * a.out_stride;
        for (uint32_t e0 = threadIdx.x * VEC; e0 < total; e0 += kThreads * kLookupUnits * VEC) {
            float v[kLookupUnits][VEC];
            uint32_t rk = r, ck = c;
#pragma unroll
            for (int k = 0; k < kLookupUnits; ++k) {
                const uint32_t e = e0 + k * kThreads * VEC;
                if (!FLAT || ck + VEC <= dim) {
                    const int64_t from = e < total ? start[rk] : -1;
                    if (from >= 0) {
                        load_any<VEC>(table + from + ck, v[k]);
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
                    }
                } else {
                    uint32_t rj = rk, cj = ck;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int64_t from = e + j < total ? start[rj] : -1;
                        v[k][j] = from >= 0 ? to_float(table[from + cj]) : 0.0f;
                        if (++cj == dim) {
                            cj = 0;
                            ++rj;
                        }
                    }
                }
                rk += step_r;
                ck += step_c;
                if (ck >= dim) {
                    ck -= dim;
                    ++rk;
                }
            }
#pragma unroll
            for (int k = 0; k < kLookupUnits; ++k) {
                const uint32_t e = e0 + k * kThreads * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[k][j] *= a.scale;
                if (FLAT) {
                    if (e + VEC <= total) {
                        store_nt<VEC>(to + e, v[k]);
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            if (e + j < total) to[e + j] = from_float<TO>(v[k][j]);
                    }
                } else if (e < total) {
                    store_nt<VEC>(to + r * a.out_stride + c, v[k]);
                }
                r += step_r;
                c += step_c;
                if (c >= dim) {
                    c -= dim;
                    ++r;
                }
            }
        }
    }
}

template <typename TT, typename TO, int VEC, bool FLAT>
hipError_t lookup_run(const LookupArgs& a, hipStream_t st) {
    // about kLookupUnits units a thread, whole groups of 8 rows (16-byte multiples)
    const int64_t want = (int64_t)kThreads * kLookupUnits * VEC;
    int64_t R = (want / a.dim + 7) / 8 * 8;
    R = R < 8 ? 8 : (R > kLookupRows ? kLookupRows : R);
    // fewer where that leaves compute units idle
    while (R > 8 && a.n / R < 1024) R = R / 2 / 8 * 8 < 8 ? 8 : R / 2 / 8 * 8;
    const int64_t blocks = (a.n + R - 1) / R;
    const dim3 grid((unsigned)(blocks < (1 << 30) ? blocks : (1 << 30)));
    k_lookup<TT, TO, VEC, FLAT><<<grid, kThreads, 0, st>>>(a, (int)R);
    return hipGetLastError();
}

// Gapless aligned outputs by 16 bytes; else the widest unit that divides a row and
// every output row's address.
template <typename TT, typename TO>
hipError_t lookup_typed(const LookupArgs& a, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(TO);
    if ((a.out_stride == a.dim || a.n == 1) && aligned_rows<TO>(a.out, 0, VEC))
        return lookup_run<TT, TO, VEC, true>(a, st);
    auto fits = [&](int v) { return a.dim % v == 0 && aligned_rows<TO>(a.out, a.out_stride, v); };
    if (fits(4)) return lookup_run<TT, TO, 4, false>(a, st);
    if (fits(2)) return lookup_run<TT, TO, 2, false>(a, st);
    return lookup_run<TT, TO, 1, false>(a, st);
}

// ---------------------------------------------------------------- sort
// Stable LSD radix sort of (id, position), 8 bits a pass at most: per block the
// digits' counts, per digit the blocks' offsets, then the scatter. The first
// pass reads the caller's ids; those outside the table get the key `rows` and
// end last.
__device__ __forceinline__ uint32_t sort_key(const LookupGradArgs& a, const uint2* pairs,
                                             int64_t i, uint32_t* flags) {
    if (pairs != nullptr) return pairs[i].x;
    const int32_t t = load_id(a.ids, a.ids64, i, a.rows, flags);
    return t >= 0 ? (uint32_t)t : (uint32_t)a.rows;
}

// Rank of a wave's keys among its earlier ones of the same digit, 64 keys a call
// in order: the lanes of equal digit are found with one ballot a bit; `seen` (LDS,
// this wave's) counts each digit so far.
__device__ __forceinline__ uint32_t wave_rank(uint32_t digit, bool on, int bits, uint32_t* seen) {
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((digit >> b) & 1u);
        same &= ((digit >> b) & 1u) ? m : ~m;
    }
    const uint32_t before = __popcll(same & ((1ull << (threadIdx.x & 63)) - 1ull));
    volatile uint32_t* mine = seen + digit;  // other lanes of the wave write it
    const uint32_t n = on ? *mine : 0u;
    __builtin_amdgcn_wave_barrier();
    if (on && before == 0) *mine = n + (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
    return n + before;
}

// Also clears the ids' runs, which k_run_sums fills in.
template <int ITEMS>
__global__ __launch_bounds__(kThreads) void k_sort_count(LookupGradArgs a, const uint2* pairs,
                                                         int shift, int bits, uint32_t* counts,
                                                         uint2* runs) {
    __shared__ uint32_t hist[256];
    hist[threadIdx.x] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (kThreads * ITEMS);
    const uint32_t mask = (1u << bits) - 1u;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = base + k * kThreads + threadIdx.x;
        if (i < a.n) atomicAdd(&hist[(sort_key(a, pairs, i, a.flags) >> shift) & mask], 1u);
    }
    if (runs != nullptr)
        for (int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x; v < a.rows;
             v += (int64_t)gridDim.x * kThreads)
            runs[v] = make_uint2(0u, 0u);
    __syncthreads();
    if (threadIdx.x < (1u << bits))
        counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x] = hist[threadIdx.x];
}

// One workgroup per digit: exclusive prefix of its blocks' counts, and its total.
__global__ __launch_bounds__(kThreads) void k_sort_scan(uint32_t* counts, int blocks,
                                                        uint32_t* totals) {
    __shared__ uint32_t part[kThreads / 64];
    uint32_t* row = counts + (size_t)blockIdx.x * blocks;
    uint32_t base = 0;
    for (int i0 = 0; i0 < blocks; i0 += kThreads * 4) {
        uint32_t c[4], sum = 0;
        const int i = i0 + threadIdx.x * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            c[k] = i + k < blocks ? row[i + k] : 0u;
            sum += c[k];
        }
        uint32_t total;
        uint32_t at = base + block_excl_scan<kThreads>(sum, part, &total);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k < blocks) row[i + k] = at;
            at += c[k];
        }
        base += total;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = base;
}

template <int ITEMS>
__global__ __launch_bounds__(kThreads) void k_sort_scatter(LookupGradArgs a, const uint2* pairs,
                                                           int shift, int bits,
                                                           const uint32_t* counts,
                                                           const uint32_t* totals, uint2* out) {
    constexpr int kWaves = kThreads / 64;
    __shared__ uint32_t cnt[kWaves][256];
    __shared__ uint32_t part[kWaves];
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    const int digits = 1 << bits;
    const uint32_t mask = digits - 1u;
    const uint32_t mine = t < digits ? totals[t] : 0u;
    const uint32_t offset = t < digits ? counts[(size_t)t * gridDim.x + blockIdx.x] : 0u;
    for (int k = 0; k < kWaves; ++k) cnt[k][t] = 0u;
    const int64_t base = (int64_t)blockIdx.x * (kThreads * ITEMS) + (int64_t)w * 64 * ITEMS;
    uint2 pair[ITEMS];
    uint32_t rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = base + k * 64 + lane;
        pair[k] = make_uint2(0u, (uint32_t)i);
        if (i < a.n) {
            if (pairs != nullptr)
                pair[k] = pairs[i];
            else
                pair[k].x = sort_key(a, nullptr, i, nullptr);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        rank[k] = wave_rank((pair[k].x >> shift) & mask, base + k * 64 + lane < a.n, bits, cnt[w]);
    // digit starts: all smaller digits' totals, this block's offset, earlier waves
    uint32_t all;
    uint32_t at = block_excl_scan<kThreads>(mine, part, &all) + offset;
    if (t < digits)
        for (int k = 0; k < kWaves; ++k) {
            const uint32_t c = cnt[k][t];
            cnt[k][t] = at;
            at += c;
        }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (base + k * 64 + lane < a.n)
            out[cnt[w][(pair[k].x >> shift) & mask] + rank[k]] = pair[k];
}

// ---------------------------------------------------------------- run sums
// A workgroup takes a span of (id, position) in id order, its slots of `lpr` lanes
// (VEC columns a lane) equal stretches of it. Runs inside a stretch are finished
// at once; each stretch's first and last run are joined over the slots in LDS,
// in order.
//
// Two uses. Where ids have to be sorted over the whole list (LOCAL false), spans
// follow that order: a run inside a span is a row's whole sum, and a span's first
// and last run, where they go on in its neighbours, are added up by k_run_join
// from `part` (span, 2, dim). With few rows (LOCAL) no such sort is needed: a span
// is some consecutive ids that the workgroup sorts itself, and each row's sum
// over it goes to `part` (span, rows, dim). That reads dout almost in order, in 2
// launches instead of 5.
constexpr int kSpan = 1024;      // most entries of a span
constexpr int kLocalRows = 128;  // most rows for LOCAL: an eighth or a quarter of the span

template <typename TD, int VEC>
__device__ __forceinline__ void put_row(TD* out, const float* acc, float scale, int accumulate,
                                        int n = VEC) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (j < n) {
            float s = acc[j] * scale;
            if (accumulate) s += to_float(out[j]);
            out[j] = from_float<TD>(s);
        }
}

template <typename TI, typename TD, int VEC, bool LOCAL>
__global__ __launch_bounds__(kThreads) void k_run_sums(LookupGradArgs a, const uint2* pairs,
                                                       int span, int lpr, int bits, float* part,
                                                       uint2* runs) {
    constexpr int kWaves = kThreads / 64;
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    __shared__ uint32_t skey[kSpan], spos[kSpan];
    __shared__ float ends[kThreads * 2 * VEC];  // (slot, first or last, column)
    __shared__ uint32_t end_key[kThreads * 2];
    const TI* dout = static_cast<const TI*>(a.dout);
    TD* dtable = static_cast<TD*>(a.dtable);
    const int t = threadIdx.x, cols = lpr * VEC, c0 = blockIdx.y * cols;
    const int slots = kThreads / lpr, slot = t / lpr, lane = t % lpr;
    const int c = c0 + lane * VEC;
    const uint32_t rows = (uint32_t)a.rows;
    const int64_t base = (int64_t)blockIdx.x * span;
    const int m = (int)min((int64_t)span, a.n - base);
    uint32_t before = kNone, after = kNone;  // the neighbours' keys
    if (LOCAL) {
        __shared__ uint32_t cnt[kWaves][kLocalRows + 1];
        __shared__ uint32_t scan[kWaves];
        for (int k = t; k < kWaves * (kLocalRows + 1); k += kThreads) (&cnt[0][0])[k] = 0u;
        __syncthreads();
        const int w = t >> 6, l = t & 63;
        uint32_t key[kSpan / kThreads], rank[kSpan / kThreads];
#pragma unroll
        for (int k = 0; k < kSpan / kThreads; ++k) {
            if (k >= span / kThreads) break;
            const int i = w * (span / kWaves) + k * 64 + l;
            key[k] = i < m ? sort_key(a, nullptr, base + i, blockIdx.y == 0 ? a.flags : nullptr) : 0u;
            rank[k] = wave_rank(key[k], i < m, bits, cnt[w]);
        }
        __syncthreads();
        uint32_t mine = 0, all;
        if (t <= (int)rows)
            for (int k = 0; k < kWaves; ++k) mine += cnt[k][t];
        uint32_t at = block_excl_scan<kThreads>(mine, scan, &all);
        if (t <= (int)rows)
            for (int k = 0; k < kWaves; ++k) {
                const uint32_t n = cnt[k][t];
                cnt[k][t] = at;
                at += n;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSpan / kThreads; ++k) {
            const int i = w * (span / kWaves) + k * 64 + l;
            if (k < span / kThreads && i < m) {
                const uint32_t to = cnt[w][key[k]] + rank[k];
                skey[to] = key[k];
                spos[to] = (uint32_t)(base + i);
            }
        }
        __syncthreads();
        // rows that no id of the span names
        float* row0 = part + (size_t)blockIdx.x * rows * a.dim;
        for (uint32_t v = slot; v < rows; v += slots) {
            const uint32_t lo = cnt[0][v];
            if (lo < (uint32_t)m && skey[lo] == v) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < a.dim) row0[(size_t)v * a.dim + c + j] = 0.0f;
        }
    } else {
        for (int i = t; i < m; i += kThreads) {
            const uint2 p = pairs[base + i];
            skey[i] = p.x;
            spos[i] = p.y;
        }
        if (base > 0) before = pairs[base - 1].x;
        if (base + m < a.n) after = pairs[base + m].x;
        __syncthreads();
        if (blockIdx.y == 0)
            for (int i = t; i < m; i += kThreads) {
                const uint32_t k = skey[i];
                if (k >= rows) continue;
                if ((i > 0 ? skey[i - 1] : before) != k) runs[k].x = (uint32_t)(base + i);
                if ((i + 1 < m ? skey[i + 1] : after) != k) runs[k].y = (uint32_t)(base + i + 1);
            }
    }
    // a run's sum over the span; `which`: 0 it holds the span's first entry, 1 only
    // its last, 2 neither
    auto finish = [&](uint32_t key, const float* acc, int at, int which, auto width) {
        constexpr int W = decltype(width)::value;
        if (key >= rows) return;
        const int n = min(W, a.dim - at);
        if (LOCAL || which < 2) {
            const size_t row = LOCAL ? (size_t)blockIdx.x * rows + key
                                     : (size_t)blockIdx.x * 2 + which;
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (j < n) part[row * a.dim + at + j] = acc[j];
        } else {
            put_row<TD, W>(dtable + (int64_t)key * a.dtable_stride + at, acc, a.scale,
                           a.accumulate, n);
        }
    };

    const int per = span / slots, lo = min(m, slot * per), hi = min(m, lo + per);
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    uint32_t cur = lo < hi ? skey[lo] : kNone, first = cur;
    bool single = true;
    const bool col_on = c < a.dim, whole = c + VEC <= a.dim;
    constexpr int U = 8;  // rows in flight
    for (int i0 = lo; i0 < hi; i0 += U) {
        float v[U][VEC];
        uint32_t k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = i0 + u < hi ? skey[i0 + u] : kNone;
            const bool on = k[u] < rows && col_on;
            const TI* src = dout + (on ? (int64_t)spos[i0 + u] * a.dout_stride + c : 0);
            if (on && whole) {
                load_any<VEC>(src, v[u]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    v[u][j] = on && c + j < a.dim ? to_float(src[j]) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k[u] == kNone) continue;
            if (k[u] != cur) {
                if (single) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ends[(slot * 2) * cols + lane * VEC + j] = acc[j];
                    single = false;
                } else if (col_on) {
                    finish(cur, acc, c, 2, std::integral_constant<int, VEC>());
                }
                cur = k[u];
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        ends[(slot * 2 + (single ? 0 : 1)) * cols + lane * VEC + j] = acc[j];
    if (lane == 0) {
        end_key[slot * 2] = first;
        end_key[slot * 2 + 1] = single ? kNone : cur;
    }
    __syncthreads();
    for (int j = t; j < cols && c0 + j < a.dim; j += kThreads) {
        uint32_t key = end_key[0];
        const uint32_t span_first = key;
        float sum = 0.0f;
        bool begin = true;  // the run holds the span's first entry
        constexpr int E = 8;
        for (int e0 = 0; e0 < slots * 2; e0 += E) {
            uint32_t k[E];
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool on = e0 + e < slots * 2;
                k[e] = on ? end_key[e0 + e] : kNone;
                v[e] = on ? ends[(e0 + e) * cols + j] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (k[e] == kNone) continue;
                if (k[e] != key) {
                    finish(key, &sum, c0 + j, begin && before == span_first ? 0 : 2,
                           std::integral_constant<int, 1>());
                    begin = false;
                    key = k[e];
                    sum = 0.0f;
                }
                sum += v[e];
            }
        }
        const bool more = after == key;
        const int which = begin ? (before == span_first || more ? 0 : 2) : (more ? 1 : 2);
        finish(key, &sum, c0 + j, which, std::integral_constant<int, 1>());
    }
}

// Rows whose run crosses spans: the sum of the spans' pieces in order; zeros for
// rows that no id names. A wave a row; a row of many pieces takes the workgroup,
// each wave every fourth piece.
constexpr int kWavePieces = 32;

template <typename TD>
__global__ __launch_bounds__(kThreads) void k_run_join(LookupGradArgs a, const uint2* runs,
                                                       int span, const float* part) {
    __shared__ float sums[kThreads];
    TD* dtable = static_cast<TD*>(a.dtable);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // sum of pieces s0 + k, s0 + k + by, .. of column c
    auto pieces = [&](uint2 run, uint32_t k, uint32_t by, int c) {
        const uint32_t s0 = run.x / (uint32_t)span, s1 = (run.y - 1u) / (uint32_t)span;
        float acc = 0.0f;
        for (uint32_t s = s0 + k; s <= s1; s += by * 4) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t q = s + u * by;
                const int which = q == s0 && run.x % (uint32_t)span != 0u ? 1 : 0;
                v[u] = q <= s1 ? part[((size_t)q * 2 + which) * a.dim + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) acc += v[u];
        }
        return acc;
    };
    auto count = [&](uint2 run) {
        return run.x == run.y ? 0u : (run.y - 1u) / (uint32_t)span - run.x / (uint32_t)span + 1u;
    };
    for (int64_t v0 = (int64_t)blockIdx.x * 4; v0 < a.rows; v0 += (int64_t)gridDim.x * 4) {
        const int64_t v = v0 + w;
        if (v < a.rows) {
            const uint2 run = runs[v];
            const uint32_t n = count(run);
            TD* out = dtable + v * a.dtable_stride;
            if (n == 0 && !a.accumulate)
                for (int c = lane; c < a.dim; c += 64) out[c] = from_float<TD>(0.0f);
            if (n > 1 && n <= kWavePieces)
                for (int c = lane; c < a.dim; c += 64) {
                    const float acc = pieces(run, 0, 1, c);
                    put_row<TD, 1>(out + c, &acc, a.scale, a.accumulate);
                }
        }
        for (int k = 0; k < 4 && v0 + k < a.rows; ++k) {
            const uint2 run = runs[v0 + k];
            if (count(run) <= kWavePieces) continue;
            for (int cb = 0; cb < a.dim; cb += 64) {
                const int c = cb + lane;
                float acc = c < a.dim ? pieces(run, w, kThreads / 64, c) : 0.0f;
                __syncthreads();
                sums[threadIdx.x] = acc;
                __syncthreads();
                if (w == 0 && c < a.dim) {
                    for (int q = 1; q < kThreads / 64; ++q) acc += sums[q * 64 + lane];
                    put_row<TD, 1>(dtable + (v0 + k) * a.dtable_stride + c, &acc, a.scale,
                                   a.accumulate);
                }
            }
        }
    }
}

// LOCAL's join: a workgroup per row and 16 columns, 16 slots over the spans.
template <typename TD>
__global__ __launch_bounds__(kThreads) void k_local_join(LookupGradArgs a, int spans,
                                                         const float* part) {
    __shared__ float sums[16][17];
    const int slot = threadIdx.x >> 4, j = threadIdx.x & 15;
    const int64_t v = blockIdx.x;
    const int c = blockIdx.y * 16 + j;
    float acc = 0.0f;
    if (c < a.dim)
        for (int s0 = slot; s0 < spans; s0 += 16 * 8) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = s0 + u * 16;
                x[u] = s < spans ? part[((size_t)s * a.rows + v) * a.dim + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) acc += x[u];
        }
    sums[slot][j] = acc;
    __syncthreads();
    if (slot == 0 && c < a.dim) {
        for (int q = 1; q < 16; ++q) acc += sums[q][j];
        put_row<TD, 1>(static_cast<TD*>(a.dtable) + v * a.dtable_stride + c, &acc, a.scale,
                       a.accumulate);
    }
}

int key_bits(int64_t rows) {  // keys 0 .. rows
    int b = 1;
    while (((int64_t)1 << b) <= rows) ++b;
    return b;
}

// Consecutive ids of a LOCAL span: fewer where that fills the chip.
int local_span(int64_t n) { return n <= (1 << 19) ? kSpan / 2 : kSpan; }

bool is_local(int64_t n, int64_t rows) { return rows <= kLocalRows && n > 0; }

// Entries of a span of the sorted list: at most 4096 spans while spans can grow,
// so that one row's pieces stay few.
int span_of(int64_t n) {
    int s = 256;
    while (s < kSpan && n / s > 4096) s *= 2;
    return s;
}

// Keys of a sort block's thread: fewer where that fills the chip.
int sort_items(int64_t n) { return n <= (1 << 21) ? 4 : 16; }

struct GradWs {
    uint2 *pairs[2], *runs;
    uint32_t *counts, *totals;
    float* part;
    size_t bytes;
    GradWs(void* base, int64_t n, int64_t rows, int dim) {
        Carve c(base);
        if (is_local(n, rows)) {
            const int span = local_span(n);
            part = c.take<float>((size_t)((n + span - 1) / span) * rows * dim);
        } else {
            const int64_t tile = (int64_t)kThreads * sort_items(n);
            for (int k = 0; k < 2; ++k) pairs[k] = c.take<uint2>((size_t)n);
            counts = c.take<uint32_t>((size_t)((n + tile - 1) / tile) * 256);
            totals = c.take<uint32_t>(256);
            runs = c.take<uint2>((size_t)rows);
            const int span = span_of(n);
            part = c.take<float>((size_t)((n + span - 1) / span) * 2 * dim);
        }
        bytes = c.bytes();
    }
};

template <typename TI, typename TD>
hipError_t grad_typed(const LookupGradArgs& a, const GradWs& w, const uint2* pairs,
                      hipStream_t st) {
    constexpr int VEC = 16 / sizeof(TI);
    const int units = (a.dim + VEC - 1) / VEC;
    int lpr = 1;
    while (lpr < 64 && lpr < units) lpr *= 2;
    const unsigned cols = (unsigned)((units + lpr - 1) / lpr);
    if (is_local(a.n, a.rows)) {
        const int span = local_span(a.n), spans = (int)((a.n + span - 1) / span);
        k_run_sums<TI, TD, VEC, true><<<dim3((unsigned)spans, cols), kThreads, 0, st>>>(
            a, nullptr, span, lpr, key_bits(a.rows), w.part, nullptr);
        k_local_join<TD><<<dim3((unsigned)a.rows, (unsigned)((a.dim + 15) / 16)), kThreads, 0, st>>>(
            a, spans, w.part);
        return hipGetLastError();
    }
    const int span = span_of(a.n);
    if (a.n > 0)
        k_run_sums<TI, TD, VEC, false>
            <<<dim3((unsigned)((a.n + span - 1) / span), cols), kThreads, 0, st>>>(
                a, pairs, span, lpr, 0, w.part, w.runs);
    const int64_t joins = (a.rows + 3) / 4;
    k_run_join<TD><<<(unsigned)(joins < 65536 ? joins : 65536), kThreads, 0, st>>>(a, w.runs, span,
                                                                                w.part);
    return hipGetLastError();
}

template <int ITEMS>
const uint2* sort_ids(const LookupGradArgs& a, const GradWs& w, hipStream_t st) {
    const int bits = key_bits(a.rows), passes = (bits + 7) / 8;
    const unsigned blocks = (unsigned)((a.n + kThreads * ITEMS - 1) / (kThreads * ITEMS));
    const uint2* pairs = nullptr;
    for (int p = 0, done = 0; p < passes; ++p) {
        const int b = (bits - done + passes - p - 1) / (passes - p);
        k_sort_count<ITEMS><<<blocks, kThreads, 0, st>>>(a, pairs, done, b, w.counts,
                                                         p == 0 ? w.runs : nullptr);
        k_sort_scan<<<1u << b, kThreads, 0, st>>>(w.counts, (int)blocks, w.totals);
        k_sort_scatter<ITEMS><<<blocks, kThreads, 0, st>>>(a, pairs, done, b, w.counts, w.totals,
                                                           w.pairs[p & 1]);
        pairs = w.pairs[p & 1];
        done += b;
    }
    return pairs;
}

__global__ __launch_bounds__(kThreads) void k_run_clear(uint2* runs, int64_t rows) {
    const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (v < rows) runs[v] = make_uint2(0u, 0u);
}

}  // namespace

hipError_t launch_lookup(const LookupArgs& a, hipStream_t st) {
    if (a.n == 0) return hipSuccess;
    if (a.table_dtype == 0)
        return a.out_dtype == 0 ? lookup_typed<float, float>(a, st)
                                : lookup_typed<float, bf16>(a, st);
    return a.out_dtype == 0 ? lookup_typed<bf16, float>(a, st) : lookup_typed<bf16, bf16>(a, st);
}

size_t lookup_grad_ws(int64_t n, int64_t rows, int dim) {
    return GradWs(nullptr, n, rows, dim).bytes;
}

hipError_t launch_lookup_grad(const LookupGradArgs& a, hipStream_t st) {
    if (a.rows == 0) return hipSuccess;
    const GradWs w(a.ws, a.n, a.rows, a.dim);
    const uint2* pairs = nullptr;
    if (a.n == 0)
        k_run_clear<<<(unsigned)((a.rows + kThreads - 1) / kThreads), kThreads, 0, st>>>(w.runs,
                                                                                      a.rows);
    else if (!is_local(a.n, a.rows))
        pairs = sort_items(a.n) == 4 ? sort_ids<4>(a, w, st) : sort_ids<16>(a, w, st);
    if (a.dout_dtype == 0)
        return a.dtable_dtype == 0 ? grad_typed<float, float>(a, w, pairs, st)
                                   : grad_typed<float, bf16>(a, w, pairs, st);
    return a.dtable_dtype == 0 ? grad_typed<bf16, float>(a, w, pairs, st)
                               : grad_typed<bf16, bf16>(a, w, pairs, st);
}

}  // namespace gs
