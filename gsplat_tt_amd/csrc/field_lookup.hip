// field_lookup.hip - rows of a feature table by id, and the table's gradient.
//
//   out[i]    = scale * table[ids[i]]            (zeros for an id outside [0, rows))
//   dtable[v] = scale * sum over ids[i] = v of dout[i]
//
// The gradient is by sorted ids: a stable radix sort of (id, position), then
// each id's run of rows is summed in position order, so the result does not
// depend on timing. Sums are held in fp32.
#include <algorithm>

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
// past the caches, which are left to the table. Bound by the output's bytes: 6000000
// rows of 45 fp32 from 65536 take 215 us, 5.1 TB/s, as fast as a copy; by divisors
// of a row 288. 4096 rows of 32 take 4 us, 9 with the call.
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
    k_lookup<TT, TO, VEC, FLAT><<<blocks_of(a.n, R), kThreads, 0, st>>>(a, (int)R);
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
// end last. Bound by launches and latency up to a few million ids: 1000000 ids of 4096
// rows take 35 us in 6 launches, of the gradient's 87.
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

// Also clears the ids' runs (unless null), which k_run_sums fills in.
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

// The whole sort of a short list in one workgroup's LDS.
constexpr int kShortThreads = 1024;
constexpr int kShort = 4096;

__global__ __launch_bounds__(kShortThreads) void k_sort_short(LookupGradArgs a, int bits_all,
                                                              uint2* out, uint2* runs) {
    constexpr int kWaves = kShortThreads / 64, kItems = kShort / kShortThreads;
    __shared__ uint2 list[kShort];
    __shared__ uint32_t cnt[kWaves][256];
    __shared__ uint32_t part[kWaves];
    const int t = threadIdx.x, w = t >> 6, lane = t & 63, n = (int)a.n;
    const int base = w * 64 * kItems;
    for (int64_t v = t; v < a.rows; v += kShortThreads) runs[v] = make_uint2(0u, 0u);
    uint2 pair[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int i = base + k * 64 + lane;
        pair[k] = make_uint2(i < n ? sort_key(a, nullptr, i, a.flags) : 0u, (uint32_t)i);
    }
    const int passes = (bits_all + 7) / 8;
    for (int p = 0, done = 0; p < passes; ++p) {
        const int bits = (bits_all - done + passes - p - 1) / (passes - p), digits = 1 << bits;
        for (int k = t; k < kWaves * 256; k += kShortThreads) (&cnt[0][0])[k] = 0u;
        __syncthreads();
        uint32_t rank[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            rank[k] = wave_rank((pair[k].x >> done) & (digits - 1u), base + k * 64 + lane < n, bits,
                                cnt[w]);
        __syncthreads();
        uint32_t mine = 0, all;
        if (t < digits)
            for (int k = 0; k < kWaves; ++k) mine += cnt[k][t];
        uint32_t at = block_excl_scan<kShortThreads>(mine, part, &all);
        if (t < digits)
            for (int k = 0; k < kWaves; ++k) {
                const uint32_t c = cnt[k][t];
                cnt[k][t] = at;
                at += c;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (base + k * 64 + lane < n)
                list[cnt[w][(pair[k].x >> done) & (digits - 1u)] + rank[k]] = pair[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (base + k * 64 + lane < n) pair[k] = list[base + k * 64 + lane];
        done += bits;
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k)
        if (base + k * 64 + lane < n) out[base + k * 64 + lane] = pair[k];
}

// ---------------------------------------------------------------- run sums
// A workgroup takes a span of (id, position) in id order, its slots of `lpr` lanes
// (VEC columns a lane) equal stretches of it. Runs inside a stretch are finished
// at once; runs over several stretches are joined by a segmented scan over the
// slots, in a fixed order.
//
// Three uses. Where ids have to be sorted over the whole list (kSorted), spans
// follow that order: a run inside a span is a row's whole sum, and a span's first
// and last run, where they go on in its neighbours, are added up by k_run_join
// from `part` (span, 2, dim). With few rows (kLocal) no such sort is needed: a span
// is some consecutive ids that the workgroup sorts itself, and each row's sum
// over it goes to `part` (span, rows, dim). That reads dout almost in order, in 2
// launches instead of 5. With few ids (kOwn) each workgroup takes kLocalRows rows
// of the table, looks through all ids for them and writes those rows whole: one
// launch.
//
// Bound by dout's bytes and their latency: sorted, rows of dout come in random order,
// 1000000 of 48 fp32 in 42 us, 4.6 TB/s, and 9 for the join. 307200 x 64 bf16 into 24
// rows: 20 us and 4, sorted 59 in all.
enum { kSorted = 0, kLocal = 1, kOwn = 2 };
constexpr int kSpan = 4096;      // most entries of a span
constexpr int kLocalRows = 128;  // most rows for kLocal: a quarter of the least span

// scale * acc into (or onto) values lo .. hi - 1 of VEC ones of a row, at once where
// that is all of them.
template <typename TD, int VEC>
__device__ __forceinline__ void put_row(TD* out, const float* acc, float scale, int accumulate,
                                        int lo = 0, int hi = VEC) {
    float s[VEC];
    if (lo == 0 && hi == VEC) {
        if (accumulate) {
            load_any<VEC>(out, s);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j] += acc[j] * scale;
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j] = acc[j] * scale;
        }
        store_any<VEC>(out, s);
        return;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (j >= lo && j < hi) {
            float v = acc[j] * scale;
            if (accumulate) v += to_float(out[j]);
            out[j] = from_float<TD>(v);
        }
}

template <typename TI, typename TD, int VEC, int MODE>
__global__ __launch_bounds__(kThreads) void k_run_sums(LookupGradArgs a, const uint2* pairs,
                                                       int span, int lpr, int bits, float* part,
                                                       uint2* runs) {
    constexpr int kWaves = kThreads / 64;
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    extern __shared__ uint32_t entries[];
    uint32_t *skey = entries, *spos = entries + span;
    __shared__ float carry[kThreads / 64][64 * VEC];     // the waves' last runs
    __shared__ uint32_t carry_flags[kThreads / 64];
    __shared__ uint32_t first_key[kThreads], last_key[kThreads];
    const TI* dout = static_cast<const TI*>(a.dout);
    TD* dtable = static_cast<TD*>(a.dtable);
    const int t = threadIdx.x, cols = lpr * VEC, c0 = blockIdx.y * cols;
    const int slots = kThreads / lpr, slot = t / lpr, lane = t % lpr;
    // the lane's columns: of a row's last ones that make no vector, a vector that ends
    // with the row is read, and its first values, the lane before's, are not written
    const bool col_on = c0 + lane * VEC < a.dim, whole = a.dim >= VEC;
    const int c = whole ? min(c0 + lane * VEC, a.dim - VEC) : 0;
    const int c_lo = c0 + lane * VEC - c, c_hi = whole ? VEC : a.dim;
    // kOwn: the workgroup's rows of the table, and keys counted from their first
    const int64_t row0 = MODE == kOwn ? (int64_t)blockIdx.x * kLocalRows : 0;
    const uint32_t rows = (uint32_t)(MODE == kOwn ? min((int64_t)kLocalRows, a.rows - row0) : a.rows);
    const int64_t base = MODE == kOwn ? 0 : (int64_t)blockIdx.x * span;
    int m = (int)min((int64_t)span, a.n - base);
    uint32_t before = kNone, after = kNone;  // the neighbours' keys
    if (MODE != kSorted) {
        uint32_t* const flags = blockIdx.y == 0 && (MODE == kLocal || blockIdx.x == 0) ? a.flags
                                                                                     : nullptr;
        __shared__ uint32_t cnt[kWaves][kLocalRows + 1];
        __shared__ uint32_t scan[kWaves];
        for (int k = t; k < kWaves * (kLocalRows + 1); k += kThreads) (&cnt[0][0])[k] = 0u;
        __syncthreads();
        const int w = t >> 6, l = t & 63;
        uint32_t key[kSpan / kThreads], rank[kSpan / kThreads];
#pragma unroll
        for (int k = 0; k < kSpan / kThreads; ++k) {
            const int i = w * (span / kWaves) + k * 64 + l;
            if (k < span / kThreads) {
                key[k] = i < m ? sort_key(a, nullptr, base + i, flags) : 0u;
                if (MODE == kOwn) {
                    const int64_t own = (int64_t)key[k] - row0;
                    key[k] = own >= 0 && own < rows ? (uint32_t)own : rows;
                }
                rank[k] = wave_rank(key[k], i < m, bits, cnt[w]);
            }
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
        if (MODE == kOwn) m = (int)cnt[0][rows];  // those of other rows came last
        // rows that no id of the span names
        if (MODE == kLocal || !a.accumulate)
            for (uint32_t v = slot; v < rows; v += slots) {
                const uint32_t lo = cnt[0][v];
                if ((lo < (uint32_t)m && skey[lo] == v) || !col_on) continue;
                const float zero[VEC] = {};
                if (MODE == kLocal)
                    put_row<float, VEC>(part + ((size_t)blockIdx.x * rows + v) * a.dim + c, zero,
                                        1.0f, 0, c_lo, c_hi);
                else
                    put_row<TD, VEC>(dtable + (row0 + v) * a.dtable_stride + c, zero, 1.0f, 0, c_lo,
                                     c_hi);
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
    auto finish = [&](uint32_t key, const float* acc, int which) {
        if (key >= rows) return;
        if (MODE == kLocal || (MODE == kSorted && which < 2)) {
            const size_t row = MODE == kLocal ? (size_t)blockIdx.x * rows + key
                                              : (size_t)blockIdx.x * 2 + which;
            put_row<float, VEC>(part + row * a.dim + c, acc, 1.0f, 0, c_lo, c_hi);
        } else {
            put_row<TD, VEC>(dtable + (row0 + key) * a.dtable_stride + c, acc, a.scale,
                             a.accumulate, c_lo, c_hi);
        }
    };

    const int per = ((MODE == kOwn ? m : span) + slots - 1) / slots, lo = min(m, slot * per), hi = min(m, lo + per);
    float acc[VEC], head[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = head[j] = 0.0f;
    uint32_t cur = lo < hi ? skey[lo] : kNone;
    const uint32_t first = cur;
    bool single = true;
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
                    for (int j = 0; j < VEC; ++j) head[j] = acc[j];
                    single = false;
                } else if (col_on) {
                    finish(cur, acc, 2);
                }
                cur = k[u];
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
        }
    }
    if (lane == 0) {
        first_key[slot] = first;
        last_key[slot] = cur;
    }
    __syncthreads();
    const uint32_t prev = slot > 0 ? last_key[slot - 1] : kNone;
    uint32_t next = slot + 1 < slots ? first_key[slot + 1] : kNone;
    // Segmented inclusive scan of the slots' last runs: `cut`: the run starts in
    // this slot (or the scan has met such a one); `begin`: it holds the span's
    // first entry.
    bool cut = !single || first != prev || first == kNone;
    bool begin = slot == 0 && single;
    for (int o = lpr; o < 64; o <<= 1) {
        const bool in = (t & 63) >= o;
        const bool ucut = __shfl_up((int)cut, o, 64), ubegin = __shfl_up((int)begin, o, 64);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float u = __shfl_up(acc[j], o, 64);
            if (in && !cut) acc[j] += u;
        }
        if (in && !cut) {
            begin = ubegin;
            cut = ucut;
        }
    }
    const int w = t >> 6, in_wave = t & 63;
    if (in_wave >= 64 - lpr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) carry[w][(in_wave - (64 - lpr)) * VEC + j] = acc[j];
        if (in_wave == 63) carry_flags[w] = (cut ? 1u : 0u) | (begin ? 2u : 0u);
    }
    __syncthreads();
    // what the earlier waves bring to this one
    float in[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) in[j] = 0.0f;
    bool in_begin = false;
    for (int k = 0; k < w; ++k) {
        const bool kcut = carry_flags[k] & 1u;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            in[j] = (kcut ? 0.0f : in[j]) + carry[k][(in_wave % lpr) * VEC + j];
        in_begin = kcut ? (carry_flags[k] & 2u) != 0u : in_begin;
    }
    if (!cut) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += in[j];
        begin = in_begin;
    }
    // the previous slot's run, which this slot's first one may continue
    float before_sum[VEC];
    bool before_begin = __shfl_up((int)begin, lpr, 64);
#pragma unroll
    for (int j = 0; j < VEC; ++j) before_sum[j] = __shfl_up(acc[j], lpr, 64);
    if (in_wave < lpr) {
        before_begin = in_begin;
#pragma unroll
        for (int j = 0; j < VEC; ++j) before_sum[j] = in[j];
    }
    if (!col_on || first == kNone) return;
    if (!single) {
        const bool joins = prev == first;
        if (joins)
#pragma unroll
            for (int j = 0; j < VEC; ++j) head[j] += before_sum[j];
        const bool from_begin = slot == 0 || (joins && before_begin);
        finish(first, head, from_begin && before == first ? 0 : 2);
    }
    if (next == kNone) next = after;  // the last slot with entries
    else if (next == cur) return;
    const bool more = next == cur;
    finish(cur, acc, begin ? (before == cur || more ? 0 : 2) : (more ? 1 : 2));
}

// Rows whose run crosses spans: the sum of the spans' pieces in order; zeros for
// rows that no id names. `lpr` lanes a row, 4 columns a lane; a row of many pieces
// takes the workgroup, whose slots share the pieces out.
constexpr uint32_t kSlotPieces = 32;

template <typename TD>
__global__ __launch_bounds__(kThreads) void k_run_join(LookupGradArgs a, const uint2* runs,
                                                       int span, int lpr, const float* part) {
    __shared__ float sums[kThreads][4];
    __shared__ uint32_t many[kThreads], n_many;
    TD* dtable = static_cast<TD*>(a.dtable);
    const int slots = kThreads / lpr, slot = threadIdx.x / lpr, lane = threadIdx.x % lpr;
    auto pieces_of = [&](uint2 run) {
        return run.x == run.y ? 0u : (run.y - 1u) / (uint32_t)span - run.x / (uint32_t)span + 1u;
    };
    // pieces k, k + by, .. of columns c.. c + 3
    auto add = [&](uint2 run, uint32_t n, uint32_t k, uint32_t by, int c, float* acc) {
        const uint32_t s0 = run.x / (uint32_t)span;
        const uint32_t from = run.x % (uint32_t)span != 0u ? 1u : 0u;  // the first piece's place
        const int nv = min(4, a.dim - c);
        for (; k < n; k += by * 4) {
            float v[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t q = k + u * by;
                const float* p = part + ((size_t)(s0 + q) * 2 + (q == 0 ? from : 0)) * a.dim + c;
                if (q < n && nv == 4) {
                    load_any<4>(p, v[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] = q < n && j < nv ? p[j] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += v[u][j];
        }
    };
    for (int64_t v0 = (int64_t)blockIdx.x * slots; v0 < a.rows; v0 += (int64_t)gridDim.x * slots) {
        if (threadIdx.x == 0) n_many = 0u;
        __syncthreads();
        const int64_t v = v0 + slot;
        if (v < a.rows) {
            const uint2 run = runs[v];
            const uint32_t n = pieces_of(run);
            if (n > kSlotPieces) {
                if (lane == 0) many[atomicAdd(&n_many, 1u)] = (uint32_t)slot;
            } else if (n > 1 || (n == 0 && !a.accumulate)) {
                for (int c = lane * 4; c < a.dim; c += lpr * 4) {
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    add(run, n, 0, 1, c, acc);
                    put_row<TD, 4>(dtable + v * a.dtable_stride + c, acc, a.scale, a.accumulate,
                                   0, min(4, a.dim - c));
                }
            }
        }
        __syncthreads();
        for (uint32_t k = 0; k < n_many; ++k) {
            const int64_t row = v0 + many[k];
            const uint2 run = runs[row];
            const uint32_t n = pieces_of(run);
            for (int c0 = 0; c0 < a.dim; c0 += lpr * 4) {
                const int c = c0 + lane * 4;
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (c < a.dim) add(run, n, slot, slots, c, acc);
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[threadIdx.x][j] = acc[j];
                __syncthreads();
                if (slot == 0 && c < a.dim) {
                    for (int q = 1; q < slots; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] += sums[q * lpr + lane][j];
                    put_row<TD, 4>(dtable + row * a.dtable_stride + c, acc, a.scale, a.accumulate,
                                   0, min(4, a.dim - c));
                }
            }
        }
        __syncthreads();
    }
}

// kLocal's join: a workgroup per row and 16 columns, 16 slots over the spans.
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

// Consecutive ids of a kLocal span: as many as leave two workgroups a compute unit.
int local_span(int64_t n) {
    int s = 512;
    while (s < kSpan && n / (2 * s) >= 512) s *= 2;
    return s;
}

// Few enough ids that every workgroup may look through them all, and that one
// workgroup may sum them all, should they be one row's (with more than a few where
// the table gives kLocal no work to share: 4096 x 32 into one row took 41 us so, 13
// by kLocal; 1000 x 32 into 5000 rows 11, and 20 sorted). Up to 4096 ids are a trade:
// into 5000 rows of 32 they took 28 us (with the call) and sorted 30, into 100000 rows
// 45 and 67; were all of them one row's 57, and sorted 29.
bool is_own(int64_t n, int64_t rows, int dim) {
    return n > 0 && n <= (rows > kLocalRows ? kSpan : 1024) && n * dim <= (1 << 17) &&
           rows <= (1 << 20);
}

bool is_local(int64_t n, int64_t rows) { return rows <= kLocalRows && n > 0; }

// A list for one workgroup, which also clears the rows' runs: 4000 x 64 into 3000 rows
// 24 us, by the long sort 33.
bool is_short(int64_t n, int64_t rows) {
    return n <= kShort && rows <= 65536 && !is_local(n, rows);
}

// Entries of a span of the sorted list: at most 4096 spans while spans can grow,
// so that one row's pieces stay few.
int span_of(int64_t n) {
    int s = 256;
    while (s < 1024 && n / s > 4096) s *= 2;
    return s;
}

// Keys of a sort block's thread: fewer where that fills the chip (20000000 ids: 916 us
// of gradient with 16, 985 with 4; 3000000: 236 and 227; 1000000: 88 with 4, 92 with 8).
int sort_items(int64_t n) { return n <= (1 << 22) ? 4 : 16; }

struct GradWs {
    uint2 *pairs[2], *runs;
    uint32_t *counts, *totals;
    float* part;
    size_t bytes;
    GradWs(void* base, int64_t n, int64_t rows, int dim) {
        Carve c(base);
        if (is_own(n, rows, dim)) {
            totals = c.take<uint32_t>(1);  // not used: every size asks for a workspace
        } else if (is_local(n, rows)) {
            const int span = local_span(n);
            part = c.take<float>((size_t)((n + span - 1) / span) * rows * dim);
        } else {
            const int64_t tile = (int64_t)kThreads * sort_items(n);
            for (int k = 0; k < 2; ++k) pairs[k] = c.take<uint2>((size_t)n);
            counts = c.take<uint32_t>((size_t)((n + tile - 1) / tile) * 256);
            totals = c.take<uint32_t>(256);
            runs = c.take<uint2>((size_t)rows);
            const int span = span_of(n);  // or longer, with fewer pieces
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
    if (is_own(a.n, a.rows, a.dim)) {
        const int span = (int)((a.n + kThreads - 1) / kThreads) * kThreads;
        k_run_sums<TI, TD, VEC, kOwn>
            <<<dim3((unsigned)((a.rows + kLocalRows - 1) / kLocalRows), cols), kThreads, span * 8, st>>>(
                a, nullptr, span, lpr, key_bits(kLocalRows), nullptr, nullptr);
        return hipGetLastError();
    }
    if (is_local(a.n, a.rows)) {
        const int span = local_span(a.n), spans = (int)((a.n + span - 1) / span);
        k_run_sums<TI, TD, VEC, kLocal><<<dim3((unsigned)spans, cols), kThreads, span * 8, st>>>(
            a, nullptr, span, lpr, key_bits(a.rows), w.part, nullptr);
        GS_LAUNCHED();
        k_local_join<TD><<<dim3((unsigned)a.rows, (unsigned)((a.dim + 15) / 16)), kThreads, 0, st>>>(
            a, spans, w.part);
        return hipGetLastError();
    }
    // a slot's stretch holds the 8 rows that it loads at a time
    const int span = std::max(span_of(a.n), std::min(kSpan, kThreads / lpr * 8));
    if (a.n > 0)
        k_run_sums<TI, TD, VEC, kSorted>
            <<<dim3((unsigned)((a.n + span - 1) / span), cols), kThreads, span * 8, st>>>(
                a, pairs, span, lpr, 0, w.part, w.runs);
    GS_LAUNCHED();
    int join_lpr = 1;
    while (join_lpr < 64 && join_lpr * 4 < a.dim) join_lpr *= 2;
    const int64_t joins = (a.rows + kThreads / join_lpr - 1) / (kThreads / join_lpr);
    k_run_join<TD><<<(unsigned)(joins < 65536 ? joins : 65536), kThreads, 0, st>>>(
        a, w.runs, span, join_lpr, w.part);
    return hipGetLastError();
}

__global__ __launch_bounds__(kThreads) void k_run_clear(uint2* runs, int64_t rows) {
    const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (v < rows) runs[v] = make_uint2(0u, 0u);
}

template <int ITEMS>
hipError_t sort_ids(const LookupGradArgs& a, const GradWs& w, const uint2** sorted,
                    hipStream_t st) {
    const int bits = key_bits(a.rows), passes = (bits + 7) / 8;
    const unsigned blocks = (unsigned)((a.n + kThreads * ITEMS - 1) / (kThreads * ITEMS));
    const uint2* pairs = nullptr;
    // The runs are cleared in passing by the first count, whose blocks are the ids'; where
    // that leaves a thread more than 256 rows, by the whole chip: 5000 ids into 2^27 rows
    // took 3.31 ms, so 0.69 (into 100000 rows 62 us in passing, 71 with the launch).
    uint2* in_passing = w.runs;
    if (a.rows > (int64_t)blocks * kThreads * 256) {
        k_run_clear<<<(unsigned)((a.rows + kThreads - 1) / kThreads), kThreads, 0, st>>>(w.runs,
                                                                                      a.rows);
        GS_LAUNCHED();
        in_passing = nullptr;
    }
    for (int p = 0, done = 0; p < passes; ++p) {
        const int b = (bits - done + passes - p - 1) / (passes - p);
        k_sort_count<ITEMS><<<blocks, kThreads, 0, st>>>(a, pairs, done, b, w.counts,
                                                         p == 0 ? in_passing : nullptr);
        GS_LAUNCHED();
        k_sort_scan<<<1u << b, kThreads, 0, st>>>(w.counts, (int)blocks, w.totals);
        GS_LAUNCHED();
        k_sort_scatter<ITEMS><<<blocks, kThreads, 0, st>>>(a, pairs, done, b, w.counts, w.totals,
                                                           w.pairs[p & 1]);
        GS_LAUNCHED();
        pairs = w.pairs[p & 1];
        done += b;
    }
    *sorted = pairs;
    return hipSuccess;
}

// Of a table without rows nothing is summed, but every id is past it.
__global__ __launch_bounds__(kThreads) void k_report_ids(LookupGradArgs a) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < a.n;
         i += (int64_t)gridDim.x * kThreads)
        load_id(a.ids, a.ids64, i, a.rows, a.flags);
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
    if (a.rows == 0) {
        if (a.n == 0 || a.flags == nullptr) return hipSuccess;
        k_report_ids<<<blocks_of(a.n, kThreads), kThreads, 0, st>>>(a);
        return hipGetLastError();
    }
    const GradWs w(a.ws, a.n, a.rows, a.dim);
    const uint2* pairs = nullptr;
    hipError_t e = hipSuccess;
    if (a.n == 0)
        k_run_clear<<<(unsigned)((a.rows + kThreads - 1) / kThreads), kThreads, 0, st>>>(w.runs,
                                                                                      a.rows);
    else if (is_own(a.n, a.rows, a.dim)) {
        // the one launch of grad_typed
    } else if (is_short(a.n, a.rows)) {
        k_sort_short<<<1, kShortThreads, 0, st>>>(a, key_bits(a.rows), w.pairs[0], w.runs);
        pairs = w.pairs[0];
    } else if (!is_local(a.n, a.rows))
        e = sort_items(a.n) == 4 ? sort_ids<4>(a, w, &pairs, st) : sort_ids<16>(a, w, &pairs, st);
    if (e != hipSuccess) return e;
    GS_LAUNCHED();
    if (a.dout_dtype == 0)
        return a.dtable_dtype == 0 ? grad_typed<float, float>(a, w, pairs, st)
                                   : grad_typed<float, bf16>(a, w, pairs, st);
    return a.dtable_dtype == 0 ? grad_typed<bf16, float>(a, w, pairs, st)
                               : grad_typed<bf16, bf16>(a, w, pairs, st);
}

}  // namespace gs
