// field_lookup.hip - rows of a feature table by id, and the table's gradient.
//
//   out[i]    = scale * table[ids[i]]            (zeros for an id outside [0, rows))
//   dtable[v] = scale * sum over ids[i] = v of dout[i]
//
// The gradient is by sorted ids: a stable radix sort of (id, position), then
// each id's run of rows is summed in position order, so the result does not
// depend on timing. Sums are held in fp32.
#include "field.h"

#include "field_device.h"

namespace gs {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- lookup
// A workgroup takes R consecutive ids, stages their rows' numbers in LDS and
// writes the R * dim values in memory order, VEC at a time.
constexpr int kLookupRows = 1024;  // most ids of a workgroup

template <typename TT, typename TO, int VEC, bool VLOAD, bool VSTORE>
__global__ __launch_bounds__(kThreads) void k_lookup(LookupArgs a, int R) {
    __shared__ int32_t row_of[kLookupRows];
    const TT* table = static_cast<const TT*>(a.table);
    TO* out = static_cast<TO*>(a.out);
    const uint32_t dim = (uint32_t)a.dim;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.n; r0 += (int64_t)gridDim.x * R) {
        const int nr = (int)min((int64_t)R, a.n - r0);
        __syncthreads();
        for (int i = threadIdx.x; i < nr; i += kThreads)
            row_of[i] = load_id(a.ids, a.ids64, r0 + i, a.rows, a.flags);
        __syncthreads();
        const uint32_t total = (uint32_t)nr * dim;
        for (uint32_t l = threadIdx.x * VEC; l < total; l += kThreads * VEC) {
            uint32_t r = l / dim, c = l - r * dim;
            float v[VEC];
            if (VLOAD) {
                const int32_t t = row_of[r];
                if (t >= 0) {
                    load_vec<VEC>(table + t * a.table_stride + c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
                }
            } else {
                uint32_t rr = r, cc = c;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int32_t t = l + j < total ? row_of[rr] : -1;
                    v[j] = t >= 0 ? to_float(table[t * a.table_stride + cc]) : 0.0f;
                    if (++cc == dim) {
                        cc = 0;
                        ++rr;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= a.scale;
            if (VSTORE && l + VEC <= total) {
                if (VLOAD)
                    store_vec<VEC>(out + (r0 + r) * a.out_stride + c, v);
                else  // rows without gaps: out_stride == dim
                    store_vec<VEC>(out + r0 * (int64_t)dim + l, v);
            } else {
                uint32_t rr = r, cc = c;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (l + j < total) out[(r0 + rr) * a.out_stride + cc] = from_float<TO>(v[j]);
                    if (++cc == dim) {
                        cc = 0;
                        ++rr;
                    }
                }
            }
        }
    }
}

template <typename TT, typename TO>
hipError_t lookup_typed(const LookupArgs& a, hipStream_t st) {
    constexpr int VEC = (sizeof(TT) == 2 && sizeof(TO) == 2) ? 8 : 4;
    const int64_t want = (int64_t)kThreads * VEC * 4;
    int64_t R = (want + a.dim - 1) / a.dim;
    R = ((R + 7) / 8) * 8;
    if (R > kLookupRows) R = kLookupRows;
    const int64_t blocks = (a.n + R - 1) / R;
    const dim3 grid((unsigned)(blocks < (1 << 30) ? blocks : (1 << 30)));
    const bool vload = a.dim % VEC == 0 && aligned_rows<TT>(a.table, a.table_stride, VEC) &&
                       aligned_rows<TO>(a.out, a.out_stride, VEC);
    const bool flat = a.out_stride == a.dim && aligned_rows<TO>(a.out, 0, VEC);
    if (vload)
        k_lookup<TT, TO, VEC, true, true><<<grid, kThreads, 0, st>>>(a, (int)R);
    else if (flat)
        k_lookup<TT, TO, VEC, false, true><<<grid, kThreads, 0, st>>>(a, (int)R);
    else
        k_lookup<TT, TO, VEC, false, false><<<grid, kThreads, 0, st>>>(a, (int)R);
    return hipGetLastError();
}

// ---------------------------------------------------------------- sort
// Stable LSD radix sort of (id, position), 8 bits a pass at most: per block the
// digits' counts, per digit the blocks' offsets, then the scatter. Ids outside
// the table get the key `rows` and end last.
constexpr int kSortItems = 16;                      // keys of a thread
constexpr int kSortTile = kThreads * kSortItems;    // keys of a workgroup

__global__ __launch_bounds__(kThreads) void k_sort_count(LookupGradArgs a, const uint32_t* keys,
                                                         uint32_t* first, int shift, int bits,
                                                         uint32_t* counts) {
    __shared__ uint32_t hist[256];
    hist[threadIdx.x] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile;
    const uint32_t mask = (1u << bits) - 1u;
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * kThreads + threadIdx.x;
        if (i < a.n) {
            uint32_t key;
            if (first != nullptr) {  // the first pass reads the caller's ids
                const int32_t t = load_id(a.ids, a.ids64, i, a.rows, a.flags);
                key = t >= 0 ? (uint32_t)t : (uint32_t)a.rows;
                first[i] = key;
            } else {
                key = keys[i];
            }
            atomicAdd(&hist[(key >> shift) & mask], 1u);
        }
    }
    __syncthreads();
    if (threadIdx.x < (1u << bits))
        counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x] = hist[threadIdx.x];
}

// One workgroup per digit: exclusive prefix of its blocks' counts, and its total.
__global__ __launch_bounds__(kThreads) void k_sort_scan(uint32_t* counts, int blocks,
                                                        uint32_t* totals) {
    __shared__ uint32_t part[kThreads];
    uint32_t* row = counts + (size_t)blockIdx.x * blocks;
    const int per = (blocks + kThreads - 1) / kThreads;
    const int lo = min((int)threadIdx.x * per, blocks), hi = min(lo + per, blocks);
    uint32_t sum = 0;
    for (int i = lo; i < hi; ++i) sum += row[i];
    uint32_t total;
    uint32_t at = block_excl_scan<kThreads>(sum, part, &total);
    for (int i = lo; i < hi; ++i) {
        const uint32_t c = row[i];
        row[i] = at;
        at += c;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = total;
}

// A wave ranks its keys in order, 64 at a time: the lanes of equal digit are
// found with one ballot per digit bit, and the wave's count of each digit so far
// is kept in LDS.
__global__ __launch_bounds__(kThreads) void k_sort_scatter(const uint32_t* keys,
                                                           const uint32_t* vals, int64_t n,
                                                           int shift, int bits,
                                                           const uint32_t* counts,
                                                           const uint32_t* totals, uint32_t* keys_o,
                                                           uint32_t* vals_o) {
    constexpr int kWaves = kThreads / 64;
    __shared__ uint32_t cnt[kWaves][256];
    __shared__ uint32_t part[kThreads];
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    const int digits = 1 << bits;
    const uint32_t mask = digits - 1u;
    for (int k = 0; k < kWaves; ++k) cnt[k][t] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile + (int64_t)w * 64 * kSortItems;
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * 64 + lane;
        const bool on = i < n;
        key[k] = on ? keys[i] : 0u;
        const uint32_t d = (key[k] >> shift) & mask;
        uint64_t same = __ballot(on);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((d >> b) & 1u);
            same &= ((d >> b) & 1u) ? m : ~m;
        }
        const uint32_t before = __popcll(same & ((1ull << lane) - 1ull));
        uint32_t seen = 0;
        volatile uint32_t* mine = &cnt[w][d];  // other lanes of the wave write it
        if (on) seen = *mine;
        rank[k] = seen + before;
        __builtin_amdgcn_wave_barrier();
        if (on && before == 0) *mine = seen + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // digit starts: all smaller digits' totals, this block's offset, earlier waves
    const uint32_t mine = t < digits ? totals[t] : 0u;
    uint32_t all;
    uint32_t at = block_excl_scan<kThreads>(mine, part, &all);
    if (t < digits) {
        at += counts[(size_t)t * gridDim.x + blockIdx.x];
        for (int k = 0; k < kWaves; ++k) {
            const uint32_t c = cnt[k][t];
            cnt[k][t] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * 64 + lane;
        if (i < n) {
            const uint32_t to = cnt[w][(key[k] >> shift) & mask] + rank[k];
            keys_o[to] = key[k];
            vals_o[to] = vals != nullptr ? vals[i] : (uint32_t)i;
        }
    }
}

// Run of every id in the sorted keys; [0, 0) for ids without one.
__global__ __launch_bounds__(kThreads) void k_run_clear(uint2* runs, int64_t rows) {
    const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (v < rows) runs[v] = make_uint2(0u, 0u);
}
__global__ __launch_bounds__(kThreads) void k_run_bounds(const uint32_t* keys, int64_t n,
                                                         int64_t rows, uint2* runs) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const uint32_t k = keys[i];
    if (k >= (uint32_t)rows) return;
    if (i == 0 || keys[i - 1] != k) runs[k].x = (uint32_t)i;
    if (i == n - 1 || keys[i + 1] != k) runs[k].y = (uint32_t)(i + 1);
}

// ---------------------------------------------------------------- run sums
// The sorted list is cut into stretches of S entries; a slot of LPR lanes sums
// one, VEC columns a lane. A run inside one stretch is written at once; the
// pieces of a longer one go to `part` (two rows a stretch: the run that holds
// its first entry, and the last run) and k_run_join adds them in order.
template <typename TD, int VEC>
__device__ __forceinline__ void put_row(TD* out, const float* acc, float scale, int accumulate,
                                        int nvalid) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (j < nvalid) {
            float s = acc[j] * scale;
            if (accumulate) s += to_float(out[j]);
            out[j] = from_float<TD>(s);
        }
}

template <typename TI, typename TD, int VEC>
__global__ __launch_bounds__(kThreads) void k_run_sums(LookupGradArgs a, const uint32_t* keys,
                                                       const uint32_t* pos, int S, int lpr,
                                                       float* part) {
    const TI* dout = static_cast<const TI*>(a.dout);
    TD* dtable = static_cast<TD*>(a.dtable);
    const int slots = kThreads / lpr;
    const int lane = threadIdx.x % lpr;
    const int64_t s = (int64_t)blockIdx.x * slots + threadIdx.x / lpr;
    const int c = (blockIdx.y * lpr + lane) * VEC;
    const int64_t lo = s * S;
    if (lo >= a.n || c >= a.dim) return;
    const int64_t hi = min(lo + S, a.n);
    const int nv = min(VEC, a.dim - c);
    const uint32_t rows = (uint32_t)a.rows;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    uint32_t cur = keys[lo];
    int64_t from = lo;
    auto flush = [&](int64_t end) {
        if (cur >= rows) return;
        const bool starts = from > lo || lo == 0 || keys[lo - 1] != cur;
        const bool ends = end < hi || hi == a.n || keys[hi] != cur;
        if (starts && ends) {
            put_row<TD, VEC>(dtable + (int64_t)cur * a.dtable_stride + c, acc, a.scale,
                             a.accumulate, nv);
        } else {
            float* p = part + ((size_t)s * 2 + (from == lo ? 0 : 1)) * a.dim + c;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < nv) p[j] = acc[j];
        }
    };
    for (int64_t i = lo; i < hi; ++i) {
        const uint32_t k = keys[i];
        if (k != cur) {
            flush(i);
            cur = k;
            from = i;
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        }
        if (k >= rows) break;
        const TI* src = dout + (int64_t)pos[i] * a.dout_stride + c;
        float v[VEC];
        if (nv == VEC && VEC > 1) {
            load_vec<VEC>(src, v);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = j < nv ? to_float(src[j]) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[j];
    }
    flush(hi);
}

// One workgroup per table row: zeros for a row no id names, the sum of the
// pieces for a run of several stretches (each slot of lanes adds every slots-th
// piece, then the slots' sums are added in order).
template <typename TD>
__global__ __launch_bounds__(kThreads) void k_run_join(LookupGradArgs a, const uint2* runs, int S,
                                                       const float* part) {
    __shared__ float sums[kThreads];
    TD* dtable = static_cast<TD*>(a.dtable);
    for (int64_t v = blockIdx.x; v < a.rows; v += gridDim.x) {
        const uint2 run = runs[v];
        TD* out = dtable + v * a.dtable_stride;
        if (run.x == run.y) {
            if (!a.accumulate)
                for (int c = threadIdx.x; c < a.dim; c += kThreads) out[c] = from_float<TD>(0.0f);
            continue;
        }
        const uint32_t s0 = run.x / (uint32_t)S, s1 = (run.y - 1u) / (uint32_t)S;
        if (s0 == s1) continue;
        const int w = min(a.dim, kThreads), slots = kThreads / w;
        const int slot = threadIdx.x / w, lane = threadIdx.x % w;
        for (int c0 = 0; c0 < a.dim; c0 += w) {
            const int c = c0 + lane;
            float acc = 0.0f;
            if (slot < slots && c < a.dim)
                for (uint32_t s = s0 + slot; s <= s1; s += slots) {
                    const int which = s == s0 && run.x % (uint32_t)S != 0u ? 1 : 0;
                    acc += part[((size_t)s * 2 + which) * a.dim + c];
                }
            __syncthreads();
            sums[threadIdx.x] = acc;
            __syncthreads();
            if (slot == 0 && c < a.dim) {
                for (int k = 1; k < slots; ++k) acc += sums[k * w + lane];
                put_row<TD, 1>(out + c, &acc, a.scale, a.accumulate, 1);
            }
        }
    }
}

int stretch_of(int64_t n) {
    int S = 16;
    while (S < 1024 && n / S > 16384) S *= 2;
    return S;
}

int key_bits(int64_t rows) {  // keys 0 .. rows
    int b = 1;
    while (((int64_t)1 << b) <= rows) ++b;
    return b;
}

struct GradWs {
    uint32_t *key[2], *val[2], *counts, *totals;
    uint2* runs;
    float* part;
    size_t bytes;
    GradWs(void* base, int64_t n, int64_t rows, int dim) {
        Carve c(base);
        const size_t blocks = (size_t)((n + kSortTile - 1) / kSortTile);
        for (int k = 0; k < 2; ++k) {
            key[k] = c.take<uint32_t>((size_t)n);
            val[k] = c.take<uint32_t>((size_t)n);
        }
        counts = c.take<uint32_t>(blocks * 256);
        totals = c.take<uint32_t>(256);
        runs = c.take<uint2>((size_t)rows);
        const int S = stretch_of(n);
        part = c.take<float>((size_t)((n + S - 1) / S) * 2 * dim);
        bytes = c.bytes();
    }
};

template <typename TI, typename TD>
hipError_t grad_typed(const LookupGradArgs& a, const GradWs& w, const uint32_t* keys,
                      const uint32_t* vals, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(TI);
    const int S = stretch_of(a.n);
    const bool vec = a.dim % VEC == 0 && aligned_rows<TI>(a.dout, a.dout_stride, VEC);
    const int cols = vec ? a.dim / VEC : a.dim;
    int lpr = 1;
    while (lpr < 64 && lpr < cols) lpr *= 2;
    const int64_t stretches = (a.n + S - 1) / S;
    const int slots = kThreads / lpr;
    if (stretches > 0) {
        const dim3 grid((unsigned)((stretches + slots - 1) / slots),
                        (unsigned)((cols + lpr - 1) / lpr));
        if (vec)
            k_run_sums<TI, TD, VEC><<<grid, kThreads, 0, st>>>(a, keys, vals, S, lpr, w.part);
        else
            k_run_sums<TI, TD, 1><<<grid, kThreads, 0, st>>>(a, keys, vals, S, lpr, w.part);
    }
    const unsigned joins = (unsigned)(a.rows < 65536 ? a.rows : 65536);
    k_run_join<TD><<<joins, kThreads, 0, st>>>(a, w.runs, S, w.part);
    return hipGetLastError();
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
    GradWs w(a.ws, a.n, a.rows, a.dim);
    const int bits = key_bits(a.rows), passes = (bits + 7) / 8;
    const unsigned blocks = (unsigned)((a.n + kSortTile - 1) / kSortTile);
    const uint32_t *keys = w.key[0], *vals = nullptr;
    int cur = 0, done = 0;
    for (int p = 0; p < passes && a.n > 0; ++p) {
        const int b = (bits - done + passes - p - 1) / (passes - p);
        k_sort_count<<<blocks, kThreads, 0, st>>>(a, keys, p == 0 ? w.key[0] : nullptr, done, b,
                                                  w.counts);
        k_sort_scan<<<1u << b, kThreads, 0, st>>>(w.counts, (int)blocks, w.totals);
        k_sort_scatter<<<blocks, kThreads, 0, st>>>(keys, vals, a.n, done, b, w.counts, w.totals,
                                                    w.key[cur ^ 1], w.val[cur ^ 1]);
        cur ^= 1;
        keys = w.key[cur];
        vals = w.val[cur];
        done += b;
    }
    k_run_clear<<<(unsigned)((a.rows + kThreads - 1) / kThreads), kThreads, 0, st>>>(w.runs, a.rows);
    if (a.n > 0)
        k_run_bounds<<<(unsigned)((a.n + kThreads - 1) / kThreads), kThreads, 0, st>>>(
            keys, a.n, a.rows, w.runs);
    if (a.dout_dtype == 0)
        return a.dtable_dtype == 0 ? grad_typed<float, float>(a, w, keys, vals, st)
                                   : grad_typed<float, bf16>(a, w, keys, vals, st);
    return a.dtable_dtype == 0 ? grad_typed<bf16, float>(a, w, keys, vals, st)
                               : grad_typed<bf16, bf16>(a, w, keys, vals, st);
}

}  // namespace gs
