// lookup.cu -- rows of a descriptor table for a list of hits, with scaling, and the table's gradient.
//
//   out[i]    = s w_i E[idx_i]                    (0 where idx_i names no row)
//   dE[p]     = s sum_{i: idx_i = p} w_i dout_i   (ascending i)
//   dw_i      = s <dout_i, E[idx_i]>
//
// The forward is bound by memory: it reads the index and each distinct row once from HBM (further hits of a row
// mostly come from L2) and writes n rows.  The gradient sorts the entries by row first (a stable radix sort of
// (row, i) pairs, so that the order of every sum is fixed and no float atomics are needed), after which each
// row's entries lie together and a group of lanes adds them in registers and writes the row once.
#include <algorithm>

#include "ops.cuh"

namespace flare {

constexpr int LK_THREADS = 256, LK_ITEMS = 4;

struct LookupArgs {
    const void *table;
    const unsigned char *scales;
    const void *index;
    const float *weight;
    void *out;
    long long rows, table_stride, scale_stride, out_stride, first;  // first: first entry of this launch
    unsigned items;  // vectors of this launch
    FastDiv vpr;     // vectors per row
    float scale;
};

template <class I>
__device__ __forceinline__ long long row_of(const void *index, long long i, long long rows) {
    const long long p = (long long)__ldg(static_cast<const I *>(index) + i);
    return p >= 0 && p < rows ? p : -1;
}

// VE consecutive values of one row of a 4-bit table, columns v * VE ...
template <int VE>
__device__ __forceinline__ void micro_load(const LookupArgs &a, long long p, unsigned v, float *f) {
    const unsigned char *codes = static_cast<const unsigned char *>(a.table) + p * a.table_stride;
    const unsigned col = v * VE;
    const float s = micro_scale(__ldg(a.scales + p * a.scale_stride + (col >> 5)));
    if constexpr (VE == 1) {
        const float2 t = micro_pair(__ldg(codes + (v >> 1)));
        f[0] = (v & 1 ? t.y : t.x) * s;
    } else {
        unsigned bits;
        if (VE == 8) bits = __ldg(reinterpret_cast<const unsigned *>(codes) + v);
        else if (VE == 4) bits = __ldg(reinterpret_cast<const unsigned short *>(codes) + v);
        else bits = __ldg(codes + v);
#pragma unroll
        for (int e = 0; e < VE / 2; ++e) {
            const float2 t = micro_pair((bits >> (8 * e)) & 255u);
            f[2 * e] = t.x * s;
            f[2 * e + 1] = t.y * s;
        }
    }
}

// One vector of VE elements per item, LK_ITEMS items in flight per thread so that the index loads and then the
// row loads of several entries overlap.  T = void: a 4-bit table.
template <class T, class O, class I, int VE>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(const LookupArgs a) {
    const unsigned base = blockIdx.x * (LK_THREADS * LK_ITEMS) + threadIdx.x;
    long long p[LK_ITEMS];
    unsigned row[LK_ITEMS], v[LK_ITEMS];
    float f[LK_ITEMS][VE];
#pragma unroll
    for (int k = 0; k < LK_ITEMS; ++k) {
        const unsigned it = base + k * LK_THREADS;
        p[k] = -1;
        row[k] = a.vpr.div(it);
        v[k] = it - row[k] * a.vpr.d;
        if (it < a.items) p[k] = row_of<I>(a.index, a.first + row[k], a.rows);
    }
#pragma unroll
    for (int k = 0; k < LK_ITEMS; ++k) {
        if (p[k] < 0) {
#pragma unroll
            for (int e = 0; e < VE; ++e) f[k][e] = 0.0f;
            continue;
        }
        const float s = a.weight ? a.scale * __ldg(a.weight + a.first + row[k]) : a.scale;
        if constexpr (std::is_void_v<T>) {
            micro_load<VE>(a, p[k], v[k], f[k]);
        } else {
            Vec<T, VE> t;
            t.load(static_cast<const T *>(a.table) + p[k] * a.table_stride + (long long)v[k] * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[k][e] = t.get(e);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) f[k][e] *= s;
    }
#pragma unroll
    for (int k = 0; k < LK_ITEMS; ++k) {
        if (base + k * LK_THREADS >= a.items) break;
        Vec<O, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.set(e, f[k][e]);
        o.store_stream(static_cast<O *>(a.out) + (a.first + row[k]) * a.out_stride + (long long)v[k] * VE);
    }
}

template <class T, class O, class I>
void launch_lookup(const LookupArgs &a, int ve, cudaStream_t st) {
    const unsigned blocks = (a.items + LK_THREADS * LK_ITEMS - 1) / (LK_THREADS * LK_ITEMS);
    switch (ve) {
        case 8: lookup_kernel<T, O, I, 8><<<blocks, LK_THREADS, 0, st>>>(a); break;
        case 4: lookup_kernel<T, O, I, 4><<<blocks, LK_THREADS, 0, st>>>(a); break;
        case 2: lookup_kernel<T, O, I, 2><<<blocks, LK_THREADS, 0, st>>>(a); break;
        default: lookup_kernel<T, O, I, 1><<<blocks, LK_THREADS, 0, st>>>(a); break;
    }
}

int run_lookup(const flare_lookup_args *in, cudaStream_t st) {
    LookupArgs a{};
    a.table = in->table;
    a.scales = in->scales;
    a.index = in->index;
    a.weight = in->weight;
    a.out = in->out;
    a.rows = in->rows;
    a.out_stride = in->out_stride;
    a.scale = in->scale;
    const bool micro = in->table_type == FLARE_MICRO;
    const int blocks32 = (in->width + 31) / 32;
    a.table_stride = micro ? 16ll * blocks32 : in->table_stride;
    a.scale_stride = 4ll * ((blocks32 + 3) / 4);
    int ve = 8;
    while (ve > 1 && !(in->width % ve == 0 && fits_vec(in->out, in->out_stride, type_size(in->out_type), ve) &&
                       (micro || fits_vec(in->table, in->table_stride, type_size(in->table_type), ve))))
        ve >>= 1;
    const unsigned vpr = (unsigned)(in->width / ve);
    a.vpr = FastDiv(vpr);
    // item numbers stay below 2^31, so that the quotient by vpr is one multiplication
    const long long per_launch = std::max<long long>(1, (1ll << 30) / vpr);
    for (a.first = 0; a.first < in->n; a.first += per_launch) {
        a.items = (unsigned)(std::min(per_launch, in->n - a.first) * vpr);
        with_type(in->out_type, [&](auto o) {
            using O = typename decltype(o)::type;
            auto go = [&](auto idx) {
                using I = typename decltype(idx)::type;
                if (micro) launch_lookup<void, O, I>(a, ve, st);
                else
                    with_type(in->table_type, [&](auto t) {
                        launch_lookup<typename decltype(t)::type, O, I>(a, ve, st);
                        return 0;
                    });
            };
            if (in->index_type == FLARE_I64) go(TypeTag<long long>{});
            else go(TypeTag<int>{});
            return 0;
        });
        OPS_LAUNCHED("flare_lookup");
    }
    return FLARE_OK;
}

// ------------------------------------------------------------------------------------------------
// Stable radix sort of the entries by row; entries that name no row get key `rows` and end behind all others.
// Per digit of up to 11 bits: count per tile, scan over tiles, scatter.  A tile is 4096 consecutive entries of one block;
// warp w ranks entries [512 w, 512 w + 512) of it 32 at a time, so ranks follow the entries' order.  Lanes with equal
// digits find one another by a ballot per bit (match.any took three times the whole kernel's time).  Up to one tile of
// entries is sorted by one block in shared memory.
// ------------------------------------------------------------------------------------------------
constexpr int RS_THREADS = 256, RS_WARPS = RS_THREADS / 32, RS_ROUNDS = 16, RS_TILE = RS_THREADS * RS_ROUNDS;
constexpr int RS_MAX_BITS = 11, RS_BINS = 1 << RS_MAX_BITS, RS_SMALL_BITS = 8;

struct SortArgs {
    const void *index;              // first pass: keys come from the index, values are the entry numbers
    const uint2 *in;                // (key, entry)
    uint2 *out;
    unsigned *key_out, *val_out;    // last pass
    unsigned *hist;                 // digit-major (bins, tiles)
    unsigned *total;                // per digit
    float *dweight;                 // 0 for entries without a row, or NULL
    long long rows;
    unsigned n, tiles;
    int shift, bits, key_bits, index_type, first, last;
};

__device__ __forceinline__ unsigned index_key(const SortArgs &a, unsigned i) {
    const long long p = a.index_type == FLARE_I64 ? row_of<long long>(a.index, i, a.rows) : row_of<int>(a.index, i, a.rows);
    return p < 0 ? (unsigned)a.rows : (unsigned)p;
}
__device__ __forceinline__ uint2 sort_entry(const SortArgs &a, unsigned i) {
    return a.first ? make_uint2(index_key(a, i), i) : a.in[i];
}

// lanes of the warp with the same `bits`-bit digit (and the same `in`)
__device__ __forceinline__ unsigned lanes_with(unsigned digit, int bits, bool in) {
    const unsigned some = __ballot_sync(0xffffffffu, in);
    unsigned same = in ? some : ~some;
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1u;
        const unsigned ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
    }
    return same;
}

__global__ void __launch_bounds__(RS_THREADS) sort_count_kernel(const SortArgs a) {
    __shared__ unsigned h[RS_BINS];
    const unsigned bins = 1u << a.bits, mask = bins - 1u;
    for (unsigned b = threadIdx.x; b < bins; b += RS_THREADS) h[b] = 0;
    __syncthreads();
    const unsigned base = blockIdx.x * RS_TILE;
#pragma unroll 8
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const unsigned i = base + r * RS_THREADS + threadIdx.x;
        if (i >= a.n) continue;
        const unsigned key = a.first ? index_key(a, i) : __ldg(&a.in[i].x);
        atomicAdd(&h[(key >> a.shift) & mask], 1u);
        if (a.first && a.dweight && key == (unsigned)a.rows) a.dweight[i] = 0.0f;
    }
    __syncthreads();
    for (unsigned b = threadIdx.x; b < bins; b += RS_THREADS) a.hist[(size_t)b * a.tiles + blockIdx.x] = h[b];
}

// exclusive sum over the block, `total` gets the sum of all
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned *warp_sums, unsigned *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 31) warp_sums[w] = inc;
    __syncthreads();
    unsigned before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < RS_WARPS; ++k) {
        if (k < w) before += warp_sums[k];
        all += warp_sums[k];
    }
    *total = all;
    return before + inc - v;
}

// block d: exclusive scan of digit d's counts over the tiles
__global__ void __launch_bounds__(RS_THREADS) sort_scan_kernel(const SortArgs a) {
    __shared__ unsigned sums[RS_WARPS];
    unsigned *h = a.hist + (size_t)blockIdx.x * a.tiles;
    unsigned carry = 0;
    for (unsigned t0 = 0; t0 < a.tiles; t0 += RS_THREADS) {
        const unsigned t = t0 + threadIdx.x;
        const unsigned v = t < a.tiles ? h[t] : 0u;
        unsigned all;
        const unsigned ex = block_exclusive(v, sums, &all);
        if (t < a.tiles) h[t] = carry + ex;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = carry;
}

// counts entry (of digit d) into its warp's counters; its rank among the warp's entries of that digit
__device__ __forceinline__ unsigned warp_rank(unsigned short *cnt, unsigned d, int bits, bool in) {
    const int lane = threadIdx.x & 31;
    const unsigned same = lanes_with(d, bits, in);
    const unsigned below = __popc(same & ((1u << lane) - 1u));
    const unsigned before = in ? cnt[d] : 0u;
    __syncwarp();
    if (in && below == 0) cnt[d] = (unsigned short)(before + __popc(same));
    __syncwarp();
    return before + below;
}

__global__ void __launch_bounds__(RS_THREADS) sort_scatter_kernel(const SortArgs a) {
    extern __shared__ unsigned smem[];
    __shared__ unsigned sums[RS_WARPS];
    const unsigned bins = 1u << a.bits, mask = bins - 1u;
    unsigned *at = smem;                                                   // (bins): first position of the tile's entries of a digit
    unsigned short *cnt = reinterpret_cast<unsigned short *>(smem + bins); // (warps, bins)
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (unsigned b = threadIdx.x; b < bins * RS_WARPS / 2; b += RS_THREADS) smem[bins + b] = 0;
    const unsigned base = blockIdx.x * RS_TILE + w * (32 * RS_ROUNDS) + lane;
    uint2 e[RS_ROUNDS];
    unsigned short rank[RS_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) e[r] = base + r * 32 < a.n ? sort_entry(a, base + r * 32) : make_uint2(0, 0);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r)
        rank[r] = (unsigned short)warp_rank(cnt + w * bins, (e[r].x >> a.shift) & mask, a.bits, base + r * 32 < a.n);
    __syncthreads();
    // first positions: digits before this one, tiles before this one; then warps before this one
    unsigned carry = 0;
    for (unsigned b0 = 0; b0 < bins; b0 += RS_THREADS) {
        const unsigned d = b0 + threadIdx.x;
        unsigned all;
        const unsigned digit = block_exclusive(d < bins ? a.total[d] : 0u, sums, &all);
        if (d < bins) {
            at[d] = carry + digit + a.hist[(size_t)d * a.tiles + blockIdx.x];
            unsigned short before = 0;
#pragma unroll
            for (int k = 0; k < RS_WARPS; ++k) {
                const unsigned short c = cnt[k * bins + d];
                cnt[k * bins + d] = before;
                before += c;
            }
        }
        carry += all;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        if (base + r * 32 >= a.n) continue;
        const unsigned d = (e[r].x >> a.shift) & mask;
        const unsigned pos = at[d] + cnt[w * bins + d] + rank[r];
        if (a.last) {
            a.key_out[pos] = e[r].x;
            a.val_out[pos] = e[r].y;
        } else {
            a.out[pos] = e[r];
        }
    }
}

// at most one tile: all digits by one block, entries in registers between passes through shared memory
__global__ void __launch_bounds__(RS_THREADS) sort_small_kernel(const SortArgs a) {
    constexpr unsigned BINS = 1u << RS_SMALL_BITS;
    __shared__ uint2 entry[RS_TILE];
    __shared__ unsigned short cnt[RS_WARPS * BINS];
    __shared__ unsigned at[BINS], sums[RS_WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const unsigned base = w * (32 * RS_ROUNDS) + lane;
    uint2 e[RS_ROUNDS];
    unsigned short rank[RS_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const unsigned i = base + r * 32;
        e[r] = i < a.n ? make_uint2(index_key(a, i), i) : make_uint2(0, 0);
        if (i < a.n && a.dweight && e[r].x == (unsigned)a.rows) a.dweight[i] = 0.0f;
    }
    for (int shift = 0; shift < a.key_bits; shift += RS_SMALL_BITS) {
        for (unsigned b = threadIdx.x; b < BINS * RS_WARPS / 2; b += RS_THREADS) reinterpret_cast<unsigned *>(cnt)[b] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_ROUNDS; ++r)
            rank[r] = (unsigned short)warp_rank(cnt + w * BINS, (e[r].x >> shift) & (BINS - 1), RS_SMALL_BITS, base + r * 32 < a.n);
        __syncthreads();
        unsigned all = 0, before = 0;
#pragma unroll
        for (int k = 0; k < RS_WARPS; ++k) {
            const unsigned c = cnt[k * BINS + threadIdx.x];
            cnt[k * BINS + threadIdx.x] = (unsigned short)before;
            before += c;
        }
        at[threadIdx.x] = block_exclusive(before, sums, &all);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_ROUNDS; ++r) {
            const unsigned d = (e[r].x >> shift) & (BINS - 1);
            if (base + r * 32 < a.n) entry[at[d] + cnt[w * BINS + d] + rank[r]] = e[r];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_ROUNDS; ++r)
            if (base + r * 32 < a.n) e[r] = entry[base + r * 32];
    }
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r)
        if (base + r * 32 < a.n) {
            a.key_out[base + r * 32] = e[r].x;
            a.val_out[base + r * 32] = e[r].y;
        }
}

// ------------------------------------------------------------------------------------------------
// Sums per row.  A row whose entries fill a whole aligned chunk of LG_CHUNK sorted entries is "long": its chunks are
// summed by blocks of their own into partial rows, and the partial rows are added in order; all others are added
// by a group of lanes.  Where a lane's one vector covers its share of the columns (DOT), the same pass forms dweight:
// the entry's dout row is in registers, and the table's row is read once for all its entries.
// ------------------------------------------------------------------------------------------------
constexpr int LG_THREADS = 256, LG_WARPS = LG_THREADS / 32, LG_CHUNK = 256;

struct GradArgs {
    const void *dout, *table, *index;
    const float *weight;
    float *dtable, *dweight, *partial;  // partial: (2 * chunks, width)
    const unsigned *key, *order;
    long long rows, dout_stride, table_stride;
    unsigned n, chunks, chunk_blocks, col_tiles;  // chunk_blocks * col_tiles blocks work on chunks, those behind them on rows
    int width, index_type, rows_per_warp;
    float scale;
};

__device__ __forceinline__ unsigned lower_bound(const unsigned *key, unsigned n, unsigned v) {
    unsigned lo = 0, len = n;
    while (len) {
        const unsigned half = len >> 1;
        if (__ldg(key + lo + half) < v) {
            lo += half + 1;
            len -= half + 1;
        } else {
            len = half;
        }
    }
    return lo;
}

__device__ __forceinline__ bool is_long(unsigned s, unsigned e) {
    const unsigned full = (s + LG_CHUNK - 1) / LG_CHUNK * LG_CHUNK;
    return full + LG_CHUNK <= e;
}

// acc += sum over sorted entries s, s + step, ... below e of scale * weight * dout, columns col, col + col_step, ...
// DOT: also dweight of those entries, e the table row's columns, summed over the G lanes of `lanes`
template <class D, int VE, int NV, int G, bool DOT>
__device__ __forceinline__ void add_entries(const GradArgs &a, unsigned s, unsigned e, unsigned step, int col, int col_step,
                                            float (&acc)[NV][VE], const float (&row)[VE], unsigned lanes) {
    constexpr int U = NV == 1 ? 4 : 2;  // entries in flight
    for (unsigned j = s; j < e; j += step * U) {
        unsigned i[U];
        float f[U];
        Vec<D, VE> d[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u) i[u] = j + u * step < e ? __ldg(a.order + j + u * step) : 0xffffffffu;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f[u] = i[u] == 0xffffffffu ? 0.0f : a.weight ? a.scale * __ldg(a.weight + i[u]) : a.scale;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const int c = col + q * col_step;
                if (i[u] != 0xffffffffu && c < a.width)
                    d[u][q].load_stream(static_cast<const D *>(a.dout) + (long long)i[u] * a.dout_stride + c);
                else d[u][q].zero();
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i[u] == 0xffffffffu) break;
            float dot = 0.0f;
#pragma unroll
            for (int q = 0; q < NV; ++q)
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    const float x = d[u][q].get(v);
                    acc[q][v] = fmaf(f[u], x, acc[q][v]);
                    if (DOT) dot = fmaf(x, row[v], dot);
                }
            if (DOT) {
#pragma unroll
                for (int o = G / 2; o; o >>= 1) dot += __shfl_xor_sync(lanes, dot, o);
                if (col == 0) a.dweight[i[u]] = a.scale * dot;
            }
        }
    }
}

template <int VE>
__device__ __forceinline__ void store_row(float *p, const float (&acc)[VE]) {
    Vec<float, VE> o;
#pragma unroll
    for (int v = 0; v < VE; ++v) o.el[v] = acc[v];
    o.store_stream(p);
}

template <class T, int VE>
__device__ __forceinline__ void load_row(const GradArgs &a, long long p, int col, bool some, float (&row)[VE]) {
    Vec<T, VE> t;
    if (some && col < a.width) t.load_stream(static_cast<const T *>(a.table) + p * a.table_stride + col);
    else t.zero();
#pragma unroll
    for (int v = 0; v < VE; ++v) row[v] = t.get(v);
}

// whether the row that chunk c begins with (side 0) or the one that it ends with (1) is long.  The keys are sorted, so
// equal keys at both ends of a chunk mean that all of it is one row.
__device__ __forceinline__ bool chunk_long(const GradArgs &a, unsigned c, int side) {
    const unsigned c0 = c * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n);
    const unsigned first = __ldg(a.key + c0), last = __ldg(a.key + c1 - 1);
    if ((side ? last : first) >= (unsigned)a.rows) return false;  // entries without a row
    if (side == 0) return (c0 + LG_CHUNK <= a.n && last == first) || (c0 >= LG_CHUNK && __ldg(a.key + c0 - LG_CHUNK) == first);
    return last != first && c1 + LG_CHUNK <= a.n && __ldg(a.key + c1 + LG_CHUNK - 1) == last;
}

// Eight chunks per block: the part of the rows at a chunk's ends that are long -> partial rows 2c (the row that the
// chunk begins with) and 2c + 1 (the row that begins inside it).  Column tiles of 32 VE.
template <class D, class T, int VE, bool DOT>
__device__ __forceinline__ void grad_chunks(const GradArgs &a, unsigned block, unsigned col_tile) {
    __shared__ float part[LG_WARPS][32 * VE];
    __shared__ unsigned todo;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (w == 0) {
        const unsigned c = block * LG_WARPS + (lane >> 1);
        const unsigned mask = __ballot_sync(0xffffffffu, lane < 2 * LG_WARPS && c < a.chunks && chunk_long(a, c, lane & 1));
        if (lane == 0) todo = mask;
    }
    __syncthreads();
    const int col = (col_tile * 32 + lane) * VE;
    for (unsigned left = todo; left; left &= left - 1) {
        const int bit = __ffs(left) - 1, side = bit & 1;
        const unsigned c = block * LG_WARPS + (bit >> 1), c0 = c * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n);
        const unsigned first = __ldg(a.key + c0), last = __ldg(a.key + c1 - 1);
        unsigned s = c0, e = c1;
        if (first != last) {
            const unsigned cut = c0 + lower_bound(a.key + c0, c1 - c0, side ? last : first + 1);
            if (side) s = cut;
            else e = cut;
        }
        float acc[1][VE] = {}, row[VE];
        if (DOT) load_row<T, VE>(a, side ? last : first, col, true, row);
        add_entries<D, VE, 1, 32, DOT>(a, s + w, e, LG_WARPS, col, 0, acc, row, 0xffffffffu);
#pragma unroll
        for (int v = 0; v < VE; ++v) part[w][lane * VE + v] = acc[0][v];
        __syncthreads();
        if (w == 0 && col < a.width) {
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                float t = 0.0f;
                for (int k = 0; k < LG_WARPS; ++k) t += part[k][lane * VE + v];
                acc[0][v] = t;
            }
            store_row<VE>(a.partial + ((size_t)2 * c + side) * a.width + col, acc[0]);
        }
        __syncthreads();
    }
}

// Eight chunks per block: for a long row that begins in one of them, adds its partial rows in order and writes the row.
template <int VE>
__global__ void __launch_bounds__(LG_THREADS) grad_join_kernel(const GradArgs a) {
    __shared__ float part[LG_WARPS][32 * VE];
    __shared__ unsigned todo;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (w == 0) {
        // a long row begins in c if it is what c ends with and c is where it starts: inside c (side 1), or at its first entry
        const unsigned c = blockIdx.x * LG_WARPS + lane;
        bool begins = false;
        if (lane < LG_WARPS && c < a.chunks) {
            const unsigned c0 = c * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n), first = __ldg(a.key + c0);
            begins = chunk_long(a, c, 1) || (__ldg(a.key + c1 - 1) == first && chunk_long(a, c, 0) &&
                                             (c0 == 0 || __ldg(a.key + c0 - 1) != first));
        }
        const unsigned mask = __ballot_sync(0xffffffffu, begins);
        if (lane == 0) todo = mask;
    }
    __syncthreads();
    const int col = (blockIdx.y * 32 + lane) * VE;
    for (unsigned left = todo; left; left &= left - 1) {
        const unsigned b = blockIdx.x * LG_WARPS + __ffs(left) - 1, c0 = b * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n);
        const unsigned row = __ldg(a.key + c1 - 1);
        const bool inside = __ldg(a.key + c0) != row;
        const unsigned e = c0 + lower_bound(a.key + c0, a.n - c0, row + 1), last = (e - 1) / LG_CHUNK;
        float acc[VE] = {};
        if (col < a.width) {
#pragma unroll 4
            for (unsigned c = b + w; c <= last; c += LG_WARPS) {
                const unsigned slot = 2 * c + (c == b && inside ? 1 : 0);
                Vec<float, VE> d;
                d.load(a.partial + (size_t)slot * a.width + col);
#pragma unroll
                for (int v = 0; v < VE; ++v) acc[v] += d.el[v];
            }
        }
#pragma unroll
        for (int v = 0; v < VE; ++v) part[w][lane * VE + v] = acc[v];
        __syncthreads();
        if (w == 0 && col < a.width) {
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                float t = 0.0f;
                for (int k = 0; k < LG_WARPS; ++k) t += part[k][lane * VE + v];
                acc[v] = t;
            }
            store_row<VE>(a.dtable + (size_t)row * a.width + col, acc);
        }
        __syncthreads();
    }
}

// A group of G lanes per row (32 / G rows at a time per warp), each lane NV vectors of VE columns per column tile.
template <class D, class T, int VE, int NV, int G, bool DOT>
__device__ __forceinline__ void grad_rows(const GradArgs &a, unsigned block) {
    constexpr int RPW = 32 / G;
    const int lane = threadIdx.x & 31, sub = lane % G;
    const unsigned lanes = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << (lane / G * G);
    const long long warp = (long long)block * LG_WARPS + (threadIdx.x >> 5), row0 = warp * a.rows_per_warp;
    if (row0 >= a.rows) return;
    // lane k finds where row row0 + k begins; the last lane's row ends where the next one begins
    const unsigned begin = lower_bound(a.key, a.n, (unsigned)min(row0 + lane, a.rows));
    const unsigned after = lower_bound(a.key, a.n, (unsigned)min(row0 + 32, a.rows));
    for (int r = 0; r < a.rows_per_warp; r += RPW) {
        const int k = r + lane / G;
        const unsigned s = __shfl_sync(0xffffffffu, begin, k & 31), next = __shfl_sync(0xffffffffu, begin, (k + 1) & 31);
        const unsigned e = k == 31 ? after : next;
        const long long row = row0 + k;
        if (row >= a.rows || k >= a.rows_per_warp || is_long(s, e)) continue;
        for (int c0 = 0; c0 < a.width; c0 += G * NV * VE) {
            float acc[NV][VE] = {}, held[VE];
            if (DOT) load_row<T, VE>(a, row, c0 + sub * VE, s < e, held);
            add_entries<D, VE, NV, G, DOT>(a, s, e, 1, c0 + sub * VE, G * VE, acc, held, lanes);
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const int c = c0 + sub * VE + q * G * VE;
                if (c < a.width) store_row<VE>(a.dtable + row * a.width + c, acc[q]);
            }
        }
    }
}

template <class D, class T, int VE, int NV, int G, bool DOT>
__global__ void __launch_bounds__(LG_THREADS) grad_sum_kernel(const GradArgs a) {
    const unsigned chunk_part = a.chunk_blocks * a.col_tiles;
    if (blockIdx.x < chunk_part) grad_chunks<D, T, VE, DOT>(a, blockIdx.x % a.chunk_blocks, blockIdx.x / a.chunk_blocks);
    else grad_rows<D, T, VE, NV, G, DOT>(a, blockIdx.x - chunk_part);
}

// dweight: a warp per entry.
template <class D, class T, int VE>
__global__ void __launch_bounds__(LG_THREADS) grad_weight_kernel(const GradArgs a) {
    const int lane = threadIdx.x & 31;
    for (long long i = ((long long)blockIdx.x * LG_THREADS + threadIdx.x) >> 5; i < a.n; i += ((long long)gridDim.x * LG_THREADS) >> 5) {
        const long long p = a.index_type == FLARE_I64 ? row_of<long long>(a.index, i, a.rows) : row_of<int>(a.index, i, a.rows);
        float t = 0.0f;
        if (p >= 0)
            for (int c = lane * VE; c < a.width; c += 32 * VE) {
                Vec<D, VE> d;
                Vec<T, VE> e;
                d.load_stream(static_cast<const D *>(a.dout) + i * a.dout_stride + c);
                e.load(static_cast<const T *>(a.table) + p * a.table_stride + c);
#pragma unroll
                for (int v = 0; v < VE; ++v) t = fmaf(d.get(v), e.get(v), t);
            }
#pragma unroll
        for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) a.dweight[i] = p >= 0 ? a.scale * t : 0.0f;
    }
}

__global__ void zero_kernel(float *p, long long n) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
        p[i] = 0.0f;
}

struct GradPlan {
    long long entries[2], key, val, hist, total, partial, bytes;
    unsigned tiles, chunks;
    int bits, passes;
};

GradPlan grad_plan(long long rows, long long n, int width) {
    GradPlan g{};
    g.tiles = (unsigned)((n + RS_TILE - 1) / RS_TILE);
    g.chunks = (unsigned)((n + LG_CHUNK - 1) / LG_CHUNK);
    g.bits = 1;
    while ((rows >> g.bits) != 0) ++g.bits;  // keys are 0 .. rows
    g.passes = (g.bits + RS_MAX_BITS - 1) / RS_MAX_BITS;
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long p = at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    g.key = take(4 * n);
    g.val = take(4 * n);
    if (g.tiles > 1) {
        for (int b = 0; b < 2; ++b) g.entries[b] = take(b < g.passes - 1 ? 8 * n : 0);
        g.hist = take((4ll << (g.bits + g.passes - 1) / g.passes) * g.tiles);
        g.total = take(4ll * RS_BINS);
    }
    // only rows that fill a chunk have partial rows
    g.partial = take(n >= LG_CHUNK ? 8ll * g.chunks * width : 0);
    g.bytes = at;
    return g;
}

int sort_entries(const flare_lookup_grad_args *in, const GradPlan &g, bool dot, cudaStream_t st) {
    char *ws = static_cast<char *>(in->workspace);
    auto words = [&](long long at) { return reinterpret_cast<unsigned *>(ws + at); };
    SortArgs s{};
    s.index = in->index;
    s.index_type = in->index_type;
    s.key_out = words(g.key);
    s.val_out = words(g.val);
    s.dweight = dot ? in->dweight : nullptr;
    s.rows = in->rows;
    s.n = (unsigned)in->n;
    s.tiles = g.tiles;
    s.key_bits = g.bits;
    if (g.tiles == 1) {
        sort_small_kernel<<<1, RS_THREADS, 0, st>>>(s);
    } else {
        s.hist = words(g.hist);
        s.total = words(g.total);
        for (int p = 0; p < g.passes; ++p) {
            s.first = p == 0;
            s.last = p == g.passes - 1;
            s.bits = (g.bits - s.shift + (g.passes - p) - 1) / (g.passes - p);
            s.in = reinterpret_cast<uint2 *>(ws + g.entries[(p + 1) & 1]);
            s.out = reinterpret_cast<uint2 *>(ws + g.entries[p & 1]);
            const size_t smem = (4 + 2 * RS_WARPS) << s.bits;
            sort_count_kernel<<<g.tiles, RS_THREADS, 0, st>>>(s);
            sort_scan_kernel<<<1u << s.bits, RS_THREADS, 0, st>>>(s);
            sort_scatter_kernel<<<g.tiles, RS_THREADS, smem, st>>>(s);
            s.shift += s.bits;
        }
    }
    OPS_LAUNCHED("flare_lookup_backward");
    return FLARE_OK;
}

template <int VE>
using Width = std::integral_constant<int, VE>;
template <class F>
void with_width(int ve, F f) {
    switch (ve) {
        case 8: f(Width<8>{}); break;
        case 4: f(Width<4>{}); break;
        case 2: f(Width<2>{}); break;
        default: f(Width<1>{}); break;
    }
}

template <class D, class T, int VE, bool DOT>
void launch_sums(GradArgs a, cudaStream_t st) {
    const int vectors = a.width / VE;
    a.col_tiles = (vectors + 31) / 32;
    a.chunk_blocks = a.n >= LG_CHUNK ? (a.chunks + LG_WARPS - 1) / LG_WARPS : 0;
    // 32 rows a warp share a search; fewer where that leaves the machine without warps
    a.rows_per_warp = 32;
    while (a.rows_per_warp > 8 && a.rows / a.rows_per_warp < 64 * SMS) a.rows_per_warp /= 2;
    const long long per_block = (long long)a.rows_per_warp * LG_WARPS;
    const unsigned grid = a.chunk_blocks * a.col_tiles + (unsigned)((a.rows + per_block - 1) / per_block);
    if (vectors <= 8) grad_sum_kernel<D, T, VE, 1, 8, DOT><<<grid, LG_THREADS, 0, st>>>(a);
    else if (vectors <= 16) grad_sum_kernel<D, T, VE, 1, 16, DOT><<<grid, LG_THREADS, 0, st>>>(a);
    else if (vectors <= 32) grad_sum_kernel<D, T, VE, 1, 32, DOT><<<grid, LG_THREADS, 0, st>>>(a);
    else if constexpr (!DOT) grad_sum_kernel<D, T, VE, 4, 32, false><<<grid, LG_THREADS, 0, st>>>(a);
    if (a.chunk_blocks) grad_join_kernel<VE><<<dim3(a.chunk_blocks, a.col_tiles), LG_THREADS, 0, st>>>(a);
}

// widest vectors that all the given tensors allow
int grad_vec(const flare_lookup_grad_args *in, bool dtable, bool table) {
    int ve = 8;
    while (ve > 1 && !(in->width % ve == 0 && fits_vec(in->dout, in->dout_stride, type_size(in->dout_type), ve) &&
                       (!dtable || fits_vec(in->dtable, in->width, 4, ve)) &&
                       (!table || fits_vec(in->table, in->table_stride, type_size(in->table_type), ve))))
        ve >>= 1;
    return ve;
}

int run_lookup_backward(const flare_lookup_grad_args *in, cudaStream_t st) {
    GradArgs a{};
    a.dout = in->dout;
    a.table = in->table;
    a.index = in->index;
    a.weight = in->weight;
    a.dtable = in->dtable;
    a.dweight = in->dweight;
    a.rows = in->rows;
    a.dout_stride = in->dout_stride;
    a.table_stride = in->table_stride;
    a.n = (unsigned)in->n;
    a.width = in->width;
    a.index_type = in->index_type;
    a.scale = in->scale;
    if (in->n == 0) {
        if (in->dtable && in->rows) {
            const long long count = in->rows * in->width;
            zero_kernel<<<(unsigned)std::min<long long>((count + 255) / 256, SMS * 16), 256, 0, st>>>(in->dtable, count);
            OPS_LAUNCHED("flare_lookup_backward");
        }
        return FLARE_OK;
    }
    const bool sums = in->dtable && in->rows;
    // both gradients in one pass where a row's columns are one vector a lane
    const int both = sums && in->dweight ? grad_vec(in, true, true) : 0;
    const bool dot = both && in->width / both <= 32;
    if (sums) {
        const GradPlan g = grad_plan(in->rows, in->n, in->width);
        char *ws = static_cast<char *>(in->workspace);
        const int e = sort_entries(in, g, dot, st);
        if (e) return e;
        a.key = reinterpret_cast<unsigned *>(ws + g.key);
        a.order = reinterpret_cast<unsigned *>(ws + g.val);
        a.partial = reinterpret_cast<float *>(ws + g.partial);
        a.chunks = g.chunks;
        with_type(in->dout_type, [&](auto d) {
            using D = typename decltype(d)::type;
            if (dot)
                with_type(in->table_type, [&](auto t) {
                    with_width(both, [&](auto ve) { launch_sums<D, typename decltype(t)::type, decltype(ve)::value, true>(a, st); });
                    return 0;
                });
            else with_width(grad_vec(in, true, false), [&](auto ve) { launch_sums<D, float, decltype(ve)::value, false>(a, st); });
            return 0;
        });
        OPS_LAUNCHED("flare_lookup_backward");
    }
    if (in->dweight && !dot) {
        const unsigned blocks = (unsigned)std::min<long long>((in->n + 7) / 8, SMS * 64);
        with_type(in->dout_type, [&](auto d) {
            return with_type(in->table_type, [&](auto t) {
                with_width(grad_vec(in, false, true), [&](auto ve) {
                    grad_weight_kernel<typename decltype(d)::type, typename decltype(t)::type, decltype(ve)::value>
                        <<<blocks, LG_THREADS, 0, st>>>(a);
                });
                return 0;
            });
        });
        OPS_LAUNCHED("flare_lookup_backward");
    }
    return FLARE_OK;
}

}  // namespace flare

using namespace flare;

extern "C" {

int flare_lookup(const flare_lookup_args *a, void *stream) {
    OPS_CHECK(a, "flare_lookup: NULL argument");
    OPS_CHECK(is_float_type(a->table_type) || a->table_type == FLARE_MICRO, "flare_lookup: unknown table type %d", a->table_type);
    OPS_CHECK(is_float_type(a->out_type), "flare_lookup: unknown output type %d", a->out_type);
    OPS_CHECK(a->index_type == FLARE_I32 || a->index_type == FLARE_I64, "flare_lookup: unknown index type %d", a->index_type);
    OPS_CHECK(a->n >= 0 && a->rows >= 0 && a->width >= 0, "flare_lookup: negative size");
    if (a->n == 0 || a->width == 0) return FLARE_OK;
    OPS_CHECK(a->index && a->out && (a->table || a->rows == 0), "flare_lookup: NULL buffer");
    OPS_CHECK(a->table_type != FLARE_MICRO || a->scales || a->rows == 0, "flare_lookup: a 4-bit table needs its scales");
    OPS_CHECK(a->out_stride >= a->width, "flare_lookup: output rows of stride %lld overlap", a->out_stride);
    return run_lookup(a, static_cast<cudaStream_t>(stream));
}

long long flare_lookup_workspace(long long rows, long long n, int width) {
    return rows > 0 && n > 0 && width > 0 ? grad_plan(rows, n, width).bytes : 0;
}

int flare_lookup_backward(const flare_lookup_grad_args *a, void *stream) {
    OPS_CHECK(a, "flare_lookup_backward: NULL argument");
    OPS_CHECK(is_float_type(a->dout_type), "flare_lookup_backward: unknown gradient type %d", a->dout_type);
    OPS_CHECK(!a->dweight || is_float_type(a->table_type), "flare_lookup_backward: table type %d has no gradient", a->table_type);
    OPS_CHECK(a->index_type == FLARE_I32 || a->index_type == FLARE_I64, "flare_lookup_backward: unknown index type %d", a->index_type);
    OPS_CHECK(a->n >= 0 && a->rows >= 0 && a->width >= 0, "flare_lookup_backward: negative size");
    OPS_CHECK(a->rows < 0x7fffffffll && a->n < 0x7fffffffll - RS_TILE, "flare_lookup_backward: %lld rows, %lld entries",
              a->rows, a->n);
    OPS_CHECK(a->n == 0 || (a->index && (a->dout || a->width == 0)), "flare_lookup_backward: NULL buffer");
    OPS_CHECK(!a->dweight || a->n == 0 || a->table || a->rows == 0 || a->width == 0, "flare_lookup_backward: dweight needs the table");
    const long long need = a->dtable ? flare_lookup_workspace(a->rows, a->n, a->width) : 0;
    OPS_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && (reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0),
              "flare_lookup_backward: workspace of %lld bytes, %lld needed (16-byte aligned)", a->workspace_bytes, need);
    if (a->width == 0) {
        flare_lookup_grad_args b = *a;
        b.dtable = nullptr;
        return run_lookup_backward(&b, static_cast<cudaStream_t>(stream));
    }
    return run_lookup_backward(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
