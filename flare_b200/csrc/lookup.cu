// lookup.cu -- rows of a descriptor table for a list of hits, with scaling, and the table's gradient.
//
//   out[i]    = s w_i E[idx_i]                    (0 where idx_i names no row)
//   dE[p]     = s sum_{i: idx_i = p} w_i dout_i   (in a fixed order)
//   dw_i      = s <dout_i, E[idx_i]>
//
// The forward is bound by memory: it reads the index and each distinct row once from HBM (further hits of a row
// mostly come from L2) and writes n rows.  The gradient sorts the entries by row first (a stable radix sort of
// (row, i) pairs, so that the order of every sum is fixed and no float atomics are needed), after which each
// row's entries lie together and a group of lanes adds them in registers and writes the row once.
#include <algorithm>

#include "ops.cuh"

namespace flare {

constexpr int LK_THREADS = 256, LK_BLOCKS = 16;  // per multiprocessor at most

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

// Items in flight per thread: 16-byte loads need no more than 2 (4: 229 us instead of 172 for 2.56M rows of 96 f16), narrow ones 4.
template <class T, int VE>
constexpr int lookup_items() {
    if constexpr (std::is_void_v<T>) return 2;
    else return VE * (int)sizeof(T) >= 16 ? 2 : 4;
}

// One vector of VE elements per item.  A block takes tiles of LK_THREADS * ITEMS items in turn and asks for the next tile's
// indices while it waits for this tile's rows.  T = void: a 4-bit table.
template <class T, class O, class I, int VE>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(const LookupArgs a) {
    constexpr int ITEMS = lookup_items<T, VE>();
    const unsigned tiles = (a.items + LK_THREADS * ITEMS - 1) / (LK_THREADS * ITEMS);
    long long next[ITEMS];
    float factor[ITEMS];
    auto ask = [&](unsigned tile) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const unsigned it = tile * (LK_THREADS * ITEMS) + k * LK_THREADS + threadIdx.x;
            next[k] = -1;
            factor[k] = a.scale;
            if (tile < tiles && it < a.items) {
                const unsigned row = a.vpr.div(it);
                next[k] = row_of<I>(a.index, a.first + row, a.rows);
                if (a.weight) factor[k] = a.scale * __ldg(a.weight + a.first + row);
            }
        }
    };
    ask(blockIdx.x);
    for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const unsigned base = tile * (LK_THREADS * ITEMS) + threadIdx.x;
        long long p[ITEMS];
        float s[ITEMS], f[ITEMS][VE];
        unsigned row[ITEMS], v[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            p[k] = next[k];
            s[k] = factor[k];
            row[k] = a.vpr.div(base + k * LK_THREADS);
            v[k] = base + k * LK_THREADS - row[k] * a.vpr.d;
        }
        if constexpr (std::is_void_v<T>) {
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
                if (p[k] >= 0) micro_load<VE>(a, p[k], v[k], f[k]);
            ask(tile + gridDim.x);
        } else {
            Vec<T, VE> t[ITEMS];
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
                if (p[k] >= 0) t[k].load(static_cast<const T *>(a.table) + p[k] * a.table_stride + (long long)v[k] * VE);
            ask(tile + gridDim.x);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
#pragma unroll
                for (int e = 0; e < VE; ++e) f[k][e] = t[k].get(e);
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if (base + k * LK_THREADS >= a.items) break;
            Vec<O, VE> o;
#pragma unroll
            for (int e = 0; e < VE; ++e) o.set(e, p[k] >= 0 ? f[k][e] * s[k] : 0.0f);
            o.store_stream(static_cast<O *>(a.out) + (a.first + row[k]) * a.out_stride + (long long)v[k] * VE);
        }
    }
}

// Rows whose elements go one or two at a time: a warp per row and 32 UNROLL VE columns of it, so that the index, the weight and
// the addresses are worked out once and not per element (16383 rows of 1023 bf16: 17 us, per element 48).
constexpr int LK_UNROLL = 8;
template <class T, class O, class I, int VE>
__global__ void __launch_bounds__(LK_THREADS) lookup_wide_kernel(const LookupArgs a, const unsigned items, const FastDiv parts) {
    const int lane = threadIdx.x & 31;
    for (unsigned it = (blockIdx.x * LK_THREADS + threadIdx.x) >> 5; it < items; it += gridDim.x * (LK_THREADS / 32)) {
        const unsigned r = parts.div(it), c0 = (it - r * parts.d) * (32 * LK_UNROLL) + lane;  // vectors
        const long long i = a.first + r, p = row_of<I>(a.index, i, a.rows);
        const float s = a.weight ? a.scale * __ldg(a.weight + i) : a.scale;
        const T *from = static_cast<const T *>(a.table) + (p < 0 ? 0 : p) * a.table_stride;
        O *to = static_cast<O *>(a.out) + i * a.out_stride;
        Vec<T, VE> t[LK_UNROLL];
        if (p >= 0)
#pragma unroll
            for (int k = 0; k < LK_UNROLL; ++k)
                if (c0 + 32 * k < a.vpr.d) t[k].load(from + (c0 + 32 * k) * VE);
#pragma unroll
        for (int k = 0; k < LK_UNROLL; ++k)
            if (c0 + 32 * k < a.vpr.d) {
                Vec<O, VE> o;
#pragma unroll
                for (int e = 0; e < VE; ++e) o.set(e, p < 0 ? 0.0f : t[k].get(e) * s);
                o.store_stream(to + (c0 + 32 * k) * VE);
            }
    }
}

template <class T, class O, class I>
void launch_lookup(const LookupArgs &a, int ve, cudaStream_t st) {
    if constexpr (!std::is_void_v<T>)
        if (ve <= 2 && a.vpr.d >= 64) {
            const FastDiv parts((a.vpr.d + 32 * LK_UNROLL - 1) / (32 * LK_UNROLL));
            const unsigned items = a.items / a.vpr.d * parts.d, per_block = LK_THREADS / 32;
            const unsigned blocks = std::min((items + per_block - 1) / per_block, (unsigned)(LK_BLOCKS * SMS));
            if (ve == 2) lookup_wide_kernel<T, O, I, 2><<<blocks, LK_THREADS, 0, st>>>(a, items, parts);
            else lookup_wide_kernel<T, O, I, 1><<<blocks, LK_THREADS, 0, st>>>(a, items, parts);
            return;
        }
    const unsigned blocks = std::min((a.items + LK_THREADS - 1) / LK_THREADS, (unsigned)(LK_BLOCKS * SMS));
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
// Per digit of up to 10 bits: count per tile, scan over tiles, scatter.  A tile is 512 R consecutive entries of one block;
// warp w ranks entries [32 R w, 32 R (w + 1)) of it 32 at a time, so ranks follow the entries' order.  Lanes with equal
// digits find one another by a ballot per bit (match.any took three times the whole kernel's time).  Short lists are
// sorted by one cluster in shared memory.
// ------------------------------------------------------------------------------------------------
constexpr int RS_THREADS = 512, RS_WARPS = RS_THREADS / 32, RS_MAX_ROUNDS = 9;
constexpr int RS_MAX_BITS = 10, RS_BINS = 1 << RS_MAX_BITS, RS_SMALL_BITS = 8;

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

template <int ROUNDS>
__global__ void __launch_bounds__(RS_THREADS) sort_count_kernel(const SortArgs a) {
    __shared__ unsigned h[RS_BINS];
    const unsigned bins = 1u << a.bits, mask = bins - 1u;
    for (unsigned b = threadIdx.x; b < bins; b += RS_THREADS) h[b] = 0;
    __syncthreads();
    const unsigned base = blockIdx.x * (RS_THREADS * ROUNDS);
#pragma unroll 8
    for (int r = 0; r < ROUNDS; ++r) {
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
template <int WARPS>
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
    for (int k = 0; k < WARPS; ++k) {
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
        const unsigned ex = block_exclusive<RS_WARPS>(v, sums, &all);
        if (t < a.tiles) h[t] = carry + ex;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = carry;
}

// Ranks of a warp's ROUNDS x 32 entries among those of equal digit; cnt (zeroed) ends as the digits' counts.  All ballots
// come first, as they do not depend on one another; the rounds' counts do.
template <int ROUNDS>
__device__ __forceinline__ void warp_ranks(unsigned short *cnt, const uint2 (&e)[ROUNDS], int shift, int bits, unsigned first, unsigned n,
                                           unsigned short (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 31;
    const unsigned mask = (1u << bits) - 1u;
    unsigned same[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) same[r] = __ballot_sync(0xffffffffu, first + r * 32 < n);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) same[r] = first + r * 32 < n ? same[r] : ~same[r];
    for (int b = shift; b < shift + bits; ++b)
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool one = (e[r].x >> b) & 1u;
            const unsigned ones = __ballot_sync(0xffffffffu, one);
            same[r] &= one ? ones : ~ones;
        }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool in = first + r * 32 < n;
        const unsigned d = (e[r].x >> shift) & mask, below = __popc(same[r] & ((1u << lane) - 1u));
        const unsigned before = in ? cnt[d] : 0u;
        __syncwarp();
        if (in && below == 0) cnt[d] = (unsigned short)(before + __popc(same[r]));
        __syncwarp();
        rank[r] = (unsigned short)(before + below);
    }
}

template <int ROUNDS>
__global__ void __launch_bounds__(RS_THREADS, 2) sort_scatter_kernel(const SortArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    unsigned *smem = reinterpret_cast<unsigned *>(raw);
    __shared__ unsigned sums[RS_WARPS];
    const unsigned bins = 1u << a.bits, mask = bins - 1u;
    unsigned *at = smem;                                                   // (bins): first position of the tile's entries of a digit
    unsigned short *cnt = reinterpret_cast<unsigned short *>(smem + bins); // (warps, bins)
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (unsigned b = threadIdx.x; b < bins * RS_WARPS / 2; b += RS_THREADS) smem[bins + b] = 0;
    const unsigned base = blockIdx.x * (RS_THREADS * ROUNDS) + w * (32 * ROUNDS) + lane;
    uint2 e[ROUNDS];
    unsigned short rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) e[r] = base + r * 32 < a.n ? sort_entry(a, base + r * 32) : make_uint2(0, 0);
    constexpr int PER = RS_BINS / RS_THREADS;
    unsigned total[PER], hist[PER];  // asked for early, used after the ranks
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const unsigned d = k * RS_THREADS + threadIdx.x;
        total[k] = d < bins ? __ldg(a.total + d) : 0u;
        hist[k] = d < bins ? __ldg(a.hist + (size_t)d * a.tiles + blockIdx.x) : 0u;
    }
    __syncthreads();
    warp_ranks(cnt + w * bins, e, a.shift, a.bits, base, a.n, rank);
    __syncthreads();
    // first positions: digits before this one, tiles before this one; then warps before this one
    unsigned carry = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const unsigned d = b * RS_THREADS + threadIdx.x;
        if (b * RS_THREADS >= bins) break;
        unsigned all;
        const unsigned digit = block_exclusive<RS_WARPS>(total[b], sums, &all);
        if (d < bins) {
            at[d] = carry + digit + hist[b];
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
    for (int r = 0; r < ROUNDS; ++r) {
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

// At most RS_SMALL entries: one launch instead of three a digit (16384 entries of 50k rows: 15 us instead of 18, of 1M rows 20
// instead of 25; 32768 would take 23 instead of 18, and 8192 in a single block took 20 where 8 take 11).  The blocks of a cluster
// hold equal parts of the entries, in registers between passes of 8 bits; counts of digits are read from the other blocks'
// shared memory, and entries go to their new places by stores into it.  Warp w of block b has entries [32 R (32 b + w),
// 32 R (32 b + w + 1)), R = 2^a.bits rounds.
constexpr int RS_SMALL_THREADS = 1024, RS_SMALL_WARPS = 32, RS_SMALL_ROUNDS = 2, RS_SMALL_BLOCKS = 8;
constexpr int RS_SMALL = RS_SMALL_THREADS * RS_SMALL_ROUNDS * RS_SMALL_BLOCKS;
static_assert(RS_SMALL <= 65536, "entry numbers of 16 bits");

__device__ __forceinline__ unsigned cluster_address(const void *p, unsigned block) {
    unsigned at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(block));
    return at;
}
__device__ __forceinline__ void small_sync(bool cluster) {
    if (cluster) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}

// grid: one cluster of a.tiles blocks
__global__ void __launch_bounds__(RS_SMALL_THREADS) sort_small_kernel(const SortArgs a) {
    constexpr unsigned BINS = 1u << RS_SMALL_BITS, MASK = BINS - 1;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ unsigned at[BINS], counts[BINS], sums[RS_SMALL_WARPS];
    const int rounds = 1 << a.bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const unsigned block_log = 10 + a.bits, block = blockIdx.x;  // log2 of a block's entries
    unsigned *keys = reinterpret_cast<unsigned *>(raw);
    unsigned short *nums = reinterpret_cast<unsigned short *>(keys + (1u << block_log));
    unsigned short *cnt = nums + (1u << block_log);  // (warps, bins)
    const unsigned local = w * (32 * rounds) + lane, base = (block << block_log) + local;
    unsigned key[RS_SMALL_ROUNDS];
    unsigned short num[RS_SMALL_ROUNDS], rank[RS_SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_SMALL_ROUNDS; ++r) {
        const unsigned i = base + r * 32;
        key[r] = 0;
        num[r] = (unsigned short)i;
        if (r < rounds && i < a.n) {
            key[r] = index_key(a, i);
            if (a.dweight && key[r] == (unsigned)a.rows) a.dweight[i] = 0.0f;
        }
    }
    for (int shift = 0; shift < a.key_bits; shift += RS_SMALL_BITS) {
        for (unsigned b = threadIdx.x; b < BINS * RS_SMALL_WARPS / 2; b += RS_SMALL_THREADS) reinterpret_cast<unsigned *>(cnt)[b] = 0;
        __syncthreads();
        unsigned short *mine = cnt + w * BINS;
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r) {
            if (r >= rounds) break;
            const bool in = base + r * 32 < a.n;
            const unsigned d = (key[r] >> shift) & MASK, some = __ballot_sync(0xffffffffu, in);
            unsigned same = in ? some : ~some;
#pragma unroll
            for (int b = 0; b < RS_SMALL_BITS; ++b) {
                const bool one = (d >> b) & 1u;
                const unsigned ones = __ballot_sync(0xffffffffu, one);
                same &= one ? ones : ~ones;
            }
            const unsigned below = __popc(same & ((1u << lane) - 1u)), before = in ? mine[d] : 0u;
            __syncwarp();
            if (in && below == 0) mine[d] = (unsigned short)(before + __popc(same));
            __syncwarp();
            rank[r] = (unsigned short)(before + below);
        }
        __syncthreads();
        // first positions: digits before this one, then warps before this one
        unsigned count = 0, all = 0;
        if (threadIdx.x < BINS)
#pragma unroll 8
            for (int k = 0; k < RS_SMALL_WARPS; ++k) {
                const unsigned c = cnt[k * BINS + threadIdx.x];
                cnt[k * BINS + threadIdx.x] = (unsigned short)count;
                count += c;
            }
        unsigned before = 0;  // of this digit in the blocks before this one
        if (a.tiles > 1) {
            if (threadIdx.x < BINS) counts[threadIdx.x] = count;
            small_sync(true);
            if (threadIdx.x < BINS) {
                count = 0;
#pragma unroll
                for (unsigned b = 0; b < RS_SMALL_BLOCKS; ++b) {
                    unsigned c = 0;
                    if (b < a.tiles)
                        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(cluster_address(counts + threadIdx.x, b)) : "memory");
                    before += b < block ? c : 0u;
                    count += c;
                }
            }
        }
        const unsigned digit = block_exclusive<RS_SMALL_WARPS>(count, sums, &all);
        if (threadIdx.x < BINS) at[threadIdx.x] = digit + before;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r) {
            if (r >= rounds || base + r * 32 >= a.n) break;
            const unsigned d = (key[r] >> shift) & MASK, pos = at[d] + mine[d] + rank[r];
            const unsigned to = pos >> block_log, slot = pos & ((1u << block_log) - 1);
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(keys + slot, to)), "r"(key[r]) : "memory");
            asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(cluster_address(nums + slot, to)), "h"(num[r]) : "memory");
        }
        small_sync(a.tiles > 1);
#pragma unroll
        for (int r = 0; r < RS_SMALL_ROUNDS; ++r)
            if (r < rounds && base + r * 32 < a.n) {
                key[r] = keys[local + r * 32];
                num[r] = nums[local + r * 32];
            }
    }
#pragma unroll
    for (int r = 0; r < RS_SMALL_ROUNDS; ++r)
        if (r < rounds && base + r * 32 < a.n) {
            a.key_out[base + r * 32] = key[r];
            a.val_out[base + r * 32] = num[r];
        }
}

// ------------------------------------------------------------------------------------------------
// Sums per row.  The sorted entries are cut into ranges of equal length, one per warp (or group of lanes) and column
// tile, whatever rows they belong to, so a row that many entries name is no special case.  A row inside one range is
// written at once; the parts of rows that cross a range's border go to partial rows, which are then added in order.
// Rows that no entry names get zeros from other blocks of the same launch.
// dout's rows are fetched at random, so what counts is how many are under way: a group of lanes keeps a ring of RING_STAGES x
// RING_ENTRIES entries in shared memory, filled by asynchronous copies (96 f16 columns: 150 KB under way per multiprocessor).  Where a
// row is one column tile (DOT), the same pass forms dweight: the table's rows take part in the ring.  Rows that
// 16-byte copies do not fit, or that are shorter than 64 bytes, go through registers, 4 entries at a time.
// ------------------------------------------------------------------------------------------------
constexpr int LG_THREADS = 256, LG_WARPS = LG_THREADS / 32;
constexpr int RING_WARPS = 2, RING_ENTRIES = 8, RING_STAGES = 2;  // 3 stages (fewer warps): 317 us where 2 take 244

struct GradArgs {
    const void *dout, *table, *index;
    const float *weight;
    float *dtable, *dweight, *partial;  // partial: (2 * ranges, width), the rows that a range begins (0) and ends (1) with
    const unsigned *key, *order;
    long long rows, dout_stride, table_stride;
    unsigned n, range, ranges, work_blocks;  // entries per range; blocks on entries, before those on rows without any
    int width, tiles, pieces, index_type;  // column tiles, 16-byte pieces of dout's row in one
    int empty_rows;
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

template <int VE>
__device__ __forceinline__ void store_row(float *p, const float (&acc)[VE]) {
    Vec<float, VE> o;
#pragma unroll
    for (int v = 0; v < VE; ++v) o.el[v] = acc[v];
    o.store_stream(p);
}

// The row that a range's stream of entries is in, and its sum so far: NQ vectors of VE columns per lane of G.
template <int VE, int NQ, int G>
struct RowSum {
    float acc[NQ][VE];
    unsigned row, before;  // before: the row of the entry before the range
    bool started;
    __device__ __forceinline__ RowSum(unsigned before_) : row(0xffffffffu), before(before_), started(false) { clear(); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int v = 0; v < VE; ++v) acc[q][v] = 0.0f;
    }
    // the stream leaves its row; `more`: the row has entries behind the range
    __device__ __forceinline__ void leave(const GradArgs &a, unsigned range, int col, bool more) {
        if (!started) return;
        float *to = row == before ? a.partial + (size_t)2 * range * a.width
                    : more        ? a.partial + ((size_t)2 * range + 1) * a.width
                                  : a.dtable + (size_t)row * a.width;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int c = col + q * G * VE;
            if (c < a.width) store_row<VE>(to + c, acc[q]);
        }
        clear();
    }
    __device__ __forceinline__ void enter(const GradArgs &a, unsigned range, int col, unsigned r) {
        if (r == row) return;
        leave(a, range, col, false);
        row = r;
        started = true;
    }
};

// a.empty_rows (at most 128) rows a warp: zeros in those that no entry names
__device__ __forceinline__ void grad_empty(const GradArgs &a, unsigned block, unsigned *words) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long row0 = ((long long)block * (blockDim.x >> 5) + w) * a.empty_rows, row1 = min(row0 + a.empty_rows, a.rows);
    if (row0 >= a.rows) return;
    // the entries of the warp's rows: both borders at once, 16 probes a step for each
    unsigned lo = 0, len = a.n;
    {
        const unsigned v = (unsigned)(lane < 16 ? row0 : row1);
        const int p = lane & 15;
        while (__any_sync(0xffffffffu, len != 0)) {
            const unsigned at = lo + (unsigned)((unsigned long long)len * (p + 1) / 17);
            const bool less = len != 0 && __ldg(a.key + at) < v;
            const unsigned below = __popc((__ballot_sync(0xffffffffu, less) >> (lane & 16)) & 0xffffu);
            if (len != 0) {
                const unsigned from = below ? lo + (unsigned)((unsigned long long)len * below / 17) + 1 : lo;
                const unsigned to = below < 16 ? lo + (unsigned)((unsigned long long)len * (below + 1) / 17) : lo + len;
                lo = from;
                len = to - from;
            }
        }
    }
    const unsigned s = __shfl_sync(0xffffffffu, lo, 0), e = __shfl_sync(0xffffffffu, lo, 16);
    unsigned *named = words + 4 * w;
    if (lane < 4) named[lane] = 0;
    __syncwarp();
    if (e - s < 1024) {
        for (unsigned j = s + lane; j < e; j += 32) {
            const unsigned r = __ldg(a.key + j) - (unsigned)row0;
            atomicOr(&named[r >> 5], 1u << (r & 31));
        }
    } else {  // few rows, many entries: look each row up
        for (int k = 0; k < 4; ++k) {
            const unsigned r = (unsigned)min(row0 + 32 * k + lane, row1);
            const unsigned at = s + lower_bound(a.key + s, e - s, r);
            const unsigned m = __ballot_sync(0xffffffffu, at < e && __ldg(a.key + at) == r);
            if (lane == 0) named[k] = m;
        }
    }
    __syncwarp();
    for (int k = 0; k < 4; ++k) {
        const long long left = row1 - row0 - 32 * k;
        unsigned empty = left <= 0 ? 0u : ~named[k] & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
        while (empty) {
            // a run of empty rows is one stretch of memory: 16 bytes at a time between its unaligned ends
            const int first = __ffs(empty) - 1;
            const unsigned after = ~(empty >> first);
            const int run = min(after ? __ffs(after) - 1 : 32, 32 - first);
            empty &= run + first >= 32 ? (1u << first) - 1u : ~(((1u << run) - 1u) << first);
            float *p = a.dtable + (row0 + 32 * k + first) * a.width;
            const long long n = (long long)run * a.width;
            const int head = (int)min(n, (long long)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / 4);
            const long long body = (n - head) / 4;
            if (lane < head) p[lane] = 0.0f;
            float4 *q = reinterpret_cast<float4 *>(p + head);
            for (long long c = lane; c < body; c += 32) __stcs(q + c, make_float4(0, 0, 0, 0));
            if (lane < n - head - 4 * body) p[head + 4 * body + lane] = 0.0f;
        }
    }
}

// rows per warp there: 128 share a search, fewer where that leaves the machine without warps
inline int empty_rows(long long rows) {
    int r = 128;
    while (r > 8 && rows / r < 24ll * SMS) r /= 2;
    return r;
}

__device__ __forceinline__ unsigned shared_addr(const void *p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(shared_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A lane's 16 bytes of a row of dout and its share of the table's row, per entry; with the stage's keys, entry numbers and
// weights a group of G lanes has RING_ENTRIES of them in a stage
template <class D, class T, bool DOT>
struct RingPiece {
    static constexpr int VE = 16 / (int)sizeof(D), TB = DOT ? VE * (int)sizeof(T) : 0;
    // bytes of a stage whose rows have `pieces` of them
    __host__ __device__ static constexpr int bytes(int pieces) { return RING_ENTRIES * (pieces * (16 + TB) + 3 * 4); }
};

// A group of G lanes per range and column tile, a lane for every 16 bytes of dout's row.  A lane copies what it will read
// itself; the lane's piece of entry e is at e * pieces + its number, dout's first, then the table's, then the numbers.
template <class D, class T, int G, bool DOT>
__global__ void __launch_bounds__(32 * RING_WARPS) grad_ring_kernel(const GradArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ unsigned words[4 * RING_WARPS];
    if (blockIdx.x >= a.work_blocks) {
        grad_empty(a, blockIdx.x - a.work_blocks, words);
        return;
    }
    using Piece = RingPiece<D, T, DOT>;
    constexpr int VE = Piece::VE, TB = Piece::TB, E = RING_ENTRIES;
    const int P = a.pieces, stage_bytes = Piece::bytes(P);
    const int sub = threadIdx.x % G;
    const unsigned lanes = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << (threadIdx.x % 32 / G * G);
    const unsigned item = blockIdx.x * (32 * RING_WARPS / G) + threadIdx.x / G, range = item / a.tiles;
    if (range >= a.ranges) return;
    const int col = (int)(item % a.tiles) * (G * VE) + sub * VE;
    const bool mine = col < a.width;
    const unsigned j0 = range * a.range, end = min(j0 + a.range, a.n);
    // entries without a row are the last ones
    unsigned j1 = end;
    if (__ldg(a.key + end - 1) >= (unsigned)a.rows) j1 = j0 + lower_bound(a.key + j0, end - j0, (unsigned)a.rows);
    if (j1 == j0) return;
    const int count = (int)(j1 - j0), stages = (count + E - 1) / E;
    unsigned char *ring = raw + (threadIdx.x / G) * (RING_STAGES * stage_bytes);
    const D *dout = static_cast<const D *>(a.dout) + col;
    const T *table = static_cast<const T *>(a.table) + col;
    // lane l < E: entry number and row of entry l of a stage
    unsigned num = 0, key = 0;
    auto numbers = [&](int st) {
        const unsigned j = j0 + st * E + sub;
        if (sub < E && j < j1) {
            num = __ldg(a.order + j);
            key = __ldg(a.key + j);
        }
    };
    auto issue = [&](int st, int slot) {
        unsigned char *to = ring + slot * stage_bytes;
        unsigned *meta = reinterpret_cast<unsigned *>(to + E * P * (16 + TB));
        const int left = count - st * E;
        if (sub < E && sub < left) {
            meta[sub] = key;
            meta[E + sub] = num;
            if (a.weight) copy4(meta + 2 * E + sub, a.weight + num);
            else meta[2 * E + sub] = __float_as_uint(1.0f);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const unsigned i = __shfl_sync(lanes, num, e, G), k = __shfl_sync(lanes, key, e, G);
            if (mine && e < left) {
                copy16(to + (e * P + sub) * 16, dout + (long long)i * a.dout_stride);
                if (DOT) {
                    const char *from = reinterpret_cast<const char *>(table + (long long)k * a.table_stride);
                    unsigned char *at = to + E * P * 16 + (e * P + sub) * TB;
                    if (TB == 8) copy8(at, from);
#pragma unroll
                    for (int b = 0; b + 16 <= TB; b += 16) copy16(at + b, from + b);
                }
            }
        }
    };
    RowSum<VE, 1, G> sum(j0 ? __ldg(a.key + j0 - 1) : 0xffffffffu);
    numbers(0);
#pragma unroll
    for (int st = 0; st < RING_STAGES - 1; ++st) {
        if (st < stages) issue(st, st);
        copies_commit();
        numbers(st + 1);
    }
    int slot = 0, fill = RING_STAGES - 1;
    for (int st = 0; st < stages; ++st) {
        if (st + RING_STAGES - 1 < stages) issue(st + RING_STAGES - 1, fill);
        copies_commit();
        numbers(st + RING_STAGES);
        copies_wait<RING_STAGES - 1>();
        __syncwarp(lanes);
        const unsigned char *from = ring + slot * stage_bytes;
        const unsigned *meta = reinterpret_cast<const unsigned *>(from + E * P * (16 + TB));
        // lanes without a piece read the last one's
        const unsigned char *mine_d = from + min(sub, P - 1) * 16, *mine_t = from + E * P * 16 + min(sub, P - 1) * TB;
        const int left = count - st * E;
        auto entries = [&](int e0, int m) {  // m <= 4 entries
            const uint4 keys = *reinterpret_cast<const uint4 *>(meta + e0);
            const float4 ws = *reinterpret_cast<const float4 *>(meta + 2 * E + e0);
            const unsigned k[4] = {keys.x, keys.y, keys.z, keys.w};
            const float f[4] = {ws.x, ws.y, ws.z, ws.w};
            float dot[4] = {};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (u >= m) break;
                sum.enter(a, range, col, k[u]);
                const float s = a.scale * f[u];
                Vec<D, VE> d;
                d.raw[0] = *reinterpret_cast<const uint4 *>(mine_d + (e0 + u) * P * 16);
                Vec<T, VE> t;
                if (DOT)
#pragma unroll
                    for (int b = 0; b < Vec<T, VE>::R::N; ++b)
                        t.raw[b] = reinterpret_cast<const typename Vec<T, VE>::R::type *>(mine_t + (e0 + u) * P * TB)[b];
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    const float x = d.get(v);
                    sum.acc[0][v] = fmaf(s, x, sum.acc[0][v]);
                    if (DOT) dot[u] = fmaf(x, t.get(v), dot[u]);
                }
                if (DOT && !mine) dot[u] = 0.0f;
            }
            if (DOT) {
                // four sums over the group: two exchanges leave each lane one of them, by two bits of its number
                const bool hi = sub & (G / 2), mid = sub & (G / 4);
                const float x = (hi ? dot[2] : dot[0]) + __shfl_xor_sync(lanes, hi ? dot[0] : dot[2], G / 2);
                const float y = (hi ? dot[3] : dot[1]) + __shfl_xor_sync(lanes, hi ? dot[1] : dot[3], G / 2);
                float z = (mid ? y : x) + __shfl_xor_sync(lanes, mid ? x : y, G / 4);
#pragma unroll
                for (int o = G / 8; o; o >>= 1) z += __shfl_xor_sync(lanes, z, o);
                const int u = (hi ? 2 : 0) + (mid ? 1 : 0);
                if (sub % (G / 4) == 0 && u < m) a.dweight[meta[E + e0 + u]] = a.scale * z;
            }
        };
        if (left >= E) {
#pragma unroll
            for (int e0 = 0; e0 < E; e0 += 4) entries(e0, 4);
        } else {
            for (int e0 = 0; e0 < left; e0 += 4) entries(e0, min(4, left - e0));
        }
        __syncwarp(lanes);  // the stage is filled again
        slot = slot + 1 == RING_STAGES ? 0 : slot + 1;
        fill = fill + 1 == RING_STAGES ? 0 : fill + 1;
    }
    copies_wait<0>();
    sum.leave(a, range, col, j1 == end && end < a.n && __ldg(a.key + end) == sum.row);
}

// A group of G lanes per range and column tile, entries through registers.  NQ vectors of VE columns per lane
template <class D, int VE, int NQ, int G>
__global__ void __launch_bounds__(LG_THREADS) grad_plain_kernel(const GradArgs a) {
    __shared__ unsigned words[4 * LG_WARPS];
    if (blockIdx.x >= a.work_blocks) {
        grad_empty(a, blockIdx.x - a.work_blocks, words);
        return;
    }
    constexpr int U = 4;
    const unsigned item = blockIdx.x * (LG_THREADS / G) + threadIdx.x / G, range = item / a.tiles;
    if (range >= a.ranges) return;
    const int col = (int)(item % a.tiles) * (G * VE * NQ) + threadIdx.x % G * VE;
    const unsigned j0 = range * a.range, j1 = min(j0 + a.range, a.n);
    RowSum<VE, NQ, G> sum(j0 ? __ldg(a.key + j0 - 1) : 0xffffffffu);
    unsigned i[U], k[U];
    auto fetch = [&](unsigned j) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            i[u] = j + u < j1 ? __ldg(a.order + j + u) : 0u;
            k[u] = j + u < j1 ? __ldg(a.key + j + u) : 0xffffffffu;
        }
    };
    fetch(j0);
    bool over = false;
    for (unsigned j = j0; j < j1 && !over; j += U) {
        unsigned ck[U];
        float f[U];
        Vec<D, VE> d[U][NQ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ck[u] = k[u];
            const bool in = ck[u] < (unsigned)a.rows;
            f[u] = in && a.weight ? a.scale * __ldg(a.weight + i[u]) : a.scale;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const int c = col + q * G * VE;
                if (in && c < a.width) d[u][q].load_stream(static_cast<const D *>(a.dout) + (long long)i[u] * a.dout_stride + c);
                else d[u][q].zero();
            }
        }
        fetch(j + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (ck[u] >= (unsigned)a.rows) {
                over = true;
                break;
            }
            sum.enter(a, range, col, ck[u]);
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int v = 0; v < VE; ++v) sum.acc[q][v] = fmaf(f[u], d[u][q].get(v), sum.acc[q][v]);
        }
    }
    sum.leave(a, range, col, j1 < a.n && __ldg(a.key + j1) == sum.row);
}

// A warp per range: if a row begins in it and goes on behind it, adds the row's partial rows in order and writes it.  Rows of
// more than JOIN_WARP ranges are added by the whole block.  grid.y: tiles of 32 VE columns
constexpr int JOIN_WARP = 32;
template <int VE>
__global__ void __launch_bounds__(LG_THREADS) grad_join_kernel(const GradArgs a) {
    __shared__ float part[LG_WARPS][32 * VE];
    __shared__ unsigned first_of[LG_WARPS], last_of[LG_WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = (blockIdx.y * 32 + lane) * VE;
    const unsigned c = blockIdx.x * LG_WARPS + w;
    auto add = [&](unsigned slot, float (&acc)[VE]) {
        Vec<float, VE> d;
        if (col < a.width) d.load(a.partial + (size_t)slot * a.width + col);
        else d.zero();
#pragma unroll
        for (int v = 0; v < VE; ++v) acc[v] += d.el[v];
    };
    unsigned row = 0, last = 0, slot = 0;
    bool many = false;
    if (c + 1 < a.ranges) {  // the last range's row ends there
        const unsigned c0 = c * a.range, c1 = c0 + a.range;
        row = __ldg(a.key + c1 - 1);
        const bool before = c0 && __ldg(a.key + c0 - 1) == row;
        if (row < (unsigned)a.rows && !before && __ldg(a.key + c1) == row) {
            slot = 2 * c + 1;  // the row begins in this range
            // its last range, by growing strides of ranges and then a search
            unsigned lo = c + 1, step = 1;  // range lo has an entry of the row
            while (lo + step < a.ranges && __ldg(a.key + (lo + step) * a.range) == row) {
                lo += step;
                step *= 2;
            }
            for (; step; step >>= 1)
                if (lo + step < a.ranges && __ldg(a.key + (lo + step) * a.range) == row) lo += step;
            last = lo;
            many = last - c > JOIN_WARP;
            if (!many) {
                float acc[VE] = {};
                add(slot, acc);
#pragma unroll 4
                for (unsigned r = c + 1; r <= last; ++r) add(2 * r, acc);
                if (col < a.width) store_row<VE>(a.dtable + (size_t)row * a.width + col, acc);
            }
        }
    }
    if (!__syncthreads_or(many)) return;
    if (lane == 0) {
        first_of[w] = many ? c : 0xffffffffu;
        last_of[w] = last;
    }
    __syncthreads();
    for (int k = 0; k < LG_WARPS; ++k) {
        const unsigned first = first_of[k], end = last_of[k];
        if (first == 0xffffffffu) continue;
        float acc[VE] = {};
        if (w == 0) add(2 * first + 1, acc);
#pragma unroll 8
        for (unsigned r = first + 1 + w; r <= end; r += LG_WARPS) add(2 * r, acc);
#pragma unroll
        for (int v = 0; v < VE; ++v) part[w][lane * VE + v] = acc[v];
        __syncthreads();
        if (w == 0 && col < a.width) {
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                float t = 0.0f;
                for (int o = 0; o < LG_WARPS; ++o) t += part[o][lane * VE + v];
                acc[v] = t;
            }
            const unsigned at = __ldg(a.key + (first + 1) * a.range);
            store_row<VE>(a.dtable + (size_t)at * a.width + col, acc);
        }
        __syncthreads();
    }
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
    unsigned tiles, range, ranges;
    int bits, passes, rounds;
};

GradPlan grad_plan(long long rows, long long n, int width) {
    GradPlan g{};
    // A wave of two blocks a multiprocessor takes as long as R + 4 rounds (about 0.9 us each): the tile for which the waves
    // that n takes are over first (2.56M entries: 9 rounds 108 us, 8 rounds 115; 1.28M: 62 and 73; 40k: 2 rounds 26, 8 rounds 38)
    long long least = 0;
    for (int r = 2; r <= RS_MAX_ROUNDS; ++r) {
        const long long tiles = (n + RS_THREADS * r - 1) / (RS_THREADS * r), time = (tiles + 2 * SMS - 1) / (2 * SMS) * (r + 4);
        if (r > 2 && time > least) continue;
        least = time;
        g.rounds = r;
        g.tiles = (unsigned)tiles;
    }
    // ranges of 256 entries, shorter where that leaves multiprocessors without a warp
    g.range = 256;
    const long long col_tiles = (width + 255) / 256;
    while (g.range > 32 && (n + g.range - 1) / g.range * col_tiles < 16ll * SMS) g.range /= 2;
    g.ranges = (unsigned)((n + g.range - 1) / g.range);
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
    if (n > RS_SMALL) {
        for (int b = 0; b < 2; ++b) g.entries[b] = take(b < g.passes - 1 ? 8 * n : 0);
        g.hist = take((4ll << (g.bits + g.passes - 1) / g.passes) * g.tiles);
        g.total = take(4ll * RS_BINS);
    }
    g.partial = take(g.ranges > 1 ? 8ll * g.ranges * width : 0);
    g.bytes = at;
    return g;
}

template <int R = RS_MAX_ROUNDS, class F>
void with_rounds(int rounds, F f) {
    if constexpr (R > 2)
        if (rounds < R) return with_rounds<R - 1>(rounds, f);
    f(std::integral_constant<int, R>{});
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
    if (in->n <= RS_SMALL) {
        const int e = allow_shared_memory<sort_small_kernel>("flare_lookup_backward");
        if (e) return e;
        s.tiles = 1;
        while (s.tiles < RS_SMALL_BLOCKS && (long long)s.tiles * RS_SMALL_THREADS < in->n) s.tiles *= 2;
        while (((long long)s.tiles * RS_SMALL_THREADS << s.bits) < in->n) ++s.bits;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = s.tiles;
        cfg.blockDim = RS_SMALL_THREADS;
        cfg.dynamicSmemBytes = (size_t)((RS_SMALL_THREADS << s.bits) * 6 + RS_SMALL_WARPS * 2 * (1 << RS_SMALL_BITS));
        cfg.stream = st;
        cudaLaunchAttribute cluster{};
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = s.tiles;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        cfg.attrs = &cluster;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, sort_small_kernel, s);
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
            with_rounds(g.rounds, [&](auto rounds) {
                sort_count_kernel<decltype(rounds)::value><<<g.tiles, RS_THREADS, 0, st>>>(s);
                sort_scan_kernel<<<1u << s.bits, RS_THREADS, 0, st>>>(s);
                sort_scatter_kernel<decltype(rounds)::value><<<g.tiles, RS_THREADS, smem, st>>>(s);
            });
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
        case 4: f(Width<4>{}); break;
        case 2: f(Width<2>{}); break;
        default: f(Width<1>{}); break;
    }
}

template <int VE>
void launch_join(const GradArgs &a, cudaStream_t st) {
    if (a.ranges > 1)
        grad_join_kernel<VE><<<dim3((a.ranges + LG_WARPS - 1) / LG_WARPS, (a.width / VE + 31) / 32), LG_THREADS, 0, st>>>(a);
}

template <class D, class T, int G, bool DOT>
int launch_ring(GradArgs a, cudaStream_t st) {
    using Piece = RingPiece<D, T, DOT>;
    constexpr int GROUPS = 32 * RING_WARPS / G;
    a.pieces = std::min(G, a.width / Piece::VE);
    a.tiles = (a.width + G * Piece::VE - 1) / (G * Piece::VE);
    a.work_blocks = (unsigned)(((long long)a.ranges * a.tiles + GROUPS - 1) / GROUPS);
    a.empty_rows = empty_rows(a.rows);
    const unsigned empty_blocks = (unsigned)((a.rows + a.empty_rows * RING_WARPS - 1) / (a.empty_rows * RING_WARPS));
    const int e = allow_shared_memory<grad_ring_kernel<D, T, G, DOT>>("flare_lookup_backward");
    if (e) return e;
    grad_ring_kernel<D, T, G, DOT><<<a.work_blocks + empty_blocks, 32 * RING_WARPS, GROUPS * RING_STAGES * Piece::bytes(a.pieces), st>>>(a);
    launch_join<Piece::VE>(a, st);
    return FLARE_OK;
}

template <class D, class T, bool DOT>
int launch_ring(const GradArgs &a, cudaStream_t st) {
    const int pieces = a.width * (int)sizeof(D) / 16;
    if (pieces <= 8) return launch_ring<D, T, 8, DOT>(a, st);
    if (pieces <= 16) return launch_ring<D, T, 16, DOT>(a, st);
    return launch_ring<D, T, 32, DOT>(a, st);
}

template <class D, int VE, int NQ, int G>
void launch_plain(GradArgs a, cudaStream_t st) {
    a.tiles = (a.width + G * VE * NQ - 1) / (G * VE * NQ);
    const unsigned per_block = LG_THREADS / G;
    a.work_blocks = (unsigned)(((long long)a.ranges * a.tiles + per_block - 1) / per_block);
    a.empty_rows = empty_rows(a.rows);
    const unsigned empty_blocks = (unsigned)((a.rows + a.empty_rows * LG_WARPS - 1) / (a.empty_rows * LG_WARPS));
    grad_plain_kernel<D, VE, NQ, G><<<a.work_blocks + empty_blocks, LG_THREADS, 0, st>>>(a);
    launch_join<VE>(a, st);
}

// widest vectors, up to 4 elements, that dout and dtable allow (or, without dtable, dout and table)
int grad_vec(const flare_lookup_grad_args *in, bool dtable) {
    int ve = 4;
    while (ve > 1 && !(in->width % ve == 0 && fits_vec(in->dout, in->dout_stride, type_size(in->dout_type), ve) &&
                       (dtable ? fits_vec(in->dtable, in->width, 4, ve)
                               : fits_vec(in->table, in->table_stride, type_size(in->table_type), ve))))
        ve >>= 1;
    return ve;
}

// whether 16-byte copies fit a matrix's rows
bool fits_copies(const void *p, long long stride, int width, int type) {
    const int per = 16 / type_size(type);
    return width % per == 0 && stride % per == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
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
    // rows of at least 64 bytes that 16-byte copies fit pass through the ring, both gradients at once where a row is one tile
    const bool ring = sums && in->width * type_size(in->dout_type) >= 64 &&
                      fits_copies(in->dout, in->dout_stride, in->width, in->dout_type) && fits_copies(in->dtable, in->width, in->width, FLARE_F32);
    const int per_piece = 16 / type_size(in->dout_type);  // columns of a lane
    const bool dot = ring && in->dweight && in->width <= 32 * per_piece &&
                     fits_vec(in->table, in->table_stride, type_size(in->table_type), per_piece);
    if (sums) {
        const GradPlan g = grad_plan(in->rows, in->n, in->width);
        char *ws = static_cast<char *>(in->workspace);
        int e = sort_entries(in, g, dot, st);
        if (e) return e;
        a.key = reinterpret_cast<unsigned *>(ws + g.key);
        a.order = reinterpret_cast<unsigned *>(ws + g.val);
        a.partial = reinterpret_cast<float *>(ws + g.partial);
        a.range = g.range;
        a.ranges = g.ranges;
        e = with_type(in->dout_type, [&](auto d) {
            using D = typename decltype(d)::type;
            if (dot)
                return with_type(in->table_type, [&](auto t) {
                    using T = typename decltype(t)::type;
                    return launch_ring<D, T, true>(a, st);
                });
            if (ring) return launch_ring<D, float, false>(a, st);
            const int ve = grad_vec(in, true);
            with_width(ve, [&](auto w) {
                constexpr int VE = decltype(w)::value;
                if (in->width / VE <= 8) launch_plain<D, VE, 1, 8>(a, st);
                else if (in->width / VE <= 32) launch_plain<D, VE, 1, 32>(a, st);
                else launch_plain<D, VE, 4, 32>(a, st);
            });
            return FLARE_OK;
        });
        if (e) return e;
        OPS_LAUNCHED("flare_lookup_backward");
    }
    if (in->dweight && !dot) {
        const unsigned blocks = (unsigned)std::min<long long>((in->n + 7) / 8, SMS * 64);
        with_type(in->dout_type, [&](auto d) {
            return with_type(in->table_type, [&](auto t) {
                with_width(grad_vec(in, false), [&](auto ve) {
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
    OPS_CHECK(a->rows < 0x7fffffffll && a->n < 0x80000000ll - 8192, "flare_lookup_backward: %lld rows, %lld entries",
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
