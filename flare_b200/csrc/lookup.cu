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
// Per digit: count per tile, scan over tiles, scatter.  A tile is 4096 consecutive entries of one block; warp w
// ranks entries [512 w, 512 w + 512) of it 32 at a time, so ranks follow the entries' order.
// ------------------------------------------------------------------------------------------------
constexpr int RS_THREADS = 256, RS_WARPS = RS_THREADS / 32, RS_ROUNDS = 16, RS_TILE = RS_THREADS * RS_ROUNDS;
constexpr int RS_MAX_BITS = 8, RS_BINS = 1 << RS_MAX_BITS;

struct SortArgs {
    const void *index;              // first pass: keys come from the index, values are the entry numbers
    const unsigned *key_in, *val_in;
    unsigned *key_out, *val_out, *hist;  // hist: digit-major (bins, tiles)
    unsigned *total;                // per digit
    long long rows;
    unsigned n, tiles;
    int shift, bits, index_type, first;
};

__device__ __forceinline__ unsigned sort_key(const SortArgs &a, unsigned i) {
    if (!a.first) return a.key_in[i];
    const long long p = a.index_type == FLARE_I64 ? row_of<long long>(a.index, i, a.rows) : row_of<int>(a.index, i, a.rows);
    return p < 0 ? (unsigned)a.rows : (unsigned)p;
}

__global__ void __launch_bounds__(RS_THREADS) sort_count_kernel(const SortArgs a) {
    __shared__ unsigned h[RS_BINS];
    const unsigned mask = (1u << a.bits) - 1u;
    h[threadIdx.x] = 0;
    __syncthreads();
    const unsigned base = blockIdx.x * RS_TILE;
#pragma unroll 4
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const unsigned i = base + r * RS_THREADS + threadIdx.x;
        if (i < a.n) atomicAdd(&h[(sort_key(a, i) >> a.shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x <= mask) a.hist[(size_t)threadIdx.x * a.tiles + blockIdx.x] = h[threadIdx.x];
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
    for (int k = 0; k < (int)(blockDim.x >> 5); ++k) {
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

__global__ void __launch_bounds__(RS_THREADS) sort_scatter_kernel(const SortArgs a) {
    __shared__ unsigned cnt[RS_WARPS][RS_BINS];
    __shared__ unsigned sums[RS_WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const unsigned mask = (1u << a.bits) - 1u;
    for (int k = 0; k < RS_WARPS; ++k) cnt[k][threadIdx.x] = 0;
    __syncthreads();
    const unsigned base = blockIdx.x * RS_TILE + w * (32 * RS_ROUNDS) + lane;
    unsigned key[RS_ROUNDS], val[RS_ROUNDS], rank[RS_ROUNDS];
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const unsigned i = base + r * 32;
        key[r] = i < a.n ? sort_key(a, i) : 0u;
        val[r] = i < a.n ? (a.first ? i : a.val_in[i]) : 0u;
    }
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        const bool in = base + r * 32 < a.n;
        const unsigned d = in ? (key[r] >> a.shift) & mask : RS_BINS;  // lanes past the end match one another only
        const unsigned same = __match_any_sync(0xffffffffu, d);
        const unsigned below = __popc(same & ((1u << lane) - 1u));
        const unsigned before = in ? cnt[w][d] : 0u;
        rank[r] = before + below;
        __syncwarp();
        if (in && below == 0) cnt[w][d] = before + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    {   // counts become first positions: digits before this one, tiles before this one, warps before this one
        unsigned all;
        const unsigned d = threadIdx.x;
        const unsigned digit = block_exclusive(d <= mask ? a.total[d] : 0u, sums, &all);
        if (d <= mask) {
            unsigned at = digit + a.hist[(size_t)d * a.tiles + blockIdx.x];
            for (int k = 0; k < RS_WARPS; ++k) {
                const unsigned c = cnt[k][d];
                cnt[k][d] = at;
                at += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; ++r) {
        if (base + r * 32 >= a.n) continue;
        const unsigned pos = cnt[w][(key[r] >> a.shift) & mask] + rank[r];
        a.key_out[pos] = key[r];
        a.val_out[pos] = val[r];
    }
}

// ------------------------------------------------------------------------------------------------
// Sums per row.  A row whose entries fill a whole aligned chunk of LG_CHUNK sorted entries is "long": its chunks are
// summed by blocks of their own into partial rows, and the partial rows are added in order; all others are added
// by a group of lanes.
// ------------------------------------------------------------------------------------------------
constexpr int LG_THREADS = 256, LG_CHUNK = 256;

struct GradArgs {
    const void *dout, *table, *index;
    const float *weight;
    float *dtable, *dweight, *partial;  // partial: (2 * chunks, width)
    const unsigned *key, *order;
    long long rows, dout_stride, table_stride;
    unsigned n;
    int width, index_type;
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

// acc += sum over sorted entries [s, e) of scale * weight * dout, columns col0 + (lane-owned vectors)
template <class D, int VE, int NV>
__device__ __forceinline__ void add_entries(const GradArgs &a, unsigned s, unsigned e, unsigned step, int col, int col_step,
                                            float (&acc)[NV][VE]) {
    constexpr int U = 4;  // entries in flight
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
        for (int u = 0; u < U; ++u)
            if (i[u] != 0xffffffffu)
#pragma unroll
                for (int q = 0; q < NV; ++q)
#pragma unroll
                    for (int v = 0; v < VE; ++v) acc[q][v] = fmaf(f[u], d[u][q].get(v), acc[q][v]);
    }
}

template <int VE>
__device__ __forceinline__ void store_row(float *p, const float (&acc)[VE]) {
    Vec<float, VE> o;
#pragma unroll
    for (int v = 0; v < VE; ++v) o.el[v] = acc[v];
    o.store(p);
}

// Block c: the part of the rows at chunk c's ends that are long -> partial rows 2c (the row that the chunk begins
// with) and 2c + 1 (the row that begins inside it).  grid.y: column tiles of 32 VE.
template <class D, int VE>
__global__ void __launch_bounds__(LG_THREADS) grad_chunk_kernel(const GradArgs a) {
    constexpr int W = LG_THREADS / 32;
    __shared__ float part[W][32 * VE];
    const unsigned c0 = blockIdx.x * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n);
    const unsigned first = __ldg(a.key + c0), last = __ldg(a.key + c1 - 1);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = (blockIdx.y * 32 + lane) * VE;
    for (int side = 0; side < 2; ++side) {
        const unsigned row = side ? last : first;
        if (side && last == first) break;
        if (row >= (unsigned)a.rows) break;  // entries without a row
        // the keys are sorted, so equal keys at both ends of a chunk mean that all of it is this row
        bool lng;
        if (side == 0)
            lng = (c0 + LG_CHUNK <= a.n && last == first) || (c0 >= LG_CHUNK && __ldg(a.key + c0 - LG_CHUNK) == first);
        else lng = c1 + LG_CHUNK <= a.n && __ldg(a.key + c1 + LG_CHUNK - 1) == last;
        if (!lng) continue;
        unsigned s = c0, e = c1;
        if (first != last) {
            const unsigned cut = c0 + lower_bound(a.key + c0, c1 - c0, side ? last : first + 1);
            if (side) s = cut;
            else e = cut;
        }
        float acc[1][VE] = {};
        add_entries<D, VE, 1>(a, s + w, e, W, col, 0, acc);
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VE; ++v) part[w][lane * VE + v] = acc[0][v];
        __syncthreads();
        if (w == 0 && col < a.width) {
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                float t = 0.0f;
                for (int k = 0; k < W; ++k) t += part[k][lane * VE + v];
                acc[0][v] = t;
            }
            store_row<VE>(a.partial + ((size_t)2 * blockIdx.x + side) * a.width + col, acc[0]);
        }
        __syncthreads();
    }
}

// Block c: if a long row begins in chunk c, adds its partial rows in order and writes the row.
template <int VE>
__global__ void __launch_bounds__(LG_THREADS) grad_join_kernel(const GradArgs a) {
    constexpr int W = LG_THREADS / 32;
    __shared__ float part[W][32 * VE];
    const unsigned c0 = blockIdx.x * LG_CHUNK, c1 = min(c0 + LG_CHUNK, a.n);
    const unsigned row = __ldg(a.key + c1 - 1);  // the only row that can begin here and be long
    if (row >= (unsigned)a.rows) return;
    const unsigned s = lower_bound(a.key, a.n, row);
    if (s < c0) return;  // it began before
    const unsigned e = lower_bound(a.key, a.n, row + 1);
    if (!is_long(s, e)) return;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = (blockIdx.y * 32 + lane) * VE;
    const unsigned last = (e - 1) / LG_CHUNK;
    float acc[VE] = {};
    if (col < a.width) {
#pragma unroll 4
        for (unsigned c = blockIdx.x + w; c <= last; c += W) {
            // the row's part of its first chunk is side 1 unless the chunk begins with it
            const unsigned slot = 2 * c + (c == blockIdx.x && s != c0 ? 1 : 0);
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
            for (int k = 0; k < W; ++k) t += part[k][lane * VE + v];
            acc[v] = t;
        }
        store_row<VE>(a.dtable + (size_t)row * a.width + col, acc);
    }
}

// A group of G lanes per row (32 / G rows per warp), each lane NV vectors of VE columns per column tile.
template <class D, int VE, int NV, int G>
__global__ void __launch_bounds__(LG_THREADS) grad_rows_kernel(const GradArgs a) {
    constexpr int RPW = 32 / G;
    const int lane = threadIdx.x & 31, sub = lane % G;
    const long long warp = ((long long)blockIdx.x * LG_THREADS + threadIdx.x) >> 5;
    // the warp's 32 rows: lane k finds where row 32 warp + k begins
    const long long row0 = warp * 32;
    if (row0 >= a.rows) return;
    const unsigned begin = lower_bound(a.key, a.n, (unsigned)min(row0 + lane, a.rows));
    const unsigned end31 = lower_bound(a.key, a.n, (unsigned)min(row0 + 32, a.rows));
    for (int r = 0; r < 32; r += RPW) {
        const int k = r + lane / G;
        const unsigned s = __shfl_sync(0xffffffffu, begin, k);
        const unsigned nxt = __shfl_sync(0xffffffffu, begin, (k + 1) & 31);
        const unsigned e = k == 31 ? end31 : nxt;
        const long long row = row0 + k;
        if (row >= a.rows || is_long(s, e)) continue;
        for (int c0 = 0; c0 < a.width; c0 += G * NV * VE) {
            float acc[NV][VE] = {};
            add_entries<D, VE, NV>(a, s, e, 1, c0 + sub * VE, G * VE, acc);
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const int c = c0 + sub * VE + q * G * VE;
                if (c < a.width) store_row<VE>(a.dtable + row * a.width + c, acc[q]);
            }
        }
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
    long long key[2], val[2], hist, total, partial, bytes;
    unsigned tiles, chunks;
};

GradPlan grad_plan(long long n, int width) {
    GradPlan g{};
    g.tiles = (unsigned)((n + RS_TILE - 1) / RS_TILE);
    g.chunks = (unsigned)((n + LG_CHUNK - 1) / LG_CHUNK);
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long p = at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    for (int b = 0; b < 2; ++b) g.key[b] = take(4 * n);
    for (int b = 0; b < 2; ++b) g.val[b] = take(4 * n);
    g.hist = take(4ll * RS_BINS * g.tiles);
    g.total = take(4ll * RS_BINS);
    // only rows that fill a chunk have partial rows
    g.partial = take(n >= LG_CHUNK ? 8ll * g.chunks * width : 0);
    g.bytes = at;
    return g;
}

template <class D>
void launch_grad(const GradArgs &a, int ve, unsigned chunks, cudaStream_t st) {
    auto go = [&](auto tag) {
        constexpr int VE = decltype(tag)::value;
        const int vectors = a.width / VE;
        if (a.n >= LG_CHUNK) {
            const dim3 grid(chunks, (vectors + 31) / 32);
            grad_chunk_kernel<D, VE><<<grid, LG_THREADS, 0, st>>>(a);
        }
        const unsigned blocks = (unsigned)((a.rows + 32 * (LG_THREADS / 32) - 1) / (32 * (LG_THREADS / 32)));
        if (vectors <= 4) grad_rows_kernel<D, VE, 1, 4><<<blocks, LG_THREADS, 0, st>>>(a);
        else if (vectors <= 8) grad_rows_kernel<D, VE, 1, 8><<<blocks, LG_THREADS, 0, st>>>(a);
        else if (vectors <= 16) grad_rows_kernel<D, VE, 1, 16><<<blocks, LG_THREADS, 0, st>>>(a);
        else if (vectors <= 32) grad_rows_kernel<D, VE, 1, 32><<<blocks, LG_THREADS, 0, st>>>(a);
        else grad_rows_kernel<D, VE, 4, 32><<<blocks, LG_THREADS, 0, st>>>(a);
        if (a.n >= LG_CHUNK) {
            const dim3 grid(chunks, (vectors + 31) / 32);
            grad_join_kernel<VE><<<grid, LG_THREADS, 0, st>>>(a);
        }
    };
    switch (ve) {
        case 8: go(std::integral_constant<int, 8>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 2: go(std::integral_constant<int, 2>{}); break;
        default: go(std::integral_constant<int, 1>{}); break;
    }
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
    if (in->dtable && in->rows) {
        const GradPlan g = grad_plan(in->n, in->width);
        char *ws = static_cast<char *>(in->workspace);
        SortArgs s{};
        s.index = in->index;
        s.index_type = in->index_type;
        s.hist = reinterpret_cast<unsigned *>(ws + g.hist);
        s.total = reinterpret_cast<unsigned *>(ws + g.total);
        s.rows = in->rows;
        s.n = a.n;
        s.tiles = g.tiles;
        int bits = 1;
        while ((in->rows >> bits) != 0) ++bits;  // keys are 0 .. rows
        const int passes = (bits + RS_MAX_BITS - 1) / RS_MAX_BITS;
        for (int p = 0, shift = 0; p < passes; ++p) {
            s.first = p == 0;
            s.shift = shift;
            s.bits = (bits - shift + (passes - p) - 1) / (passes - p);
            s.key_in = reinterpret_cast<unsigned *>(ws + g.key[(p + 1) & 1]);
            s.val_in = reinterpret_cast<unsigned *>(ws + g.val[(p + 1) & 1]);
            s.key_out = reinterpret_cast<unsigned *>(ws + g.key[p & 1]);
            s.val_out = reinterpret_cast<unsigned *>(ws + g.val[p & 1]);
            sort_count_kernel<<<g.tiles, RS_THREADS, 0, st>>>(s);
            sort_scan_kernel<<<1u << s.bits, RS_THREADS, 0, st>>>(s);
            sort_scatter_kernel<<<g.tiles, RS_THREADS, 0, st>>>(s);
            OPS_LAUNCHED("flare_lookup_backward");
            shift += s.bits;
        }
        a.key = s.key_out;
        a.order = s.val_out;
        a.partial = reinterpret_cast<float *>(ws + g.partial);
        int ve = 8;
        while (ve > 1 && !(in->width % ve == 0 && fits_vec(in->dout, in->dout_stride, type_size(in->dout_type), ve) &&
                           fits_vec(in->dtable, in->width, 4, ve)))
            ve >>= 1;
        with_type(in->dout_type, [&](auto d) {
            launch_grad<typename decltype(d)::type>(a, ve, g.chunks, st);
            return 0;
        });
        OPS_LAUNCHED("flare_lookup_backward");
    }
    if (in->dweight) {
        int ve = 8;
        while (ve > 1 && !(in->width % ve == 0 && fits_vec(in->dout, in->dout_stride, type_size(in->dout_type), ve) &&
                           fits_vec(in->table, in->table_stride, type_size(in->table_type), ve)))
            ve >>= 1;
        const unsigned blocks = (unsigned)std::min<long long>((in->n + 7) / 8, SMS * 64);
        with_type(in->dout_type, [&](auto d) {
            return with_type(in->table_type, [&](auto t) {
                using D = typename decltype(d)::type;
                using T = typename decltype(t)::type;
                switch (ve) {
                    case 8: grad_weight_kernel<D, T, 8><<<blocks, LG_THREADS, 0, st>>>(a); break;
                    case 4: grad_weight_kernel<D, T, 4><<<blocks, LG_THREADS, 0, st>>>(a); break;
                    case 2: grad_weight_kernel<D, T, 2><<<blocks, LG_THREADS, 0, st>>>(a); break;
                    default: grad_weight_kernel<D, T, 1><<<blocks, LG_THREADS, 0, st>>>(a); break;
                }
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
    return rows > 0 && n > 0 && width > 0 ? grad_plan(n, width).bytes : 0;
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
