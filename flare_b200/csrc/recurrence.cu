// recurrence.cu -- the gated linear recurrence h_t = a_t h_{t-1} + x_t over many sequences, and its gradient.
//
// A stretch of steps maps the state that enters it to A h + H (A the product of its gates, H what it yields from 0), and
// two stretches join to (A2 A1, A2 H1 + H2), so a sequence can be cut in time:
//   * a thread holds SPAN = 16 steps of VE neighbouring channels in registers, all loaded before the first is used;
//   * the W warps of a tile take W consecutive spans, pass the state through their (A, H) in shared memory and run their own
//     span again from the state that enters it (from registers: every input is read once);
//   * with few channels and many steps, S blocks share a sequence: a first kernel writes each block's (A, H), the
//     second folds the ones before its own (the inputs are then read twice, the second time mostly from L2).
// The fold's order is fixed by the sizes alone, so results repeat bit for bit.
//
// The gradient runs the same scheme from the last step: mu = a_t lambda_t is what step t hands to step t - 1, lambda_t =
// dh_t + mu_{t+1}, dx_t = lambda_t, da_t = lambda_t h_{t-1}.  h_{t-1} is formed again in 32 bits from x and the state saved
// before every span (1/16 of a float per element), not read from rounded outputs.
// Bound by memory: gate, x (dh) in, h (dx, dgate) out.  State, products and sums are 32-bit floats.
#include <algorithm>
#include <cstdlib>

#include "ops.cuh"

namespace flare {

constexpr int SPAN = FLARE_RECURRENCE_SPAN;
static_assert(SPAN == 16, "shifts by 4");
constexpr int WARPS = 8;         // warps per block: W along time times WARPS / W tiles of channels
constexpr int MAX_SPLITS = 128;  // blocks along time

struct RecArgs {
    const void *gate, *x, *dh, *offsets;
    const float *state, *dlast;
    void *h, *dgate, *dx;
    float *last, *saved, *dstate;
    float *agg;      // (splits, 2, seqs * width)
    float *partial;  // (parts, rows, groups): sums over parts of a group's channels
    long long seqs, rows;
    long long gate_s, x_s, h_s, dh_s, dgate_s, dx_s;   // elements
    int gate_t, x_t, h_t, dh_t, dgate_t, dx_t;         // elements; less than 2^31 bytes
    int steps, width, groups;
    FastDiv share;             // channels per gate
    int off64, reverse, packed;
    int wlog, splits, per;     // log2 W; dense: steps per split
    unsigned tiles, units;     // units: lanes' worth of channels, seqs * width / VE
    FastDiv upr;               // units per sequence
    int group_units, groups_per_tile, parts;  // backward tiles of whole groups, see Place
    FastDiv gunits, fparts;    // by group_units and parts
    int spans;                 // dense: spans per sequence
};

__device__ __forceinline__ int offset_at(const RecArgs &a, long long s) {
    const long long o = a.off64 ? __ldg(static_cast<const long long *>(a.offsets) + s) : (long long)__ldg(static_cast<const int *>(a.offsets) + s);
    return (int)min(max(o, 0ll), (long long)a.steps);
}

// Where a lane's channels lie.  LANES > 0: tiles of LANES lanes consist of whole groups of channels that share a gate, or of
// a part of one such group, so that sums over a group need no other tile.
template <int VE, int LANES>
struct Place {
    bool active;
    int seq, row0, len;  // row0: the sequence's first row (packed), len: its steps
    int c;               // first channel
    unsigned chain;      // seq * width + c
    int part;            // LANES: part of the group
    int group, member;   // LANES: group of the tile, place in it
    // lanes without channels of their own (!active) walk along with another's and store nothing
    __device__ __forceinline__ Place(const RecArgs &a, unsigned tile) {
        const int lane = threadIdx.x & ((LANES ? LANES : 32) - 1);
        unsigned u;
        part = group = 0;
        member = lane;
        if (!LANES) {
            u = tile * 32 + lane;
            active = u < a.units;
        } else if (a.parts == 1) {
            const unsigned g = a.gunits.div(lane);
            group = (int)g;
            member = lane - group * a.group_units;
            u = (tile * a.groups_per_tile + g) * a.group_units + member;
            active = (int)g < a.groups_per_tile && u < a.units;
            if ((int)g >= a.groups_per_tile) u = (tile * a.groups_per_tile + g) * a.group_units - 1;
        } else {
            const unsigned t = a.fparts.div(tile);
            part = tile - t * a.parts;
            const int pos = part * LANES + lane;
            u = t * a.group_units + min(pos, a.group_units - 1);
            active = pos < a.group_units;
        }
        const bool some = tile < a.tiles;
        active = active && some;
        u = some ? min(u, a.units - 1) : 0u;
        seq = (int)a.upr.div(u);
        c = (int)(u - seq * a.upr.d) * VE;
        chain = u * VE;
        row0 = 0;
        len = some ? a.steps : 0;
        if (a.packed && some) {
            row0 = offset_at(a, seq);
            len = max(offset_at(a, seq + 1) - row0, 0);
        }
    }
    // element offset of the first step's row in a tensor (the next step's is stride_t further on, or before if reversed)
    __device__ __forceinline__ long long first(const RecArgs &a, long long stride_s, int stride_t) const {
        const long long base = a.packed ? (long long)row0 * stride_t : seq * stride_s;
        return a.reverse ? base + (long long)(len - 1) * stride_t : base;
    }
    // row of `saved` that holds the state before span k >= 1
    __device__ __forceinline__ long long saved_row(const RecArgs &a, int k) const {
        return a.packed ? (long long)row0 / SPAN + seq + k : (long long)seq * (a.spans - 1) + k - 1;
    }
    // the steps that block `split` works on, in whole rounds of W spans
    __device__ __forceinline__ void range(const RecArgs &a, int split, int &t0, int &t1) const {
        t0 = 0;
        t1 = len;
        if (a.splits > 1) {
            unsigned per = a.per;
            if (a.packed) {
                const unsigned round = SPAN << a.wlog, rounds = ((unsigned)len + round - 1) / round;
                per = (rounds + a.splits - 1) / a.splits * round;
            }
            t0 = (int)min((long long)len, (long long)split * per);
            t1 = (int)min((long long)len, (long long)t0 + per);
        }
    }
};

// What a stretch (A, H) makes of the state c.  A state of exactly 0 adds nothing, also where the product of the gates
// has left the range of a float.
__device__ __forceinline__ float through(float A, float H, float c) { return c == 0.0f ? H : fmaf(A, c, H); }

// SPAN steps of N channels as they lie in memory, `step` elements apart.
template <class T, int N>
struct Span {
    Vec<T, N> d[SPAN];
    // FULL: all steps are there, else the ones past n are filled with `rest`.  KEEP: others read it again soon
    template <bool FULL, bool KEEP>
    __device__ __forceinline__ void load(const T *p, int step, int n, float rest) {
        const int bytes = step * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < SPAN; ++i) {
            const T *at = reinterpret_cast<const T *>(reinterpret_cast<const char *>(p) + (long long)bytes * i);
            if (!FULL && i >= n)
#pragma unroll
                for (int v = 0; v < N; ++v) d[i].set(v, rest);
            else if (KEEP) d[i].load(at);
            else d[i].load_stream(at);
        }
    }
    __device__ __forceinline__ float at(int i, int v) const { return d[i].get(N == 1 ? 0 : v); }
    // step i is unpacked to 32 bits here and not before, so that a span waits in its packed form
    __device__ __forceinline__ void hold(int i) {
        if constexpr (N * sizeof(T) == 2) asm volatile("" : "+h"(d[i].raw[0]));
        else if constexpr (N * sizeof(T) == 4) asm volatile("" : "+r"(d[i].raw[0]));
        else if constexpr (N * sizeof(T) == 8) asm volatile("" : "+r"(d[i].raw[0].x), "+r"(d[i].raw[0].y));
        else if constexpr (N * sizeof(T) == 16)
            asm volatile("" : "+r"(d[i].raw[0].x), "+r"(d[i].raw[0].y), "+r"(d[i].raw[0].z), "+r"(d[i].raw[0].w));
    }
};

// (A, H) of a span, walked from its first step (forward) or its last (backward, where H collects a_t dh_t)
template <bool BACK, class T, class GT, int VE, int GN>
__device__ __forceinline__ void stretch(const Span<GT, GN> &g, const Span<T, VE> &x, float (&A)[VE], float (&H)[VE]) {
#pragma unroll
    for (int v = 0; v < VE; ++v) {
        A[v] = 1.0f;
        H[v] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < SPAN; ++k) {
        const int i = BACK ? SPAN - 1 - k : k;
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            const float a = g.at(i, v);
            H[v] = BACK ? a * (H[v] + x.at(i, v)) : fmaf(a, H[v], x.at(i, v));
            A[v] *= a;
        }
    }
}

// barrier of the W warps that share a tile
__device__ __forceinline__ void tile_sync(int wlog) {
    const int id = 1 + (threadIdx.x >> (5 + wlog));
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(32 << wlog) : "memory");
}

// How the W warps of a tile pass the state along time.  Of a lane's VE channels thread (w, lane) looks after v = w, w + W, ...:
// it holds their state at the round's border and passes it through all W stretches, so that the walk over the warps is
// done once per channel and not once per warp (which took 2.5 of the 8 instructions an element took).
// BACK: warps are passed from the last to the first.
template <bool BACK, int VE>
struct Pass {
    static constexpr int MINE = (VE + 1) / 2;  // W > 1
    float *sa, *sh;                            // (W, VE, 32) each
    int wlog, w, lane;
    float carry[MINE];
    __device__ __forceinline__ Pass(float *smem, int wlog_) : wlog(wlog_), w((threadIdx.x >> 5) & ((1 << wlog_) - 1)), lane(threadIdx.x & 31) {
        sa = smem + ((threadIdx.x >> (5 + wlog)) << wlog) * (2 * VE * 32);
        sh = sa + (VE * 32 << wlog);
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {  // f(q, v) for the channels that this thread looks after
#pragma unroll
        for (int q = 0; q < MINE; ++q) {
            const int v = w + (q << wlog);
            if (v < VE) f(q, v);
        }
    }
    __device__ __forceinline__ void begin(const float *ends, unsigned chain) {
        each([&](int q, int v) { carry[q] = ends ? ends[chain + v] : 0.0f; });
    }
    __device__ __forceinline__ void finish(float *ends, unsigned chain) {
        each([&](int q, int v) { ends[chain + v] = carry[q]; });
    }
    // (A, H): this warp's stretch; in: the state that enters it.  prod (optional): times the product of all stretches' A
    __device__ __forceinline__ void run(const float (&A)[VE], const float (&H)[VE], float (&in)[VE], float *prod = nullptr) {
        const int W = 1 << wlog;
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            sa[(w * VE + v) * 32 + lane] = A[v];
            sh[(w * VE + v) * 32 + lane] = H[v];
        }
        tile_sync(wlog);
        each([&](int q, int v) {
            float c = carry[q];
#pragma unroll 4
            for (int k = 0; k < W; ++k) {
                const int at = ((BACK ? W - 1 - k : k) * VE + v) * 32 + lane;
                const float a = sa[at];
                sa[at] = c;
                c = through(a, sh[at], c);
                if (prod) prod[q] *= a;
            }
            carry[q] = c;
        });
        tile_sync(wlog);
#pragma unroll
        for (int v = 0; v < VE; ++v) in[v] = sa[(w * VE + v) * 32 + lane];
    }
};

// The state that enters block `split`: pass.carry through the blocks before it in the walk.  Each of the W warps joins a
// part of them, then the parts are passed in order.
template <bool BACK, int VE>
__device__ __forceinline__ void fold_splits(const RecArgs &a, unsigned chain, int split, Pass<BACK, VE> &pass) {
    const long long chains = a.seqs * a.width;
    const int W = 1 << a.wlog, w = pass.w;
    const int n = BACK ? a.splits - 1 - split : split;
    if (n == 0) return;
    // parts in the order of the walk: warp w (BACK: W - 1 - w) has the w-th
    const int k0 = n * (BACK ? W - 1 - w : w) / W, k1 = n * (BACK ? W - w : w + 1) / W;
    float A[VE], H[VE], unused[VE];
#pragma unroll
    for (int v = 0; v < VE; ++v) {
        A[v] = 1.0f;
        H[v] = 0.0f;
    }
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
        const float *p = a.agg + (long long)(BACK ? a.splits - 1 - k : k) * 2 * chains + chain;
        Vec<float, VE> pa, ph;
        pa.load(p);
        ph.load(p + chains);
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            H[v] = through(pa.get(v), ph.get(v), H[v]);
            A[v] *= pa.get(v);
        }
    }
    pass.run(A, H, unused);
}

// plain loads: `last` may be `state` and `dstate` may be `dlast`, each written by the lanes that have read it
template <int VE>
__device__ __forceinline__ void load_ends(const float *p, unsigned chain, bool some, float (&f)[VE]) {
    Vec<float, VE> v;
    if (p && some) v.load_plain(p + chain);
    else v.zero();
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = v.get(e);
}
template <int VE>
__device__ __forceinline__ void store_ends(float *p, const float (&f)[VE]) {
    Vec<float, VE> v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v.el[e] = f[e];
    v.store(p);
}

// zeros in the rows of a packed tensor that belong to no sequence, shared among all blocks
template <class T>
__device__ __forceinline__ void clear_rest(const RecArgs &a, void *out, long long stride, int width) {
    const int tail = offset_at(a, a.seqs), head = min(offset_at(a, 0), tail);
    const long long n = ((long long)head + a.steps - tail) * width;
    const long long block = blockIdx.y * (long long)gridDim.x + blockIdx.x, blocks = (long long)gridDim.x * gridDim.y;
    for (long long i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) {
        const long long r = i / width;
        static_cast<T *>(out)[(r < head ? r : tail + r - head) * stride + (i - r * width)] = from_f32<T>(0.0f);
    }
}

__device__ __forceinline__ unsigned my_tile(const RecArgs &a) {
    return blockIdx.x * (WARPS >> a.wlog) + (threadIdx.x >> (5 + a.wlog));
}
__device__ __forceinline__ int warp_max(int v) { return __reduce_max_sync(0xffffffffu, v); }

// BACK false: (A, H) of x; true: of dh, from the end.  grid (tiles, splits); W > 1
template <bool BACK, class T, class GT, int VE, bool SHARED>
__global__ void __launch_bounds__(32 * WARPS) recurrence_split_kernel(const RecArgs a) {
    extern __shared__ __align__(16) float smem[];
    const int W = 1 << a.wlog, w = (threadIdx.x >> 5) & (W - 1), split = blockIdx.y;
    const Place<VE, 0> me(a, my_tile(a));
    int t0, t1;
    me.range(a, split, t0, t1);
    Pass<BACK, VE> pass(smem, a.wlog);
    const int round = W * SPAN, n = (warp_max(t1 - t0) + round - 1) >> (4 + a.wlog);
    const T *src = static_cast<const T *>(BACK ? a.dh : a.x);
    const int src_t = BACK ? a.dh_t : a.x_t;
    const int gs = a.reverse ? -a.gate_t : a.gate_t, xs = a.reverse ? -src_t : src_t;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + a.share.div(me.c);
    const T *xp = src + me.first(a, BACK ? a.dh_s : a.x_s, src_t) + me.c;
    float A[VE], H[VE], unused[VE], prod[Pass<BACK, VE>::MINE];
    pass.begin(nullptr, 0);
#pragma unroll
    for (int q = 0; q < Pass<BACK, VE>::MINE; ++q) prod[q] = 1.0f;
    for (int k = 0; k < n; ++k) {
        const int t = t0 + (BACK ? n - 1 - k : k) * round + w * SPAN, left = t1 - t;
        Span<GT, SHARED ? 1 : VE> g;
        Span<T, VE> x;
        if (__all_sync(0xffffffffu, left >= SPAN) && src) {
            g.template load<true, true>(gp + (long long)t * gs, gs, 0, 1.0f);
            x.template load<true, true>(xp + (long long)t * xs, xs, 0, 0.0f);
        } else {
            g.template load<false, true>(gp + (long long)t * gs, gs, left, 1.0f);
            x.template load<false, true>(xp + (long long)t * xs, xs, src ? left : 0, 0.0f);
        }
        stretch<BACK>(g, x, A, H);
        pass.run(A, H, unused, prod);
    }
    if (me.active) {
        const long long chains = a.seqs * a.width;
        float *p = a.agg + (long long)split * 2 * chains;
        pass.each([&](int q, int v) { p[me.chain + v] = prod[q]; });
        pass.finish(p + chains, me.chain);
    }
}

template <class T, class GT, int VE, bool SHARED>
__global__ void __launch_bounds__(32 * WARPS) recurrence_forward_kernel(const RecArgs a) {
    extern __shared__ __align__(16) float smem[];
    const int W = 1 << a.wlog, w = (threadIdx.x >> 5) & (W - 1), split = blockIdx.y;
    const Place<VE, 0> me(a, my_tile(a));
    int t0, t1;
    me.range(a, split, t0, t1);
    Pass<false, VE> pass(smem, a.wlog);
    const int round = SPAN << a.wlog, n = (warp_max(t1 - t0) + round - 1) >> (4 + a.wlog);
    const int gs = a.reverse ? -a.gate_t : a.gate_t, xs = a.reverse ? -a.x_t : a.x_t, hs = a.reverse ? -a.h_t : a.h_t;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + a.share.div(me.c);
    const T *xp = static_cast<const T *>(a.x) + me.first(a, a.x_s, a.x_t) + me.c;
    T *hp = static_cast<T *>(a.h) + me.first(a, a.h_s, a.h_t) + me.c;
    float carry[VE], h[VE], A[VE], H[VE];
    if (W > 1) pass.begin(a.state, me.chain);
    else load_ends<VE>(a.state, me.chain, true, carry);
    if (a.splits > 1) fold_splits<false, VE>(a, me.chain, split, pass);
    // a span of which every lane has all steps needs no tests
    auto span = [&](auto full, int t, int left) {
        constexpr bool FULL = decltype(full)::value;
        Span<GT, SHARED ? 1 : VE> g;
        Span<T, VE> x;
        g.template load<FULL, SHARED>(gp + (long long)t * gs, gs, left, 1.0f);
        x.template load<FULL, false>(xp + (long long)t * xs, xs, left, 0.0f);
        if (W > 1) {
            stretch<false>(g, x, A, H);
            pass.run(A, H, h);
        } else {
#pragma unroll
            for (int v = 0; v < VE; ++v) h[v] = carry[v];
        }
        if (a.saved && me.active && left > 0 && t > 0) store_ends<VE>(a.saved + me.saved_row(a, t / SPAN) * a.width + me.c, h);
        if (a.h) {
            const int bytes = hs * (int)sizeof(T);
            char *p = reinterpret_cast<char *>(hp + (long long)t * hs);
#pragma unroll
            for (int i = 0; i < SPAN; ++i) {
                Vec<T, VE> o;
                x.hold(i);
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    h[v] = fmaf(g.at(i, v), h[v], x.at(i, v));
                    o.set(v, h[v]);
                }
                if (me.active && (FULL || i < left)) o.store_stream(reinterpret_cast<T *>(p + (long long)bytes * i));
            }
        } else {
#pragma unroll
            for (int i = 0; i < SPAN; ++i) {
                x.hold(i);
#pragma unroll
                for (int v = 0; v < VE; ++v) h[v] = fmaf(g.at(i, v), h[v], x.at(i, v));
            }
        }
        if (W == 1)
#pragma unroll
            for (int v = 0; v < VE; ++v) carry[v] = h[v];
    };
    for (int k = 0; k < n; ++k) {
        const int t = t0 + k * round + w * SPAN, left = t1 - t;
        if (__all_sync(0xffffffffu, left >= SPAN)) span(std::true_type{}, t, left);
        else span(std::false_type{}, t, left);
    }
    if (split == a.splits - 1 && me.active) {
        if (W > 1) pass.finish(a.last, me.chain);
        else store_ends<VE>(a.last + me.chain, carry);
    }
    if (a.packed && a.h) clear_rest<T>(a, a.h, a.h_t, a.width);
}

// smem: what the warps pass, then SHARED: 16 x 32 sums of products per warp, a lane's channels each.  The states before a span's
// steps stay in registers: in shared memory, for a third block per multiprocessor, 160k x 16 x 96 f16 took 15 % longer.
// DH: whether there is a gradient of every state, not of the last ones alone
// LANES: lanes of a tile of groups (0: a gate per channel)
template <class T, class GT, int VE, int LANES, bool DH>
__global__ void __launch_bounds__(32 * WARPS, 2) recurrence_backward_kernel(const RecArgs a) {
    extern __shared__ __align__(16) float smem[];
    const int W = 1 << a.wlog, w = (threadIdx.x >> 5) & (W - 1), split = blockIdx.y;
    constexpr bool SHARED = LANES > 0, BLOCK = LANES > 32;
    const Place<VE, LANES> me(a, BLOCK ? blockIdx.x : my_tile(a));
    int t0, t1;
    me.range(a, split, t0, t1);
    Pass<true, VE> pass(smem, a.wlog);
    // SHARED, several groups in a tile: where a group's sums of this span go and how many they are
    __shared__ char *group_at[SHARED ? 32 * WARPS : 1];
    __shared__ int group_steps[SHARED ? 32 * WARPS : 1], longest;
    constexpr int STRIDE = LANES + 1;  // of the sums' 16 rows, off the banks' 32
    const int lane = threadIdx.x & ((BLOCK ? LANES : 32) - 1), first_group = threadIdx.x - lane;
    float *sums = smem + (W > 1 ? 2 * WARPS * 32 * VE : 0) + (BLOCK ? 0 : (threadIdx.x >> 5) * (SPAN * STRIDE));
    int most = warp_max(t1 - t0);
    if (BLOCK && a.packed) {  // the block walks together
        if (threadIdx.x == 0) longest = 0;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) atomicMax(&longest, most);
        __syncthreads();
        most = longest;
    }
    const int round = SPAN << a.wlog, n = (most + round - 1) >> (4 + a.wlog);
    const int gc = (int)a.share.div(me.c);
    const int gs = a.reverse ? -a.gate_t : a.gate_t, xs = a.reverse ? -a.x_t : a.x_t;
    const int dhs = a.reverse ? -a.dh_t : a.dh_t, dxs = a.reverse ? -a.dx_t : a.dx_t, dgs = a.reverse ? -a.dgate_t : a.dgate_t;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + gc;
    const T *xp = static_cast<const T *>(a.x) + me.first(a, a.x_s, a.x_t) + me.c;
    const T *dhp = DH ? static_cast<const T *>(a.dh) + me.first(a, a.dh_s, a.dh_t) + me.c : nullptr;
    T *dxp = static_cast<T *>(a.dx) + me.first(a, a.dx_s, a.dx_t) + me.c;
    GT *dgp = static_cast<GT *>(a.dgate) + me.first(a, a.dgate_s, a.dgate_t) + gc;
    // SHARED: where the group's sums of step 0 go, and the next step's from there
    char *sum_at = reinterpret_cast<char *>(dgp);
    int sum_t = dgs * (int)sizeof(GT);
    if (SHARED && a.parts > 1) {
        const long long row = (a.packed ? me.row0 : (long long)me.seq * a.steps) + (a.reverse ? me.len - 1 : 0);
        sum_at = reinterpret_cast<char *>(a.partial + (me.part * a.rows + row) * a.groups + gc);
        sum_t = (a.reverse ? -4 : 4) * a.groups;
    }
    float carry[VE], mu[VE], A[VE], H[VE];
    if (W > 1) pass.begin(a.dlast, me.chain);
    else load_ends<VE>(a.dlast, me.chain, true, carry);
    if (a.splits > 1) fold_splits<true, VE>(a, me.chain, split, pass);
    auto span = [&](auto full, int t, int left) {
        constexpr bool FULL = decltype(full)::value;
        Span<GT, SHARED ? 1 : VE> g;
        Span<T, VE> x, dh;
        g.template load<FULL, SHARED>(gp + (long long)t * gs, gs, left, 1.0f);
        if (DH) dh.template load<FULL, false>(dhp + (long long)t * dhs, dhs, left, 0.0f);
        x.template load<FULL, false>(xp + (long long)t * xs, xs, left, 0.0f);
        float before[SPAN][VE];  // the state before each step
        if (t > 0) load_ends<VE>(a.saved + me.saved_row(a, t / SPAN) * a.width, me.c, left > 0, before[0]);
        else load_ends<VE>(a.state, me.chain, left > 0, before[0]);
        if (W > 1) {
            if (!DH) dh.template load<false, false>(nullptr, 0, 0, 0.0f);
            stretch<true>(g, dh, A, H);
            pass.run(A, H, mu);
        } else {
#pragma unroll
            for (int v = 0; v < VE; ++v) mu[v] = carry[v];
        }
#pragma unroll
        for (int i = 0; i + 1 < SPAN; ++i) {
            x.hold(i);
#pragma unroll
            for (int v = 0; v < VE; ++v) before[i + 1][v] = fmaf(g.at(i, v), before[i][v], x.at(i, v));
        }
        const int dxb = dxs * (int)sizeof(T), dgb = dgs * (int)sizeof(GT);
        char *px = reinterpret_cast<char *>(dxp + (long long)t * dxs), *pg = reinterpret_cast<char *>(dgp + (long long)t * dgs);
#pragma unroll
        for (int i = SPAN - 1; i >= 0; --i) {
            Vec<T, VE> o;
            Vec<GT, SHARED ? 1 : VE> og;
            float sum = 0.0f;
            if (DH) dh.hold(i);
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                const float lambda = DH ? dh.at(i, v) + mu[v] : mu[v];
                o.set(v, lambda);
                if (SHARED) sum = fmaf(lambda, before[i][v], sum);
                else og.set(v, lambda * before[i][v]);
                mu[v] = g.at(i, v) * lambda;
            }
            const bool mine = me.active && (FULL || i < left);
            if (mine) o.store_stream(reinterpret_cast<T *>(px + (long long)dxb * i));
            if (SHARED) sums[i * STRIDE + lane] = sum;
            else if (mine) og.store_stream(reinterpret_cast<GT *>(pg + (long long)dgb * i));
        }
        if (W == 1)
#pragma unroll
            for (int v = 0; v < VE; ++v) carry[v] = mu[v];
    };
    for (int k = 0; k < n; ++k) {
        const int t = t0 + (n - 1 - k) * round + w * SPAN, left = t1 - t;
        if (__all_sync(0xffffffffu, left >= SPAN)) span(std::true_type{}, t, left);
        else span(std::false_type{}, t, left);
        if (SHARED) {
            // (step, group) sums over the group's lanes of this tile, in the lanes' order
            const bool one = a.groups_per_tile == 1;
            char *mine = sum_at + (long long)sum_t * t;
            if (!one && me.member == 0 && me.group < a.groups_per_tile) {
                group_at[first_group + me.group] = mine;
                group_steps[first_group + me.group] = me.active ? left : 0;
            }
            if (BLOCK) __syncthreads();
            else __syncwarp();
            const int units = min(a.group_units - me.part * LANES, LANES), outs = SPAN * a.groups_per_tile;
            for (int o = lane; o < outs; o += LANES) {
                const int i = o % SPAN, g = o / SPAN;
                if (i >= (one ? left : group_steps[first_group + g])) continue;
                const float *p = sums + i * STRIDE + g * a.group_units;
                float sum = 0.0f;
#pragma unroll 4
                for (int l = 0; l < units; ++l) sum += p[l];
                char *to = (one ? mine : group_at[first_group + g]) + (long long)sum_t * i;
                if (a.parts == 1) *reinterpret_cast<GT *>(to) = from_f32<GT>(sum);
                else *reinterpret_cast<float *>(to) = sum;
            }
            if (BLOCK) __syncthreads();
            else __syncwarp();
        }
    }
    if (a.dstate && split == 0 && me.active) {
        if (W > 1) pass.finish(a.dstate, me.chain);
        else store_ends<VE>(a.dstate + me.chain, carry);
    }
    if (a.packed) {
        clear_rest<T>(a, a.dx, a.dx_t, a.width);
        if (a.parts == 1) clear_rest<GT>(a, a.dgate, a.dgate_t, a.groups);
    }
}

// dgate from the partial sums of its parts, in order; zeros in rows of no sequence
template <class GT>
__global__ void recurrence_join_kernel(const RecArgs a) {
    const long long n = a.rows * a.groups;
    const int tail = a.packed ? offset_at(a, a.seqs) : a.steps, head = a.packed ? min(offset_at(a, 0), tail) : 0;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / a.groups, g = i - row * a.groups;
        const long long s = a.packed ? 0 : row / a.steps, at = a.packed ? row : row - s * a.steps;
        float t = 0.0f;
        if (!a.packed || (row >= head && row < tail))
            for (int p = 0; p < a.parts; ++p) t += a.partial[p * n + i];
        static_cast<GT *>(a.dgate)[s * a.dgate_s + at * a.dgate_t + g] = from_f32<GT>(t);
    }
}

// ------------------------------------------------------------------------------------------------

struct RecPlan {
    int ve, warps, splits, parts, group_units, groups_per_tile;
    bool shared, block;  // block: a tile is the block's 256 lanes, not a warp's
    long long tiles, rows, agg_bytes, ends_bytes, bytes;
};

// The ends that a call reads (state, or dlast), if it writes the new ones in their place.
const float *ends_in_place(const flare_recurrence_args *a, bool backward) {
    const float *in = backward ? a->dlast : a->state, *out = backward ? a->dstate : a->last;
    return a->seqs && in == out ? in : nullptr;
}

// Vectors of `ve` channels: whole within a group of channels that share a gate, aligned in every tensor.
bool vec_fits(const flare_recurrence_args *a, int ve, bool backward) {
    const int xs = type_size(a->x_type), gs = type_size(a->gate_type), share = a->width / a->groups;
    if (a->width % ve || (share > 1 && share % ve)) return false;
    auto ok = [&](const void *p, long long s, long long t, int size) {
        return !p || (fits_vec(p, t, size, ve) && (a->offsets || s % ve == 0));
    };
    if (!ok(a->x, a->x_s, a->x_t, xs)) return false;
    if (share == 1 && !ok(a->gate, a->gate_s, a->gate_t, gs)) return false;
    for (const void *p : {(const void *)a->state, (const void *)a->last, (const void *)a->saved, (const void *)a->dlast, (const void *)a->dstate})
        if (reinterpret_cast<uintptr_t>(p) % (4 * ve)) return false;
    if (!backward) return ok(a->h, a->h_s, a->h_t, xs);
    return ok(a->dh, a->dh_s, a->dh_t, xs) && ok(a->dx, a->dx_s, a->dx_t, xs) &&
           (share > 1 || ok(a->dgate, a->dgate_s, a->dgate_t, gs));
}

// channels per lane: the gradient holds x, dh, 32-bit states and gates of a span in 128 registers a thread
constexpr int widest_backward(bool f32, bool shared) { return (f32 ? 1 : 2) * (shared ? 2 : 1); }

RecPlan rec_plan(const flare_recurrence_args *a, bool backward) {
    RecPlan p{};
    const int share = a->width / a->groups;
    p.shared = share > 1;
    p.rows = a->offsets ? a->steps : a->seqs * a->steps;
    const long long chains = a->seqs * a->width;
    // the widest vectors that leave the machine enough warps
    // forward 16 bytes a lane where gates take no more than a register a step (160k x 16 x 96 f16: 90 us, with 8 bytes 125 us)
    const bool f32 = a->x_type == FLARE_F32;
    const int widest = backward ? widest_backward(f32, p.shared) : p.shared && !f32 ? 8 : 4;
    p.ve = widest;
    while (p.ve > 1 && (!vec_fits(a, p.ve, backward) || chains / p.ve < 32ll * 8 * SMS)) p.ve >>= 1;
    while (p.ve < 2 && a->x_type != FLARE_F32 && vec_fits(a, 2 * p.ve, backward)) p.ve *= 2;  // 4 bytes a lane at least
    // sums over a group stay within a warp where wider vectors allow it
    if (backward && p.shared)
        while (p.ve < widest && share / p.ve > 32 && vec_fits(a, 2 * p.ve, backward)) p.ve *= 2;
    p.group_units = p.parts = p.groups_per_tile = 1;
    p.tiles = (chains / p.ve + 31) / 32;
    auto group_tiles = [&](int lanes) {
        p.group_units = share / p.ve;
        p.parts = (p.group_units + lanes - 1) / lanes;
        p.groups_per_tile = p.parts > 1 ? 1 : lanes / p.group_units;
        const long long groups = a->seqs * a->groups;
        p.tiles = p.parts > 1 ? groups * p.parts : (groups + p.groups_per_tile - 1) / p.groups_per_tile;
    };
    if (backward && p.shared) group_tiles(32);
    // time is cut only as far as it takes to fill the machine: W spans at a time, then S blocks
    const long long mean = std::max<long long>(1, a->offsets ? a->steps / std::max<long long>(1, a->seqs) : a->steps);
    const long long spans = (mean + SPAN - 1) / SPAN;
    p.warps = 1;
    while (p.warps < WARPS && 2 * p.warps <= spans && p.tiles * p.warps < 16ll * SMS) p.warps *= 2;
    // packed sequences are uneven: the longest ones finish last, so each gets several warps if the mean one can use them
    if (a->offsets)
        while (p.warps < WARPS && 2 * p.warps <= spans) p.warps *= 2;
    // where no warps share a tile, the block is one tile if groups leave lanes of a warp idle: 96 channels are 24 lanes, of which
    // 10 fit a block and 1 a warp (160k x 16 x 96 f16: 233 us, by warps 280; 30k x 64 x 4 groups of 8 lanes: 201, by warps 181)
    p.block = backward && p.shared && p.warps == 1 && 32 % p.group_units != 0;
    if (p.block) group_tiles(32 * WARPS);
    p.splits = 1;
    const long long have = p.tiles * p.warps, want = 24ll * SMS;
    if (p.warps == WARPS && have > 0 && have * 2 <= want) {
        const long long rounds = (mean + p.warps * SPAN - 1) / (p.warps * SPAN);
        p.splits = (int)std::max(1ll, std::min({want / have, rounds, (long long)MAX_SPLITS}));
    }
    p.agg_bytes = p.splits > 1 ? (8ll * p.splits * chains + 15) / 16 * 16 : 0;
    // blocks that share a sequence all start from its state, and one of them writes the new one at a time of its own: where that
    // takes the old one's place they start from a copy
    p.ends_bytes = p.splits > 1 && ends_in_place(a, backward) ? (4 * chains + 15) / 16 * 16 : 0;
    p.bytes = p.agg_bytes + p.ends_bytes + (p.parts > 1 ? 4ll * p.parts * p.rows * a->groups : 0);
    return p;
}

RecArgs rec_args(const flare_recurrence_args *in, const RecPlan &p) {
    RecArgs a{};
    a.gate = in->gate, a.x = in->x, a.dh = in->dh, a.offsets = in->offsets;
    if (in->seqs) a.state = in->state, a.dlast = in->dlast;
    a.h = in->h, a.dgate = in->dgate, a.dx = in->dx;
    a.last = in->last, a.saved = in->saved, a.dstate = in->dstate;
    a.agg = static_cast<float *>(in->workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(in->workspace) + p.agg_bytes + p.ends_bytes);
    a.seqs = in->seqs, a.steps = (int)in->steps, a.rows = p.rows;
    a.gate_s = in->gate_s, a.x_s = in->x_s, a.h_s = in->h_s, a.dh_s = in->dh_s, a.dgate_s = in->dgate_s, a.dx_s = in->dx_s;
    a.gate_t = (int)in->gate_t, a.x_t = (int)in->x_t, a.h_t = (int)in->h_t;
    a.dh_t = (int)in->dh_t, a.dgate_t = (int)in->dgate_t, a.dx_t = (int)in->dx_t;
    a.width = in->width, a.groups = in->groups, a.share = FastDiv((unsigned)(in->width / in->groups));
    a.off64 = in->offsets_type == FLARE_I64, a.reverse = in->reverse != 0, a.packed = in->offsets != nullptr;
    while ((1 << a.wlog) < p.warps) ++a.wlog;
    a.splits = p.splits, a.tiles = (unsigned)p.tiles;
    const long long round = (long long)p.warps * SPAN, rounds = (in->steps + round - 1) / round;
    a.per = (int)std::min<long long>((rounds + p.splits - 1) / p.splits * round, 0x7fffffff);
    a.units = (unsigned)(in->seqs * in->width / p.ve);
    a.upr = FastDiv((unsigned)(in->width / p.ve));
    a.group_units = p.group_units, a.groups_per_tile = p.groups_per_tile, a.parts = p.parts;
    a.gunits = FastDiv((unsigned)p.group_units), a.fparts = FastDiv((unsigned)p.parts);
    a.spans = (int)((in->steps + SPAN - 1) / SPAN);
    return a;
}

template <class F>
int rec_dispatch(const flare_recurrence_args *in, const RecPlan &p, F f) {
    return with_type(in->x_type, [&](auto t) {
        using T = typename decltype(t)::type;
        auto gates = [&](auto gt) {
            auto vec = [&](auto ve) {
                if (p.shared) f(t, gt, ve, std::true_type{});
                else f(t, gt, ve, std::false_type{});
            };
            if constexpr (!std::is_same_v<T, float>)
                if (p.ve == 8) return f(t, gt, std::integral_constant<int, 8>{}, std::true_type{});  // shared gates, forward
            if (p.ve == 4) vec(std::integral_constant<int, 4>{});
            else if (p.ve == 2) vec(std::integral_constant<int, 2>{});
            else vec(std::integral_constant<int, 1>{});
        };
        if (in->gate_type == in->x_type) gates(TypeTag<T>{});
        else gates(TypeTag<float>{});
        return 0;
    });
}

int run_recurrence(const flare_recurrence_args *in, bool backward, cudaStream_t st) {
    const RecPlan p = rec_plan(in, backward);
    RecArgs a = rec_args(in, p);
    if (p.ends_bytes) {
        float *copy = reinterpret_cast<float *>(static_cast<char *>(in->workspace) + p.agg_bytes);
        const cudaError_t e = cudaMemcpyAsync(copy, ends_in_place(in, backward), sizeof(float) * (size_t)(in->seqs * in->width),
                                              cudaMemcpyDeviceToDevice, st);
        if (e != cudaSuccess) {
            set_error("%s: %s", backward ? "flare_recurrence_backward" : "flare_recurrence_forward", cudaGetErrorString(e));
            return FLARE_E_CUDA;
        }
        (backward ? a.dlast : a.state) = copy;
    }
    const int at_once = WARPS / p.warps;  // tiles of warps per block
    // a block is launched for rows of no sequence even where there is no sequence
    const dim3 grid((unsigned)std::max(1ll, p.block ? p.tiles : (p.tiles + at_once - 1) / at_once), (unsigned)p.splits);
    const size_t buffers = p.warps > 1 ? sizeof(float) * 2 * WARPS * 32 * p.ve : 0;
    rec_dispatch(in, p, [&](auto t, auto gt, auto ve, auto shared) {
        using T = typename decltype(t)::type;
        using GT = typename decltype(gt)::type;
        constexpr int VE = decltype(ve)::value;
        constexpr bool SH = decltype(shared)::value;
        // the split kernel's tiles are plain ones, whatever the main kernel's
        RecArgs plain = a;
        plain.tiles = (a.units + 31) / 32;
        const dim3 sgrid((plain.tiles + at_once - 1) / at_once, (unsigned)p.splits);
        if (!backward) {
            // 8 channels a lane take 300,000 channels, which leave nothing to split
            if constexpr (VE < 8)
                if (p.splits > 1) recurrence_split_kernel<false, T, GT, VE, SH><<<sgrid, 32 * WARPS, buffers, st>>>(plain);
            recurrence_forward_kernel<T, GT, VE, SH><<<grid, 32 * WARPS, buffers, st>>>(a);
            return;
        }
        if constexpr (VE <= widest_backward(sizeof(T) == 4, SH)) {
            if (p.splits > 1) recurrence_split_kernel<true, T, GT, VE, SH><<<sgrid, 32 * WARPS, buffers, st>>>(plain);
            const size_t sums = SH ? sizeof(float) * WARPS * SPAN * 33 : 0;
            auto launch = [&](auto lanes) {
                constexpr int LANES = decltype(lanes)::value;
                if (a.dh) recurrence_backward_kernel<T, GT, VE, LANES, true><<<grid, 32 * WARPS, buffers + sums, st>>>(a);
                else recurrence_backward_kernel<T, GT, VE, LANES, false><<<grid, 32 * WARPS, buffers + sums, st>>>(a);
            };
            if constexpr (!SH) launch(std::integral_constant<int, 0>{});
            else if (p.block) launch(std::integral_constant<int, 32 * WARPS>{});
            else launch(std::integral_constant<int, 32>{});
            if (p.parts > 1) {
                const long long n = p.rows * in->groups;
                recurrence_join_kernel<GT><<<(unsigned)std::min<long long>((n + 255) / 256, 16 * SMS), 256, 0, st>>>(a);
            }
        }
    });
    OPS_LAUNCHED(backward ? "flare_recurrence_backward" : "flare_recurrence_forward");
    return FLARE_OK;
}

int rec_check(const flare_recurrence_args *a, bool backward, const char *what) {
    OPS_CHECK(a, "%s: NULL argument", what);
    OPS_CHECK(is_float_type(a->x_type) && is_float_type(a->gate_type), "%s: unknown type", what);
    OPS_CHECK(a->gate_type == a->x_type || a->gate_type == FLARE_F32, "%s: gates of type %d with x of type %d", what, a->gate_type,
              a->x_type);
    OPS_CHECK(a->seqs >= 0 && a->steps >= 0 && a->width >= 1 && a->groups >= 1 && a->width % a->groups == 0,
              "%s: %lld sequences of %lld steps, %d channels in %d groups", what, a->seqs, a->steps, a->width, a->groups);
    OPS_CHECK(a->seqs < 0x40000000ll && a->seqs * a->width < 0x40000000ll && a->steps < 0x40000000ll,
              "%s: %lld sequences of %lld steps, %d channels", what, a->seqs, a->steps, a->width);
    // a tensor's steps are addressed by 32-bit distances
    const long long gate = std::max(std::abs(a->gate_t), std::abs(a->dgate_t)) * type_size(a->gate_type);
    const long long rest = std::max({std::abs(a->x_t), std::abs(a->h_t), std::abs(a->dh_t), std::abs(a->dx_t)}) * type_size(a->x_type);
    OPS_CHECK(gate < 0x7fffffffll && rest < 0x7fffffffll, "%s: steps %lld bytes apart, less than 2^31 needed", what, std::max(gate, rest));
    const bool some = a->seqs > 0, data = (some || a->offsets) && a->steps > 0;
    OPS_CHECK(!data || (a->gate && a->x), "%s: NULL gate or x", what);
    const long long ends = 4 * a->seqs * a->width;
    if (!backward) {
        OPS_CHECK(!some || a->last, "%s: NULL last", what);
        OPS_CHECK(a->last == a->state || !overlaps(a->last, ends, a->state, ends), "%s: last overlaps state", what);
        // a step's caller chooses where the new state goes; element for element it may take an input's place, as each
        // thread reads all of its own before it writes
        if (a->steps == 1 && !a->offsets && a->last) {
            auto apart = [&](const void *p, long long stride, int width, int type) {
                const int size = type_size(type);
                return (p == a->last && type == FLARE_F32 && width == a->width && (stride == width || a->seqs == 1)) ||
                       !overlaps_rows(a->last, ends, p, a->seqs, (long long)width * size, stride * size);
            };
            OPS_CHECK(apart(a->x, a->x_s, a->width, a->x_type), "%s: last overlaps x", what);
            OPS_CHECK(apart(a->gate, a->gate_s, a->groups, a->gate_type), "%s: last overlaps gate", what);
        }
    } else {
        OPS_CHECK(a->dstate == a->dlast || !overlaps(a->dstate, ends, a->dlast, ends), "%s: dstate overlaps dlast", what);
        const bool spans = some && a->steps > SPAN;
        OPS_CHECK(!data || (a->dgate && a->dx), "%s: NULL gradient", what);
        OPS_CHECK(!spans || a->saved, "%s: NULL saved", what);
    }
    OPS_CHECK(a->offsets_type == FLARE_I32 || a->offsets_type == FLARE_I64, "%s: unknown offsets type %d", what, a->offsets_type);
    return FLARE_OK;
}

}  // namespace flare

using namespace flare;

extern "C" {

long long flare_recurrence_saved(long long seqs, long long steps, int width, int packed) {
    if (seqs <= 0 || steps <= SPAN || width <= 0) return 0;
    const long long spans = (steps + SPAN - 1) / SPAN;
    return (packed ? steps / SPAN + seqs + 1 : seqs * (spans - 1)) * width;
}

long long flare_recurrence_workspace(const flare_recurrence_args *a, int backward) {
    if (!a || a->seqs < 0 || a->steps <= 0 || a->width <= 0 || a->groups <= 0 || a->width % a->groups) return 0;
    return rec_plan(a, backward != 0).bytes;
}

static int recurrence_entry(const flare_recurrence_args *a, bool backward, void *stream, const char *what) {
    int e = rec_check(a, backward, what);
    if (e) return e;
    if (a->seqs == 0 && !(a->offsets && a->steps)) return FLARE_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->steps == 0) {
        // nothing steps: the state passes through, its gradient too
        float *dst = backward ? a->dstate : a->last;
        const float *src = backward ? a->dlast : a->state;
        const size_t bytes = sizeof(float) * (size_t)(a->seqs * a->width);
        cudaError_t ce = cudaSuccess;
        if (dst && bytes && src) {
            if (dst != src) ce = cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice, st);
        } else if (dst && bytes) {
            ce = cudaMemsetAsync(dst, 0, bytes, st);
        }
        if (ce != cudaSuccess) {
            set_error("%s: %s", what, cudaGetErrorString(ce));
            return FLARE_E_CUDA;
        }
        return FLARE_OK;
    }
    const long long need = flare_recurrence_workspace(a, backward);
    OPS_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && reinterpret_cast<uintptr_t>(a->workspace) % 16 == 0),
              "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what, a->workspace_bytes, need);
    return run_recurrence(a, backward, st);
}

int flare_recurrence_forward(const flare_recurrence_args *a, void *stream) {
    return recurrence_entry(a, false, stream, "flare_recurrence_forward");
}

int flare_recurrence_backward(const flare_recurrence_args *a, void *stream) {
    return recurrence_entry(a, true, stream, "flare_recurrence_backward");
}

}  // extern "C"
