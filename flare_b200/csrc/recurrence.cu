// recurrence.cu -- the gated linear recurrence h_t = a_t h_{t-1} + x_t over many sequences, and its gradient.
//
// A stretch of steps maps the state that enters it to A h + H (A the product of its gates, H what it yields from 0), and
// two stretches join to (A2 A1, A2 H1 + H2), so a sequence can be cut in time:
//   * a thread holds SPAN = 16 steps of VE neighbouring channels in registers, all loaded before the first is used;
//   * the W warps of a block take W consecutive spans, exchange their (A, H) through shared memory and run their own
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

#include "ops.cuh"

namespace flare {

constexpr int SPAN = FLARE_RECURRENCE_SPAN;
constexpr int MAX_W = 8;        // warps per block along time
constexpr int MAX_SPLITS = 64;  // blocks along time

struct RecArgs {
    const void *gate, *x, *dh, *offsets;
    const float *state, *dlast;
    void *h, *dgate, *dx;
    float *last, *saved, *dstate;
    float *agg;      // (splits, 2, seqs * width)
    float *partial;  // (parts, rows, groups): sums over parts of a group's channels
    long long seqs, steps, rows;
    long long gate_s, gate_t, x_s, x_t, h_s, h_t, dh_s, dh_t, dgate_s, dgate_t, dx_s, dx_t;
    int width, groups, share;  // share: channels per gate
    int off64, reverse, packed;
    int splits;
    unsigned units;            // lanes' worth of channels: seqs * width / VE
    FastDiv upr;               // units per sequence
    int group_units, groups_per_tile, parts;  // backward tiles of whole groups, see Place
    long long spans;           // dense: spans per sequence
};

__device__ __forceinline__ long long offset_at(const RecArgs &a, long long s) {
    const long long o = a.off64 ? __ldg(static_cast<const long long *>(a.offsets) + s) : (long long)__ldg(static_cast<const int *>(a.offsets) + s);
    return min(max(o, 0ll), a.steps);
}

// Where a lane's channels lie.  GROUPED: tiles consist of whole groups of channels that share a gate, or of a part of
// one such group (32 lanes at a time), so that sums over a group need no other block.
template <int VE, bool GROUPED>
struct Place {
    bool active;
    long long seq, row0, len;  // row0: first row of the sequence in memory terms (packed), len: its steps
    int c;                     // first channel
    long long chain;           // seq * width + c
    int pos, part;
    __device__ __forceinline__ Place(const RecArgs &a, unsigned tile) {
        const int lane = threadIdx.x & 31;
        unsigned u;
        if (!GROUPED) {
            u = tile * 32 + lane;
            active = u < a.units;
            pos = part = 0;
        } else if (a.parts == 1) {
            const unsigned g = lane / a.group_units;
            pos = lane - g * a.group_units;
            u = (tile * a.groups_per_tile + g) * a.group_units + pos;
            active = (int)g < a.groups_per_tile && u < a.units;
            part = 0;
        } else {
            part = tile % a.parts;
            pos = part * 32 + lane;
            u = tile / a.parts * a.group_units + pos;
            active = pos < a.group_units;
        }
        if (!active) u = 0;
        const unsigned s = a.upr.div(u);
        seq = s;
        c = (int)(u - s * a.upr.d) * VE;
        chain = seq * a.width + c;
        row0 = 0;
        len = a.steps;
        if (a.packed) {
            row0 = offset_at(a, seq);
            len = max(offset_at(a, seq + 1) - row0, 0ll);
        }
        if (!active) len = 0;
    }
    // element offset of step 0's row in a tensor and the distance to the next step's
    __device__ __forceinline__ long long first(const RecArgs &a, long long stride_s, long long stride_t) const {
        const long long base = a.packed ? row0 * stride_t : seq * stride_s;
        return base + (a.reverse ? (len - 1) * stride_t : 0);
    }
    // row of `saved` that holds the state before span k >= 1
    __device__ __forceinline__ long long saved_row(const RecArgs &a, long long k) const {
        return a.packed ? row0 / SPAN + seq + k : seq * (a.spans - 1) + k - 1;
    }
};

// the steps of a lane that block `split` of a.splits works on, in whole rounds of W spans
__device__ __forceinline__ void split_range(const RecArgs &a, long long len, int W, int split, long long &t0, long long &t1) {
    const long long round = (long long)W * SPAN;
    const long long rounds = (len + round - 1) / round;
    const long long per = (rounds + a.splits - 1) / a.splits * round;
    t0 = min(len, split * per);
    t1 = min(len, t0 + per);
}

__device__ __forceinline__ long long warp_max(long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// What a stretch (A, H) makes of the state c.  A state of exactly 0 adds nothing, also where the product of the gates
// has left the range of a float.
__device__ __forceinline__ float through(float A, float H, float c) { return c == 0.0f ? H : fmaf(A, c, H); }

// A lane's gates of one span: one per channel, or one for all its channels.
template <class GT, int VE, bool SHARED>
struct Gates {
    static constexpr int N = SHARED ? 1 : VE;
    Vec<GT, N> g[SPAN];
    __device__ __forceinline__ void load(const GT *p, long long step, long long n) {
#pragma unroll
        for (int i = 0; i < SPAN; ++i) {
            if (i < n) g[i].load(p + i * step);
            else
#pragma unroll
                for (int v = 0; v < N; ++v) g[i].set(v, 1.0f);
        }
    }
    __device__ __forceinline__ float at(int i, int v) const { return g[i].get(SHARED ? 0 : v); }
};

template <class T, int VE>
struct Span {
    Vec<T, VE> d[SPAN];
    __device__ __forceinline__ void load(const T *p, long long step, long long n) {
#pragma unroll
        for (int i = 0; i < SPAN; ++i) {
            if (i < n) d[i].load(p + i * step);
            else d[i].zero();
        }
    }
};

// (A, H) of a span, walked from its first step (forward) or its last (backward, where H collects a_t dh_t)
template <bool BACK, class T, class GT, int VE, bool SHARED>
__device__ __forceinline__ void stretch(const Gates<GT, VE, SHARED> &g, const Span<T, VE> &x, float (&A)[VE], float (&H)[VE]) {
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
            H[v] = BACK ? a * (H[v] + x.d[i].get(v)) : fmaf(a, H[v], x.d[i].get(v));
            A[v] *= a;
        }
    }
}

// The state that enters warp w's span, from the state `carry` that enters the round; carry becomes what leaves the round.
// BACK: warps are passed from the last to the first.  buf: (2, W, 32 VE) floats, not the one of the round before.
template <bool BACK, int VE>
__device__ __forceinline__ void exchange(float *buf, int W, const float (&A)[VE], const float (&H)[VE], float (&carry)[VE], float (&in)[VE]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    float *sa = buf, *sh = buf + W * 32 * VE;
#pragma unroll
    for (int v = 0; v < VE; ++v) {
        sa[(w * VE + v) * 32 + lane] = A[v];
        sh[(w * VE + v) * 32 + lane] = H[v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VE; ++v) in[v] = carry[v];
    for (int k = 0; k < W; ++k) {
        const int o = BACK ? W - 1 - k : k;
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            if (o == w) in[v] = carry[v];
            carry[v] = through(sa[(o * VE + v) * 32 + lane], sh[(o * VE + v) * 32 + lane], carry[v]);
        }
    }
}

// state entering block `split`: `c` through the blocks that come before it in the walk
template <bool BACK, int VE>
__device__ __forceinline__ void fold_splits(const RecArgs &a, long long chain, int split, float (&c)[VE]) {
    const long long chains = a.seqs * a.width;
    const int n = BACK ? a.splits - 1 - split : split;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
        const int o = BACK ? a.splits - 1 - k : k;
        const float *p = a.agg + (long long)o * 2 * chains + chain;
#pragma unroll
        for (int v = 0; v < VE; ++v) c[v] = through(__ldg(p + v), __ldg(p + chains + v), c[v]);
    }
}

// BACK false: (A, H) of x; true: of dh, from the end.  grid (tiles, splits)
template <bool BACK, class T, class GT, int VE, bool SHARED>
__global__ void __launch_bounds__(32 * MAX_W) recurrence_split_kernel(const RecArgs a) {
    extern __shared__ float smem[];
    const int W = blockDim.x >> 5, lane = threadIdx.x & 31, w = threadIdx.x >> 5, split = blockIdx.y;
    const Place<VE, false> me(a, blockIdx.x);
    long long t0, t1;
    split_range(a, me.len, W, split, t0, t1);
    const long long span = warp_max(t1 - t0), round = (long long)W * SPAN;
    const long long dir = a.reverse ? -1 : 1;
    const void *src = BACK ? a.dh : a.x;
    const long long src_s = BACK ? a.dh_s : a.x_s, src_t = BACK ? a.dh_t : a.x_t;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + me.c / a.share;
    const T *xp = static_cast<const T *>(src) + me.first(a, src_s, src_t) + me.c;
    float A[VE], H[VE], tA[VE], tH[VE], unused[VE];
#pragma unroll
    for (int v = 0; v < VE; ++v) {
        tA[v] = 1.0f;
        tH[v] = 0.0f;
    }
    const long long n = (span + round - 1) / round;
    for (long long k = 0; k < n; ++k) {
        const long long r = BACK ? n - 1 - k : k;
        const long long t = t0 + r * round + w * SPAN, left = t1 - t;
        Gates<GT, VE, SHARED> g;
        Span<T, VE> x;
        g.load(gp + t * dir * a.gate_t, dir * a.gate_t, left);
        if (src) x.load(xp + t * dir * src_t, dir * src_t, left);
        else x.load(xp, 0, 0);
        stretch<BACK>(g, x, A, H);
        float *buf = smem + (k & 1) * 2 * W * 32 * VE;
        exchange<BACK>(buf, W, A, H, tH, unused);
        // the product of the round's gates, in the same buffer
        for (int o = 0; o < W; ++o)
#pragma unroll
            for (int v = 0; v < VE; ++v) tA[v] *= buf[(o * VE + v) * 32 + lane];
    }
    if (w == 0 && me.active) {
        const long long chains = a.seqs * a.width;
        float *p = a.agg + (long long)split * 2 * chains + me.chain;
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            p[v] = tA[v];
            p[chains + v] = tH[v];
        }
    }
}

template <class T, class GT, int VE, bool SHARED>
__global__ void __launch_bounds__(32 * MAX_W) recurrence_forward_kernel(const RecArgs a) {
    extern __shared__ float smem[];
    const int W = blockDim.x >> 5, w = threadIdx.x >> 5, split = blockIdx.y;
    const Place<VE, false> me(a, blockIdx.x);
    long long t0, t1;
    split_range(a, me.len, W, split, t0, t1);
    const long long span = warp_max(t1 - t0), round = (long long)W * SPAN;
    const long long dir = a.reverse ? -1 : 1;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + me.c / a.share;
    const T *xp = static_cast<const T *>(a.x) + me.first(a, a.x_s, a.x_t) + me.c;
    T *hp = a.h ? static_cast<T *>(a.h) + me.first(a, a.h_s, a.h_t) + me.c : nullptr;
    float carry[VE], h[VE], A[VE], H[VE];
#pragma unroll
    for (int v = 0; v < VE; ++v) carry[v] = me.active && a.state ? a.state[me.chain + v] : 0.0f;
    if (me.active) fold_splits<false, VE>(a, me.chain, split, carry);
    const long long n = (span + round - 1) / round;
    for (long long k = 0; k < n; ++k) {
        const long long t = t0 + k * round + w * SPAN, left = t1 - t;
        Gates<GT, VE, SHARED> g;
        Span<T, VE> x;
        g.load(gp + t * dir * a.gate_t, dir * a.gate_t, left);
        x.load(xp + t * dir * a.x_t, dir * a.x_t, left);
        if (W > 1) {
            stretch<false>(g, x, A, H);
            exchange<false>(smem + (k & 1) * 2 * W * 32 * VE, W, A, H, carry, h);
        } else {
#pragma unroll
            for (int v = 0; v < VE; ++v) h[v] = carry[v];
        }
        if (a.saved && left > 0 && t > 0) {
            float *p = a.saved + me.saved_row(a, t / SPAN) * a.width + me.c;
#pragma unroll
            for (int v = 0; v < VE; ++v) p[v] = h[v];
        }
#pragma unroll
        for (int i = 0; i < SPAN; ++i) {
            Vec<T, VE> o;
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                h[v] = fmaf(g.at(i, v), h[v], x.d[i].get(v));
                o.set(v, h[v]);
            }
            if (hp && i < left) o.store(hp + (t + i) * dir * a.h_t);
        }
        if (W == 1)
#pragma unroll
            for (int v = 0; v < VE; ++v) carry[v] = h[v];
    }
    if (w == 0 && split == a.splits - 1 && me.active)
#pragma unroll
        for (int v = 0; v < VE; ++v) a.last[me.chain + v] = carry[v];
}

template <class T, class GT, int VE, bool SHARED>
__global__ void __launch_bounds__(32 * MAX_W) recurrence_backward_kernel(const RecArgs a) {
    extern __shared__ float smem[];
    const int W = blockDim.x >> 5, w = threadIdx.x >> 5, split = blockIdx.y;
    const Place<VE, SHARED> me(a, blockIdx.x);
    long long t0, t1;
    split_range(a, me.len, W, split, t0, t1);
    const long long span = warp_max(t1 - t0), round = (long long)W * SPAN;
    const long long dir = a.reverse ? -1 : 1;
    const int gc = me.c / a.share;
    const GT *gp = static_cast<const GT *>(a.gate) + me.first(a, a.gate_s, a.gate_t) + gc;
    const T *xp = static_cast<const T *>(a.x) + me.first(a, a.x_s, a.x_t) + me.c;
    const T *dhp = a.dh ? static_cast<const T *>(a.dh) + me.first(a, a.dh_s, a.dh_t) + me.c : nullptr;
    T *dxp = static_cast<T *>(a.dx) + me.first(a, a.dx_s, a.dx_t) + me.c;
    GT *dgp = static_cast<GT *>(a.dgate) + me.first(a, a.dgate_s, a.dgate_t) + gc;
    float carry[VE], mu[VE], A[VE], H[VE];
#pragma unroll
    for (int v = 0; v < VE; ++v) carry[v] = me.active && a.dlast ? a.dlast[me.chain + v] : 0.0f;
    if (me.active) fold_splits<true, VE>(a, me.chain, split, carry);
    const long long n = (span + round - 1) / round;
    for (long long k = 0; k < n; ++k) {
        const long long t = t0 + (n - 1 - k) * round + w * SPAN, left = t1 - t;
        Gates<GT, VE, SHARED> g;
        Span<T, VE> x, dh;
        g.load(gp + t * dir * a.gate_t, dir * a.gate_t, left);
        if (dhp) dh.load(dhp + t * dir * a.dh_t, dir * a.dh_t, left);
        else dh.load(xp, 0, 0);
        x.load(xp + t * dir * a.x_t, dir * a.x_t, left);
        float before[SPAN][VE];  // the state before each step
#pragma unroll
        for (int v = 0; v < VE; ++v) before[0][v] = 0.0f;
        if (left > 0) {
            const float *p = t > 0 ? a.saved + me.saved_row(a, t / SPAN) * a.width + me.c : a.state ? a.state + me.chain : nullptr;
            if (p)
#pragma unroll
                for (int v = 0; v < VE; ++v) before[0][v] = p[v];
        }
        if (W > 1) {
            stretch<true>(g, dh, A, H);
            exchange<true>(smem + (k & 1) * 2 * W * 32 * VE, W, A, H, carry, mu);
        } else {
#pragma unroll
            for (int v = 0; v < VE; ++v) mu[v] = carry[v];
        }
#pragma unroll
        for (int i = 0; i + 1 < SPAN; ++i)
#pragma unroll
            for (int v = 0; v < VE; ++v) before[i + 1][v] = fmaf(g.at(i, v), before[i][v], x.d[i].get(v));
#pragma unroll
        for (int i = SPAN - 1; i >= 0; --i) {
            Vec<T, VE> o;
            Vec<GT, SHARED ? 1 : VE> og;
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                const float lambda = dh.d[i].get(v) + mu[v];
                o.set(v, lambda);
                const float d = lambda * before[i][v];
                if (SHARED) sum += d;
                else og.set(v, d);
                mu[v] = g.at(i, v) * lambda;
            }
            if (i < left) o.store(dxp + (t + i) * dir * a.dx_t);
            if (!SHARED) {
                if (i < left) og.store(dgp + (t + i) * dir * a.dgate_t);
            } else {
                // sum over the group's lanes of this tile; steps past the end and lanes without channels add 0
                const int units = min(a.group_units - me.part * 32, 32);
                const int pos = me.pos - me.part * 32;
                if (!(i < left)) sum = 0.0f;
                for (int d = 1; d < units; d <<= 1) {
                    const float other = __shfl_down_sync(0xffffffffu, sum, d);
                    if (pos + d < units) sum += other;
                }
                if (pos == 0 && i < left) {
                    if (a.parts == 1) {
                        dgp[(t + i) * dir * a.dgate_t] = from_f32<GT>(sum);
                    } else {
                        const long long at = a.reverse ? me.len - 1 - (t + i) : t + i;
                        const long long row = (a.packed ? me.row0 : me.seq * a.steps) + at;
                        a.partial[(me.part * a.rows + row) * a.groups + gc] = sum;
                    }
                }
            }
        }
        if (W == 1)
#pragma unroll
            for (int v = 0; v < VE; ++v) carry[v] = mu[v];
    }
    if (a.dstate && w == 0 && split == 0 && me.active)
#pragma unroll
        for (int v = 0; v < VE; ++v) a.dstate[me.chain + v] = carry[v];
}

// dgate from the partial sums of its parts, in order
template <class GT>
__global__ void recurrence_join_kernel(const RecArgs a) {
    const long long n = a.rows * a.groups;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        float t = 0.0f;
        for (int p = 0; p < a.parts; ++p) t += a.partial[p * n + i];
        const long long row = i / a.groups, g = i - row * a.groups;
        const long long s = a.packed ? 0 : row / a.steps, at = a.packed ? row : row - s * a.steps;
        static_cast<GT *>(a.dgate)[s * a.dgate_s + at * a.dgate_t + g] = from_f32<GT>(t);
    }
}

// zeros in the rows of a packed tensor that belong to no sequence
template <class T>
__global__ void recurrence_rest_kernel(const RecArgs a, T *out, long long stride, int width) {
    const long long head = min(offset_at(a, 0), offset_at(a, a.seqs)), tail = offset_at(a, a.seqs);
    const long long rows = head + a.steps - tail, n = rows * width;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / width;
        out[(r < head ? r : tail + r - head) * stride + (i - r * width)] = from_f32<T>(0.0f);
    }
}

// ------------------------------------------------------------------------------------------------

struct RecPlan {
    int ve, warps, splits, parts, group_units, groups_per_tile;
    bool shared;
    long long tiles, rows, agg_bytes, bytes;
};

// Vectors of `ve` channels: whole within a group of channels that share a gate, aligned in every tensor.
bool vec_fits(const flare_recurrence_args *a, int ve, bool backward) {
    const int xs = type_size(a->x_type), gs = type_size(a->gate_type), share = a->width / a->groups;
    if (a->width % ve || (share > 1 && share % ve)) return false;
    auto ok = [&](const void *p, long long s, long long t, int size) {
        return !p || (fits_vec(p, t, size, ve) && (a->offsets || s % ve == 0));
    };
    if (!ok(a->x, a->x_s, a->x_t, xs)) return false;
    if (share == 1 && !ok(a->gate, a->gate_s, a->gate_t, gs)) return false;
    if (!backward) return ok(a->h, a->h_s, a->h_t, xs);
    return ok(a->dh, a->dh_s, a->dh_t, xs) && ok(a->dx, a->dx_s, a->dx_t, xs) &&
           (share > 1 || ok(a->dgate, a->dgate_s, a->dgate_t, gs));
}

RecPlan rec_plan(const flare_recurrence_args *a, bool backward) {
    RecPlan p{};
    const int share = a->width / a->groups;
    p.shared = share > 1;
    p.rows = a->offsets ? a->steps : a->seqs * a->steps;
    // 4 bytes a lane make whole 128-byte lines of a warp; wider vectors only where a group of channels then fits a warp
    p.ve = a->x_type == FLARE_F32 ? 1 : 2;
    if (backward && p.shared)
        while (p.ve < 4 && share / p.ve > 32) p.ve *= 2;
    while (p.ve > 1 && !vec_fits(a, p.ve, backward)) p.ve >>= 1;
    const long long units = a->seqs * a->width / p.ve;
    p.group_units = p.parts = p.groups_per_tile = 1;
    if (backward && p.shared) {
        p.group_units = share / p.ve;
        p.parts = (p.group_units + 31) / 32;
        p.groups_per_tile = p.parts > 1 ? 1 : 32 / p.group_units;
        const long long groups = a->seqs * a->groups;
        p.tiles = p.parts > 1 ? groups * p.parts : (groups + p.groups_per_tile - 1) / p.groups_per_tile;
    } else {
        p.tiles = (units + 31) / 32;
    }
    // time is cut only as far as it takes to fill the machine: W spans a block, then S blocks
    const long long mean = std::max<long long>(1, a->offsets ? a->steps / std::max<long long>(1, a->seqs) : a->steps);
    const long long spans = (mean + SPAN - 1) / SPAN;
    p.warps = 1;
    while (p.warps < MAX_W && 2 * p.warps <= spans && p.tiles * p.warps < 12ll * SMS) p.warps *= 2;
    p.splits = 1;
    const long long have = p.tiles * p.warps, want = 8ll * SMS;
    if (have > 0 && have * 2 <= want) {
        const long long rounds = (mean + p.warps * SPAN - 1) / (p.warps * SPAN);
        p.splits = (int)std::min({want / have, rounds, (long long)MAX_SPLITS});
        if (p.splits < 1) p.splits = 1;
    }
    p.agg_bytes = p.splits > 1 ? (8ll * p.splits * a->seqs * a->width + 15) / 16 * 16 : 0;
    p.bytes = p.agg_bytes + (p.parts > 1 ? 4ll * p.parts * p.rows * a->groups : 0);
    return p;
}

RecArgs rec_args(const flare_recurrence_args *in, const RecPlan &p) {
    RecArgs a{};
    a.gate = in->gate, a.x = in->x, a.dh = in->dh, a.offsets = in->offsets;
    a.state = in->state, a.dlast = in->dlast;
    a.h = in->h, a.dgate = in->dgate, a.dx = in->dx;
    a.last = in->last, a.saved = in->saved, a.dstate = in->dstate;
    a.agg = static_cast<float *>(in->workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(in->workspace) + p.agg_bytes);
    a.seqs = in->seqs, a.steps = in->steps, a.rows = p.rows;
    a.gate_s = in->gate_s, a.gate_t = in->gate_t, a.x_s = in->x_s, a.x_t = in->x_t, a.h_s = in->h_s, a.h_t = in->h_t;
    a.dh_s = in->dh_s, a.dh_t = in->dh_t, a.dgate_s = in->dgate_s, a.dgate_t = in->dgate_t, a.dx_s = in->dx_s, a.dx_t = in->dx_t;
    a.width = in->width, a.groups = in->groups, a.share = in->width / in->groups;
    a.off64 = in->offsets_type == FLARE_I64, a.reverse = in->reverse != 0, a.packed = in->offsets != nullptr;
    a.splits = p.splits;
    a.units = (unsigned)(in->seqs * in->width / p.ve);
    a.upr = FastDiv((unsigned)(in->width / p.ve));
    a.group_units = p.group_units, a.groups_per_tile = p.groups_per_tile, a.parts = p.parts;
    a.spans = (in->steps + SPAN - 1) / SPAN;
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
            if (p.ve == 4) vec(std::integral_constant<int, 4>{});
            else if (p.ve == 2) vec(std::integral_constant<int, 2>{});
            else vec(std::integral_constant<int, 1>{});
        };
        if (in->gate_type == in->x_type) gates(TypeTag<T>{});
        else gates(TypeTag<float>{});
        return 0;
    });
}

template <class T>
void launch_rest(const RecArgs &a, void *out, long long stride, int width, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<long long>((a.steps * width + 255) / 256, 2 * SMS);
    recurrence_rest_kernel<T><<<blocks, 256, 0, st>>>(a, static_cast<T *>(out), stride, width);
}

int run_recurrence(const flare_recurrence_args *in, bool backward, cudaStream_t st) {
    const RecPlan p = rec_plan(in, backward);
    const RecArgs a = rec_args(in, p);
    const dim3 grid((unsigned)p.tiles, (unsigned)p.splits);
    const int threads = 32 * p.warps;
    const size_t smem = p.warps > 1 ? sizeof(float) * 4 * p.warps * 32 * p.ve : 0;
    const char *what = backward ? "flare_recurrence_backward" : "flare_recurrence_forward";
    rec_dispatch(in, p, [&](auto t, auto gt, auto ve, auto shared) {
        using T = typename decltype(t)::type;
        using GT = typename decltype(gt)::type;
        constexpr int VE = decltype(ve)::value;
        constexpr bool SH = decltype(shared)::value;
        if (p.tiles == 0) {  // packed rows without a sequence
        } else if (p.splits > 1) {
            // the split kernel's tiles are plain ones, whatever the main kernel's
            const dim3 sgrid((a.units + 31) / 32, (unsigned)p.splits);
            const size_t ss = sizeof(float) * 4 * p.warps * 32 * VE;
            if (backward) recurrence_split_kernel<true, T, GT, VE, SH><<<sgrid, threads, ss, st>>>(a);
            else recurrence_split_kernel<false, T, GT, VE, SH><<<sgrid, threads, ss, st>>>(a);
        }
        if (p.tiles == 0) {
        } else if (backward) recurrence_backward_kernel<T, GT, VE, SH><<<grid, threads, smem, st>>>(a);
        else recurrence_forward_kernel<T, GT, VE, SH><<<grid, threads, smem, st>>>(a);
        if (p.tiles && backward && p.parts > 1) {
            const long long n = p.rows * in->groups;
            recurrence_join_kernel<GT><<<(unsigned)std::min<long long>((n + 255) / 256, 16 * SMS), 256, 0, st>>>(a);
        }
        if (a.packed) {
            if (!backward && a.h) launch_rest<T>(a, a.h, a.h_t, a.width, st);
            if (backward) {
                launch_rest<T>(a, a.dx, a.dx_t, a.width, st);
                launch_rest<GT>(a, a.dgate, a.dgate_t, a.groups, st);
            }
        }
    });
    OPS_LAUNCHED(what);
    return FLARE_OK;
}

int rec_check(const flare_recurrence_args *a, bool backward, const char *what) {
    OPS_CHECK(a, "%s: NULL argument", what);
    OPS_CHECK(is_float_type(a->x_type) && is_float_type(a->gate_type), "%s: unknown type", what);
    OPS_CHECK(a->gate_type == a->x_type || a->gate_type == FLARE_F32, "%s: gates of type %d with x of type %d", what, a->gate_type,
              a->x_type);
    OPS_CHECK(a->seqs >= 0 && a->steps >= 0 && a->width >= 1 && a->groups >= 1 && a->width % a->groups == 0,
              "%s: %lld sequences of %lld steps, %d channels in %d groups", what, a->seqs, a->steps, a->width, a->groups);
    OPS_CHECK(a->seqs * a->width < 0x40000000ll && a->seqs < 0x40000000ll, "%s: %lld sequences of %d channels", what, a->seqs, a->width);
    OPS_CHECK(a->offsets_type == FLARE_I32 || a->offsets_type == FLARE_I64, "%s: unknown offsets type %d", what, a->offsets_type);
    const bool some = a->seqs > 0, data = (some || a->offsets) && a->steps > 0;
    OPS_CHECK(!data || (a->gate && a->x), "%s: NULL gate or x", what);
    if (!backward) {
        OPS_CHECK(!some || a->last, "%s: NULL last", what);
    } else {
        const bool spans = some && a->steps > SPAN;
        OPS_CHECK(!data || (a->dgate && a->dx), "%s: NULL gradient", what);
        OPS_CHECK(!spans || a->saved, "%s: NULL saved", what);
    }
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
