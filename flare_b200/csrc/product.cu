// product.cu -- out = A B^T of two matrices held in microscaled 4-bit floats, on the tensor cores.
//
// tcgen05.mma kind::mxf4 multiplies 4-bit elements and applies the block scales itself: D (TMEM, f32) += (A * 2^sa)
// (B * 2^sb)^T for 64 elements of K at a time, two scales per row.  The larger matrix gives the 128 rows of a tile (P), the
// other its BN columns (Q); where that is B, the tile is stored transposed.  One block per multiprocessor walks over tiles;
// per 256 elements of K (a stage):
//   * warp 8 brings the codes, 128 bytes a row, by TMA into 128-byte-swizzled tiles;
//   * warps 4-7 bring the scales: asynchronous copies of 16 bytes a row (two stages) into a ring, three such groups ahead, from
//     which each warp stores the words of tile rows l, l + 32, l + 64, l + 96 to lane l of its quarter of TMEM.  (tcgen05.cp from
//     shared memory takes 80 cycles of the tensor pipe for each of six pieces a stage, whose products take 384: 54 us at
//     4096 x 4096 x 4096, where this takes 44; scales through registers were waited for, 52; scales never fetched would be 39.)
//   * warp 9 issues the products; its commit frees the stage.
// Warps 0-3 read a finished D from TMEM, a row per thread, round it once and store it through shared memory by TMA, while
// the next tile goes into the other half of TMEM.  Few tiles and a long K: up to 8 blocks of a cluster take a part of K
// each (product_plan.h) and add their tiles through distributed shared memory, in order.
// A few rows that are not quantised yet (at most 16) are Q as they come: four times warps 4-7 quantise a stage of them on the way
// into shared memory, a block of 32 elements per thread, which saves such a call a launch and a matrix.  Scales then lie there
// too, 32 rows of 16 bytes, row r the words of tile rows r, r + 32, r + 64, r + 96, and warp 9 spreads them over TMEM.
// Every wait is bounded; where one ran out the block's tiles are NaN and a bit of the status word is set.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "ops.cuh"
#include "product_plan.h"
#include "umma.cuh"

namespace flare {

constexpr int PT = 128;          // rows of P per tile
constexpr int KSTAGE = 256;      // elements of K per stage
constexpr int KBYTES = KSTAGE / 2;
constexpr int PR_WARPS = 10, PR_THREADS = 32 * PR_WARPS;
constexpr int SMEM_MAX = 227 * 1024, SMEM_FIXED = 2048;  // static shared memory and alignment
constexpr int OUT_BYTES = 32 * 128;                      // a warp's piece of the output on its way
constexpr int TMEM_COLS = 512;

struct ProductArgs {
    const unsigned char *ps, *qs;
    void *out;
    int *status;
    long long p, q, out_stride;
    int k, blocks, pitch;         // blocks of 32 per row, scale bytes per row
    int stages, swap, vec, bulk;  // vec: 16-byte stores of a row's columns are aligned; bulk: the output has a tensor map
    int accs;                     // accumulators in TMEM
    unsigned ptiles, tiles;
    int wide;                     // scales may be read 16 bytes at a time
    const void *x;                // Q before quantisation, else NULL
    long long x_stride;
    int x_vec;                    // its rows may be read 16 bytes at a time
};

// threads of a product whose Q is quantised on the way: a stage takes a warp longer (0.8 us) than its codes need to arrive, so
// four teams of four warps take the stages in turn
constexpr int X_TEAMS = 4, X_THREADS = PR_THREADS + 128 * (X_TEAMS - 1);
constexpr int X_ROWS = FLARE_PRODUCT_ROWS;
static_assert(X_ROWS * (KSTAGE / 32) == 128, "a block of 32 elements per thread of four warps");

// 32 elements of a row, in flight
template <class X>
struct Raw32 {
    static constexpr int N = 16 / (int)sizeof(X);  // elements of a 16-byte piece
    unsigned w[8 * (int)sizeof(X)];
    // left: elements from p to the row's end
    __device__ __forceinline__ void load(const X *p, int left, bool vec) {
#pragma unroll
        for (int i = 0; i < 32 / N; ++i) {
            Vec<X, N> v;
            if (vec && left >= (i + 1) * N) {
                v.load(p + i * N);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v.el[e] = i * N + e < left ? p[i * N + e] : from_f32<X>(0.0f);
            }
            w[4 * i] = v.raw[0].x, w[4 * i + 1] = v.raw[0].y, w[4 * i + 2] = v.raw[0].z, w[4 * i + 3] = v.raw[0].w;
        }
    }
    // its 16 bytes of codes and scale byte
    __device__ __forceinline__ uint4 quantize(unsigned *byte) const {
        float inv;
        *byte = micro_byte(words_most<X, 8 * (int)sizeof(X)>(w), &inv);
        if (*byte == 255) return make_uint4(0, 0, 0, 0);
        return make_uint4(micro_codes8<X>(w, 0, inv), micro_codes8<X>(w, 4, inv), micro_codes8<X>(w, 8, inv), micro_codes8<X>(w, 12, inv));
    }
};
template <>
struct Raw32<void> {};

// A matrix descriptor's words: the low one is the address / 16 and a leading offset of 16 bytes, so that tiles, stages and steps of
// K add to it; the high one is fixed.  One thread issues all products, so its own instructions count (4096 x 4096 x 4096: 57 us
// with whole descriptors built for each of them, 53.5 us so).
constexpr uint32_t DESC_ROWS = 64u | (1u << 14) | (2u << 29);  // 8 rows are 1024 bytes, version 1, 128-byte swizzle
constexpr uint32_t DESC_SCALES = 8u | (1u << 14);              // 8 rows are 128 bytes, version 1, no swizzle
__device__ __forceinline__ uint32_t desc_low(const void *p) { return (smem_u32(p) >> 4) | (1u << 16); }

// D (+)= A B^T, 64 elements of K; the scales' columns in TMEM, which half of their words in idesc
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 da, {%1, %7};\n\t"
        "mov.b64 db, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}\n"
        :
        : "r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(sa), "r"(sb), "r"(acc), "r"(DESC_ROWS)
        : "memory");
}
// 32 rows x 16 bytes of shared memory to 4 columns of TMEM, the same in all four quarters of the lanes
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t low) {
    asm volatile(
        "{\n\t.reg .b64 d;\n\t"
        "mov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}\n"
        :
        : "r"(taddr), "r"(low), "r"(DESC_SCALES)
        : "memory");
}
// N pieces of 4 words a lane to 4 N columns of this warp's quarter of the lanes
template <int N>
__device__ __forceinline__ void words_to_tmem(uint32_t taddr, const uint4 *v) {
    if constexpr (N >= 4) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
                         taddr),
                     "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w), "r"(v[2].x),
                     "r"(v[2].y), "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w)
                     : "memory");
        if constexpr (N > 4) words_to_tmem<N - 4>(taddr + 16, v + 4);
    } else {
        static_assert(N == 2, "4 or 6 pieces");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0].x), "r"(v[0].y),
                     "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w)
                     : "memory");
    }
}
// instruction descriptor of kind::mxf4: [4,6) scale id of B, [7,10) A and [10,12) B element type (1: e2m1), [17,23) N >> 3,
// [23] scales are powers of two, [27,29) M >> 7, [29,31) scale id of A
__host__ __device__ constexpr uint32_t idesc_mxf4(int N, int half) {
    return ((uint32_t)(2 * half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | (1u << 27) |
           ((uint32_t)(2 * half) << 29);
}
__device__ __forceinline__ void tma_rows(void *dst, const CUtensorMap *map, int x, int y, void *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
// a box of the output from shared memory; what lies outside the output is left out
__device__ __forceinline__ void tma_store(const CUtensorMap *map, int x, int y, const void *src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
                 "r"(smem_u32(src))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void stores_have_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void arrive(void *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive_expect(void *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float remote_f32(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// PLAIN: both matrices are quantised already
template <int BN, bool PLAIN>
struct ProductTile {
    static constexpr int QBLOCKS = (BN + 127) / 128;                      // 128-row pieces of Q's scales
    static constexpr int ROWS = 1 + QBLOCKS;                              // scale rows per thread
    static constexpr int CODES = (PT + BN) * KBYTES;                      // bytes of codes per stage
    static constexpr int SCALES = PLAIN ? 0 : 2 * 512 * ROWS;             // bytes of scales per stage
    static constexpr int AHEAD = 4, GROUP = PLAIN ? 128 * 16 * ROWS : 0;  // PLAIN: 16 bytes of scales per row, for two stages
    static constexpr int STAGE = CODES + SCALES;                          // a multiple of 1024
    static constexpr int SCOLS = 2 * 4 * ROWS;                            // TMEM columns of a stage's scales
    static constexpr int FIT = (SMEM_MAX - SMEM_FIXED - 4 * OUT_BYTES - AHEAD * GROUP) / STAGE;
    static constexpr int MAX_STAGES = FIT > 8 ? 8 : FIT;
    static_assert(STAGE % 1024 == 0, "tiles start on swizzle atoms");
    static_assert(2 * BN + MAX_STAGES * SCOLS <= TMEM_COLS, "two accumulators and the scales fit TMEM");
};

// 16 columns of one row (or, transposed, 16 rows of one column)
template <class O>
__device__ __forceinline__ void product_store(const ProductArgs &a, long long p, long long q0, const float *f) {
    if (p >= a.p) return;
    O *out = static_cast<O *>(a.out);
    if (a.swap) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (q0 + i < a.q) out[(q0 + i) * a.out_stride + p] = from_f32<O>(f[i]);
        return;
    }
    O *row = out + p * a.out_stride + q0;
    if (a.vec && q0 + 16 <= a.q) {
        constexpr int N = 16 / sizeof(O);
#pragma unroll
        for (int i = 0; i < 16; i += N) {
            Vec<O, N> v;
#pragma unroll
            for (int e = 0; e < N; ++e) v.set(e, f[i + e]);
            v.store(row + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (q0 + i < a.q) row[i] = from_f32<O>(f[i]);
    }
}

// The 32 rows of a warp, columns [c, c + 128 bytes) of the accumulator, rounded and laid out as the tensor map's swizzle wants:
// row r's 16-byte piece b at 128 r + 16 (b ^ (r mod 8)).
template <class O>
__device__ __forceinline__ void stage_output(unsigned char *to, uint32_t tmem) {
    constexpr int COLS = 128 / (int)sizeof(O), N = 16 / (int)sizeof(O);
    const int lane = threadIdx.x & 31;
    float f[COLS];
#pragma unroll
    for (int c = 0; c < COLS; c += 16) tmem_ld16(tmem + c, f + c);
    tmem_wait_ld();
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        Vec<O, N> v;
#pragma unroll
        for (int e = 0; e < N; ++e) v.set(e, f[b * N + e]);
        *reinterpret_cast<uint4 *>(to + lane * 128 + ((b ^ (lane & 7)) << 4)) = v.raw[0];
    }
}

// X: the type of a Q that is quantised here, or void
template <int BN, class O, class X>
__global__ void __launch_bounds__(std::is_void_v<X> ? PR_THREADS : X_THREADS) product_kernel(const __grid_constant__ CUtensorMap pmap, const __grid_constant__ CUtensorMap qmap,
                                                             const __grid_constant__ CUtensorMap omap, const ProductArgs a) {
    using Tile = ProductTile<BN, std::is_void_v<X>>;
    constexpr int ROWS = Tile::ROWS;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up, copies;
    __shared__ __align__(8) uint64_t full[8], empty[8], ready[2], taken[2];
    // tiles need 1024-byte alignment; the block's own offset is the same in all blocks of a cluster
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    unsigned char *outs = smem + a.stages * Tile::STAGE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = gridDim.z, rank = blockIdx.z;
    const int all = (a.k + KSTAGE - 1) / KSTAGE, per = part_of_k(all, S);
    const int s0 = min(rank * per, all), s1 = min(s0 + per, all), steps = s1 - s0;
    const unsigned mine = blockIdx.x < a.tiles ? (a.tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;  // tiles of this block
    auto tile_p = [&](unsigned n) { return (long long)((blockIdx.x + n * gridDim.x) % a.ptiles) * PT; };
    auto tile_q = [&](unsigned n) { return (long long)((blockIdx.x + n * gridDim.x) / a.ptiles) * BN; };
    uint32_t cols = 32;
    while (cols < (uint32_t)(a.accs * BN + a.stages * Tile::SCOLS)) cols *= 2;

    if (warp == 9) tmem_alloc(&tmem_slot, cols);
    if (threadIdx.x == 256) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&pmap) : "memory");
        if constexpr (std::is_void_v<X>) asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    }
    if (threadIdx.x == 0) {
        gave_up = copies = 0;
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&full[s], 1 + 4);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ready[b], 1);
            mbar_init(&taken[b], 4);
        }
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, scales = tmem + a.accs * BN;

    if (warp == 8) {
        if (lane == 0) {
            int st = 0, round = 0, issued = 0;
            bool ok = true;
            for (unsigned n = 0; n < mine && ok; ++n) {
                const int y = (int)tile_p(n), z = (int)tile_q(n);
                for (int i = 0; i < steps; ++i) {
                    if (round) ok = mbar_wait(&empty[st], (round - 1) & 1);
                    if (!ok) break;
                    unsigned char *t = smem + st * Tile::STAGE;
                    arrive_expect(&full[st], std::is_void_v<X> ? Tile::CODES : PT * KBYTES);
                    tma_rows(t, &pmap, (s0 + i) * KBYTES, y, &full[st]);
                    if constexpr (std::is_void_v<X>) tma_rows(t + PT * KBYTES, &qmap, (s0 + i) * KBYTES, z, &full[st]);
                    ++issued;
                    if (++st == a.stages) st = 0, ++round;
                }
            }
            copies = issued;
            if (!ok) atomicExch(&gave_up, 1);
        }
    } else if (warp == 9) {
        if (lane == 0) {
            int st = 0, round = 0;
            bool ok = true;
            const uint32_t low0 = desc_low(smem);
            for (unsigned n = 0; n < mine && ok; ++n) {
                const int buf = a.accs == 2 ? n & 1 : 0;
                const unsigned use = a.accs == 2 ? n >> 1 : n;  // how often the accumulator was used before
                if (use) ok = mbar_wait(&taken[buf], (use - 1) & 1);
                const uint32_t d = tmem + buf * BN;
                for (int i = 0; i < steps && ok; ++i) {
                    ok = mbar_wait(&full[st], round & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t t = low0 + st * (Tile::STAGE / 16), scol = scales + st * Tile::SCOLS;
                    // half h of the stage: the word of P's rows, then those of Q's
                    if constexpr (!std::is_void_v<X>)
#pragma unroll
                        for (int b = 0; b < 2 * ROWS; ++b) scales_to_tmem(scol + 4 * b, t + Tile::CODES / 16 + 32 * b);
                    const int left = a.k - (s0 + i) * KSTAGE;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        if (m * 64 >= left) break;
                        const uint32_t sa = scol + (m / 2) * 4 * ROWS;
                        mma_mxf4(d, t + 2 * m, t + PT * KBYTES / 16 + 2 * m, idesc_mxf4(BN, m & 1), sa, sa + 4, (i | m) != 0);
                    }
                    mma_commit(&empty[st]);
                    if (++st == a.stages) st = 0, ++round;
                }
                if (!ok) {  // known before the tile counts as ready
                    atomicExch(&gave_up, 1);
                    __threadfence_block();
                }
                mma_commit(&ready[buf]);
            }
        }
    } else if (warp >= 4 && !std::is_void_v<X>) {
        if constexpr (!std::is_void_v<X>) {
            // thread r of a team has row r of P's scales, two words a stage, and block r mod 8 of row r / 8 of Q
            constexpr int AHEAD = 2;
            const int team = warp < 8 ? 0 : 1 + (warp - 10) / 4, r = (warp < 8 ? warp - 4 : (warp - 10) & 3) * 32 + lane;
            const int qr = r >> 3, qb = r & 7, total = (int)mine * steps;
            unsigned w[AHEAD][2];
            Raw32<X> x[AHEAD];
            unsigned fn = 0;
            int fi = team;
            auto fetch = [&](unsigned (&word)[2], Raw32<X> &raw) {
                while (fi >= steps && fn < mine) fi -= steps, ++fn;
                if (fn >= mine) return;
                const long long row = tile_p(fn) + r;
                const int first = (s0 + fi) * 2, e0 = (s0 + fi) * KSTAGE + qb * 32;
                word[0] = word[1] = 0;
                if (row < a.p) {
                    const unsigned *src = reinterpret_cast<const unsigned *>(a.ps + row * a.pitch);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int left = a.blocks - 4 * (first + h);
                        if (left > 0) word[h] = __ldg(src + first + h) & (left < 4 ? (1u << (8 * left)) - 1u : 0xffffffffu);
                    }
                }
                raw.load(static_cast<const X *>(a.x) + qr * a.x_stride + e0, qr < a.q ? a.k - e0 : 0, a.x_vec);
                fi += X_TEAMS;
            };
            if (total)
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) fetch(w[u], x[u]);
            int st = team, round = 0;
            bool ok = true;
            for (int i0 = team; i0 < total && ok; i0 += AHEAD * X_TEAMS)
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    if (i0 + u * X_TEAMS >= total || !ok) break;
                    while (st >= a.stages) st -= a.stages, ++round;
                    if (round) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (round - 1) & 1));
                    if (!ok) break;
                    unsigned char *t = smem + st * Tile::STAGE, *sc = t + Tile::CODES;
                    const int at = (r & 31) * 16 + (r >> 5) * 4;
                    *reinterpret_cast<unsigned *>(sc + at) = w[u][0];
                    *reinterpret_cast<unsigned *>(sc + ROWS * 512 + at) = w[u][1];
                    unsigned byte;
                    const uint4 codes = x[u].quantize(&byte);
                    *reinterpret_cast<uint4 *>(t + PT * KBYTES + qr * 128 + ((qb ^ (qr & 7)) << 4)) = codes;
                    sc[((qb >> 2) * ROWS + 1) * 512 + qr * 16 + (qb & 3)] = (unsigned char)byte;
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) arrive(&full[st]);
                    st += X_TEAMS;
                    fetch(w[u], x[u]);
                }
            if (!ok && lane == 0) atomicExch(&gave_up, 1);
        }
    } else if (warp >= 4) {
        // thread r copies the scales of row r of P and rows r, r + 128 of Q, 4 words (2 stages) at a time: groups (tile, pair of
        // stages), in a ring of AHEAD.  Lane l of each warp then has the words of rows l + 32 j, which are columns j of its quarter.
        constexpr int AHEAD = Tile::AHEAD;
        const int r = threadIdx.x - 128, pairs = (steps + 1) / 2, words = a.pitch / 4;
        const unsigned groups = mine * (unsigned)pairs;
        unsigned char *ring = outs + 4 * OUT_BYTES;
        unsigned ftile = 0, fgroup = 0;
        int fpair = 0;
        const unsigned *src[ROWS];  // of the tile being fetched
        bool some[ROWS];
        auto fetch = [&] {
            if (fgroup < groups) {
                if (fpair == 0) {
                    const long long p0 = tile_p(ftile), q0 = tile_q(ftile);
#pragma unroll
                    for (int b = 0; b < ROWS; ++b) {
                        const int o = b ? (b - 1) * 128 + r : r;
                        const long long row = (b ? q0 : p0) + o;
                        some[b] = row < (b ? a.q : a.p) && (!b || o < BN);
                        src[b] = reinterpret_cast<const unsigned *>((b ? a.qs : a.ps) + (some[b] ? row * a.pitch : 0)) + s0 * 2;
                    }
                }
                const int left = words - (s0 * 2 + 4 * fpair);  // of the row, at least 1
                const uint32_t to = smem_u32(ring) + (fgroup % AHEAD) * Tile::GROUP + r * 16;
#pragma unroll
                for (int b = 0; b < ROWS; ++b) {
                    if (a.wide) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + b * 2048), "l"(src[b]), "r"(some[b] ? 16 : 0)
                                     : "memory");
                    } else {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const bool in = some[b] && w < left;
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + b * 2048 + w * 4), "l"(src[b] + (in ? w : 0)),
                                         "r"(in ? 4 : 0)
                                         : "memory");
                        }
                    }
                    src[b] += 4;
                }
                if (++fpair == pairs) fpair = 0, ++ftile;
            }
            ++fgroup;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int u = 0; u < AHEAD - 1; ++u) fetch();
        int st = 0, round = 0, pair = 0;
        bool ok = true;
        const uint32_t quarter = scales + ((uint32_t)((warp & 3) * 32) << 16);
        // a warp whose wait ran out still meets the others at every barrier
        for (unsigned g = 0; g < groups; ++g) {
            asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 2) : "memory");
            asm volatile("bar.sync 1, 128;" ::: "memory");
            fetch();  // into the place that all four warps have read
            const uint4 *from = reinterpret_cast<const uint4 *>(ring + (g % AHEAD) * Tile::GROUP) + lane;
            uint4 v[ROWS][4];
#pragma unroll
            for (int b = 0; b < ROWS; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[b][j] = from[b * 128 + j * 32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * pair + h;
                if (i >= steps) break;
                if (round && ok) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (round - 1) & 1));
                if (ok) {
                    tc_fence_after();
                    // bytes past the last block are not scales
                    const int left = a.blocks - (s0 + i) * 8;
                    const unsigned lo = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
                    const unsigned hi = left >= 8 ? 0xffffffffu : left > 4 ? (1u << (8 * (left - 4))) - 1u : 0u;
                    uint4 piece[2 * ROWS];
#pragma unroll
                    for (int b = 0; b < ROWS; ++b) {
                        const uint4 *x = v[b];
                        piece[b] = h ? make_uint4(x[0].z & lo, x[1].z & lo, x[2].z & lo, x[3].z & lo)
                                     : make_uint4(x[0].x & lo, x[1].x & lo, x[2].x & lo, x[3].x & lo);
                        piece[ROWS + b] = h ? make_uint4(x[0].w & hi, x[1].w & hi, x[2].w & hi, x[3].w & hi)
                                            : make_uint4(x[0].y & hi, x[1].y & hi, x[2].y & hi, x[3].y & hi);
                    }
                    words_to_tmem<2 * ROWS>(quarter + st * Tile::SCOLS, piece);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(&full[st]);
                }
                if (++st == a.stages) st = 0, ++round;
            }
            if (++pair == pairs) pair = 0;
        }
        if (!ok && lane == 0) atomicExch(&gave_up, 1);
    } else if (S == 1) {
        constexpr int OC = 128 / (int)sizeof(O);  // output columns of 128 bytes
        unsigned char *out = outs + warp * OUT_BYTES;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        bool ok = true;
        for (unsigned n = 0; n < mine; ++n) {
            const int buf = a.accs == 2 ? n & 1 : 0;
            const unsigned use = a.accs == 2 ? n >> 1 : n;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&ready[buf], use & 1));
            // a wait that ran out before this tile's commit shows here
            if (*(volatile int *)&gave_up) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const long long p0 = tile_p(n), q0 = tile_q(n);
            const uint32_t d = tmem + lanes + buf * BN;
            if (ok && a.bulk && BN >= OC) {
                for (int c = 0; c < BN && q0 + c < a.q && p0 + warp * 32 < a.p; c += OC) {
                    if (lane == 0) stores_have_read();
                    __syncwarp();
                    stage_output<O>(out, d + c);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) tma_store(&omap, (int)(q0 + c), (int)p0 + warp * 32, out);
                }
            } else {
#pragma unroll 2
                for (int c = 0; c < BN; c += 16) {
                    float f[16];
                    tmem_ld16(d + c, f);
                    tmem_wait_ld();
                    if (!ok)
#pragma unroll
                        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(0x7fc00000u);
                    if (q0 + c < a.q) product_store<O>(a, p0 + threadIdx.x, q0 + c, f);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&taken[buf]);
        }
        if (!ok && lane == 0) atomicExch(&gave_up, 1);
        if (lane == 0) stores_done();
    } else {
        if (!mbar_wait(&ready[0], 0)) atomicExch(&gave_up, 1);
        tc_fence_after();
    }
    __syncthreads();
    const bool bad = *(volatile int *)&gave_up != 0;
    if (bad && threadIdx.x == 0) {
        // copies may still be under way: they end before the block's shared memory is let go
        for (int i = max(0, copies - a.stages); i < copies; ++i) mbar_wait(&full[i % a.stages], (i / a.stages) & 1);
        if (a.status) atomicOr(a.status, (int)ERR_MBAR);
    }
    if (S > 1) {
        // every block leaves its tile in its shared memory (the stages are free), then adds a share of the columns
        float *part = reinterpret_cast<float *>(smem);
        if (warp < 4) {
            for (int c = 0; c < BN; c += 16) {
                float f[16];
                tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, f);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(c + i) * PT + threadIdx.x] = bad ? __uint_as_float(0x7fc00000u) : steps ? f[i] : 0.0f;
            }
        }
        cluster_sync();
        if (warp < 4) {
            const long long p = tile_p(0) + threadIdx.x, q0 = tile_q(0);
            O *out = static_cast<O *>(a.out);
            for (int c = rank; c < BN; c += S) {
                const long long q = q0 + c;
                if (q >= a.q || p >= a.p) continue;
                float v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = r < S ? remote_f32(smem_u32(part + c * PT + threadIdx.x), r) : 0.0f;
                float t = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; ++r) t += v[r];
                out[a.swap ? q * a.out_stride + p : p * a.out_stride + q] = from_f32<O>(t);
            }
        }
        cluster_sync();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, cols);
}

// ------------------------------------------------------------------------------------------------
// One stage of K (k <= 256) and one tile of Q: a small layer over very many rows.  Q and its scales stay in shared memory and
// TMEM; what moves is P, 16 ceil(k / 32) contiguous bytes a row, and the output.  TMA takes such short rows one by one (147
// us for 1M x 64 x 96), so warps 4-7 copy P's tile by 16-byte asynchronous copies, consecutive threads consecutive pieces, into
// the swizzled layout, NARROW_AHEAD tiles ahead.  Pieces past a row's end stay zero from the start.
// ------------------------------------------------------------------------------------------------
constexpr int NARROW_STAGES = 4, NARROW_AHEAD = 2, NARROW_BLOCKS = 2;  // blocks per multiprocessor

template <int BN>
struct NarrowTile {
    static constexpr int P = PT * KBYTES, PS = 2 * 512;              // a stage: codes, scales
    static constexpr int Q = BN * KBYTES, QS = 2 * 512;
    static constexpr int ACCS = BN > 64 ? 1 : 2;                     // two blocks share TMEM
    static constexpr int COLS = ACCS * BN + 8 * NARROW_STAGES + 8 <= 64 ? 64 : ACCS * BN + 8 * NARROW_STAGES + 8 <= 128 ? 128 : 256;
    static constexpr int SMEM = 1024 + Q + NARROW_STAGES * P + NARROW_STAGES * PS + QS + 4 * OUT_BYTES;
    static_assert(BN <= 128 && ACCS * BN + 8 * NARROW_STAGES + 8 <= 256, "TMEM of two blocks");
};

template <int BN, class O>
__global__ void __launch_bounds__(PR_THREADS, NARROW_BLOCKS) product_narrow_kernel(const __grid_constant__ CUtensorMap omap, const unsigned char *pc,
                                                                                   const unsigned char *qc, const ProductArgs a) {
    using Tile = NarrowTile<BN>;
    constexpr int ST = NARROW_STAGES;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    __shared__ __align__(8) uint64_t full[ST], empty[ST], ready[2], taken[2];
    unsigned char *qtile = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    unsigned char *ptile = qtile + Tile::Q, *outs = ptile + ST * Tile::P;
    unsigned char *pscale = outs + 4 * OUT_BYTES, *qscale = pscale + ST * Tile::PS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned mine = blockIdx.x < a.tiles ? (a.tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    auto tile_p = [&](unsigned n) { return (long long)(blockIdx.x + n * gridDim.x) * PT; };
    // byte of piece b (16 bytes) of row r in a 128-byte-swizzled tile
    auto place = [](int r, int b) { return r * 128 + ((b ^ (r & 7)) << 4); };
    // half h of 128 rows' scales: row r's word
    auto scale_place = [](int r, int h) { return h * 512 + (r & 31) * 16 + (r >> 5) * 4; };
    auto scale_word = [&](const unsigned char *scales, long long row, int h) {
        const int left = a.blocks - 4 * h;
        if (left <= 0) return 0u;
        const unsigned v = __ldg(reinterpret_cast<const unsigned *>(scales + row * a.pitch) + h);
        return left < 4 ? v & ((1u << (8 * left)) - 1u) : v;  // bytes past the last block are not scales
    };

    if (warp == 9) tmem_alloc(&tmem_slot, Tile::COLS);
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 4);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ready[b], 1);
            mbar_init(&taken[b], 4);
        }
        fence_mbar_init();
    }
    // Q, and zeros where P's rows have no pieces
    for (int c = threadIdx.x; c < BN * 8; c += PR_THREADS) {
        const int r = c >> 3, b = c & 7;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (b < a.blocks && r < a.q) v = __ldg(reinterpret_cast<const uint4 *>(qc + (long long)r * 16 * a.blocks) + b);
        *reinterpret_cast<uint4 *>(qtile + place(r, b)) = v;
    }
    for (int c = threadIdx.x; c < 256; c += PR_THREADS) {
        const int r = c & 127, h = c >> 7;
        *reinterpret_cast<unsigned *>(qscale + scale_place(r, h)) = r < BN && r < a.q ? scale_word(a.qs, r, h) : 0u;
    }
    for (int c = threadIdx.x; c < ST * PT * 8; c += PR_THREADS)
        if ((c & 7) >= a.blocks) *reinterpret_cast<uint4 *>(ptile + (c >> 10) * Tile::P + place((c >> 3) & 127, c & 7)) = make_uint4(0, 0, 0, 0);
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, pscol = tmem + Tile::ACCS * BN, qscol = pscol + 8 * ST;

    if (warp == 9) {
        if (lane == 0) {
            bool ok = true;
            const uint32_t qlow = desc_low(qtile), plow = desc_low(ptile), slow = desc_low(pscale);
            for (int h = 0; h < 2; ++h) scales_to_tmem(qscol + 4 * h, desc_low(qscale) + 32 * h);
            for (unsigned n = 0; n < mine && ok; ++n) {
                const int st = n % ST, buf = n % Tile::ACCS;
                const unsigned use = n / Tile::ACCS;
                if (use) ok = mbar_wait(&taken[buf], (use - 1) & 1);
                if (ok) ok = mbar_wait(&full[st], (n / ST) & 1);
                if (ok) {
                    tc_fence_after();
                    const uint32_t t = plow + st * (Tile::P / 16), scol = pscol + 8 * st;
#pragma unroll
                    for (int h = 0; h < 2; ++h) scales_to_tmem(scol + 4 * h, slow + st * (Tile::PS / 16) + 32 * h);
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        if (m * 64 < a.k)
                            mma_mxf4(tmem + buf * BN, t + 2 * m, qlow + 2 * m, idesc_mxf4(BN, m & 1), scol + (m / 2) * 4, qscol + (m / 2) * 4, m != 0);
                    mma_commit(&empty[st]);
                } else {
                    atomicExch(&gave_up, 1);
                    __threadfence_block();
                }
                mma_commit(&ready[buf]);
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const int r = threadIdx.x - 128;
        // this thread's pieces of a tile, at most 8: piece c of the tile's contiguous bytes
        int to[8], row[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = j * 128 + r;
            row[j] = j < a.blocks ? c / a.blocks : 0;
            to[j] = j < a.blocks ? place(row[j], c - row[j] * a.blocks) : 0;
        }
        bool ok = true;
        unsigned w0 = 0, w1 = 0;
        auto words = [&](unsigned n) {
            w0 = w1 = 0;
            if (n < mine && tile_p(n) + r < a.p) {
                w0 = scale_word(a.ps, tile_p(n) + r, 0);
                w1 = scale_word(a.ps, tile_p(n) + r, 1);
            }
        };
        words(0);
        for (unsigned n = 0; n < mine + NARROW_AHEAD && ok; ++n) {
            if (n < mine) {
                const int st = n % ST;
                if (n >= ST) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (n / ST - 1) & 1));
                if (!ok) break;
                const long long p0 = tile_p(n);
                const unsigned char *from = pc + p0 * 16 * a.blocks + r * 16;
                const uint32_t at = smem_u32(ptile + st * Tile::P);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    // rows past the last are left as they are: their outputs are not stored
                    if (j < a.blocks && p0 + row[j] < a.p)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + to[j]), "l"(from + j * 2048) : "memory");
                unsigned char *sc = pscale + st * Tile::PS;
                *reinterpret_cast<unsigned *>(sc + scale_place(r, 0)) = w0;
                *reinterpret_cast<unsigned *>(sc + scale_place(r, 1)) = w1;
                words(n + 1);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (n >= NARROW_AHEAD) {
                asm volatile("cp.async.wait_group %0;" ::"n"(NARROW_AHEAD) : "memory");
                fence_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&full[(n - NARROW_AHEAD) % ST]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (!ok && lane == 0) atomicExch(&gave_up, 1);
    } else if (warp < 4) {
        constexpr int OC = 128 / (int)sizeof(O);
        unsigned char *out = outs + warp * OUT_BYTES;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        bool ok = true;
        for (unsigned n = 0; n < mine; ++n) {
            const int buf = n % Tile::ACCS;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&ready[buf], (n / Tile::ACCS) & 1));
            if (*(volatile int *)&gave_up) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const long long p0 = tile_p(n);
            const uint32_t d = tmem + lanes + buf * BN;
            if (ok && a.bulk && BN >= OC) {
                for (int c = 0; c < BN && c < a.q && p0 + warp * 32 < a.p; c += OC) {
                    if (lane == 0) stores_have_read();
                    __syncwarp();
                    stage_output<O>(out, d + c);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) tma_store(&omap, c, (int)p0 + warp * 32, out);
                }
            } else {
#pragma unroll 2
                for (int c = 0; c < BN; c += 16) {
                    float f[16];
                    tmem_ld16(d + c, f);
                    tmem_wait_ld();
                    if (!ok)
#pragma unroll
                        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(0x7fc00000u);
                    if (c < a.q) product_store<O>(a, p0 + threadIdx.x, c, f);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive(&taken[buf]);
        }
        if (!ok && lane == 0) atomicExch(&gave_up, 1);
        if (lane == 0) stores_done();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *(volatile int *)&gave_up && a.status) atomicOr(a.status, (int)ERR_MBAR);
    if (warp == 9) tmem_dealloc(tmem, Tile::COLS);
}

// ------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess) return (EncodeTiled) nullptr;
        return q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : (EncodeTiled) nullptr;
    }();
    return fn;
}

// rows of `cols` elements, in boxes of 128 bytes by box_rows
int matrix_map(CUtensorMap *map, CUtensorMapDataType type, int size, const void *p, long long rows, long long cols, long long stride, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) {
        set_error("flare_micro_product: the driver has no cuTensorMapEncodeTiled");
        return FLARE_E_CUDA;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(stride * size)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = encode(map, type, 2, const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("flare_micro_product: tensor map of %lld rows of %lld: error %d", rows, cols, (int)r);
        return FLARE_E_CUDA;
    }
    return FLARE_OK;
}

template <int BN, class O, class X>
int launch_product(const CUtensorMap &pm, const CUtensorMap &qm, const CUtensorMap &om, ProductArgs a, int split, cudaStream_t st) {
    using Tile = ProductTile<BN, std::is_void_v<X>>;
    const int per = part_of_k((a.k + KSTAGE - 1) / KSTAGE, split);
    a.ptiles = (unsigned)((a.p + PT - 1) / PT);
    const long long tiles = (long long)a.ptiles * ((a.q + BN - 1) / BN);
    if (tiles > 0x7fffffff) {
        set_error("flare_micro_product: %lld tiles", tiles);
        return FLARE_E_INVALID;
    }
    a.tiles = (unsigned)tiles;
    const unsigned grid = split > 1 ? a.tiles : (unsigned)std::min<long long>(tiles, SMS);
    a.accs = grid < a.tiles ? 2 : 1;
    // no more stages than the block's tiles have
    a.stages = (int)std::min<long long>(Tile::MAX_STAGES, per * ((tiles + grid - 1) / grid));
    int smem = a.stages * Tile::STAGE + 4 * OUT_BYTES + Tile::AHEAD * Tile::GROUP + 1024;
    if (split > 1) smem = std::max(smem, PT * BN * 4 + 1024);
    const int e0 = allow_shared_memory<product_kernel<BN, O, X>>("flare_micro_product");
    if (e0) return e0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, 1, (unsigned)split);
    cfg.blockDim = dim3(std::is_void_v<X> ? PR_THREADS : X_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = (unsigned)split;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, product_kernel<BN, O, X>, pm, qm, om, a);
    if (e != cudaSuccess) {
        set_error("flare_micro_product: %s", cudaGetErrorString(e));
        return FLARE_E_CUDA;
    }
    return FLARE_OK;
}

template <int BN, class O>
int launch_narrow(const CUtensorMap &om, const unsigned char *pc, const unsigned char *qc, ProductArgs a, cudaStream_t st) {
    a.tiles = (unsigned)((a.p + PT - 1) / PT);
    const int e = allow_shared_memory<product_narrow_kernel<BN, O>>("flare_micro_product");
    if (e) return e;
    product_narrow_kernel<BN, O><<<std::min(a.tiles, (unsigned)(NARROW_BLOCKS * SMS)), PR_THREADS, NarrowTile<BN>::SMEM, st>>>(om, pc, qc, a);
    OPS_LAUNCHED("flare_micro_product");
    return FLARE_OK;
}

int run_product(const flare_product_args *in, cudaStream_t st) {
    ProductArgs a{};
    a.swap = in->m < in->n || in->x;  // the larger matrix gives the tiles' 128 rows
    const unsigned char *pc = a.swap ? in->b_codes : in->a_codes, *qc = a.swap ? in->a_codes : in->b_codes;
    a.ps = a.swap ? in->b_scales : in->a_scales;
    a.qs = a.swap ? in->a_scales : in->b_scales;
    a.p = a.swap ? in->n : in->m;
    a.q = a.swap ? in->m : in->n;
    a.out = in->out;
    a.status = in->status;
    a.out_stride = in->out_stride;
    a.x = in->x;
    a.x_stride = in->x_stride;
    a.x_vec = in->x && fits_vec(in->x, in->x_stride, type_size(in->x_type), 16 / type_size(in->x_type));
    a.k = in->k;
    a.blocks = (in->k + 31) / 32;
    a.pitch = 4 * ((a.blocks + 3) / 4);
    a.wide = a.pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(a.ps) | reinterpret_cast<uintptr_t>(a.qs)) % 16 == 0;
    const int size = type_size(in->out_type);
    a.vec = fits_vec(in->out, in->out_stride, size, 16 / size);
    const CUtensorMapDataType out_map = size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    CUtensorMap pm, qm, om{};
    int e = FLARE_OK;
    // one stage of K and one tile of Q, over at least two tiles a multiprocessor
    if (!in->x && in->k <= KSTAGE && a.q <= 128 && a.p >= 2ll * SMS * PT) {
        int bn = 16;
        while (bn < a.q) bn *= 2;
        a.bulk = !a.swap && a.vec && bn * size >= 128;
        if (a.bulk) e = matrix_map(&om, out_map, size, in->out, in->m, in->n, in->out_stride, 32);
        if (e) return e;
        return with_type(in->out_type, [&](auto t) {
            using O = typename decltype(t)::type;
            switch (bn) {
                case 16: return launch_narrow<16, O>(om, pc, qc, a, st);
                case 32: return launch_narrow<32, O>(om, pc, qc, a, st);
                case 64: return launch_narrow<64, O>(om, pc, qc, a, st);
                default: return launch_narrow<128, O>(om, pc, qc, a, st);
            }
        });
    }
    // columns per tile: what Q has, at most 192 (two accumulators of 192 and the scales fill TMEM); narrower where that leaves
    // multiprocessors without a tile
    int bn = 16;
    while (bn < 128 && bn < a.q) bn *= 2;
    const long long ptiles = (a.p + PT - 1) / PT;
    auto tiles = [&](int b) { return ptiles * ((a.q + b - 1) / b); };
    if (bn < a.q && tiles(192) >= SMS) bn = 192;
    while (bn > 64 && tiles(bn) < SMS) bn /= 2;
    // and then parts of K
    const int split = parts_of_k((in->k + KSTAGE - 1) / KSTAGE, tiles(bn), (int)std::min<long long>(a.q, bn), in->x != nullptr,
                                 a.swap ? Store::columns : a.vec ? Store::rows_of_16 : Store::rows);
    // whole 128-byte pieces of output rows go by TMA
    a.bulk = !a.swap && split == 1 && a.vec && bn * size >= 128;
    e = matrix_map(&pm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pc, a.p, 16ll * a.blocks, 16ll * a.blocks, PT);
    if (!e && !in->x) e = matrix_map(&qm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, qc, a.q, 16ll * a.blocks, 16ll * a.blocks, bn);
    if (!e && a.bulk)
        e = matrix_map(&om, out_map, size, in->out, in->m, in->n, in->out_stride, 32);
    if (e) return e;
    return with_type(in->out_type, [&](auto t) {
        using O = typename decltype(t)::type;
        if (in->x)
            return with_type(in->x_type, [&](auto x) { return launch_product<16, O, typename decltype(x)::type>(pm, qm, om, a, split, st); });
        switch (bn) {
            case 16: return launch_product<16, O, void>(pm, qm, om, a, split, st);
            case 32: return launch_product<32, O, void>(pm, qm, om, a, split, st);
            case 64: return launch_product<64, O, void>(pm, qm, om, a, split, st);
            case 128: return launch_product<128, O, void>(pm, qm, om, a, split, st);
            default: return launch_product<192, O, void>(pm, qm, om, a, split, st);
        }
    });
}

}  // namespace flare

using namespace flare;

extern "C" {

long long flare_micro_product_workspace(long long m, long long n, int k) {
    (void)m, (void)n, (void)k;
    return 0;  // blocks that share a tile add up in their shared memory
}

int flare_micro_product(const flare_product_args *a, void *stream) {
    OPS_CHECK(a, "flare_micro_product: NULL argument");
    OPS_CHECK(is_float_type(a->out_type), "flare_micro_product: unknown type %d", a->out_type);
    OPS_CHECK(a->m >= 0 && a->n >= 0 && a->k >= 1 && a->k <= (1 << 30), "flare_micro_product: %lld x %lld x %d", a->m, a->n, a->k);
    OPS_CHECK(a->m < 0x40000000ll && a->n < 0x40000000ll, "flare_micro_product: %lld x %lld outputs", a->m, a->n);
    if (a->m == 0 || a->n == 0) return FLARE_OK;
    OPS_CHECK(((a->a_codes && a->a_scales) || a->x) && a->b_codes && a->b_scales && a->out, "flare_micro_product: NULL buffer");
    OPS_CHECK(!a->x || (is_float_type(a->x_type) && a->m <= FLARE_PRODUCT_ROWS && a->x_stride >= a->k),
              "flare_micro_product: x of type %d, %lld rows (at most %d) of stride %lld", a->x_type, a->m, FLARE_PRODUCT_ROWS, a->x_stride);
    OPS_CHECK(a->out_stride >= a->n, "flare_micro_product: output rows of stride %lld overlap", a->out_stride);
    for (const void *p : {(const void *)a->a_codes, (const void *)a->b_codes})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0, "flare_micro_product: codes must be 16-byte aligned");
    for (const void *p : {(const void *)a->a_scales, (const void *)a->b_scales})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 4 == 0, "flare_micro_product: scales must be 4-byte aligned");
    return run_product(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
