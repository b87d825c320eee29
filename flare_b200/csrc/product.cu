// product.cu -- out = A B^T of two matrices held in microscaled 4-bit floats, on the tensor cores.
//
// tcgen05.mma kind::mxf4 multiplies 4-bit elements and applies the block scales itself: D (TMEM, f32) += (A * 2^sa)
// (B * 2^sb)^T for 64 elements of K at a time, two scales per row.  The larger matrix gives the 128 rows of a tile (P), the
// other its BN columns (Q); where that is B, the tile is stored transposed.  Per 256 elements of K (a stage):
//   * warp 4 brings the codes, 128 bytes a row, by TMA into 128-byte-swizzled tiles;
//   * warps 0-3 bring the scales, a word (128 elements of K) per row and half stage, into the order that tcgen05.cp spreads
//     over TMEM: 32 rows of 16 bytes, row r the words of tile rows r, r + 32, r + 64, r + 96;
//   * warp 5 copies the scales to TMEM and issues the products; its commit frees the stage.
// Then warps 0-3 read D from TMEM, a row per thread, and store it rounded once.  Few tiles and a long K: up to 8 blocks of a
// cluster take a part of K each and add their tiles through distributed shared memory, in order.
// Every wait is bounded; a block in which one ran out stores NaN and sets a bit of the status word.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "ops.cuh"
#include "umma.cuh"

namespace flare {

constexpr int PT = 128;          // rows of P per tile
constexpr int KSTAGE = 256;      // elements of K per stage
constexpr int KBYTES = KSTAGE / 2;
constexpr int PR_THREADS = 192;
constexpr int SMEM_MAX = 227 * 1024, SMEM_HEAD = 1024;

struct ProductArgs {
    const unsigned char *ps, *qs;
    void *out;
    int *status;
    long long p, q, out_stride;
    int k, blocks, pitch;   // blocks of 32 per row, scale bytes per row
    int stages, swap, vec;  // vec: 16-byte stores of a row's columns are aligned
};

// D (+)= A B^T, 64 elements of K; the scales' columns in TMEM, which half of their words in idesc
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
        :
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
        : "memory");
}
// 32 rows x 16 bytes of shared memory to 4 columns of TMEM, the same in all four quarters of the lanes
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// instruction descriptor of kind::mxf4: [4,6) scale id of B, [7,10) A and [10,12) B element type (1: e2m1), [17,23) N >> 3,
// [23] scales are powers of two, [27,29) M >> 7, [29,31) scale id of A
__host__ __device__ constexpr uint32_t idesc_mxf4(int N, int half) {
    return ((uint32_t)(2 * half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | (1u << 27) |
           ((uint32_t)(2 * half) << 29);
}
// matrix descriptor of a K-major tile of 128-byte rows, 128-byte swizzle: 8 rows are 1024 bytes
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) { return sdesc(saddr, 16, 1024) | (2ull << 61); }

__device__ __forceinline__ void tma_rows(void *dst, const CUtensorMap *map, int x, int y, void *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
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

template <int BN>
struct ProductTile {
    static constexpr int QBLOCKS = (BN + 127) / 128;                      // 128-row pieces of Q's scales
    static constexpr int CODES = (PT + BN) * KBYTES;                      // bytes of codes per stage
    static constexpr int SCALES = 2 * 512 * (1 + QBLOCKS);                // bytes of scales per stage
    static constexpr int STAGE = CODES + SCALES;                          // a multiple of 1024
    static constexpr int SCOLS = 2 * 4 * (1 + QBLOCKS);                   // TMEM columns of a stage's scales
    static constexpr int MAX_STAGES = (SMEM_MAX - SMEM_HEAD - 1024) / STAGE > 8 ? 8 : (SMEM_MAX - SMEM_HEAD - 1024) / STAGE;
    static_assert(STAGE % 1024 == 0, "tiles start on swizzle atoms");
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

template <int BN, class O>
__global__ void __launch_bounds__(PR_THREADS) product_kernel(const __grid_constant__ CUtensorMap pmap,
                                                             const __grid_constant__ CUtensorMap qmap, const ProductArgs a) {
    using Tile = ProductTile<BN>;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up, copies;
    __shared__ __align__(8) uint64_t full[8], empty[8], done;
    // tiles need 1024-byte alignment; the block's own offset is the same in all blocks of a cluster
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = gridDim.z, rank = blockIdx.z;
    const long long p0 = (long long)blockIdx.x * PT, q0 = (long long)blockIdx.y * BN;
    const int all = (a.k + KSTAGE - 1) / KSTAGE;
    const int per = (all + S - 1) / S;
    const int s0 = min(rank * per, all), s1 = min(s0 + per, all), steps = s1 - s0;
    uint32_t cols = 32;
    while (cols < (uint32_t)(BN + a.stages * Tile::SCOLS)) cols *= 2;

    if (warp == 5) tmem_alloc(&tmem_slot, cols);
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&full[s], 1 + 4);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 4) {
        if (lane == 0) {
            int issued = 0;
            for (; issued < steps; ++issued) {
                const int st = issued % a.stages, round = issued / a.stages;
                if (round && !mbar_wait(&empty[st], (round - 1) & 1)) {
                    atomicExch(&gave_up, 1);
                    break;
                }
                unsigned char *t = smem + st * Tile::STAGE;
                arrive_expect(&full[st], Tile::CODES);
                tma_rows(t, &pmap, (s0 + issued) * KBYTES, (int)p0, &full[st]);
                tma_rows(t + PT * KBYTES, &qmap, (s0 + issued) * KBYTES, (int)q0, &full[st]);
            }
            copies = issued;
        }
    } else if (warp == 5) {
        if (lane == 0) {
            bool ok = true;
            for (int i = 0; i < steps && ok; ++i) {
                const int st = i % a.stages;
                ok = mbar_wait(&full[st], (i / a.stages) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t t = smem_u32(smem + st * Tile::STAGE), sc = t + Tile::CODES;
                const uint32_t scol = tmem + BN + st * Tile::SCOLS;
                // half h of the stage: the word of P's rows, then those of Q's
#pragma unroll
                for (int b = 0; b < 2 * (1 + Tile::QBLOCKS); ++b) scales_to_tmem(scol + 4 * b, sdesc(sc + 512 * b, 16, 128));
                const int left = a.k - (s0 + i) * KSTAGE;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    if (m * 64 >= left) break;
                    const uint32_t sa = scol + (m / 2) * 4 * (1 + Tile::QBLOCKS);
                    mma_mxf4(tmem, desc_sw128(t + m * 32), desc_sw128(t + PT * KBYTES + m * 32), idesc_mxf4(BN, m & 1), sa, sa + 4,
                             (i | m) != 0);
                }
                mma_commit(&empty[st]);
            }
            if (!ok) atomicExch(&gave_up, 1);
            mma_commit(&done);
        }
    } else {
        // scales: thread r has row r of P and rows r, r + 128 of Q; the words of 4 stages are loaded together, one such group ahead
        constexpr int G = 4, ROWS = 1 + Tile::QBLOCKS;
        const unsigned *src[ROWS];
        src[0] = p0 + threadIdx.x < a.p ? reinterpret_cast<const unsigned *>(a.ps + (p0 + threadIdx.x) * a.pitch) : nullptr;
#pragma unroll
        for (int b = 0; b < Tile::QBLOCKS; ++b) {
            const int r = b * 128 + threadIdx.x;
            src[1 + b] = r < BN && q0 + r < a.q ? reinterpret_cast<const unsigned *>(a.qs + (q0 + r) * a.pitch) : nullptr;
        }
        unsigned next[G][ROWS][2], cur[G][ROWS][2];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int b = 0; b < ROWS; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int word = (s0 + i0 + g) * 2 + h, left = a.blocks - word * 4;
                        unsigned v = 0;
                        if (src[b] && i0 + g < steps && left > 0) {
                            v = __ldg(src[b] + word);
                            if (left < 4) v &= (1u << (8 * left)) - 1u;  // bytes past the last block are not scales
                        }
                        next[g][b][h] = v;
                    }
        };
        fetch(0);
        bool ok = true;
        for (int i0 = 0; i0 < steps && ok; i0 += G) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int b = 0; b < ROWS; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) cur[g][b][h] = next[g][b][h];
            if (i0 + G < steps) fetch(i0 + G);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int i = i0 + g;
                if (i >= steps || !ok) break;
                const int st = i % a.stages, round = i / a.stages;
                if (round) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (round - 1) & 1));
                if (!ok) break;
                unsigned *sc = reinterpret_cast<unsigned *>(smem + st * Tile::STAGE + Tile::CODES);
                const int at = (threadIdx.x & 31) * 4 + warp;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int b = 0; b < ROWS; ++b) sc[(h * ROWS + b) * 128 + at] = cur[g][b][h];
                fence_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&full[st]);
            }
        }
        if (!ok && lane == 0) atomicExch(&gave_up, 1);
        if (!mbar_wait(&done, 0)) atomicExch(&gave_up, 1);
        tc_fence_after();
    }
    __syncthreads();
    const bool bad = *(volatile int *)&gave_up != 0;
    if (bad && threadIdx.x == 0) {
        // copies may still be under way: they end before the block's shared memory is let go
        for (int i = max(0, copies - a.stages); i < copies; ++i) mbar_wait(&full[i % a.stages], (i / a.stages) & 1);
        if (a.status) atomicOr(a.status, (int)ERR_MBAR);
    }
    const float nan = __uint_as_float(0x7fc00000u);
    if (S == 1) {
        if (warp < 4) {
            const long long p = p0 + threadIdx.x;
#pragma unroll 2
            for (int c = 0; c < BN; c += 16) {
                float f[16];
                tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, f);
                tmem_wait_ld();
                if (bad)
#pragma unroll
                    for (int i = 0; i < 16; ++i) f[i] = nan;
                if (q0 + c < a.q) product_store<O>(a, p, q0 + c, f);
            }
        }
    } else {
        // every block leaves its tile in its shared memory (the stages are free), then adds a share of the columns
        float *part = reinterpret_cast<float *>(smem);
        if (warp < 4) {
            for (int c = 0; c < BN; c += 16) {
                float f[16];
                tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, f);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(c + i) * PT + threadIdx.x] = bad ? nan : steps ? f[i] : 0.0f;
            }
        }
        cluster_sync();
        if (warp < 4) {
            const long long p = p0 + threadIdx.x;
            O *out = static_cast<O *>(a.out);
            for (int c = rank; c < BN; c += S) {
                const long long q = q0 + c;
                if (q >= a.q || p >= a.p) continue;
                float t = 0.0f;
                for (int r = 0; r < S; ++r) t += remote_f32(smem_u32(part + c * PT + threadIdx.x), r);
                out[a.swap ? q * a.out_stride + p : p * a.out_stride + q] = from_f32<O>(t);
            }
        }
        cluster_sync();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) tmem_dealloc(tmem, cols);
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

int code_map(CUtensorMap *map, const unsigned char *codes, long long rows, int blocks, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) {
        set_error("flare_micro_product: the driver has no cuTensorMapEncodeTiled");
        return FLARE_E_CUDA;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)16 * blocks, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)16 * blocks};
    const cuuint32_t box[2] = {KBYTES, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<unsigned char *>(codes), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("flare_micro_product: tensor map of %lld rows of %d bytes: error %d", rows, 16 * blocks, (int)r);
        return FLARE_E_CUDA;
    }
    return FLARE_OK;
}

template <int BN, class O>
int launch_product(const CUtensorMap &pm, const CUtensorMap &qm, ProductArgs a, int split, cudaStream_t st) {
    using Tile = ProductTile<BN>;
    const int steps = (a.k + KSTAGE - 1) / KSTAGE, per = (steps + split - 1) / split;
    a.stages = std::min(Tile::MAX_STAGES, std::max(per, 1));
    int smem = a.stages * Tile::STAGE + 1024;
    if (split > 1) smem = std::max(smem, PT * BN * 4 + 1024);
    auto fn = product_kernel<BN, O>;
    const int e0 = allow_shared_memory(reinterpret_cast<const void *>(fn), "flare_micro_product");
    if (e0) return e0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((a.p + PT - 1) / PT), (unsigned)((a.q + BN - 1) / BN), (unsigned)split);
    cfg.blockDim = dim3(PR_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = (unsigned)split;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, pm, qm, a);
    if (e != cudaSuccess) {
        set_error("flare_micro_product: %s", cudaGetErrorString(e));
        return FLARE_E_CUDA;
    }
    return FLARE_OK;
}

int run_product(const flare_product_args *in, cudaStream_t st) {
    ProductArgs a{};
    a.swap = in->m < in->n;  // the larger matrix gives the tiles' 128 rows
    const unsigned char *pc = a.swap ? in->b_codes : in->a_codes, *qc = a.swap ? in->a_codes : in->b_codes;
    a.ps = a.swap ? in->b_scales : in->a_scales;
    a.qs = a.swap ? in->a_scales : in->b_scales;
    a.p = a.swap ? in->n : in->m;
    a.q = a.swap ? in->m : in->n;
    a.out = in->out;
    a.status = in->status;
    a.out_stride = in->out_stride;
    a.k = in->k;
    a.blocks = (in->k + 31) / 32;
    a.pitch = 4 * ((a.blocks + 3) / 4);
    a.vec = fits_vec(in->out, in->out_stride, type_size(in->out_type), 16 / type_size(in->out_type));
    // columns per tile: what Q has, at most 256; narrower where that leaves multiprocessors without a tile
    int bn = 16;
    while (bn < 256 && bn < a.q) bn *= 2;
    const long long ptiles = (a.p + PT - 1) / PT;
    auto tiles = [&](int b) { return ptiles * ((a.q + b - 1) / b); };
    while (bn > 64 && tiles(bn) < SMS) bn /= 2;
    // and then parts of K, at least two stages each
    const int steps = (in->k + KSTAGE - 1) / KSTAGE;
    int split = 1;
    while (split < 8 && tiles(bn) * split * 2 <= SMS && steps >= split * 4) split *= 2;
    CUtensorMap pm, qm;
    int e = code_map(&pm, pc, a.p, a.blocks, PT);
    if (!e) e = code_map(&qm, qc, a.q, a.blocks, bn);
    if (e) return e;
    return with_type(in->out_type, [&](auto t) {
        using O = typename decltype(t)::type;
        switch (bn) {
            case 16: return launch_product<16, O>(pm, qm, a, split, st);
            case 32: return launch_product<32, O>(pm, qm, a, split, st);
            case 64: return launch_product<64, O>(pm, qm, a, split, st);
            case 128: return launch_product<128, O>(pm, qm, a, split, st);
            default: return launch_product<256, O>(pm, qm, a, split, st);
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
    OPS_CHECK(a->a_codes && a->a_scales && a->b_codes && a->b_scales && a->out, "flare_micro_product: NULL buffer");
    OPS_CHECK(a->out_stride >= a->n, "flare_micro_product: output rows of stride %lld overlap", a->out_stride);
    for (const void *p : {(const void *)a->a_codes, (const void *)a->b_codes})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0, "flare_micro_product: codes must be 16-byte aligned");
    for (const void *p : {(const void *)a->a_scales, (const void *)a->b_scales})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 4 == 0, "flare_micro_product: scales must be 4-byte aligned");
    return run_product(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
