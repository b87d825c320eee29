// product.cu -- out = A B^T of two matrices held in microscaled 4-bit floats.
#include <algorithm>

#include "ops.cuh"

namespace flare {

struct ProductArgs {
    const unsigned char *ac, *as, *bc, *bs;
    void *out;
    long long m, n, out_stride;
    int blocks, pitch;
};

// 64 x 64 outputs per block, 4 x 4 per thread, one 32-element block of K at a time, values in shared memory.
template <class O>
__global__ void __launch_bounds__(256) product_kernel(const ProductArgs a) {
    __shared__ float sa[32][65], sb[32][65];
    const long long m0 = (long long)blockIdx.x * 64;
    const long long n0 = (long long)blockIdx.y * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int row = threadIdx.x >> 2, piece = threadIdx.x & 3;
    float acc[4][4] = {};
    for (int b = 0; b < a.blocks; ++b) {
        for (int side = 0; side < 2; ++side) {
            const long long r = (side ? n0 : m0) + row;
            const bool in = r < (side ? a.n : a.m);
            unsigned bits = 0;
            float s = 0.0f;
            if (in) {
                bits = __ldg(reinterpret_cast<const unsigned *>((side ? a.bc : a.ac) + (r * a.blocks + b) * 16) + piece);
                s = micro_scale((side ? a.bs : a.as)[r * a.pitch + b]);
            }
            float(*dst)[65] = side ? sb : sa;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float2 t = micro_pair((bits >> (8 * p)) & 255u);
                dst[piece * 8 + 2 * p][row] = t.x * s;
                dst[piece * 8 + 2 * p + 1][row] = t.y * s;
            }
        }
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
            if (r < a.m && c < a.n) static_cast<O *>(a.out)[r * a.out_stride + c] = from_f32<O>(acc[i][j]);
        }
}

}  // namespace flare

using namespace flare;

extern "C" {

long long flare_micro_product_workspace(long long m, long long n, int k) { return 0; }

int flare_micro_product(const flare_product_args *a, void *stream) {
    OPS_CHECK(a, "flare_micro_product: NULL argument");
    OPS_CHECK(is_float_type(a->out_type), "flare_micro_product: unknown type %d", a->out_type);
    OPS_CHECK(a->m >= 0 && a->n >= 0 && a->k >= 1 && a->k <= (1 << 30), "flare_micro_product: %lld x %lld x %d", a->m, a->n, a->k);
    OPS_CHECK(a->m < 0x40000000ll && a->n < 64 * 65535ll, "flare_micro_product: %lld x %lld outputs", a->m, a->n);
    if (a->m == 0 || a->n == 0) return FLARE_OK;
    OPS_CHECK(a->a_codes && a->a_scales && a->b_codes && a->b_scales && a->out, "flare_micro_product: NULL buffer");
    OPS_CHECK(a->out_stride >= a->n, "flare_micro_product: output rows of stride %lld overlap", a->out_stride);
    for (const void *p : {(const void *)a->a_codes, (const void *)a->b_codes})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0, "flare_micro_product: codes must be 16-byte aligned");
    for (const void *p : {(const void *)a->a_scales, (const void *)a->b_scales})
        OPS_CHECK(reinterpret_cast<uintptr_t>(p) % 4 == 0, "flare_micro_product: scales must be 4-byte aligned");
    const int blocks = (a->k + 31) / 32;
    ProductArgs p{a->a_codes, a->a_scales, a->b_codes, a->b_scales, a->out, a->m, a->n, a->out_stride, blocks,
                  4 * ((blocks + 3) / 4)};
    const dim3 grid((unsigned)((a->m + 63) / 64), (unsigned)((a->n + 63) / 64));
    with_type(a->out_type, [&](auto t) {
        product_kernel<typename decltype(t)::type><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
        return 0;
    });
    OPS_LAUNCHED("flare_micro_product");
    return FLARE_OK;
}

}  // extern "C"
