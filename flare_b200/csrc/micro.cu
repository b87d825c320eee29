// micro.cu -- microscaled 4-bit floats: to codes and scales and back (the format is described in the header).
//
// Both directions are bound by memory: 2.03 (16-bit input) to 4.53 bytes (f32) an element.  Four lanes share a block of
// 32, 8 elements each, so that a warp's 16-byte loads are contiguous; the block's largest magnitude is exchanged by two
// shuffles.
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "ops.cuh"

namespace flare {

int allow_shared_memory(const void *kernel, const char *what) {
    static std::mutex lock;
    static std::set<std::pair<const void *, int>> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) {
        std::lock_guard<std::mutex> hold(lock);
        if (allowed.count({kernel, device})) return FLARE_OK;
        cudaFuncAttributes at{};
        e = cudaFuncGetAttributes(&at, kernel);
        // 227 KB a block, less what the kernel has already
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)at.sharedSizeBytes);
        if (e == cudaSuccess) allowed.insert({kernel, device});
    }
    if (e == cudaSuccess) return FLARE_OK;
    set_error("%s: %s", what, cudaGetErrorString(e));
    return FLARE_E_CUDA;
}

constexpr int MQ_THREADS = 256;

struct MicroArgs {
    const void *x;
    void *out;
    unsigned char *codes, *scales;
    const unsigned char *codes_in, *scales_in;
    long long stride, first;  // first: first row of this launch
    unsigned items;           // 8-element pieces of this launch
    int width, blocks, pitch;
    FastDiv ppr;              // pieces per row: 4 * blocks
};

template <class T, bool VEC>
__global__ void __launch_bounds__(MQ_THREADS) micro_quantize_kernel(const MicroArgs a) {
    const unsigned it = blockIdx.x * MQ_THREADS + threadIdx.x;
    const unsigned r = a.ppr.div(it), piece = it - r * a.ppr.d;
    const long long row = a.first + r;
    const int col = (int)piece * 8;
    const bool in = it < a.items;
    float f[8];
    if (VEC) {
        Vec<T, 8> v;
        if (in && col < a.width) v.load_stream(static_cast<const T *>(a.x) + row * a.stride + col);
        else v.zero();
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v.get(e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            f[e] = in && col + e < a.width ? to_f32(static_cast<const T *>(a.x)[row * a.stride + col + e]) : 0.0f;
    }
    // magnitudes compare as their bits do; infinities and NaN are the largest
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(f[e]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    unsigned byte, bits = 0;
    if (most >= 0x7f800000u) {
        byte = 255;
    } else {
        // floor(log2) of the largest is its exponent field - 127; below 2^-125 (subnormal ones too) the clamp decides
        const int e = most == 0 ? -127 : max((int)(most >> 23) - 127 - 2, -127);
        byte = (unsigned)(e + 127);
        const float inv = __uint_as_float((unsigned)(127 - e) << 23);  // 2^-e, e in [-127, 125]
#pragma unroll
        for (int p = 0; p < 4; ++p) bits |= micro_code_pair(f[2 * p] * inv, f[2 * p + 1] * inv) << (8 * p);
    }
    if (!in) return;
    *reinterpret_cast<unsigned *>(a.codes + row * (16ll * a.blocks) + 4 * piece) = bits;
    if ((piece & 3) == 0) {
        unsigned char *s = a.scales + row * a.pitch;
        const int b = (int)piece >> 2;
        s[b] = (unsigned char)byte;
        if (b == a.blocks - 1)
            for (int k = a.blocks; k < a.pitch; ++k) s[k] = 0;
    }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(MQ_THREADS) micro_dequantize_kernel(const MicroArgs a) {
    const unsigned it = blockIdx.x * MQ_THREADS + threadIdx.x;
    if (it >= a.items) return;
    const unsigned r = a.ppr.div(it), piece = it - r * a.ppr.d;
    const long long row = a.first + r;
    const int col = (int)piece * 8;
    if (col >= a.width) return;
    const unsigned bits = __ldcs(reinterpret_cast<const unsigned *>(a.codes_in + row * (16ll * a.blocks)) + piece);
    const float s = micro_scale(__ldg(a.scales_in + row * a.pitch + (piece >> 2)));
    Vec<T, 8> v;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float2 t = micro_pair((bits >> (8 * p)) & 255u);
        v.set(2 * p, t.x * s);
        v.set(2 * p + 1, t.y * s);
    }
    T *o = static_cast<T *>(a.out) + row * a.stride + col;
    if (VEC) {
        v.store_stream(o);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < a.width) o[e] = v.el[e];
    }
}

// runs f(args) over launches whose piece numbers stay below 2^31
template <class F>
int micro_launches(MicroArgs &a, long long rows, int width, F f) {
    a.width = width;
    a.blocks = (width + 31) / 32;
    a.pitch = 4 * ((a.blocks + 3) / 4);
    const unsigned ppr = 4u * (unsigned)a.blocks;
    a.ppr = FastDiv(ppr);
    const long long per_launch = std::max<long long>(1, (1ll << 30) / ppr);
    for (a.first = 0; a.first < rows; a.first += per_launch) {
        a.items = (unsigned)(std::min(per_launch, rows - a.first) * ppr);
        f((a.items + MQ_THREADS - 1) / MQ_THREADS);
    }
    return FLARE_OK;
}

}  // namespace flare

using namespace flare;

extern "C" {

int flare_micro_quantize(const void *x, int type, long long rows, int width, long long stride, unsigned char *codes,
                         unsigned char *scales, void *stream) {
    OPS_CHECK(is_float_type(type), "flare_micro_quantize: unknown type %d", type);
    OPS_CHECK(rows >= 0 && width >= 1 && width <= (1 << 30), "flare_micro_quantize: %lld rows of %d", rows, width);
    if (rows == 0) return FLARE_OK;
    OPS_CHECK(x && codes && scales, "flare_micro_quantize: NULL buffer");
    OPS_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
              "flare_micro_quantize: codes must be 16-byte and scales 4-byte aligned");
    MicroArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.stride = stride;
    const bool vec = width % 8 == 0 && fits_vec(x, stride, type_size(type), 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return micro_launches(a, rows, width, [&](unsigned blocks) {
            if (vec) micro_quantize_kernel<T, true><<<blocks, MQ_THREADS, 0, st>>>(a);
            else micro_quantize_kernel<T, false><<<blocks, MQ_THREADS, 0, st>>>(a);
        });
    });
    OPS_LAUNCHED("flare_micro_quantize");
    return FLARE_OK;
}

int flare_micro_dequantize(const unsigned char *codes, const unsigned char *scales, long long rows, int width, void *out,
                           int type, long long stride, void *stream) {
    OPS_CHECK(is_float_type(type), "flare_micro_dequantize: unknown type %d", type);
    OPS_CHECK(rows >= 0 && width >= 1 && width <= (1 << 30), "flare_micro_dequantize: %lld rows of %d", rows, width);
    if (rows == 0) return FLARE_OK;
    OPS_CHECK(out && codes && scales, "flare_micro_dequantize: NULL buffer");
    OPS_CHECK(stride >= width, "flare_micro_dequantize: output rows of stride %lld overlap", stride);
    OPS_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
              "flare_micro_dequantize: codes must be 16-byte and scales 4-byte aligned");
    MicroArgs a{};
    a.out = out;
    a.codes_in = codes;
    a.scales_in = scales;
    a.stride = stride;
    const bool vec = width % 8 == 0 && fits_vec(out, stride, type_size(type), 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return micro_launches(a, rows, width, [&](unsigned blocks) {
            if (vec) micro_dequantize_kernel<T, true><<<blocks, MQ_THREADS, 0, st>>>(a);
            else micro_dequantize_kernel<T, false><<<blocks, MQ_THREADS, 0, st>>>(a);
        });
    });
    OPS_LAUNCHED("flare_micro_dequantize");
    return FLARE_OK;
}

}  // extern "C"
