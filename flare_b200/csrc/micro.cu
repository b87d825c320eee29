// micro.cu -- microscaled 4-bit floats: to codes and scales and back (the format is described in the header).
//
// Both directions are bound by memory: 2.53 (16-bit values) to 4.53 bytes (f32) an element.  Where rows allow it a lane
// has 16 consecutive elements, half a block, and reads or writes 32 bytes at a time; the block's largest magnitude takes one
// exchange.  With 8 elements a lane the instructions per element bound it (3M x 96 f16: 207 us to codes and 150 us back).
// Other rows go by 8 elements a lane, four lanes to a block.
#include <algorithm>

#include "ops.cuh"

namespace flare {

constexpr int MQ_THREADS = 256;

struct MicroArgs {
    const void *x;
    void *out;
    unsigned char *codes, *scales;
    const unsigned char *codes_in, *scales_in;
    long long stride, first;  // first: first row of this launch
    unsigned items;           // 8- or 16-element pieces of this launch
    int width, blocks, pitch;
    FastDiv ppr;              // pieces per row: 4 or 2 per block
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
    float inv;
    const unsigned byte = micro_byte(most, &inv);
    unsigned bits = 0;
    if (byte != 255)
#pragma unroll
        for (int p = 0; p < 4; ++p) bits |= micro_code_pair(f[2 * p] * inv, f[2 * p + 1] * inv) << (8 * p);
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

// 32 bytes, aligned to as many
__device__ __forceinline__ void load32(const void *p, unsigned *w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void store32(void *p, const unsigned (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// 16 elements of T
template <class T>
struct Sixteen {
    static constexpr int N = (int)sizeof(T) / 2;  // 32-byte pieces
    unsigned w[8 * N];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N; ++i) load32(reinterpret_cast<const char *>(p) + 32 * i, w + 8 * i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < 8 * N; ++k) w[k] = 0;
    }
};

// A lane per 16 elements of a row, two lanes per block
template <class T>
__global__ void __launch_bounds__(MQ_THREADS) micro_quantize16_kernel(const MicroArgs a) {
    const unsigned it = blockIdx.x * MQ_THREADS + threadIdx.x;
    const unsigned r = a.ppr.div(it), piece = it - r * a.ppr.d;
    const long long row = a.first + r;
    const bool in = it < a.items;
    Sixteen<T> x;
    if (in && (int)piece * 16 < a.width) x.load(static_cast<const T *>(a.x) + row * a.stride + piece * 16);
    else x.zero();
    unsigned most = words_most<T, 8 * Sixteen<T>::N>(x.w);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    float inv;
    const unsigned byte = micro_byte(most, &inv);
    unsigned lo = 0, hi = 0;
    if (byte != 255) {
        lo = micro_codes8<T>(x.w, 0, inv);
        hi = micro_codes8<T>(x.w, 4, inv);
    }
    if (!in) return;
    __stcs(reinterpret_cast<uint2 *>(a.codes + row * (16ll * a.blocks)) + piece, make_uint2(lo, hi));
    if ((piece & 1) == 0) {
        unsigned char *s = a.scales + row * a.pitch;
        const int b = (int)piece >> 1;
        s[b] = (unsigned char)byte;
        if (b == a.blocks - 1)
            for (int k = a.blocks; k < a.pitch; ++k) s[k] = 0;
    }
}

template <class T>
__global__ void __launch_bounds__(MQ_THREADS) micro_dequantize16_kernel(const MicroArgs a) {
    const unsigned it = blockIdx.x * MQ_THREADS + threadIdx.x;
    if (it >= a.items) return;
    const unsigned r = a.ppr.div(it), piece = it - r * a.ppr.d;
    const long long row = a.first + r;
    if ((int)piece * 16 >= a.width) return;
    const uint2 c = __ldcs(reinterpret_cast<const uint2 *>(a.codes_in + row * (16ll * a.blocks)) + piece);
    const unsigned byte = __ldg(a.scales_in + row * a.pitch + (piece >> 1));
    const float s = micro_scale(byte);
    unsigned w[(int)sizeof(T) / 2][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float2 t = micro_pair(((k < 4 ? c.x : c.y) >> (8 * (k & 3))) & 255u);
        const float x = t.x * s, y = t.y * s;
        if constexpr (sizeof(T) == 4) {
            w[k / 4][2 * k % 8] = __float_as_uint(x);
            w[k / 4][2 * k % 8 + 1] = __float_as_uint(y);
        } else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(x, y);
            w[0][k] = *reinterpret_cast<const unsigned *>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            w[0][k] = *reinterpret_cast<const unsigned *>(&h);
        }
    }
    T *o = static_cast<T *>(a.out) + row * a.stride + piece * 16;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) store32(reinterpret_cast<char *>(o) + 32 * i, w[i]);
}

// whether rows allow 32-byte accesses of 16 elements
inline bool fits_sixteen(const void *p, long long stride, int width, int size) {
    return width % 16 == 0 && stride * size % 32 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0;
}

// runs f(args) over launches whose piece numbers stay below 2^31
template <class F>
int micro_launches(MicroArgs &a, long long rows, int width, int per_block, F f) {
    a.width = width;
    a.blocks = (width + 31) / 32;
    a.pitch = 4 * ((a.blocks + 3) / 4);
    const unsigned ppr = (unsigned)per_block * (unsigned)a.blocks;  // pieces per block and row
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
    const bool vec = width % 8 == 0 && fits_vec(x, stride, type_size(type), 8), wide = fits_sixteen(x, stride, width, type_size(type));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return micro_launches(a, rows, width, wide ? 2 : 4, [&](unsigned blocks) {
            if (wide) micro_quantize16_kernel<T><<<blocks, MQ_THREADS, 0, st>>>(a);
            else if (vec) micro_quantize_kernel<T, true><<<blocks, MQ_THREADS, 0, st>>>(a);
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
    const bool vec = width % 8 == 0 && fits_vec(out, stride, type_size(type), 8), wide = fits_sixteen(out, stride, width, type_size(type));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return micro_launches(a, rows, width, wide ? 2 : 4, [&](unsigned blocks) {
            if (wide) micro_dequantize16_kernel<T><<<blocks, MQ_THREADS, 0, st>>>(a);
            else if (vec) micro_dequantize_kernel<T, true><<<blocks, MQ_THREADS, 0, st>>>(a);
            else micro_dequantize_kernel<T, false><<<blocks, MQ_THREADS, 0, st>>>(a);
        });
    });
    OPS_LAUNCHED("flare_micro_dequantize");
    return FLARE_OK;
}

}  // extern "C"
