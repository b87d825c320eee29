// ops.cuh -- shared by the operators outside the render path (lookup.cu, recurrence.cu, micro.cu, product.cu): element
// types, vector loads and stores through 32-bit floats, the 4-bit format, argument checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/flare_b200.h"

namespace flare {

void set_error(const char *fmt, ...);

#define OPS_CHECK(cond, ...)          \
    do {                              \
        if (!(cond)) {                \
            flare::set_error(__VA_ARGS__); \
            return FLARE_E_INVALID;   \
        }                             \
    } while (0)

#define OPS_LAUNCHED(what)                                              \
    do {                                                                \
        cudaError_t ce_ = cudaGetLastError();                           \
        if (ce_ != cudaSuccess) {                                       \
            flare::set_error("%s: %s", what, cudaGetErrorString(ce_));  \
            return FLARE_E_CUDA;                                        \
        }                                                               \
    } while (0)

constexpr int SMS = 148;  // streaming multiprocessors of a B200

__host__ __device__ constexpr int type_size(int type) { return type == FLARE_F32 ? 4 : 2; }
inline bool is_float_type(int type) { return type == FLARE_F32 || type == FLARE_F16 || type == FLARE_BF16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// BYTES of raw storage moved by accesses of at most 16 bytes; the address is aligned to min(BYTES, 16).
template <int BYTES>
struct Raw;
template <>
struct Raw<2> { using type = unsigned short; static constexpr int N = 1; };
template <>
struct Raw<4> { using type = unsigned; static constexpr int N = 1; };
template <>
struct Raw<8> { using type = uint2; static constexpr int N = 1; };
template <>
struct Raw<16> { using type = uint4; static constexpr int N = 1; };
template <>
struct Raw<32> { using type = uint4; static constexpr int N = 2; };

// N elements of T as they lie in memory.
template <class T, int N>
struct Vec {
    using R = Raw<N * (int)sizeof(T)>;
    union {
        typename R::type raw[R::N];
        T el[N];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) raw[i] = __ldg(reinterpret_cast<const typename R::type *>(p) + i);
    }
    // for memory that this kernel writes too, after reading it
    __device__ __forceinline__ void load_plain(const T *p) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) raw[i] = *(reinterpret_cast<const typename R::type *>(p) + i);
    }
    // read once: no line is kept for it
    __device__ __forceinline__ void load_stream(const T *p) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) raw[i] = __ldcs(reinterpret_cast<const typename R::type *>(p) + i);
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < R::N; ++i) reinterpret_cast<typename R::type *>(p)[i] = raw[i];
    }
    __device__ __forceinline__ void store_stream(T *p) const {
#pragma unroll
        for (int i = 0; i < R::N; ++i) __stcs(reinterpret_cast<typename R::type *>(p) + i, raw[i]);
    }
    __device__ __forceinline__ float get(int i) const { return to_f32(el[i]); }
    __device__ __forceinline__ void set(int i, float v) { el[i] = from_f32<T>(v); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N; ++i) el[i] = from_f32<T>(0.0f);
    }
};

// Whether vectors of `n` elements of `size` bytes may be used at p with rows `stride` elements apart.
inline bool fits_vec(const void *p, long long stride, int size, int n) {
    const int bytes = n * size < 16 ? n * size : 16;
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride % n == 0;
}

// Whether two stretches of memory share a byte.
inline bool overlaps(const void *p, long long p_bytes, const void *q, long long q_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return p && q && p_bytes > 0 && q_bytes > 0 && a < b + (uintptr_t)q_bytes && b < a + (uintptr_t)p_bytes;
}

// The same for a stretch and `rows` rows of row_bytes, `stride` bytes apart.
inline bool overlaps_rows(const void *p, long long p_bytes, const void *q, long long rows, long long row_bytes, long long stride) {
    if (rows <= 0 || stride == 0) return overlaps(p, p_bytes, q, rows > 0 ? row_bytes : 0);
    if (stride < 0) return overlaps_rows(p, p_bytes, static_cast<const char *>(q) + (rows - 1) * stride, rows, row_bytes, -stride);
    // the first row that ends behind the stretch's start
    const long long before = (long long)(reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) - row_bytes;
    const long long row = before < 0 ? 0 : before / stride + 1;
    return row < rows && overlaps(p, p_bytes, static_cast<const char *>(q) + row * stride, row_bytes);
}

// 2^(byte - 127); byte 255 stands for NaN
__device__ __forceinline__ float micro_scale(unsigned byte) {
    if (byte == 0) return __uint_as_float(0x00400000u);
    return __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23);
}

// Two codes in the low byte of `pair` -> their values (exact in f16), low code first.
__device__ __forceinline__ float2 micro_pair(unsigned pair) {
    unsigned h;
    asm("{\n\t.reg .b8 c;\n\tcvt.u8.u32 c, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(h) : "r"(pair));
    return __half22float2(*reinterpret_cast<__half2 *>(&h));
}
// Nearest code of lo (low four bits) and of hi (high four bits): ties to even, magnitudes above 6 to 6.
__device__ __forceinline__ unsigned micro_code_pair(float lo, float hi) {
    unsigned c;
    asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\tcvt.u32.u8 %0, c;\n\t}" : "=r"(c) : "f"(hi), "f"(lo));
    return c;
}

__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b) {
    unsigned d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Elements 2k and 2k + 1 of T as they lie in 32-bit words.
template <class T>
__device__ __forceinline__ float2 words_pair(const unsigned *w, int k) {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
    else return make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
}
// The largest magnitude in N words, as a float's bits.  Magnitudes compare as their bits do; infinities and NaN are the largest.
template <class T, int N>
__device__ __forceinline__ unsigned words_most(const unsigned *w) {
    unsigned m[4] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) m[k & 3] = sizeof(T) == 4 ? max(m[k & 3], w[k] & 0x7fffffffu) : max_u16x2(m[k & 3], w[k] & 0x7fff7fffu);
    if constexpr (sizeof(T) == 4) return max(max(m[0], m[1]), max(m[2], m[3]));
    const unsigned p = max_u16x2(max_u16x2(m[0], m[1]), max_u16x2(m[2], m[3])), h = max(p & 0xffffu, p >> 16);
    if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    else return h << 16;
}
// The scale byte of a block whose largest magnitude is `most`, and 2^-e for its elements (0 where the block stands for NaN).
__device__ __forceinline__ unsigned micro_byte(unsigned most, float *inv) {
    *inv = 0.0f;
    if (most >= 0x7f800000u) return 255;
    // floor(log2) of the largest is its exponent field - 127; below 2^-125 (subnormal ones too) the clamp decides
    const int e = max((int)(most >> 23) - 127 - 2, -127);
    *inv = __uint_as_float((unsigned)(127 - e) << 23);  // e in [-127, 125]
    return (unsigned)(e + 127);
}
// Codes of eight elements, from the 4 pairs k, k + 1, ...
template <class T>
__device__ __forceinline__ unsigned micro_codes8(const unsigned *w, int k, float inv) {
    unsigned c = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float2 v = words_pair<T>(w, k + p);
        c |= micro_code_pair(v.x * inv, v.y * inv) << (8 * p);
    }
    return c;
}

// Exact quotient of 31-bit values by a fixed divisor d >= 1 (multiply and shift, Granlund and Montgomery 1994).
struct FastDiv {
    unsigned d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(unsigned divisor) : d(divisor) {
        shift = 0;
        while ((1ull << shift) < divisor) ++shift;
        mul = (unsigned)(((1ull << 32) * ((1ull << shift) - divisor)) / divisor + 1);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// Lets kernel K have all of a multiprocessor's shared memory, once per device.
template <auto K>
int allow_shared_memory(const char *what) {
    static std::atomic<unsigned long long> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (e == cudaSuccess && (done.load() & bit)) return FLARE_OK;
    cudaFuncAttributes at{};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, K);
    // 227 KB a block, less what the kernel has already
    if (e == cudaSuccess) e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)at.sharedSizeBytes);
    if (e != cudaSuccess) {
        set_error("%s: %s", what, cudaGetErrorString(e));
        return FLARE_E_CUDA;
    }
    done.fetch_or(bit);
    return FLARE_OK;
}

template <class T>
struct TypeTag { using type = T; };
// f(tag) for the C++ type of a FLARE_* float type
template <class F>
int with_type(int type, F f) {
    switch (type) {
        case FLARE_F32: return f(TypeTag<float>{});
        case FLARE_F16: return f(TypeTag<__half>{});
        default: return f(TypeTag<__nv_bfloat16>{});
    }
}

}  // namespace flare
