// ops.cuh -- shared by the operators outside the render path (lookup.cu, recurrence.cu, micro.cu): element
// types, vector loads and stores through 32-bit floats, argument checks.
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
