// feq_token.cuh -- shared pieces of the row operators on token features in float32, bfloat16 and
// float16 (layer norm, expert routing, expert linear): element types, vector loads and stores of
// any power-of-two width, and the sums within a group of lanes.  Arithmetic is in float32
// everywhere; a value is rounded to its 16-bit type once, when it is stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "feq_internal.cuh"

namespace feq {
namespace token {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements, moved as one access of sizeof(T) * V bytes (2 .. 16).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// A 1-D parameter stored in the features' type or in float32.
template <typename T>
__device__ __forceinline__ float param_at(const void *p, int is_f32, int64_t i) {
    return is_f32 ? static_cast<const float *>(p)[i] : to_f32(static_cast<const T *>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void param_put(void *p, int is_f32, int64_t i, float v) {
    if (is_f32)
        static_cast<float *>(p)[i] = v;
    else
        static_cast<T *>(p)[i] = from_f32<T>(v);
}

// Sum over groups of `width` lanes (a power of two up to 32), the same value in every lane.
__device__ __forceinline__ float lane_sum(float v, int width) {
    for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

inline size_t dtype_bytes(int dtype) { return dtype == FEQ_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == FEQ_DTYPE_F32 || dtype == FEQ_DTYPE_BF16 || dtype == FEQ_DTYPE_F16; }

// Widest power-of-two vector, in elements and at most 16 bytes, that divides every address and
// row length (in bytes) or-ed into `bits`.
inline int vector_elems(uint64_t bits, size_t elem_bytes) {
    size_t b = 16;
    while (b > elem_bytes && (bits & (b - 1))) b >>= 1;
    return (int)(b / elem_bytes);
}

inline int pow2_ceil(int64_t n) {
    int p = 1;
    while (p < n && p < (1 << 30)) p <<= 1;
    return p;
}

inline int sm_count() {
    static std::atomic<int> known[64];       // by device; 0: not asked yet
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) return sms;
    if (dev >= 0 && dev < 64 && known[dev].load(std::memory_order_relaxed)) return known[dev].load(std::memory_order_relaxed);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && dev >= 0 && dev < 64)
        known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

// Calls f with a value of the element type and an integral constant for the vector width.
#define FEQ_TOKEN_VEC(T, vec, ...)                                                     \
    switch (vec) {                                                                     \
        case 8: if constexpr (sizeof(T) == 2) { constexpr int V = 8; __VA_ARGS__ } break;   \
        case 4: { constexpr int V = 4; __VA_ARGS__ } break;                            \
        case 2: { constexpr int V = 2; __VA_ARGS__ } break;                            \
        default: { constexpr int V = 1; __VA_ARGS__ } break;                           \
    }
#define FEQ_TOKEN_TYPE(dtype, ...)                                                     \
    switch (dtype) {                                                                   \
        case FEQ_DTYPE_F32: { using T = float; __VA_ARGS__ } break;                    \
        case FEQ_DTYPE_BF16: { using T = __nv_bfloat16; __VA_ARGS__ } break;           \
        default: { using T = __half; __VA_ARGS__ } break;                              \
    }

}  // namespace token
}  // namespace feq
