// Pieces the row-wise kernels (norm, row quantiser, distillation loss) share: 16-byte vector loads of any float type
// into fp32 registers and back, NaN-propagating maxima, block reductions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace ntb200 {

template <class T> struct RowType;
template <> struct RowType<float> {
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct RowType<__half> {
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <> struct RowType<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// V consecutive elements: V * sizeof(T) is 16, 8, 4 or 2 bytes, and addresses are aligned to that.
template <class T, int V>
struct __align__(sizeof(T) * V) Pack {
    T e[V];
    // one instruction per value: a BFloat16 is the upper half of a Float32, so the pair's word is shifted or masked
    // (extracting the 16 bits first costs a second one)
    __device__ __forceinline__ float up(int i) const {
        if constexpr (std::is_same<T, __nv_bfloat16>::value && V % 2 == 0) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(e)[i >> 1];
            return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
        } else if constexpr (std::is_same<T, __half>::value && V % 2 == 0) {
            const __half2 h = reinterpret_cast<const __half2*>(e)[i >> 1];
            return i & 1 ? __high2float(h) : __low2float(h);
        } else {
            return RowType<T>::up(e[i]);
        }
    }
    __device__ __forceinline__ void set(int i, float v) { e[i] = RowType<T>::down(v); }
    // all of them, rounded; 16-bit values two at a time (one conversion instruction a pair)
    __device__ __forceinline__ void put(const float* v) {
        if constexpr (sizeof(T) == 2 && V % 2 == 0) {
            uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                if constexpr (std::is_same<T, __half>::value) {
                    const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
                    w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
                    w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = RowType<T>::down(v[i]);
        }
    }
};

// The hardware's exponential and reciprocal alone (relative error about 2^-22): results below 2^-126 are zero.
__device__ __forceinline__ float exp2_hw(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_hw(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is NaN
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

}  // namespace ntb200
