// What follows the product in ntb200_linear_act, on fp32 registers: scales, bias, activation, residual, one rounding.
// Shared by the epilogues of the GEMM kernels and the elementwise kernels of linear.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

namespace ntb200 {

// kFast: results that are rounded to 16 bits use the hardware exponential and reciprocal (relative error about 2^-21,
// a hundredth of half a Float16 step); Float32 results use the full-precision functions.
template <bool kFast>
__device__ __forceinline__ float sigmoid_times(float z, float u) {   // z / (1 + e^-u)
    if constexpr (kFast) return __fdividef(z, 1.f + __expf(-u));
    return z / (1.f + expf(-u));
}

constexpr float kGeluScale = 1.5957691216057308f;   // 2 sqrt(2 / pi): z/2 (1 + tanh u) = z sigmoid(2 u)
constexpr float kGeluCubic = 0.044715f;

// Phi(z) = erfc(-z / sqrt 2) / 2 for results of 16 bits, e = e^(-z^2 / 2).  Phi(-a) = e t P(t) with t = 1 / (1 + 0.36 a): P is
// a degree-6 fit of erfcx(a / sqrt 2) / (2 t), relative error below 1.1e-6 over 0 <= a <= 14 (least squares reweighted
// towards the minimax, evaluated in fp32), so the tail keeps its relative precision.  15 instructions; erfcf takes 40.
__device__ __forceinline__ float phi_fast(float z, float e) {
    const float t = __fdividef(1.f, 1.f + 0.36f * fabsf(z));
    const float q = e * t * (0.14371304f + t * (0.14177254f + t * (0.13971882f + t * (0.026550606f + t * (0.1809521f + t * (-0.17976327f + t * 0.047055867f))))));
    return z < 0.f ? q : 1.f - q;
}

// Full precision, out of line: Float32 results are few and these functions long.
static __device__ __noinline__ float act_value_full(int act, float z) {
    switch (act) {
        case NTB200_ACT_RELU: return z < 0.f ? 0.f : z;
        case NTB200_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678118654752f);
        case NTB200_ACT_GELU_TANH: return sigmoid_times<false>(z, kGeluScale * (z + kGeluCubic * z * z * z));
        case NTB200_ACT_SILU: return sigmoid_times<false>(z, z);
        default: return z;
    }
}

template <bool kFast>
__device__ __forceinline__ float act_value(int act, float z) {
    if constexpr (!kFast) return act_value_full(act, z);
    switch (act) {
        case NTB200_ACT_RELU: return z < 0.f ? 0.f : z;
        case NTB200_ACT_GELU: return z * phi_fast(z, __expf(-0.5f * z * z));
        case NTB200_ACT_GELU_TANH: return sigmoid_times<true>(z, kGeluScale * (z + kGeluCubic * z * z * z));
        case NTB200_ACT_SILU: return sigmoid_times<true>(z, z);
        default: return z;
    }
}

template <bool kFast>
__device__ __forceinline__ float act_slope(int act, float z) {
    switch (act) {
        case NTB200_ACT_RELU: return z < 0.f ? 0.f : 1.f;
        case NTB200_ACT_GELU: {
            const float e = kFast ? __expf(-0.5f * z * z) : expf(-0.5f * z * z);
            if constexpr (kFast) return phi_fast(z, e) + z * e * 0.39894228040143268f;
            return 0.5f * erfcf(z * -0.70710678118654752f) + z * e * 0.39894228040143268f;
        }
        case NTB200_ACT_GELU_TANH: {
            if (fabsf(z) > 20.f) return z > 0.f ? 1.f : 0.f;   // the tails, before z^3 can overflow
            const float g = sigmoid_times<kFast>(1.f, kGeluScale * (z + kGeluCubic * z * z * z));
            return g + z * g * (1.f - g) * kGeluScale * (1.f + 3.f * kGeluCubic * z * z);
        }
        case NTB200_ACT_SILU: {
            const float g = sigmoid_times<kFast>(1.f, z);
            return g * (1.f + z * (1.f - g));
        }
        default: return 1.f;
    }
}

// The activation of N values, decided once.
template <bool kFast, int N>
__device__ __forceinline__ void act_values(int act, float (&f)[N]) {
    if constexpr (!kFast) {
        if (act == NTB200_ACT_NONE) return;
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = act_value_full(act, f[j]);
        return;
    }
#define NTB200_ACT_CASE(A)                                            \
    case A:                                                           \
        _Pragma("unroll") for (int j = 0; j < N; ++j) f[j] = act_value<kFast>(A, f[j]); \
        break;
    switch (act) {
        NTB200_ACT_CASE(NTB200_ACT_RELU)
        NTB200_ACT_CASE(NTB200_ACT_GELU)
        NTB200_ACT_CASE(NTB200_ACT_GELU_TANH)
        NTB200_ACT_CASE(NTB200_ACT_SILU)
        default: break;
    }
#undef NTB200_ACT_CASE
}

__device__ __forceinline__ float lin_up16(uint32_t bits, int dtype) {
    return dtype == NTB200_F16 ? __half2float(__ushort_as_half((unsigned short)bits))
                               : __bfloat162float(__ushort_as_bfloat16((unsigned short)bits));
}
__device__ __forceinline__ uint32_t lin_pack2(float lo, float hi, int dtype) {
    if (dtype == NTB200_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lin_load(const void* p, long long i, int dtype) {
    return dtype == NTB200_F32 ? static_cast<const float*>(p)[i] : lin_up16(static_cast<const uint16_t*>(p)[i], dtype);
}
__device__ __forceinline__ void lin_store(void* p, long long i, float v, int dtype) {
    if (dtype == NTB200_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = uint16_t(lin_pack2(v, 0.f, dtype));
}

// v[0..32) += 32 consecutive elements at p + i (16-byte aligned).
__device__ __forceinline__ void lin_add32(const void* p, long long i, int dtype, float (&v)[32]) {
    if (dtype == NTB200_F32) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float4 o = s[q];
            v[4 * q] += o.x; v[4 * q + 1] += o.y; v[4 * q + 2] += o.z; v[4 * q + 3] += o.w;
        }
        return;
    }
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint4 o = s[q];
        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[8 * q + 2 * j] += lin_up16(w[j] & 0xffffu, dtype);
            v[8 * q + 2 * j + 1] += lin_up16(w[j] >> 16, dtype);
        }
    }
}
__device__ __forceinline__ void lin_store32(void* p, long long i, int dtype, const float (&v)[32]) {
    if (dtype == NTB200_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
        for (int q = 0; q < 8; ++q) d[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        return;
    }
    uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        d[q] = make_uint4(lin_pack2(v[8 * q], v[8 * q + 1], dtype), lin_pack2(v[8 * q + 2], v[8 * q + 3], dtype),
                          lin_pack2(v[8 * q + 4], v[8 * q + 5], dtype), lin_pack2(v[8 * q + 6], v[8 * q + 7], dtype));
}

// Scales and bias of 32 consecutive products of one row; wide: every column is there and the vectors start on 16 bytes.
__device__ __forceinline__ void linear_scale_bias32(const LinearParams& l, int n, int col0, float rs, bool wide, float (&f)[32]) {
    if (l.col_scale) {
        if (wide) {
            const float4* cs = reinterpret_cast<const float4*>(l.col_scale + col0);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 o = cs[q];
                f[4 * q] *= rs * o.x; f[4 * q + 1] *= rs * o.y; f[4 * q + 2] *= rs * o.z; f[4 * q + 3] *= rs * o.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col0 + j < n) f[j] *= rs * l.col_scale[col0 + j];
        }
    }
    if (l.bias) {
        if (wide) {
            lin_add32(l.bias, col0, l.out_dtype, f);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col0 + j < n) f[j] += lin_load(l.bias, col0 + j, l.out_dtype);
        }
    }
}

// Everything after the product for four neighbouring products of one row (K slices: the sums come four at a time).
__device__ __forceinline__ void linear_finish4(const LinearParams& l, int n, int row, int col, float (&f)[4]) {
    const int dt = l.out_dtype;
    const float rs = l.row_scale ? l.row_scale[row] : 1.f;
    const long long y0 = (long long)row * l.y_rs + col, r0 = (long long)row * l.residual_rs + col, p0 = (long long)row * l.pre_rs + col;
    float r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool in = col + j < n;
        if (l.col_scale && in) f[j] *= rs * l.col_scale[col + j];
        if (l.bias && in) f[j] += lin_load(l.bias, col + j, dt);
        r[j] = l.residual && in ? lin_load(l.residual, r0 + j, dt) : 0.f;
    }
    float z[4] = {f[0], f[1], f[2], f[3]};
    if (dt == NTB200_F32) act_values<false>(l.act, f);
    else act_values<true>(l.act, f);
    if (l.vec_ok && col + 4 <= n) {
        if (dt == NTB200_F32) {
            if (l.pre) *reinterpret_cast<float4*>(static_cast<float*>(l.pre) + p0) = make_float4(z[0], z[1], z[2], z[3]);
            *reinterpret_cast<float4*>(static_cast<float*>(l.y) + y0) = make_float4(f[0] + r[0], f[1] + r[1], f[2] + r[2], f[3] + r[3]);
        } else {
            if (l.pre) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(l.pre) + p0) = make_uint2(lin_pack2(z[0], z[1], dt), lin_pack2(z[2], z[3], dt));
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(l.y) + y0) = make_uint2(lin_pack2(f[0] + r[0], f[1] + r[1], dt), lin_pack2(f[2] + r[2], f[3] + r[3], dt));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < n) {
            if (l.pre) lin_store(l.pre, p0 + j, z[j], dt);
            lin_store(l.y, y0 + j, f[j] + r[j], dt);
        }
}

// 32 consecutive products of one row, columns col0 ..: everything after the product, stored.
__device__ __forceinline__ void linear_finish32(const LinearParams& l, int n, int row, int col0, float (&f)[32]) {
    const int dt = l.out_dtype;
    const bool full = col0 + 32 <= n && l.vec_ok;
    linear_scale_bias32(l, n, col0, l.row_scale ? l.row_scale[row] : 1.f, full, f);
    const long long y0 = (long long)row * l.y_rs + col0, r0 = (long long)row * l.residual_rs + col0, p0 = (long long)row * l.pre_rs + col0;
    if (full) {
        if (l.pre) lin_store32(l.pre, p0, dt, f);
        if (dt == NTB200_F32) act_values<false>(l.act, f);
        else act_values<true>(l.act, f);
        if (l.residual) lin_add32(l.residual, r0, dt, f);
        lin_store32(l.y, y0, dt, f);
        return;
    }
    if (l.pre) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (col0 + j < n) lin_store(l.pre, p0 + j, f[j], dt);
    }
    if (dt == NTB200_F32) act_values<false>(l.act, f);
    else act_values<true>(l.act, f);
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (col0 + j < n) lin_store(l.y, y0 + j, f[j] + (l.residual ? lin_load(l.residual, r0 + j, dt) : 0.f), dt);
}

}  // namespace ntb200
