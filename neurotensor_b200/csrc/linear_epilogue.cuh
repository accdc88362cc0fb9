// What follows the product in ntb200_linear_act, on fp32 registers: scales, bias, activation, residual, one rounding.
// Shared by the epilogues of the GEMM kernels and the elementwise kernels of linear.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "row_ops.cuh"

namespace ntb200 {

// e^x for Float32 results: the hardware exponential of the rounded x log2(e), corrected to first order by what the rounding
// left out (relative error about 2^-22; without the correction it grows with |x|).  Straight-line code: calls of expf and
// erfcf, one value at a time, made the Float32 epilogue the longest part of its kernel.
__device__ __forceinline__ float exp_full(float x) {
    x = fminf(fmaxf(x, -150.f), 150.f);
    const float t = x * 1.44269504f;
    const float r = fmaf(x, 1.44269504f, -t) + x * 1.9259630e-8f;
    return exp2_hw(t) * fmaf(r, 0.69314718f, 1.f);
}
// kFast: results that are rounded to 16 bits use the hardware exponential as it is (a hundredth of half a Float16 step).
template <bool kFast>
__device__ __forceinline__ float sigmoid_times(float z, float u) {   // z / (1 + e^-u)
    return z * rcp_hw(1.f + (kFast ? exp2_hw(-1.4426950408889634f * u) : exp_full(-u)));
}

constexpr float kGeluScale = 1.5957691216057308f;   // 2 sqrt(2 / pi): z/2 (1 + tanh u) = z sigmoid(2 u)
constexpr float kGeluCubic = 0.044715f;

// Phi(z) = erfc(-z / sqrt 2) / 2 from e = e^(-z^2 / 2): Phi(-a) = e t P(t) with t = 1 / (1 + p a), P a fit of
// erfcx(a / sqrt 2) / (2 t) over 0 <= a <= 14 by least squares reweighted towards the minimax of the relative error, so the
// tail keeps its precision.  Relative error with the constants below, evaluated in 64 bits: degree 6, p = 0.36, below 1.1e-6 for
// 16-bit results; degree 8, p = 0.21, below 7e-8 (1.1e-7 rms with fp32's roundings) for Float32.
template <bool kFast>
__device__ __forceinline__ float gauss(float z) {
    if constexpr (kFast) return exp2_hw(-0.72134752044448170f * z * z);
    const float s = fminf(z * z, 400.f), low = z * z < 400.f ? fmaf(z, z, -s) : 0.f;   // the square's own rounding matters for large z
    return exp_full(-0.5f * s) * fmaf(-0.5f, low, 1.f);
}
template <bool kFast>
__device__ __forceinline__ float phi(float z, float e) {
    float q;
    if constexpr (kFast) {
        const float t = rcp_hw(1.f + 0.36f * fabsf(z));
        q = e * t * (0.14371304f + t * (0.14177254f + t * (0.13971882f + t * (0.026550606f + t * (0.1809521f + t * (-0.17976327f + t * 0.047055867f))))));
    } else {
        const float t = rcp_hw(1.f + 0.21f * fabsf(z));
        q = e * t * (0.08371158f + t * (0.085068814f + t * (0.069192477f + t * (0.1248716f + t * (-0.09392268f + t * (0.34939754f + t * (-0.33025047f +
                                                                                                                                     t * (0.28358722f + t * -0.071656048f))))))));
    }
    return z < 0.f ? q : 1.f - q;
}

template <bool kFast>
__device__ __forceinline__ float act_value(int act, float z) {
    switch (act) {
        case NTB200_ACT_RELU: return z < 0.f ? 0.f : z;
        case NTB200_ACT_GELU: return z * phi<kFast>(z, gauss<kFast>(z));
        case NTB200_ACT_GELU_TANH: return sigmoid_times<kFast>(z, kGeluScale * (z + kGeluCubic * z * z * z));
        case NTB200_ACT_SILU: return sigmoid_times<kFast>(z, z);
        default: return z;
    }
}

template <bool kFast>
__device__ __forceinline__ float act_slope(int act, float z) {
    switch (act) {
        case NTB200_ACT_RELU: return z < 0.f ? 0.f : 1.f;
        case NTB200_ACT_GELU: {
            const float e = gauss<kFast>(z);
            return fmaf(z * 0.39894228040143268f, e, phi<kFast>(z, e));
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

// A product times its row's and its column's scale.  kWide (Float32 results, whose operands' scales span the type's whole
// range): in an order whose steps neither overflow nor vanish unless the result does.
template <bool kWide>
__device__ __forceinline__ float scaled(float v, float rs, float cs) {
    if constexpr (!kWide) return v * rs * cs;
    const bool apart = (rs < 1.f) != (cs < 1.f);
    return v * (apart ? rs * cs : rs) * (apart ? 1.f : cs);
}

// Scales and bias of 32 consecutive products of one row; wide: every column is there and the vectors start on 16 bytes.
__device__ __forceinline__ void linear_scale_bias32(const LinearParams& l, int n, int col0, float rs, bool wide, float (&f)[32]) {
    if (l.col_scale) {
        if (wide) {
            const float4* cs = reinterpret_cast<const float4*>(l.col_scale + col0);
            if (l.out_dtype == NTB200_F32) {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 o = cs[q];
                    f[4 * q] = scaled<true>(f[4 * q], rs, o.x); f[4 * q + 1] = scaled<true>(f[4 * q + 1], rs, o.y);
                    f[4 * q + 2] = scaled<true>(f[4 * q + 2], rs, o.z); f[4 * q + 3] = scaled<true>(f[4 * q + 3], rs, o.w);
                }
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 o = cs[q];
                    f[4 * q] = scaled<false>(f[4 * q], rs, o.x); f[4 * q + 1] = scaled<false>(f[4 * q + 1], rs, o.y);
                    f[4 * q + 2] = scaled<false>(f[4 * q + 2], rs, o.z); f[4 * q + 3] = scaled<false>(f[4 * q + 3], rs, o.w);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col0 + j < n)
                    f[j] = l.out_dtype == NTB200_F32 ? scaled<true>(f[j], rs, l.col_scale[col0 + j]) : scaled<false>(f[j], rs, l.col_scale[col0 + j]);
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

// What four neighbouring products of one row need besides themselves; K-slice kernels load it before the sums are there.
struct LinearAhead4 {
    float rs, cs[4], bias[4], res[4];
};
__device__ __forceinline__ void linear_load_ahead4(const LinearParams& l, int n, int row, int col, LinearAhead4& a) {
    a.rs = l.row_scale ? l.row_scale[row] : 1.f;
    const long long r0 = (long long)row * l.residual_rs + col;
    if (l.vec_ok && col + 4 <= n) {
        if (l.col_scale) *reinterpret_cast<float4*>(a.cs) = *reinterpret_cast<const float4*>(l.col_scale + col);
        auto four = [&](const void* p, long long i, float (&o)[4]) {
            if (l.out_dtype == NTB200_F32) {
                *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
                o[0] = lin_up16(w.x & 0xffffu, l.out_dtype); o[1] = lin_up16(w.x >> 16, l.out_dtype);
                o[2] = lin_up16(w.y & 0xffffu, l.out_dtype); o[3] = lin_up16(w.y >> 16, l.out_dtype);
            }
        };
        if (l.bias) four(l.bias, col, a.bias);
        if (l.residual) four(l.residual, r0, a.res);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool in = col + j < n;
        if (l.col_scale) a.cs[j] = in ? l.col_scale[col + j] : 1.f;
        if (l.bias) a.bias[j] = in ? lin_load(l.bias, col + j, l.out_dtype) : 0.f;
        if (l.residual) a.res[j] = in ? lin_load(l.residual, r0 + j, l.out_dtype) : 0.f;
    }
}
// Everything after the product for them, stored.
__device__ __forceinline__ void linear_finish4(const LinearParams& l, int n, int row, int col, float (&f)[4], const LinearAhead4& a) {
    const int dt = l.out_dtype;
    const long long y0 = (long long)row * l.y_rs + col, p0 = (long long)row * l.pre_rs + col;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (l.col_scale) f[j] = dt == NTB200_F32 ? scaled<true>(f[j], a.rs, a.cs[j]) : scaled<false>(f[j], a.rs, a.cs[j]);
        if (l.bias) f[j] += a.bias[j];
    }
    const float z[4] = {f[0], f[1], f[2], f[3]};
    if (dt == NTB200_F32) act_values<false>(l.act, f);
    else act_values<true>(l.act, f);
    if (l.residual)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] += a.res[j];
    if (l.vec_ok && col + 4 <= n) {
        if (dt == NTB200_F32) {
            if (l.pre) *reinterpret_cast<float4*>(static_cast<float*>(l.pre) + p0) = make_float4(z[0], z[1], z[2], z[3]);
            *reinterpret_cast<float4*>(static_cast<float*>(l.y) + y0) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            if (l.pre) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(l.pre) + p0) = make_uint2(lin_pack2(z[0], z[1], dt), lin_pack2(z[2], z[3], dt));
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(l.y) + y0) = make_uint2(lin_pack2(f[0], f[1], dt), lin_pack2(f[2], f[3], dt));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < n) {
            if (l.pre) lin_store(l.pre, p0 + j, z[j], dt);
            lin_store(l.y, y0 + j, f[j], dt);
        }
}

// One element of y's type.
template <int kDt>
__device__ __forceinline__ float lin_get(const char* p) {
    if constexpr (kDt == NTB200_F32) return *reinterpret_cast<const float*>(p);
    else return lin_up16(*reinterpret_cast<const uint16_t*>(p), kDt);
}
template <int kDt>
__device__ __forceinline__ void lin_set(char* p, float v) {
    if constexpr (kDt == NTB200_F32) *reinterpret_cast<float*>(p) = v;
    else *reinterpret_cast<uint16_t*>(p) = uint16_t(lin_pack2(v, 0.f, kDt));
}

// What a warp needs besides the products of 32 rows x 32 columns, lane = column: the column's scale and bias, the
// residuals of its 32 rows, and (lane = row) the rows' scales.  Loaded before the products are there, all loads on their way together.
struct LinearAhead {
    float cs, bias, rs, res[32];
};
template <int kDt>
__device__ __forceinline__ void linear_load_ahead(const LinearParams& l, int m, int n, int row0, int col0, int lane, LinearAhead& a) {
    constexpr int es = kDt == NTB200_F32 ? 4 : 2;
    const int col = col0 + lane;
    const bool in = col < n;
    a.rs = l.row_scale && row0 + lane < m ? l.row_scale[row0 + lane] : 1.f;
    a.cs = l.col_scale && in ? l.col_scale[col] : 1.f;
    a.bias = l.bias && in ? lin_get<kDt>(static_cast<const char*>(l.bias) + (long long)col * es) : 0.f;
    if (l.residual && in) {
        const char* p = static_cast<const char*>(l.residual) + ((long long)row0 * l.residual_rs + col) * es;
        const long long step = l.residual_rs * es;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            a.res[r] = row0 + r < m ? lin_get<kDt>(p) : 0.f;
            p += step;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 32; ++r) a.res[r] = 0.f;
    }
}

// kRows x 32 products staged in shared memory (row pitch 33 floats; rows first .. first + kRows of the warp's 32), finished
// by a warp with lane = column: pre and y leave in runs of 32 elements of a row, whatever their alignment.
template <int kDt, int kRows>
__device__ __forceinline__ void linear_finish_block(const LinearParams& l, int m, int n, const float* staged, int row0, int first, int col0, int lane,
                                                    const LinearAhead& a) {
    constexpr int es = kDt == NTB200_F32 ? 4 : 2;
    const int col = col0 + lane;
    const bool in = col < n;
    char* y = static_cast<char*>(l.y) + ((long long)(row0 + first) * l.y_rs + col) * es;
    char* pre = static_cast<char*>(l.pre) + ((long long)(row0 + first) * l.pre_rs + col) * es;
    const long long y_step = l.y_rs * es, pre_step = l.pre_rs * es;
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 8) {
        if (row0 + first + r0 >= m) break;   // uniform across the warp
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = first + r0 + i;
            f[i] = staged[(r0 + i) * 33 + lane];
            if (l.row_scale) f[i] = scaled<kDt == NTB200_F32>(f[i], __shfl_sync(0xffffffffu, a.rs, r), a.cs);
            f[i] += a.bias;
            if (l.pre && in && row0 + r < m) lin_set<kDt>(pre, f[i]);
            pre += pre_step;
        }
        act_values<kDt != NTB200_F32>(l.act, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (in && row0 + first + r0 + i < m) lin_set<kDt>(y, f[i] + a.res[first + r0 + i]);
            y += y_step;
        }
    }
}

}  // namespace ntb200
