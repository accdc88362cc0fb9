// ntb200_linear_act and its backward pass: y = act(x w [* scales] + bias) + residual.
//
// The product runs on the tcgen05 kernels of gemm_umma.cu, whose epilogue does everything that follows the product on
// the fp32 accumulator (linear_epilogue.cuh): one launch, one rounding, no intermediate in memory but the
// pre-activation that the backward pass asks for.  Operands that TMA cannot address (rows that do not start on 16
// bytes) are copied once into padded rows in the caller's workspace.  Float32 has three kernels: few rows (or few terms) on
// the CUDA cores here, tiny K on the exact CUDA-core kernel, both finished by an elementwise pass, and everything else as
// three Float16 products on the tensor cores.
#include <algorithm>
#include <cstdlib>
#include <cstring>

#include "internal.h"
#include "linear_epilogue.cuh"
#include "row_ops.cuh"

namespace ntb200 {
namespace {

bool linear_float(int d) { return d == NTB200_F32 || d == NTB200_F16 || d == NTB200_BF16; }
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// y = act(z + bias) + residual, pre = z + bias, from an fp32 product in `slabs` partial sums (0: K = 0), added in their order.
__global__ void linear_finish_kernel(const float* __restrict__ z, int slabs, const LinearParams l, long long m, int n) {
    const long long total = m * n;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / n;
        const int col = int(i - row * n);
        float v = 0.f;
#pragma unroll 8
        for (int s = 0; s < slabs; ++s) v += z[s * total + i];
        if (l.bias) v += lin_load(l.bias, col, l.out_dtype);
        if (l.pre) lin_store(l.pre, row * l.pre_rs + col, v, l.out_dtype);
        v = l.out_dtype == NTB200_F32 ? act_value<false>(l.act, v) : act_value<true>(l.act, v);
        if (l.residual) v += lin_load(l.residual, row * l.residual_rs + col, l.out_dtype);
        lin_store(l.y, row * l.y_rs + col, v, l.out_dtype);
    }
}

// dst[r][c] = src[r * rs + c * cs], rows of dst ld elements apart (a multiple of 16 bytes), for one or two matrices in one
// launch.  One 16-byte store per thread; neighbouring threads read neighbouring elements where cs is 1.
struct PadJob {
    const void* src;
    void* dst;
    long long rs, cs, ld, rows, cols;
};
template <class U>
__global__ void pad_rows_kernel(const PadJob first, const PadJob second) {
    constexpr int V = 16 / sizeof(U);
    const long long total_first = first.rows * (first.ld / V), total = total_first + second.rows * (second.ld / V);
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const bool one = i < total_first;
        const PadJob& j = one ? first : second;
        const long long at = one ? i : i - total_first, per_row = j.ld / V;
        const long long r = at / per_row, c0 = (at - r * per_row) * V;
        const U* src = static_cast<const U*>(j.src) + r * j.rs + c0 * j.cs;
        Pack<U, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = c0 + k < j.cols ? src[k * j.cs] : U(0);
        *reinterpret_cast<Pack<U, V>*>(static_cast<U*>(j.dst) + r * j.ld + c0) = o;
    }
}

// ---- Float32, few rows ---------------------------------------------------------------------------------------------------
// y of up to 64 rows: the weight is what has to be read, so it is read as it is, 16 rows to a pass, and multiplied on the CUDA
// cores; splitting it first would cost three times its bytes, and few tiles would walk a long K one after another
// ([8, 4096] x [4096, 4096]: 101 us as three Float16 products).  K is cut into slices of whole 128s until there are six blocks per
// SM; their sums go to the workspace and are added in order by linear_finish_kernel.
struct FewRows {
    const float* a; long long a_ms, a_ks;
    const float* b; long long b_s;          // elements from one row (kAlongN) or column of b to the next
    float* out; long long out_rs;           // [slices][m] rows of n
    int m, n, k, slice;
};
constexpr int kFewRows = 16, kFewStep = 128, kFewThreads = 128;

// kAlongN: the weight's rows are dense along n; a thread takes two columns.  Otherwise dense along k: a warp takes four columns,
// its lanes 32 neighbouring k.
template <bool kAlongN>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const FewRows f) {
    __shared__ float xs[kAlongN ? kFewStep * (kFewRows + 4) : kFewRows * kFewStep];
    const int tid = threadIdx.x, lane = tid & 31;
    const int r0 = int(blockIdx.z) * kFewRows, rows = min(kFewRows, f.m - r0);
    const int k0 = int(blockIdx.y) * f.slice, k1 = min(f.k, k0 + f.slice);
    constexpr int kCols = kAlongN ? 2 : 4;
    const int col = kAlongN ? int(blockIdx.x) * (2 * kFewThreads) + tid : (int(blockIdx.x) * (kFewThreads / 32) + (tid >> 5)) * 4;
    constexpr int kNext = kAlongN ? kFewThreads : 1;   // from one of a thread's columns to its next
    float acc[kCols][kFewRows];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) acc[c][r] = 0.f;
    for (int kb = k0; kb < k1; kb += kFewStep) {
        __syncthreads();
        for (int r = 0; r < kFewRows; ++r)
            xs[kAlongN ? tid * (kFewRows + 4) + r : r * kFewStep + tid] = r < rows && kb + tid < k1 ? f.a[(r0 + r) * f.a_ms + (kb + tid) * f.a_ks] : 0.f;
        __syncthreads();
        if constexpr (kAlongN) {
            for (int kk = 0; kk < kFewStep && kb + kk < k1; kk += 8) {
                float w[2][8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        w[c][u] = kb + kk + u < k1 && col + c * kNext < f.n ? f.b[(kb + kk + u) * f.b_s + col + c * kNext] : 0.f;
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int r = 0; r < kFewRows; r += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(&xs[(kk + u) * (kFewRows + 4) + r]);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            acc[c][r] = fmaf(w[c][u], x.x, acc[c][r]);
                            acc[c][r + 1] = fmaf(w[c][u], x.y, acc[c][r + 1]);
                            acc[c][r + 2] = fmaf(w[c][u], x.z, acc[c][r + 2]);
                            acc[c][r + 3] = fmaf(w[c][u], x.w, acc[c][r + 3]);
                        }
                    }
            }
        } else {
            float w[kFewStep / 32][4];
#pragma unroll
            for (int u = 0; u < kFewStep / 32; ++u)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    w[u][c] = kb + lane + 32 * u < k1 && col + c < f.n ? f.b[(col + c) * f.b_s + kb + lane + 32 * u] : 0.f;
#pragma unroll
            for (int u = 0; u < kFewStep / 32; ++u)
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) {
                    const float x = xs[r * kFewStep + lane + 32 * u];
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[c][r] = fmaf(w[u][c], x, acc[c][r]);
                }
        }
    }
    float* out = f.out + ((long long)blockIdx.y * f.m + r0) * f.out_rs;
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        if (r >= rows) break;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const float v = kAlongN ? acc[c][r] : warp_sum(acc[c][r]);
            if ((kAlongN || lane == 0) && col + c * kNext < f.n) out[r * f.out_rs + col + c * kNext] = v;
        }
    }
}

// ---- Float32 as three Float16 products ----------------------------------------------------------------------------------
// A row of A (a column of B) is scaled by a power of two that brings its largest finite value to [2^14, 2^15), then
// x = hi + lo with hi = fp16(x), lo = fp16(x - hi): |x - hi| <= 2^-11 |x| and |x - hi - lo| <= 2^-23 |x| down to 2^-16 of the
// largest value (below that lo is subnormal: the error stays below 2^-39 of the largest value).  a.b = hi.hi + hi.lo + lo.hi, less
// lo.lo, up to 2^-22 |a||b|, and the parts' own errors, up to 2^-22 together; by their norm the three come to 8e-8 of the result.
// kind::f16 runs at twice TF32's rate and a value's two parts take 4 bytes instead of 8: [512, 1024] x [1024, 4096] took 30 us as
// three TF32 products.  The scales are undone by the epilogue's row and column factors (powers of two, exact).  Parts keep the
// operand's direction (tcgen05 takes Float16 tiles along either axis), so nothing is transposed.  [512, 1024] x [1024, 4096] with
// gelu: 34 us (46 when the split read its operands twice).
struct SplitF16Job {
    const float* src;
    __half* hi;
    __half* lo;
    float* unscale;                 // [mn]: what a product has to be multiplied by for this operand
    long long mn, k, mn_s, k_s, ld; // source strides; rows of the parts (along K, or along mn) are ld elements apart
    int along_k, blocks;
    int pairs;                      // values 2 i, 2 i + 1 of a row are neighbours and start on 8 bytes
};
constexpr int kSplitThreads = 1024;

__device__ __forceinline__ float split_scale(float top, float* unscale) {
    const int e = top > 0.f ? int(__float_as_uint(top) >> 23) : 141;
    const int bits = min(253, 268 - e);
    *unscale = __uint_as_float(uint32_t(254 - bits) << 23);
    return __uint_as_float(uint32_t(bits) << 23);
}
// Both parts of a pair of values.  An infinity is the largest Float16 of its sign and an infinite low part: its one infinite
// product is with the other value's high part, so the sum is the product's infinity (infinite high parts would meet low parts of
// zero or of the other sign).  A NaN's low part is NaN.
__device__ __forceinline__ void split_pair(float x, float y, float scale, __half2& hi, __half2& lo) {
    x *= scale;
    y *= scale;
    hi = __floats2half2_rn(fminf(fmaxf(x, -65504.f), 65504.f), fminf(fmaxf(y, -65504.f), 65504.f));
    lo = __floats2half2_rn(x - __low2float(hi), y - __high2float(hi));
}
__device__ __forceinline__ float max_finite(float top, float x) {
    const float a = fabsf(x);
    return a < INFINITY ? fmaxf(top, a) : top;
}

// Row and column jobs alike: a thread's values come in pairs that are neighbours in memory (where the source allows it:
// kPairs), and their parts leave as half2.
template <bool kPairs>
__device__ __forceinline__ float2 load_pair(const float* p, long long step, bool second) {
    if constexpr (kPairs) return *reinterpret_cast<const float2*>(p);
    return make_float2(p[0], second ? p[step] : 0.f);
}
__device__ __forceinline__ void store_parts(__half* hi, __half* lo, __half2 h, __half2 l) {   // rows of the parts are padded: a pair always fits
    *reinterpret_cast<__half2*>(hi) = h;
    *reinterpret_cast<__half2*>(lo) = l;
}

// Up to kHeld pairs of a thread stay in registers between the maximum and the split (K <= 1024): one read, all of it on its way at
// once.  Longer ones are read twice, the second time from L1 / L2.
constexpr int kHeld = 16, kHeldK = kHeld * 64;

template <bool kPairs>
__device__ __forceinline__ void split_rows(const SplitF16Job& j, int block, int warp, int lane) {   // a warp per row
    const long long r = (long long)block * 32 + warp;
    if (r >= j.mn) return;
    const int k = int(j.k);
    const long long step = j.k_s;
    const float* src = j.src + r * j.mn_s;
    __half* hi = j.hi + r * j.ld;
    __half* lo = j.lo + r * j.ld;
    float top = 0.f;
    if (k <= kHeldK) {
        float2 v[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int c = 2 * lane + 64 * i;
            v[i] = c < k ? load_pair<kPairs>(src + c * step, step, c + 1 < k) : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) top = max_finite(max_finite(top, v[i].x), v[i].y);
        top = warp_max_nan(top);
        float unscale;
        const float scale = split_scale(top, &unscale);
        if (lane == 0) j.unscale[r] = unscale;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int c = 2 * lane + 64 * i;
            __half2 h, l;
            split_pair(v[i].x, v[i].y, scale, h, l);
            if (c < k) store_parts(hi + c, lo + c, h, l);
        }
        return;
    }
#pragma unroll 8
    for (int c = 2 * lane; c < k; c += 64) {
        const float2 v = load_pair<kPairs>(src + c * step, step, c + 1 < k);
        top = max_finite(max_finite(top, v.x), v.y);
    }
    top = warp_max_nan(top);
    float unscale;
    const float scale = split_scale(top, &unscale);
    if (lane == 0) j.unscale[r] = unscale;
#pragma unroll 8
    for (int c = 2 * lane; c < k; c += 64) {   // from L1 / L2
        const float2 v = load_pair<kPairs>(src + c * step, step, c + 1 < k);
        __half2 h, l;
        split_pair(v.x, v.y, scale, h, l);
        store_parts(hi + c, lo + c, h, l);
    }
}

// 32 columns per block: 16 lanes on their pairs, 64 rows of K at a time.
template <bool kPairs>
__device__ __forceinline__ void split_columns(const SplitF16Job& j, int block, int warp, int lane, float (*red)[33]) {
    const int mn = int(j.mn), k = int(j.k);
    const int at = 2 * (lane & 15), c = block * 32 + at, row0 = 2 * warp + (lane >> 4);
    const bool in = c < mn, both = c + 1 < mn;
    const float* src = j.src + (long long)(in ? c : 0) * j.mn_s + row0 * j.k_s;
    const long long down = 64 * j.k_s;
    float tx = 0.f, ty = 0.f;
    const bool held = k <= kHeldK;
    float2 kept[kHeld];
    if (held) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) kept[i] = in && row0 + 64 * i < k ? load_pair<kPairs>(src + i * down, j.mn_s, both) : make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            tx = max_finite(tx, kept[i].x);
            ty = max_finite(ty, kept[i].y);
        }
    } else if (in) {
        const float* p = src;
#pragma unroll 8
        for (int r = row0; r < k; r += 64, p += down) {
            const float2 v = load_pair<kPairs>(p, j.mn_s, both);
            tx = max_finite(tx, v.x);
            ty = max_finite(ty, v.y);
        }
    }
    tx = fmaxf(tx, __shfl_xor_sync(0xffffffffu, tx, 16));
    ty = fmaxf(ty, __shfl_xor_sync(0xffffffffu, ty, 16));
    if (lane < 16) { red[warp][at] = tx; red[warp][at + 1] = ty; }
    __syncthreads();
    const float top = warp_max_nan(red[lane][warp]);   // warp w: the maximum of column w
    __syncthreads();
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
    if (!in) return;
    float ux, uy;
    const float sx = split_scale(red[0][at], &ux), sy = split_scale(red[0][at + 1], &uy);
    if (row0 == 0) {
        j.unscale[c] = ux;
        if (both) j.unscale[c + 1] = uy;
    }
    __half* hi = j.hi + row0 * j.ld + c;
    __half* lo = j.lo + row0 * j.ld + c;
    const long long out_down = 64 * j.ld;
    if (held) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            __half2 h, l;
            split_pair(kept[i].x * sx, kept[i].y * sy, 1.f, h, l);
            if (row0 + 64 * i < k) store_parts(hi + i * out_down, lo + i * out_down, h, l);
        }
        return;
    }
#pragma unroll 8
    for (int r = row0; r < k; r += 64, src += down, hi += out_down, lo += out_down) {
        const float2 v = load_pair<kPairs>(src, j.mn_s, both);
        __half2 h, l;
        split_pair(v.x * sx, v.y * sy, 1.f, h, l);
        store_parts(hi, lo, h, l);
    }
}

__global__ void __launch_bounds__(kSplitThreads) split_f16_kernel(const SplitF16Job ja, const SplitF16Job jb) {
    __shared__ float red[32][33];
    const bool second = int(blockIdx.x) >= ja.blocks;
    const SplitF16Job j = second ? jb : ja;
    const int block = int(blockIdx.x) - (second ? ja.blocks : 0), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (j.along_k) {
        if (j.pairs) split_rows<true>(j, block, warp, lane);
        else split_rows<false>(j, block, warp, lane);
    } else {
        if (j.pairs) split_columns<true>(j, block, warp, lane, red);
        else split_columns<false>(j, block, warp, lane, red);
    }
}

// gz = gy act'(pre), and the column sums of gz of one slab of rows per blockIdx.y (partial: [slabs, n]).  32 x 8 threads,
// each on V columns of every eighth row of the slab; the sums use gz before it is rounded.
// kAct is the activation, decided once per launch: a switch per value costs as much as the slope.  8192 x 16384 bf16 with the
// bias sums: relu and silu 136 us (5.9 TB/s), gelu 179 us (instructions of the two exponent and division steps and the fit).
template <class T, int V, int kAct>
__global__ void __launch_bounds__(256, 4) act_backward_kernel(const T* __restrict__ gy, long long gy_rs, const T* __restrict__ pre, long long pre_rs,
                                                           T* __restrict__ gz, long long gz_rs, float* __restrict__ partial, long long m,
                                                           int n, long long slab_rows) {
    __shared__ float red[8][32 * V + 1];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int col = (blockIdx.x * 32 + x) * V;
    const long long r0 = blockIdx.y * slab_rows, r1 = min(m, r0 + slab_rows);
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    if (col < n) {
#pragma unroll 4
        for (long long r = r0 + y; r < r1; r += 8) {
            const Pack<T, V> g = *reinterpret_cast<const Pack<T, V>*>(gy + r * gy_rs + col);
            Pack<T, V> o;
            if constexpr (kAct != NTB200_ACT_NONE) {
                const Pack<T, V> z = *reinterpret_cast<const Pack<T, V>*>(pre + r * pre_rs + col);
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[i] = g.up(i) * act_slope<sizeof(T) == 2>(kAct, z.up(i));
                    sum[i] += v[i];
                }
                o.put(v);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += g.up(i);
                o = g;
            }
            if (gz) *reinterpret_cast<Pack<T, V>*>(gz + r * gz_rs + col) = o;
        }
    }
    if (!partial) return;
#pragma unroll
    for (int i = 0; i < V; ++i) red[y][x * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        const int c = blockIdx.x * 32 * V + i;
        if (c >= n) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += red[k][i];
        partial[(long long)blockIdx.y * n + c] = v;
    }
}

template <class T>
__global__ void __launch_bounds__(256) join_slabs_kernel(const float* __restrict__ partial, T* __restrict__ out, int slabs, int n) {
    __shared__ float s[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < n)
        for (int i = y; i < slabs; i += 8) v += partial[(long long)i * n + c];
    s[y][x] = v;
    __syncthreads();
    if (y == 0 && c < n) {
        for (int i = 1; i < 8; ++i) v += s[i][x];
        out[c] = RowType<T>::down(v);
    }
}

// Slabs of rows of the bias gradient's partial sums: four blocks per SM, all resident at once, of at least 64 rows each.  148 SMs
// here and in plan_few: the workspace's size, which follows, depends on the call's sizes alone.
long long act_slabs(int64_t m, int64_t n, int vec) {
    const int64_t col_blocks = (n + 32 * vec - 1) / (32 * vec);
    int64_t slabs = std::max<int64_t>(1, std::min<int64_t>((m + 63) / 64, 148 * 4 / std::min<int64_t>(col_blocks, 148 * 4)));
    return std::min<int64_t>(slabs, 65535);
}

// A GEMM operand as [mn, k] with element strides.
struct Operand {
    const void* p;
    int64_t mn, k, mn_s, k_s;
};
// TMA can address it: one direction dense, the other in steps of 16 bytes that do not overlap (an expanded matrix repeats
// one row with a step of 0).
bool tma_ready(const Operand& o, int es) {
    if (!on16(o.p)) return false;
    return ((o.k_s == 1 || o.k == 1) && (o.mn == 1 || (o.mn_s * es % 16 == 0 && o.mn_s >= o.k))) ||
           ((o.mn_s == 1 || o.mn == 1) && (o.k == 1 || (o.k_s * es % 16 == 0 && o.k_s >= o.mn)));
}
// Bytes of the padded copy (0: none needed).
size_t padded_bytes(const Operand& o, int es) {
    if (tma_ready(o, es)) return 0;
    const bool along_k = o.k_s <= o.mn_s;
    const int64_t rows = along_k ? o.mn : o.k, cols = along_k ? o.k : o.mn, v = 16 / es;
    return round256(size_t(rows) * size_t((cols + v - 1) / v * v) * size_t(es));
}
int plan_pad(Operand& o, int es, PadJob* job, cudaStream_t stream) {
    *job = PadJob{nullptr, nullptr, 0, 0, 16, 0, 0};
    const size_t bytes = padded_bytes(o, es);
    if (bytes == 0) return NTB200_OK;
    void* copy = nullptr;
    if (int rc = scratch_acquire(&copy, bytes, stream)) return rc;
    const bool along_k = o.k_s <= o.mn_s;
    const int64_t rows = along_k ? o.mn : o.k, cols = along_k ? o.k : o.mn, v = 16 / es, ld = (cols + v - 1) / v * v;
    *job = PadJob{o.p, copy, along_k ? o.mn_s : o.k_s, along_k ? o.k_s : o.mn_s, ld, rows, cols};
    o.p = copy;
    o.mn_s = along_k ? ld : 1;
    o.k_s = along_k ? 1 : ld;
    return NTB200_OK;
}
// Padded copies of the operands that need one.
int pad_operands(Operand& a, Operand& b, int es, cudaStream_t stream) {
    PadJob ja, jb;
    if (int rc = plan_pad(a, es, &ja, stream)) return rc;
    if (int rc = plan_pad(b, es, &jb, stream)) return rc;
    const int64_t work = (ja.rows * ja.ld + jb.rows * jb.ld) / (16 / es);
    if (work == 0) return NTB200_OK;
    const int blocks = int(std::min<int64_t>((work + 255) / 256, int64_t(sm_count()) * 16));
    if (es == 1) pad_rows_kernel<uint8_t><<<blocks, 256, 0, stream>>>(ja, jb);
    else pad_rows_kernel<uint16_t><<<blocks, 256, 0, stream>>>(ja, jb);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

GemmArgs gemm_of(int dtype, const Operand& a, const Operand& b, void* c, int64_t c_rs) {
    GemmArgs g{};
    g.dtype = dtype;
    g.f16_rounding = NTB200_F16_ROUND_ONCE;
    g.m = a.mn; g.n = b.mn; g.k = a.k; g.batch = 1;
    g.a = a.p; g.a_rs = a.mn_s; g.a_cs = a.k_s; g.a_bs = 0;
    g.b = b.p; g.b_rs = b.k_s; g.b_cs = b.mn_s; g.b_bs = 0;
    g.c = c; g.c_rs = c_rs; g.c_bs = 0;
    return g;
}

// Float32 products for the exact CUDA-core kernel: few sums of few terms.  Its time grows with K alone while its tiles do not fill
// the GPU ([45, 2048] x [2048, 448]: 291 us, 42 on the tensor cores; K = 128: 27 and 17, K = 64: 19 and 17).
// NTB200_FP32_MODE=ffma asks for that kernel always.
bool f32_exact_only() {
    static const bool exact_only = [] { const char* e = getenv("NTB200_FP32_MODE"); return e && std::strcmp(e, "ffma") == 0; }();
    return exact_only;
}
bool small_f32(const GemmArgs& g) { return f32_exact_only() || (g.k <= 32 && double(g.m) * double(g.n) * double(g.k) < 6.0e7); }
// Slices of K for few_rows_kernel, 0 where another kernel takes the product.  Few rows: [64, 2048] x [2048, 2048] (2.7e8 multiply-adds)
// takes 30 us, as three Float16 products 42; further up the multiply-adds bound it.  Few terms (plain: the weight's gradient of few rows): the result
// is what has to be written, and it is written once, straight to its place.
struct FewPlan { int slices, slice; bool direct; };
FewPlan plan_few(const Operand& a, const Operand& b, bool plain) {
    const double work = double(a.mn) * double(b.mn) * double(a.k);
    if (f32_exact_only() || a.k == 0) return {0, 0, false};
    if (plain && a.k <= 32 && b.mn_s == 1 && work < 2.0e9 && a.mn <= 65535 * kFewRows) return {1, kFewStep, true};
    if (a.mn > 64 || (b.mn_s != 1 && b.k_s != 1) || work >= 3.0e8) return {0, 0, false};
    const int64_t cols = b.mn_s == 1 ? 2 * kFewThreads : 16, steps = (a.k + kFewStep - 1) / kFewStep;
    const int64_t blocks = (b.mn + cols - 1) / cols * ((a.mn + kFewRows - 1) / kFewRows);
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(steps, 148 * 6 / blocks)), per = (steps + want - 1) / want;
    const int slices = int((steps + per - 1) / per);
    return {slices, int(per * kFewStep), plain && slices == 1};
}
size_t few_bytes(const FewPlan& p, int64_t m, int64_t n) { return p.direct ? 0 : round256(size_t(p.slices) * size_t(m) * size_t(n) * 4); }
int few_product(const Operand& a, const Operand& b, const FewPlan& p, const LinearParams& l, cudaStream_t stream) {
    void* partial = l.y;
    if (!p.direct)
        if (int rc = scratch_acquire(&partial, few_bytes(p, a.mn, b.mn), stream)) return rc;
    const bool along_n = b.mn_s == 1;
    const FewRows f{static_cast<const float*>(a.p), a.mn_s, a.k_s, static_cast<const float*>(b.p), along_n ? b.k_s : b.mn_s,
                    static_cast<float*>(partial), p.direct ? l.y_rs : b.mn, int(a.mn), int(b.mn), int(a.k), p.slice};
    const int cols = along_n ? 2 * kFewThreads : 16;
    const dim3 grid(unsigned((b.mn + cols - 1) / cols), unsigned(p.slices), unsigned((a.mn + kFewRows - 1) / kFewRows));
    if (along_n) few_rows_kernel<true><<<grid, kFewThreads, 0, stream>>>(f);
    else few_rows_kernel<false><<<grid, kFewThreads, 0, stream>>>(f);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    if (p.direct) return NTB200_OK;
    const int blocks = int(std::min<int64_t>((a.mn * b.mn + 255) / 256, int64_t(sm_count()) * 16));
    linear_finish_kernel<<<blocks, 256, 0, stream>>>(static_cast<const float*>(partial), p.slices, l, a.mn, int(b.mn));
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

// Parts of one operand: rows along the direction in which its elements are closer together.
size_t parts_elements(const Operand& o) {
    const bool along_k = o.k_s <= o.mn_s;
    const int64_t rows = along_k ? o.mn : o.k, cols = along_k ? o.k : o.mn;
    return size_t(rows) * size_t((cols + 7) / 8 * 8);
}
size_t f16x3_bytes(const Operand& a, const Operand& b) {
    return 2 * 2 * (round256(parts_elements(a)) + round256(parts_elements(b))) + 4 * round256(size_t(a.mn)) + 4 * round256(size_t(b.mn)) + 4096;
}
// y of `l` from Float32 operands on the tensor cores; l's scales are free.
int f16x3_product(const Operand& a, const Operand& b, LinearParams l, cudaStream_t stream) {
    Operand parts[2] = {a, b};
    SplitF16Job jobs[2];
    void* lo[2];
    for (int i = 0; i < 2; ++i) {
        Operand& o = parts[i];
        const bool along_k = o.k_s <= o.mn_s;
        const int64_t ld = ((along_k ? o.k : o.mn) + 7) / 8 * 8;
        const size_t bytes = 2 * round256(parts_elements(o));
        void *hi = nullptr, *unscale = nullptr;
        if (int rc = scratch_acquire(&hi, 2 * bytes, stream)) return rc;
        if (int rc = scratch_acquire(&unscale, 4 * size_t(o.mn), stream)) return rc;
        lo[i] = static_cast<char*>(hi) + bytes;
        jobs[i] = SplitF16Job{static_cast<const float*>(o.p), static_cast<__half*>(hi), static_cast<__half*>(lo[i]), static_cast<float*>(unscale),
                              o.mn, o.k, o.mn_s, o.k_s, ld, along_k ? 1 : 0, int((o.mn + 31) / 32),
                              (along_k ? o.k_s == 1 && o.mn_s % 2 == 0 && o.k % 2 == 0 : o.mn_s == 1 && o.k_s % 2 == 0 && o.mn % 2 == 0) &&
                                      reinterpret_cast<uintptr_t>(o.p) % 8 == 0 ? 1 : 0};
        o.p = hi;
        o.mn_s = along_k ? ld : 1;
        o.k_s = along_k ? 1 : ld;
    }
    split_f16_kernel<<<unsigned(jobs[0].blocks + jobs[1].blocks), kSplitThreads, 0, stream>>>(jobs[0], jobs[1]);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    l.row_scale = jobs[0].unscale;
    l.col_scale = jobs[1].unscale;
    GemmArgs g = gemm_of(NTB200_F16, parts[0], parts[1], l.y, l.y_rs);
    g.linear = &l;
    return launch_umma_f16x3(g, lo[0], lo[1], stream);
}

// One plain product of the backward pass: its scratch beyond padded copies.
size_t product_bytes(const GemmArgs& g, const Operand& a, const Operand& b) {
    if (g.dtype == NTB200_F32) {
        const FewPlan few = plan_few(a, b, true);
        return few.slices ? few_bytes(few, a.mn, b.mn) : small_f32(g) ? 0 : f16x3_bytes(a, b);
    }
    return umma_scratch_bytes(g) + gemv_scratch_bytes(g) + 1024;
}
int plain_product(int dtype, Operand a, Operand b, void* c, int64_t c_rs, cudaStream_t stream) {
    if (a.mn == 0 || b.mn == 0) return NTB200_OK;
    if (dtype != NTB200_F32)
        if (int rc = pad_operands(a, b, 2, stream)) return rc;
    GemmArgs g = gemm_of(dtype, a, b, c, c_rs);
    // Rows that TMA cannot store would leave a plain GEMM element by element, thread by thread: ntb200_linear_act's
    // epilogue moves them by rows.  Large Float32 products are three Float16 ones.
    LinearParams l{};
    l.y = c; l.y_rs = c_rs; l.act = NTB200_ACT_NONE; l.out_dtype = dtype;
    if (dtype == NTB200_F32) {
        const FewPlan few = plan_few(a, b, true);
        if (few.slices) return few_product(a, b, few, l, stream);
        if (!small_f32(g)) return f16x3_product(a, b, l, stream);
    }
    if (dtype != NTB200_F32 && (c_rs % 8 != 0 || !on16(c))) {
        g.linear = &l;
        return launch_umma_gemm(g, stream);
    }
    return route_gemm(g, NTB200_ROUTE_AUTO, stream);
}

int check_linear(const ntb200_linear_desc* d) {
    const char* what = "linear_act";
    if (!d) return fail(NTB200_ERR_INVALID_ARG, "%s: null descriptor", what);
    const bool int8 = d->dtype == NTB200_I8;
    if (!int8 && !linear_float(d->dtype))
        return fail(NTB200_ERR_UNSUPPORTED, "%s: Float32, Float16, BFloat16 and Int8 only, got %s", what, dtype_name(d->dtype));
    if (!linear_float(d->out_dtype) || (!int8 && d->out_dtype != d->dtype))
        return fail(NTB200_ERR_INVALID_ARG, "%s: the output of %s operands cannot be %s", what, dtype_name(d->dtype), dtype_name(d->out_dtype));
    if (d->activation < NTB200_ACT_NONE || d->activation > NTB200_ACT_SILU)
        return fail(NTB200_ERR_INVALID_ARG, "%s: unknown activation %d", what, d->activation);
    if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > (int64_t(1) << 30) || d->n > (int64_t(1) << 30) || d->k > (int64_t(1) << 30))
        return fail(NTB200_ERR_INVALID_ARG, "%s: bad extent", what);
    if (int8 && d->k > 131071) return fail(NTB200_ERR_INVALID_ARG, "%s: Int8 sums are exact up to K = 131071, got %lld", what, (long long)d->k);
    if (d->x_row_stride < 0 || d->x_col_stride < 0 || d->w_row_stride < 0 || d->w_col_stride < 0)
        return fail(NTB200_ERR_INVALID_ARG, "%s: negative stride", what);
    if (d->m > 1 && (d->y_row_stride < d->n || (d->pre && d->pre_row_stride < d->n) || (d->residual && d->residual_row_stride < d->n)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: a row stride is shorter than a row", what);
    if (d->m == 0 || d->n == 0) return NTB200_OK;
    if (!d->y || (d->k > 0 && (!d->x || !d->w)) || (int8 && (!d->x_scale || !d->w_scale)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    if (!int8 && (d->x_scale || d->w_scale)) return fail(NTB200_ERR_INVALID_ARG, "%s: scales belong to Int8 operands", what);
    if (d->pre && (d->pre == d->y || d->pre == d->residual))
        return fail(NTB200_ERR_INVALID_ARG, "%s: the pre-activation needs memory of its own", what);
    if (d->y == d->x || d->y == d->w || (d->pre && (d->pre == d->x || d->pre == d->w)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: an output in an operand's place", what);
    if (d->residual && d->residual == d->y && d->residual_row_stride != d->y_row_stride)
        return fail(NTB200_ERR_INVALID_ARG, "%s: an output in the residual's place must have its row stride", what);
    return NTB200_OK;
}

Operand x_of(const ntb200_linear_desc& d) { return Operand{d.x, d.m, d.k, d.x_row_stride, d.x_col_stride}; }
Operand w_of(const ntb200_linear_desc& d) { return Operand{d.w, d.n, d.k, d.w_col_stride, d.w_row_stride}; }

int check_backward(const ntb200_linear_backward_desc* d) {
    const char* what = "linear_act_backward";
    if (!d) return fail(NTB200_ERR_INVALID_ARG, "%s: null descriptor", what);
    if (!linear_float(d->dtype)) return fail(NTB200_ERR_UNSUPPORTED, "%s: Float32, Float16 and BFloat16 only, got %s", what, dtype_name(d->dtype));
    if (d->activation < NTB200_ACT_NONE || d->activation > NTB200_ACT_SILU)
        return fail(NTB200_ERR_INVALID_ARG, "%s: unknown activation %d", what, d->activation);
    if (d->m < 0 || d->n <= 0 || d->k <= 0 || d->m > (int64_t(1) << 30) || d->n > (int64_t(1) << 30) || d->k > (int64_t(1) << 30))
        return fail(NTB200_ERR_INVALID_ARG, "%s: bad extent", what);
    if (d->x_row_stride < 0 || d->x_col_stride < 0 || d->w_row_stride < 0 || d->w_col_stride < 0)
        return fail(NTB200_ERR_INVALID_ARG, "%s: negative stride", what);
    if (d->m > 1 && (d->grad_out_row_stride < d->n || (d->pre && d->pre_row_stride < d->n)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: a row stride is shorter than a row", what);
    if (d->m == 0) return NTB200_OK;
    if (!d->grad_out || (d->activation != NTB200_ACT_NONE && !d->pre) || (d->grad_x && !d->w) || (d->grad_w && !d->x))
        return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    for (const void* out : {static_cast<const void*>(d->grad_x), static_cast<const void*>(d->grad_w), static_cast<const void*>(d->grad_bias)})
        if (out && (out == d->grad_out || out == d->pre || out == d->x || out == d->w))
            return fail(NTB200_ERR_INVALID_ARG, "%s: a gradient in an input's place", what);
    return NTB200_OK;
}

// How the backward pass forms gz: its row stride (rows start on 16 bytes), whether it is grad_out itself, and whether
// grad_out and pre can be read 16 bytes at a time.
struct GzPlan { int64_t ld; bool own; bool vec; long long slabs; };
GzPlan plan_gz(const ntb200_linear_backward_desc& d) {
    const int es = int(dtype_size(d.dtype)), v = 16 / es;
    const bool act = d.activation != NTB200_ACT_NONE;
    const bool rows16 = on16(d.grad_out) && (d.m == 1 || d.grad_out_row_stride * es % 16 == 0);
    GzPlan p;
    p.vec = d.n % v == 0 && rows16 && (!act || (on16(d.pre) && (d.m == 1 || d.pre_row_stride * es % 16 == 0)));
    p.own = act || (!rows16 && d.dtype != NTB200_F32);
    p.ld = p.own ? (d.n + v - 1) / v * v : d.grad_out_row_stride;
    p.slabs = act_slabs(d.m, d.n, p.vec ? v : 1);
    return p;
}

template <class T>
int launch_gz(const ntb200_linear_backward_desc& d, const GzPlan& p, void* gz, float* partial, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    const long long per = (d.m + p.slabs - 1) / p.slabs;
    const int slabs = int((d.m + per - 1) / per);
    const T* gy = static_cast<const T*>(d.grad_out);
    const T* pre = d.activation != NTB200_ACT_NONE ? static_cast<const T*>(d.pre) : nullptr;
    const int v = p.vec ? kVec : 1;
    const dim3 grid(unsigned((d.n + 32 * v - 1) / (32 * v)), unsigned(slabs));
#define NTB200_GZ(VV, AA) \
    act_backward_kernel<T, VV, AA><<<grid, 256, 0, stream>>>(gy, d.grad_out_row_stride, pre, d.pre_row_stride, static_cast<T*>(gz), p.ld, partial, d.m, int(d.n), per)
#define NTB200_GZ_ACT(AA)              \
    case AA:                           \
        if (p.vec) NTB200_GZ(kVec, AA); \
        else NTB200_GZ(1, AA);         \
        break
    switch (d.activation) {
        NTB200_GZ_ACT(NTB200_ACT_NONE);
        NTB200_GZ_ACT(NTB200_ACT_RELU);
        NTB200_GZ_ACT(NTB200_ACT_GELU);
        NTB200_GZ_ACT(NTB200_ACT_GELU_TANH);
        NTB200_GZ_ACT(NTB200_ACT_SILU);
    }
#undef NTB200_GZ_ACT
#undef NTB200_GZ
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    if (partial) {
        join_slabs_kernel<T><<<unsigned((d.n + 31) / 32), 256, 0, stream>>>(partial, static_cast<T*>(d.grad_bias), slabs, int(d.n));
        count_launch();
        NTB200_CUDA(cudaGetLastError());
    }
    return NTB200_OK;
}

// The two products of the backward pass over gz: operands in the order GemmArgs wants them.
void backward_operands(const ntb200_linear_backward_desc& d, const void* gz, int64_t ld, Operand (&dx)[2], Operand (&dw)[2]) {
    dx[0] = Operand{gz, d.m, d.n, ld, 1};                               // gx[m, k] = gz[m, n] . w[k, n]^T
    dx[1] = Operand{d.w, d.k, d.n, d.w_row_stride, d.w_col_stride};
    dw[0] = Operand{d.x, d.k, d.m, d.x_col_stride, d.x_row_stride};     // gw[k, n] = x^T . gz
    dw[1] = Operand{gz, d.n, d.m, 1, ld};
    if (d.grad_w_transposed) std::swap(dw[0], dw[1]);                   // gw[n, k] = gz^T . x
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" {

size_t ntb200_linear_act_workspace_bytes(const ntb200_linear_desc* d) {
    if (check_linear(d) || d->m == 0 || d->n == 0 || d->k == 0) return 0;
    if (d->dtype == NTB200_F32) {
        const GemmArgs g = gemm_of(d->dtype, x_of(*d), w_of(*d), d->y, d->y_row_stride);
        const FewPlan few = plan_few(x_of(*d), w_of(*d), false);
        return few.slices ? few_bytes(few, d->m, d->n) : small_f32(g) ? round256(size_t(d->m) * size_t(d->n) * 4) : f16x3_bytes(x_of(*d), w_of(*d));
    }
    const int es = int(dtype_size(d->dtype));
    GemmArgs g = gemm_of(d->dtype, x_of(*d), w_of(*d), d->y, d->y_row_stride);
    const LinearParams l{};
    g.linear = &l;
    return padded_bytes(x_of(*d), es) + padded_bytes(w_of(*d), es) + umma_scratch_bytes(g);
}

int ntb200_linear_act(const ntb200_linear_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_linear(d)) return rc;
    if (d->m == 0 || d->n == 0) return NTB200_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (workspace_bytes > 0 && (!workspace || !on16(workspace)))
        return fail(NTB200_ERR_INVALID_ARG, "linear_act: the workspace must start on 16 bytes");
    const ScratchArena arena(workspace, workspace_bytes);
    const int oes = int(dtype_size(d->out_dtype));
    LinearParams l{};
    l.row_scale = d->x_scale; l.col_scale = d->w_scale;
    l.bias = d->bias;
    l.residual = d->residual; l.residual_rs = d->residual_row_stride;
    l.y = d->y; l.y_rs = d->y_row_stride;
    l.pre = d->pre; l.pre_rs = d->pre_row_stride;
    l.act = d->activation; l.out_dtype = d->out_dtype;
    auto rows16 = [&](const void* p, int64_t rs) { return !p || (on16(p) && (d->m == 1 || rs * oes % 16 == 0)); };
    l.vec_ok = rows16(l.y, l.y_rs) && rows16(l.residual, l.residual_rs) && rows16(l.pre, l.pre_rs) && on16(l.bias) && on16(l.col_scale);
    Operand x = x_of(*d), w = w_of(*d);
    GemmArgs g = gemm_of(d->dtype, x, w, d->y, d->y_row_stride);
    const FewPlan few = d->dtype == NTB200_F32 ? plan_few(x, w, false) : FewPlan{};
    if (few.slices) return few_product(x, w, few, l, s);
    if (d->k == 0 || (d->dtype == NTB200_F32 && small_f32(g))) {
        void* z = nullptr;
        if (d->k > 0) {
            if (int rc = scratch_acquire(&z, size_t(d->m) * size_t(d->n) * 4, s)) return rc;
            g.c = z; g.c_rs = d->n;
            if (int rc = launch_simt_gemm(g, s)) return rc;
        }
        const int blocks = int(std::min<int64_t>((d->m * d->n + 255) / 256, int64_t(sm_count()) * 16));
        linear_finish_kernel<<<blocks, 256, 0, s>>>(static_cast<const float*>(z), z ? 1 : 0, l, d->m, int(d->n));
        count_launch();
        NTB200_CUDA(cudaGetLastError());
        return NTB200_OK;
    }
    if (d->dtype == NTB200_F32) return f16x3_product(x, w, l, s);
    if (int rc = pad_operands(x, w, int(dtype_size(d->dtype)), s)) return rc;
    g = gemm_of(d->dtype, x, w, d->y, d->y_row_stride);
    g.linear = &l;
    return launch_umma_gemm(g, s);
}

size_t ntb200_linear_act_backward_workspace_bytes(const ntb200_linear_backward_desc* d) {
    if (check_backward(d) || d->m == 0) return 0;
    const int es = int(dtype_size(d->dtype));
    const GzPlan p = plan_gz(*d);
    size_t bytes = 1024;
    if (p.own) bytes += round256(size_t(d->m) * size_t(p.ld) * size_t(es));
    if (d->grad_bias) bytes += round256(size_t(p.slabs) * size_t(d->n) * 4);
    Operand dx[2], dw[2];
    backward_operands(*d, p.own ? nullptr : d->grad_out, p.ld, dx, dw);
    for (const auto* o : {dx, dw}) {
        if (o == dx ? !d->grad_x : !d->grad_w) continue;
        if (d->dtype != NTB200_F32) bytes += padded_bytes(o[0], es) + padded_bytes(o[1], es);
        bytes += product_bytes(gemm_of(d->dtype, o[0], o[1], nullptr, o[1].mn), o[0], o[1]);
    }
    return bytes;
}

int ntb200_linear_act_backward(const ntb200_linear_backward_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_backward(d)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (workspace_bytes > 0 && (!workspace || !on16(workspace)))
        return fail(NTB200_ERR_INVALID_ARG, "linear_act_backward: the workspace must start on 16 bytes");
    const size_t es = dtype_size(d->dtype);
    if (d->m == 0) {   // no rows: the weights' gradients are sums of nothing
        if (d->grad_w) NTB200_CUDA(cudaMemsetAsync(d->grad_w, 0, size_t(d->k) * size_t(d->n) * es, s));
        if (d->grad_bias) NTB200_CUDA(cudaMemsetAsync(d->grad_bias, 0, size_t(d->n) * es, s));
        return NTB200_OK;
    }
    const ScratchArena arena(workspace, workspace_bytes);
    const GzPlan p = plan_gz(*d);
    const void* gz = d->grad_out;
    void* own = nullptr;
    float* partial = nullptr;
    if (p.own) {
        if (int rc = scratch_acquire(&own, size_t(d->m) * size_t(p.ld) * es, s)) return rc;
        gz = own;
    }
    if (d->grad_bias)
        if (int rc = scratch_acquire(reinterpret_cast<void**>(&partial), size_t(p.slabs) * size_t(d->n) * 4, s)) return rc;
    if (p.own || partial) {
        int rc;
        if (d->dtype == NTB200_F32) rc = launch_gz<float>(*d, p, own, partial, s);
        else if (d->dtype == NTB200_F16) rc = launch_gz<__half>(*d, p, own, partial, s);
        else rc = launch_gz<__nv_bfloat16>(*d, p, own, partial, s);
        if (rc) return rc;
    }
    Operand dx[2], dw[2];
    backward_operands(*d, gz, p.ld, dx, dw);
    if (d->grad_x && d->grad_w && d->dtype != NTB200_F32)   // both copies in one launch
        if (int rc = pad_operands(dx[1], dw[d->grad_w_transposed ? 1 : 0], int(es), s)) return rc;
    if (d->grad_x)
        if (int rc = plain_product(d->dtype, dx[0], dx[1], d->grad_x, d->k, s)) return rc;
    if (d->grad_w)
        if (int rc = plain_product(d->dtype, dw[0], dw[1], d->grad_w, d->grad_w_transposed ? d->k : d->n, s)) return rc;
    return NTB200_OK;
}

}  // extern "C"
