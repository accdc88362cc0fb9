// Distillation from a teacher's top logits: loss and gradient of the student's logits in one call.
//
//   p = softmax over the row's present entries of t / T          (K entries: values t, columns i; a column outside
//   q = softmax(s / T) over all V columns                          [0, V) or a value of -inf: an entry that is not there)
//   L = T^2 sum_j p_j (log p_j - log q_{i_j})                    loss = sum over rows of weight L
//   dloss/ds_v = weight T (q_v - sum_{j: i_j = v} p_j)
//
// A row without entries, or with weight 0, has L = 0 and a zero gradient and its logits are not read.  The softmax
// statistics are fp32: a running maximum and sum per thread, joined in a fixed order.  The kernel moves bytes: the
// logits once in, the gradient once out.
#include <algorithm>

#include "internal.h"
#include "row_ops.cuh"

namespace ntb200 {
namespace {

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    const void* s; long long s_rs;
    const void* t;                       // [rows, top], f32 / f16 / bf16 (t_kind)
    const void* idx;                     // [rows, top], int32 or int64
    const float* weight;                 // [rows]; null: 1 / rows
    void* grad; long long g_rs;          // null: loss only
    float* row_loss;                     // [rows]
    long long rows;
    int vocab, top, t_kind, idx64;
    float temp, even_weight;
};

// (m, z): maximum and sum of 2^((x - m) c); joining two of them.  An empty one is (-inf, 0).
__device__ __forceinline__ void join(float& m, float& z, float m2, float z2, float c) {
    const float top = fmaxf(m, m2);
    const float ref = top == -INFINITY ? 0.f : top;
    z = z * exp2f((m - ref) * c) + z2 * exp2f((m2 - ref) * c);
    m = top;
}

template <int kThreads>
struct RowShared {
    float p[kMaxTop], x[kMaxTop];        // teacher's probabilities, the student's logits at the same places
    int at[kMaxTop];
    float red_m[kThreads / 32], red_z[kThreads / 32];
};

__device__ __forceinline__ float teacher_value(const DistillArgs& a, long long i) {
    if (a.t_kind == NTB200_F32) return static_cast<const float*>(a.t)[i];
    if (a.t_kind == NTB200_F16) return __half2float(static_cast<const __half*>(a.t)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.t)[i]);
}

template <int kThreads>
__device__ __forceinline__ float block_max(float v, float* red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < kThreads / 32 ? red[lane] : -INFINITY;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return warp_sum(lane < kThreads / 32 ? red[lane] : 0.f);
}

// One block per row.
template <class T, int V, int kThreads>
__global__ void __launch_bounds__(kThreads) distill_kernel(const DistillArgs a) {
    __shared__ RowShared<kThreads> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = kLog2e / a.temp;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* s = static_cast<const T*>(a.s) + row * a.s_rs;
        T* grad = a.grad ? static_cast<T*>(a.grad) + row * a.g_rs : nullptr;
        const float weight = a.weight ? a.weight[row] : a.even_weight;
        const int nv = a.vocab / V;
        // the teacher's entries
        float tmax = -INFINITY;
        int present = 0;
        __syncthreads();   // the previous row's readers are done with the shared arrays
        if (weight != 0.f)
            for (int j = tid; j < a.top; j += kThreads) {
                const long long i = a.idx64 ? static_cast<const long long*>(a.idx)[row * a.top + j]
                                            : static_cast<const int*>(a.idx)[row * a.top + j];
                const float t = i >= 0 && i < a.vocab ? teacher_value(a, row * a.top + j) : -INFINITY;
                const bool in = t != -INFINITY;
                sh.at[j] = in ? int(i) : -1;
                sh.p[j] = t;
                sh.x[j] = in ? RowType<T>::up(s[i]) : 0.f;
                present |= in;
                tmax = fmaxf(tmax, t);
            }
        present = __syncthreads_or(present);
        if (!present) {
            if (grad) {
                Pack<T, V> zero;
#pragma unroll
                for (int i = 0; i < V; ++i) zero.set(i, 0.f);
                for (int v = tid; v < nv; v += kThreads) reinterpret_cast<Pack<T, V>*>(grad)[v] = zero;
            }
            if (tid == 0) a.row_loss[row] = 0.f;
            continue;
        }
        tmax = block_max<kThreads>(tmax, sh.red_m);
        float tsum = 0.f;
        for (int j = tid; j < a.top; j += kThreads) {
            const float e = sh.at[j] < 0 ? 0.f : exp2f((sh.p[j] - tmax) * c);
            tsum += e;
        }
        tsum = block_sum<kThreads>(tsum, sh.red_z);
        // the student's maximum and sum
        const Pack<T, V>* sv = reinterpret_cast<const Pack<T, V>*>(s);
        float m = -INFINITY, z = 0.f;
        for (int v = tid; v < nv; v += kThreads) {
            const Pack<T, V> x = sv[v];
            float top = x.up(0);
#pragma unroll
            for (int i = 1; i < V; ++i) top = fmaxf(top, x.up(i));
            if (top > m) {
                z *= exp2f((m - top) * c);
                m = top;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < V; ++i) z += exp2f((x.up(i) - ref) * c);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o);
            join(m, z, m2, z2, c);
        }
        __syncthreads();
        if (lane == 0) { sh.red_m[warp] = m; sh.red_z[warp] = z; }
        __syncthreads();
        m = lane < kThreads / 32 ? sh.red_m[lane] : -INFINITY;
        z = lane < kThreads / 32 ? sh.red_z[lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o);
            join(m, z, m2, z2, c);
        }
        const float log2z = log2f(z);
        // the row's loss: sum_j p_j (log p_j - log q_{i_j})
        float loss = 0.f;
        for (int j = tid; j < a.top; j += kThreads) {
            float p = 0.f;
            if (sh.at[j] >= 0) {
                const float lt = (sh.p[j] - tmax) * c;
                p = exp2f(lt) / tsum;
                if (p > 0.f) loss += p * ((lt - log2f(tsum)) - ((sh.x[j] - m) * c - log2z));
                else if (!(p == 0.f)) loss = p;
            }
            sh.p[j] = p;
        }
        loss = block_sum<kThreads>(loss, sh.red_z);
        if (tid == 0) a.row_loss[row] = a.temp * a.temp * loss / kLog2e;
        if (!grad) continue;
        const float coef = weight * a.temp, scale = coef / z;
        for (int v = tid; v < nv; v += kThreads) {
            const Pack<T, V> x = sv[v];
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.set(i, scale * exp2f((x.up(i) - m) * c));
            reinterpret_cast<Pack<T, V>*>(grad)[v] = o;
        }
        __syncthreads();
        // the teacher's places: the first entry of a column writes it, with the probabilities of all its entries
        for (int j = tid; j < a.top; j += kThreads) {
            const int at = sh.at[j];
            if (at < 0) continue;
            bool first = true;
            for (int k = 0; k < j; ++k) first = first && sh.at[k] != at;
            if (!first) continue;
            float p = sh.p[j];
            for (int k = j + 1; k < a.top; ++k)
                if (sh.at[k] == at) p += sh.p[k];
            grad[at] = RowType<T>::down(scale * exp2f((sh.x[j] - m) * c) - coef * p);
        }
    }
}

// loss = sum over rows of weight times row loss, in a fixed order; rows of weight 0 are left out
__global__ void __launch_bounds__(1024) distill_total_kernel(const float* __restrict__ row_loss, const float* __restrict__ weight,
                                                             float even_weight, long long rows, float* loss) {
    __shared__ float red[32];
    float v = 0.f;
    for (long long r = threadIdx.x; r < rows; r += 1024) {
        const float w = weight ? weight[r] : even_weight;
        if (w != 0.f) v += w * row_loss[r];
    }
    v = block_sum<1024>(v, red);
    if (threadIdx.x == 0) *loss = v;
}

template <class T>
int launch_distill(const DistillArgs& a, bool vec_ok, float* loss, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    const int grid = int(std::min<long long>(a.rows, 1ll << 30));
    if (vec_ok) distill_kernel<T, kVec, 512><<<grid, 512, 0, stream>>>(a);
    else distill_kernel<T, 1, 512><<<grid, 512, 0, stream>>>(a);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    distill_total_kernel<<<1, 1024, 0, stream>>>(a.row_loss, a.weight, a.even_weight, a.rows, loss);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" int ntb200_distill_topk(int dtype, const void* logits, int64_t logits_row_stride, int teacher_dtype, const void* teacher,
                                   int index_dtype, const void* index, const float* row_weight, void* grad, int64_t grad_row_stride,
                                   float* row_loss, float* loss, int64_t rows, int64_t vocab, int64_t top, double temperature,
                                   void* stream) {
    const char* what = "distill_topk";
    auto is_float = [](int d) { return d == NTB200_F32 || d == NTB200_F16 || d == NTB200_BF16; };
    if (!is_float(dtype) || !is_float(teacher_dtype))
        return fail(NTB200_ERR_UNSUPPORTED, "%s: Float32, Float16 and BFloat16 only, got %s and %s", what, dtype_name(dtype), dtype_name(teacher_dtype));
    if (index_dtype != NTB200_I32 && index_dtype != NTB200_I64)
        return fail(NTB200_ERR_UNSUPPORTED, "%s: the teacher's columns must be Int32 or Int64, got %s", what, dtype_name(index_dtype));
    if (rows < 0 || vocab <= 0 || vocab > (int64_t(1) << 30) || top <= 0) return fail(NTB200_ERR_INVALID_ARG, "%s: bad extent", what);
    if (top > kMaxTop) return fail(NTB200_ERR_INVALID_ARG, "%s: at most %d teacher entries per row, got %lld", what, kMaxTop, (long long)top);
    if (!(temperature > 0) || !(temperature < 1e30)) return fail(NTB200_ERR_INVALID_ARG, "%s: the temperature must be positive and finite", what);
    if (!loss) return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        NTB200_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), s));
        return NTB200_OK;
    }
    if (!logits || !teacher || !index || !row_loss) return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows > 1 && (logits_row_stride < vocab || (grad && grad_row_stride < vocab)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: a row stride is shorter than a row", what);
    if (grad == logits && grad_row_stride != logits_row_stride)
        return fail(NTB200_ERR_INVALID_ARG, "%s: a gradient in the logits' place must have their row stride", what);
    const int64_t es = int64_t(dtype_size(dtype));
    const bool vec_ok = vocab * es % 16 == 0 && logits_row_stride * es % 16 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 &&
                        (!grad || (grad_row_stride * es % 16 == 0 && reinterpret_cast<uintptr_t>(grad) % 16 == 0));
    const DistillArgs a{logits, logits_row_stride, teacher, index, row_weight, grad, grad_row_stride, row_loss, rows, int(vocab), int(top),
                        teacher_dtype, index_dtype == NTB200_I64 ? 1 : 0, float(temperature), float(1.0 / double(rows))};
    switch (dtype) {
        case NTB200_F32: return launch_distill<float>(a, vec_ok, loss, s);
        case NTB200_F16: return launch_distill<__half>(a, vec_ok, loss, s);
        default: return launch_distill<__nv_bfloat16>(a, vec_ok, loss, s);
    }
}
