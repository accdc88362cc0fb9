// Distillation from a teacher's top logits: loss and gradient of the student's logits in one call.
//
//   p = softmax over the row's present entries of t / T          (K entries: values t, columns i; a column outside
//   q = softmax(s / T) over all V columns                          [0, V) or a value of -inf: an entry that is not there)
//   L = T^2 sum_j p_j (log p_j - log q_{i_j})                    loss = sum over rows of weight L
//   dloss/ds_v = weight T (q_v - sum_{j: i_j = v} p_j)
//
// A row without entries, or with weight 0, has L = 0 and a zero gradient, whatever its logits are (those of a row of weight 0
// are not read).  The softmax statistics are fp32: a running maximum and sum per thread, joined in a fixed order.  The kernel
// moves bytes: the logits once in, the gradient once out.
#include <algorithm>

#include "internal.h"
#include "row_ops.cuh"
#include "sm100_ptx.cuh"

namespace ntb200 {
namespace {

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kModerate = 64.f;   // |m c| up to which an exponent's error is below 2^-18

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

// T^2 (logs - cross / T) without T^2 and x / T, which leave the type's range at temperatures and logits whose loss does not.
__device__ __forceinline__ float row_loss_of(float temp, float logs, float cross) { return temp * (temp * logs - cross); }

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

// ---- one cluster per row: the row stays in shared memory ------------------------------------------------------------
// The C blocks of a cluster hold one row, a piece each, fetched once by an untiled bulk copy; maximum, sum and
// gradient then come from shared memory, and only (max, sum, teacher's share) of each piece crosses the cluster.  A block
// that re-read its row from L2 instead took 623 us for 4096 x 131072 bf16 logits: the rows in flight (592 x 256 KB) do not
// fit L2, so the second read went to memory again.  Pieces are at most 72 KB where C <= 8 allows it, so that three blocks
// per SM overlap loading, arithmetic and storing (36 KB: 562 us, 512 threads per block: 566 us; four barriers per copy to
// start earlier: 488 against 477 us; the gradient formed in shared memory and sent by a bulk store: 502 against 474).  Measured:
// 4096 x 131072 bf16 with 64 entries 466 - 506 us (4.2 - 4.6 TB/s), loss alone 297 us; bound by the chain a block goes through
// (load, maximum, sum, exchange, store) with three blocks per SM, not by the exponential unit (a polynomial for a quarter of the
// exponentials: 469 us).
// Rows need not start on 16 bytes: the piece's whole 16-byte granules are copied, the elements of a cut first or last
// granule are loaded one by one, and what else lies in those two granules is set to -inf, which adds nothing.
constexpr int kPieceThreads = 256, kMaxCluster = 8;

// Behind the piece in dynamic shared memory: three arrays of `top` entries (the teacher's probabilities; the same with
// those of a column's later entries added to its first, -1 for the later ones; the columns within this piece, -1: not there or
// in another block's piece).
struct PieceShared {
    float red[4][kPieceThreads / 32];
    float4 share[kMaxCluster];           // (max, sum, sum p (x - max), sum p) of every block's piece, by rank
    unsigned long long bar;
    uint32_t abort_flag;
};

// A maximum, or up to four sums, over the block in one exchange.
__device__ __forceinline__ float piece_max(float u, PieceShared& sh) {
    constexpr int W = kPieceThreads / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, o));
    if (lane == 0) sh.red[0][warp] = u;
    __syncthreads();
    u = sh.red[0][0];
#pragma unroll
    for (int i = 1; i < W; ++i) u = fmaxf(u, sh.red[0][i]);
    __syncthreads();
    return u;
}
template <int N>
__device__ __forceinline__ void piece_sums(float (&u)[N], PieceShared& sh) {
    constexpr int W = kPieceThreads / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        u[k] = warp_sum(u[k]);
        if (lane == 0) sh.red[k][warp] = u[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        u[k] = sh.red[k][0];
#pragma unroll
        for (int i = 1; i < W; ++i) u[k] += sh.red[k][i];
    }
    __syncthreads();
}

// The largest of V elements.  16-bit types compare two at a time, which changes no value (NaN is ignored either way and
// shows in the sum).
template <class T, int V>
__device__ __forceinline__ float pack_max(const Pack<T, V>& x) {
    if constexpr (sizeof(T) == 4) {
        float top = x.up(0);
#pragma unroll
        for (int k = 1; k < V; ++k) top = fmaxf(top, x.up(k));
        return top;
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2* p = reinterpret_cast<const T2*>(x.e);
        T2 top = p[0];
#pragma unroll
        for (int k = 1; k < V / 2; ++k) top = __hmax2(top, p[k]);
        return fmaxf(RowType<T>::up(top.x), RowType<T>::up(top.y));
    }
}

__device__ __forceinline__ void st_cluster_f4(uint32_t local_addr, uint32_t cta_rank, float4 v) {
    asm volatile(
        "{\n\t.reg .b32 remote;\n\t"
        "mapa.shared::cluster.u32 remote, %0, %1;\n\t"
        "st.shared::cluster.v4.f32 [remote], {%2, %3, %4, %5};\n\t}"
        ::"r"(local_addr), "r"(cta_rank), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// kBlocks: blocks per SM that registers shall allow (shared memory allows three of 72 KB, five of 42 KB).
template <class T, int kBlocks>
__global__ void __launch_bounds__(kPieceThreads, kBlocks) distill_piece_kernel(const DistillArgs a, int C, int piece, bool same_align, unsigned int* status) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t piece_mem[];
    __shared__ PieceShared sh;
    float* sh_p = reinterpret_cast<float*>(piece_mem + (size_t(piece) * sizeof(T) + 32));
    float* sh_q = sh_p + a.top;
    int* sh_at = reinterpret_cast<int*>(sh_q + a.top);
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t rank = C > 1 ? cluster_cta_rank() : 0u;
    const long long row = blockIdx.x / C;
    const float c = kLog2e / a.temp;
    const int first = int(rank) * piece, count = max(0, min(piece, a.vocab - first));
    const T* s = static_cast<const T*>(a.s) + row * a.s_rs + first;
    T* grad = a.grad ? static_cast<T*>(a.grad) + row * a.g_rs + first : nullptr;
    const float weight = a.weight ? a.weight[row] : a.even_weight;
    // granules of 16 bytes: element e of the piece sits at e + lead; granules [g0, g1) are whole
    const int lead = int((reinterpret_cast<uintptr_t>(s) & 15) / sizeof(T));
    const int granules = count ? (lead + count + V - 1) / V : 0;
    const int g0 = lead ? 1 : 0, g1 = (lead + count) / V;
    auto zeros = [&]() {
        if (!grad) return;
        const bool wide = same_align && g1 > g0;
        const int w0 = wide ? g0 * V - lead : 0, w1 = wide ? g1 * V - lead : 0;   // elements written 16 bytes at a time
        Pack<T, V> zero;
#pragma unroll
        for (int k = 0; k < V; ++k) zero.set(k, 0.f);
        for (int v = g0 + tid; wide && v < g1; v += kPieceThreads) reinterpret_cast<Pack<T, V>*>(grad - lead)[v] = zero;
        for (int v = tid; v < count - (w1 - w0); v += kPieceThreads) grad[v < w0 ? v : v + (w1 - w0)] = RowType<T>::down(0.f);
    };
    if (weight == 0.f) {
        zeros();
        if (rank == 0 && tid == 0) a.row_loss[row] = 0.f;
        return;
    }
    T* mem = reinterpret_cast<T*>(piece_mem);
    if (tid == 0) {
        sh.abort_flag = 0;
        mbar_init(smem_u32(&sh.bar), 1);
        fence_barrier_init();
        fence_proxy_async_smem();
        if (g1 > g0) {
            mbar_expect_tx(smem_u32(&sh.bar), uint32_t(g1 - g0) * 16u);
            bulk_load(smem_u32(piece_mem) + uint32_t(g0) * 16u, s + (g0 * V - lead), uint32_t(g1 - g0) * 16u, smem_u32(&sh.bar));
        }
    }
    if (tid < V && granules) {   // the cut granules
        if (g0 == 1) mem[tid] = tid >= lead && tid - lead < count ? s[tid - lead] : RowType<T>::down(-INFINITY);
        if (granules > g1 && (granules - 1 >= g0)) {
            const int e = (granules - 1) * V + tid - lead;
            mem[(granules - 1) * V + tid] = e < count ? s[e] : RowType<T>::down(-INFINITY);
        }
    }
    // the teacher's entries, in every block
    float tmax = -INFINITY;
    int present = 0;
    for (int j = tid; j < a.top; j += kPieceThreads) {
        const long long i = a.idx64 ? static_cast<const long long*>(a.idx)[row * a.top + j] : static_cast<const int*>(a.idx)[row * a.top + j];
        const float value = teacher_value(a, row * a.top + j);   // on its way together with the column
        const float t = i >= 0 && i < a.vocab ? value : -INFINITY;
        sh_at[j] = t != -INFINITY && i >= first && i < first + count ? int(i - first) : -1;
        sh_p[j] = t;
        present |= t != -INFINITY;
        tmax = fmaxf(tmax, t);
    }
    // their probabilities, while the piece is on its way
    present = __syncthreads_or(present);
    tmax = piece_max(tmax, sh);
    float tsums[1] = {0.f};
    for (int j = tid; j < a.top; j += kPieceThreads) tsums[0] += sh_p[j] == -INFINITY ? 0.f : exp2f((sh_p[j] - tmax) * c);
    piece_sums(tsums, sh);
    float sums[4] = {0.f, 0.f, 0.f, 0.f};   // sum p log2 p, and this piece's z, sum p and sum p (x - m)
    const float log2t = log2f(tsums[0]);
    for (int j = tid; j < a.top; j += kPieceThreads) {
        const float t = sh_p[j];
        float p = 0.f;
        if (t != -INFINITY) {
            const float lt = (t - tmax) * c;
            p = exp2f(lt) / tsums[0];
            if (p != 0.f) sums[0] += p * (lt - log2t);
        }
        sh_p[j] = p;
    }
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this block runs: its shared memory may be written
    float m = -INFINITY;
    if (granules > g1 && granules - 1 >= g0 && tid < V) m = RowType<T>::up(mem[(granules - 1) * V + tid]);
    if (g0 == 1 && tid < V) m = fmaxf(m, RowType<T>::up(mem[tid]));
    const bool landed = __all_sync(0xffffffffu, g1 <= g0 || mbar_wait(smem_u32(&sh.bar), 0, &sh.abort_flag));   // for every lane of the warp
#pragma unroll 4
    for (int v = g0 + tid; v < g1; v += kPieceThreads) m = fmaxf(m, pack_max(reinterpret_cast<const Pack<T, V>*>(mem)[v]));
    if (!landed && lane == 0) {
        sh.abort_flag = 1;
        atomicExch(status, 0x151u);
    }
    m = piece_max(m, sh);
    const float ref = m == -INFINITY ? 0.f : m, mc = ref * c;
    // 16-bit logits take one multiply-add to the exponent, x c - m c, as long as the rounding of m c (2^-24 of it) stays far
    // below the gradient's own; not so where all of a piece is masked by the type's lowest value
    const bool moderate = sizeof(T) == 2 && fabsf(mc) <= kModerate;
    for (int j = tid; j < a.top; j += kPieceThreads) {   // a thread's own entries of above
        const float p = sh_p[j];
        if (sh_at[j] < 0) continue;
        if (p != 0.f) {
            sums[2] += p;
            sums[3] += p * (RowType<T>::up(mem[sh_at[j] + lead]) - ref);
        }
    }
    float z0 = 0.f, z1 = 0.f;
    if (moderate) {
#pragma unroll 2
        for (int v = tid; v < granules; v += kPieceThreads) {
            const Pack<T, V> x = reinterpret_cast<const Pack<T, V>*>(mem)[v];
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                z0 += exp2_hw(fmaf(x.up(k), c, -mc));
                z1 += exp2_hw(fmaf(x.up(k + 1), c, -mc));
            }
        }
    } else {
#pragma unroll 2
        for (int v = tid; v < granules; v += kPieceThreads) {
            const Pack<T, V> x = reinterpret_cast<const Pack<T, V>*>(mem)[v];
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                z0 += exp2_hw((x.up(k) - ref) * c);
                z1 += exp2_hw((x.up(k + 1) - ref) * c);
            }
        }
    }
    sums[1] = z0 + z1;
    piece_sums(sums, sh);
    const float entropy = sums[0], z = sums[1], own_p = sums[2], own_x = sums[3];
    if (C > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (tid < C) st_cluster_f4(smem_u32(&sh.share[rank]), uint32_t(tid), make_float4(m, z, own_x, own_p));
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    // while the cluster meets: of a column's entries the first will write it, with the probabilities of all; a warp per entry
    for (int j = tid >> 5; grad && j < a.top; j += kPieceThreads / 32) {
        const int at = sh_at[j];
        if (at < 0) continue;
        float p = 0.f;
        bool first_one = true;
        for (int k0 = 0; k0 < a.top; k0 += 32) {
            unsigned same = __ballot_sync(0xffffffffu, k0 + lane < a.top && sh_at[min(k0 + lane, a.top - 1)] == at);
            if (same && k0 + __ffs(same) - 1 < j) first_one = false;
            for (; same; same &= same - 1) p += sh_p[k0 + __ffs(same) - 1];
        }
        if (lane == 0) sh_q[j] = first_one ? p : -1.f;
    }
    if (C > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        if (tid == 0) sh.share[0] = make_float4(m, z, own_x, own_p);
        __syncthreads();
    }
    if (sh.abort_flag) {   // a copy did not land in time (the status word tells): it may still, so the block waits once more
        volatile uint32_t never = 0;
        if (tid == 0 && g1 > g0) (void)mbar_wait(smem_u32(&sh.bar), 0, &never);
        __syncthreads();
        return;
    }
    float gm = -INFINITY, gz = 0.f, cross = 0.f;
    for (int i = 0; i < C; ++i) gm = fmaxf(gm, sh.share[i].x);
    for (int i = 0; i < C; ++i) {
        const float4 q = sh.share[i];
        const float d = q.x == -INFINITY ? 0.f : q.x - gm;
        gz += q.y * exp2f(d * c);        // an empty piece's sum is 0; one of nothing but NaN has the maximum of an empty one, and a NaN
        cross += q.w == 0.f ? q.z : q.z + q.w * d;   // sum p (x - gm); a piece far below may have an infinite d
    }
    if (gm == -INFINITY) gz = NAN;       // every column of the student masked out
    if (!present) {
        zeros();
        if (rank == 0 && tid == 0) a.row_loss[row] = 0.f;
        return;
    }
    if (rank == 0 && tid == 0) a.row_loss[row] = row_loss_of(a.temp, (entropy + log2f(gz)) / kLog2e, cross);
    if (!grad) return;
    const float coef = weight * a.temp, scale = coef / gz;
    // q times its factor: for 16-bit gradients one multiply-add and one exponential, the factor inside the exponent
    const bool fold = sizeof(T) == 2 && scale > 0.f && fabsf(gm) * c <= kModerate;
    const float off = fold ? fmaf(-gm, c, log2f(scale)) : 0.f;
    auto value = [&](float x) { return fold ? exp2_hw(fmaf(x, c, off)) : exp2_hw((x - gm) * c) * scale; };
    if (same_align && fold) {
        Pack<T, V>* gv = reinterpret_cast<Pack<T, V>*>(grad - lead);
#pragma unroll 2
        for (int v = g0 + tid; v < g1; v += kPieceThreads) {
            const Pack<T, V> x = reinterpret_cast<const Pack<T, V>*>(mem)[v];
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = exp2_hw(fmaf(x.up(k), c, off));
            Pack<T, V> q;
            q.put(o);
            gv[v] = q;
        }
    } else if (same_align) {
        Pack<T, V>* gv = reinterpret_cast<Pack<T, V>*>(grad - lead);
        for (int v = g0 + tid; v < g1; v += kPieceThreads) {
            const Pack<T, V> x = reinterpret_cast<const Pack<T, V>*>(mem)[v];
            Pack<T, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) o.set(k, value(x.up(k)));
            gv[v] = o;
        }
    }
    if (same_align) {
        if (tid < V && granules) {
            if (g0 == 1 && tid >= lead && tid - lead < count) grad[tid - lead] = RowType<T>::down(value(RowType<T>::up(mem[tid])));
            const int e = (granules - 1) * V + tid - lead;
            if (granules > g1 && granules - 1 >= g0 && e < count) grad[e] = RowType<T>::down(value(RowType<T>::up(mem[e + lead])));
        }
    } else {
        for (int v = tid; v < count; v += kPieceThreads) grad[v] = RowType<T>::down(value(RowType<T>::up(mem[v + lead])));
    }
    __syncthreads();
    for (int j = tid; j < a.top; j += kPieceThreads) {   // the teacher's places
        const int at = sh_at[j];
        if (at >= 0 && !(sh_q[j] < 0.f)) grad[at] = RowType<T>::down(scale * exp2f((RowType<T>::up(mem[at + lead]) - gm) * c) - coef * sh_q[j]);
    }
}

// One block per row, the row read twice: rows too long for eight blocks' shared memory.
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
                if (p > 0.f) loss += p * (a.temp * (((lt - log2f(tsum)) + log2z) / kLog2e) - (sh.x[j] - m));
                else if (!(p == 0.f)) loss = p;
            }
            sh.p[j] = p;
        }
        loss = block_sum<kThreads>(loss, sh.red_z);
        if (tid == 0) a.row_loss[row] = a.temp * loss;
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

// Blocks per row: the smallest power of two whose pieces are at most 72 KB (three blocks per SM), more while the rows leave
// SMs without a block and pieces stay above 8 KB; then whatever fits a block's shared memory.  0: the row does not.
int cluster_size(long long rows, int vocab, int es) {
    constexpr long long kMany = 72 * 1024, kMost = 200 * 1024;
    const long long bytes = (long long)vocab * es;
    int C = 1;
    while (C < kMaxCluster && (bytes > kMany * C || (rows * C * 2 <= sm_count() && bytes > 16 * 1024 * C))) C *= 2;
    return bytes > kMost * C ? 0 : C;
}

template <class T>
int launch_distill(const DistillArgs& a, bool vec_ok, float* loss, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    const int C = cluster_size(a.rows, a.vocab, int(sizeof(T)));
    if (C > 0 && a.rows * C < (1ll << 31)) {
        const int piece = int(((long long)a.vocab + C - 1) / C + 63) / 64 * 64;
        const uint32_t smem = uint32_t(piece) * uint32_t(sizeof(T)) + 32u + 12u * uint32_t(a.top);
        const bool same_align = a.grad && (reinterpret_cast<uintptr_t>(a.grad) - reinterpret_cast<uintptr_t>(a.s)) % 16 == 0 &&
                                ((a.g_rs - a.s_rs) * (long long)sizeof(T)) % 16 == 0;
        auto kernel = smem <= 42 * 1024 ? distill_piece_kernel<T, 5> : distill_piece_kernel<T, 3>;
        NTB200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 213 * 1024));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(a.rows * C), 1, 1);
        cfg.blockDim = dim3(kPieceThreads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = unsigned(C);
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        NTB200_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, C, piece, same_align, device_status_word()));
    } else {
        const int grid = int(std::min<long long>(a.rows, 1ll << 30));
        if (vec_ok) distill_kernel<T, kVec, 512><<<grid, 512, 0, stream>>>(a);
        else distill_kernel<T, 1, 512><<<grid, 512, 0, stream>>>(a);
    }
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
    if (!(temperature >= 1e-30) || !(temperature <= 1e30))
        return fail(NTB200_ERR_INVALID_ARG, "%s: the temperature must be positive and finite (1e-30 to 1e30)", what);
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
