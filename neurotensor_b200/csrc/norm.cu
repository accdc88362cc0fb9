// Root-mean-square norm with the residual's addition, its backward pass, and the quantisation of rows to Int8.
//
//   h = x + r        rstd = (mean(h^2) + eps)^-1/2        y = h rstd w
//   Int8:   u = h w,  A = max |u|,  q = rint(u 127 / A),  scale = A rstd / 127        (y = q scale; rstd cancels out of q)
//   backward, given h, rstd, gy = dL/dy and gh = dL/dh over the residual stream:
//           g = gy w,  xhat = h rstd,  gx = rstd (g - xhat mean(g xhat)) + gh,  gw = sum over rows of gy xhat
//
// All sums run in fp32 on the unrounded h; y, h and gx are rounded once, when they are stored.  These kernels move
// bytes: 8 per element for a 16-bit forward pass with residual (x, r in; y, h out), as many for the backward pass.
// The backward pass starts from h as it was stored, which is what a training step keeps: for 16 bits that rounding puts an
// error of its own, as large as the last rounding's, into the weight's gradient (x and r read again would cost 25 % more bytes).
#include <algorithm>

#include "internal.h"
#include "row_ops.cuh"
#include "sm100_ptx.cuh"

namespace ntb200 {
namespace {

enum RowOut : int { kSame = 0, kInt8 = 1 };

struct RowArgs {
    const void* x; long long x_rs;
    const void* r; long long r_rs;      // null: no residual
    const void* w;                      // null: no norm, quantise the row itself
    void* y;                            // [rows, cols], type of x or int8
    void* h; float* stat;               // stat: rstd (16 / 32-bit output) or the row's scale (Int8 output)
    long long rows; int cols;
    float eps;
};

// q = rint(u * 127 / A), which lies within +-127 but for roundings; a row of zeros gives zeros, and so does a row with a NaN or
// an infinity (its scale is not finite, so the product that reads it is NaN).  A below 2^-100 is scaled up first: 127 / A would
// overflow.
struct Quant {
    float up, inv;
    __device__ __forceinline__ explicit Quant(float top) {
        up = top < 0x1p-100f ? 0x1p100f : 1.f;
        inv = top > 0.f && top < INFINITY ? __fdiv_rn(127.f, __fmul_rn(top, up)) : (top == 0.f ? 0.f : NAN);
    }
    // V values, packed.  Adding 1.5 2^23 rounds to a whole number (ties to even, as rint does) and leaves it in the low byte
    // of the sum's bits: no conversion, which the hardware does at a quarter of the rate.  127 (1 + 2^-22) at most comes out
    // of the product, so no value needs a clamp; NaN quotients are replaced, their low byte could be anything.
    template <int V>
    __device__ __forceinline__ void put(Pack<int8_t, V>& o, const float* u) const {
        uint32_t q[V];
#pragma unroll
        for (int i = 0; i < V; ++i) q[i] = __float_as_uint(__fadd_rn(__fmul_rn(u[i], inv), 12582912.f));
        if (up != 1.f) {   // a tiny row
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = __float_as_uint(__fadd_rn(__fmul_rn(__fmul_rn(u[i], up), inv), 12582912.f));
        }
        if (!(fabsf(inv) < INFINITY)) {   // a NaN or an infinity in the row
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = 0;
        }
        if constexpr (V % 4 == 0) {
            uint32_t* w = reinterpret_cast<uint32_t*>(o.e);
#pragma unroll
            for (int i = 0; i < V; i += 4) w[i / 4] = __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o.e[i] = int8_t(q[i] & 0xffu);
        }
    }
};

// Rows that do not start on 16 bytes, but do so alike in every tensor of the call (contiguous tensors of an odd width):
// element e of a row sits in 16-byte granule (e + lead) / V, lead being what the row's start is past a 16-byte boundary.
// Whole granules move as vectors, the cut first and last one element by element; what they hold besides is 0.
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_granule(const T* row, int e0, int cols) {
    if (e0 >= 0 && e0 + V <= cols) return *reinterpret_cast<const Pack<T, V>*>(row + e0);
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.e[i] = unsigned(e0 + i) < unsigned(cols) ? row[e0 + i] : T(0.f);
    return o;
}
template <class T, int V>
__device__ __forceinline__ void store_granule(T* row, int e0, int cols, const Pack<T, V>& v) {
    if (e0 >= 0 && e0 + V <= cols) {
        *reinterpret_cast<Pack<T, V>*>(row + e0) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (unsigned(e0 + i) < unsigned(cols)) row[e0 + i] = v.e[i];
}
template <class T>
__device__ __forceinline__ int row_lead(const T* row) { return int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }

// G threads (whole warps) hold one row in registers, P vectors of V elements each; a block takes blockDim / G rows at a
// time.  One pass over memory: load, reduce, scale, store.  One row of 8192 bf16 takes 2.1 us in a captured graph, a launch's own
// time; 16384 rows of 4096 with residual took 103 us this way (5.2 TB/s), which is why many rows go through the ring below.
// kCut: rows laid out as above; the weight, whose start is not cut, is then read element by element (from L1).
template <class T, int V, int P, int kOut, bool kCut, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 512 && P * V <= 16 ? 2 : 1) norm_rows_kernel(const RowArgs a, int G) {
    __shared__ float s_sum[2][32], s_top[2][32];
    const int groups = blockDim.x / G, group = threadIdx.x / G, t = threadIdx.x - group * G;
    const int warps = G >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first_warp = group * warps;
    const T* w = static_cast<const T*>(a.w);
    int flip = 0;
    for (long long base = (long long)blockIdx.x * groups; base < a.rows; base += (long long)gridDim.x * groups, flip ^= 1) {
        const long long row = base + group;
        const bool live = row < a.rows;
        const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_rs;
        const T* r = static_cast<const T*>(a.r) + (live && a.r ? row : 0) * a.r_rs;
        const int lead = kCut ? row_lead(x) : 0;
        const int nv = live ? (lead + a.cols + V - 1) / V : 0;
        float f[P * V];
        Pack<T, V> px[P], pr[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G, e0 = c * V - lead;
            if (c < nv) {
                px[p] = kCut ? load_granule<T, V>(x, e0, a.cols) : *reinterpret_cast<const Pack<T, V>*>(x + e0);
                if (a.r) pr[p] = kCut ? load_granule<T, V>(r, e0, a.cols) : *reinterpret_cast<const Pack<T, V>*>(r + e0);
            }
        }
        float sum = 0.f, top = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G, e0 = c * V - lead;
            if (c >= nv) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = px[p].up(i);
                if (a.r) v = __fadd_rn(v, pr[p].up(i));
                f[p * V + i] = v;
                sum = fmaf(v, v, sum);
            }
            if (a.h) {
                Pack<T, V> o;
                o.put(f + p * V);
                T* h = static_cast<T*>(a.h) + row * a.cols;
                if constexpr (kCut) store_granule<T, V>(h, e0, a.cols, o);
                else *reinterpret_cast<Pack<T, V>*>(h + e0) = o;
            }
            if (kOut == kInt8) {
                if (w) {
                    if constexpr (kCut) {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            f[p * V + i] = unsigned(e0 + i) < unsigned(a.cols) ? __fmul_rn(f[p * V + i], RowType<T>::up(w[e0 + i])) : 0.f;
                    } else {
                        const Pack<T, V> pw = *reinterpret_cast<const Pack<T, V>*>(w + e0);
#pragma unroll
                        for (int i = 0; i < V; ++i) f[p * V + i] = __fmul_rn(f[p * V + i], pw.up(i));
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) top = max_nan(top, fabsf(f[p * V + i]));
            }
        }
        sum = warp_sum(sum);
        if (kOut == kInt8) top = warp_max_nan(top);
        if (warps > 1) {
            if (lane == 0) {
                s_sum[flip][warp] = sum;
                if (kOut == kInt8) s_top[flip][warp] = top;
            }
            __syncthreads();   // the two buffers alternate, so one barrier per row is enough
            sum = lane < warps ? s_sum[flip][first_warp + lane] : 0.f;
            sum = warp_sum(sum);
            if (kOut == kInt8) {
                top = lane < warps ? s_top[flip][first_warp + lane] : 0.f;
                top = warp_max_nan(top);
            }
        }
        const float rstd = w ? __frsqrt_rn(sum / float(a.cols) + a.eps) : 1.f;
        const Quant quant(top);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G, e0 = c * V - lead;
            if (c >= nv) continue;
            if (kOut == kInt8) {
                Pack<int8_t, V> o;
                quant.put(o, f + p * V);
                int8_t* q = static_cast<int8_t*>(a.y) + row * a.cols;
                if constexpr (kCut) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (unsigned(e0 + i) < unsigned(a.cols)) q[e0 + i] = o.e[i];
                } else {
                    *reinterpret_cast<Pack<int8_t, V>*>(q + e0) = o;
                }
            } else {
                T* y = static_cast<T*>(a.y) + row * a.cols;
                Pack<T, V> o;
                float v[V];
                if constexpr (kCut) {
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = unsigned(e0 + i) < unsigned(a.cols) ? f[p * V + i] * rstd * RowType<T>::up(w[e0 + i]) : 0.f;
                    o.put(v);
                    store_granule<T, V>(y, e0, a.cols, o);
                } else {
                    const Pack<T, V> pw = *reinterpret_cast<const Pack<T, V>*>(w + e0);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = f[p * V + i] * rstd * pw.up(i);
                    o.put(v);
                    *reinterpret_cast<Pack<T, V>*>(y + e0) = o;
                }
            }
        }
        if (live && t == 0 && a.stat) a.stat[row] = kOut == kInt8 ? __fdiv_rn(__fmul_rn(top, rstd), 127.f) : rstd;
    }
}

template <int kThreads>
__device__ __forceinline__ void block_sum_top(float& sum, float& top) {
    __shared__ float s_sum[kThreads / 32], s_top[kThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    sum = warp_sum(sum);
    top = warp_max_nan(top);
    __syncthreads();
    if (lane == 0) { s_sum[warp] = sum; s_top[warp] = top; }
    __syncthreads();
    sum = warp_sum(lane < kThreads / 32 ? s_sum[lane] : 0.f);
    top = warp_max_nan(lane < kThreads / 32 ? s_top[lane] : 0.f);
}

// Rows too long for a block's registers: the row is read twice (the second time from L2).  Every element is read and
// written by one thread, so h may be x or r here as well.
template <class T, int kOut>
__global__ void __launch_bounds__(1024) norm_long_rows_kernel(const RowArgs a) {
    const T* w = static_cast<const T*>(a.w);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
        const T* r = a.r ? static_cast<const T*>(a.r) + row * a.r_rs : nullptr;
        float sum = 0.f, top = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            float v = RowType<T>::up(x[c]);
            if (r) v = __fadd_rn(v, RowType<T>::up(r[c]));
            if (w) sum += v * v;
            if (kOut == kInt8) top = max_nan(top, fabsf(w ? __fmul_rn(v, RowType<T>::up(w[c])) : v));
        }
        block_sum_top<1024>(sum, top);
        const float rstd = w ? __frsqrt_rn(sum / float(a.cols) + a.eps) : 1.f;
        const Quant quant(top);
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            float v = RowType<T>::up(x[c]);
            if (r) v = __fadd_rn(v, RowType<T>::up(r[c]));
            if (a.h) static_cast<T*>(a.h)[row * a.cols + c] = RowType<T>::down(v);
            if (kOut == kInt8)
            {
                const float u = w ? __fmul_rn(v, RowType<T>::up(w[c])) : v;
                Pack<int8_t, 1> o;
                quant.put(o, &u);
                static_cast<int8_t*>(a.y)[row * a.cols + c] = o.e[0];
            }
            else
                static_cast<T*>(a.y)[row * a.cols + c] = RowType<T>::down(v * rstd * RowType<T>::up(w[c]));
        }
        if (threadIdx.x == 0) {
            if (kOut == kInt8) a.stat[row] = __fdiv_rn(__fmul_rn(top, rstd), 127.f);
            else if (a.stat) a.stat[row] = rstd;
        }
    }
}

// ---- many rows: each group of G threads streams its rows through a ring of shared-memory stages --------------------
// A group takes rows first, first + step, ...; one thread of it keeps `stages` rows on their way with untiled bulk
// copies (one per tensor and row) while the group reduces and writes the row that has landed.  Loads in flight cost no
// registers and no barrier, so the memory system always has the next rows to fetch.  A row is read from its stage into
// registers before the barrier of its reduction; the thread that passes that barrier refills the stage.  Bound by memory:
// 16384 x 4096 bf16 with residual 87 - 93 us (5.8 - 6.2 TB/s of 6.5 copied), 8192 x 8192 89 us; as Int8 rows 84 us.
constexpr int kForwardThreads = 512, kForwardBlocks = 2;   // two blocks per SM, 64 registers per thread
constexpr uint32_t kRingBytes = 200u * 1024u;               // an SM's shared memory for stages
struct RowRing {
    uint32_t data, bars;             // shared-memory addresses of this group's stages and their barriers
    uint32_t row_bytes;
    int tensors, stages;
    __device__ __forceinline__ uint32_t at(int stage, int tensor) const { return data + uint32_t(stage * tensors + tensor) * row_bytes; }
    __device__ __forceinline__ uint32_t bar(int stage) const { return bars + 8u * uint32_t(stage); }
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> ld_shared_pack(uint32_t addr) {
    static_assert(sizeof(Pack<T, V>) == 16, "16-byte vectors");
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return *reinterpret_cast<Pack<T, V>*>(&v);
}

// The G threads of a group meet: a warp by itself, more than one warp on a named barrier of their own.  They agree there on
// whether any of them gave up waiting, so that they leave together: a flag read after the barrier may be set between the reads of two
// warps, and the one that stayed would wait at the next barrier, which has no limit, for threads that are gone.
__device__ __forceinline__ bool group_gave_up(int group, int G, bool mine) {
    if (G == 32) {
        __syncwarp();
        return __any_sync(0xffffffffu, mine);
    }
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any) : "r"(uint32_t(mine)), "r"(group + 1), "r"(G) : "memory");
    return any != 0;
}

struct RingShape { int G, stages; unsigned int* status; };

// Start of a ring kernel: barriers initialised, the group's first rows on their way.
template <class Load>
__device__ __forceinline__ RowRing ring_start(const RingShape& rs, uint32_t smem, uint32_t bars, int group, int t, int tensors, uint32_t row_bytes,
                                              long long row, long long step, long long rows, const Load& load) {
    RowRing ring{smem + uint32_t(group * rs.stages * tensors) * row_bytes, bars + 8u * uint32_t(group * rs.stages), row_bytes, tensors, rs.stages};
    if (t == 0) {
        for (int s = 0; s < rs.stages; ++s) mbar_init(ring.bar(s), 1);
        fence_barrier_init();
        fence_proxy_async_smem();
        for (int s = 0; s < rs.stages && row + s * step < rows; ++s) load(ring, s, row + s * step);
    }
    return ring;
}

// A wait that ran out: the device status word is raised, the flag ends the block's other waits that are still open, each group
// leaves at its next barrier (group_gave_up), and its copying thread waits (bounded again) for the copies still on their way before
// the block ends.
__device__ __forceinline__ void ring_gave_up(unsigned int* status, volatile uint32_t* abort_flag, unsigned int where) {
    *abort_flag = 1;
    atomicExch(status, 0x100u | where);
}
__device__ __forceinline__ void ring_drain(const RowRing& ring, int stage, uint32_t phase, long long row, long long step, long long rows) {
    volatile uint32_t never = 0;
    for (int s = 0; s < ring.stages && row < rows; ++s, row += step) {
        (void)mbar_wait(ring.bar(stage), phase, &never);
        if (++stage == ring.stages) { stage = 0; phase ^= 1u; }
    }
}

template <class T, int P, int kOut, bool kResidual>
__global__ void __launch_bounds__(kForwardThreads, kForwardBlocks) norm_ring_kernel(const RowArgs a, const RingShape rs) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t ring_mem[];
    __shared__ __align__(8) unsigned long long s_bar[128];
    __shared__ float s_sum[2][32], s_top[2][32];
    __shared__ uint32_t s_abort;
    const int G = rs.G, groups = blockDim.x / G, group = threadIdx.x / G, t = threadIdx.x - group * G;
    const int warps = G >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first_warp = group * warps;
    const int nv = a.cols / V;
    const long long step = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + group;
    if (threadIdx.x == 0) s_abort = 0;
    auto load = [&](const RowRing& ring, int s, long long r) {
        mbar_expect_tx(ring.bar(s), ring.row_bytes * uint32_t(ring.tensors));
        bulk_load(ring.at(s, 0), static_cast<const T*>(a.x) + r * a.x_rs, ring.row_bytes, ring.bar(s));
        if (kResidual) bulk_load(ring.at(s, 1), static_cast<const T*>(a.r) + r * a.r_rs, ring.row_bytes, ring.bar(s));
    };
    const RowRing ring = ring_start(rs, smem_u32(ring_mem), smem_u32(s_bar), group, t, kResidual ? 2 : 1, uint32_t(a.cols) * uint32_t(sizeof(T)), row, step,
                                    a.rows, load);
    const Pack<T, V>* w = static_cast<const Pack<T, V>*>(a.w);
    __syncthreads();
    int flip = 0, stage = 0;
    uint32_t phase = 0;
    for (; row < a.rows; row += step, flip ^= 1) {
        const bool landed = mbar_wait(ring.bar(stage), phase, &s_abort);
        if (!landed) ring_gave_up(rs.status, &s_abort, 0x41);
        float f[P * V];
        float sum = 0.f, top = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c < nv) {
                const Pack<T, V> x = ld_shared_pack<T, V>(ring.at(stage, 0) + uint32_t(c) * 16u);
                if (kResidual) {
                    const Pack<T, V> r = ld_shared_pack<T, V>(ring.at(stage, 1) + uint32_t(c) * 16u);
                    Pack<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) f[p * V + i] = __fadd_rn(x.up(i), r.up(i));
                    o.put(f + p * V);
                    reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.h) + row * a.cols)[c] = o;
                } else {
                    if (a.h) reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.h) + row * a.cols)[c] = x;
#pragma unroll
                    for (int i = 0; i < V; ++i) f[p * V + i] = x.up(i);
                }
                if (a.w) {
#pragma unroll
                    for (int i = 0; i < V; ++i) sum += f[p * V + i] * f[p * V + i];
                }
                if (kOut == kInt8) {
                    if (a.w) {
                        const Pack<T, V> pw = w[c];
#pragma unroll
                        for (int i = 0; i < V; ++i) f[p * V + i] = __fmul_rn(f[p * V + i], pw.up(i));
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) top = max_nan(top, fabsf(f[p * V + i]));
                }
            }
        }
        sum = warp_sum(sum);
        if (kOut == kInt8) top = warp_max_nan(top);
        if (warps > 1 && lane == 0) {
            s_sum[flip][warp] = sum;
            if (kOut == kInt8) s_top[flip][warp] = top;
        }
        if (group_gave_up(group, G, !landed)) break;     // else the row is in registers and its partial sums are in place
        if (t == 0 && row + ring.stages * step < a.rows) load(ring, stage, row + ring.stages * step);
        if (++stage == ring.stages) { stage = 0; phase ^= 1u; }
        if (warps > 1) {
            sum = warp_sum(lane < warps ? s_sum[flip][first_warp + lane] : 0.f);
            if (kOut == kInt8) top = warp_max_nan(lane < warps ? s_top[flip][first_warp + lane] : 0.f);
        }
        const float rstd = a.w ? __frsqrt_rn(sum / float(a.cols) + a.eps) : 1.f;
        const Quant quant(top);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c >= nv) continue;
            if (kOut == kInt8) {
                Pack<int8_t, V> o;
                quant.put(o, f + p * V);
                reinterpret_cast<Pack<int8_t, V>*>(static_cast<int8_t*>(a.y) + row * a.cols)[c] = o;
            } else {
                const Pack<T, V> pw = w[c];
                Pack<T, V> o;
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = f[p * V + i] * rstd * pw.up(i);
                o.put(v);
                reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.y) + row * a.cols)[c] = o;
            }
        }
        if (t == 0 && a.stat) a.stat[row] = kOut == kInt8 ? __fdiv_rn(__fmul_rn(top, rstd), 127.f) : rstd;
    }
    if (t == 0 && s_abort) ring_drain(ring, stage, phase, row, step, a.rows);
}

// Self-test of the rings' way out: in every odd group the second half of the threads waits, at turn 3, on a barrier that nothing
// signals, while the first half has nothing to wait for.  The wait runs out, the status word is raised, and all threads of such a
// group leave at that turn; the even groups go on to the last.  left_at[thread]: the turn at which it left.
constexpr int kSelftestTurns = 8, kSelftestStalls = 3;
__global__ void __launch_bounds__(512) ring_timeout_selftest_kernel(int G, unsigned long long limit_ns, unsigned int* status, int* left_at) {
    __shared__ __align__(8) unsigned long long s_bar[16];
    __shared__ uint32_t s_abort;
    const int group = threadIdx.x / G, t = threadIdx.x - group * G;
    if (t == 0) mbar_init(smem_u32(&s_bar[group]), 1);
    if (threadIdx.x == 0) s_abort = 0;
    fence_barrier_init();
    __syncthreads();
    int turn = 0;
    for (; turn < kSelftestTurns; ++turn) {
        const bool waits = (group & 1) && t >= G / 2 && turn == kSelftestStalls;
        const bool landed = !waits || mbar_wait(smem_u32(&s_bar[group]), 0, &s_abort, limit_ns);
        if (!landed) ring_gave_up(status, &s_abort, 0x43);
        if (group_gave_up(group, G, !landed)) break;
    }
    left_at[threadIdx.x] = turn;
}

struct BackArgs {
    const void* h; long long h_rs;
    const void* w; const float* rstd;
    const void* gy; long long gy_rs;
    const void* gh; long long gh_rs;    // null: nothing arrives over the residual stream
    void* gx; float* partial;           // partial: [grid, cols] sums of gy xhat, one row per block; null: no weight gradient
    long long rows; int cols;
};

// The same layout; each thread keeps the sums of gy xhat of its columns in registers over all rows its block takes.
// kCut: a thread's columns are the same for all rows of one lead, so a block takes rows of one lead only: rows first,
// first + step, ... with a step that is a multiple of `period`, the number of rows after which the leads repeat.
// 3406 x 14054 bf16 (rows 12 bytes past a boundary, then 8, ...): forward 136 us, backward 205 us; element by element the two took
// 851 us.  What bounds them: the cut granules' instructions and the weight's single loads, and in the backward pass registers: at
// 1024 threads a thread's two granules, their weights and sums do not fit the 64 it may have (spill stores of <.., 8, 2, true, 1024>
// 220 bytes in BFloat16, 896 in Float16, which the compiler holds to 32 registers; of <.., 8, 4, *, 1024>, rows above 16384, 1108 to
// 1768).
template <class T, int V, int P, bool kCut, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(const BackArgs a, int G, int period) {
    extern __shared__ float s_gw[];      // [groups - 1][cols] while the groups of a block are joined
    __shared__ float s_dot[2][32];
    const int groups = blockDim.x / G, group = threadIdx.x / G, t = threadIdx.x - group * G;
    const int warps = G >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first_warp = group * warps;
    const T* w = static_cast<const T*>(a.w);
    // block b takes the rows of class b mod period: class + period (b / period * groups + group), ...
    const long long first = blockIdx.x % period + (long long)period * ((long long)(blockIdx.x / period) * groups);
    const long long step = (long long)gridDim.x * groups;   // gridDim is a multiple of the period
    const int lead = kCut ? row_lead(static_cast<const T*>(a.h) + min(first, a.rows - 1) * a.h_rs) : 0;
    const int nv = (lead + a.cols + V - 1) / V;
    float gw[P * V];
    Pack<T, V> pw[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = t + p * G, e0 = c * V - lead;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            gw[p * V + i] = 0.f;
            pw[p].e[i] = c < nv && unsigned(e0 + i) < unsigned(a.cols) ? w[e0 + i] : T(0.f);
        }
    }
    int flip = 0;
    for (long long base = first; base < a.rows; base += step, flip ^= 1) {
        const long long row = base + (long long)period * group;
        const bool live = row < a.rows;
        const T* h = static_cast<const T*>(a.h) + (live ? row : 0) * a.h_rs;
        const T* gy = static_cast<const T*>(a.gy) + (live ? row : 0) * a.gy_rs;
        const T* gh = static_cast<const T*>(a.gh) + (live && a.gh ? row : 0) * a.gh_rs;
        const float rstd = live ? a.rstd[row] : 0.f;
        Pack<T, V> ph[P], pg[P], pr[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G, e0 = c * V - lead;
            if (live && c < nv) {
                ph[p] = kCut ? load_granule<T, V>(h, e0, a.cols) : *reinterpret_cast<const Pack<T, V>*>(h + e0);
                pg[p] = kCut ? load_granule<T, V>(gy, e0, a.cols) : *reinterpret_cast<const Pack<T, V>*>(gy + e0);
                if (a.gh) pr[p] = kCut ? load_granule<T, V>(gh, e0, a.cols) : *reinterpret_cast<const Pack<T, V>*>(gh + e0);
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!live || t + p * G >= nv) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float g = pg[p].up(i) * ph[p].up(i);      // the row's rstd joins the sums below
                gw[p * V + i] = fmaf(g, rstd, gw[p * V + i]);
                dot = fmaf(g, pw[p].up(i), dot);
            }
        }
        dot = warp_sum(dot);
        if (warps > 1) {
            if (lane == 0) s_dot[flip][warp] = dot;
            __syncthreads();
            dot = warp_sum(lane < warps ? s_dot[flip][first_warp + lane] : 0.f);
        }
        if (!live) continue;
        const float c0 = rstd * (rstd * dot) / float(a.cols);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G, e0 = c * V - lead;
            if (c >= nv) continue;
            Pack<T, V> o;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = fmaf(-ph[p].up(i), c0, pg[p].up(i) * pw[p].up(i));
                v[i] = a.gh ? fmaf(rstd, d, pr[p].up(i)) : rstd * d;
            }
            o.put(v);
            T* gx = static_cast<T*>(a.gx) + row * a.cols;
            if constexpr (kCut) store_granule<T, V>(gx, e0, a.cols, o);
            else *reinterpret_cast<Pack<T, V>*>(gx + e0) = o;
        }
    }
    if (!a.partial) return;
    // join the block's groups in their order, then one row of partial sums per block
    __syncthreads();
    if (group > 0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int e0 = (t + p * G) * V - lead;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (unsigned(e0 + i) < unsigned(a.cols)) s_gw[(group - 1) * a.cols + e0 + i] = gw[p * V + i];
        }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int e0 = (t + p * G) * V - lead;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (unsigned(e0 + i) >= unsigned(a.cols)) continue;
                float v = gw[p * V + i];
                for (int g = 1; g < groups; ++g) v += s_gw[(g - 1) * a.cols + e0 + i];
                a.partial[(long long)blockIdx.x * a.cols + e0 + i] = v;
            }
        }
    }
}

// The backward pass over the ring: h, gy and gh (kStream) of a row land together.  8192 x 8192 bf16: 101 us, 5.3 TB/s.
template <class T, int P, bool kStream, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_backward_ring_kernel(const BackArgs a, const RingShape rs) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t ring_mem[];
    __shared__ __align__(8) unsigned long long s_bar[128];
    __shared__ float s_dot[2][32];
    __shared__ uint32_t s_abort;
    const int G = rs.G, groups = blockDim.x / G, group = threadIdx.x / G, t = threadIdx.x - group * G;
    const int warps = G >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first_warp = group * warps;
    const int nv = a.cols / V;
    const long long step = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + group;
    if (threadIdx.x == 0) s_abort = 0;
    auto load = [&](const RowRing& ring, int s, long long r) {
        mbar_expect_tx(ring.bar(s), ring.row_bytes * uint32_t(ring.tensors));
        bulk_load(ring.at(s, 0), static_cast<const T*>(a.h) + r * a.h_rs, ring.row_bytes, ring.bar(s));
        bulk_load(ring.at(s, 1), static_cast<const T*>(a.gy) + r * a.gy_rs, ring.row_bytes, ring.bar(s));
        if (kStream) bulk_load(ring.at(s, 2), static_cast<const T*>(a.gh) + r * a.gh_rs, ring.row_bytes, ring.bar(s));
    };
    const RowRing ring = ring_start(rs, smem_u32(ring_mem), smem_u32(s_bar), group, t, kStream ? 3 : 2, uint32_t(a.cols) * uint32_t(sizeof(T)), row, step,
                                    a.rows, load);
    Pack<T, V> w[P];
    float gw[P * V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (t + p * G < nv) w[p] = static_cast<const Pack<T, V>*>(a.w)[t + p * G];
#pragma unroll
        for (int i = 0; i < V; ++i) gw[p * V + i] = 0.f;
    }
    __syncthreads();
    int flip = 0, stage = 0;
    uint32_t phase = 0;
    const float inv_cols = 1.f / float(a.cols);
    for (; row < a.rows; row += step, flip ^= 1) {
        const float rstd = a.rstd[row];
        const bool landed = mbar_wait(ring.bar(stage), phase, &s_abort);
        if (!landed) ring_gave_up(rs.status, &s_abort, 0x42);
        Pack<T, V> h[P], gy[P], gh[P];
        float dot = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c < nv) {
                h[p] = ld_shared_pack<T, V>(ring.at(stage, 0) + uint32_t(c) * 16u);
                gy[p] = ld_shared_pack<T, V>(ring.at(stage, 1) + uint32_t(c) * 16u);
                if (kStream) gh[p] = ld_shared_pack<T, V>(ring.at(stage, 2) + uint32_t(c) * 16u);
#pragma unroll
                for (int i = 0; i < V; ++i) {
    const float hv = h[p].up(i), g = gy[p].up(i) * hv;      // the row's rstd joins the sums below
                    gw[p * V + i] = fmaf(g, rstd, gw[p * V + i]);
                    dot = fmaf(g, w[p].up(i), dot);
                }
            }
        }
        dot = warp_sum(dot);
        if (warps > 1 && lane == 0) s_dot[flip][warp] = dot;
        if (group_gave_up(group, G, !landed)) break;
        if (t == 0 && row + ring.stages * step < a.rows) load(ring, stage, row + ring.stages * step);
        if (++stage == ring.stages) { stage = 0; phase ^= 1u; }
        if (warps > 1) dot = warp_sum(lane < warps ? s_dot[flip][first_warp + lane] : 0.f);
        const float c0 = rstd * (rstd * dot) * inv_cols;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c >= nv) continue;
            Pack<T, V> o;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = fmaf(-h[p].up(i), c0, gy[p].up(i) * w[p].up(i));
                v[i] = kStream ? fmaf(rstd, d, gh[p].up(i)) : rstd * d;
            }
            o.put(v);
            reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.gx) + row * a.cols)[c] = o;
        }
    }
    if (t == 0 && s_abort) ring_drain(ring, stage, phase, row, step, a.rows);
    if (!a.partial) return;
    // the ring is empty: join the block's groups in their order there, then one row of partial sums per block
    __syncthreads();
    float* s_gw = reinterpret_cast<float*>(ring_mem);
    if (group > 0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c < nv)
#pragma unroll
                for (int i = 0; i < V; ++i) s_gw[(group - 1) * a.cols + c * V + i] = gw[p * V + i];
        }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = t + p * G;
            if (c >= nv) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = gw[p * V + i];
                for (int g = 1; g < groups; ++g) v += s_gw[(g - 1) * a.cols + c * V + i];
                a.partial[(long long)blockIdx.x * a.cols + c * V + i] = v;
            }
        }
    }
}

// Rows too long for registers: gx row by row (two passes over the row) ...
template <class T>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const BackArgs a) {
    const T* w = static_cast<const T*>(a.w);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* h = static_cast<const T*>(a.h) + row * a.h_rs;
        const T* gy = static_cast<const T*>(a.gy) + row * a.gy_rs;
        const T* gh = a.gh ? static_cast<const T*>(a.gh) + row * a.gh_rs : nullptr;
        const float rstd = a.rstd[row];
        float dot = 0.f, none = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += 1024)
            dot += RowType<T>::up(gy[c]) * RowType<T>::up(w[c]) * (RowType<T>::up(h[c]) * rstd);
        block_sum_top<1024>(dot, none);
        dot /= float(a.cols);
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            float v = rstd * (RowType<T>::up(gy[c]) * RowType<T>::up(w[c]) - RowType<T>::up(h[c]) * rstd * dot);
            if (gh) v += RowType<T>::up(gh[c]);
            static_cast<T*>(a.gx)[row * a.cols + c] = RowType<T>::down(v);
        }
    }
}
// ... and the weight gradient's partial sums column by column, one slab of rows per blockIdx.y.
template <class T>
__global__ void norm_weight_long_kernel(const BackArgs a, long long slab_rows) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.cols) return;
    const long long r0 = blockIdx.y * slab_rows, r1 = min(a.rows, r0 + slab_rows);
    float v = 0.f;
    for (long long row = r0; row < r1; ++row)
        v += RowType<T>::up(static_cast<const T*>(a.gy)[row * a.gy_rs + c]) *
             (RowType<T>::up(static_cast<const T*>(a.h)[row * a.h_rs + c]) * a.rstd[row]);
    a.partial[(long long)blockIdx.y * a.cols + c] = v;
}

// out[c] = sum over the slabs of partial[s][c], in a fixed order: 16 threads per column take every sixteenth slab.
template <class T>
__global__ void __launch_bounds__(512) sum_partials_kernel(const float* __restrict__ partial, T* __restrict__ out, int slabs, int cols) {
    __shared__ float s[16][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int i = y; i < slabs; i += 16) v += partial[(long long)i * cols + c];
    }
    s[y][x] = v;
    __syncthreads();
    if (y == 0 && c < cols) {
        for (int i = 1; i < 16; ++i) v += s[i][x];
        out[c] = RowType<T>::down(v);
    }
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// How rows meet 16-byte boundaries: every row of every tensor starts on one, or all tensors' rows start alike past one (see
// load_granule; period: the rows after which that repeats), or neither.
enum Layout : int { kAligned, kCutAlike, kScattered };
struct RowLayout {
    Layout kind = kAligned;
    int period = 1;
    long long lead = -1, step = -1;
    void add(const void* p, long long row_bytes) {   // one tensor of the call
        if (!p) return;
        const long long l = reinterpret_cast<uintptr_t>(p) % 16, s = row_bytes % 16;
        if (lead < 0) { lead = l; step = s; }
        else if (l != lead || s != step) kind = kScattered;
    }
    void finish(int es) {
        if (kind == kScattered || lead < 0) return;
        if (lead == 0 && step == 0) return;
        if (lead % es || step % es) { kind = kScattered; return; }
        kind = kCutAlike;
        while (step * period % 16) period *= 2;
    }
};

// How a row is laid over threads: V elements per vector (16 bytes, or one where rows are scattered), P vectors per thread,
// G threads per row, `threads` per block.  Few vectors per thread as long as 512 threads hold the row; a row that needs
// more than 128 threads has a block of its own, of just the warps it needs (4095 BFloat16 on 1024 threads left half of
// them idle: 314 us for 16384 rows), shorter ones share blocks of 256.  g = 0: too long for registers.
struct RowPlan { int v, p, g, threads; };
RowPlan plan_row(int cols, int vec, Layout layout) {
    RowPlan r{layout == kScattered ? 1 : vec, 0, 0, 0};
    const int nv = cols / r.v + (layout == kCutAlike ? 2 : 0);   // two cut granules at most
    const int least = layout == kScattered ? 4 : 1, most = layout == kScattered ? 16 : 4;
    for (int limit : {512, 1024}) {
        const int last = limit == 512 ? most / 2 : most;   // the most vectors per thread only where 1024 threads need them
        for (r.p = limit == 512 ? least : most / 2; r.p <= last; r.p *= 2) {
            const int need = (nv + r.p - 1) / r.p;
            if (need > limit) continue;
            if (need > 128) {
                r.g = r.threads = (need + 31) / 32 * 32;
            } else {
                for (r.g = 32; r.g < need; r.g *= 2) {}
                r.threads = 256;
            }
            return r;
        }
    }
    r.g = 0;
    return r;
}

// The ring's shape for rows of `tensors` x cols elements: p vectors per thread, the smallest power of two of threads per
// row (32 or more) that covers the row, as many stages as `bytes` of shared memory hold, up to 8.  stages < 2: no ring,
// the row is too long.
struct RingPlan { int p, g, threads, stages; uint32_t smem; };
RingPlan plan_ring(int cols, int vec, int es, int tensors, int p, int threads, uint32_t bytes) {
    const int nv = cols / vec;
    RingPlan r{p, 32, threads, 0, 0};
    while (r.g < threads && r.p * r.g < nv) r.g *= 2;
    if (r.p * r.g < nv) return r;
    const uint32_t stage = uint32_t(tensors) * uint32_t(cols) * uint32_t(es), groups = uint32_t(threads / r.g);
    r.stages = int(std::min<uint32_t>(8, bytes / (stage * groups)));
    r.smem = stage * groups * uint32_t(std::max(r.stages, 1));
    return r;
}
RingPlan plan_forward(int cols, int vec, int es, int tensors) {
    const int nv = cols / vec;
    return plan_ring(cols, vec, es, tensors, nv <= 32 ? 1 : (nv <= 2 * kForwardThreads ? 2 : 4), kForwardThreads, kRingBytes / kForwardBlocks);
}
RingPlan plan_backward(int cols, int vec, int es, int tensors) {
    const int nv = cols / vec;
    // groups of more than one warp meet on named barriers, of which a block has 15: at most 8 such groups, or 16 warps
    if (nv <= 64) return plan_ring(cols, vec, es, tensors, 1, 512, kRingBytes);
    if (nv <= 1024) return plan_ring(cols, vec, es, tensors, 2, 512, kRingBytes);
    return plan_ring(cols, vec, es, tensors, 4, 512, kRingBytes);
}

// Kernel attributes are per device and kernel, and only ever raised.
int allow_smem(const void* kernel, uint32_t bytes) {
    if (bytes <= 40 * 1024) return NTB200_OK;   // the 48 KB every kernel may have, less static shared memory
    NTB200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
    return NTB200_OK;
}

template <class T, int P, int kOut, bool kResidual>
int launch_ring(const RowArgs& a, const RingPlan& r, cudaStream_t stream) {
    auto kernel = norm_ring_kernel<T, P, kOut, kResidual>;
    if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), r.smem)) return rc;
    const int groups = r.threads / r.g;
    const int grid = int(std::min<long long>((a.rows + groups - 1) / groups, (long long)sm_count() * kForwardBlocks));
    kernel<<<grid, r.threads, r.smem, stream>>>(a, RingShape{r.g, r.stages, device_status_word()});
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

template <class T, int kOut>
int launch_rows(const RowArgs& a, Layout layout, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    if (layout == kAligned && (a.h || !a.r)) {
        const RingPlan r = plan_forward(a.cols, kVec, int(sizeof(T)), a.r ? 2 : 1);
        // each group has several rows to stream
        if (r.stages >= 2 && a.rows >= 4ll * sm_count() * (r.threads / r.g)) {
            if (a.r) {
                if (r.p == 1) return launch_ring<T, 1, kOut, true>(a, r, stream);
                if (r.p == 2) return launch_ring<T, 2, kOut, true>(a, r, stream);
                return launch_ring<T, 4, kOut, true>(a, r, stream);
            }
            if (r.p == 1) return launch_ring<T, 1, kOut, false>(a, r, stream);
            if (r.p == 2) return launch_ring<T, 2, kOut, false>(a, r, stream);
            return launch_ring<T, 4, kOut, false>(a, r, stream);
        }
    }
    const RowPlan pl = plan_row(a.cols, kVec, layout);
    const int sms = sm_count();
    if (pl.g == 0) {
        const int grid = int(std::min<long long>(a.rows, 2ll * sms));
        norm_long_rows_kernel<T, kOut><<<grid, 1024, 0, stream>>>(a);
    } else {
        const int threads = pl.threads, groups = threads / pl.g;
        const long long want = (a.rows + groups - 1) / groups;
        const int grid = int(std::min<long long>(want, (long long)sms * 16));
#define NTB200_ROWS(VV, PP, CUT, TT) norm_rows_kernel<T, VV, PP, kOut, CUT, TT><<<grid, threads, 0, stream>>>(a, pl.g)
        if (layout == kAligned) {
            if (threads > 512 && pl.p == 2) NTB200_ROWS(kVec, 2, false, 1024);
            else if (threads > 512) NTB200_ROWS(kVec, 4, false, 1024);
            else if (pl.p == 1) NTB200_ROWS(kVec, 1, false, 512);
            else NTB200_ROWS(kVec, 2, false, 512);
        } else if (layout == kCutAlike) {
            if (threads > 512 && pl.p == 2) NTB200_ROWS(kVec, 2, true, 1024);
            else if (threads > 512) NTB200_ROWS(kVec, 4, true, 1024);
            else if (pl.p == 1) NTB200_ROWS(kVec, 1, true, 512);
            else NTB200_ROWS(kVec, 2, true, 512);
        } else {
            if (threads > 512 && pl.p == 8) NTB200_ROWS(1, 8, false, 1024);
            else if (threads > 512) NTB200_ROWS(1, 16, false, 1024);
            else if (pl.p == 4) NTB200_ROWS(1, 4, false, 512);
            else NTB200_ROWS(1, 8, false, 512);
        }
#undef NTB200_ROWS
    }
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

constexpr int64_t kMaxCols = int64_t(1) << 30;

// Slabs of the weight gradient's partial sums, and so the grid of the backward kernel: depends on sizes alone, so that
// the workspace can be sized before the call.
int backward_slabs(int64_t rows) { return int(std::max<int64_t>(1, std::min<int64_t>(rows, 2 * 148))); }

template <class T, int P, bool kStream, int kThreads>
int launch_backward_ring(const BackArgs& a, const RingPlan& r, int grid, cudaStream_t stream) {
    auto kernel = norm_backward_ring_kernel<T, P, kStream, kThreads>;
    const uint32_t smem = std::max(r.smem, uint32_t(r.threads / r.g - 1) * uint32_t(a.cols) * 4u);
    if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    kernel<<<grid, r.threads, smem, stream>>>(a, RingShape{r.g, r.stages, device_status_word()});
    count_launch();
    return NTB200_OK;
}

template <class T>
int launch_backward(const BackArgs& a, void* grad_weight, const RowLayout& layout, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    const RowPlan pl = plan_row(a.cols, kVec, layout.kind);
    int slabs = backward_slabs(a.rows);
    const RingPlan r = layout.kind == kAligned ? plan_backward(a.cols, kVec, int(sizeof(T)), a.gh ? 3 : 2) : RingPlan{};
    if (r.stages >= 2 && a.rows >= 4ll * sm_count() * (r.threads / r.g)) {
        slabs = std::min(slabs, sm_count());
        int rc;
        if (a.gh) rc = r.p == 1 ? launch_backward_ring<T, 1, true, 512>(a, r, slabs, stream)
                     : r.p == 2 ? launch_backward_ring<T, 2, true, 512>(a, r, slabs, stream) : launch_backward_ring<T, 4, true, 512>(a, r, slabs, stream);
        else rc = r.p == 1 ? launch_backward_ring<T, 1, false, 512>(a, r, slabs, stream)
                : r.p == 2 ? launch_backward_ring<T, 2, false, 512>(a, r, slabs, stream) : launch_backward_ring<T, 4, false, 512>(a, r, slabs, stream);
        if (rc) return rc;
    } else if (pl.g == 0) {
        if (a.partial) {   // before gx, which may take the place of gy
            const long long per = (a.rows + slabs - 1) / slabs;
            slabs = int((a.rows + per - 1) / per);
            norm_weight_long_kernel<T><<<dim3(unsigned((a.cols + 255) / 256), unsigned(slabs)), 256, 0, stream>>>(a, per);
            count_launch();
        }
        norm_backward_long_kernel<T><<<int(std::min<long long>(a.rows, 2ll * sm_count())), 1024, 0, stream>>>(a);
        count_launch();
    } else {
        const int threads = pl.threads, groups = threads / pl.g;
        const int period = layout.kind == kCutAlike ? layout.period : 1;
        // two blocks per SM; a whole number of blocks for every class of rows (a class without rows leaves sums of zero)
        slabs = int(std::min<long long>(std::min(slabs, 2 * sm_count()), (a.rows + groups - 1) / groups));
        slabs = (slabs + period - 1) / period * period;
        // at most 7 groups of 512 columns
        const size_t smem = a.partial ? size_t(groups - 1) * a.cols * sizeof(float) : 0;
#define NTB200_BACK(VV, PP, CUT, TT) norm_backward_kernel<T, VV, PP, CUT, TT><<<slabs, threads, smem, stream>>>(a, pl.g, period)
        if (layout.kind == kAligned) {
            if (threads > 512 && pl.p == 2) NTB200_BACK(kVec, 2, false, 1024);
            else if (threads > 512) NTB200_BACK(kVec, 4, false, 1024);
            else if (pl.p == 1) NTB200_BACK(kVec, 1, false, 512);
            else NTB200_BACK(kVec, 2, false, 512);
        } else if (layout.kind == kCutAlike) {
            if (threads > 512 && pl.p == 2) NTB200_BACK(kVec, 2, true, 1024);
            else if (threads > 512) NTB200_BACK(kVec, 4, true, 1024);
            else if (pl.p == 1) NTB200_BACK(kVec, 1, true, 512);
            else NTB200_BACK(kVec, 2, true, 512);
        } else {
            if (threads > 512 && pl.p == 8) NTB200_BACK(1, 8, false, 1024);
            else if (threads > 512) NTB200_BACK(1, 16, false, 1024);
            else if (pl.p == 4) NTB200_BACK(1, 4, false, 512);
            else NTB200_BACK(1, 8, false, 512);
        }
#undef NTB200_BACK
        count_launch();
    }
    NTB200_CUDA(cudaGetLastError());
    if (a.partial) {
        sum_partials_kernel<T><<<unsigned((a.cols + 31) / 32), 512, 0, stream>>>(a.partial, static_cast<T*>(grad_weight), slabs, a.cols);
        count_launch();
        NTB200_CUDA(cudaGetLastError());
    }
    return NTB200_OK;
}

#define NTB200_ROW_SWITCH(dtype, ...)                                                       \
    switch (dtype) {                                                                        \
        case NTB200_F32: { using T = float; return __VA_ARGS__; }                           \
        case NTB200_F16: { using T = __half; return __VA_ARGS__; }                          \
        default: { using T = __nv_bfloat16; return __VA_ARGS__; }                           \
    }

int check_rows(const char* what, int dtype, int64_t rows, int64_t cols) {
    if (dtype != NTB200_F32 && dtype != NTB200_F16 && dtype != NTB200_BF16)
        return fail(NTB200_ERR_UNSUPPORTED, "%s: Float32, Float16 and BFloat16 only, got %s", what, dtype_name(dtype));
    if (rows < 0 || cols <= 0 || cols > kMaxCols) return fail(NTB200_ERR_INVALID_ARG, "%s: bad extent", what);
    return NTB200_OK;
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" {

static int norm_forward(const char* what, int dtype, const void* x, int64_t x_rs, const void* r, int64_t r_rs, const void* w, void* y,
                        bool int8, void* h, float* stat, int64_t rows, int64_t cols, double eps, void* stream) {
    if (int rc = check_rows(what, dtype, rows, cols)) return rc;
    if (rows == 0) return NTB200_OK;
    if (!x || !y || (int8 && !stat)) return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    if (!(eps >= 0)) return fail(NTB200_ERR_INVALID_ARG, "%s: epsilon must not be negative", what);
    if ((rows > 1 && x_rs < cols) || (r && rows > 1 && r_rs < cols))
        return fail(NTB200_ERR_INVALID_ARG, "%s: a row stride is shorter than a row", what);
    if (rows > 1 && h && ((h == x && x_rs != cols) || (h == r && r_rs != cols)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: h in the place of an input must have its row stride (h is contiguous)", what);
    if (y == h || (int8 && (y == x || y == r)) || (rows > 1 && ((y == x && x_rs != cols) || (y == r && r_rs != cols))))
        return fail(NTB200_ERR_INVALID_ARG, "%s: the output in the place of h, or of an input whose rows lie elsewhere", what);
    const int es = int(dtype_size(dtype));
    RowLayout layout;
    layout.add(x, x_rs * es);
    layout.add(r, r_rs * es);
    if (!int8) layout.add(y, cols * es);
    layout.add(h, cols * es);
    layout.finish(es);
    // Int8 rows start where `cols` bytes end: vectors of them need whole vectors of x, and the weight its own boundary
    if (layout.kind == kAligned && ((cols * es) % 16 != 0 || !aligned(w, 16) || (int8 && !aligned(y, size_t(16 / es))))) layout.kind = kScattered;
    const RowArgs a{x, x_rs, r, r_rs, w, y, h, stat, rows, int(cols), float(eps)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (int8) { NTB200_ROW_SWITCH(dtype, (launch_rows<T, kInt8>(a, layout.kind, s))) }
    NTB200_ROW_SWITCH(dtype, (launch_rows<T, kSame>(a, layout.kind, s)))
}

int ntb200_rms_norm(int dtype, const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, const void* weight,
                    void* y, void* h, float* rstd, int64_t rows, int64_t cols, double eps, void* stream) {
    if (rows > 0 && !weight) return fail(NTB200_ERR_INVALID_ARG, "rms_norm: null pointer");
    return norm_forward("rms_norm", dtype, x, x_row_stride, residual, residual_row_stride, weight, y, false, h, rstd, rows, cols, eps, stream);
}

int ntb200_rms_norm_int8(int dtype, const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride,
                         const void* weight, int8_t* q, float* scale, void* h, int64_t rows, int64_t cols, double eps, void* stream) {
    if (rows > 0 && !weight) return fail(NTB200_ERR_INVALID_ARG, "rms_norm_int8: null pointer");
    return norm_forward("rms_norm_int8", dtype, x, x_row_stride, residual, residual_row_stride, weight, q, true, h, scale, rows, cols, eps,
                        stream);
}

int ntb200_quantize_rows(int dtype, const void* x, int64_t x_row_stride, int8_t* q, float* scale, int64_t rows, int64_t cols, void* stream) {
    return norm_forward("quantize_rows", dtype, x, x_row_stride, nullptr, 0, nullptr, q, true, nullptr, scale, rows, cols, 0.0, stream);
}

int ntb200_selftest_ring_timeout(int group_threads, unsigned int limit_ms, int32_t* left_at, void* stream) {
    const bool known = group_threads == 32 || group_threads == 64 || group_threads == 128 || group_threads == 256;
    if (!known || limit_ms == 0 || limit_ms > 1000 || !left_at)
        return fail(NTB200_ERR_INVALID_ARG, "selftest_ring_timeout: groups of 32, 64, 128 or 256 threads, a limit of 1..1000 ms, and 512 results");
    ring_timeout_selftest_kernel<<<1, 512, 0, static_cast<cudaStream_t>(stream)>>>(group_threads, 1000000ull * limit_ms, device_status_word(), left_at);
    count_launch();
    NTB200_CUDA(cudaGetLastError());
    return NTB200_OK;
}

size_t ntb200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return size_t(backward_slabs(rows) + 8) * size_t(cols) * sizeof(float);   // whole classes of up to 8 rows
}

int ntb200_rms_norm_backward(int dtype, const void* h, int64_t h_row_stride, const void* weight, const float* rstd, const void* grad_y,
                             int64_t grad_y_row_stride, const void* grad_h, int64_t grad_h_row_stride, void* grad_x, void* grad_weight,
                             void* workspace, int64_t rows, int64_t cols, void* stream) {
    const char* what = "rms_norm_backward";
    if (int rc = check_rows(what, dtype, rows, cols)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (grad_weight) NTB200_CUDA(cudaMemsetAsync(grad_weight, 0, size_t(cols) * dtype_size(dtype), s));
        return NTB200_OK;
    }
    if (!h || !weight || !rstd || !grad_y || !grad_x || (grad_weight && !workspace))
        return fail(NTB200_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows > 1 && (h_row_stride < cols || grad_y_row_stride < cols || (grad_h && grad_h_row_stride < cols)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: a row stride is shorter than a row", what);
    if (rows > 1 && ((grad_x == h && h_row_stride != cols) || (grad_x == grad_y && grad_y_row_stride != cols) ||
                     (grad_h && grad_x == grad_h && grad_h_row_stride != cols)))
        return fail(NTB200_ERR_INVALID_ARG, "%s: grad_x in the place of an input must have its row stride (grad_x is contiguous)", what);
    const int es = int(dtype_size(dtype));
    RowLayout layout;
    layout.add(h, h_row_stride * es);
    layout.add(grad_y, grad_y_row_stride * es);
    layout.add(grad_h, grad_h_row_stride * es);
    layout.add(grad_x, cols * es);
    layout.finish(es);
    if (layout.kind == kAligned && ((cols * es) % 16 != 0 || !aligned(weight, 16))) layout.kind = kScattered;
    const BackArgs a{h, h_row_stride, weight, rstd, grad_y, grad_y_row_stride, grad_h, grad_h_row_stride, grad_x,
                     grad_weight ? static_cast<float*>(workspace) : nullptr, rows, int(cols)};
    NTB200_ROW_SWITCH(dtype, (launch_backward<T>(a, grad_weight, layout, s)))
}

}  // extern "C"
