// distill_topk.cuh -- distillation from a teacher's K largest logits, forward and backward.
//   p = softmax over the row's K teacher logits / tau (entries whose index names no column take no part)
//   q = softmax over the student's vocab logits / tau;  lse = log sum_j exp(z_j / tau)
//   loss = tau^2 * sum_k p_k * (log p_k - log q_idx(k));   dz_j = gy * tau * (q_j - sum over k with idx(k) = j of p_k)
// A row is cut into one slice per CTA of a cluster (one slice where there are rows enough for the whole GPU); a CTA runs
// over its slice once with a running maximum and sum per thread, the cluster joins the pairs through distributed shared
// memory, and the backward writes the slice and then sets the K columns of the teacher again from the unrounded values.
// Bound by memory: the K columns are a few KB against a row of hundreds.
#pragma once
#include <cooperative_groups.h>

#include "agb_device.cuh"
#include "layernorm_affine.cuh"

namespace agb {

constexpr int kKdThreads = 512;
constexpr int kKdMaxK = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct KdArgs {
    const void* z;
    const void* idx;
    const void* teacher;
    int idx64, teacher_bf16;
    float *loss, *lse;             // written by the forward; lse is read by the backward alone
    const float* gy;
    const void* dz_add;
    void* dz;
    int64_t vocab;
    int k;
    float tau, inv_tau;
    int64_t slice;                 // columns per CTA of the cluster
};

__device__ __forceinline__ float ex2f(float u) {
    float p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(u));
    return p;
}
// (max, sum of exp(. - max)) pairs: join b into a.  An empty pair has max = -inf and sum 0.
__device__ __forceinline__ void join_pair(float& m, float& s, float mb, float sb) {
    const float top = fmaxf(m, mb);
    // equal maxima (two empty sides or two infinities among them) are not rescaled: inf - inf would be NaN
    const float a = m == top ? 1.f : exp2f(__fmul_rn(__fsub_rn(m, top), kLog2e));
    const float b = mb == top ? 1.f : exp2f(__fmul_rn(__fsub_rn(mb, top), kLog2e));
    s = __fmaf_rn(s, a, __fmul_rn(sb, b));
    m = top;
}

// (max, sum) of n values (already divided by tau on the way in), n <= N, per thread
template <int N>
__device__ __forceinline__ void online_add(const float (&f)[N], float inv_tau, float& m, float& s) {
    float c = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) c = fmaxf(c, f[e]);
    c = __fmul_rn(c, inv_tau);
    if (c > m) {
        s = __fmul_rn(s, ex2f(__fmul_rn(__fsub_rn(m, c), kLog2e)));
        m = c;
    }
    const float shift = m == -INFINITY ? 0.f : m;      // nothing but masked columns so far: they add exp(-inf) = 0
#pragma unroll
    for (int e = 0; e < N; ++e) s = __fadd_rn(s, ex2f(__fmul_rn(__fmaf_rn(f[e], inv_tau, -shift), kLog2e)));
}

// MODE 0: loss and lse.  1: loss, lse and dz.  2: dz from a saved lse.
template <typename T, int MODE>
__global__ void __launch_bounds__(kKdThreads) kd_kernel(const KdArgs a) {
    namespace cg = cooperative_groups;
    typedef Unit<T, 16> U;
    constexpr int N = U::N;
    __shared__ float sp[kKdMaxK], sz[kKdMaxK], sadd[kKdMaxK];
    __shared__ int sidx[kKdMaxK];
    __shared__ float red[64];
    __shared__ float pair[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int64_t r = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = kKdThreads / 32;
    const T* z = static_cast<const T*>(a.z) + r * a.vocab;
    const int64_t lo = rank * a.slice < a.vocab ? rank * a.slice : a.vocab;
    const int64_t hi = lo + a.slice < a.vocab ? lo + a.slice : a.vocab;
    const T* add = (MODE > 0 && a.dz_add) ? static_cast<const T*>(a.dz_add) + r * a.vocab : nullptr;

    pdl_wait();
    pdl_trigger();
    // ---- the teacher's row: p_k in shared memory, the same bits in every CTA
    float tmax = -INFINITY;
    for (int k = tid; k < a.k; k += kKdThreads) {
        const int64_t e = r * a.k + k;
        const int64_t j = a.idx64 ? static_cast<const int64_t*>(a.idx)[e] : static_cast<const int32_t*>(a.idx)[e];
        const bool there = j >= 0 && j < a.vocab;
        float t = -INFINITY, zk = 0.f, ak = 0.f;
        if (there) {
            t = a.teacher_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher)[e]) : static_cast<const float*>(a.teacher)[e];
            t = __fmul_rn(t, a.inv_tau);
            zk = __fmul_rn(Vec<T>::load1(z + j), a.inv_tau);
            if (add) ak = Vec<T>::load1(add + j);
        }
        sidx[k] = there ? static_cast<int>(j) : -1;
        sp[k] = t;
        sz[k] = zk;
        sadd[k] = ak;
        tmax = (t > tmax || t != t) ? t : tmax;
    }
    auto block_max = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, v, o);
            v = (w > v || w != w) ? w : v;
        }
        __syncthreads();
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = red[0];
        for (int i = 1; i < NW; ++i) v = (red[i] > v || red[i] != red[i]) ? red[i] : v;
        return v;
    };
    auto block_sum = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
        __syncthreads();
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = red[0];
        for (int i = 1; i < NW; ++i) v = __fadd_rn(v, red[i]);
        return v;
    };
    tmax = block_max(tmax);
    // no entry takes part (none, none that names a column, or none above -inf): the row has no loss and no gradient
    const bool on = !(tmax == -INFINITY);
    T* dz = MODE > 0 ? static_cast<T*>(a.dz) + r * a.vocab : nullptr;
    if (!on) {
        if (MODE < 2 && rank == 0 && tid == 0) {
            a.loss[r] = 0.f;
            a.lse[r] = 0.f;
        }
        if (MODE > 0)
            for (int64_t j = lo + tid; j < hi; j += kKdThreads) Vec<T>::store1(dz + j, add ? Vec<T>::load1(add + j) : 0.f);
        return;                                        // every CTA of the cluster takes this way
    }
    float tsum = 0.f;
    for (int k = tid; k < a.k; k += kKdThreads) tsum = __fadd_rn(tsum, exp2f(__fmul_rn(__fsub_rn(sp[k], tmax), kLog2e)));
    tsum = block_sum(tsum);
    const float tlse = __fadd_rn(tmax, logf(tsum));

    // ---- the student's slice
    // columns up to the first 16-byte boundary, whole vectors, the rest
    const int64_t mis = (16 - (reinterpret_cast<uintptr_t>(z + lo) & 15)) & 15;
    int64_t head = lo + mis / static_cast<int>(sizeof(T));
    if (head > hi) head = hi;
    const int64_t nvec = (hi - head) / N;
    const int64_t tail = head + nvec * N;
    float lse;
    if (MODE < 2) {
        float m = -INFINITY, s = 0.f;
        const uint4* zv = reinterpret_cast<const uint4*>(z + head);
        int64_t i = tid;
        for (; i + 3 * kKdThreads < nvec; i += 4 * kKdThreads) {
            uint4 u[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) u[q] = zv[i + q * kKdThreads];
            float f[4 * N];
#pragma unroll
            for (int q = 0; q < 4; ++q) U::unpack(u[q], f + q * N);
            online_add(f, a.inv_tau, m, s);
        }
        for (; i < nvec; i += kKdThreads) {
            float f[N];
            U::unpack(zv[i], f);
            online_add(f, a.inv_tau, m, s);
        }
        for (int64_t j = lo + tid; j < head; j += kKdThreads) {
            float f[1] = {Vec<T>::load1(z + j)};
            online_add(f, a.inv_tau, m, s);
        }
        for (int64_t j = tail + tid; j < hi; j += kKdThreads) {
            float f[1] = {Vec<T>::load1(z + j)};
            online_add(f, a.inv_tau, m, s);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float mb = __shfl_xor_sync(0xffffffffu, m, o), sb = __shfl_xor_sync(0xffffffffu, s, o);
            join_pair(m, s, mb, sb);
        }
        __syncthreads();
        if (lane == 0) {
            red[warp] = m;
            red[32 + warp] = s;
        }
        __syncthreads();
        m = red[0];
        s = red[32];
        for (int w = 1; w < NW; ++w) join_pair(m, s, red[w], red[32 + w]);
        if (C > 1) {
            if (tid == 0) {
                pair[0] = m;
                pair[1] = s;
            }
            cluster.sync();
            m = *cluster.map_shared_rank(&pair[0], 0);
            s = *cluster.map_shared_rank(&pair[1], 0);
            for (int c = 1; c < C; ++c) join_pair(m, s, *cluster.map_shared_rank(&pair[0], c), *cluster.map_shared_rank(&pair[1], c));
            cluster.sync();                            // nobody leaves while its pair may be read
        }
        lse = __fadd_rn(m, logf(s));
        if (rank == 0) {
            float l = 0.f;
            for (int k = tid; k < a.k; k += kKdThreads) {
                const float lp = __fsub_rn(sp[k], tlse), p = exp2f(__fmul_rn(lp, kLog2e));
                if (!(p == 0.f)) l = __fmaf_rn(p, __fsub_rn(lp, __fsub_rn(sz[k], lse)), l);   // 0 * log 0 = 0
            }
            l = block_sum(l);
            if (tid == 0) {
                a.loss[r] = __fmul_rn(__fmul_rn(a.tau, a.tau), l);
                a.lse[r] = lse;
            }
        }
    } else {
        lse = a.lse[r];
    }

    // ---- the gradient of the slice
    if (MODE > 0) {
        const float g = __fmul_rn(a.gy[r], a.tau);
        auto grad = [&](float zz) { return __fmul_rn(g, ex2f(__fmul_rn(__fmaf_rn(zz, a.inv_tau, -lse), kLog2e))); };
        const bool together = ((reinterpret_cast<uintptr_t>(dz + head) | (add ? reinterpret_cast<uintptr_t>(add + head) : 0)) & 15) == 0;
        if (together) {
            const uint4* zv = reinterpret_cast<const uint4*>(z + head);
            const uint4* av = add ? reinterpret_cast<const uint4*>(add + head) : nullptr;
            uint4* dv = reinterpret_cast<uint4*>(dz + head);
            auto one = [&](uint4 u, uint4 w, int64_t i) {
                float f[N];
                U::unpack(u, f);
                if (av) {
                    float p[N];
                    U::unpack(w, p);
#pragma unroll
                    for (int e = 0; e < N; ++e) f[e] = __fadd_rn(grad(f[e]), p[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) f[e] = grad(f[e]);
                }
                store_vec_streaming(dv + i, U::pack(f));
            };
            int64_t i = tid;
            for (; i + 3 * kKdThreads < nvec; i += 4 * kKdThreads) {
                uint4 u[4], w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) u[q] = zv[i + q * kKdThreads];
                if (av) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) w[q] = av[i + q * kKdThreads];
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) one(u[q], w[q], i + q * kKdThreads);
            }
            for (; i < nvec; i += kKdThreads) one(zv[i], av ? av[i] : make_uint4(0, 0, 0, 0), i);
        }
        const int64_t stop = together ? head : hi;
        for (int64_t j = lo + tid; j < stop; j += kKdThreads) {
            const float v = grad(Vec<T>::load1(z + j));
            Vec<T>::store1(dz + j, add ? __fadd_rn(v, Vec<T>::load1(add + j)) : v);
        }
        if (together)
            for (int64_t j = tail + tid; j < hi; j += kKdThreads) {
                const float v = grad(Vec<T>::load1(z + j));
                Vec<T>::store1(dz + j, add ? __fadd_rn(v, Vec<T>::load1(add + j)) : v);
            }
        __syncthreads();                               // the slice is written: its teacher columns are set again
        for (int k = tid; k < a.k; k += kKdThreads) {
            const int j = sidx[k];
            if (j < lo || j >= hi) continue;
            bool first = true;
            float p = 0.f;
            for (int i = 0; i < a.k; ++i)
                if (sidx[i] == j) {
                    if (i < k) first = false;
                    p = __fadd_rn(p, exp2f(__fmul_rn(__fsub_rn(sp[i], tlse), kLog2e)));
                }
            if (!first) continue;                      // a column named twice is set once, with both shares
            const float q = exp2f(__fmul_rn(__fsub_rn(sz[k], lse), kLog2e));
            const float v = __fmul_rn(g, __fsub_rn(q, p));
            Vec<T>::store1(dz + j, add ? __fadd_rn(v, sadd[k]) : v);
        }
    }
}

}  // namespace agb
