// distill_topk.cuh -- distillation from a teacher's K largest logits, forward and backward.
//   p = softmax over the row's K teacher logits / tau (entries whose index names no column take no part)
//   q = softmax over the student's vocab logits / tau;  lse = log sum_j exp(z_j / tau)
//   loss = tau^2 * sum_k p_k * (log p_k - log q_idx(k));   dz_j = gy * tau * (q_j - sum over k with idx(k) = j of p_k)
// Three shapes of one kernel.  Many long rows: a block per row, or per slice of it (the CTAs of a cluster send each other their sums through
// distributed shared memory), with a running maximum and sum; the backward reads the slice again, from L2, and writes it.  Few rows:
// eight slices in a cluster, short enough to be loaded into registers before anything else is done and to stay there.  Short rows: a
// warp each, no block barrier anywhere.  The K columns of the teacher are set again after the slice is written, from unrounded values.
// Bound by memory: the K columns are a few KB against a row of hundreds.  4096 x 131072 bf16, k = 64: forward 168 us (the copy rate), backward
// 353 us (94 % of it), both in one call 495 us (67 %): there a row's sum and its gradient follow one another, and a block that joins its
// sums or gathers the teacher's columns loads nothing.  Tried and slower: a ring of bulk copies that run ahead into the next row (612 us),
// slices of 32 KB in registers (976 us: the fixed 14000 clocks of a block against 6000 for its slice), L2 eviction hints (no change).
#pragma once
#include <cooperative_groups.h>

#include "agb_device.cuh"
#include "layernorm_affine.cuh"
#include "umma.cuh"

namespace agb {

constexpr int kKdMaxK = 1024;
constexpr int kKdWarpK = 128;          // most entries of a row that a warp takes alone
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
    int64_t rows, vocab;
    int k;
    float tau, inv_tau;
    int64_t slice;                 // columns per CTA of the cluster
    int* status;
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

// The student's sum, as exp2: a thread holds its largest z, the shift sh = max * c (c = log2(e) / tau) and the sum of exp2(z * c - sh),
// one multiply-add and one ex2 per column.  sh is whatever the product rounds to: the sum is relative to it, so that rounding
// costs nothing.  |max * c| beyond 3e38 (a row at its type's lowest value) is clamped; such a row ends with a sum that is zero or not finite
// and is summed again from (z - max) (kd_kernel).
struct KdSum {
    float m, sh;
    float2 s;
};
__device__ __forceinline__ float kd_shift(float m, float c) { return m == -INFINITY ? 0.f : fminf(fmaxf(__fmul_rn(m, c), -3e38f), 3e38f); }

template <typename T>
__device__ __forceinline__ float word_max(const uint4& u);
template <>
__device__ __forceinline__ float word_max<float>(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
template <>
__device__ __forceinline__ float word_max<__nv_bfloat16>(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ void kd_raise(KdSum& k, float top, float c) {
    if (top > k.m) {
        const float sh = kd_shift(top, c);
        // an empty sum stays empty, whatever the two shifts are
        const float f = k.m == -INFINITY ? 0.f : ex2f(__fsub_rn(k.sh, sh));
        k.s = mul2(k.s, pk(f));
        k.m = top;
        k.sh = sh;
    }
}
template <typename T, int W>
__device__ __forceinline__ void kd_add(KdSum& k, const uint4 (&u)[W], float c) {
    typedef Unit<T, 16> U;
    float top = word_max<T>(u[0]);
#pragma unroll
    for (int q = 1; q < W; ++q) top = fmaxf(top, word_max<T>(u[q]));
    kd_raise(k, top, c);
#pragma unroll
    for (int q = 0; q < W; ++q) {
        float f[U::N];
        U::unpack(u[q], f);
#pragma unroll
        for (int e = 0; e < U::N; e += 2) {
            const float2 x = fma2p(make_float2(f[e], f[e + 1]), pk(c), pk(-k.sh));
            k.s = add2(k.s, make_float2(ex2f(x.x), ex2f(x.y)));
        }
    }
}
__device__ __forceinline__ void kd_add1(KdSum& k, float z, float c) {
    kd_raise(k, z, c);
    k.s.x = __fadd_rn(k.s.x, ex2f(__fmaf_rn(z, c, -k.sh)));
}
// Joins another thread's sum.
__device__ __forceinline__ void kd_join(float& m, float& sh, float& s, float mb, float shb, float sb) {
    const float top = fmaxf(sh, shb);
    // a side without columns has sum 0 and a shift of 0 that must not count
    const bool ea = m == -INFINITY && s == 0.f, eb = mb == -INFINITY && sb == 0.f;
    const float to = ea ? shb : eb ? sh : top;
    s = __fadd_rn(ea ? 0.f : __fmul_rn(s, ex2f(__fsub_rn(sh, to))), eb ? 0.f : __fmul_rn(sb, ex2f(__fsub_rn(shb, to))));
    sh = to;
    m = fmaxf(m, mb);
}

// Another CTA's shared memory.
__device__ __forceinline__ uint32_t peer_address(const void* p, int rank) {
    uint32_t out;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_u32(p)), "r"(rank));
    return out;
}
__device__ __forceinline__ void store_peer(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_peer(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// MODE 0: loss and lse.  1: loss, lse and dz.  2: dz from a saved lse.  NT threads work on a row's slice together: a block, or a warp of
// a block of eight.  KEEP: the slice stays in registers.
template <typename T, int MODE, int NT, int KEEP>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT) kd_kernel(const KdArgs a) {
    namespace cg = cooperative_groups;
    typedef Unit<T, 16> U;
    constexpr int N = U::N, ROWS = NT == 32 ? 8 : 1, K = NT == 32 ? kKdWarpK : kKdMaxK, NW = NT / 32;
    __shared__ float sp_all[ROWS * K], sprob_all[ROWS * K], sz_all[ROWS * K], sadd_all[MODE > 0 ? ROWS * K : 1], sraw_all[MODE > 0 ? ROWS * K : 1];
    __shared__ int sidx_all[MODE > 0 ? ROWS * K : 1];
    __shared__ float red[96];
    __shared__ float pairs[8][3];
    __shared__ __align__(8) uint64_t pair_bar;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = NT == 32 ? lane : threadIdx.x;
    const int which = NT == 32 ? warp : 0;
    float* sp = sp_all + which * K;
    float* sprob = sprob_all + which * K;
    float* sz = sz_all + which * K;
    [[maybe_unused]] float* sadd = sadd_all + (MODE > 0 ? which * K : 0);
    [[maybe_unused]] float* sraw = sraw_all + (MODE > 0 ? which * K : 0);
    [[maybe_unused]] int* sidx = sidx_all + (MODE > 0 ? which * K : 0);
    const int C = NT == 32 ? 1 : static_cast<int>(cg::this_cluster().num_blocks());
    const int rank = NT == 32 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
    const int64_t r = NT == 32 ? static_cast<int64_t>(blockIdx.x) * ROWS + warp : blockIdx.x / C;
    if (NT == 32 && r >= a.rows) return;               // warps do not wait for one another
    const T* z = static_cast<const T*>(a.z) + r * a.vocab;
    const int64_t lo = rank * a.slice < a.vocab ? rank * a.slice : a.vocab;
    const int64_t hi = lo + a.slice < a.vocab ? lo + a.slice : a.vocab;
    const T* add = (MODE > 0 && a.dz_add) ? static_cast<const T*>(a.dz_add) + r * a.vocab : nullptr;
    auto sync = [] {
        if constexpr (NT == 32) __syncwarp();
        else __syncthreads();
    };

    if constexpr (NT > 32 && MODE < 2) {
        if (C > 1) {                                   // the barrier is ready long before a peer's sums arrive
            if (tid == 0) {
                mbar_init(&pair_bar, C);
                mbar_fence_init();
            }
            asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        }
    }
    pdl_wait();
    pdl_trigger();
    [[maybe_unused]] const float gy = MODE > 0 ? a.gy[r] : 0.f;
    // ---- the student's slice: columns up to the first 16-byte boundary, whole vectors, the rest
    const int64_t mis = (16 - (reinterpret_cast<uintptr_t>(z + lo) & 15)) & 15;
    int64_t head = lo + mis / static_cast<int>(sizeof(T));
    if (head > hi) head = hi;
    const int64_t nvec = (hi - head) / N;
    const int64_t tail = head + nvec * N;
    [[maybe_unused]] uint4 kz[KEEP ? KEEP : 1];
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int q = 0; q < KEEP; ++q)
            if (tid + q * NT < nvec) kz[q] = zv[tid + q * NT];
    }
    // ---- the teacher's row: p_k in shared memory, the same bits in every CTA
    float tmax = -INFINITY, tsum = 0.f;                // of the thread's entries, then of all
    for (int k = tid; k < a.k; k += NT) {
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
        sp[k] = t;
        sz[k] = zk;
        if constexpr (MODE > 0) {
            sraw[k] = there ? Vec<T>::load1(z + j) : 0.f;
            sidx[k] = there ? static_cast<int>(j) : -1;
            sadd[k] = ak;
        }
        join_pair(tmax, tsum, t, t == -INFINITY ? 0.f : 1.f);
    }
    auto block_sum = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
        if constexpr (NT > 32) {
            __syncthreads();
            if (lane == 0) red[warp] = v;
            __syncthreads();
            v = lane < NW ? red[lane] : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
        }
        return v;
    };
    auto join_teacher = [&] {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float mb = __shfl_xor_sync(0xffffffffu, tmax, o), sb = __shfl_xor_sync(0xffffffffu, tsum, o);
            join_pair(tmax, tsum, mb, sb);
        }
    };
    join_teacher();
    if constexpr (NT > 32) {
        if (lane == 0) {
            red[warp] = tmax;
            red[32 + warp] = tsum;
        }
        __syncthreads();
        tmax = lane < NW ? red[lane] : -INFINITY;
        tsum = lane < NW ? red[32 + lane] : 0.f;
        join_teacher();
    } else {
        __syncwarp();                                  // the entries are in shared memory
    }
    // no entry takes part (none, none that names a column, or none above -inf; a NaN counts): the row has no loss and no gradient
    const bool on = !(tsum == 0.f);
    T* dz = MODE > 0 ? static_cast<T*>(a.dz) + r * a.vocab : nullptr;
    if (!on) {
        if (MODE < 2 && rank == 0 && tid == 0) {
            a.loss[r] = 0.f;
            a.lse[r] = 0.f;
        }
        if (MODE > 0)
            for (int64_t j = lo + tid; j < hi; j += NT) Vec<T>::store1(dz + j, add ? Vec<T>::load1(add + j) : 0.f);
        if constexpr (NT > 32 && MODE < 2) {
            if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        }
        return;                                        // every CTA of the cluster takes this way
    }
    const float tlse = __fadd_rn(tmax, logf(tsum));
    for (int k = tid; k < a.k; k += NT) sprob[k] = exp2f(__fmul_rn(__fsub_rn(sp[k], tlse), kLog2e));

    const float c = __fmul_rn(a.inv_tau, kLog2e);
    // the gradient's form: q_j = exp2(z_j * c - sh) * scale, or with `slow` exp2((z_j - zm) * c) * scale
    float lse, sh, scale, zm = 0.f;
    bool slow;
    if (MODE < 2) {
        KdSum k{-INFINITY, 0.f, make_float2(0.f, 0.f)};
        if constexpr (KEEP > 0) {
#pragma unroll
            for (int q = 0; q < KEEP; q += 2) {
                if (tid + (q + 1) * NT < nvec) {
                    const uint4 u[2] = {kz[q], kz[q + 1]};
                    kd_add<T>(k, u, c);
                } else if (tid + q * NT < nvec) {
                    const uint4 u[1] = {kz[q]};
                    kd_add<T>(k, u, c);
                }
            }
        } else {
            int64_t i = tid;
            for (; i + 3 * NT < nvec; i += 4 * NT) {
                uint4 u[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) u[q] = zv[i + q * NT];
                kd_add<T>(k, u, c);
            }
            for (; i < nvec; i += NT) {
                const uint4 u[1] = {zv[i]};
                kd_add<T>(k, u, c);
            }
        }
        for (int64_t j = lo + tid; j < head; j += NT) kd_add1(k, Vec<T>::load1(z + j), c);
        for (int64_t j = tail + tid; j < hi; j += NT) kd_add1(k, Vec<T>::load1(z + j), c);
        float m = k.m, s = __fadd_rn(k.s.x, k.s.y);
        sh = k.sh;
        auto join_warp = [&] {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float mb = __shfl_xor_sync(0xffffffffu, m, o), hb = __shfl_xor_sync(0xffffffffu, sh, o),
                            sb = __shfl_xor_sync(0xffffffffu, s, o);
                kd_join(m, sh, s, mb, hb, sb);
            }
        };
        if constexpr (NT > 32) {
            if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        }
        // over the row's threads, then over the slices: the same bits everywhere
        uint32_t turn = 0;
        auto join_all = [&] {
            join_warp();
            if constexpr (NT > 32) {
                __syncthreads();
                if (lane == 0) {
                    red[warp] = m;
                    red[32 + warp] = sh;
                    red[64 + warp] = s;
                }
                __syncthreads();
                m = lane < NW ? red[lane] : -INFINITY;
                sh = lane < NW ? red[32 + lane] : 0.f;
                s = lane < NW ? red[64 + lane] : 0.f;
                join_warp();
                if (C > 1) {
                    // each CTA sends its sum to all (itself among them) and waits for theirs: nobody reads another's memory
                    if (tid < C) {
                        const uint32_t to = peer_address(&pairs[rank][0], tid);
                        store_peer(to, m);
                        store_peer(to + 4, sh);
                        store_peer(to + 8, s);
                        mbar_arrive_peer(peer_address(&pair_bar, tid));
                    }
                    bool here = false;
                    for (int i = 0; i < kTcPollLimit && !here; ++i) here = mbar_poll(&pair_bar, turn);
                    if (!here) atomicExch(a.status, 6 /* AGB_ERR_TIMEOUT */);
                    asm volatile("fence.acq_rel.cluster;" ::: "memory");
                    turn ^= 1;
                    m = pairs[0][0];
                    sh = pairs[0][1];
                    s = pairs[0][2];
                    for (int q = 1; q < C; ++q) kd_join(m, sh, s, pairs[q][0], pairs[q][1], pairs[q][2]);
                }
            }
        };
        join_all();
        slow = !(s > 0.f && s < INFINITY) && m != -INFINITY;
        if (slow) {                                    // see KdSum; NaN and infinities come out as in the formula
            zm = m;
            if constexpr (NT > 32) {
                if (C > 1) cg::this_cluster().sync();  // everyone has read the first round
            }
            float t = 0.f;
            for (int64_t j = lo + tid; j < hi; j += NT) t = __fadd_rn(t, ex2f(__fmul_rn(__fsub_rn(Vec<T>::load1(z + j), zm), c)));
            m = 0.f;
            sh = 0.f;
            s = t;
            join_all();
            lse = __fmaf_rn(zm, a.inv_tau, logf(s));
        } else {
            lse = __fmul_rn(kLn2, __fadd_rn(sh, log2f(s)));
        }
        scale = __fdiv_rn(1.f, s);
        if (rank == 0) {
            float l = 0.f;
            for (int k = tid; k < a.k; k += NT) {
                const float lp = __fsub_rn(sp[k], tlse), p = sprob[k];
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
        sh = __fmul_rn(lse, kLog2e);
        slow = !(fabsf(sh) < 3e38f);
        scale = exp2f(-__fmaf_rn(lse, kLog2e, -sh));   // what the product's rounding left
    }

    // ---- the gradient of the slice
    if (MODE > 0) {
        const float g = __fmul_rn(gy, a.tau), gs = __fmul_rn(g, scale);
        auto grad = [&](float zz) {
            if (!slow) return __fmul_rn(gs, ex2f(__fmaf_rn(zz, c, -sh)));
            if (MODE == 2) return __fmul_rn(g, ex2f(__fmul_rn(__fmaf_rn(zz, a.inv_tau, -lse), kLog2e)));
            return __fmul_rn(gs, ex2f(__fmul_rn(__fsub_rn(zz, zm), c)));
        };
        const bool together = !slow && ((reinterpret_cast<uintptr_t>(dz + head) | (add ? reinterpret_cast<uintptr_t>(add + head) : 0)) & 15) == 0;
        if (together) {
            const uint4* av = add ? reinterpret_cast<const uint4*>(add + head) : nullptr;
            uint4* dv = reinterpret_cast<uint4*>(dz + head);
            auto one = [&](const uint4& u, int64_t i) {
                float f[N];
                U::unpack(u, f);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float2 x = fma2p(make_float2(f[e], f[e + 1]), pk(c), pk(-sh));
                    const float2 d = mul2(pk(gs), make_float2(ex2f(x.x), ex2f(x.y)));
                    f[e] = d.x;
                    f[e + 1] = d.y;
                }
                if (av) {
                    float p[N];
                    U::unpack(av[i], p);
#pragma unroll
                    for (int e = 0; e < N; ++e) f[e] = __fadd_rn(f[e], p[e]);
                }
                store_vec_streaming(dv + i, U::pack(f));
            };
            if constexpr (KEEP > 0) {
#pragma unroll
                for (int q = 0; q < KEEP; ++q)
                    if (tid + q * NT < nvec) one(kz[q], tid + q * NT);
            } else {
                int64_t i = tid;
                for (; i + 3 * NT < nvec; i += 4 * NT) {
                    uint4 u[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) u[q] = zv[i + q * NT];
#pragma unroll
                    for (int q = 0; q < 4; ++q) one(u[q], i + q * NT);
                }
                for (; i < nvec; i += NT) one(zv[i], i);
            }
        }
        const int64_t stop = together ? head : hi;
        for (int64_t j = lo + tid; j < stop; j += NT) {
            const float v = grad(Vec<T>::load1(z + j));
            Vec<T>::store1(dz + j, add ? __fadd_rn(v, Vec<T>::load1(add + j)) : v);
        }
        if (together)
            for (int64_t j = tail + tid; j < hi; j += NT) {
                const float v = grad(Vec<T>::load1(z + j));
                Vec<T>::store1(dz + j, add ? __fadd_rn(v, Vec<T>::load1(add + j)) : v);
            }
        sync();                                        // the slice is written: its teacher columns are set again
        // a column named twice is set once, with all its shares, by its first entry
        auto set = [&](int k, float p) {
            const float v = __fsub_rn(grad(sraw[k]), __fmul_rn(g, p));
            Vec<T>::store1(dz + sidx[k], add ? __fadd_rn(v, sadd[k]) : v);
        };
        if constexpr (NT == 32) {
            for (int k = lane; k < a.k; k += 32) {
                const int j = sidx[k];
                if (j < lo || j >= hi) continue;
                bool first = true;
                float p = 0.f;
                for (int i = 0; i < a.k; ++i)
                    if (sidx[i] == j) {
                        first = first && i >= k;
                        p = __fadd_rn(p, sprob[i]);
                    }
                if (first) set(k, p);
            }
        } else {
            // a warp per entry: its lanes look for the column among the others (one thread per entry took 4100 clocks at k = 64)
            for (int k = warp; k < a.k; k += NW) {
                const int j = sidx[k];
                if (j < lo || j >= hi) continue;
                bool first = true;
                float p = 0.f;
                for (int i0 = 0; i0 < a.k; i0 += 32) {
                    const int i = i0 + lane;
                    const bool same = i < a.k && sidx[i] == j;
                    if (same) p = __fadd_rn(p, sprob[i]);
                    if (__any_sync(0xffffffffu, same && i < k)) first = false;
                }
                if (!first) continue;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) p = __fadd_rn(p, __shfl_xor_sync(0xffffffffu, p, o));
                if (lane == 0) set(k, p);
            }
        }
    }
}

}  // namespace agb
