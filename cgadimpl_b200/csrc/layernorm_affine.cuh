// layernorm_affine.cuh -- LayerNorm with weight and bias, forward and VJP.
//   mean = sum_j x / H;  rstd = 1 / sqrt(sum_j (x - mean)^2 / H + eps);  xh = (x - mean) * rstd;  y = xh * gamma + beta
//   v = gy * gamma;  dx = rstd * (v - sum_j v / H - xh * (sum_j v * xh) / H)
//   dgamma[j] = sum_r gy * xh;  dbeta[j] = sum_r gy
// Every sum is carried in fp32, column sums over the CTAs in fp64; outputs are rounded once.  The variance is taken from
// the centred values (a second pass over registers), so an offset of the row costs no digits.
// No contraction of a size that matters: bound by memory.
#pragma once
#include "agb_device.cuh"

namespace agb {

// UB bytes of T at once: 16 where rows and pointers allow it, else the widest of 4 and 2 that divides a row.
template <typename T, int UB>
struct Unit;
template <>
struct Unit<float, 16> {
    typedef uint4 raw;
    static constexpr int N = 4;
    __device__ __forceinline__ static void unpack(const raw& u, float* f) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    __device__ __forceinline__ static raw pack(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <>
struct Unit<float, 4> {
    typedef uint32_t raw;
    static constexpr int N = 1;
    __device__ __forceinline__ static void unpack(const raw& u, float* f) { f[0] = __uint_as_float(u); }
    __device__ __forceinline__ static raw pack(const float* f) { return __float_as_uint(f[0]); }
};
__device__ __forceinline__ void unpack_bf16x2(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
}
template <>
struct Unit<__nv_bfloat16, 16> {
    typedef uint4 raw;
    static constexpr int N = 8;
    __device__ __forceinline__ static void unpack(const raw& u, float* f) {
        unpack_bf16x2(u.x, f); unpack_bf16x2(u.y, f + 2); unpack_bf16x2(u.z, f + 4); unpack_bf16x2(u.w, f + 6);
    }
    __device__ __forceinline__ static raw pack(const float* f) {
        return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
};
template <>
struct Unit<__nv_bfloat16, 4> {
    typedef uint32_t raw;
    static constexpr int N = 2;
    __device__ __forceinline__ static void unpack(const raw& u, float* f) { unpack_bf16x2(u, f); }
    __device__ __forceinline__ static raw pack(const float* f) { return pack_bf16x2(f[0], f[1]); }
};
template <>
struct Unit<__nv_bfloat16, 2> {
    typedef uint16_t raw;
    static constexpr int N = 1;
    __device__ __forceinline__ static void unpack(const raw& u, float* f) { f[0] = __uint_as_float(static_cast<uint32_t>(u) << 16); }
    __device__ __forceinline__ static raw pack(const float* f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f[0])); }
};

// Sum over the G threads of a row, the same bits in each of them.  G is a power of two up to 32 (parts of a warp; several rows
// to a warp) or the whole block.  `scratch`: one float per warp, reused after the second barrier.
__device__ __forceinline__ float row_sum(float v, int G, float* scratch) {
    for (int o = (G < 32 ? G : 32) >> 1; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (G <= 32) return v;
    const int nw = blockDim.x >> 5;
    __syncthreads();                                   // the previous sum has been read
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < nw ? scratch[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

struct LnaFwdArgs {
    const void *x, *gamma, *beta;
    void* y;
    float *mean, *rstd;
    int64_t rows;
    int hidden, G;
    float eps;
};

// One row per G threads, UPT units per thread held in registers between the two passes.
template <typename T, int UB, int UPT>
__global__ void __launch_bounds__(512) lna_fwd_kernel(const LnaFwdArgs a) {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    __shared__ float scratch[32];
    const int G = a.G, t = threadIdx.x & (G <= 32 ? G - 1 : 1023);
    const int per_block = blockDim.x / G, nunits = a.hidden / U::N;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(a.hidden));
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per_block;
    const int64_t groups = (a.rows + per_block - 1) / per_block * per_block;   // whole warps take every turn (shuffles)
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * per_block + (G <= 32 ? threadIdx.x / G : 0); r < groups; r += stride) {
        const bool live = r < a.rows;
        const raw* x = reinterpret_cast<const raw*>(static_cast<const T*>(a.x) + r * a.hidden);
        float f[UPT][U::N];
        float s = 0.f;
        raw u[UPT];
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (live && t + i * G < nunits) u[i] = x[t + i * G];
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (live && t + i * G < nunits) {
                U::unpack(u[i], f[i]);
#pragma unroll
                for (int e = 0; e < U::N; ++e) s = __fadd_rn(s, f[i][e]);
            }
        const float mean = __fmul_rn(row_sum(s, G, scratch), inv_h);
        s = 0.f;
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (live && t + i * G < nunits) {
#pragma unroll
                for (int e = 0; e < U::N; ++e) {
                    f[i][e] = __fsub_rn(f[i][e], mean);
                    s = __fmaf_rn(f[i][e], f[i][e], s);
                }
            }
        const float rstd = __fdiv_rn(1.f, __fsqrt_rn(__fmaf_rn(row_sum(s, G, scratch), inv_h, a.eps)));
        if (!live) continue;
        if (t == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        raw* y = reinterpret_cast<raw*>(static_cast<T*>(a.y) + r * a.hidden);
        const raw* gamma = reinterpret_cast<const raw*>(a.gamma);
        const raw* beta = reinterpret_cast<const raw*>(a.beta);
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (t + i * G < nunits) {
                float g[U::N], b[U::N];
                U::unpack(gamma[t + i * G], g);
                if (beta) U::unpack(beta[t + i * G], b);
#pragma unroll
                for (int e = 0; e < U::N; ++e) {
                    const float h = __fmul_rn(f[i][e], rstd);
                    f[i][e] = beta ? __fmaf_rn(h, g[e], b[e]) : __fmul_rn(h, g[e]);
                }
                y[t + i * G] = U::pack(f[i]);
            }
    }
}

// Rows that do not fit the registers of a block: three passes over global memory.
template <typename T, int UB>
__global__ void __launch_bounds__(1024) lna_fwd_wide(const LnaFwdArgs a) {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    __shared__ float scratch[32];
    const int nunits = a.hidden / U::N, G = blockDim.x;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(a.hidden));
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const raw* x = reinterpret_cast<const raw*>(static_cast<const T*>(a.x) + r * a.hidden);
        raw* y = reinterpret_cast<raw*>(static_cast<T*>(a.y) + r * a.hidden);
        float f[U::N], g[U::N], b[U::N];
        float s = 0.f;
        for (int i = threadIdx.x; i < nunits; i += G) {
            U::unpack(x[i], f);
#pragma unroll
            for (int e = 0; e < U::N; ++e) s = __fadd_rn(s, f[e]);
        }
        const float mean = __fmul_rn(row_sum(s, G, scratch), inv_h);
        s = 0.f;
        for (int i = threadIdx.x; i < nunits; i += G) {
            U::unpack(x[i], f);
#pragma unroll
            for (int e = 0; e < U::N; ++e) {
                const float c = __fsub_rn(f[e], mean);
                s = __fmaf_rn(c, c, s);
            }
        }
        const float rstd = __fdiv_rn(1.f, __fsqrt_rn(__fmaf_rn(row_sum(s, G, scratch), inv_h, a.eps)));
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int i = threadIdx.x; i < nunits; i += G) {
            U::unpack(x[i], f);
            U::unpack(reinterpret_cast<const raw*>(a.gamma)[i], g);
            if (a.beta) U::unpack(reinterpret_cast<const raw*>(a.beta)[i], b);
#pragma unroll
            for (int e = 0; e < U::N; ++e) {
                const float h = __fmul_rn(__fsub_rn(f[e], mean), rstd);
                f[e] = a.beta ? __fmaf_rn(h, g[e], b[e]) : __fmul_rn(h, g[e]);
            }
            y[i] = U::pack(f);
        }
    }
}

struct LnaBwdArgs {
    const void *x, *gamma;
    const float *mean, *rstd;
    const void *gy, *dx_add;
    void* dx;
    int64_t rows;
    int hidden, G;
};

// dx alone, one row per G threads, UPT units per thread.
template <typename T, int UB, int UPT>
__global__ void __launch_bounds__(512) lna_dx_kernel(const LnaBwdArgs a) {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    __shared__ float scratch[32];
    const int G = a.G, t = threadIdx.x & (G <= 32 ? G - 1 : 1023);
    const int per_block = blockDim.x / G, nunits = a.hidden / U::N;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(a.hidden));
    const int64_t stride = static_cast<int64_t>(gridDim.x) * per_block;
    const int64_t groups = (a.rows + per_block - 1) / per_block * per_block;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * per_block + (G <= 32 ? threadIdx.x / G : 0); r < groups; r += stride) {
        const bool live = r < a.rows;
        const raw* x = reinterpret_cast<const raw*>(static_cast<const T*>(a.x) + r * a.hidden);
        const raw* gy = reinterpret_cast<const raw*>(static_cast<const T*>(a.gy) + r * a.hidden);
        const raw* add = a.dx_add ? reinterpret_cast<const raw*>(static_cast<const T*>(a.dx_add) + r * a.hidden) : nullptr;
        const raw* gamma = reinterpret_cast<const raw*>(a.gamma);
        raw ux[UPT], ug[UPT];
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (live && t + i * G < nunits) {
                ux[i] = x[t + i * G];
                ug[i] = gy[t + i * G];
            }
        const float mean = live ? a.mean[r] : 0.f, rstd = live ? a.rstd[r] : 0.f;
        float sv = 0.f, svh = 0.f;
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (live && t + i * G < nunits) {
                float f[U::N], g[U::N], w[U::N];
                U::unpack(ux[i], f);
                U::unpack(ug[i], g);
                U::unpack(gamma[t + i * G], w);
#pragma unroll
                for (int e = 0; e < U::N; ++e) {
                    const float v = __fmul_rn(g[e], w[e]);
                    sv = __fadd_rn(sv, v);
                    svh = __fmaf_rn(v, __fmul_rn(__fsub_rn(f[e], mean), rstd), svh);
                }
            }
        const float c1 = __fmul_rn(row_sum(sv, G, scratch), inv_h);
        const float c2 = __fmul_rn(row_sum(svh, G, scratch), inv_h);
        if (!live) continue;
        raw* dx = reinterpret_cast<raw*>(static_cast<T*>(a.dx) + r * a.hidden);
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (t + i * G < nunits) {
                float f[U::N], g[U::N], w[U::N], p[U::N];
                U::unpack(ux[i], f);
                U::unpack(ug[i], g);
                U::unpack(gamma[t + i * G], w);
                if (add) U::unpack(add[t + i * G], p);
#pragma unroll
                for (int e = 0; e < U::N; ++e) {
                    const float h = __fmul_rn(__fsub_rn(f[e], mean), rstd);
                    const float q = __fmaf_rn(-h, c2, __fsub_rn(__fmul_rn(g[e], w[e]), c1));
                    f[e] = add ? __fmaf_rn(rstd, q, p[e]) : __fmul_rn(rstd, q);
                }
                dx[t + i * G] = U::pack(f);
            }
    }
}

// dx alone for rows that do not fit the registers of a block.
template <typename T, int UB>
__global__ void __launch_bounds__(1024) lna_dx_wide(const LnaBwdArgs a) {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    __shared__ float scratch[32];
    const int nunits = a.hidden / U::N, G = blockDim.x;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(a.hidden));
    const raw* gamma = reinterpret_cast<const raw*>(a.gamma);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const raw* x = reinterpret_cast<const raw*>(static_cast<const T*>(a.x) + r * a.hidden);
        const raw* gy = reinterpret_cast<const raw*>(static_cast<const T*>(a.gy) + r * a.hidden);
        const raw* add = a.dx_add ? reinterpret_cast<const raw*>(static_cast<const T*>(a.dx_add) + r * a.hidden) : nullptr;
        raw* dx = reinterpret_cast<raw*>(static_cast<T*>(a.dx) + r * a.hidden);
        const float mean = a.mean[r], rstd = a.rstd[r];
        float f[U::N], g[U::N], w[U::N], p[U::N];
        float sv = 0.f, svh = 0.f;
        for (int i = threadIdx.x; i < nunits; i += G) {
            U::unpack(x[i], f);
            U::unpack(gy[i], g);
            U::unpack(gamma[i], w);
#pragma unroll
            for (int e = 0; e < U::N; ++e) {
                const float v = __fmul_rn(g[e], w[e]);
                sv = __fadd_rn(sv, v);
                svh = __fmaf_rn(v, __fmul_rn(__fsub_rn(f[e], mean), rstd), svh);
            }
        }
        const float c1 = __fmul_rn(row_sum(sv, G, scratch), inv_h);
        const float c2 = __fmul_rn(row_sum(svh, G, scratch), inv_h);
        for (int i = threadIdx.x; i < nunits; i += G) {
            U::unpack(x[i], f);
            U::unpack(gy[i], g);
            U::unpack(gamma[i], w);
            if (add) U::unpack(add[i], p);
#pragma unroll
            for (int e = 0; e < U::N; ++e) {
                const float h = __fmul_rn(__fsub_rn(f[e], mean), rstd);
                const float q = __fmaf_rn(-h, c2, __fsub_rn(__fmul_rn(g[e], w[e]), c1));
                f[e] = add ? __fmaf_rn(rstd, q, p[e]) : __fmul_rn(rstd, q);
            }
            dx[i] = U::pack(f);
        }
    }
}

// Column sums of gy * xh and of gy over a run of rows: thread = column, blockIdx.y = run.  partial: [runs][2][hidden] fp32.
template <typename T>
__global__ void __launch_bounds__(256) lna_columns(const T* x, const T* gy, const float* mean, const float* rstd, float* partial,
                                                   int64_t rows, int hidden, int64_t run) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= hidden) return;
    const int64_t r0 = blockIdx.y * run, r1 = r0 + run < rows ? r0 + run : rows;
    float sg = 0.f, sb = 0.f;
#pragma unroll 8
    for (int64_t r = r0; r < r1; ++r) {
        const float g = Vec<T>::load1(gy + r * hidden + j), f = Vec<T>::load1(x + r * hidden + j);
        sg = __fmaf_rn(g, __fmul_rn(__fsub_rn(f, mean[r]), rstd[r]), sg);
        sb = __fadd_rn(sb, g);
    }
    float* p = partial + static_cast<int64_t>(blockIdx.y) * 2 * hidden;
    p[j] = sg;
    p[hidden + j] = sb;
}

// Sums the partial rows in a fixed order, in fp64.  partial: [n][2][hidden]; blockDim (32, 8): eight runs of rows per column.
__global__ void __launch_bounds__(256) lna_column_reduce(const float* partial, int n, int hidden, float* dgamma, float* dbeta,
                                                         int accumulate) {
    __shared__ double part[8][33];
    const int j = blockIdx.x * 32 + threadIdx.x;       // over 2 * hidden
    double s = 0.0;
    if (j < 2 * hidden)
        for (int i = threadIdx.y; i < n; i += 8) s += static_cast<double>(partial[static_cast<int64_t>(i) * 2 * hidden + j]);
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y || j >= 2 * hidden) return;
    for (int k = 1; k < 8; ++k) s += part[k][threadIdx.x];
    float* out = j < hidden ? dgamma : dbeta;
    if (!out) return;
    float* o = out + (j < hidden ? j : j - hidden);
    *o = accumulate ? static_cast<float>(s + static_cast<double>(*o)) : static_cast<float>(s);
}

}  // namespace agb
