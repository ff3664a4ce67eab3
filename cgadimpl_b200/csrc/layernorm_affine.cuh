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

// The whole backward in one pass over x and gy.  A persistent CTA walks tiles of `rows_per_tile` consecutive rows; one thread keeps a ring
// of tiles filled by bulk copies, so the bytes in flight are the ring's and not the registers'.  G threads own a row (parts of a warp, a
// warp or several), UPT units of N columns each, always the same columns: their sums for dgamma and dbeta stay in registers over all
// rows of the CTA and leave as one fp32 partial row.  The tile is read twice from shared memory, once for the two row sums and once for
// dx.  One block barrier per tile joins the row sums of several warps and frees the tile before.
//   xc = x - mean;  s1 = sum v, s2 = sum v * xc  (v = gy * gamma);  dx = rstd * v + k1 + k2 * xc,  k1 = -rstd * s1 / H,
//   k2 = -rstd^3 * s2 / H;  dgamma += (gy * rstd) * xc;  dbeta += gy
// Rows that are no multiple of 16 bytes (UB < 16): the tile's bytes are one run all the same.  It is copied from the 16-byte boundary
// before it to the one behind it, which lies within the tensor except at its two ends; what the ends hold beyond whole words is copied
// by the thread itself.  Columns are then taken one by one.
struct LnaRing {
    int rows_per_tile, stages, tile_stride;    // bytes of a tile's slot for one array
    int64_t tiles;
};

// Issues tile k into a slot.  `bytes` of the tensor end at `total`.
template <bool WHOLE>
__device__ __forceinline__ void lna_copy(uint8_t* slot, const uint8_t* base, int64_t at, int bytes, int64_t total, uint64_t* bar, int elem) {
    if (WHOLE) {
        bulk_load(slot, base + at, bytes, bar);
        return;
    }
    const uint8_t* p = base + at;
    const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    int lo = -lead, hi = (lead + bytes + 15) / 16 * 16 - lead;                 // relative to p
    if (at + lo < 0) lo += 16;
    if (at + hi > total) hi -= 16;
    // the ends of the tensor, at most 15 bytes each (and the whole of a tile of a few bytes)
    const int head = lo < 0 ? 0 : (lo < bytes ? lo : bytes);
    for (int i = 0; i < head; i += elem)
        for (int b = 0; b < elem; b += 2) *reinterpret_cast<uint16_t*>(slot + lead + i + b) = *reinterpret_cast<const uint16_t*>(p + i + b);
    for (int i = hi > head ? hi : head; i < bytes; i += elem)
        for (int b = 0; b < elem; b += 2) *reinterpret_cast<uint16_t*>(slot + lead + i + b) = *reinterpret_cast<const uint16_t*>(p + i + b);
    mbar_arrive_expect_tx(bar, hi > lo ? hi - lo : 0);
    if (hi > lo) bulk_load(slot + lead + lo, p + lo, hi - lo, bar);
}

template <typename T, int UB, int UPT, int MAXT>
__global__ void __launch_bounds__(MAXT) lna_bwd_ring(const LnaBwdArgs a, const LnaRing g, float* partial, int* status) {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    constexpr int N = U::N, S = 8;
    constexpr bool WHOLE = UB == 16;
    extern __shared__ __align__(128) uint8_t lna_smem[];
    __shared__ __align__(8) uint64_t full[S];
    __shared__ float2 scratch[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.G, t = tid % G, mine = tid / G;            // this thread's place in its row, its row of the tile
    const int H = a.hidden, nunits = H / N;
    const int64_t row_bytes = static_cast<int64_t>(H) * sizeof(T), total = a.rows * row_bytes;
    const uint8_t* xb = static_cast<const uint8_t*>(a.x);
    const uint8_t* gb = static_cast<const uint8_t*>(a.gy);
    if (tid == 0) {
        for (int s = 0; s < g.stages; ++s) mbar_init(&full[s], WHOLE ? 1 : 2);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    auto issue = [&](int64_t k, int s) {
        const int64_t r0 = k * g.rows_per_tile;
        const int rows = static_cast<int>(a.rows - r0 < g.rows_per_tile ? a.rows - r0 : g.rows_per_tile);
        const int bytes = static_cast<int>(rows * row_bytes);
        uint8_t* slot = lna_smem + static_cast<int64_t>(2 * s) * g.tile_stride;
        if (WHOLE) mbar_arrive_expect_tx(&full[s], 2 * bytes);
        lna_copy<WHOLE>(slot, xb, r0 * row_bytes, bytes, total, &full[s], sizeof(T));
        lna_copy<WHOLE>(slot + g.tile_stride, gb, r0 * row_bytes, bytes, total, &full[s], sizeof(T));
    };
    const int64_t step = gridDim.x;
    if (tid == 0) {
        int64_t k = blockIdx.x;
        for (int s = 0; s < g.stages && k < g.tiles; ++s, k += step) issue(k, s);
    }
    float dg[UPT][N], db[UPT][N];
    const raw* gamma = reinterpret_cast<const raw*>(a.gamma);   // from L1 each time: the sums take the registers
#pragma unroll
    for (int i = 0; i < UPT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) dg[i][e] = db[i][e] = 0.f;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(H));
    int s = 0, prev = 0, n = 0;
    uint32_t phase = 0;
    float next_mean = 0.f, next_rstd = 0.f;
    {
        const int64_t r = static_cast<int64_t>(blockIdx.x) * g.rows_per_tile + mine;
        if (r < a.rows && mine < g.rows_per_tile) {
            next_mean = a.mean[r];
            next_rstd = a.rstd[r];
        }
    }
    bool ok = true;
    for (int64_t k = blockIdx.x; k < g.tiles; k += step, ++n) {
        const int64_t r = k * g.rows_per_tile + mine;
        const bool live = r < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        const int64_t rn = r + step * g.rows_per_tile;
        if (rn < a.rows) {
            next_mean = a.mean[rn];
            next_rstd = a.rstd[rn];
        }
        ok = mbar_wait_bounded(&full[s], phase) && ok;
        const uint8_t* slot = lna_smem + static_cast<int64_t>(2 * s) * g.tile_stride;
        const int64_t at = k * g.rows_per_tile * row_bytes;
        const int ox = WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(xb + at) & 15);
        const int og = WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(gb + at) & 15);
        const raw* x = reinterpret_cast<const raw*>(slot + ox + mine * row_bytes);
        const raw* gy = reinterpret_cast<const raw*>(slot + g.tile_stride + og + mine * row_bytes);
        float s1 = 0.f, s2 = 0.f;
        if (live) {
#pragma unroll
            for (int i = 0; i < UPT; ++i)
                if (t + i * G < nunits) {
                    float f[N], q[N], w[N];
                    U::unpack(x[t + i * G], f);
                    U::unpack(gy[t + i * G], q);
                    U::unpack(__ldg(gamma + t + i * G), w);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float v = __fmul_rn(q[e], w[e]);
                        s1 = __fadd_rn(s1, v);
                        s2 = __fmaf_rn(v, __fsub_rn(f[e], mean), s2);
                    }
                }
        }
        for (int o = (G < 32 ? G : 32) >> 1; o > 0; o >>= 1) {
            s1 = __fadd_rn(s1, __shfl_xor_sync(0xffffffffu, s1, o));
            s2 = __fadd_rn(s2, __shfl_xor_sync(0xffffffffu, s2, o));
        }
        if (G > 32 && lane == 0) scratch[n & 1][warp] = make_float2(s1, s2);
        __syncthreads();                               // the sums are there, and everyone has left the tile before
        if (tid == 0 && n > 0 && g.stages > 1) {
            const int64_t kn = k + (g.stages - 1) * step;
            if (kn < g.tiles) issue(kn, prev);
        }
        if (G > 32) {
            const int w0 = mine * (G >> 5);
            s1 = s2 = 0.f;
            for (int w = w0; w < w0 + (G >> 5); ++w) {
                const float2 q = scratch[n & 1][w];
                s1 = __fadd_rn(s1, q.x);
                s2 = __fadd_rn(s2, q.y);
            }
        }
        if (live) {
            const float k1 = -__fmul_rn(rstd, __fmul_rn(s1, inv_h));
            const float k2 = -__fmul_rn(__fmul_rn(rstd, rstd), __fmul_rn(rstd, __fmul_rn(s2, inv_h)));
            raw* dx = reinterpret_cast<raw*>(static_cast<T*>(a.dx) + r * H);
            const raw* add = a.dx_add ? reinterpret_cast<const raw*>(static_cast<const T*>(a.dx_add) + r * H) : nullptr;
#pragma unroll
            for (int i = 0; i < UPT; ++i)
                if (t + i * G < nunits) {
                    float f[N], q[N], w[N], p[N];
                    U::unpack(x[t + i * G], f);
                    U::unpack(gy[t + i * G], q);
                    U::unpack(__ldg(gamma + t + i * G), w);
                    if (add) U::unpack(add[t + i * G], p);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float xc = __fsub_rn(f[e], mean), gr = __fmul_rn(q[e], rstd);
                        db[i][e] = __fadd_rn(db[i][e], q[e]);
                        dg[i][e] = __fmaf_rn(gr, xc, dg[i][e]);
                        float d = __fmaf_rn(gr, w[e], __fmaf_rn(xc, k2, k1));
                        if (add) d = __fadd_rn(d, p[e]);
                        f[e] = d;
                    }
                    const raw out = U::pack(f);
                    if constexpr (UB == 16) store_vec_streaming(dx + t + i * G, out);
                    else dx[t + i * G] = out;
                }
        }
        if (g.stages == 1) {                           // a ring of one: the next tile once everyone has left this one
            __syncthreads();
            if (tid == 0 && k + step < g.tiles) issue(k + step, 0);
        }
        prev = s;
        if (++s == g.stages) {
            s = 0;
            phase ^= 1;
        }
    }
    if (!ok) {
        if (tid == 0) atomicExch(status, 6 /* AGB_ERR_TIMEOUT */);
    }
    if (!partial) return;
    // ---- the CTA's partial row: rows of a warp first, then warps of the same columns in order
    for (int o = 16; o >= G; o >>= 1) {
#pragma unroll
        for (int i = 0; i < UPT; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                dg[i][e] = __fadd_rn(dg[i][e], __shfl_xor_sync(0xffffffffu, dg[i][e], o));
                db[i][e] = __fadd_rn(db[i][e], __shfl_xor_sync(0xffffffffu, db[i][e], o));
            }
    }
    float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * H;
    const int per = G < 32 ? 32 : G, groups = blockDim.x / per, group = tid / per;      // threads that hold all columns once
    if (groups == 1) {
        if (tid < G) {
#pragma unroll
            for (int i = 0; i < UPT; ++i)
                if (t + i * G < nunits)
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        out[(t + i * G) * N + e] = dg[i][e];
                        out[H + (t + i * G) * N + e] = db[i][e];
                    }
        }
        return;
    }
    float* sums = reinterpret_cast<float*>(lna_smem);  // the ring is empty: every tile issued has been waited for
    for (int q = 0; q < groups; ++q) {
        __syncthreads();
        if (group == q && tid % per < G) {
#pragma unroll
            for (int i = 0; i < UPT; ++i)
                if (t + i * G < nunits)
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int c = (t + i * G) * N + e;
                        sums[c] = q ? __fadd_rn(sums[c], dg[i][e]) : dg[i][e];
                        sums[H + c] = q ? __fadd_rn(sums[H + c], db[i][e]) : db[i][e];
                    }
        }
    }
    __syncthreads();
    for (int c = tid; c < 2 * H; c += blockDim.x) out[c] = sums[c];
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

// Sums the partial rows in a fixed order, in fp64.  partial: [n][2][hidden]; blockDim (32, 32): 32 runs of rows per column.
__global__ void __launch_bounds__(1024) lna_column_reduce(const float* partial, int n, int hidden, float* dgamma, float* dbeta,
                                                          int accumulate) {
    __shared__ double part[32][33];
    pdl_wait();
    pdl_trigger();
    const int j = blockIdx.x * 32 + threadIdx.x;       // over 2 * hidden
    double s = 0.0;
    if (j < 2 * hidden) {
#pragma unroll 4
        for (int i = threadIdx.y; i < n; i += 32) s += static_cast<double>(partial[static_cast<int64_t>(i) * 2 * hidden + j]);
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    // warp y joins the 32 runs of column y
    const int jj = blockIdx.x * 32 + threadIdx.y;
    s = warp_sum(part[threadIdx.x][threadIdx.y]);
    if (threadIdx.x || jj >= 2 * hidden) return;
    float* out = jj < hidden ? dgamma : dbeta;
    if (!out) return;
    float* o = out + (jj < hidden ? jj : jj - hidden);
    *o = accumulate ? static_cast<float>(s + static_cast<double>(*o)) : static_cast<float>(s);
}

}  // namespace agb
