// layernorm_affine.cuh -- LayerNorm with weight and bias, forward and VJP.
//   mean = sum_j x / H;  rstd = 1 / sqrt(sum_j (x - mean)^2 / H + eps);  xh = (x - mean) * rstd;  y = xh * gamma + beta
//   v = gy * gamma;  dx = rstd * (v - sum_j v / H - xh * (sum_j v * xh) / H)
//   dgamma[j] = sum_r gy * xh;  dbeta[j] = sum_r gy
// Every sum is carried in fp32, column sums over the CTAs in fp64; outputs are rounded once.  The variance is taken from
// the centred values (a second pass over registers), so an offset of the row costs no digits.
// No contraction of a size that matters: bound by memory.  16384 x 8192 bf16: forward 105 us (79 % of the copy rate), backward 163 us (76 %);
// 8192 x 4096 fp32: 47 us (89 %) and 83 us (75 %).  What is left is latency: 16 warps an SM and two block barriers a row (ncu: issue slots 55 %
// busy, DRAM 54 %); a third block an SM at 80 registers spills (forward 151 us).
#pragma once
#include <type_traits>

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

// Two lanes of fp32 at once (one instruction each on sm_100a).
__device__ __forceinline__ float2 pk(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2p(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
// A thread's UPT units of a row as pairs of fp32 (a unit of one element shares a pair with the next unit).  The units lie 32 apart, so
// that a warp reads neighbours and every offset is a constant of the instruction.  Units at or behind `lim` do not exist: they load as
// zeros and are not stored; FULL says that there are none.
template <typename T, int UB, int UPT>
struct Slice {
    typedef Unit<T, UB> U;
    typedef typename U::raw raw;
    static constexpr int N = U::N, NV = UPT * N, P = (NV + 1) / 2;
    template <bool FULL, typename L>
    __device__ __forceinline__ static void load(float2 (&f)[P], int lim, L get) {
        float v[2 * P];
        v[2 * P - 1] = 0.f;
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
            raw u{};
            if (FULL || 32 * i < lim) u = get(32 * i);
            U::unpack(u, v + i * N);
        }
#pragma unroll
        for (int e = 0; e < P; ++e) f[e] = make_float2(v[2 * e], v[2 * e + 1]);
    }
    template <bool FULL, typename F>
    __device__ __forceinline__ static void store(const float2 (&f)[P], int lim, F put) {
        float v[2 * P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
            v[2 * e] = f[e].x;
            v[2 * e + 1] = f[e].y;
        }
#pragma unroll
        for (int i = 0; i < UPT; ++i)
            if (FULL || 32 * i < lim) put(32 * i, U::pack(v + i * N));
    }
    __device__ __forceinline__ static float at(const float2 (&f)[P], int e) { return e & 1 ? f[e >> 1].y : f[e >> 1].x; }
};
// First unit of thread t of a row of G threads (G below 32: one unit per thread).
__device__ __forceinline__ int first_unit(int t, int G, int upt) { return G <= 32 ? t : (t >> 5) * 32 * upt + (t & 31); }

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

struct LnaRing {
    int rows_per_tile, stages, tile_stride;    // bytes of a tile's slot for one array
    int64_t tiles;
};

// Copies a tile's bytes [at, at + bytes) of a tensor of `total` bytes into a slot.
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


// Forward.  The ring of lna_bwd_ring with one array; a thread takes its slice of the row out of the tile into registers, and the mean and
// the centred squares are summed from there.  Two block barriers per tile where a row is several warps, the first of which also frees
// the slot.
template <typename T, int UB, int UPT, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? 3 : 1) lna_fwd_ring(const LnaFwdArgs a, const LnaRing g, int* status) {
    typedef Slice<T, UB, UPT> L;
    typedef typename L::raw raw;
    constexpr int N = L::N, P = L::P, S = 8;
    constexpr bool WHOLE = UB == 16;
    extern __shared__ __align__(128) uint8_t lna_smem[];
    __shared__ __align__(8) uint64_t full[S];
    __shared__ float scratch[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.G, t = tid % G, mine = tid / G;
    const int H = a.hidden, first = first_unit(t, G, UPT), lim = H / N - first;
    const bool all = __all_sync(0xffffffffu, lim > 32 * (UPT - 1));
    const int64_t row_bytes = static_cast<int64_t>(H) * sizeof(T), total = a.rows * row_bytes;
    const uint8_t* xb = static_cast<const uint8_t*>(a.x);
    if (tid == 0) {
        for (int s = 0; s < g.stages; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
    auto issue = [&](int64_t k, int s) {
        const int64_t r0 = k * g.rows_per_tile;
        const int rows = static_cast<int>(a.rows - r0 < g.rows_per_tile ? a.rows - r0 : g.rows_per_tile);
        const int bytes = static_cast<int>(rows * row_bytes);
        if (WHOLE) mbar_arrive_expect_tx(&full[s], bytes);
        lna_copy<WHOLE>(lna_smem + static_cast<int64_t>(s) * g.tile_stride, xb, r0 * row_bytes, bytes, total, &full[s], sizeof(T));
    };
    const int64_t step = gridDim.x;
    if (tid == 0) {
        int64_t k = blockIdx.x;
        for (int s = 0; s < g.stages && k < g.tiles; ++s, k += step) issue(k, s);
    }
    const raw* gamma = reinterpret_cast<const raw*>(a.gamma) + first;
    const raw* beta = reinterpret_cast<const raw*>(a.beta) + first;
    const bool with_beta = a.beta != nullptr;
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(H));
    const int w0 = mine * (G >> 5), w1 = w0 + (G >> 5);
    // sum over the row's threads; the scratch of the two sums of a tile alternates, so that one barrier each is enough
    auto row_total = [&](float v, int which) {
        for (int o = (G < 32 ? G : 32) >> 1; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
        if (G <= 32) return v;
        if (lane == 0) scratch[which][warp] = v;
        __syncthreads();
        v = 0.f;
        for (int w = w0; w < w1; w += 4) {             // four loads in flight
            float q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = w + u < w1 ? scratch[which][w + u] : 0.f;
            v = __fadd_rn(v, __fadd_rn(__fadd_rn(q[0], q[1]), __fadd_rn(q[2], q[3])));
        }
        return v;
    };
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto tile = [&](auto full_tag, int64_t k) {
        constexpr bool FULL = decltype(full_tag)::value;
        const int64_t r = k * g.rows_per_tile + mine;
        const bool live = r < a.rows;
        const int n = live ? lim : 0;
        const int ox = WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(xb + k * g.rows_per_tile * row_bytes) & 15);
        const raw* x = reinterpret_cast<const raw*>(lna_smem + static_cast<int64_t>(s) * g.tile_stride + ox + mine * row_bytes) + first;
        float2 f[P];
        L::template load<FULL>(f, n, [&](int u) { return x[u]; });
        float2 v = f[0];
#pragma unroll
        for (int e = 1; e < P; ++e) v = add2(v, f[e]);
        if (G <= 32) __syncthreads();                  // everyone has taken the tile out of its slot
        const float mean = __fmul_rn(row_total(__fadd_rn(v.x, v.y), 0), inv_h);
        if (tid == 0 && k + g.stages * step < g.tiles) issue(k + g.stages * step, s);      // row_total's barrier has been passed
        v = pk(0.f);
#pragma unroll
        for (int e = 0; e < P; ++e) {
            // columns that do not exist add nothing to the squares
            const bool x0 = FULL && 2 * e < L::NV ? true : 32 * (2 * e / N) < n, x1 = (2 * e + 1 < L::NV) && (FULL || 32 * ((2 * e + 1) / N) < n);
            f[e] = add2(f[e], make_float2(x0 ? -mean : 0.f, x1 ? -mean : 0.f));
            v = fma2p(f[e], f[e], v);
        }
        const float rstd = rsqrtf(__fmaf_rn(row_total(__fadd_rn(v.x, v.y), 1), inv_h, a.eps));
        if (live && t == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        raw* y = reinterpret_cast<raw*>(static_cast<T*>(a.y) + r * H) + first;
        float2 w[P];
        L::template load<FULL>(w, n, [&](int u) { return __ldg(gamma + u); });
        if (with_beta) {
            float2 b[P];
            L::template load<FULL>(b, n, [&](int u) { return __ldg(beta + u); });
#pragma unroll
            for (int e = 0; e < P; ++e) f[e] = fma2p(mul2(f[e], pk(rstd)), w[e], b[e]);
        } else {
#pragma unroll
            for (int e = 0; e < P; ++e) f[e] = mul2(mul2(f[e], pk(rstd)), w[e]);
        }
        L::template store<FULL>(f, n, [&](int u, const raw& out) {
            if constexpr (UB == 16) store_vec_streaming(y + u, out);
            else y[u] = out;
        });
    };
    for (int64_t k = blockIdx.x; k < g.tiles; k += step) {
        ok = mbar_wait_bounded(&full[s], phase) && ok;
        // the whole warp has all its units, and all rows of the tile exist
        if (all && (k + 1) * g.rows_per_tile <= a.rows) tile(std::true_type{}, k);
        else tile(std::false_type{}, k);
        if (++s == g.stages) {
            s = 0;
            phase ^= 1;
        }
    }
    pdl_trigger();                                     // at the end: 1 to 7 % ahead of triggering at the start
    if (!ok && tid == 0) atomicExch(status, 6 /* AGB_ERR_TIMEOUT */);
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
            U::unpack(__ldg(reinterpret_cast<const raw*>(a.gamma) + i), g);
            if (a.beta) U::unpack(__ldg(reinterpret_cast<const raw*>(a.beta) + i), b);
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
template <typename T, int UB, int UPT, int MAXT>
__global__ void __launch_bounds__(MAXT) lna_bwd_ring(const LnaBwdArgs a, const LnaRing g, float* partial, int* status) {
    // the slice is worked through in parts, so that the sums of all of it and the values of one part fit the registers
    constexpr int NU = Unit<T, UB>::N, PART = UPT * NU > 8 ? (8 / NU > 0 ? 8 / NU : 1) : UPT, PARTS = UPT / PART;
    typedef Slice<T, UB, PART> L;
    typedef typename L::raw raw;
    constexpr int N = L::N, P = L::P, S = 8;
    constexpr bool WHOLE = UB == 16;
    extern __shared__ __align__(128) uint8_t lna_smem[];
    __shared__ __align__(8) uint64_t full[S];
    __shared__ float2 scratch[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.G, t = tid % G, mine = tid / G;            // this thread's place in its row, its row of the tile
    const int H = a.hidden, first = first_unit(t, G, UPT), lim = H / N - first;
    const bool all = __all_sync(0xffffffffu, lim > 32 * (UPT - 1));
    const int64_t row_bytes = static_cast<int64_t>(H) * sizeof(T), total = a.rows * row_bytes;
    const uint8_t* xb = static_cast<const uint8_t*>(a.x);
    const uint8_t* gb = static_cast<const uint8_t*>(a.gy);
    if (tid == 0) {
        for (int s = 0; s < g.stages; ++s) mbar_init(&full[s], WHOLE ? 1 : 2);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
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
    float2 dg[PARTS][P], db[PARTS][P];
    const raw* gamma = reinterpret_cast<const raw*>(a.gamma) + first;   // from L1 each time: the sums take the registers
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
        for (int e = 0; e < P; ++e) dg[i][e] = db[i][e] = pk(0.f);
    const float inv_h = __fdiv_rn(1.f, static_cast<float>(H));
    int s = 0, prev = 0, n = 0;
    uint32_t phase = 0;
    float next_mean = 0.f, next_rstd = 0.f;
    {
        const int64_t r = static_cast<int64_t>(blockIdx.x) * g.rows_per_tile + mine;
        if (r < a.rows) {
            next_mean = a.mean[r];
            next_rstd = a.rstd[r];
        }
    }
    bool ok = true;
    auto tile = [&](auto full_tag, int64_t k) {
        constexpr bool FULL = decltype(full_tag)::value;
        const int64_t r = k * g.rows_per_tile + mine;
        const float mean = next_mean, rstd = next_rstd;
        const int64_t rn = r + step * g.rows_per_tile;
        if (rn < a.rows) {
            next_mean = a.mean[rn];
            next_rstd = a.rstd[rn];
        }
        const int have = r < a.rows ? lim : 0;
        const uint8_t* slot = lna_smem + static_cast<int64_t>(2 * s) * g.tile_stride;
        const int64_t at = k * g.rows_per_tile * row_bytes;
        const int ox = WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(xb + at) & 15);
        const int og = WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(gb + at) & 15);
        const raw* x = reinterpret_cast<const raw*>(slot + ox + mine * row_bytes) + first;
        const raw* gy = reinterpret_cast<const raw*>(slot + g.tile_stride + og + mine * row_bytes) + first;
        // columns that do not exist come as zeros of gy and gamma, which adds nothing to any of the sums
        float2 t1 = pk(0.f), t2 = pk(0.f);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int o = 32 * PART * i;
            float2 f[P], q[P], w[P];
            L::template load<FULL>(f, have - o, [&](int u) { return x[o + u]; });
            L::template load<FULL>(q, have - o, [&](int u) { return gy[o + u]; });
            L::template load<FULL>(w, have - o, [&](int u) { return __ldg(gamma + o + u); });
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 v = mul2(q[e], w[e]);
                t1 = add2(t1, v);
                t2 = fma2p(v, add2(f[e], pk(-mean)), t2);
            }
        }
        float s1 = __fadd_rn(t1.x, t1.y), s2 = __fadd_rn(t2.x, t2.y);
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
            const int w0 = mine * (G >> 5), w1 = w0 + (G >> 5);
            s1 = s2 = 0.f;
            for (int w = w0; w < w1; w += 4) {         // four loads in flight
                float2 q[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) q[u] = w + u < w1 ? scratch[n & 1][w + u] : pk(0.f);
                s1 = __fadd_rn(s1, __fadd_rn(__fadd_rn(q[0].x, q[1].x), __fadd_rn(q[2].x, q[3].x)));
                s2 = __fadd_rn(s2, __fadd_rn(__fadd_rn(q[0].y, q[1].y), __fadd_rn(q[2].y, q[3].y)));
            }
        }
        const float k1 = -__fmul_rn(rstd, __fmul_rn(s1, inv_h));
        const float k2 = -__fmul_rn(__fmul_rn(rstd, rstd), __fmul_rn(rstd, __fmul_rn(s2, inv_h)));
        raw* dx = reinterpret_cast<raw*>(static_cast<T*>(a.dx) + r * H) + first;
        const raw* add = a.dx_add ? reinterpret_cast<const raw*>(static_cast<const T*>(a.dx_add) + r * H) + first : nullptr;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int o = 32 * PART * i;
            float2 f[P], q[P], w[P];
            L::template load<FULL>(f, have - o, [&](int u) { return x[o + u]; });
            L::template load<FULL>(q, have - o, [&](int u) { return gy[o + u]; });
            L::template load<FULL>(w, have - o, [&](int u) { return __ldg(gamma + o + u); });
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 xc = add2(f[e], pk(-mean)), gr = mul2(q[e], pk(rstd));
                db[i][e] = add2(db[i][e], q[e]);
                dg[i][e] = fma2p(gr, xc, dg[i][e]);
                f[e] = fma2p(gr, w[e], fma2p(xc, pk(k2), pk(k1)));
            }
            if (add) {
                float2 p[P];
                L::template load<FULL>(p, have - o, [&](int u) { return add[o + u]; });
#pragma unroll
                for (int e = 0; e < P; ++e) f[e] = add2(f[e], p[e]);
            }
            L::template store<FULL>(f, have - o, [&](int u, const raw& out) {
                if constexpr (UB == 16) store_vec_streaming(dx + o + u, out);
                else dx[o + u] = out;
            });
        }
    };
    for (int64_t k = blockIdx.x; k < g.tiles; k += step, ++n) {
        ok = mbar_wait_bounded(&full[s], phase) && ok;
        // the whole warp has all its units, and all rows of the tile exist
        if (all && (k + 1) * g.rows_per_tile <= a.rows) tile(std::true_type{}, k);
        else tile(std::false_type{}, k);
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
    pdl_trigger();                                     // at the end: 1 to 7 % ahead of triggering at the start
    if (!ok && tid == 0) atomicExch(status, 6 /* AGB_ERR_TIMEOUT */);
    if (!partial) return;
    // ---- the CTA's partial row: rows of a warp first, then warps of the same columns in order
    for (int o = 16; o >= G; o >>= 1) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
            for (int e = 0; e < P; ++e) {
                dg[i][e] = add2(dg[i][e], make_float2(__shfl_xor_sync(0xffffffffu, dg[i][e].x, o), __shfl_xor_sync(0xffffffffu, dg[i][e].y, o)));
                db[i][e] = add2(db[i][e], make_float2(__shfl_xor_sync(0xffffffffu, db[i][e].x, o), __shfl_xor_sync(0xffffffffu, db[i][e].y, o)));
            }
    }
    float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * H;
    const int per = G < 32 ? 32 : G, groups = blockDim.x / per, group = tid / per;      // threads that hold all columns once
    float* sums = groups == 1 ? out : reinterpret_cast<float*>(lna_smem);               // the ring is empty: every tile has been waited for
    for (int q = 0; q < groups; ++q) {
        __syncthreads();
        if (group != q || tid % per >= G) continue;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
            for (int u = 0; u < PART; ++u) {
                const int unit = 32 * (PART * i + u);
                if (unit >= lim) continue;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int c = (first + unit) * N + e;
                    const float vg = L::at(dg[i], u * N + e), vb = L::at(db[i], u * N + e);
                    sums[c] = q ? __fadd_rn(sums[c], vg) : vg;
                    sums[H + c] = q ? __fadd_rn(sums[H + c], vb) : vb;
                }
            }
    }
    if (groups == 1) return;
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
