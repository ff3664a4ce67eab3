// linear_ce.cuh -- softmax cross entropy taken straight from the hidden states, the logits never kept.
//   z = h W';  lse_t = log sum_v exp z_tv;  loss_t = lse_t - z_t,target(t)
//   g_tv = gy_t * (exp(z_tv - lse_t) - [v = target(t)]);  dh = g W;  dW = g' h
// Rows whose target names no column take no part: they are left out when h is laid out for the products (rows in order, no gaps), so
// they cost nothing and what they hold (padding, NaN) reaches nothing.
//
// Bound by the tensor cores: 2 * rows * hidden * vocab operations forward, three times that backward (the logits again, dh, dw).  ncu, 2048 x
// 4096 x 32768 bf16: tensor pipe active 92 % (logits, 340 us), 89 % (g, 352 us), 90 % (dh and dw, 761 us), DRAM 11 to 22 %.  Events: 4096 x 4096 x
// 18944 forward 409 us, 1556 TFLOP/s in a burst; 8192 x 4096 x 131072 with a quarter of the rows left out, forward and backward 20.2 ms, 1.31
// PFLOP/s under the power cap.  With few rows the forward reads W once: 16 x 4096 x 32768 58 us for 268 MB.  fp32, 1023 x 1024 x 50001: six
// products each at 1430 (logits), 1070 (g) and 1310 TFLOP/s (dh and dw).
//
// One persistent kernel does all the products.  Tiles of 128 x 256 with fp32 accumulators in tensor memory (two of them: the
// epilogue of a tile runs under the products of the next), operands in 64-wide slabs through a ring of TMA loads; CTA pairs
// (cta_group::2) on tiles of 256 x 256 read half of B each, which is what 64 bytes a clock from L2 allow.  Forward: the
// epilogue turns a tile of logits into a (max, sum of exp) pair per row and half tile; a small kernel joins the pairs.  Backward,
// piece by piece of the vocabulary: the logits again with an epilogue that writes g in 16 bits, then dh += g W and dW = g' h in one
// launch.  dh is kept in fp32 over the pieces; where rows are few the vocabulary axis is cut between CTAs and the parts are summed
// in order.
//
// What the tensor cores keep of a sum: their fp32 accumulators cut instead of rounding, so a logit of 4096 terms comes out about 1e-6 of
// itself too small.  The target's logit is computed apart (ce_join_kernel); the others enter lse as they are: a loss of 8 is off by about 1e-5.
// g is kept relative to the largest |gy| (a mean's gy, all alike, would otherwise round every target's g the same way), and what
// rounding takes from the target's g is given back to dh in fp32 (ce_dh_kernel).
//
// fp32 operands are split into three bf16 planes (x = x1 + x2 + x3 exactly: 8 bits of mantissa each), and a product is the sum
// of the six plane products down to 2^-16 of the largest; the three left out are below 2^-24 of it.  g in 16-bit mode is rounded to
// bf16 before the two gradient products (half a step, 2^-8 relative to each g, independent over the sum): the operand type of the
// matrix instruction, the accuracy that dh and dW are rounded to themselves.
#pragma once
#include "distill_topk.cuh"
#include "umma.cuh"

namespace agb {

constexpr int kTM = 128, kTN = 256, kTK = 64;          // rows of A per CTA, most columns of a tile, depth of a slab
constexpr int kCeThreads = 384;        // TMA, MMA, TMEM, idle, and eight warps of epilogue
// CG CTAs work on a tile of CG * 128 rows together (tcgen05 cta_group): each holds its 128 rows of A, its share of the columns of
// B and the accumulators of its rows.  A pair reads half of B per CTA, so its ring is deeper for the same bytes.
// Behind the ring each epilogue warp has boxes of 4 KB (32 rows of 128 bytes) in which its results leave by TMA, in turn.
constexpr int kBoxBytes = 32 * 128;
template <int CG, int PHASE>
struct CeRing {
    static constexpr int kStages = CG == 1 ? 4 : 6;
    static constexpr int kBoxes = PHASE == 0 ? 0 : 1;
    static constexpr int kBytesA = kTM * kTK * 2, kBytesB = kTN / CG * kTK * 2;
    static constexpr int kStageBytes = kBytesA + kBytesB;
    static constexpr int kSmem = kStages * kStageBytes + 8 * kBoxes * kBoxBytes + 1024;
};

// What an epilogue does with its tile.
enum CeEpi { kEpiPairs = 0, kEpiG = 1, kEpiDh = 2, kEpiDw = 3 };

struct CeJob {
    int epi;
    int a_mn, b_mn;                    // operand major-ness: 0 K-major, 1 MN-major
    int a_planes3, b_row0, a_row0;     // a_planes3: the six products of split fp32 operands; row offsets of the piece in B (A)
    int m, n, k;                       // extents; m < 0 or k < 0: the number of rows that take part, read on the device
    int splits, k_per_split;           // K cut into `splits` parts of k_per_split (a multiple of kTK)
    int n_first;                       // tile order: 1 N fastest, 0 M fastest in groups of kMGroup rows
    int tn;                            // columns of a tile, at most 256
    int b_box;                         // rows of B's TMA box: 64 where B is MN-major, else a CTA's whole share of the columns
};
constexpr int kMGroup = 4096;

// dw leaves by TMA to its place; or, where its rows are no multiple of 16 bytes, to a buffer with rows that are (in 32 bits if it is to be
// added), from which ce_unpack_kernel takes it; or, where only its base lies between, element by element.
enum CeDw { kDwTma = 0, kDwStaged = 1, kDwScalar = 2 };

struct CeArgs {
    CUtensorMap A[2], B[2];
    CUtensorMap out[2];                // of the job's results, boxes of 32 rows of 128 bytes
    CeJob job[2];
    int jobs;
    const int* count;                  // rows that take part
    int* status;
    int64_t rows_pad;                  // row stride of the per-row arrays below
    // pairs
    float2* pairs;                     // [rows_pad][half tiles of the vocabulary]
    int64_t n_pairs;
    float* z_target;                   // [rows_pad]
    const int* target;                 // [rows_pad]
    int pair0;                         // first half tile of this piece
    int col0, vocab;                   // first column of the piece
    // g
    const float *lse, *gy;             // [rows_pad]
    __nv_bfloat16* g;                  // [planes][rows_pad][g_stride]
    float* left_over;                  // [rows_pad]: what rounding took from g at the row's target (one plane only, else NULL)
    const float* gy_scale;             // the largest |gy|: g is kept relative to it
    int64_t g_stride;
    int planes;
    // dh: fp32 parts [split][rows_pad][dh_stride]
    float* dh;
    int64_t dh_stride;
    int dh_add;                        // 0 the first piece: write, 1 add
    // dw
    void* dw;
    int hidden, dw_add, dw_f32;
    int dw_out;                        // how dw leaves: CeDw
};

struct CeTile {
    int m0, n0, k0, iters, split;
};

// The extents of a job with the device's row count filled in, and its number of tiles.
struct CeShape {
    int m, n, k, tm, mt, nt, tiles;
    __device__ __forceinline__ CeShape(const CeJob& j, int count, int tile_m) {
        m = j.m < 0 ? count : j.m;
        k = j.k < 0 ? count : j.k;
        n = j.n;
        tm = tile_m;
        mt = (m + tm - 1) / tm;
        nt = (n + j.tn - 1) / j.tn;
        tiles = mt * nt * j.splits;
    }
};
__device__ __forceinline__ CeTile ce_tile(const CeJob& j, const CeShape& s, int t) {
    CeTile o;
    int m, n;
    o.split = t / (s.mt * s.nt);
    t -= o.split * s.mt * s.nt;
    if (j.n_first) {
        n = t % s.nt;
        m = t / s.nt;
    } else {
        const int tall = kMGroup / s.tm, group = t / (tall * s.nt), first = group * tall;
        const int height = s.mt - first < tall ? s.mt - first : tall;
        t -= first * s.nt;
        m = first + t % height;
        n = t / height;
    }
    o.m0 = m * s.tm;
    o.n0 = n * j.tn;
    o.k0 = o.split * j.k_per_split;
    const int k1 = o.k0 + j.k_per_split < s.k ? o.k0 + j.k_per_split : s.k;
    const int blocks = k1 > o.k0 ? (k1 - o.k0 + kTK - 1) / kTK : 0;
    o.iters = blocks * (j.a_planes3 ? 6 : 1);
    return o;
}
// Plane pairs of the six products, smallest first.
__device__ __forceinline__ void plane_pair(int p, int& a, int& b) {
    // (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
    a = p == 1 ? 2 : (p == 2 || p == 4) ? 1 : 0;
    b = p == 0 ? 2 : (p == 2 || p == 3) ? 1 : 0;
}

// x = hi + mid + lo, each with 8 bits of mantissa, cut (not rounded) so that none overflows; what is not finite stays in hi.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const uint32_t u = __float_as_uint(x);
    hi = u & 0xffff0000u;
    if ((u & 0x7f800000u) == 0x7f800000u) {
        if (u & 0x007fffffu) hi |= 0x00400000u;        // NaN stays NaN when its low bits are cut
        mid = lo = 0;
        return;
    }
    const float r = __fsub_rn(x, __uint_as_float(hi));
    mid = __float_as_uint(r) & 0xffff0000u;
    lo = __float_as_uint(__fsub_rn(r, __uint_as_float(mid))) & 0xffff0000u;
}

// ---------------------------------------------------------------- laying out
// Rows of x [rows][cols] whose target names a column, in order and without gaps, into dst [planes][rows_pad][stride] bf16;
// zeros behind the last column up to `stride` and, for the backward, behind the last row up to a multiple of kTK.  Also the
// per-row arrays.
// A block takes `per_block` (at most 32) rows; it counts the targets before its own to know where they go.  kRowsEnd blocks behind them
// count all targets and do what needs that number.
struct CeRowsArgs {
    const void* x;
    const void* target;
    int target64;
    int64_t rows;
    int cols, vocab, planes, per_block;
    __nv_bfloat16* dst;
    int64_t rows_pad, stride;
    int* count;
    int* row_of;                       // [rows_pad]: the row that went there
    int* pos_of;                       // [rows]: where the row went, or -1
    int* target_of;                    // [rows_pad]
    const float *lse, *gy;             // backward: [rows]; NULL in the forward
    float *lse_of, *gy_of, *gy_scale;
    float *loss, *lse_out;             // forward: rows that take no part get 0
};
constexpr int kRowsBlock = 32;         // most rows of a block
constexpr int kRowsEnd = 8;

__device__ __forceinline__ int ce_target(const CeRowsArgs& a, int64_t r) {
    const int64_t t = a.target64 ? static_cast<const int64_t*>(a.target)[r] : static_cast<const int32_t*>(a.target)[r];
    return t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
}

// One row into its planes; `vec`: 16-byte loads are possible.  Loads are issued in batches before the stores that may alias them.
template <typename T>
__device__ __forceinline__ void ce_copy_row(const T* src, __nv_bfloat16* dst, int cols, int64_t stride, int64_t plane, bool vec, int lane,
                                            int lanes) {
    constexpr int B = 8;
    if (sizeof(T) == 2 && vec) {
        const uint4* s = reinterpret_cast<const uint4*>(src);
        uint4* d = reinterpret_cast<uint4*>(dst);
        const int n = cols / 8;
        for (int i0 = lane; i0 < n; i0 += lanes * B) {
            uint4 v[B];
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (i0 + lanes * b < n) v[b] = s[i0 + lanes * b];
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (i0 + lanes * b < n) d[i0 + lanes * b] = v[b];
        }
        return;
    }
    uint32_t* d = reinterpret_cast<uint32_t*>(dst);    // two columns at a time: the stride is a multiple of 8
    const int n = static_cast<int>(stride / 2);
    const int64_t p32 = plane / 2;
    for (int i0 = lane; i0 < n; i0 += lanes * B) {
        T v[B][2];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int c = 2 * (i0 + lanes * b);
            v[b][0] = c < cols ? src[c] : T(0.f);
            v[b][1] = c + 1 < cols ? src[c + 1] : T(0.f);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int i = i0 + lanes * b;
            if (i >= n) continue;
            if (sizeof(T) == 2) {
                d[i] = (__float_as_uint(Vec<T>::load1(&v[b][0])) >> 16) | (__float_as_uint(Vec<T>::load1(&v[b][1])) & 0xffff0000u);
            } else {
                uint32_t h0, m0, l0, h1, m1, l1;
                split3(Vec<T>::load1(&v[b][0]), h0, m0, l0);
                split3(Vec<T>::load1(&v[b][1]), h1, m1, l1);
                d[i] = (h0 >> 16) | h1;
                d[p32 + i] = (m0 >> 16) | m1;
                d[2 * p32 + i] = (l0 >> 16) | l1;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) ce_rows_kernel(const CeRowsArgs a) {
    __shared__ int warp_count[8];
    __shared__ int where[kRowsBlock];
    __shared__ float scale_of[8];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t plane = a.rows_pad * a.stride;
    const int end = static_cast<int>(blockIdx.x) - (static_cast<int>(gridDim.x) - kRowsEnd);   // >= 0: one of the last blocks
    const int64_t r0 = end >= 0 ? a.rows : static_cast<int64_t>(blockIdx.x) * a.per_block;
    int n = 0;
#pragma unroll 4
    for (int64_t r = threadIdx.x; r < r0; r += 256) n += ce_target(a, r) >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) warp_count[warp] = n;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < 8; ++w) base += warp_count[w];
    if (end >= 0) {
        if (a.lse) {                                   // rows of dW's sum behind the last one, up to a whole slab, are zeros
            const int stop = (base + kTK - 1) / kTK * kTK;
            for (int p = 0; p < a.planes; ++p)
                for (int i = base + end; i < stop; i += kRowsEnd) {
                    uint4* d = reinterpret_cast<uint4*>(a.dst + p * plane + i * a.stride);
                    for (int64_t c = threadIdx.x; c < a.stride / 8; c += 256) d[c] = make_uint4(0, 0, 0, 0);
                }
        }
        if (end > 0) return;
        if (threadIdx.x == 0) *a.count = base;
        if (a.lse) {                                   // the largest |gy| of the rows that take part, 1 where that is no scale
            float top = 0.f;
#pragma unroll 4
            for (int64_t r = threadIdx.x; r < a.rows; r += 256)
                if (ce_target(a, r) >= 0) top = fmaxf(top, fabsf(a.gy[r]));
            top = warp_max(top);
            if (lane == 0) scale_of[warp] = top;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int w = 1; w < 8; ++w) top = fmaxf(top, scale_of[w]);
                *a.gy_scale = top > 0x1p-100f && top < 0x1p100f ? top : 1.f;
            }
        }
        return;
    }
    if (threadIdx.x < 32) {
        const int64_t r = r0 + threadIdx.x;
        const bool mine = threadIdx.x < a.per_block && r < a.rows;
        const int t = mine ? ce_target(a, r) : -1;
        const uint32_t mask = __ballot_sync(0xffffffffu, t >= 0);
        const int at = base + __popc(mask & ((1u << threadIdx.x) - 1));
        where[threadIdx.x] = t >= 0 ? at : -1;
        if (t >= 0) {
            a.row_of[at] = static_cast<int>(r);
            a.target_of[at] = t;
            if (a.lse) {
                a.lse_of[at] = a.lse[r];
                a.gy_of[at] = a.gy[r];
            }
        } else if (mine && a.loss) {
            a.loss[r] = 0.f;
            a.lse_out[r] = 0.f;
        }
        if (mine) a.pos_of[r] = t >= 0 ? at : -1;
    }
    __syncthreads();
    const bool vec = sizeof(T) == 2 && a.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    // a warp per row, or the block where it has one row only
    const bool alone = a.per_block == 1;
    for (int i = alone ? 0 : warp; i < a.per_block; i += 8)
        if (where[i] >= 0)
            ce_copy_row(static_cast<const T*>(a.x) + (r0 + i) * a.cols, a.dst + where[i] * a.stride, a.cols, a.stride, plane, vec,
                        alone ? threadIdx.x : lane, alone ? 256 : 32);
}

// Rows [row0, row0 + rows) of w into dst [planes][rows_pad][stride]: what W needs where TMA cannot read it as it is.  LONG: a warp per row.
// Else a thread takes pairs of columns wherever they lie, so that short rows fill the warps too, at the price of a division per pair.
template <typename T, bool LONG>
__global__ void __launch_bounds__(256) ce_pack_kernel(const T* w, int64_t rows, int cols, __nv_bfloat16* dst, int64_t rows_pad, int64_t stride) {
    pdl_wait();
    pdl_trigger();
    if constexpr (LONG) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + warp; r < rows; r += static_cast<int64_t>(gridDim.x) * 8)
            ce_copy_row(w + r * cols, dst + r * stride, cols, stride, rows_pad * stride, false, lane, 32);
        return;
    }
    constexpr int B = 8;
    const uint32_t per_row = static_cast<uint32_t>(stride / 2);
    const int64_t total = rows * per_row, step = static_cast<int64_t>(gridDim.x) * 256, p32 = rows_pad * per_row;
    uint32_t* d = reinterpret_cast<uint32_t*>(dst);
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i0 < total; i0 += step * B) {
        T v[B][2];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int64_t i = i0 + b * step;
            const uint32_t r = static_cast<uint32_t>(i < total ? i : 0) / per_row;      // a piece has less than 2^32 pairs
            const int c = 2 * static_cast<int>(static_cast<uint32_t>(i < total ? i : 0) - r * per_row);
            const T* src = w + static_cast<int64_t>(r) * cols + c;
            v[b][0] = i < total && c < cols ? src[0] : T(0.f);
            v[b][1] = i < total && c + 1 < cols ? src[1] : T(0.f);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int64_t i = i0 + b * step;
            if (i >= total) continue;
            if (sizeof(T) == 2) {
                d[i] = (__float_as_uint(Vec<T>::load1(&v[b][0])) >> 16) | (__float_as_uint(Vec<T>::load1(&v[b][1])) & 0xffff0000u);
            } else {
                uint32_t h0, m0, l0, h1, m1, l1;
                split3(Vec<T>::load1(&v[b][0]), h0, m0, l0);
                split3(Vec<T>::load1(&v[b][1]), h1, m1, l1);
                d[i] = (h0 >> 16) | h1;
                d[p32 + i] = (m0 >> 16) | m1;
                d[2 * p32 + i] = (l0 >> 16) | l1;
            }
        }
    }
}

// ---------------------------------------------------------------- the epilogue's stores
// Eight 16-byte words of a row (thread = row) into the next swizzled box, then one lane sends it off: send(box).
template <int BOXES, typename F>
__device__ __forceinline__ void ce_send(uint8_t* boxes, int& turn, const uint4 (&w)[8], int lane, F send) {
    tma_store_wait_read<BOXES - 1>();                  // the lane that sent this box last: it has been read
    __syncwarp();
    uint8_t* box = boxes + turn * kBoxBytes;
    if (++turn == BOXES) turn = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = w[q];
    fence_async();
    __syncwarp();
    if (lane == 0) {
        send(box);
        tma_store_commit();
    }
}

// A staged piece of dw [rows][stride] (S: bf16, or fp32 that is still to be rounded or added) to its place [rows][cols].  LONG: a warp per row;
// 16-bit rows that start between two words are written as a single element and pairs.  Else element by element, wherever they lie.
template <typename S, typename T, bool LONG>
__global__ void __launch_bounds__(256) ce_unpack_kernel(const S* src, int64_t rows, int cols, int64_t stride, T* dw, int add) {
    constexpr int B = 8;
    pdl_wait();
    pdl_trigger();
    if constexpr (!LONG) {
        const int64_t total = rows * cols, step = static_cast<int64_t>(gridDim.x) * 256;
        for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i0 < total; i0 += step * B) {
            float v[B], o[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int64_t i = i0 + b * step;
                const uint32_t at = static_cast<uint32_t>(i < total ? i : 0), r = at / cols;   // a piece has less than 2^32 elements
                v[b] = Vec<S>::load1(src + static_cast<int64_t>(r) * stride + (at - r * cols));
                o[b] = add ? Vec<T>::load1(dw + at) : 0.f;
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (i0 + b * step < total) Vec<T>::store1(dw + i0 + b * step, add ? __fadd_rn(v[b], o[b]) : v[b]);
        }
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + warp; r < rows; r += static_cast<int64_t>(gridDim.x) * 8) {
        const S* s = src + r * stride;
        T* d = dw + r * cols;
        const int odd = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(d) & 2) ? 1 : 0;
        if (odd && lane == 0) {
            const float v = Vec<S>::load1(s);
            Vec<T>::store1(d, add ? __fadd_rn(v, Vec<T>::load1(d)) : v);
        }
        for (int c0 = odd + 2 * lane; c0 < cols; c0 += 64 * B) {
            float v[B][2], o[B][2];
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = c0 + 64 * b + e;
                    v[b][e] = c < cols ? Vec<S>::load1(s + c) : 0.f;
                    o[b][e] = add && c < cols ? Vec<T>::load1(d + c) : 0.f;
                }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int c = c0 + 64 * b;
                if (c >= cols) continue;
                const float x = add ? __fadd_rn(v[b][0], o[b][0]) : v[b][0], y = add ? __fadd_rn(v[b][1], o[b][1]) : v[b][1];
                if (sizeof(T) == 2 && c + 1 < cols) {
                    *reinterpret_cast<uint32_t*>(d + c) = pack_bf16x2(x, y);
                } else {
                    Vec<T>::store1(d + c, x);
                    if (c + 1 < cols) Vec<T>::store1(d + c + 1, y);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- the products
// PHASE 0: logits into pairs.  1: logits into g, one plane.  3: g in three planes.  2: dh and dw, one or both.
template <int CG, int PHASE>
__global__ void __launch_bounds__(kCeThreads, 1) ce_gemm_kernel(const __grid_constant__ CeArgs a) {
    typedef CeRing<CG, PHASE> R;
    constexpr int kStages = R::kStages;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 1 ? 0 : static_cast<int>(cluster_rank());
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8 * CG);
        }
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 2) tmem_alloc<CG>(&tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_barrier();                    // the leader's barriers are ready before the other CTA's copies arrive
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    pdl_wait();                                        // barriers and tensor memory were set up under the kernel before
    pdl_trigger();
    const int count = *a.count;
    const CeShape s0(a.job[0], count, kTM * CG), s1(a.job[a.jobs - 1], count, kTM * CG);
    const int total = s0.tiles + (PHASE == 2 && a.jobs > 1 ? s1.tiles : 0);
    const int first = blockIdx.x / CG, stride = gridDim.x / CG;

    if (warp == 0) {
        if (elect_one()) {
            const uint32_t full0 = leader_address(&full[0]);
            int fills = 0, s = 0;                      // s: slot of the ring
            uint32_t wrap = 1;                         // parity of the slot's previous use
            bool ok = true;
            for (int t = first; t < total && ok; t += stride) {
                const int j = PHASE != 2 || t < s0.tiles ? 0 : 1;
                const CeTile tile = ce_tile(a.job[j], j ? s1 : s0, j ? t - s0.tiles : t);
                // everything that the inner loop needs, in registers: one thread feeds the tensor cores of the CTA, and a
                // division or a load from the argument's memory per slab cost it more than the slab's products take
                const bool a_mn = a.job[j].a_mn, b_mn = a.job[j].b_mn;
                const int share = a.job[j].tn / CG;                     // columns of B that this CTA holds
                const int box = a.job[j].b_box, boxes = share / box;
                const int am = (a_mn ? a.job[j].a_row0 : 0) + tile.m0 + rank * kTM;
                const int b_row0 = a.job[j].b_row0, bn = tile.n0 + rank * share;
                const uint32_t bytes = CG * (R::kBytesA + share * kTK * 2);
                const CUtensorMap* ma = &a.A[j];
                const CUtensorMap* mb = &a.B[j];
                const int products = a.job[j].a_planes3 ? 6 : 1, blocks = tile.iters / products;
                for (int p = 0; p < products && ok; ++p) {
                    int pa = 0, pb = 0;
                    if (products == 6) plane_pair(p, pa, pb);
                    int k = tile.k0;
                    for (int it = 0; it < blocks; ++it, ++fills, k += kTK) {
                        if (fills >= kStages && !wait_or_abort(&empty[s], wrap, &abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        uint8_t* sa = ring + s * R::kStageBytes;
                        uint8_t* sb = sa + R::kBytesA;
                        const uint32_t bar = CG == 1 ? smem_u32(&full[s]) : full0 + s * 8;
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);     // both CTAs' bytes
                        if (a_mn) {
#pragma unroll
                            for (int b = 0; b < kTM / 64; ++b) tma_load_3d<CG>(sa + b * (kTK * 128), ma, am + b * 64, k, pa, bar);
                        } else {
                            tma_load_3d<CG>(sa, ma, k, am, pa, bar);
                        }
                        if (b_mn) {
                            for (int b = 0; b < boxes; ++b) tma_load_3d<CG>(sb + b * (kTK * 128), mb, bn + b * 64, b_row0 + k, pb, bar);
                        } else {
                            for (int b = 0; b < boxes; ++b) tma_load_3d<CG>(sb + b * box * 128, mb, k, b_row0 + bn + b * box, pb, bar);
                        }
                        if (++s == kStages) {
                            s = 0;
                            wrap ^= 1;
                        }
                    }
                }
            }
            if (!ok) {                                 // the copies still in flight land before the CTA leaves
                if (CG == 1)
                    for (int f = fills > kStages ? fills - kStages : 0; f < fills; ++f) mbar_wait_bounded(&full[f % kStages], (f / kStages) & 1);
                else
                    for (int i = 0; i < 2000; ++i) __nanosleep(1000);   // counted on the leader's barrier: given two milliseconds
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int n = 0, s = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t ring0 = smem_u32(ring);
            const uint64_t desc = smem_desc(0, kTK * 128);
            for (int t = first; t < total && ok; t += stride, ++n) {
                const int j = PHASE != 2 || t < s0.tiles ? 0 : 1;
                const CeTile tile = ce_tile(a.job[j], j ? s1 : s0, j ? t - s0.tiles : t);
                const uint32_t idesc = mma_idesc(kTM * CG, a.job[j].tn, a.job[j].a_mn, a.job[j].b_mn);
                const uint32_t step_a = (a.job[j].a_mn ? 2048 : 32) >> 4, step_b = (a.job[j].b_mn ? 2048 : 32) >> 4;
                const int acc = n & 1, iters = tile.iters;
                if (n >= 2 && !wait_or_abort(&acc_empty[acc], (n / 2 - 1) & 1, &abort_flag, a.status)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * kTN;
                for (int it = 0; it < iters; ++it) {
                    if (!wait_or_abort(&full[s], phase, &abort_flag, a.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = desc + ((ring0 + s * R::kStageBytes) >> 4), db = da + (R::kBytesA >> 4);
#pragma unroll
                    for (int k = 0; k < kTK / 16; ++k) mma_bf16<CG>(d, da + k * step_a, db + k * step_b, idesc, it > 0 || k > 0);
                    mma_commit<CG>(&empty[s]);
                    if (++s == kStages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                mma_commit<CG>(&acc_full[acc]);
            }
            if (!ok) {
                mma_commit<CG>(&drained);
                mbar_wait_bounded(&drained, 0);
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, part = (warp - 4) >> 2;     // lanes 32 * quarter.., the part-th half of the columns
        [[maybe_unused]] uint8_t* boxes = ring + kStages * R::kStageBytes + (warp - 4) * R::kBoxes * kBoxBytes;
        [[maybe_unused]] int turn = 0;
        const uint32_t acc_empty_at[2] = {leader_address(&acc_empty[0]), leader_address(&acc_empty[1])};
        int n = 0;
        for (int t = first; t < total; t += stride, ++n) {
            const int j = PHASE != 2 || t < s0.tiles ? 0 : 1;
            const CeJob& job = a.job[j];
            const CeShape& sh = j ? s1 : s0;
            const CeTile tile = ce_tile(job, sh, j ? t - s0.tiles : t);
            const int acc = n & 1, width = job.tn >> 1;
            const int row0 = tile.m0 + rank * kTM + quarter * 32, row = row0 + lane;
            const bool live = row < sh.m;
            const int c0 = tile.n0 + part * width;
            const int c1 = c0 + width < sh.n ? c0 + width : sh.n;          // this thread's columns that exist
            if (!wait_or_abort(&acc_full[acc], (n / 2) & 1, &abort_flag, a.status)) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * kTN + part * width + (static_cast<uint32_t>(quarter * 32) << 16);
            [[maybe_unused]] const bool empty_sum = tile.iters == 0;       // nothing was multiplied: the accumulators hold something old
            if constexpr (PHASE == 0) {
                float m = -INFINITY, s = 0.f;
                const int tgt = live ? a.target[row] - a.col0 : -1;
                for (int c = c0; c < c0 + width; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
                    const int left = c1 - c;
                    if (left < 32) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= left) v[e] = -INFINITY;
                    }
                    if (tgt >= c && tgt < c1 && tgt < c + 32) {
                        float zt = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (tgt == c + e) zt = v[e];
                        a.z_target[row] = zt;
                    }
                    online_add(v, 1.f, m, s);
                }
                if (live) a.pairs[row * a.n_pairs + a.pair0 + c0 / width] = make_float2(m, s);
            } else if constexpr (PHASE == 1 || PHASE == 3) {
                // columns behind the last one are zeros up to the tile's end: dh and dW read whole slabs of 64
                const int tgt = live ? a.target[row] - a.col0 : -1;
                const float lse = live ? a.lse[row] : 0.f, gy = live ? __fdiv_rn(a.gy[row], *a.gy_scale) : 0.f;
#pragma unroll 1
                for (int c = c0; c < c0 + width; c += 64) {
#pragma unroll 1
                    for (int p = 0; p < (PHASE == 3 ? 3 : 1); ++p) {
                        uint4 w[8];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int ch = c + 32 * half;
                            float v[32];
                            tmem_load32(d + (ch - c0), v);
                            const bool here = tgt >= ch && tgt < c1 && tgt < ch + 32;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                float q = ex2f(__fmul_rn(__fsub_rn(v[e], lse), kLog2e));
                                if (here && tgt == ch + e) q = __fsub_rn(q, 1.f);
                                v[e] = live && ch + e < c1 ? __fmul_rn(gy, q) : 0.f;
                            }
                            if (PHASE == 1 && here) {
                                float g = 0.f;
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (tgt == ch + e) g = v[e];
                                a.left_over[row] = __fsub_rn(g, __bfloat162float(__float2bfloat16_rn(g)));
                            }
                            if (PHASE == 3) {          // this plane's 16 bits of each
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    uint32_t hi, mid, lo;
                                    split3(v[e], hi, mid, lo);
                                    v[e] = __uint_as_float(p == 0 ? hi : p == 1 ? mid : lo);
                                }
                            }
#pragma unroll
                            for (int q = 0; q < 4; ++q) w[4 * half + q] = Unit<__nv_bfloat16, 16>::pack(v + 8 * q);
                        }
                        ce_send<R::kBoxes>(boxes, turn, w, lane, [&](const uint8_t* box) { tma_store_3d(&a.out[j], box, c, row0, p); });
                    }
                }
            } else if (job.epi == kEpiDh || a.dw_out != kDwScalar) {
                // rows behind the last one of dh's parts are scratch; those of dW are cut off by the map
                const bool dh = job.epi == kEpiDh, staged = !dh && a.dw_out == kDwStaged, f32 = dh || a.dw_f32;
                const float scale = dh ? 1.f : *a.gy_scale;
                const int step = f32 ? 32 : 64, y = dh || staged ? row0 : a.col0 + row0;
                // a box that starts behind the last row has nothing to write
#pragma unroll 1
                for (int c = c0; c < c1 && row0 < sh.m; c += step) {
                    uint4 w[8];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (f32 && half) break;
                        float v[32];
                        tmem_load32(d + (c - c0) + 32 * half, v);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = empty_sum ? 0.f : __fmul_rn(scale, v[e]);
                        if (f32) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) w[q] = Unit<float, 16>::pack(v + 4 * q);
                        } else {
                            if (a.dw_add && !staged && live) {
                                const uint4* o = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.dw) +
                                                                                static_cast<int64_t>(y + lane) * a.hidden + c + 32 * half);
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    if (c + 32 * half + 8 * q < c1) {
                                        float f[8];
                                        Unit<__nv_bfloat16, 16>::unpack(o[q], f);
#pragma unroll
                                        for (int e = 0; e < 8; ++e) v[8 * q + e] = __fadd_rn(v[8 * q + e], f[e]);
                                    }
                            }
#pragma unroll
                            for (int q = 0; q < 4; ++q) w[4 * half + q] = Unit<__nv_bfloat16, 16>::pack(v + 8 * q);
                        }
                    }
                    ce_send<R::kBoxes>(boxes, turn, w, lane, [&](const uint8_t* box) {
                        if (dh ? a.dh_add : (a.dw_add && f32 && !staged)) tma_add_3d(&a.out[j], box, c, y, tile.split);
                        else tma_store_3d(&a.out[j], box, c, y, tile.split);
                    });
                }
            } else {                                   // a base that TMA cannot write to: element by element
                const int64_t at = static_cast<int64_t>(a.col0 + row) * a.hidden;
                const float scale = *a.gy_scale;
#pragma unroll 1
                for (int c = c0; c < c1; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        if (!live || c + e >= c1) continue;
                        const float x = empty_sum ? 0.f : __fmul_rn(scale, v[e]);
                        if (a.dw_f32) {
                            float* o = static_cast<float*>(a.dw) + at + c + e;
                            *o = a.dw_add ? __fadd_rn(x, *o) : x;
                        } else {
                            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.dw) + at + c + e;
                            *o = __float2bfloat16_rn(a.dw_add ? __fadd_rn(x, __bfloat162float(*o)) : x);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) mbar_arrive(&acc_empty[acc]);
                else mbar_arrive_cluster(acc_empty_at[acc]);
            }
        }
        tma_store_wait();                              // this thread's boxes have been written
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_barrier();                    // neither CTA leaves while the other may still reach its memory
    tc_fence_after();
    if (warp == 2) tmem_free<CG>(tmem, 512);
}

// ---------------------------------------------------------------- joining
// lse and loss of the rows that take part, W warps per row (one where rows fill the GPU, eight where they are few).  The loss is a
// difference of two numbers of the size of the logits, and the tensor cores cut (not round) every partial sum: z_target there was off by
// 1.5e-5 at 4096 terms of one sign.  So z_target is computed once more, in fp32, and takes its own place in the sum of exponentials as
// well: the two agree, and the loss of a target with p near one is not a difference of two errors.
template <typename T, int W>
__global__ void __launch_bounds__(256) ce_join_kernel(const float2* pairs, int n, int64_t n_pairs, const int* count, const float* z_target,
                                                      const int* target_of, const int* row_of, const T* h, const T* w, int hidden, float* loss,
                                                      float* lse) {
    __shared__ float part[8][3];
    // what the dot product reads was written before the products started: it runs under their end
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = blockIdx.x * (8 / W) + warp / W, me = threadIdx.x % (32 * W);
    const bool live = i < *count;                      // the same for all threads of the block where W > 1
    typedef Unit<T, 16> U;
    float z = 0.f;
    int r = 0;
    if (live) {
        r = row_of[i];
        const T* hr = h + static_cast<int64_t>(r) * hidden;
        const T* wr = w + static_cast<int64_t>(target_of[i]) * hidden;
        if (hidden % U::N == 0 && ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(w)) & 15) == 0) {
            const uint4* hv = reinterpret_cast<const uint4*>(hr);
            const uint4* wv = reinterpret_cast<const uint4*>(wr);
#pragma unroll 4
            for (int c = me; c < hidden / U::N; c += 32 * W) {
                float f[U::N], g[U::N];
                U::unpack(hv[c], f);
                U::unpack(wv[c], g);
#pragma unroll
                for (int e = 0; e < U::N; ++e) z = __fmaf_rn(f[e], g[e], z);
            }
        } else {
#pragma unroll 8
            for (int c = me; c < hidden; c += 32 * W) z = __fmaf_rn(Vec<T>::load1(hr + c), Vec<T>::load1(wr + c), z);
        }
    }
    pdl_wait();
    pdl_trigger();
    float m = -INFINITY, s = 0.f;
    if (live) {
#pragma unroll 4
        for (int p = me; p < n; p += 32 * W) {
            const float2 q = pairs[i * n_pairs + p];
            join_pair(m, s, q.x, q.y);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        z = __fadd_rn(z, __shfl_xor_sync(0xffffffffu, z, o));
        const float mb = __shfl_xor_sync(0xffffffffu, m, o), sb = __shfl_xor_sync(0xffffffffu, s, o);
        join_pair(m, s, mb, sb);
    }
    if (W > 1) {
        if (lane == 0) {
            part[warp][0] = z;
            part[warp][1] = m;
            part[warp][2] = s;
        }
        __syncthreads();
        if (warp) return;
        for (int q = 1; q < W; ++q) {
            z = __fadd_rn(z, part[q][0]);
            join_pair(m, s, part[q][1], part[q][2]);
        }
    }
    if (lane || !live) return;
    s = __fadd_rn(s, __fsub_rn(exp2f(__fmul_rn(__fsub_rn(z, m), kLog2e)), exp2f(__fmul_rn(__fsub_rn(z_target[i], m), kLog2e))));
    const float l = __fadd_rn(m, logf(s));
    lse[r] = l;
    loss[r] = __fsub_rn(l, z);
}

// Few tiles and a long sum: the logits as fp32 parts [splits][rows_pad][stride] of K, each part a CTA's.  This is the join for them: a block
// per row adds the parts, takes the maximum and the sum, and goes on as ce_join_kernel does.
template <typename T>
__global__ void __launch_bounds__(1024) ce_join_parts_kernel(const float* parts, int splits, int64_t rows_pad, int64_t stride, int vocab,
                                                            const int* count, const int* target_of, const int* row_of, const T* h, const T* w,
                                                            int hidden, float* loss, float* lse) {
    __shared__ float red[32][3];
    __shared__ float z_there;
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (i >= *count) return;
    const int r = row_of[i], target = target_of[i];
    float z = 0.f;
    const T* hr = h + static_cast<int64_t>(r) * hidden;
    const T* wr = w + static_cast<int64_t>(target) * hidden;
#pragma unroll 4
    for (int c = threadIdx.x; c < hidden; c += blockDim.x) z = __fmaf_rn(Vec<T>::load1(hr + c), Vec<T>::load1(wr + c), z);
    float m = -INFINITY, s = 0.f;
    const float* p = parts + i * stride;
    for (int c = threadIdx.x * 4; c < vocab; c += 4 * blockDim.x) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < splits; ++k) {
            const float4 q = *reinterpret_cast<const float4*>(p + k * rows_pad * stride + c);
            v[0] = __fadd_rn(v[0], q.x);
            v[1] = __fadd_rn(v[1], q.y);
            v[2] = __fadd_rn(v[2], q.z);
            v[3] = __fadd_rn(v[3], q.w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (c + e == target) z_there = v[e];
            if (c + e >= vocab) v[e] = -INFINITY;
        }
        online_add(v, 1.f, m, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        z = __fadd_rn(z, __shfl_xor_sync(0xffffffffu, z, o));
        const float mb = __shfl_xor_sync(0xffffffffu, m, o), sb = __shfl_xor_sync(0xffffffffu, s, o);
        join_pair(m, s, mb, sb);
    }
    if (lane == 0) {
        red[warp][0] = z;
        red[warp][1] = m;
        red[warp][2] = s;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int q = 1; q < static_cast<int>(blockDim.x >> 5); ++q) {
        z = __fadd_rn(z, red[q][0]);
        join_pair(m, s, red[q][1], red[q][2]);
    }
    s = __fadd_rn(s, __fsub_rn(exp2f(__fmul_rn(__fsub_rn(z, m), kLog2e)), exp2f(__fmul_rn(__fsub_rn(z_there, m), kLog2e))));
    const float l = __fadd_rn(m, logf(s));
    lse[r] = l;
    loss[r] = __fsub_rn(l, z);
}

// g of the same parts, what the epilogue of PHASE 1 (3) writes; zeros up to whole slabs of rows and columns.
__global__ void __launch_bounds__(256) ce_g_parts_kernel(const float* parts, int splits, int64_t rows_pad, int64_t stride, int vocab,
                                                         const int* count, const int* target_of, const float* lse_of, const float* gy_of,
                                                         const float* gy_scale, __nv_bfloat16* g, int64_t g_stride, int planes, float* left_over) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 2, n = *count;
    if (i >= (n + kTK - 1) / kTK * kTK || c >= g_stride) return;
    float v[2] = {0.f, 0.f};
    if (i < n) {
        const float lse = lse_of[i], gy = __fdiv_rn(gy_of[i], *gy_scale);
        const int target = target_of[i];
        const float* p = parts + i * stride + c;
        float2 z = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < splits; ++k) z = add2(z, *reinterpret_cast<const float2*>(p + k * rows_pad * stride));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float q = ex2f(__fmul_rn(__fsub_rn(e ? z.y : z.x, lse), kLog2e));
            if (target == c + e) q = __fsub_rn(q, 1.f);
            v[e] = c + e < vocab ? __fmul_rn(gy, q) : 0.f;
            if (planes == 1 && target == c + e) left_over[i] = __fsub_rn(v[e], __bfloat162float(__float2bfloat16_rn(v[e])));
        }
    }
    uint32_t* o = reinterpret_cast<uint32_t*>(g + i * g_stride + c);
    if (planes == 1) {
        *o = pack_bf16x2(v[0], v[1]);
    } else {
        const int64_t plane = rows_pad * g_stride / 2;
        uint32_t h0, m0, l0, h1, m1, l1;
        split3(v[0], h0, m0, l0);
        split3(v[1], h1, m1, l1);
        o[0] = (h0 >> 16) | h1;
        o[plane] = (m0 >> 16) | m1;
        o[2 * plane] = (l0 >> 16) | l1;
    }
}

// dh of every row: the parts summed in order, what rounding took from g at the target times that row of W, rounded once; zeros where
// the row took no part.  A thread takes four neighbouring columns.
template <typename T>
__global__ void __launch_bounds__(256) ce_dh_kernel(const float* parts, int splits, int64_t rows_pad, int64_t stride, const int* pos_of,
                                                    const int* target_of, const float* left_over, const float* gy_scale, const T* w, T* dh,
                                                    int64_t rows, int hidden) {
    pdl_wait();
    pdl_trigger();
    const float scale = *gy_scale;
    const int quads = (hidden + 3) / 4;
    const bool vec = sizeof(T) == 4 ? hidden % 4 == 0 && (reinterpret_cast<uintptr_t>(dh) & 15) == 0
                                    : hidden % 4 == 0 && (reinterpret_cast<uintptr_t>(dh) & 7) == 0;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const int p = pos_of[r];
        const T* wr = p >= 0 && left_over ? w + static_cast<int64_t>(target_of[p]) * hidden : nullptr;
        const float left = wr ? left_over[p] : 0.f;
        for (int q = blockIdx.x * 256 + threadIdx.x; q < quads; q += gridDim.x * 256) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            if (p >= 0) {
#pragma unroll 4
                for (int k = 0; k < splits; ++k) {
                    const float4 v = *reinterpret_cast<const float4*>(parts + (k * rows_pad + p) * stride + 4 * q);
                    s[0] = __fadd_rn(s[0], v.x);
                    s[1] = __fadd_rn(s[1], v.y);
                    s[2] = __fadd_rn(s[2], v.z);
                    s[3] = __fadd_rn(s[3], v.w);
                }
                if (wr) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * q + e < hidden) s[e] = __fmaf_rn(left, Vec<T>::load1(wr + 4 * q + e), s[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __fmul_rn(scale, s[e]);
            T* o = dh + r * hidden + 4 * q;
            if (vec && sizeof(T) == 4) {
                *reinterpret_cast<float4*>(o) = make_float4(s[0], s[1], s[2], s[3]);
            } else if (vec) {
                *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * q + e < hidden) Vec<T>::store1(o + e, s[e]);
            }
        }
    }
}

}  // namespace agb
