// linear_ce.cuh -- softmax cross entropy taken straight from the hidden states, the logits never kept.
//   z = h W';  lse_t = log sum_v exp z_tv;  loss_t = lse_t - z_t,target(t)
//   g_tv = gy_t * (exp(z_tv - lse_t) - [v = target(t)]);  dh = g W;  dW = g' h
// Rows whose target names no column take no part: they are left out when h is laid out for the products (rows in order, no gaps), so
// they cost nothing and what they hold (padding, NaN) reaches nothing.
//
// One persistent kernel does all the products.  Tiles of 128 x 256 with fp32 accumulators in tensor memory (two of them: the
// epilogue of a tile runs under the products of the next), operands in 64-wide slabs through a ring of TMA loads.  Forward: the
// epilogue turns a tile of logits into a (max, sum of exp) pair per row and half tile; a small kernel joins the pairs.  Backward,
// piece by piece of the vocabulary: the logits again with an epilogue that writes g in 16 bits, then dh += g W and dW = g' h in one
// launch.  dh is kept in fp32 over the pieces; where rows are few the vocabulary axis is cut between CTAs and the parts are summed
// in order.
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
template <int CG>
struct CeRing {
    static constexpr int kStages = CG == 1 ? 4 : 6;
    static constexpr int kBytesA = kTM * kTK * 2, kBytesB = kTN / CG * kTK * 2;
    static constexpr int kStageBytes = kBytesA + kBytesB;
    static constexpr int kSmem = kStages * kStageBytes + 1024;
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
    int tn;                            // columns of a tile: 256, 128 or 64 (a pair: 256)
    int b_box;                         // rows of B's TMA box: 64 where B is MN-major, else 128 or a CTA's whole share
};
constexpr int kMGroup = 4096;

struct CeArgs {
    CUtensorMap A[2], B[2];
    CeJob job[2];
    int jobs;
    const int* count;                  // rows that take part
    int* status;
    int64_t rows_pad;                  // row stride of the per-row arrays below
    // pairs
    float2* pairs;                     // [half tiles of the vocabulary][rows_pad]
    float* z_target;                   // [rows_pad]
    const int* target;                 // [rows_pad]
    int pair0;                         // first half tile of this piece
    int col0, vocab;                   // first column of the piece
    // g
    const float *lse, *gy;             // [rows_pad]
    __nv_bfloat16* g;                  // [planes][rows_pad][g_stride]
    int64_t g_stride;
    int planes;
    // dh: fp32 parts [split][rows_pad][dh_stride]
    float* dh;
    int64_t dh_stride;
    int dh_add;                        // 0 the first piece: write, 1 add
    // dw
    void* dw;
    int hidden, dw_add, dw_f32;
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
// A block takes 32 rows; it counts the targets before its own to know where they go.
struct CeRowsArgs {
    const void* x;
    const void* target;
    int target64;
    int64_t rows;
    int cols, vocab, planes;
    __nv_bfloat16* dst;
    int64_t rows_pad, stride;
    int* count;
    int* row_of;                       // [rows_pad]: the row that went there
    int* pos_of;                       // [rows]: where the row went, or -1
    int* target_of;                    // [rows_pad]
    const float *lse, *gy;             // backward: [rows]; NULL in the forward
    float *lse_of, *gy_of;
    float *loss, *lse_out;             // forward: rows that take no part get 0
};
constexpr int kRowsBlock = 32;

__device__ __forceinline__ int ce_target(const CeRowsArgs& a, int64_t r) {
    const int64_t t = a.target64 ? static_cast<const int64_t*>(a.target)[r] : static_cast<const int32_t*>(a.target)[r];
    return t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
}

// One row into its planes; `vec`: 16-byte loads are possible.
template <typename T>
__device__ __forceinline__ void ce_copy_row(const T* src, __nv_bfloat16* dst, int cols, int64_t stride, int64_t plane, bool vec, int lane,
                                            int lanes) {
    if (sizeof(T) == 2) {
        if (vec) {
            const uint4* s = reinterpret_cast<const uint4*>(src);
            uint4* d = reinterpret_cast<uint4*>(dst);
            for (int i = lane; i < cols / 8; i += lanes) d[i] = s[i];
        } else {
            const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
            uint16_t* d = reinterpret_cast<uint16_t*>(dst);
            for (int i = lane; i < stride; i += lanes) d[i] = i < cols ? s[i] : static_cast<uint16_t>(0);
        }
    } else {
        uint16_t* d = reinterpret_cast<uint16_t*>(dst);
        for (int i = lane; i < stride; i += lanes) {
            uint32_t hi = 0, mid = 0, lo = 0;
            if (i < cols) split3(Vec<T>::load1(src + i), hi, mid, lo);
            d[i] = static_cast<uint16_t>(hi >> 16);
            d[plane + i] = static_cast<uint16_t>(mid >> 16);
            d[2 * plane + i] = static_cast<uint16_t>(lo >> 16);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) ce_rows_kernel(const CeRowsArgs a) {
    __shared__ int warp_count[8];
    __shared__ int where[kRowsBlock];
    __shared__ int last;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRowsBlock;
    int n = 0;
    for (int64_t r = threadIdx.x; r < r0; r += 256) n += ce_target(a, r) >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) warp_count[threadIdx.x >> 5] = n;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < 8; ++w) base += warp_count[w];
    if (threadIdx.x < 32) {
        const int64_t r = r0 + threadIdx.x;
        const int t = r < a.rows ? ce_target(a, r) : -1;
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
        } else if (r < a.rows && a.loss) {
            a.loss[r] = 0.f;
            a.lse_out[r] = 0.f;
        }
        if (r < a.rows) a.pos_of[r] = t >= 0 ? at : -1;
        if (threadIdx.x == 0) last = base + __popc(mask);
    }
    __syncthreads();
    const int64_t plane = a.rows_pad * a.stride;
    const bool vec = sizeof(T) == 2 && a.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < kRowsBlock; i += 8)
        if (where[i] >= 0)
            ce_copy_row(static_cast<const T*>(a.x) + (r0 + i) * a.cols, a.dst + where[i] * a.stride, a.cols, a.stride, plane, vec, lane, 32);
    if (blockIdx.x + 1 == gridDim.x) {                 // the last block knows the number of rows
        if (threadIdx.x == 0) *a.count = last;
        // rows of dW's sum behind the last one, up to a whole slab
        const int64_t stop = (static_cast<int64_t>(last) + kTK - 1) / kTK * kTK;
        for (int p = 0; a.lse && p < a.planes; ++p) {
            uint4* d = reinterpret_cast<uint4*>(a.dst + p * plane + last * a.stride);
            for (int64_t i = threadIdx.x; i < (stop - last) * a.stride / 8; i += 256) d[i] = make_uint4(0, 0, 0, 0);
        }
    }
}

// Rows [row0, row0 + rows) of w into dst [planes][rows_pad][stride]: what W needs where TMA cannot read it as it is.
template <typename T>
__global__ void __launch_bounds__(256) ce_pack_kernel(const T* w, int64_t rows, int cols, __nv_bfloat16* dst, int64_t rows_pad, int64_t stride) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + warp; r < rows; r += static_cast<int64_t>(gridDim.x) * 8)
        ce_copy_row(w + r * cols, dst + r * stride, cols, stride, rows_pad * stride, false, lane, 32);
}

// ---------------------------------------------------------------- the products
template <int CG>
__global__ void __launch_bounds__(kCeThreads, 1) ce_gemm_kernel(const __grid_constant__ CeArgs a) {
    typedef CeRing<CG> R;
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
    const int count = *a.count;
    const CeShape s0(a.job[0], count, kTM * CG), s1(a.job[a.jobs - 1], count, kTM * CG);
    const int total = s0.tiles + (a.jobs > 1 ? s1.tiles : 0);
    const int first = blockIdx.x / CG, stride = gridDim.x / CG;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full0 = leader_address(&full[0]);
            int fills = 0, s = 0;                      // s: slot of the ring
            uint32_t wrap = 1;                         // parity of the slot's previous use
            bool ok = true;
            for (int t = first; t < total && ok; t += stride) {
                const int j = t < s0.tiles ? 0 : 1;
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
        if (lane == 0 && rank == 0) {
            int n = 0, s = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t ring0 = smem_u32(ring);
            const uint64_t desc = smem_desc(0, kTK * 128);
            for (int t = first; t < total && ok; t += stride, ++n) {
                const int j = t < s0.tiles ? 0 : 1;
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
        const uint32_t acc_empty_at[2] = {leader_address(&acc_empty[0]), leader_address(&acc_empty[1])};
        int n = 0;
        for (int t = first; t < total; t += stride, ++n) {
            const int j = t < s0.tiles ? 0 : 1;
            const CeJob& job = a.job[j];
            const CeShape& sh = j ? s1 : s0;
            const CeTile tile = ce_tile(job, sh, j ? t - s0.tiles : t);
            const int acc = n & 1, width = job.tn >> 1;
            if (!wait_or_abort(&acc_full[acc], (n / 2) & 1, &abort_flag, a.status)) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * kTN + part * width + (static_cast<uint32_t>(quarter * 32) << 16);
            const int row = tile.m0 + rank * kTM + quarter * 32 + lane;
            const bool live = row < sh.m;
            const bool empty_sum = tile.iters == 0;    // nothing was multiplied: the accumulators hold something old
            const int c0 = tile.n0 + part * width;
            if (job.epi == kEpiPairs) {
                float m = -INFINITY, s = 0.f;
                const int tgt = live ? a.target[row] - a.col0 : -1;
                for (int c = c0; c < c0 + width; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
                    const int left = sh.n - c;
                    if (left < 32) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= left) v[e] = -INFINITY;
                    }
                    if (tgt >= c && tgt < c + 32) {
                        float zt = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (tgt == c + e) zt = v[e];
                        a.z_target[row] = zt;
                    }
                    online_add(v, 1.f, m, s);
                }
                if (live) a.pairs[static_cast<int64_t>(a.pair0 + c0 / width) * a.rows_pad + row] = make_float2(m, s);
            } else if (job.epi == kEpiG) {
                const int tgt = live ? a.target[row] - a.col0 : -1;
                const float lse = live ? a.lse[row] : 0.f, gy = live ? a.gy[row] : 0.f;
                __nv_bfloat16* out = a.g + row * a.g_stride;
                const int64_t plane = a.rows_pad * a.g_stride;
                for (int c = c0; c < c0 + width; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float p = ex2f(__fmul_rn(__fsub_rn(v[e], lse), kLog2e));
                        v[e] = live && c + e < sh.n ? __fmul_rn(gy, tgt == c + e ? __fsub_rn(p, 1.f) : p) : 0.f;
                    }
                    if (a.planes == 1) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *reinterpret_cast<uint4*>(out + c + 8 * q) = Unit<__nv_bfloat16, 16>::pack(v + 8 * q);
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            uint32_t h0, m0, l0, h1, m1, l1;
                            split3(v[2 * q], h0, m0, l0);
                            split3(v[2 * q + 1], h1, m1, l1);
                            *reinterpret_cast<uint32_t*>(out + c + 2 * q) = (h0 >> 16) | h1;
                            *reinterpret_cast<uint32_t*>(out + plane + c + 2 * q) = (m0 >> 16) | m1;
                            *reinterpret_cast<uint32_t*>(out + 2 * plane + c + 2 * q) = (l0 >> 16) | l1;
                        }
                    }
                }
            } else if (job.epi == kEpiDh) {
                float* out = a.dh + (static_cast<int64_t>(tile.split) * a.rows_pad + row) * a.dh_stride;
                for (int c = c0; c < c0 + width && c < sh.n; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
                    if (!live) continue;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        if (c + 4 * q >= a.dh_stride) break;          // the stride is the width rounded up to 4
                        float4* o = reinterpret_cast<float4*>(out + c + 4 * q);
                        float4 w = empty_sum ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        if (a.dh_add) {
                            const float4 old = *o;
                            w = make_float4(__fadd_rn(old.x, w.x), __fadd_rn(old.y, w.y), __fadd_rn(old.z, w.z), __fadd_rn(old.w, w.w));
                        }
                        *o = w;
                    }
                }
            } else {
                const int64_t at = static_cast<int64_t>(a.col0 + row) * a.hidden;
                const bool vec = a.hidden % 8 == 0 && (reinterpret_cast<uintptr_t>(a.dw) & 15) == 0;
                for (int c = c0; c < c0 + width && c < sh.n; c += 32) {
                    float v[32];
                    tmem_load32(d + (c - c0), v);
                    if (!live) continue;
                    if (empty_sum) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0.f;
                    }
                    if (a.dw_f32) {
                        float* o = static_cast<float*>(a.dw) + at + c;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (c + e < sh.n) {
                                if (a.dw_add) v[e] = __fadd_rn(v[e], o[e]);
                                if (!vec) o[e] = v[e];
                            }
                        if (vec) {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (c + 4 * q < sh.n) reinterpret_cast<float4*>(o)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                    } else {
                        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.dw) + at + c;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (c + e < sh.n) {
                                if (a.dw_add) v[e] = __fadd_rn(v[e], __bfloat162float(o[e]));
                                if (!vec) o[e] = __float2bfloat16_rn(v[e]);
                            }
                        if (vec) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                if (c + 8 * q < sh.n) reinterpret_cast<uint4*>(o)[q] = Unit<__nv_bfloat16, 16>::pack(v + 8 * q);
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
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_barrier();                    // neither CTA leaves while the other may still reach its memory
    tc_fence_after();
    if (warp == 2) tmem_free<CG>(tmem, 512);
}

// ---------------------------------------------------------------- joining
// lse and loss of the rows that take part, from their pairs.  blockDim (32, 8): 32 rows, eight runs of pairs.
__global__ void __launch_bounds__(256) ce_join_kernel(const float2* pairs, int n, int64_t rows_pad, const int* count, const float* z_target,
                                                      const int* row_of, float* loss, float* lse) {
    __shared__ float2 part[8][33];
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
    const bool live = i < *count;
    float m = -INFINITY, s = 0.f;
    if (live)
        for (int p = threadIdx.y; p < n; p += 8) {
            const float2 q = pairs[p * rows_pad + i];
            join_pair(m, s, q.x, q.y);
        }
    part[threadIdx.y][threadIdx.x] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.y || !live) return;
    for (int p = 1; p < 8; ++p) join_pair(m, s, part[p][threadIdx.x].x, part[p][threadIdx.x].y);
    const float l = __fadd_rn(m, logf(s));
    const int r = row_of[i];
    lse[r] = l;
    loss[r] = __fsub_rn(l, z_target[i]);
}

// dh of every row: the parts summed in order and rounded once, zeros where the row took no part.
template <typename T>
__global__ void __launch_bounds__(256) ce_dh_kernel(const float* parts, int splits, int64_t rows_pad, int64_t stride, const int* pos_of, T* dh,
                                                    int64_t rows, int hidden) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int p = pos_of[r];
        for (int c = threadIdx.x; c < hidden; c += 256) {
            float s = 0.f;
            if (p >= 0)
                for (int k = 0; k < splits; ++k) s = __fadd_rn(s, parts[(static_cast<int64_t>(k) * rows_pad + p) * stride + c]);
            Vec<T>::store1(dh + r * hidden + c, s);
        }
    }
}

}  // namespace agb
