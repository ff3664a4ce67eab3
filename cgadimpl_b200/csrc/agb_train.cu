// agb_train.cu -- the operators at the end of a model, behind the C ABI of include/agb/agb.h: LayerNorm with weight and
// bias, softmax cross entropy taken from the hidden states, distillation from a teacher's largest logits.
#define AGB_NO_STATUS_WORD
#include <nvtx3/nvToolsExt.h>

#include <type_traits>

#include "agb/agb.h"
#include "agb_internal.h"
#include "distill_topk.cuh"
#include "layernorm_affine.cuh"
#include "linear_ce.cuh"

namespace {

using agb_int::after_launch;
using agb_int::check_ptr;
using agb_int::cuda_fail;
using agb_int::fail;
typedef __nv_bfloat16 bf16;

#define AGB_TRY(expr)                  \
    do {                               \
        int s__ = (expr);              \
        if (s__ != AGB_OK) return s__; \
    } while (0)
#define AGB_CUDA(call)                                        \
    do {                                                      \
        cudaError_t e__ = (call);                             \
        if (e__ != cudaSuccess) return cuda_fail(e__, #call); \
    } while (0)

struct NvtxRange {
    explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
};
#define AGB_RANGE() NvtxRange nvtx_range__(__func__)

inline uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Launches with programmatic stream serialization (the kernels call pdl_wait() before they touch what the one before wrote) and, where
// `cluster` is above 1, in clusters.
template <typename... KArgs, typename... Args>
int launch(const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (agb_int::pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    AGB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
    return after_launch(what);
}

// ------------------------------------------------------------------ LayerNorm with weight and bias
int check_lna(int64_t rows, int64_t hidden, int dtype) {
    if (rows < 0 || hidden <= 0) return fail(AGB_ERR_INVALID_ARG, "rows=%lld hidden=%lld", (long long)rows, (long long)hidden);
    if (dtype != AGB_F32 && dtype != AGB_BF16) return fail(AGB_ERR_UNSUPPORTED, "dtype %d (only AGB_F32, AGB_BF16)", dtype);
    if (hidden > (1LL << 30)) return fail(AGB_ERR_UNSUPPORTED, "hidden %lld too large", (long long)hidden);
    return AGB_OK;
}

// The widest unit that divides the rows and all pointers: 16 bytes, 4 or the element.
inline int unit_bytes(uintptr_t all, int64_t row_bytes, int elem) {
    const uintptr_t m = all | static_cast<uintptr_t>(row_bytes);
    return m % 16 == 0 ? 16 : (m % 4 == 0 ? 4 : elem);
}

// Threads per row for `units` units at `upt` per thread: a power of two up to a warp (one unit each), else whole warps; 0: too many.
inline int threads_per_row(int64_t units, int upt, int limit) {
    if (units <= 32 && upt == 1) {
        int g = 1;
        while (g < units) g *= 2;
        return g;
    }
    const int64_t g = ceil_div(units, 32LL * upt) * 32;
    return g > limit ? 0 : static_cast<int>(g);
}
inline int64_t grid_for(int64_t rows, int G, int block, int sms, int per_sm) {
    const int64_t want = ceil_div(rows, G <= 32 ? block / G : 1), cap = static_cast<int64_t>(sms) * per_sm;
    return want < cap ? want : cap;
}

constexpr int kLnaRuns = 64;        // wide rows: runs of rows of the column sums, each a partial row
constexpr int kLnaCtas = 4;         // most CTAs per SM of the ring kernel
// Partial rows that a workspace has room for: four CTAs on each of 160 SMs, two where a row is long.
int64_t lna_partials(int64_t rows, int64_t hidden) {
    const int64_t most = hidden <= 2048 ? 640 : 320;
    return rows < 1 ? 1 : rows < most ? rows : most;
}

// How the ring kernel takes a call: `upt` units per thread, `block` threads, `ctas` per SM.  stages 0: rows too wide for it.
struct LnaPlan {
    int G, block, grid, smem;
    agb::LnaRing ring;
};
// Columns a thread takes: one unit where a row has no more than a warp's worth of them; eight where a warp then has the row, where rows are few and a row's latency
// counts (the threads of a row then add up to 1024), and in the backward of rows that are taken element by element, whose instructions and
// not the sums' registers are the limit (8192 x 2047 fp32: 47 us with eight, 64 us with 32; 4099 x 1001 bf16: 18 and 34 us); else 32, which
// spreads the fixed cost of a row over more columns (32768 x 4096 bf16: 149 us with 32, 281 us with eight).
enum LnaWidth { kLnaUnit = 0, kLnaEight = 1, kLnaWide = 2 };
LnaWidth lna_width(int64_t rows, int64_t units, int n, bool backward, int sms) {
    if (units <= 32) return kLnaUnit;
    if (units * n <= 256) return kLnaEight;
    return units * n <= 8192 && (rows <= 2LL * sms || (backward && n == 1)) ? kLnaEight : kLnaWide;
}

// `arrays`: 1 forward, 2 backward.
LnaPlan plan_lna(int64_t rows, int64_t hidden, int elem, bool whole, int64_t units, int upt, int limit, int arrays, const agb_int::Device& d) {
    LnaPlan p{};
    p.G = threads_per_row(units, upt, limit);
    if (!p.G) return p;
    p.block = p.G >= 256 ? p.G : 256 / p.G * p.G;
    int per_tile = p.block / p.G;
    const int64_t row_bytes = hidden * elem;
    // tiles of rows for every SM before tiles of several rows
    while (per_tile > 1 && ceil_div(rows, per_tile) < d.sms && p.block > 32 && p.G < p.block) {
        per_tile = (per_tile + 1) / 2;
        p.block = ceil_div(per_tile * p.G, 32) * 32;
        per_tile = p.block / p.G;
        if (p.block == 32) break;
    }
    const int slack = whole ? 0 : 32;
    const int64_t tile = ceil_div(per_tile * row_bytes + slack, 128) * 128, sums = arrays == 2 && per_tile > 1 ? 2 * hidden * 4 : 0;
    int ctas = (limit >= 1024 || upt == 1 ? 1024 : arrays == 1 && !whole && p.block <= 256 ? 768 : 512) / p.block;   // registers: 64, 80 or 128
    if (ctas > kLnaCtas) ctas = kLnaCtas;
    if (ctas < 1) ctas = 1;
    int stages = 0;
    for (; ctas >= 1; --ctas) {
        int64_t room = d.smem_per_sm / ctas - 1024 - 2048;
        if (room > d.smem_optin - 2048) room = d.smem_optin - 2048;
        stages = static_cast<int>(room / (arrays * tile));
        if (stages >= 3 || (ctas == 1 && stages >= 1)) break;
    }
    if (ctas < 1) return p;
    if (stages > 4) stages = 4;
    p.ring.rows_per_tile = per_tile;
    p.ring.stages = stages;
    p.ring.tile_stride = static_cast<int>(tile);
    p.ring.tiles = ceil_div(rows, per_tile);
    const int64_t bytes = arrays * tile * stages;
    p.smem = static_cast<int>(bytes > sums ? bytes : sums);
    int64_t most = static_cast<int64_t>(d.sms) * ctas;
    if (arrays == 2 && most > lna_partials(rows, hidden)) most = lna_partials(rows, hidden);
    p.grid = static_cast<int>(p.ring.tiles < most ? p.ring.tiles : most);
    return p;
}

template <typename T, int UB, int UPT, int MAXT>
int lna_fwd_launch(agb::LnaFwdArgs a, const LnaPlan& p, const agb_int::Device& d, cudaStream_t st) {
    a.G = p.G;
    AGB_CUDA(cudaFuncSetAttribute(agb::lna_fwd_ring<T, UB, UPT, MAXT>, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem));
    return launch("layernorm_affine_fwd", agb::lna_fwd_ring<T, UB, UPT, MAXT>, dim3(p.grid), dim3(p.block), p.smem, st, 1, a, p.ring, d.status);
}
template <typename T, int UB>
int lna_fwd(const agb::LnaFwdArgs& a, const agb_int::Device& d, cudaStream_t st) {
    constexpr int N = agb::Unit<T, UB>::N;
    const int64_t units = a.hidden / N;
    auto plan = [&](int upt, int limit) { return plan_lna(a.rows, a.hidden, sizeof(T), UB == 16, units, upt, limit, 1, d); };
    const LnaWidth width = lna_width(a.rows, units, N, false, d.sms);
    LnaPlan p = width == kLnaUnit ? plan(1, 512) : width == kLnaEight ? plan(8 / N, 1024) : plan(32 / N, 512);
    if (p.ring.stages > 0) {
        if (width == kLnaUnit) return lna_fwd_launch<T, UB, 1, 512>(a, p, d, st);
        if (width == kLnaEight) return lna_fwd_launch<T, UB, 8 / N, 1024>(a, p, d, st);
        // element by element: blocks of 256 at 80 registers a thread, three per SM instead of two (16384 x 4097 bf16 115 -> 102 us; the 16-byte
        // form spills there, 16384 x 8192 bf16 105 -> 151 us)
        if constexpr (UB < 16) {
            if (p.block <= 256) return lna_fwd_launch<T, UB, 32 / N, 256>(a, p, d, st);
        }
        return lna_fwd_launch<T, UB, 32 / N, 512>(a, p, d, st);
    }
    agb::lna_fwd_wide<T, UB><<<static_cast<unsigned>(grid_for(a.rows, 1024, 1024, d.sms, 2)), 1024, 0, st>>>(a);
    return after_launch("layernorm_affine_fwd");
}

template <typename T, int UB, int UPT, int MAXT>
int lna_ring(agb::LnaBwdArgs a, const LnaPlan& p, float* partial, const agb_int::Device& d, cudaStream_t st) {
    a.G = p.G;
    AGB_CUDA(cudaFuncSetAttribute(agb::lna_bwd_ring<T, UB, UPT, MAXT>, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem));
    return launch("layernorm_affine_bwd", agb::lna_bwd_ring<T, UB, UPT, MAXT>, dim3(p.grid), dim3(p.block), p.smem, st, 1, a, p.ring, partial,
                  d.status);
}

// The single pass where a row fits a block (32 columns a thread, 512 threads; 8 and 1024 where rows are few and a row's latency counts),
// else dx and the column sums one after the other.
template <typename T, int UB>
int lna_bwd(const agb::LnaBwdArgs& a, float* dgamma, float* dbeta, int accumulate, float* partial, const agb_int::Device& d, cudaStream_t st) {
    constexpr int N = agb::Unit<T, UB>::N;
    const bool columns = dgamma || dbeta;
    int runs = 0;
    if (a.rows > 0) {
        const int64_t units = a.hidden / N;
        auto plan = [&](int upt, int limit) { return plan_lna(a.rows, a.hidden, sizeof(T), UB == 16, units, upt, limit, 2, d); };
        const LnaWidth width = lna_width(a.rows, units, N, true, d.sms);
        const LnaPlan p = width == kLnaUnit ? plan(1, 512) : width == kLnaEight ? plan(8 / N, 1024) : plan(32 / N, 512);
        float* to = columns ? partial : nullptr;
        if (p.ring.stages > 0) {
            runs = p.grid;
            if (width == kLnaUnit) AGB_TRY((lna_ring<T, UB, 1, 512>(a, p, to, d, st)));
            else if (width == kLnaEight) AGB_TRY((lna_ring<T, UB, 8 / N, 1024>(a, p, to, d, st)));
            else AGB_TRY((lna_ring<T, UB, 32 / N, 512>(a, p, to, d, st)));
        } else {
            const int64_t run = ceil_div(a.rows, kLnaRuns);
            if (columns) {
                runs = static_cast<int>(ceil_div(a.rows, run));
                agb::lna_columns<T><<<dim3(static_cast<unsigned>(ceil_div(a.hidden, 256)), runs), 256, 0, st>>>(
                    static_cast<const T*>(a.x), static_cast<const T*>(a.gy), a.mean, a.rstd, partial, a.rows, a.hidden, run);
                AGB_TRY(after_launch("layernorm_affine_columns"));
            }
            agb::lna_dx_wide<T, UB><<<static_cast<unsigned>(grid_for(a.rows, 1024, 1024, d.sms, 2)), 1024, 0, st>>>(a);
            AGB_TRY(after_launch("layernorm_affine_dx"));
        }
    }
    if (!columns) return AGB_OK;
    return launch("layernorm_affine_column_reduce", agb::lna_column_reduce, dim3(static_cast<unsigned>(ceil_div(2LL * a.hidden, 32))), dim3(32, 32), 0,
                  st, 1, static_cast<const float*>(partial), runs, a.hidden, dgamma, dbeta, accumulate);
}

// ------------------------------------------------------------------ distillation
int check_kd(int64_t rows, int64_t vocab, int64_t k, float tau, int dtype, int idx_type, int teacher_dtype) {
    if (rows < 0 || vocab <= 0 || k <= 0)
        return fail(AGB_ERR_INVALID_ARG, "rows=%lld vocab=%lld k=%lld", (long long)rows, (long long)vocab, (long long)k);
    if (!(tau > 0.f) || !(tau < INFINITY) || !(1.f / tau < INFINITY))
        return fail(AGB_ERR_INVALID_ARG, "temperature %g must be positive and finite, and its reciprocal too", (double)tau);
    if (dtype != AGB_F32 && dtype != AGB_BF16) return fail(AGB_ERR_UNSUPPORTED, "dtype %d (only AGB_F32, AGB_BF16)", dtype);
    if (teacher_dtype != AGB_F32 && teacher_dtype != AGB_BF16)
        return fail(AGB_ERR_UNSUPPORTED, "teacher_dtype %d (only AGB_F32, AGB_BF16)", teacher_dtype);
    if (idx_type != AGB_I32 && idx_type != AGB_I64) return fail(AGB_ERR_INVALID_ARG, "idx_type %d (AGB_I32 or AGB_I64)", idx_type);
    if (vocab > (1LL << 30)) return fail(AGB_ERR_UNSUPPORTED, "vocab %lld too large", (long long)vocab);
    if (k > agb::kKdMaxK) return fail(AGB_ERR_UNSUPPORTED, "k=%lld (at most %d)", (long long)k, agb::kKdMaxK);
    if (rows > (1LL << 27)) return fail(AGB_ERR_UNSUPPORTED, "rows=%lld (at most 2^27)", (long long)rows);
    return AGB_OK;
}

constexpr int kKdKeep = 8;         // words of 16 bytes that a thread of a block keeps

template <typename T, int MODE>
int launch_kd(agb::KdArgs a, int64_t rows, cudaStream_t st) {
    agb_int::Device d;
    AGB_TRY(agb_int::device(&d));
    a.status = d.status;
    const int64_t word = 16 / static_cast<int64_t>(sizeof(T));
    const char* what = "distill_topk";
    a.slice = a.vocab;
    if (a.vocab <= 32 * 32 * word && a.k <= agb::kKdWarpK && rows >= d.sms) {
        const dim3 grid(static_cast<unsigned>(ceil_div(rows, 8)));
        if (a.vocab <= 32 * 8 * word) return launch(what, agb::kd_kernel<T, MODE, 32, 8>, grid, dim3(256), 0, st, 1, a);
        return launch(what, agb::kd_kernel<T, MODE, 32, 0>, grid, dim3(256), 0, st, 1, a);
    }
    // Slices per row: enough CTAs for the GPU where rows are few, none shorter than one turn of a block of 256.
    int C = 1;
    while (C < 8 && rows * C < 2 * d.sms && a.vocab / (2 * C) >= 256 * word) C *= 2;
    if (MODE < 2 && C > 1 && ceil_div(a.vocab, C) <= 256 * kKdKeep * word - 64) {
        a.slice = ceil_div(ceil_div(a.vocab, C), 64) * 64;
        return launch(what, agb::kd_kernel<T, MODE, 256, kKdKeep>, dim3(static_cast<unsigned>(rows * C)), dim3(256), 0, st, C, a);
    }
    // There and back.  Long rows: blocks of 512 and slices of up to 256 KB, since a block's joins cost the same for a short one (4096 x 131072
    // bf16: 476 us, 496 us with 256 threads and 64 KB).  Shorter rows: 256 threads (4096 x 32768 bf16: 130 us, 179 us with 512).
    const int64_t row_bytes = a.vocab * static_cast<int64_t>(sizeof(T));
    const bool wide = MODE == 1 && row_bytes >= (128 << 10);
    while (wide && C < 8 && row_bytes / C > (256 << 10)) C *= 2;
    a.slice = ceil_div(ceil_div(a.vocab, C), 64) * 64;
    const dim3 grid(static_cast<unsigned>(rows * C));
    if constexpr (MODE == 1) {
        if (wide) return launch(what, agb::kd_kernel<T, MODE, 512, 0>, grid, dim3(512), 0, st, C, a);
    }
    return launch(what, agb::kd_kernel<T, MODE, 256, 0>, grid, dim3(256), 0, st, C, a);
}

template <int MODE>
int run_kd(const void* z, const void* idx, int idx_type, const void* teacher, int teacher_dtype, float* loss, float* lse,
           const float* gy, const void* dz_add, void* dz, int64_t rows, int64_t vocab, int64_t k, float tau, int dtype, void* stream) {
    AGB_TRY(check_kd(rows, vocab, k, tau, dtype, idx_type, teacher_dtype));
    if (rows == 0) return AGB_OK;
    const int elem = dtype == AGB_F32 ? 4 : 2;
    AGB_TRY(check_ptr(z, "z", elem));
    AGB_TRY(check_ptr(idx, "idx", idx_type == AGB_I64 ? 8 : 4));
    AGB_TRY(check_ptr(teacher, "teacher", teacher_dtype == AGB_F32 ? 4 : 2));
    AGB_TRY(check_ptr(lse, "lse", 4));
    if (MODE < 2) AGB_TRY(check_ptr(loss, "loss", 4));
    if (MODE > 0) {
        AGB_TRY(check_ptr(gy, "gy", 4));
        AGB_TRY(check_ptr(dz, "dz", elem));
        AGB_TRY(check_ptr(dz_add, "dz_add", elem, false));
    }
    agb::KdArgs a{z, idx, teacher, idx_type == AGB_I64, teacher_dtype == AGB_BF16, loss, lse, gy, dz_add, dz, rows, vocab, static_cast<int>(k),
                  tau, 1.f / tau, 0, nullptr};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == AGB_F32 ? launch_kd<float, MODE>(a, rows, st) : launch_kd<bf16, MODE>(a, rows, st);
}

// ------------------------------------------------------------------ cross entropy from the hidden states
// The driver's tensor map encoder, looked up once (the runtime library is linked, the driver library is not).
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = []() -> EncodeTiled {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}
// A [planes][rows][cols] tensor (bf16, or fp32) with rows `stride` elements apart, in boxes of 128 bytes by `box_rows` rows.
int make_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int planes, int64_t stride, int64_t plane, int box_rows,
             bool f32 = false) {
    const int elem = f32 ? 4 : 2;
    EncodeTiled f = encode_tiled();
    if (!f) return fail(AGB_ERR_CUDA, "cuTensorMapEncodeTiled is not available in this driver");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride) * elem, static_cast<cuuint64_t>(plane) * elem};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / elem), static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult r = f(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(AGB_ERR_CUDA, "cuTensorMapEncodeTiled: error %d", static_cast<int>(r));
    return AGB_OK;
}

constexpr int64_t kCePackLimit = 512LL << 20;   // bytes of W laid out at once, where it has to be
constexpr int64_t kCeGLimit = 256LL << 20;      // bytes of g at once

// How a call is cut up, and where its parts lie in the workspace.
struct CePlan {
    int planes;
    bool direct_w;              // TMA reads W as it is
    bool direct_dw;             // and writes dW as it is
    int64_t rows_pad, k_stride, piece, pieces, g_stride, dh_stride, pairs;
    int pair;                   // CTAs that work on a tile together
    int tn;                     // columns of a tile of logits
    int64_t pairs_per_piece;
    int splits, k_per_split;
    int z_splits, z_per_split;  // parts of the logits' K; 1: none
    size_t z, h, w, count, row_of, pos_of, target_of, lse_of, gy_of, gy_scale, left_over, z_target, pair_at, g, dh, dw, total;
};

// Columns of a tile of logits.  A slab of a tile takes the longest of its products (2 clocks per column), its bytes from L2 at 64 a
// clock, and its share of W from memory at 24 a clock (the measured rate over the SMs), which the tiles above it share; what counts is
// that times the turns that the GPU takes.  16 x 4096 x 32768: one turn of 147 tiles of 224 columns instead of one of 128 tiles of 256.
int choose_tn(int pair, int64_t rows, int64_t columns, int step, int sms) {
    const int64_t mt = ceil_div(rows, pair * agb::kTM), units = sms / pair;
    int best = 256;
    double least = 0;
    for (int tn = 256; tn >= (step < 64 ? 64 : step); tn -= step) {
        double slab = 2.0 * tn;
        const double l2 = (agb::kTM * 128 + tn / pair * 128) / 64.0, dram = tn / pair * 128 / 24.0 / static_cast<double>(mt);
        if (l2 > slab) slab = l2;
        if (dram > slab) slab = dram;
        const double cost = slab * static_cast<double>(ceil_div(mt * ceil_div(columns, tn), units));
        if (tn == 256 || cost < 0.97 * least) {
            best = tn;
            least = cost;
        }
    }
    return best;
}

CePlan plan_ce(bool backward, int64_t rows, int64_t hidden, int64_t vocab, int dtype, bool want_dh, int sms) {
    CePlan p{};
    p.planes = dtype == AGB_F32 ? 3 : 1;
    p.direct_w = dtype == AGB_BF16 && hidden % 8 == 0;
    p.direct_dw = hidden % (dtype == AGB_BF16 ? 8 : 4) == 0;
    p.rows_pad = ceil_div(rows, 2 * agb::kTM) * 2 * agb::kTM;
    p.k_stride = ceil_div(hidden, 8) * 8;
    p.piece = ceil_div(vocab, 256) * 256;
    auto limit = [&](int64_t bytes_per_column, int64_t bytes) {
        int64_t most = bytes / bytes_per_column / 256 * 256;
        if (most < 256) most = 256;
        if (p.piece > most) p.piece = most;
    };
    if (!p.direct_w) limit(p.planes * p.k_stride * 2, kCePackLimit);
    if (backward) limit(p.planes * p.rows_pad * 2, kCeGLimit);
    p.pieces = ceil_div(vocab, p.piece);
    p.piece = ceil_div(ceil_div(vocab, p.pieces), 256) * 256;      // even pieces
    p.pieces = ceil_div(vocab, p.piece);
    p.g_stride = p.piece;
    p.dh_stride = ceil_div(hidden, 4) * 4;
    p.pair = rows <= agb::kTM ? 1 : 2;     // rows that fit one CTA's half of a pair's tile leave nothing for the other to do
    p.tn = choose_tn(p.pair, rows, p.piece < vocab ? p.piece : vocab, backward ? 128 : 32, sms);
    p.pairs_per_piece = ceil_div(p.piece, p.tn) * 2;
    p.pairs = p.pieces * p.pairs_per_piece;
    // dh: few tiles with a long sum are cut along it, until the GPU has two per SM or a part has 16 slabs
    const int64_t tiles = p.rows_pad / agb::kTM * ceil_div(hidden, agb::kTN), blocks = ceil_div(p.piece, agb::kTK);
    int64_t s = ceil_div(2 * sms, tiles);
    const int64_t slabs = blocks * (p.planes == 3 ? 6 : 1);
    if (s > slabs / 16) s = slabs / 16;
    if (s > blocks) s = blocks;
    if (s < 1) s = 1;
    p.k_per_split = static_cast<int>(ceil_div(blocks, s) * agb::kTK);
    p.splits = static_cast<int>(ceil_div(p.piece, p.k_per_split));
    // The logits of a small problem: tiles that leave most of the GPU idle, each with a long sum, are cut along it too.  1.5 us of a slab
    // of 64 saved per eighth of the sum against one more kernel: 10 x 1835 x 2235 fp32 took 71 us as nine tiles of 174 slabs.
    const int64_t z_tiles = ceil_div(rows, p.pair * agb::kTM) * ceil_div(vocab, agb::kTN), z_blocks = ceil_div(hidden, agb::kTK);
    int64_t z = (sms / p.pair) / z_tiles;
    if (z > z_blocks / 2) z = z_blocks / 2;
    p.z_splits = 1;
    if (p.pieces == 1 && z >= 2 && z_blocks * (p.planes == 3 ? 6 : 1) >= 40 && z * p.rows_pad * p.piece * 4 <= (64 << 20)) {
        p.z_per_split = static_cast<int>(ceil_div(z_blocks, z) * agb::kTK);
        p.z_splits = static_cast<int>(ceil_div(hidden, p.z_per_split));
    }
    size_t at = 0;
    auto take = [&](size_t* where, size_t bytes) {
        *where = at;
        at += (bytes + 1023) / 1024 * 1024;
    };
    take(&p.h, static_cast<size_t>(p.planes) * p.rows_pad * p.k_stride * 2);
    take(&p.count, 4);
    take(&p.row_of, p.rows_pad * 4);
    take(&p.pos_of, p.rows_pad * 4);
    take(&p.target_of, p.rows_pad * 4);
    if (p.z_splits > 1) take(&p.z, static_cast<size_t>(p.z_splits) * p.rows_pad * p.piece * 4);
    if (!p.direct_w) take(&p.w, static_cast<size_t>(p.planes) * p.piece * p.k_stride * 2);
    if (backward) {
        take(&p.lse_of, p.rows_pad * 4);
        take(&p.gy_of, p.rows_pad * 4);
        take(&p.left_over, p.rows_pad * 4);
        take(&p.gy_scale, 4);
        take(&p.g, static_cast<size_t>(p.planes) * p.rows_pad * p.g_stride * 2);
        if (!p.direct_dw) take(&p.dw, static_cast<size_t>(p.piece) * p.k_stride * 4);
        if (want_dh) take(&p.dh, static_cast<size_t>(p.splits) * p.rows_pad * p.dh_stride * 4);
    } else {
        take(&p.z_target, p.rows_pad * 4);
        take(&p.pair_at, static_cast<size_t>(p.pairs) * p.rows_pad * 8);
    }
    p.total = at + 1024;        // the caller's base may lie anywhere
    return p;
}

int check_ce(int64_t rows, int64_t hidden, int64_t vocab, int dtype, int target_type) {
    if (rows < 0 || hidden <= 0 || vocab <= 0)
        return fail(AGB_ERR_INVALID_ARG, "rows=%lld hidden=%lld vocab=%lld", (long long)rows, (long long)hidden, (long long)vocab);
    if (dtype != AGB_F32 && dtype != AGB_BF16) return fail(AGB_ERR_UNSUPPORTED, "dtype %d (only AGB_F32, AGB_BF16)", dtype);
    if (target_type != AGB_I32 && target_type != AGB_I64) return fail(AGB_ERR_INVALID_ARG, "target_type %d (AGB_I32 or AGB_I64)", target_type);
    // rows: the blocks that lay h out count the targets before their own, which grows with the square (13 ms at 2^20 rows)
    if (rows > (1LL << 20) || hidden > (1LL << 20) || vocab > (1LL << 24))
        return fail(AGB_ERR_UNSUPPORTED, "rows=%lld hidden=%lld vocab=%lld (at most 2^20, 2^20, 2^24)", (long long)rows, (long long)hidden,
                    (long long)vocab);
    return AGB_OK;
}

struct CeCall {
    const void *h, *w, *target;
    int target_type;
    int64_t rows, hidden, vocab;
    int dtype;
    char* ws;
    cudaStream_t st;
    agb_int::Device d;
    CePlan p;
    template <typename T>
    T* at(size_t off) const { return reinterpret_cast<T*>(ws + off); }
};

int ce_rows(const CeCall& c, const float* lse, const float* gy, float* loss, float* lse_out) {
    agb::CeRowsArgs a{};
    a.x = c.h;
    a.target = c.target;
    a.target64 = c.target_type == AGB_I64;
    a.rows = c.rows;
    a.cols = static_cast<int>(c.hidden);
    a.vocab = static_cast<int>(c.vocab);
    a.planes = c.p.planes;
    a.dst = c.at<bf16>(c.p.h);
    a.rows_pad = c.p.rows_pad;
    a.stride = c.p.k_stride;
    a.count = c.at<int>(c.p.count);
    a.row_of = c.at<int>(c.p.row_of);
    a.pos_of = c.at<int>(c.p.pos_of);
    a.target_of = c.at<int>(c.p.target_of);
    a.lse = lse;
    a.gy = gy;
    if (lse) {
        a.lse_of = c.at<float>(c.p.lse_of);
        a.gy_of = c.at<float>(c.p.gy_of);
        a.gy_scale = c.at<float>(c.p.gy_scale);
    }
    a.loss = loss;
    a.lse_out = lse_out;
    // a block per row, then a warp per row, while the blocks, which all count the targets before their own, stay about a thousand
    a.per_block = c.rows <= 8LL * c.d.sms ? 1 : c.rows <= 8192 ? 8 : c.rows <= 16384 ? 16 : agb::kRowsBlock;
    const dim3 grid(static_cast<unsigned>(ceil_div(c.rows, a.per_block)) + agb::kRowsEnd);
    return launch("linear_ce_rows", c.dtype == AGB_F32 ? agb::ce_rows_kernel<float> : agb::ce_rows_kernel<bf16>, grid, dim3(256), 0, c.st, 1, a);
}
int ce_pack(const CeCall& c, int64_t col0, int64_t n) {
    if (c.p.direct_w) return AGB_OK;
    const bool wide = c.hidden >= 256 && n >= 8LL * c.d.sms;
    int64_t grid = wide ? ceil_div(n, 8) : ceil_div(n * (c.p.k_stride / 2), 256 * 8);
    if (grid > 16LL * c.d.sms) grid = 16LL * c.d.sms;
    auto pack = [&](auto kernel, auto* typed) {
        typedef decltype(typed) P;
        return launch("linear_ce_pack", kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, c.st, 1, static_cast<P>(c.w) + col0 * c.hidden, n,
                      static_cast<int>(c.hidden), c.at<bf16>(c.p.w), c.p.piece, c.p.k_stride);
    };
    if (c.dtype == AGB_F32)
        return pack(wide ? agb::ce_pack_kernel<float, true> : agb::ce_pack_kernel<float, false>, static_cast<const float*>(nullptr));
    return pack(wide ? agb::ce_pack_kernel<bf16, true> : agb::ce_pack_kernel<bf16, false>, static_cast<const bf16*>(nullptr));
}
int ce_unpack(const CeCall& c, void* dw, int64_t col0, int64_t n, bool f32, int add) {
    const bool wide = c.hidden >= 256 && n >= 8LL * c.d.sms;
    int64_t grid = wide ? ceil_div(n, 8) : ceil_div(n * c.hidden, 256 * 8);
    if (grid > 16LL * c.d.sms) grid = 16LL * c.d.sms;
    auto unpack = [&](auto kernel, auto* from, auto* to) {
        return launch("linear_ce_unpack", kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, c.st, 1, from, n, static_cast<int>(c.hidden),
                      c.p.k_stride, to + col0 * c.hidden, add);
    };
    if (c.dtype == AGB_F32)
        return unpack(wide ? agb::ce_unpack_kernel<float, float, true> : agb::ce_unpack_kernel<float, float, false>, c.at<float>(c.p.dw),
                      static_cast<float*>(dw));
    if (f32)
        return unpack(wide ? agb::ce_unpack_kernel<float, bf16, true> : agb::ce_unpack_kernel<float, bf16, false>, c.at<float>(c.p.dw),
                      static_cast<bf16*>(dw));
    return unpack(wide ? agb::ce_unpack_kernel<bf16, bf16, true> : agb::ce_unpack_kernel<bf16, bf16, false>, c.at<bf16>(c.p.dw),
                  static_cast<bf16*>(dw));
}
// W, or its piece where it was laid out: rows of the map, and the map's row of the piece's first column.
int map_w(const CeCall& c, CUtensorMap* m, int64_t n, int box_rows) {
    if (c.p.direct_w) return make_map(m, c.w, c.hidden, c.vocab, 1, c.hidden, c.vocab * c.hidden, box_rows);
    return make_map(m, c.at<void>(c.p.w), c.p.k_stride, n, c.p.planes, c.p.k_stride, c.p.piece * c.p.k_stride, box_rows);
}
int map_h(const CeCall& c, CUtensorMap* m, int box_rows) {
    return make_map(m, c.at<void>(c.p.h), c.p.k_stride, c.p.rows_pad, c.p.planes, c.p.k_stride, c.p.rows_pad * c.p.k_stride, box_rows);
}
int map_g(const CeCall& c, CUtensorMap* m, int box_rows) {
    return make_map(m, c.at<void>(c.p.g), c.p.g_stride, c.p.rows_pad, c.p.planes, c.p.g_stride, c.p.rows_pad * c.p.g_stride, box_rows);
}
agb::CeArgs ce_args(const CeCall& c) {
    agb::CeArgs a{};
    a.count = c.at<int>(c.p.count);
    a.status = c.d.status;
    a.rows_pad = c.p.rows_pad;
    a.target = c.at<int>(c.p.target_of);
    a.vocab = static_cast<int>(c.vocab);
    a.planes = c.p.planes;
    a.hidden = static_cast<int>(c.hidden);
    return a;
}
// The logits of a piece: rows that take part x n columns.
agb::CeJob logits_job(const CeCall& c, int epi, int64_t col0, int64_t n) {
    agb::CeJob j{};
    j.epi = epi;
    j.a_planes3 = c.p.planes == 3;
    j.b_row0 = c.p.direct_w ? static_cast<int>(col0) : 0;
    j.m = -1;
    j.n = static_cast<int>(n);
    j.k = static_cast<int>(c.hidden);
    j.splits = 1;
    j.k_per_split = static_cast<int>(ceil_div(c.hidden, agb::kTK) * agb::kTK);
    j.tn = c.p.tn;
    j.b_box = j.tn / c.p.pair;
    return j;
}
template <int CG, int PHASE>
int launch_gemm_cg(const CeCall& c, const agb::CeArgs& a) {
    int64_t tiles = 0;
    for (int i = 0; i < a.jobs; ++i) {
        const agb::CeJob& j = a.job[i];
        tiles += ceil_div(j.m < 0 ? c.rows : j.m, CG * agb::kTM) * ceil_div(j.n, j.tn) * j.splits;
    }
    if (tiles >= (1LL << 31)) return fail(AGB_ERR_UNSUPPORTED, "too many tiles");
    AGB_CUDA(cudaFuncSetAttribute(agb::ce_gemm_kernel<CG, PHASE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (agb::CeRing<CG, PHASE>::kSmem)));
    const int64_t most = c.d.sms / CG;
    return launch("linear_ce_gemm", agb::ce_gemm_kernel<CG, PHASE>, dim3(static_cast<unsigned>((tiles < most ? tiles : most) * CG)),
                  dim3(agb::kCeThreads), agb::CeRing<CG, PHASE>::kSmem, c.st, CG, a);
}
template <int PHASE>
int launch_gemm(const CeCall& c, const agb::CeArgs& a) {
    return c.p.pair == 1 ? launch_gemm_cg<1, PHASE>(c, a) : launch_gemm_cg<2, PHASE>(c, a);
}

// The logits of a small problem as parts of K (there is one piece).
int ce_parts(const CeCall& c) {
    agb::CeArgs a = ce_args(c);
    a.jobs = 1;
    agb::CeJob& j = a.job[0];
    j = logits_job(c, agb::kEpiDh, 0, c.vocab);
    j.tn = agb::kTN;
    j.b_box = j.tn / c.p.pair;
    j.splits = c.p.z_splits;
    j.k_per_split = c.p.z_per_split;
    j.n_first = 1;
    AGB_TRY(map_h(c, &a.A[0], 128));
    AGB_TRY(map_w(c, &a.B[0], c.vocab, j.b_box));
    a.dh = c.at<float>(c.p.z);
    a.dh_stride = c.p.piece;
    AGB_TRY(make_map(&a.out[0], a.dh, c.p.piece, c.p.rows_pad, c.p.z_splits, c.p.piece, c.p.rows_pad * c.p.piece, 32, true));
    return launch_gemm<2>(c, a);
}

int start_ce(CeCall* c, bool backward, bool want_dh, void* workspace, size_t workspace_bytes, agb_stream_t stream) {
    const int elem = c->dtype == AGB_F32 ? 4 : 2;
    AGB_TRY(check_ptr(c->h, "h", elem));
    AGB_TRY(check_ptr(c->w, "w", elem));
    AGB_TRY(check_ptr(c->target, "target", c->target_type == AGB_I64 ? 8 : 4));
    if (c->dtype == AGB_BF16 && c->hidden % 8 == 0 && addr(c->w) % 16)
        return fail(AGB_ERR_MISALIGNED, "w must be aligned to 16 bytes where hidden is a multiple of 8");
    if (!workspace) return fail(AGB_ERR_WORKSPACE, "workspace is NULL");
    AGB_TRY(agb_int::device(&c->d));
    c->p = plan_ce(backward, c->rows, c->hidden, c->vocab, c->dtype, want_dh, c->d.sms);
    if (workspace_bytes < c->p.total) return fail(AGB_ERR_WORKSPACE, "workspace %zu bytes, need %zu", workspace_bytes, c->p.total);
    c->ws = reinterpret_cast<char*>((addr(workspace) + 1023) & ~static_cast<uintptr_t>(1023));
    c->st = static_cast<cudaStream_t>(stream);
    return AGB_OK;
}

}  // namespace

extern "C" {

size_t agb_linear_ce_workspace_bytes(int backward, int64_t rows, int64_t hidden, int64_t vocab, int dtype) {
    agb_int::Device d;
    if (check_ce(rows, hidden, vocab, dtype, AGB_I32) != AGB_OK || agb_int::device(&d) != AGB_OK) return 0;
    return plan_ce(backward != 0, rows > 0 ? rows : 1, hidden, vocab, dtype, true, d.sms).total;
}

int agb_linear_ce_fwd(const void* h, const void* w, const void* target, int target_type, float* loss, float* lse, int64_t rows,
                      int64_t hidden, int64_t vocab, int dtype, void* workspace, size_t workspace_bytes, agb_stream_t stream) {
    AGB_RANGE();
    AGB_TRY(check_ce(rows, hidden, vocab, dtype, target_type));
    if (rows == 0) return AGB_OK;
    AGB_TRY(check_ptr(loss, "loss", 4));
    AGB_TRY(check_ptr(lse, "lse", 4));
    CeCall c{h, w, target, target_type, rows, hidden, vocab, dtype, nullptr, nullptr, {}, {}};
    AGB_TRY(start_ce(&c, false, false, workspace, workspace_bytes, stream));
    AGB_TRY(ce_rows(c, nullptr, nullptr, loss, lse));
    if (c.p.z_splits > 1) {
        AGB_TRY(ce_pack(c, 0, vocab));
        AGB_TRY(ce_parts(c));
        auto join = [&](auto kernel, auto* typed) {
            typedef decltype(typed) P;
            return launch("linear_ce_join_parts", kernel, dim3(static_cast<unsigned>(rows)), dim3(vocab <= 2048 ? 256 : 1024), 0, c.st, 1, c.at<float>(c.p.z), c.p.z_splits,
                          c.p.rows_pad, c.p.piece, static_cast<int>(vocab), c.at<int>(c.p.count), c.at<int>(c.p.target_of), c.at<int>(c.p.row_of),
                          static_cast<P>(h), static_cast<P>(w), static_cast<int>(hidden), loss, lse);
        };
        return dtype == AGB_F32 ? join(agb::ce_join_parts_kernel<float>, static_cast<const float*>(nullptr))
                                : join(agb::ce_join_parts_kernel<bf16>, static_cast<const bf16*>(nullptr));
    }
    for (int64_t i = 0; i < c.p.pieces; ++i) {
        const int64_t col0 = i * c.p.piece, n = vocab - col0 < c.p.piece ? vocab - col0 : c.p.piece;
        AGB_TRY(ce_pack(c, col0, n));
        agb::CeArgs a = ce_args(c);
        a.jobs = 1;
        a.job[0] = logits_job(c, agb::kEpiPairs, col0, n);
        AGB_TRY(map_h(c, &a.A[0], 128));
        AGB_TRY(map_w(c, &a.B[0], n, a.job[0].b_box));
        a.pairs = c.at<float2>(c.p.pair_at);
        a.z_target = c.at<float>(c.p.z_target);
        a.col0 = static_cast<int>(col0);
        a.n_pairs = c.p.pairs;
        a.pair0 = static_cast<int>(i * c.p.pairs_per_piece);
        AGB_TRY(launch_gemm<0>(c, a));
    }
    const int64_t last = vocab - (c.p.pieces - 1) * c.p.piece;
    const int pairs = static_cast<int>((c.p.pieces - 1) * c.p.pairs_per_piece + ceil_div(last, c.p.tn) * 2);
    const bool few = rows <= 8LL * c.d.sms;
    const dim3 grid(static_cast<unsigned>(few ? rows : ceil_div(rows, 8)));
    auto join = [&](auto kernel, auto* typed) {
        typedef decltype(typed) P;
        return launch("linear_ce_join", kernel, grid, dim3(256), 0, c.st, 1, c.at<float2>(c.p.pair_at), pairs, c.p.pairs, c.at<int>(c.p.count),
                      c.at<float>(c.p.z_target), c.at<int>(c.p.target_of), c.at<int>(c.p.row_of), static_cast<P>(h), static_cast<P>(w),
                      static_cast<int>(hidden), loss, lse);
    };
    if (dtype == AGB_F32)
        return join(few ? agb::ce_join_kernel<float, 8> : agb::ce_join_kernel<float, 1>, static_cast<const float*>(nullptr));
    return join(few ? agb::ce_join_kernel<bf16, 8> : agb::ce_join_kernel<bf16, 1>, static_cast<const bf16*>(nullptr));
}

int agb_linear_ce_bwd(const void* h, const void* w, const void* target, int target_type, const float* lse, const float* gy, void* dh,
                      void* dw, int accumulate_dw, int64_t rows, int64_t hidden, int64_t vocab, int dtype, void* workspace,
                      size_t workspace_bytes, agb_stream_t stream) {
    AGB_RANGE();
    AGB_TRY(check_ce(rows, hidden, vocab, dtype, target_type));
    const int elem = dtype == AGB_F32 ? 4 : 2;
    if (!dh && !dw) return fail(AGB_ERR_INVALID_ARG, "neither dh nor dw is asked for");
    if (dw && dw == w) return fail(AGB_ERR_INVALID_ARG, "dw must not be w: w is read while dw is written");
    if (dh && (dh == w || dh == dw)) return fail(AGB_ERR_INVALID_ARG, "dh must not be w or dw");
    AGB_TRY(check_ptr(dw, "dw", elem, false));
    if (rows == 0) {
        if (dw && !accumulate_dw)
            AGB_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(vocab) * hidden * elem, static_cast<cudaStream_t>(stream)));
        return AGB_OK;
    }
    AGB_TRY(check_ptr(dh, "dh", elem, false));
    AGB_TRY(check_ptr(lse, "lse", 4));
    AGB_TRY(check_ptr(gy, "gy", 4));
    CeCall c{h, w, target, target_type, rows, hidden, vocab, dtype, nullptr, nullptr, {}, {}};
    AGB_TRY(start_ce(&c, true, dh != nullptr, workspace, workspace_bytes, stream));
    AGB_TRY(ce_rows(c, lse, gy, nullptr, nullptr));
    for (int64_t i = 0; i < c.p.pieces; ++i) {
        const int64_t col0 = i * c.p.piece, n = vocab - col0 < c.p.piece ? vocab - col0 : c.p.piece;
        AGB_TRY(ce_pack(c, col0, n));
        agb::CeArgs a = ce_args(c);
        a.jobs = 1;
        a.job[0] = logits_job(c, agb::kEpiG, col0, n);
        AGB_TRY(map_h(c, &a.A[0], 128));
        AGB_TRY(map_w(c, &a.B[0], n, a.job[0].b_box));
        a.col0 = static_cast<int>(col0);
        a.lse = c.at<float>(c.p.lse_of);
        a.gy = c.at<float>(c.p.gy_of);
        a.g = c.at<bf16>(c.p.g);
        a.g_stride = c.p.g_stride;
        a.left_over = c.p.planes == 1 ? c.at<float>(c.p.left_over) : nullptr;
        a.gy_scale = c.at<float>(c.p.gy_scale);
        AGB_TRY(map_g(c, &a.out[0], 32));
        if (c.p.z_splits > 1) {
            AGB_TRY(ce_parts(c));
            const dim3 grid(static_cast<unsigned>(ceil_div(c.p.g_stride, 512)), static_cast<unsigned>(ceil_div(rows, agb::kTK) * agb::kTK));
            AGB_TRY(launch("linear_ce_g_parts", agb::ce_g_parts_kernel, grid, dim3(256), 0, c.st, 1, c.at<float>(c.p.z), c.p.z_splits, c.p.rows_pad,
                           c.p.piece, static_cast<int>(vocab), c.at<int>(c.p.count), c.at<int>(c.p.target_of), a.lse, a.gy, a.gy_scale, a.g,
                           a.g_stride, c.p.planes, a.left_over));
        } else {
            AGB_TRY(c.p.planes == 1 ? launch_gemm<1>(c, a) : launch_gemm<3>(c, a));
        }
        a.jobs = 0;
        if (dh) {
            agb::CeJob& j = a.job[a.jobs];
            j = agb::CeJob{};
            j.epi = agb::kEpiDh;
            j.b_mn = 1;
            j.a_planes3 = c.p.planes == 3;
            j.b_row0 = c.p.direct_w ? static_cast<int>(col0) : 0;
            j.m = -1;
            j.n = static_cast<int>(hidden);
            j.k = static_cast<int>(n);
            j.splits = c.p.splits;
            j.k_per_split = c.p.k_per_split;
            j.n_first = 1;
            j.tn = agb::kTN;
            j.b_box = 64;
            AGB_TRY(map_g(c, &a.A[a.jobs], 128));
            AGB_TRY(map_w(c, &a.B[a.jobs], n, 64));
            a.dh = c.at<float>(c.p.dh);
            a.dh_stride = c.p.dh_stride;
            a.dh_add = i > 0;
            AGB_TRY(make_map(&a.out[a.jobs], a.dh, c.p.dh_stride, c.p.rows_pad, c.p.splits, c.p.dh_stride, c.p.rows_pad * c.p.dh_stride, 32, true));
            ++a.jobs;
        }
        if (dw) {
            agb::CeJob& j = a.job[a.jobs];
            j = agb::CeJob{};
            j.epi = agb::kEpiDw;
            j.a_mn = j.b_mn = 1;
            j.a_planes3 = c.p.planes == 3;
            j.m = static_cast<int>(n);
            j.n = static_cast<int>(hidden);
            j.k = -1;
            j.splits = 1;
            j.k_per_split = static_cast<int>(c.p.rows_pad);
            j.n_first = 1;
            j.tn = agb::kTN;
            j.b_box = 64;
            AGB_TRY(map_g(c, &a.A[a.jobs], 64));
            AGB_TRY(map_h(c, &a.B[a.jobs], 64));
            a.dw = dw;
            a.dw_add = accumulate_dw != 0;
            a.dw_f32 = dtype == AGB_F32;
            if (!c.p.direct_dw) {
                a.dw_out = agb::kDwStaged;
                a.dw_f32 = a.dw_f32 || a.dw_add;
                AGB_TRY(make_map(&a.out[a.jobs], c.at<void>(c.p.dw), c.p.k_stride, n, 1, c.p.k_stride, c.p.piece * c.p.k_stride, 32, a.dw_f32));
            } else if (addr(dw) % 16 == 0) {
                a.dw_out = agb::kDwTma;
                AGB_TRY(make_map(&a.out[a.jobs], dw, hidden, vocab, 1, hidden, vocab * hidden, 32, a.dw_f32));
            } else {
                a.dw_out = agb::kDwScalar;
            }
            ++a.jobs;
        }
        AGB_TRY(launch_gemm<2>(c, a));
        if (dw && a.dw_out == agb::kDwStaged) AGB_TRY(ce_unpack(c, dw, col0, n, a.dw_f32, accumulate_dw));
    }
    if (dh) {
        const dim3 grid(static_cast<unsigned>(ceil_div(ceil_div(hidden, 4), 256)), static_cast<unsigned>(rows < 32768 ? rows : 32768));
        const float* left = c.p.planes == 1 ? c.at<float>(c.p.left_over) : nullptr;
        auto add_up = [&](auto kernel, auto* to) {
            typedef std::remove_pointer_t<decltype(to)> T;
            return launch("linear_ce_dh", kernel, grid, dim3(256), 0, c.st, 1, c.at<float>(c.p.dh), c.p.splits, c.p.rows_pad, c.p.dh_stride,
                          c.at<int>(c.p.pos_of), c.at<int>(c.p.target_of), left, c.at<float>(c.p.gy_scale), static_cast<const T*>(w), to, rows,
                          static_cast<int>(hidden));
        };
        return dtype == AGB_F32 ? add_up(agb::ce_dh_kernel<float>, static_cast<float*>(dh)) : add_up(agb::ce_dh_kernel<bf16>, static_cast<bf16*>(dh));
    }
    return AGB_OK;
}

int agb_layernorm_affine_fwd(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, int64_t rows,
                             int64_t hidden, float eps, int dtype, agb_stream_t stream) {
    AGB_RANGE();
    AGB_TRY(check_lna(rows, hidden, dtype));
    if (rows == 0) return AGB_OK;
    const int elem = dtype == AGB_F32 ? 4 : 2;
    AGB_TRY(check_ptr(x, "x", elem));
    AGB_TRY(check_ptr(gamma, "gamma", elem));
    AGB_TRY(check_ptr(beta, "beta", elem, false));
    AGB_TRY(check_ptr(y, "y", elem));
    AGB_TRY(check_ptr(mean, "mean", 4));
    AGB_TRY(check_ptr(rstd, "rstd", 4));
    agb_int::Device d;
    AGB_TRY(agb_int::device(&d));
    agb::LnaFwdArgs a{x, gamma, beta, y, mean, rstd, rows, static_cast<int>(hidden), 0, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ub = unit_bytes(addr(x) | addr(gamma) | addr(beta) | addr(y), hidden * elem, elem);
    if (dtype == AGB_F32) return ub == 16 ? lna_fwd<float, 16>(a, d, st) : lna_fwd<float, 4>(a, d, st);
    return ub == 16 ? lna_fwd<bf16, 16>(a, d, st) : lna_fwd<bf16, 2>(a, d, st);
}

size_t agb_layernorm_affine_bwd_workspace_bytes(int64_t rows, int64_t hidden, int dtype) {
    (void)dtype;
    return hidden <= 0 ? 0 : static_cast<size_t>(lna_partials(rows, hidden)) * 2 * hidden * sizeof(float);
}

int agb_layernorm_affine_bwd(const void* x, const void* gamma, const float* mean, const float* rstd, const void* gy, const void* dx_add,
                             void* dx, float* dgamma, float* dbeta, int accumulate, void* workspace, size_t workspace_bytes, int64_t rows,
                             int64_t hidden, int dtype, agb_stream_t stream) {
    AGB_RANGE();
    AGB_TRY(check_lna(rows, hidden, dtype));
    const int elem = dtype == AGB_F32 ? 4 : 2;
    if (rows > 0) {
        AGB_TRY(check_ptr(x, "x", elem));
        AGB_TRY(check_ptr(gamma, "gamma", elem));
        AGB_TRY(check_ptr(mean, "mean", 4));
        AGB_TRY(check_ptr(rstd, "rstd", 4));
        AGB_TRY(check_ptr(gy, "gy", elem));
        AGB_TRY(check_ptr(dx_add, "dx_add", elem, false));
        AGB_TRY(check_ptr(dx, "dx", elem));
    }
    AGB_TRY(check_ptr(dgamma, "dgamma", 4, false));
    AGB_TRY(check_ptr(dbeta, "dbeta", 4, false));
    if (dgamma || dbeta) {
        AGB_TRY(check_ptr(workspace, "workspace", 8));
        const size_t need = agb_layernorm_affine_bwd_workspace_bytes(rows, hidden, dtype);
        if (workspace_bytes < need) return fail(AGB_ERR_WORKSPACE, "workspace %zu bytes, need %zu", workspace_bytes, need);
    }
    agb_int::Device d;
    AGB_TRY(agb_int::device(&d));
    agb::LnaBwdArgs a{x, gamma, mean, rstd, gy, dx_add, dx, rows, static_cast<int>(hidden), 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* part = static_cast<float*>(workspace);
    const int ub = unit_bytes(addr(x) | addr(gamma) | addr(gy) | addr(dx_add) | addr(dx), hidden * elem, elem);
    if (dtype == AGB_F32)
        return ub == 16 ? lna_bwd<float, 16>(a, dgamma, dbeta, accumulate, part, d, st) : lna_bwd<float, 4>(a, dgamma, dbeta, accumulate, part, d, st);
    return ub == 16 ? lna_bwd<bf16, 16>(a, dgamma, dbeta, accumulate, part, d, st) : lna_bwd<bf16, 2>(a, dgamma, dbeta, accumulate, part, d, st);
}

int agb_distill_topk_fwd(const void* z, const void* idx, int idx_type, const void* teacher, int teacher_dtype, float* loss, float* lse,
                         int64_t rows, int64_t vocab, int64_t k, float temperature, int dtype, agb_stream_t stream) {
    AGB_RANGE();
    return run_kd<0>(z, idx, idx_type, teacher, teacher_dtype, loss, lse, nullptr, nullptr, nullptr, rows, vocab, k, temperature, dtype,
                     stream);
}
int agb_distill_topk_bwd(const void* z, const void* idx, int idx_type, const void* teacher, int teacher_dtype, const float* lse,
                         const float* gy, const void* dz_add, void* dz, int64_t rows, int64_t vocab, int64_t k, float temperature,
                         int dtype, agb_stream_t stream) {
    AGB_RANGE();
    return run_kd<2>(z, idx, idx_type, teacher, teacher_dtype, nullptr, const_cast<float*>(lse), gy, dz_add, dz, rows, vocab, k, temperature,
                     dtype, stream);
}
int agb_distill_topk_fwd_bwd(const void* z, const void* idx, int idx_type, const void* teacher, int teacher_dtype, const float* gy,
                             const void* dz_add, float* loss, float* lse, void* dz, int64_t rows, int64_t vocab, int64_t k,
                             float temperature, int dtype, agb_stream_t stream) {
    AGB_RANGE();
    return run_kd<1>(z, idx, idx_type, teacher, teacher_dtype, loss, lse, gy, dz_add, dz, rows, vocab, k, temperature, dtype, stream);
}

}  // extern "C"
