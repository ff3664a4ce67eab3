// agb_train.cu -- the operators at the end of a model, behind the C ABI of include/agb/agb.h: LayerNorm with weight and
// bias, softmax cross entropy taken from the hidden states, distillation from a teacher's largest logits.
#define AGB_NO_STATUS_WORD
#include <nvtx3/nvToolsExt.h>

#include "agb/agb.h"
#include "agb_internal.h"
#include "distill_topk.cuh"
#include "layernorm_affine.cuh"

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

// Threads per row for `units` units at `upt` per thread: a power of two up to a warp, else whole warps; 0: too many.
inline int threads_per_row(int64_t units, int upt, int limit) {
    const int64_t want = ceil_div(units, upt);
    if (want <= 32) {
        int g = 1;
        while (g < want) g *= 2;
        return g;
    }
    const int64_t g = ceil_div(want, 32) * 32;
    return g > limit ? 0 : static_cast<int>(g);
}
inline int64_t grid_for(int64_t rows, int G, int block, int sms, int per_sm) {
    const int64_t want = ceil_div(rows, G <= 32 ? block / G : 1), cap = static_cast<int64_t>(sms) * per_sm;
    return want < cap ? want : cap;
}

template <typename T, int UB>
int lna_fwd(agb::LnaFwdArgs a, int sms, cudaStream_t st) {
    constexpr int N = agb::Unit<T, UB>::N, UPT = 32 / N;
    a.G = threads_per_row(a.hidden / N, UPT, 512);
    if (a.G) {
        const int block = a.G <= 32 ? 128 : a.G;
        agb::lna_fwd_kernel<T, UB, UPT><<<static_cast<unsigned>(grid_for(a.rows, a.G, block, sms, 2048 / block)), block, 0, st>>>(a);
    } else {
        agb::lna_fwd_wide<T, UB><<<static_cast<unsigned>(grid_for(a.rows, 1024, 1024, sms, 2)), 1024, 0, st>>>(a);
    }
    return after_launch("layernorm_affine_fwd");
}

template <typename T, int UB>
int lna_dx(agb::LnaBwdArgs a, int sms, cudaStream_t st) {
    constexpr int N = agb::Unit<T, UB>::N, UPT = 16 / N;
    a.G = threads_per_row(a.hidden / N, UPT, 512);
    if (a.G) {
        const int block = a.G <= 32 ? 128 : a.G;
        agb::lna_dx_kernel<T, UB, UPT><<<static_cast<unsigned>(grid_for(a.rows, a.G, block, sms, 2048 / block)), block, 0, st>>>(a);
    } else {
        agb::lna_dx_wide<T, UB><<<static_cast<unsigned>(grid_for(a.rows, 1024, 1024, sms, 2)), 1024, 0, st>>>(a);
    }
    return after_launch("layernorm_affine_bwd");
}

constexpr int kLnaRuns = 64;   // runs of rows of the column sums, each a partial row

template <typename T>
int lna_bwd(const agb::LnaBwdArgs& a, float* dgamma, float* dbeta, int accumulate, float* partial, cudaStream_t st) {
    agb_int::Device d;
    AGB_TRY(agb_int::device(&d));
    const int ub = unit_bytes(addr(a.x) | addr(a.gamma) | addr(a.gy) | addr(a.dx_add) | addr(a.dx), a.hidden * (int)sizeof(T), sizeof(T));
    const int64_t run = a.rows > 0 ? ceil_div(a.rows, kLnaRuns) : 1;
    const int runs = static_cast<int>(ceil_div(a.rows, run));
    const bool columns = dgamma || dbeta;
    if (columns && runs > 0) {
        agb::lna_columns<T><<<dim3(static_cast<unsigned>(ceil_div(a.hidden, 256)), runs), 256, 0, st>>>(
            static_cast<const T*>(a.x), static_cast<const T*>(a.gy), a.mean, a.rstd, partial, a.rows, a.hidden, run);
        AGB_TRY(after_launch("layernorm_affine_columns"));
    }
    if (a.rows > 0)
        AGB_TRY((ub == 16 ? lna_dx<T, 16>(a, d.sms, st) : ub == 4 ? lna_dx<T, 4>(a, d.sms, st) : lna_dx<T, sizeof(T)>(a, d.sms, st)));
    if (!columns) return AGB_OK;
    agb::lna_column_reduce<<<static_cast<unsigned>(ceil_div(2LL * a.hidden, 32)), dim3(32, 8), 0, st>>>(partial, runs, a.hidden, dgamma,
                                                                                                dbeta, accumulate);
    return after_launch("layernorm_affine_column_reduce");
}

// ------------------------------------------------------------------ distillation
int check_kd(int64_t rows, int64_t vocab, int64_t k, float tau, int dtype, int idx_type, int teacher_dtype) {
    if (rows < 0 || vocab <= 0 || k <= 0)
        return fail(AGB_ERR_INVALID_ARG, "rows=%lld vocab=%lld k=%lld", (long long)rows, (long long)vocab, (long long)k);
    if (!(tau > 0.f) || !(tau < INFINITY)) return fail(AGB_ERR_INVALID_ARG, "temperature %g must be positive and finite", (double)tau);
    if (dtype != AGB_F32 && dtype != AGB_BF16) return fail(AGB_ERR_UNSUPPORTED, "dtype %d (only AGB_F32, AGB_BF16)", dtype);
    if (teacher_dtype != AGB_F32 && teacher_dtype != AGB_BF16)
        return fail(AGB_ERR_UNSUPPORTED, "teacher_dtype %d (only AGB_F32, AGB_BF16)", teacher_dtype);
    if (idx_type != AGB_I32 && idx_type != AGB_I64) return fail(AGB_ERR_INVALID_ARG, "idx_type %d (AGB_I32 or AGB_I64)", idx_type);
    if (vocab > (1LL << 30)) return fail(AGB_ERR_UNSUPPORTED, "vocab %lld too large", (long long)vocab);
    if (k > agb::kKdMaxK) return fail(AGB_ERR_UNSUPPORTED, "k=%lld (at most %d)", (long long)k, agb::kKdMaxK);
    if (rows > (1LL << 27)) return fail(AGB_ERR_UNSUPPORTED, "rows=%lld (at most 2^27)", (long long)rows);
    return AGB_OK;
}

template <typename T, int MODE>
int launch_kd(agb::KdArgs a, int64_t rows, cudaStream_t st) {
    agb_int::Device d;
    AGB_TRY(agb_int::device(&d));
    // Slices per row: enough CTAs for the GPU where rows are few, none shorter than one turn of the block.
    int C = 1;
    while (C < 8 && rows * C < 2 * d.sms && a.vocab / (2 * C) >= agb::kKdThreads * (16 / static_cast<int>(sizeof(T)))) C *= 2;
    a.slice = ceil_div(ceil_div(a.vocab, C), 64) * 64;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * C));
    cfg.blockDim = dim3(agb::kKdThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    AGB_CUDA(cudaLaunchKernelEx(&cfg, agb::kd_kernel<T, MODE>, a));
    return after_launch("distill_topk");
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
    agb::KdArgs a{z, idx, teacher, idx_type == AGB_I64, teacher_dtype == AGB_BF16, loss, lse, gy, dz_add, dz, vocab, static_cast<int>(k),
                  tau, 1.f / tau, 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == AGB_F32 ? launch_kd<float, MODE>(a, rows, st) : launch_kd<bf16, MODE>(a, rows, st);
}

}  // namespace

extern "C" {

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
    if (dtype == AGB_F32) return ub == 16 ? lna_fwd<float, 16>(a, d.sms, st) : lna_fwd<float, 4>(a, d.sms, st);
    return ub == 16 ? lna_fwd<bf16, 16>(a, d.sms, st) : ub == 4 ? lna_fwd<bf16, 4>(a, d.sms, st) : lna_fwd<bf16, 2>(a, d.sms, st);
}

size_t agb_layernorm_affine_bwd_workspace_bytes(int64_t rows, int64_t hidden, int dtype) {
    (void)rows;
    (void)dtype;
    return hidden <= 0 ? 0 : static_cast<size_t>(kLnaRuns) * 2 * hidden * sizeof(float);
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
    agb::LnaBwdArgs a{x, gamma, mean, rstd, gy, dx_add, dx, rows, static_cast<int>(hidden), 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == AGB_F32 ? lna_bwd<float>(a, dgamma, dbeta, accumulate, static_cast<float*>(workspace), st)
                            : lna_bwd<bf16>(a, dgamma, dbeta, accumulate, static_cast<float*>(workspace), st);
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
