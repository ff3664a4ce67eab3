// rules_vjp.cpp -- VJP rules of the RMSNorm path, one `void vjp_X(Node*, const Tensor& gy)` per op
// as in cgadimpl/src/autodiff/autodiff_vjp_ops.cpp, and the vjp_lookup table (:506-513).
// Every rule launches on the node's creation stream (the reference's current_stream() is
// thread-local and therefore null in the worker threads of the parallel backward).
#define AG_EXPOSE_AUTODIFF_RULES
#include <algorithm>
#include <vector>

#include "ad/detail/autodiff_ops.hpp"
#include "ad/detail/host_util.hpp"

namespace ag {
namespace detail {
namespace {

ag_cuda_stream_t rule_stream(Node* n) { return n->creation_context.stream; }

// P.grad += reduce_for_broadcast(g * a, P.value)   (a may be null: plain g)
// autodiff_vjp_ops.cpp:15-35 picks the axes to sum from the shapes; here the shape class does.
void accumulate_reduced(Node* P, const Tensor& g, const Tensor* a, ag_cuda_stream_t st) {
    std::unique_lock<std::mutex> lock(P->grad_mutex);
    bool first = false;
    Tensor& G = P->open_grad(&first);   // has P's shape even when P's value has been dropped
    int mode;
    try {
        mode = classify_broadcast(g, G);
    } catch (...) {
        if (first) P->grad_live = false;
        throw;
    }
    if (mode == AGB_BCAST_FULL) {
        if (first) P->grad_live = false;  // accumulate_grad opens the slot itself
        lock.unlock();
        P->accumulate_grad(a ? binary_op(1, g, *a, st) : g);
        return;
    }
    require_cuda(G, "broadcast gradient");
    const auto rh = rows_hidden(g);
    const size_t wsb = agb_mul_reduce_workspace_bytes(rh.rows, rh.hidden);
    void* ws = workspace(wsb, g, st);
    check_status(agb_mul_reduce(g.raw(), a ? a->raw() : nullptr, G.raw(), rh.rows, rh.hidden, mode, /*accumulate=*/first ? 0 : 1,
                                ws, wsb, agb_dtype(g), st),
                 "reduce_for_broadcast");
}

// X.grad += rms_vjp(x, gamma, rstd, gy): dx_add == dx == X.grad fuses accumulate_grad's `+=`; the FIRST
// contribution to X.grad is written instead (dx_add = NULL), so the buffer is neither zero-filled nor read.
// dgamma (fp32) is written to / accumulates into G->grad when G is given.
void norm_backward(Node* X, Node* G, const Tensor& rstd, const Tensor& gy, ag_cuda_stream_t st) {
    const Tensor& x = X->value;
    const auto rh = rows_hidden(x);
    const bool want_dx = X->requires_grad();
    const bool want_dg = G && G->requires_grad();
    if (!want_dx && !want_dg) return;
    if (want_dg && G->value.dtype() != Dtype::Float32)
        throw std::runtime_error("rmsnorm backward: dgamma is produced in fp32; a non-fp32 gamma node cannot "
                                 "receive it through the graph API (use agb_rmsnorm_bwd directly)");
    size_t wsb = 0;
    void* ws = nullptr;
    if (want_dg) {
        wsb = agb_rmsnorm_bwd_workspace_bytes(rh.rows, rh.hidden, agb_dtype(x));
        ws = workspace(wsb, x, st);
    }
    Tensor scratch_dx;
    if (!want_dx) scratch_dx = Tensor(x.shape(), ag::options(x).with_req_grad(false));
    std::unique_lock<std::mutex> lx(X->grad_mutex, std::defer_lock), lg;
    if (want_dx) lx.lock();
    if (want_dg) lg = std::unique_lock<std::mutex>(G->grad_mutex);
    bool first_dx = false, first_dg = false;
    Tensor* gx = want_dx ? &X->open_grad(&first_dx) : nullptr;
    Tensor* gg = want_dg ? &G->open_grad(&first_dg) : nullptr;
    check_status(agb_rmsnorm_bwd(x.raw(), G ? G->value.raw() : nullptr, rstd.data<float>(), gy.raw(),
                                 want_dx && !first_dx ? gx->raw() : nullptr, want_dx ? gx->raw() : scratch_dx.raw(),
                                 want_dg ? gg->raw() : nullptr, AGB_F32, /*accumulate_dgamma=*/first_dg ? 0 : 1, ws, wsb,
                                 rh.rows, rh.hidden, agb_dtype(x), st),
                 "rmsnorm backward");
}

// The locks of several parents in one order (two rules that share parents run at once in the parallel backward), a parent named
// twice locked once.
struct GradLocks {
    std::vector<std::unique_lock<std::mutex>> held;
    explicit GradLocks(std::vector<Node*> nodes) {
        std::sort(nodes.begin(), nodes.end());
        nodes.erase(std::unique(nodes.begin(), nodes.end()), nodes.end());
        for (Node* p : nodes)
            if (p) held.emplace_back(p->grad_mutex);
    }
};

// LayerNorm with weight and bias: dx is added in place (dx_add == dx), the column sums accumulate in fp32.
void layernorm_affine_backward(Node* n, const Tensor& gy, ag_cuda_stream_t st) {
    Node* X = n->inputs[0].get();
    Node* G = n->inputs[1].get();
    Node* B = n->inputs.size() > 2 ? n->inputs[2].get() : nullptr;
    const Tensor& x = X->value;
    const auto rh = rows_hidden(x);
    const bool want_dx = X->requires_grad(), want_dg = G->requires_grad(), want_db = B && B->requires_grad();
    if (!want_dx && !want_dg && !want_db) return;
    for (Node* p : {want_dg ? G : nullptr, want_db ? B : nullptr})
        if (p && p->value.dtype() != Dtype::Float32)
            throw std::runtime_error("layernorm backward: the gradients of gamma and beta are produced in fp32; a non-fp32 node cannot receive "
                                     "them through the graph API (use agb_layernorm_affine_bwd directly)");
    if ((want_dg && (G == X || G == B)) || (want_db && B == X))
        throw std::runtime_error("layernorm backward: x, gamma and beta must be different nodes");
    const size_t wsb = want_dg || want_db ? agb_layernorm_affine_bwd_workspace_bytes(rh.rows, rh.hidden, agb_dtype(x)) : 0;
    void* ws = wsb ? workspace(wsb, x, st) : nullptr;
    Tensor scratch;
    if (!want_dx) scratch = Tensor(x.shape(), ag::options(x).with_req_grad(false));
    GradLocks locks({want_dx ? X : nullptr, want_dg ? G : nullptr, want_db ? B : nullptr});
    bool first_dx = false, first_dg = false, first_db = false;
    Tensor* gx = want_dx ? &X->open_grad(&first_dx) : nullptr;
    Tensor* gg = want_dg ? &G->open_grad(&first_dg) : nullptr;
    Tensor* gb = want_db ? &B->open_grad(&first_db) : nullptr;
    if (gg && gb && first_dg != first_db) {            // one of the two has a contribution already: both add
        if (first_dg) gg->zero_();
        else gb->zero_();
        first_dg = first_db = false;
    }
    const bool add_columns = gg ? !first_dg : !first_db;
    check_status(agb_layernorm_affine_bwd(x.raw(), G->value.raw(), n->tape[0]->data<float>(), n->tape[1]->data<float>(), gy.raw(),
                                          want_dx && !first_dx ? gx->raw() : nullptr, want_dx ? gx->raw() : scratch.raw(),
                                          gg ? gg->data<float>() : nullptr, gb ? gb->data<float>() : nullptr, add_columns ? 1 : 0, ws, wsb,
                                          rh.rows, rh.hidden, agb_dtype(x), st),
                 "layernorm backward");
}

[[noreturn]] void not_on_path(const char* what, const char* name) {
    throw std::runtime_error(std::string(what) + " for op '" + name + "' is not part of the RMSNorm path of this library");
}

}  // namespace

void vjp_Leaf(Node*, const Tensor&) {}

// autodiff_vjp_ops.cpp:40-45
void vjp_Add(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    for (int i = 0; i < 2; ++i) {
        Node* P = n->inputs[i].get();
        if (P->requires_grad()) accumulate_reduced(P, gy, nullptr, rule_stream(n));
    }
}

// autodiff_vjp_ops.cpp:54-59
void vjp_Mul(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* A = n->inputs[0].get();
    Node* B = n->inputs[1].get();
    if (A->requires_grad()) {
        const Tensor b = on_device_of(B->value, gy);
        if (classify_broadcast(gy, A->value) == AGB_BCAST_FULL) A->accumulate_grad(binary_op(1, gy, b, rule_stream(n)));
        else accumulate_reduced(A, gy, &b, rule_stream(n));
    }
    if (B->requires_grad()) {
        const Tensor a = on_device_of(A->value, gy);
        if (classify_broadcast(gy, B->value) == AGB_BCAST_FULL) B->accumulate_grad(binary_op(1, gy, a, rule_stream(n)));
        else accumulate_reduced(B, gy, &a, rule_stream(n));
    }
}

// autodiff_vjp_ops.cpp:351-365; X.grad += dx fused through dx_add == dx == X.grad
void vjp_LayerNorm(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    if (n->inputs.size() > 1) {
        layernorm_affine_backward(n, gy, rule_stream(n));
        return;
    }
    Node* X = n->inputs[0].get();
    if (!X->requires_grad()) return;
    const auto rh = rows_hidden(X->value);
    std::lock_guard<std::mutex> lock(X->grad_mutex);
    bool first = false;
    Tensor& G = X->open_grad(&first);
    check_status(agb_layernorm_bwd(X->value.raw(), n->tape[1]->data<float>(), n->tape[0]->data<float>(), gy.raw(),
                                   first ? nullptr : G.raw(), G.raw(), rh.rows, rh.hidden, n->eps, agb_dtype(X->value),
                                   rule_stream(n)),
                 "laynor backward");
}

// autodiff_vjp_ops.cpp:368-377
void vjp_RMSNorm(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    norm_backward(n->inputs[0].get(), nullptr, *n->tape[0], gy, rule_stream(n));
}

void vjp_RMSNormAffine(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    norm_backward(n->inputs[0].get(), n->inputs[1].get(), *n->tape[0], gy, rule_stream(n));
}

// The reference throws here (autodiff_vjp_ops.cpp:379-381).  y = yhat * G with a scalar G:
// dyhat = gy * G -> through the norm;  dG = sum(gy * yhat).
void vjp_RealRMSNorm(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* X = n->inputs[0].get();
    Node* G = n->inputs[1].get();
    if (X->requires_grad()) {
        Tensor dyhat = binary_op(1, gy, G->value, rule_stream(n));
        norm_backward(X, nullptr, *n->tape[0], dyhat, rule_stream(n));
    }
    if (G->requires_grad()) accumulate_reduced(G, gy, n->tape[1].get(), rule_stream(n));
}

// autodiff_vjp_ops.cpp:399-402: X.grad += gy (scalar broadcast)
void vjp_Sum(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* X = n->inputs[0].get();
    if (X->requires_grad()) X->accumulate_grad(gy);
}
// autodiff_vjp_ops.cpp:403-409: X.grad += gy * (1/numel)
void vjp_MeanAll(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* X = n->inputs[0].get();
    if (!X->requires_grad()) return;
    std::lock_guard<std::mutex> lock(X->grad_mutex);
    bool first = false;
    Tensor& G = X->open_grad(&first);
    if (first) G.zero_();
    const float scale = 1.0f / static_cast<float>(G.numel());
    const auto rh = rows_hidden(G);
    const Tensor src = on_device_of(gy, G);
    check_status(agb_accumulate_broadcast(G.raw(), src.raw(), rh.rows, rh.hidden, AGB_BCAST_SCALAR, scale,
                                          agb_dtype(G), rule_stream(n)),
                 "vjp_MeanAll");
}
// autodiff_vjp_ops.cpp:411-414: X.grad += gy ([B,1] broadcast)
void vjp_RowSum(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* X = n->inputs[0].get();
    if (X->requires_grad()) X->accumulate_grad(gy);
}
// autodiff_vjp_ops.cpp:416-418 throws as well
void vjp_RowMax(Node*, const Tensor&) { throw std::runtime_error("VJP for RowMax not implemented yet!"); }

// autodiff_vjp_ops.cpp:421-428: Z.grad += y * (gy - sum(y*gy)); the `+=` is fused (dz_add == dz == Z.grad)
void vjp_SoftmaxRow(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* Z = n->inputs[0].get();
    if (!Z->requires_grad()) return;
    const auto rh = rows_hidden(n->value);
    std::lock_guard<std::mutex> lock(Z->grad_mutex);
    bool first = false;
    Tensor& G = Z->open_grad(&first);
    check_status(agb_softmax_row_bwd(n->value.raw(), gy.raw(), first ? nullptr : G.raw(), G.raw(), rh.rows, rh.hidden,
                                     agb_dtype(n->value), rule_stream(n)),
                 "vjp_SoftmaxRow");
}
// autodiff_vjp_ops.cpp:430-440: softmax(z) recomputed from Z.value; Z.grad += gy[.., 1] * softmax(z)
void vjp_LogSumExpRow(Node* n, const Tensor& gy) {
    StreamGuard g(rule_stream(n));
    Node* Z = n->inputs[0].get();
    if (!Z->requires_grad()) return;
    const auto rh = rows_hidden(Z->value);
    if (gy.numel() != rh.rows) throw std::runtime_error("vjp_LogSumExpRow: gy must have one entry per row");
    std::lock_guard<std::mutex> lock(Z->grad_mutex);
    bool first = false;
    Tensor& G = Z->open_grad(&first);
    check_status(agb_logsumexp_row_bwd(Z->value.raw(), gy.raw(), first ? nullptr : G.raw(), G.raw(), rh.rows, rh.hidden,
                                       agb_dtype(Z->value), rule_stream(n)),
                 "vjp_LogSumExpRow");
}

// dh = g w, dw = g' h with the logits computed again; dw accumulates in place, a second contribution to h goes through a buffer.
void vjp_CeWithLogits(Node* n, const Tensor& gy) {
    if (n->inputs.size() < 3) not_on_path("VJP", "CeWithLogits");
    StreamGuard g(rule_stream(n));
    Node* Hn = n->inputs[0].get();
    Node* Wn = n->inputs[1].get();
    const Tensor &h = Hn->value, &w = Wn->value, &target = n->inputs[2]->value;
    const bool want_dh = Hn->requires_grad(), want_dw = Wn->requires_grad();
    if (!want_dh && !want_dw) return;
    const auto rh = rows_hidden(h);
    if (gy.numel() != rh.rows || gy.dtype() != Dtype::Float32)
        throw std::runtime_error("vjp_CeWithLogits: gy must have one fp32 entry per row");
    if (Hn == Wn) throw std::runtime_error("vjp_CeWithLogits: h and w must be different nodes");
    const int64_t vocab = w.shape().dims[0];
    const size_t wsb = agb_linear_ce_workspace_bytes(1, rh.rows, rh.hidden, vocab, agb_dtype(h));
    void* ws = workspace(wsb, h, rule_stream(n));
    Tensor dh;
    {
        GradLocks locks({want_dh ? Hn : nullptr, want_dw ? Wn : nullptr});
        bool first_dh = false, first_dw = false;
        Tensor* gh = want_dh ? &Hn->open_grad(&first_dh) : nullptr;
        Tensor* gw = want_dw ? &Wn->open_grad(&first_dw) : nullptr;
        if (want_dh && !first_dh) dh = Tensor(h.shape(), ag::options(h).with_req_grad(false));
        check_status(agb_linear_ce_bwd(h.raw(), w.raw(), target.raw(), agb_index(target, "vjp_CeWithLogits"), n->tape[0]->data<float>(),
                                       gy.data<float>(), want_dh ? (first_dh ? gh->raw() : dh.raw()) : nullptr, want_dw ? gw->raw() : nullptr,
                                       want_dw && !first_dw ? 1 : 0, rh.rows, rh.hidden, vocab, agb_dtype(h), ws, wsb, rule_stream(n)),
                     "vjp_CeWithLogits");
    }
    if (dh.defined()) Hn->accumulate_grad(dh);
}

// dz = gy * t * (softmax(z / t) - the teacher's shares), added in place.
void vjp_KLDivergence(Node* n, const Tensor& gy) {
    if (n->inputs.size() < 3) not_on_path("VJP", "KLDivergence");
    StreamGuard g(rule_stream(n));
    Node* Z = n->inputs[0].get();
    if (!Z->requires_grad()) return;
    const Tensor &idx = n->inputs[1]->value, &teacher = n->inputs[2]->value;
    const auto rh = rows_hidden(Z->value);
    if (gy.numel() != rh.rows || gy.dtype() != Dtype::Float32)
        throw std::runtime_error("vjp_KLDivergence: gy must have one fp32 entry per row");
    std::lock_guard<std::mutex> lock(Z->grad_mutex);
    bool first = false;
    Tensor& G = Z->open_grad(&first);
    check_status(agb_distill_topk_bwd(Z->value.raw(), idx.raw(), agb_index(idx, "vjp_KLDivergence"), teacher.raw(), agb_dtype(teacher),
                                      n->tape[0]->data<float>(), gy.data<float>(), first ? nullptr : G.raw(), G.raw(), rh.rows, rh.hidden,
                                      idx.numel() / rh.rows, n->eps, agb_dtype(Z->value), rule_stream(n)),
                 "vjp_KLDivergence");
}

#define AG_NOT_ON_PATH(name) \
    void vjp_##name(Node*, const Tensor&) { not_on_path("VJP", #name); }
AG_NOT_ON_PATH(Sub) AG_NOT_ON_PATH(Div) AG_NOT_ON_PATH(Exp) AG_NOT_ON_PATH(Log) AG_NOT_ON_PATH(Sqrt)
AG_NOT_ON_PATH(Reciprocal) AG_NOT_ON_PATH(Sign) AG_NOT_ON_PATH(Abs) AG_NOT_ON_PATH(Pow) AG_NOT_ON_PATH(Sin)
AG_NOT_ON_PATH(Cos) AG_NOT_ON_PATH(Tan) AG_NOT_ON_PATH(Sinh) AG_NOT_ON_PATH(Cosh) AG_NOT_ON_PATH(Asin)
AG_NOT_ON_PATH(Acos) AG_NOT_ON_PATH(Atan) AG_NOT_ON_PATH(ASinh) AG_NOT_ON_PATH(ACosh) AG_NOT_ON_PATH(ATanh)
AG_NOT_ON_PATH(Relu) AG_NOT_ON_PATH(Sigmoid) AG_NOT_ON_PATH(Tanh) AG_NOT_ON_PATH(Softplus) AG_NOT_ON_PATH(GELU)
AG_NOT_ON_PATH(SiLU) AG_NOT_ON_PATH(Mish) AG_NOT_ON_PATH(LeakyRelu) AG_NOT_ON_PATH(Gaus) AG_NOT_ON_PATH(Parcon)
AG_NOT_ON_PATH(LiSHT) AG_NOT_ON_PATH(MatMul)
AG_NOT_ON_PATH(Transpose) AG_NOT_ON_PATH(Linear) AG_NOT_ON_PATH(FMA) AG_NOT_ON_PATH(Dyntanh)
AG_NOT_ON_PATH(Attention) AG_NOT_ON_PATH(SWIGLU)
AG_NOT_ON_PATH(MSELoss) AG_NOT_ON_PATH(MAELoss)
#undef AG_NOT_ON_PATH

}  // namespace detail

VjpFn vjp_lookup(Op op) {
    switch (op) {
#define OP(name, arity, str) \
    case Op::name: return &detail::vjp_##name;
#include "ad/detail/ops.def"
#undef OP
        default: return nullptr;
    }
}

}  // namespace ag
