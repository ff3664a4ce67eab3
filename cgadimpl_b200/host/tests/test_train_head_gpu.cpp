// test_train_head_gpu.cpp -- the end of a model through the graph API, as a training step uses it: LayerNorm with weight and bias, the
// vocabulary loss on top of it, a distillation loss beside it.  Values and gradients against the same composition in double on the CPU;
// tolerances count the fp32 roundings of the sums (2^-24 a term, sums of at most a few thousand terms of size 1).
#include <cmath>
#include <cstdint>

#include "ad/ag_all.hpp"
#include "check.hpp"

using namespace ag;
static const auto kDev = DeviceIndex(Device::CUDA);
typedef std::vector<double> Vd;

static Vd wide(const std::vector<float>& v) { return Vd(v.begin(), v.end()); }
static bool near(const std::vector<float>& got, const Vd& want, double tol, const char* what) {
    if (got.size() != want.size()) return false;
    for (size_t i = 0; i < got.size(); ++i)
        if (!(std::abs(got[i] - want[i]) <= tol)) {
            std::fprintf(stderr, "  %s[%zu]: %.9g, want %.9g (tolerance %.3g)\n", what, i, got[i], want[i], tol);
            return false;
        }
    return true;
}

int main() {
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) { std::printf("no CUDA device\n"); return 2; }
    OwnTensor::manual_seed(5);
    const int64_t R = 37, H = 72, V = 203, K = 5;
    const auto opt = TensorOptions().with_device(kDev), grad = opt.with_req_grad(true);
    std::vector<int64_t> target(R), idx(R * K);
    for (int64_t r = 0; r < R; ++r) target[r] = r % 6 == 2 ? -100 : (r * 67) % V;
    for (int64_t i = 0; i < R * K; ++i) idx[i] = i % 7 == 3 ? -1 : (i * 31) % V;
    const double eps = 1e-5, tau = 2.0;

    // the step in double: loss = mean(ce) + sum(kd) * 0.1, gradients by the formulas
    struct Ref { Vd y, ce, kd, dx, dgamma, dbeta, dw, dz; };
    auto reference = [&](const Vd& x, const Vd& gamma, const Vd& beta, const Vd& w, const Vd& z, const Vd& teacher, double ce_scale, double kd_scale) {
        Ref o;
        o.y.resize(R * H); o.ce.assign(R, 0); o.kd.assign(R, 0); o.dx.assign(R * H, 0); o.dgamma.assign(H, 0); o.dbeta.assign(H, 0);
        o.dw.assign(V * H, 0); o.dz.assign(R * V, 0);
        for (int64_t r = 0; r < R; ++r) {
            double mean = 0, var = 0;
            for (int64_t j = 0; j < H; ++j) mean += x[r * H + j] / H;
            for (int64_t j = 0; j < H; ++j) var += (x[r * H + j] - mean) * (x[r * H + j] - mean) / H;
            const double rstd = 1 / std::sqrt(var + eps);
            Vd xh(H), dy(H, 0.0);
            for (int64_t j = 0; j < H; ++j) { xh[j] = (x[r * H + j] - mean) * rstd; o.y[r * H + j] = xh[j] * gamma[j] + beta[j]; }
            if (target[r] >= 0) {
                Vd p(V);
                double top = -1e300, s = 0;
                for (int64_t v = 0; v < V; ++v) { p[v] = 0; for (int64_t j = 0; j < H; ++j) p[v] += o.y[r * H + j] * w[v * H + j]; top = std::max(top, p[v]); }
                for (int64_t v = 0; v < V; ++v) s += std::exp(p[v] - top);
                const double lse = top + std::log(s);
                o.ce[r] = lse - p[target[r]];
                for (int64_t v = 0; v < V; ++v) {
                    const double g = ce_scale * (std::exp(p[v] - lse) - (v == target[r]));
                    for (int64_t j = 0; j < H; ++j) { dy[j] += g * w[v * H + j]; o.dw[v * H + j] += g * o.y[r * H + j]; }
                }
            }
            double a = 0, b = 0;
            for (int64_t j = 0; j < H; ++j) { a += dy[j] * gamma[j] / H; b += dy[j] * gamma[j] * xh[j] / H; o.dgamma[j] += dy[j] * xh[j]; o.dbeta[j] += dy[j]; }
            for (int64_t j = 0; j < H; ++j) o.dx[r * H + j] = rstd * (dy[j] * gamma[j] - a - xh[j] * b);
            double ttop = -1e300, ts = 0, ztop = -1e300, zs = 0;
            for (int64_t k = 0; k < K; ++k) if (idx[r * K + k] >= 0) ttop = std::max(ttop, teacher[r * K + k] / tau);
            for (int64_t k = 0; k < K; ++k) if (idx[r * K + k] >= 0) ts += std::exp(teacher[r * K + k] / tau - ttop);
            for (int64_t v = 0; v < V; ++v) ztop = std::max(ztop, z[r * V + v] / tau);
            for (int64_t v = 0; v < V; ++v) zs += std::exp(z[r * V + v] / tau - ztop);
            const double zl = ztop + std::log(zs), tl = ttop + std::log(ts);
            for (int64_t v = 0; v < V; ++v) o.dz[r * V + v] = kd_scale * tau * std::exp(z[r * V + v] / tau - zl);
            for (int64_t k = 0; k < K; ++k) {
                const int64_t v = idx[r * K + k];
                if (v < 0) continue;
                const double lp = teacher[r * K + k] / tau - tl, q = std::exp(lp);
                o.kd[r] += tau * tau * q * (lp - (z[r * V + v] / tau - zl));
                o.dz[r * V + v] -= kd_scale * tau * q;
            }
        }
        return o;
    };

    run_test("norm, vocabulary loss and distillation in one step", [&] {
        nn::LayerNorm norm(H);
        norm.gamma().val().copy_(Tensor::rand(Shape{{H}}, opt));
        norm.beta().val().copy_(Tensor::randn(Shape{{H}}, opt));
        Value x = make_tensor(Tensor::randn(Shape{{R, H}}, grad)), w = make_tensor(Tensor::randn(Shape{{V, H}}, grad));
        Value z = make_tensor(Tensor::randn(Shape{{R, V}}, grad));
        const Tensor t = Tensor::from_host(target.data(), Shape{{R}}, opt.with_dtype(Dtype::Int64));
        const Tensor cols = Tensor::from_host(idx.data(), Shape{{R, K}}, opt.with_dtype(Dtype::Int32));
        const Tensor teacher = Tensor::randn(Shape{{R, K}}, opt);
        Value scale = make_tensor(Tensor::full(Shape{{1}}, opt, 0.1f));
        Ref ref = reference(wide(x.val().to_vector()), wide(norm.gamma().val().to_vector()), wide(norm.beta().val().to_vector()),
                            wide(w.val().to_vector()), wide(z.val().to_vector()), wide(teacher.to_vector()), 1.0 / R, double(0.1f));
        for (int pass = 0; pass < 2; ++pass) {          // the second pass writes over the first one's gradients
            norm.zero_grad();
            Value y = norm(x), ce = linear_cross_entropy(y, w, t), kd = distill_topk(z, cols, teacher, float(tau));
            CHECK(ce.node->op == Op::CeWithLogits && kd.node->op == Op::KLDivergence && y.node->op == Op::LayerNorm);
            CHECK(ce.shape() == (std::vector<int64_t>{R, 1}));
            Value loss = add(mean_all(ce), sum(kd) * scale);
            zero_grad(loss);
            backward(loss, nullptr, pass == 1);
            CHECK(near(y.val().to_vector(), ref.y, 1e-5, "y") && near(ce.val().to_vector(), ref.ce, 2e-4, "ce"));
            CHECK(near(kd.val().to_vector(), ref.kd, 1e-4, "kd") && near(z.grad().to_vector(), ref.dz, 1e-5, "dz"));
            CHECK(near(w.grad().to_vector(), ref.dw, 2e-4, "dw") && near(x.grad().to_vector(), ref.dx, 2e-4, "dx"));
            CHECK(near(norm.gamma().grad().to_vector(), ref.dgamma, 5e-4, "dgamma"));
            CHECK(near(norm.beta().grad().to_vector(), ref.dbeta, 5e-4, "dbeta"));
        }
    });

    run_test("contributions add: a shared head, shared logits and a shared norm", [&] {
        Value x = make_tensor(Tensor::randn(Shape{{R, H}}, grad)), w = make_tensor(Tensor::randn(Shape{{V, H}}, grad));
        Value g = make_tensor(Tensor::ones(Shape{{H}}, grad)), b = make_tensor(Tensor::zeros(Shape{{H}}, grad));
        Value z = make_tensor(Tensor::randn(Shape{{R, V}}, grad));
        const Tensor t = Tensor::from_host(target.data(), Shape{{R}}, opt.with_dtype(Dtype::Int32));
        const Tensor cols = Tensor::from_host(idx.data(), Shape{{R, K}}, opt.with_dtype(Dtype::Int64));
        const Tensor teacher = Tensor::randn(Shape{{R, K}}, opt);
        auto once = [&](int times) {
            Value total;
            for (int i = 0; i < times; ++i) {
                Value part = add(sum(linear_cross_entropy(layernorm(x, g, b), w, t)), sum(distill_topk(z, cols, teacher)));
                total = i ? add(total, part) : part;
            }
            zero_grad(total);
            backward(total);
            std::vector<std::vector<float>> out;
            for (Value* v : {&x, &w, &g, &b, &z}) out.push_back(v->grad().to_vector());
            return out;
        };
        auto one = once(1), two = once(2);
        for (size_t i = 0; i < one.size(); ++i) {
            Vd want = wide(one[i]);
            double top = 0;
            for (double& v : want) { v *= 2; top = std::max(top, std::abs(v)); }
            CHECK(near(two[i], want, 1e-5 * top + 1e-6, "twice"));
        }
        Value h = make_tensor(Tensor::randn(Shape{{R, H}}, grad));       // h used twice by the same head
        auto grad_h = [&](int times) {
            Value total;
            for (int i = 0; i < times; ++i) { Value p = sum(linear_cross_entropy(h, w, t)); total = i ? add(total, p) : p; }
            zero_grad(total);
            backward(total);
            return h.grad().to_vector();
        };
        Vd want = wide(grad_h(1));
        for (double& v : want) v *= 2;
        CHECK(near(grad_h(2), want, 1e-4, "dh twice"));
    });

    run_test("recompute gives the same bits; the tangent of the norm agrees with differences", [&] {
        Value x = make_tensor(Tensor::randn(Shape{{R, H}}, grad)), w = make_tensor(Tensor::randn(Shape{{V, H}}, grad));
        Value g = make_tensor(Tensor::rand(Shape{{H}}, grad)), b = make_tensor(Tensor::randn(Shape{{H}}, grad));
        const Tensor t = Tensor::from_host(target.data(), Shape{{R}}, opt.with_dtype(Dtype::Int64));
        Value y = layernorm(x, g, b, 1e-3f), ce = linear_cross_entropy(y, w, t);
        const auto yv = y.val().to_vector(), cv = ce.val().to_vector();
        CHECK(forward_eval_node(y.node).to_vector() == yv && forward_eval_node(ce.node).to_vector() == cv);
        const Tensor dx = Tensor::randn(Shape{{R, H}}, opt), dg = Tensor::randn(Shape{{H}}, opt), db = Tensor::randn(Shape{{H}}, opt);
        const std::function<const Tensor&(Node*)> tangent = [&](Node* p) -> const Tensor& { return p == x.node.get() ? dx : p == g.node.get() ? dg : db; };
        const auto ty = jvp_lookup(Op::LayerNorm)(y.node.get(), tangent).to_vector();
        const Vd xv = wide(x.val().to_vector()), gv = wide(g.val().to_vector()), bv = wide(b.val().to_vector());
        const Vd tx = wide(dx.to_vector()), tg = wide(dg.to_vector()), tb = wide(db.to_vector());
        auto value = [&](double s) {
            Vd o(R * H);
            for (int64_t r = 0; r < R; ++r) {
                double mean = 0, var = 0;
                for (int64_t j = 0; j < H; ++j) mean += (xv[r * H + j] + s * tx[r * H + j]) / H;
                for (int64_t j = 0; j < H; ++j) { const double c = xv[r * H + j] + s * tx[r * H + j] - mean; var += c * c / H; }
                for (int64_t j = 0; j < H; ++j)
                    o[r * H + j] = (xv[r * H + j] + s * tx[r * H + j] - mean) / std::sqrt(var + double(1e-3f)) * (gv[j] + s * tg[j]) + bv[j] + s * tb[j];
            }
            return o;
        };
        Vd up = value(1e-5), down = value(-1e-5);
        for (size_t i = 0; i < up.size(); ++i) up[i] = (up[i] - down[i]) / 2e-5;
        CHECK(near(ty, up, 1e-4, "ty"));
    });

    run_test("what does not fit is refused", [&] {
        Value x = make_tensor(Tensor::randn(Shape{{R, H}}, grad)), w = make_tensor(Tensor::randn(Shape{{V, H + 1}}, grad));
        Value g = make_tensor(Tensor::ones(Shape{{H + 1}}, grad)), z = make_tensor(Tensor::randn(Shape{{R, V}}, grad));
        const Tensor t = Tensor::from_host(target.data(), Shape{{R}}, opt.with_dtype(Dtype::Int64));
        const Tensor cols = Tensor::from_host(idx.data(), Shape{{R, K}}, opt.with_dtype(Dtype::Int32));
        auto refused = [](const std::function<void()>& f) {
            try { f(); } catch (const std::exception&) { return true; }
            return false;
        };
        CHECK(refused([&] { layernorm(x, g); }));
        CHECK(refused([&] { linear_cross_entropy(x, w, t); }));
        CHECK(refused([&] { linear_cross_entropy(x, x, x.val()); }));
        CHECK(refused([&] { distill_topk(z, cols, t); }));
        CHECK(refused([&] { distill_topk(z, z.val(), Tensor::randn(Shape{{R, V}}, opt)); }));
        CHECK(refused([&] { distill_topk(z, cols, Tensor::randn(Shape{{R, K}}, opt), 0.f); }));
        CHECK(refused([&] { Tensor::from_host(target.data(), Shape{{R}}, opt); }));
        Value h16 = make_tensor(Tensor::randn(Shape{{R, H}}, grad.with_dtype(Dtype::Bfloat16)));
        Value g16 = make_tensor(Tensor::ones(Shape{{H}}, grad.with_dtype(Dtype::Bfloat16)));
        Value y = layernorm(h16, g16);
        CHECK(refused([&] { backward(sum(y)); }));      // a 16-bit weight cannot take the fp32 column sums
    });
    cudaDeviceSynchronize();
    return finish("test_train_head_gpu");
}
