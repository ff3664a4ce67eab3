"""The operators at the end of a model run together, as a training step uses them: LayerNorm with weight and bias, the vocabulary loss on
its output, a distillation loss on logits of the same output; through the Python wrappers here, through the graph API in
cgadimpl_b200/host/tests/test_train_head_gpu.cpp."""
import os
import subprocess

import pytest
import torch

from cgadimpl_b200.host import build as host_build


@pytest.mark.gpu
def test_graph_api():
    host_build.build()
    exe = os.path.join(os.path.dirname(host_build.__file__), "build", "test_train_head_gpu")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "all passed" in out and "[FAIL]" not in out, out


def make(dtype, rows=300, hidden=136, vocab=1003, k=9, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = (n(rows, hidden) + 0.3).to(dtype)
    gamma, beta = (1 + 0.1 * n(hidden)).to(dtype), (0.1 * n(hidden)).to(dtype)
    w = (n(vocab, hidden) * hidden ** -0.5).to(dtype)
    target = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    target[::5] = -100
    idx = torch.rand(rows, vocab, device="cuda", generator=g).argsort(-1)[:, :k].contiguous()
    idx[::7, 3:] = -1
    idx[::11] = -1
    return x, gamma, beta, w, target, idx, n(rows, k)


def step(ops, x, gamma, beta, w, target, idx, teacher, tau=2.0, share=0.3):
    rows = x.shape[0]
    y, mean, rstd = ops.layernorm_affine_fwd(x, gamma, beta)
    each = torch.full((rows,), 1.0 / rows, device=x.device)
    ce, lse = ops.linear_ce_fwd(y, w, target)
    dy, dw = ops.linear_ce_bwd(y, w, target, lse, each)
    z = y @ w.T
    kd, _, dz = ops.distill_topk_fwd_bwd(z, idx, teacher, share * each, tau)
    dy = dy + dz @ w
    dw = dw + dz.T @ y
    dx, dgamma, dbeta = ops.layernorm_affine_bwd(x, gamma, mean, rstd, dy)
    return ce, kd, dx, dgamma, dbeta, dw


def reference(x, gamma, beta, w, target, idx, teacher, tau=2.0, share=0.3):
    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w)]
    xd, gd, bd, wd = leaves
    y = torch.nn.functional.layer_norm(xd, (x.shape[1],), gd, bd, 1e-5)
    z = y @ wd.T
    log_q = torch.log_softmax(z, -1)
    on = target >= 0
    ce = torch.where(on, -log_q.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0)
    there = idx >= 0
    t = torch.where(there, teacher.double() / tau, -1e300)
    p = torch.softmax(t, -1) * there
    lq = torch.log_softmax(z / tau, -1).gather(1, idx.clamp(min=0))
    kd = tau * tau * (torch.special.xlogy(p, p) - p * lq).sum(-1) * there.any(-1)
    loss = ce.mean() + share * kd.mean()
    loss.backward()
    return [ce.detach(), kd.detach(), xd.grad, gd.grad, bd.grad, wd.grad]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(dtype):
    """Held to the 2-norm: every output but the losses is rounded to its type at the end, and y, dy and z once more on the way (half a step
    each, a sum of about six independent roundings for the gradients); fp32 sums of up to 1003 terms carry 1003 * 2^-24."""
    from cgadimpl_b200 import ops

    args = make(dtype)
    bound = 6 * torch.finfo(dtype).eps / 2 + 1003 * 2.0 ** -24
    for name, got, want in zip(("ce", "kd", "dx", "dgamma", "dbeta", "dw"), step(ops, *args), reference(*args)):
        err = float((got.double() - want).norm() / want.norm())
        assert err <= bound, f"{name}: {err:.3e} > {bound:.3e}"
    ops.device_status()


@pytest.mark.gpu
def test_step_captured_and_replayed():
    from cgadimpl_b200 import ops

    args = list(make(torch.bfloat16, seed=1))
    want = step(ops, *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(ops, *args)
    torch.cuda.current_stream().wait_stream(s)
    x = args[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(ops, x, *args[1:])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x.copy_(args[0].flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step(ops, x, *args[1:])))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Two steps with workspaces of their own run side by side."""
    from cgadimpl_b200 import ops

    sets = [make(torch.bfloat16, rows=700, seed=s) for s in (2, 3)]
    want = [step(ops, *a) for a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (st, a) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = step(ops, *a)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
