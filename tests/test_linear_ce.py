"""Softmax cross entropy from the hidden states (agb_linear_ce_*) against its formula in 64 bits, and its refusals.

Tolerances.  Products are summed in fp32 on the tensor cores, 16 terms of K per step, six plane products for fp32 operands: a sum of K
terms is held to S(K) * sum|terms| with S(K) = (K / 16 * products + 32) * 2^-23 (one step of fp32 per addition; cutting rather than
rounding is allowed for).  z carries S(hidden); lse carries the largest such error of its row and the sum's own; g carries z's and lse's
errors relative to p, and half a step of bf16 where it is the 16-bit operand of the gradient products; dh and dw carry g's errors
weighted with |w| and |h|, S of their own sums, and their rounding."""
import ctypes as C

import pytest
import torch

from cgadimpl_b200 import _lib, build

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def S(k, dtype):
    return (k / 16 * (6 if dtype == torch.float32 else 1) + 32) * 2 * U


@pytest.fixture(scope="module")
def ops():
    from cgadimpl_b200 import ops as _ops

    yield _ops
    if torch.cuda.is_available():
        _ops.device_status()


def make(rows, hidden, vocab, dtype, seed=0, ignored=0.0, target_dtype=torch.int64, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, hidden, device="cuda", generator=g).to(dtype)
    w = (torch.randn(vocab, hidden, device="cuda", generator=g) * scale / hidden ** 0.5).to(dtype)
    target = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    off = torch.rand(rows, device="cuda", generator=g) < ignored
    target = torch.where(off, torch.full_like(target, -100), target).to(target_dtype)
    gy = torch.randn(rows, device="cuda", generator=g)
    return h, w, target, gy


def reference(h, w, target, gy):
    vocab, dtype = w.shape[0], h.dtype
    target = target.long()
    on = (target >= 0) & (target < vocab)
    hd, wd = torch.where(on[:, None], h.double(), 0.0), w.double()
    at = torch.where(on, target, 0)
    z = hd @ wd.T
    top = z.max(-1, keepdim=True).values
    lse = (top + torch.log(torch.exp(z - top).sum(-1, keepdim=True)))[:, 0]
    loss = lse - z.gather(1, at[:, None])[:, 0]
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    gyd = torch.where(on, gy.double(), 0.0)[:, None]
    g = gyd * (p - onehot)
    ref = dict(loss=torch.where(on, loss, 0.0), lse=torch.where(on, lse, 0.0), dh=g @ wd, dw=g.T @ hd)
    # tolerances
    z_tol = S(h.shape[1], dtype) * (hd.abs() @ wd.abs().T)
    worst = z_tol.max(-1).values
    lse_tol = worst + (vocab / 16 + 64) * U + 4 * U * (lse.abs() + top[:, 0].abs())
    loss_tol = lse_tol + worst + 4 * U * (lse.abs() + top[:, 0].abs())
    rel = z_tol + lse_tol[:, None] + 8 * U * (z.abs() + lse.abs()[:, None] + 8)
    g_tol = gyd.abs() * p * rel * torch.exp(rel) + 4 * U * g.abs()
    if dtype == torch.bfloat16:
        g_tol = g_tol * 1.01 + half(dtype) * g.abs()
    dh_tol = g_tol @ wd.abs() + (S(vocab, dtype) + 8 * U) * (g.abs() @ wd.abs()) + half(dtype) * ref["dh"].abs() + 2.0 ** -126
    dw_tol = g_tol.T @ hd.abs() + (S(h.shape[0], dtype) + 8 * U) * (g.abs().T @ hd.abs()) + half(dtype) * ref["dw"].abs() + 2.0 ** -126
    return ref, dict(loss=torch.where(on, loss_tol, 0.0), lse=torch.where(on, lse_tol, 0.0), dh=dh_tol, dw=dw_tol)


def check(name, got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())}/{bad.numel()} off, worst {float((err - tol).max()):.3e} above its tolerance"


def run_case(ops, h, w, target, gy):
    ref, tol = reference(h, w, target, gy)
    loss, lse = ops.linear_ce_fwd(h, w, target)
    check("loss", loss, ref["loss"], tol["loss"])
    check("lse", lse, ref["lse"], tol["lse"])
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    check("dh", dh, ref["dh"], tol["dh"])
    check("dw", dw, ref["dw"], tol["dw"])
    return loss, lse, dh, dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,vocab", [(128, 64, 256), (1, 8, 1), (1, 1, 2), (2, 16, 100), (7, 72, 129), (128, 128, 512), (129, 64, 257),
                                               (3, 1001, 300), (130, 100, 1000), (257, 333, 2049), (64, 512, 5000), (1, 4096, 1024),
                                               (300, 96, 10007), (1000, 40, 130), (31, 2056, 777), (640, 520, 3001)])
def test_sizes(ops, rows, hidden, vocab, dtype):
    run_case(ops, *make(rows, hidden, vocab, dtype, seed=rows + vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,vocab", [(4100, 64, 600), (8200, 24, 300), (9, 128, 131072), (700, 256, 70001), (16, 1024, 32768)])
def test_many_rows_and_large_vocabularies(ops, rows, hidden, vocab, dtype):
    run_case(ops, *make(rows, hidden, vocab, dtype, seed=3, ignored=0.3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_several_pieces_of_the_vocabulary(ops, dtype):
    """Rows enough that g is written in more than one piece: 256 MB hold rows * piece * 2 bytes (6 in fp32)."""
    rows = 33000 if dtype == torch.bfloat16 else 11000
    run_case(ops, *make(rows, 40, 9001, dtype, seed=4, ignored=0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("target_dtype", [torch.int32, torch.int64])
def test_rows_that_take_no_part(ops, dtype, target_dtype):
    h, w, target, gy = make(200, 72, 500, dtype, seed=5, target_dtype=target_dtype)
    target[::3] = -100
    target[1] = -1
    target[4] = 500                                     # the first column that is not there
    target[64:160] = -1                                 # whole tiles of them
    target[7] = 2 ** 31 - 1
    if target_dtype == torch.int64:
        target[8] = 2 ** 32 + 5                         # its low 32 bits name a column
    h[0], h[70] = float("nan"), float("inf")            # what they hold reaches nothing
    gy[3] = float("nan")
    loss, lse, dh, dw = run_case(ops, h, w, target, gy)
    off = (target < 0) | (target >= 500)
    assert bool((dh[off] == 0).all()) and bool((loss[off] == 0).all()) and bool((lse[off] == 0).all())
    none = torch.full_like(target, -1)
    loss, lse, dh, dw = run_case(ops, h, w, none, gy)   # nothing takes part
    assert bool((dw == 0).all()) and bool((dh == 0).all())
    kept = torch.full_like(w, 2.0)
    ops.linear_ce_bwd(h, w, none, lse, gy, dw=kept, accumulate_dw=True)
    assert bool((kept == 2).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_left_out_rows_change_no_bit_of_the_others(ops, dtype):
    h, w, target, gy = make(150, 64, 700, dtype, seed=6, ignored=0.4)
    on = target >= 0
    loss, lse = ops.linear_ce_fwd(h, w, target)
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    l2, s2 = ops.linear_ce_fwd(h[on], w, target[on])
    dh2, dw2 = ops.linear_ce_bwd(h[on], w, target[on], s2, gy[on])
    assert torch.equal(loss[on], l2) and torch.equal(lse[on], s2) and torch.equal(dh[on], dh2) and torch.equal(dw, dw2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_accumulation_parts_and_same_bits(ops, dtype):
    h, w, target, gy = make(100, 88, 900, dtype, seed=7, ignored=0.2)
    ref, tol = reference(h, w, target, gy)
    _, lse = ops.linear_ce_fwd(h, w, target)
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    again = ops.linear_ce_bwd(h, w, target, lse, gy)
    assert torch.equal(dh, again[0]) and torch.equal(dw, again[1])
    a, b = ops.linear_ce_bwd(h, w, target, lse, gy, need_dw=False)
    assert b is None and torch.equal(a, dh)
    a, b = ops.linear_ce_bwd(h, w, target, lse, gy, need_dh=False)
    assert a is None and torch.equal(b, dw)
    old = torch.randn(w.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    got = ops.linear_ce_bwd(h, w, target, lse, gy, dw=old.clone(), accumulate_dw=True)[1]
    total = ref["dw"] + old.double()
    check("dw +=", got, total, tol["dw"] + 2 * U * old.double().abs() + half(dtype) * total.abs())
    # a workspace full of NaN from an earlier life
    n = _lib.lib().agb_linear_ce_workspace_bytes(1, 100, 88, 900, ops._dt(h))
    ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")
    got = ops.linear_ce_bwd(h, w, target, lse, gy, workspace=ws)
    assert torch.equal(got[0], dh) and torch.equal(got[1], dw)
    n = _lib.lib().agb_linear_ce_workspace_bytes(0, 100, 88, 900, ops._dt(h))
    ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")
    assert torch.equal(ops.linear_ce_fwd(h, w, target, workspace=ws)[1], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_peaked_and_large_logits(ops, dtype):
    h, w, target, gy = make(60, 64, 400, dtype, seed=8, scale=40.0)
    target[:20] = (h[:20].float() @ w.float().T).argmax(-1)      # p close to one: g cancels
    run_case(ops, h, w, target, gy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_that_are_not_finite(ops, dtype):
    h, w, target, gy = make(140, 64, 300, dtype, seed=9)
    h[5, 3] = float("nan")
    loss, lse = ops.linear_ce_fwd(h, w, target)
    rest = torch.arange(140, device="cuda") != 5
    assert bool(loss[5].isnan()) and bool(loss[rest].isfinite().all())
    dh, _ = ops.linear_ce_bwd(h, w, target, lse, gy, need_dw=False)
    assert bool(dh[5].isnan().all()) and bool(dh[rest].isfinite().all())


@pytest.mark.gpu
def test_fp32_keeps_24_bits(ops):
    """Operands that differ in their last bits only: bf16 products would see none of it."""
    h = torch.ones(4, 64, device="cuda")
    w = torch.ones(8, 64, device="cuda")
    w += torch.arange(8, device="cuda")[:, None] * 2.0 ** -20
    target = torch.arange(4, device="cuda")
    run_case(ops, h, w, target, torch.ones(4, device="cuda"))
    big = torch.full((4, 64), 3.0e38, device="cuda")    # above the largest bf16 when rounded up
    loss, lse = ops.linear_ce_fwd(big, torch.full((8, 64), 2.0 ** -126, device="cuda"), target)
    assert bool(lse.isfinite().all())


@pytest.mark.gpu
def test_alignment(ops):
    h, w, target, gy = make(40, 64, 300, torch.bfloat16, seed=10)
    hs = torch.empty(h.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(h.shape)
    hs.copy_(h)
    loss, lse = ops.linear_ce_fwd(h, w, target)
    assert torch.equal(ops.linear_ce_fwd(hs, w, target)[1], lse)
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    dws = torch.empty(w.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(w.shape)
    dhs = torch.empty(h.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(h.shape)
    ops.linear_ce_bwd(hs, w, target, lse, gy, dh=dhs, dw=dws)
    assert torch.equal(dhs, dh) and torch.equal(dws, dw)
    ws = torch.empty(w.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(w.shape)
    ws.copy_(w)
    with pytest.raises(_lib.AgbError) as e:             # refused, not read wrongly
        ops.linear_ce_fwd(h, ws, target)
    assert e.value.status == 3
    h, w, target, gy = make(40, 65, 300, torch.bfloat16, seed=10)
    ws = torch.empty(w.numel() + 1, dtype=h.dtype, device="cuda")[1:].view(w.shape)
    ws.copy_(w)                                         # a width that is laid out anyway
    assert torch.equal(ops.linear_ce_fwd(h, ws, target)[1], ops.linear_ce_fwd(h, w, target)[1])


@pytest.mark.gpu
def test_gradient_against_differences(ops):
    """sum(gy * loss) moves by <dh, d> and <dw, d> per unit along d (fp32, step 2^-5; error: the losses' own over the step, and the third
    derivative's share, bounded by step^2 times the third power of the logits' change)."""
    h, w, target, gy = make(20, 48, 200, torch.float32, seed=11, ignored=0.2)
    _, lse = ops.linear_ce_fwd(h, w, target)
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    g = torch.Generator(device="cuda").manual_seed(12)
    step = 2.0 ** -5
    size = float(gy.double().abs().sum())

    def value(h, w):
        return float((ops.linear_ce_fwd(h, w, target)[0].double() * gy.double()).sum())

    for name in ("h", "w"):
        d = torch.randn((h if name == "h" else w).shape, device="cuda", generator=g) * (1.0 if name == "h" else 48 ** -0.5)
        change = (d @ w.T if name == "h" else h @ d.T).abs().max().item()
        plus, minus = (value(h + step * d, w), value(h - step * d, w)) if name == "h" else (value(h, w + step * d), value(h, w - step * d))
        want = float(((dh if name == "h" else dw).double() * d.double()).sum())
        noise = size * 64 * S(48, torch.float32) / (2 * step) + step ** 2 * size * change ** 3
        assert abs((plus - minus) / (2 * step) - want) <= noise


@pytest.mark.gpu
def test_captured_and_replayed_and_on_another_stream(ops):
    h, w, target, gy = make(300, 136, 3000, torch.bfloat16, seed=13, ignored=0.25)

    def step(h, target):
        loss, lse = ops.linear_ce_fwd(h, w, target)
        return (loss, lse) + ops.linear_ce_bwd(h, w, target, lse, gy)

    want = step(h, target)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(h, target)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hs, ts = h.clone(), target.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(hs, ts)
    for scale, shift in ((1.0, 0), (0.5, 17)):          # another number of rows takes part on replay
        hs.copy_(h * scale)
        ts.copy_(target.roll(shift))
        ts[:shift] = -1
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step(hs, ts)))


@pytest.mark.gpu
def test_no_rows(ops):
    h = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(10, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = ops.linear_ce_fwd(h, w, t)
    assert loss.numel() == 0
    dh, dw = ops.linear_ce_bwd(h, w, t, lse, lse)
    assert dh.shape == (0, 64) and bool((dw == 0).all())
    kept = torch.full_like(w, 3.0)
    ops.linear_ce_bwd(h, w, t, lse, lse, dw=kept, accumulate_dw=True)
    assert bool((kept == 3).all())


@pytest.mark.gpu
def test_wrapper_refuses_operands_that_do_not_fit(ops):
    h, w, target, gy = make(8, 64, 100, torch.float32)
    for bad in (lambda: ops.linear_ce_fwd(h.t(), w, target), lambda: ops.linear_ce_fwd(h, w.t(), target),
                lambda: ops.linear_ce_fwd(h, w[:, :32], target), lambda: ops.linear_ce_fwd(h, w.bfloat16(), target),
                lambda: ops.linear_ce_fwd(h, w, target[:4]), lambda: ops.linear_ce_fwd(h, w, target.cpu()),
                lambda: ops.linear_ce_bwd(h, w, target, gy[:3], gy), lambda: ops.linear_ce_bwd(h, w, target, gy, gy, accumulate_dw=True)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.linear_ce_fwd(h.half(), w.half(), target), lambda: ops.linear_ce_fwd(h, w, target.short())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(_lib.AgbError):
        ops.linear_ce_fwd(h, w, target, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_refusals_need_no_device():
    build.build()
    lib = _lib.lib()
    one = C.c_void_p(0x1000)
    fwd, bwd = lib.agb_linear_ce_fwd, lib.agb_linear_ce_bwd
    big = 1 << 40
    assert fwd(one, one, one, 1, one, one, -1, 8, 8, 0, one, big, None) == 1
    assert fwd(one, one, one, 1, one, one, 4, 0, 8, 0, one, big, None) == 1
    assert fwd(one, one, one, 1, one, one, 4, 8, 0, 0, one, big, None) == 1
    assert fwd(one, one, one, 1, one, one, 4, 8, 8, 2, one, big, None) == 2
    assert fwd(one, one, one, 5, one, one, 4, 8, 8, 0, one, big, None) == 1
    assert fwd(one, one, one, 1, one, one, 4, 8, 1 << 25, 0, one, big, None) == 2
    assert fwd(one, one, one, 1, one, one, (1 << 20) + 1, 8, 8, 0, one, big, None) == 2
    assert fwd(None, one, one, 1, one, one, 4, 8, 8, 0, one, big, None) == 1
    assert fwd(one, one, C.c_void_p(0x1004), 1, one, one, 4, 8, 8, 0, one, big, None) == 3
    assert fwd(one, one, one, 1, None, one, 4, 8, 8, 0, one, big, None) == 1
    assert fwd(one, C.c_void_p(0x1002), one, 1, one, one, 4, 8, 8, 1, one, big, None) == 3
    assert fwd(one, one, one, 1, one, one, 4, 8, 8, 0, None, big, None) == 5
    assert bwd(one, one, one, 1, one, one, None, None, 0, 4, 8, 8, 0, one, big, None) == 1
    two, three = C.c_void_p(0x2000), C.c_void_p(0x3000)
    assert bwd(one, two, one, 1, None, one, one, three, 0, 4, 8, 8, 0, one, big, None) == 1
    assert bwd(one, two, one, 1, one, one, one, two, 0, 4, 8, 8, 0, one, big, None) == 1 and b"dw" in lib.agb_last_error()
    assert bwd(one, two, one, 1, one, one, two, three, 0, 4, 8, 8, 0, one, big, None) == 1
    assert fwd(None, None, None, 1, None, None, 0, 8, 8, 0, None, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,vocab", [(10, 1835, 2235), (190, 1973, 1818), (2, 4096, 300), (129, 2048, 513), (1, 8192, 255), (64, 1024, 64),
                                               (250, 4100, 1000)])
def test_few_tiles_and_a_long_sum(ops, rows, hidden, vocab, dtype):
    """Sizes whose logits are cut along the hidden axis; rows that take no part among them, and none at all."""
    h, w, target, gy = make(rows, hidden, vocab, dtype, seed=hidden, ignored=0.3)
    run_case(ops, h, w, target, gy)
    run_case(ops, h, w, torch.full_like(target, -1), gy)
    loss, lse = ops.linear_ce_fwd(h, w, target)
    n = _lib.lib().agb_linear_ce_workspace_bytes(1, rows, hidden, vocab, ops._dt(h))
    ws = torch.full((n // 4 + 1,), float("nan"), device="cuda")
    one, two = ops.linear_ce_bwd(h, w, target, lse, gy, workspace=ws), ops.linear_ce_bwd(h, w, target, lse, gy)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dh_in_place_of_h(ops, dtype):
    h, w, target, gy = make(150, 72, 900, dtype, seed=14, ignored=0.2)
    _, lse = ops.linear_ce_fwd(h, w, target)
    dh, dw = ops.linear_ce_bwd(h, w, target, lse, gy)
    over = h.clone()
    got = ops.linear_ce_bwd(over, w, target, lse, gy, dh=over)
    assert torch.equal(got[0], dh) and torch.equal(got[1], dw)
    with pytest.raises(_lib.AgbError):
        ops.linear_ce_bwd(h, w, target, lse, gy, dw=w)


@pytest.mark.gpu
def test_many_rows_of_a_small_head(ops):
    """More rows than the blocks that lay them out take 8 of each, most of them without a target."""
    h, w, target, gy = make(70000, 16, 40, torch.bfloat16, seed=15, ignored=0.9)
    run_case(ops, h, w, target, gy)


def test_matrix_kernels_do_not_spill():
    """What ptxas made of the matrix kernels: phases 0 to 2 without spills, the epilogue of split fp32 gradients with a few bytes."""
    seen = 0
    for name, r in build.kernel_resources().items():
        if "ce_gemm_kernel" not in name:
            continue
        seen += 1
        limit = 64 if "ELi3EE" in name else 0
        assert r["spill_stores"] <= limit and r["registers"] <= 168, f"{name}: {r}"
    assert seen == 8
