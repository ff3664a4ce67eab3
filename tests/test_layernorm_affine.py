"""LayerNorm with weight and bias (agb_layernorm_affine_*) against its formula in 64 bits, and its refusals.

Tolerances.  u = 2^-24 is half a step of fp32, half(dtype) half a step of the output.  A sum of n terms taken in any order in fp32 is
off by at most n * u * sum|terms|; the kernels add at most CHAIN terms one after the other per thread and join the threads in a tree, so
the row sums are held to (CHAIN + 16) * u.  An output is then off by its rounding plus the error of its parts."""
import ctypes as C

import pytest
import torch

from cgadimpl_b200 import _lib, build

U = 2.0 ** -24
CHAIN = 64


def half(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ops():
    from cgadimpl_b200 import ops as _ops

    yield _ops
    if torch.cuda.is_available():
        _ops.device_status()


def make(rows, hidden, dtype, seed=0, offset=0.5, beta=True, shift=0):
    """Inputs on the GPU; shift > 0 places every tensor that many elements behind a 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def place(t):
        buf = torch.empty(t.numel() + shift, dtype=dtype, device="cuda")
        v = buf[shift:].view(t.shape)
        v.copy_(t)
        return v

    x = place(torch.randn(rows, hidden, device="cuda", generator=g) + offset)
    gy = place(torch.randn(rows, hidden, device="cuda", generator=g))
    add = place(torch.randn(rows, hidden, device="cuda", generator=g))
    gamma = place(1 + 0.1 * torch.randn(hidden, device="cuda", generator=g))
    b = place(0.1 * torch.randn(hidden, device="cuda", generator=g)) if beta else None
    return x, gy, add, gamma, b


def reference(x, gamma, beta, gy, eps, add=None):
    x, gamma, gy = x.double(), gamma.double(), gy.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (x - mean) * rstd
    b = 0.0 if beta is None else beta.double()
    v = gy * gamma
    dx = rstd * (v - v.mean(-1, keepdim=True) - h * (v * h).mean(-1, keepdim=True))
    if add is not None:
        dx = dx + add.double()
    return dict(y=h * gamma + b, mean=mean[:, 0], rstd=rstd[:, 0], dx=dx, dgamma=(gy * h).sum(0), dbeta=gy.sum(0), h=h, v=v)


def tolerances(x, gamma, beta, gy, ref, dtype, add=None):
    n = CHAIN + 16
    x, gamma, gy = x.double().abs(), gamma.double().abs(), gy.double().abs()
    rstd = ref["rstd"][:, None]
    mean_tol = n * U * x.mean(-1)                       # the sum, its division
    # xh: the mean's error, the subtraction's and the product's rounding, half of the variance's relative error (n * u)
    h_tol = rstd * (mean_tol[:, None] + U * x) + n * U * ref["h"].abs()
    rstd_tol = n * U * ref["rstd"] + 0.5 * ref["rstd"] ** 3 * (mean_tol ** 2)
    b = 0.0 if beta is None else beta.double().abs()
    y_tol = half(dtype) * ref["y"].abs() + h_tol * gamma + 4 * U * (ref["h"].abs() * gamma + b)
    va, ha = ref["v"].abs(), ref["h"].abs()
    c1_tol = n * U * va.mean(-1, keepdim=True)
    c2 = (ref["v"] * ref["h"]).mean(-1, keepdim=True).abs()
    c2_tol = n * U * (va * ha).mean(-1, keepdim=True) + (va * h_tol).mean(-1, keepdim=True)
    dx_tol = rstd * (c1_tol + ha * c2_tol + h_tol * c2 + 8 * U * (va + ha * c2 + c1_tol / (n * U))) + n * U * ref["dx"].abs()
    if add is not None:
        dx_tol = dx_tol + 4 * U * add.double().abs()
    dx_tol = dx_tol + half(dtype) * ref["dx"].abs()
    rows = x.shape[0]
    terms = min(rows, 4096) + 16
    dg_tol = terms * U * (gy * ha).sum(0) + (gy * h_tol).sum(0) + 2 * U * ref["dgamma"].abs()
    db_tol = terms * U * gy.sum(0) + 2 * U * ref["dbeta"].abs()
    return dict(y=y_tol, mean=mean_tol + U * ref["mean"].abs(), rstd=rstd_tol, dx=dx_tol, dgamma=dg_tol, dbeta=db_tol)


def check(name, got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())}/{bad.numel()} off, worst {float((err - tol).max()):.3e} above its tolerance"


def run_case(ops, rows, hidden, dtype, beta=True, shift=0, offset=0.5, eps=1e-5, seed=0):
    x, gy, _, gamma, b = make(rows, hidden, dtype, seed, offset, beta, shift)
    ref = reference(x, gamma, b, gy, eps)
    tol = tolerances(x, gamma, b, gy, ref, dtype)
    out = None if not shift else torch.empty(rows * hidden + shift, dtype=dtype, device="cuda")[shift:].view(rows, hidden)
    y, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b, eps, out=out)
    for k, v in (("y", y), ("mean", mean), ("rstd", rstd)):
        check(k, v, ref[k], tol[k])
    dx, dgamma, dbeta = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, with_beta=beta)
    check("dx", dx, ref["dx"], tol["dx"])
    check("dgamma", dgamma, ref["dgamma"], tol["dgamma"])
    if beta:
        check("dbeta", dbeta, ref["dbeta"], tol["dbeta"])
    else:
        assert dbeta is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hidden", [1, 2, 7, 8, 31, 33, 64, 100, 257, 1000, 1001, 1024, 2050, 4096, 4097, 8192, 8200, 10001])
@pytest.mark.parametrize("rows", [1, 3, 130])
def test_sizes(ops, rows, hidden, dtype):
    run_case(ops, rows, hidden, dtype, seed=rows * 31 + hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden", [(5, 16384), (3, 16385), (2, 33000), (2, 70001), (2, 70000), (2500, 8), (40000, 3), (5000, 1001),
                                         (3000, 4096), (700, 8192), (1025, 12288)])
def test_long_rows_and_many_rows(ops, rows, hidden, dtype):
    run_case(ops, rows, hidden, dtype, beta=hidden % 2 == 0, seed=hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shift", [(torch.float32, 1), (torch.bfloat16, 1), (torch.bfloat16, 2), (torch.bfloat16, 8)])
@pytest.mark.parametrize("hidden", [64, 1000, 4096])
def test_bases_off_the_vector_boundary(ops, hidden, dtype, shift):
    run_case(ops, 37, hidden, dtype, shift=shift, seed=shift)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offset_rows_and_constant_rows(ops, dtype):
    run_case(ops, 65, 1024, dtype, offset=100.0)
    x = torch.full((3, 256), 2.5, dtype=dtype, device="cuda")
    w = torch.ones(256, dtype=dtype, device="cuda")
    y, mean, rstd = ops.layernorm_affine_fwd(x, w, None)
    assert bool((y == 0).all()) and bool((mean == 2.5).all())
    check("rstd", rstd, torch.full((3,), 1 / (1e-5 ** 0.5), dtype=torch.float64, device="cuda"), 320.0 * 4 * U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden", [(70, 1001), (70, 4096), (300, 64), (9, 16384), (2, 40000)])
def test_gradient_accumulation_forms(ops, rows, hidden, dtype):
    x, gy, add, gamma, b = make(rows, hidden, dtype, seed=5)
    _, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    ref = reference(x, gamma, b, gy, 1e-5, add)
    tol = tolerances(x, gamma, b, gy, ref, dtype, add)
    buf = add.clone()
    dg0 = torch.full((hidden,), 3.0, device="cuda")
    db0 = torch.full((hidden,), -2.0, device="cuda")
    dx, dg, db = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, dx_add=buf, dx=buf, dgamma=dg0, dbeta=db0, accumulate=True)
    assert dx.data_ptr() == buf.data_ptr() and dg.data_ptr() == dg0.data_ptr()
    check("dx += in place", dx, ref["dx"], tol["dx"])
    check("dgamma +=", dg, ref["dgamma"] + 3, tol["dgamma"] + 4 * U * 3)
    check("dbeta +=", db, ref["dbeta"] - 2, tol["dbeta"] + 4 * U * 2)
    ref2 = reference(x, gamma, b, gy, 1e-5, gy)
    dx2, _, _ = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, dx_add=gy)
    check("dx_add is gy", dx2, ref2["dx"], tolerances(x, gamma, b, gy, ref2, dtype, gy)["dx"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_every_time_and_parts_left_out(ops, dtype):
    x, gy, _, gamma, b = make(777, 1000, dtype, seed=9)
    _, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    one = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    two = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    dx, dg, _ = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, with_beta=False)
    assert torch.equal(dx, one[0]) and torch.equal(dg, one[1])
    lib = _lib.lib()
    only_dx = torch.empty_like(x)                       # a frozen norm: no column sums, no workspace
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    st = lib.agb_layernorm_affine_bwd(p(x), p(gamma), p(mean), p(rstd), p(gy), None, p(only_dx), None, None, 0, None, 0, 777, 1000,
                                      _lib.AGB_F32 if dtype == torch.float32 else _lib.AGB_BF16,
                                      C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert st == 0 and torch.equal(only_dx, one[0])


@pytest.mark.gpu
def test_no_rows(ops):
    x = torch.empty(0, 64, device="cuda")
    g = torch.ones(64, device="cuda")
    y, mean, rstd = ops.layernorm_affine_fwd(x, g, g)
    assert y.shape == (0, 64) and mean.numel() == 0
    dx, dg, db = ops.layernorm_affine_bwd(x, g, mean, rstd, x)
    assert bool((dg == 0).all()) and bool((db == 0).all())
    dg.fill_(2.0)
    db.fill_(3.0)
    ops.layernorm_affine_bwd(x, g, mean, rstd, x, dgamma=dg, dbeta=db, accumulate=True)
    assert bool((dg == 2).all()) and bool((db == 3).all())


@pytest.mark.gpu
def test_nan_stays_in_its_row(ops):
    x, gy, _, gamma, b = make(6, 1024, torch.bfloat16, seed=2)
    x[3, 17] = float("nan")
    y, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    assert bool(y[3].isnan().all()) and not bool(y[[0, 1, 2, 4, 5]].isnan().any())
    dx, _, _ = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    assert bool(dx[3].isnan().all()) and not bool(dx[[0, 1, 2, 4, 5]].isnan().any())


@pytest.mark.gpu
def test_gradient_against_differences(ops):
    """sum(gy * y) moves by <dx, d> per unit along d: fp32 forward, step 2^-6, held to the differences' own error (the third
    derivative's share step^2 and the rounding of the two sums over 2 * step)."""
    x, gy, _, gamma, b = make(4, 512, torch.float32, seed=3)
    _, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    dx, dgamma, dbeta = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    g = torch.Generator(device="cuda").manual_seed(4)
    step = 2.0 ** -6

    def value(x, gamma, b):
        return float((ops.layernorm_affine_fwd(x, gamma, b)[0].double() * gy.double()).sum())

    size = float(gy.double().abs().sum())
    noise = 32 * U * 4 * size / (2 * step)
    d = torch.randn(x.shape, device="cuda", generator=g)
    diff = (value(x + step * d, gamma, b) - value(x - step * d, gamma, b)) / (2 * step)
    assert abs(diff - float((dx.double() * d.double()).sum())) <= noise + step * step * size
    d = torch.randn(512, device="cuda", generator=g)
    diff = (value(x, gamma + step * d, b) - value(x, gamma - step * d, b)) / (2 * step)
    assert abs(diff - float((dgamma.double() * d.double()).sum())) <= 4 * noise
    diff = (value(x, gamma, b + step * d) - value(x, gamma, b - step * d)) / (2 * step)
    assert abs(diff - float((dbeta.double() * d.double()).sum())) <= 4 * noise


@pytest.mark.gpu
def test_captured_and_replayed_and_on_another_stream(ops):
    x, gy, _, gamma, b = make(333, 1000, torch.bfloat16, seed=11)
    want = ops.layernorm_affine_fwd(x, gamma, b)
    wantb = ops.layernorm_affine_bwd(x, gamma, want[1], want[2], gy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
        got = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(got, wantb))
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = ops.layernorm_affine_fwd(xs, gamma, b)
        got = ops.layernorm_affine_bwd(xs, gamma, mean, rstd, gy)
    for scale in (1.0, -3.0):
        xs.copy_(x * scale)
        graph.replay()
        want = ops.layernorm_affine_fwd(xs, gamma, b)
        wantb = ops.layernorm_affine_bwd(xs, gamma, want[1], want[2], gy)
        assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(got, wantb))


@pytest.mark.gpu
def test_wrapper_refuses_operands_that_do_not_fit(ops):
    x, gy, _, gamma, b = make(4, 64, torch.float32)
    with pytest.raises(ValueError):
        ops.layernorm_affine_fwd(x.t(), gamma, b)
    with pytest.raises(ValueError):
        ops.layernorm_affine_fwd(x, gamma[:32], b)
    with pytest.raises(ValueError):
        ops.layernorm_affine_fwd(x, gamma.bfloat16(), b)
    with pytest.raises(TypeError):
        ops.layernorm_affine_fwd(x.half(), gamma.half(), None)
    _, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    with pytest.raises(ValueError):
        ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, accumulate=True)
    with pytest.raises(ValueError):
        ops.layernorm_affine_bwd(x, gamma, mean[:2], rstd, gy)
    with pytest.raises(_lib.AgbError):
        ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))


def test_refusals_need_no_device():
    build.build()
    lib = _lib.lib()
    one, odd = C.c_void_p(0x1000), C.c_void_p(0x1002)
    fwd, bwd = lib.agb_layernorm_affine_fwd, lib.agb_layernorm_affine_bwd
    assert fwd(one, one, None, one, one, one, -1, 8, 1e-5, 0, None) == 1
    assert fwd(one, one, None, one, one, one, 4, 0, 1e-5, 0, None) == 1
    assert fwd(one, one, None, one, one, one, 4, 8, 1e-5, 2, None) == 2
    assert fwd(None, one, None, one, one, one, 4, 8, 1e-5, 0, None) == 1 and b"x is NULL" in lib.agb_last_error()
    assert fwd(one, None, None, one, one, one, 4, 8, 1e-5, 0, None) == 1
    assert fwd(one, one, odd, one, one, one, 4, 8, 1e-5, 0, None) == 3
    assert fwd(one, one, None, one, None, one, 4, 8, 1e-5, 0, None) == 1
    assert fwd(None, None, None, None, None, None, 0, 8, 1e-5, 0, None) == 0
    need = lib.agb_layernorm_affine_bwd_workspace_bytes(4, 8, 0)
    assert bwd(one, one, one, one, one, None, one, one, one, 0, None, 0, 4, 8, 0, None) == 1       # column sums without a workspace
    assert need > 0 and bwd(one, one, one, one, one, None, one, one, one, 0, one, need - 1, 4, 8, 0, None) == 5
    assert bwd(one, one, one, one, None, None, one, one, one, 0, one, need, 4, 8, 0, None) == 1
    assert bwd(one, one, one, one, one, odd, one, one, one, 0, one, need, 4, 8, 0, None) == 3
    assert lib.agb_layernorm_affine_bwd_workspace_bytes(4, 0, 0) == 0


def test_ring_kernels_do_not_spill():
    """The 16-byte forms of the one-pass kernels: their loops hold the column sums in registers."""
    seen = 0
    for name, r in build.kernel_resources().items():
        if "lna_bwd_ringI13__nv_bfloat16Li16E" in name or "lna_fwd_ringI13__nv_bfloat16Li16E" in name:
            seen += 1
            assert r["spill_stores"] == 0 and r["registers"] <= 128, f"{name}: {r}"
    assert seen == 6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hidden", [64, 1001, 4096])
def test_in_place(ops, hidden, dtype):
    """y over x, dx over gy and dx over x: every element is read before its own place is written."""
    x, gy, _, gamma, b = make(1500, hidden, dtype, seed=21)
    y, mean, rstd = ops.layernorm_affine_fwd(x, gamma, b)
    dx, dg, db = ops.layernorm_affine_bwd(x, gamma, mean, rstd, gy)
    over = x.clone()
    assert torch.equal(ops.layernorm_affine_fwd(over, gamma, b, out=over)[0], y)
    over = gy.clone()
    got = ops.layernorm_affine_bwd(x, gamma, mean, rstd, over, dx=over)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dg) and torch.equal(got[2], db)
    over = x.clone()
    got = ops.layernorm_affine_bwd(over, gamma, mean, rstd, gy, dx=over)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dg) and torch.equal(got[2], db)
