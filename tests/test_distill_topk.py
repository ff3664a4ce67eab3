"""Distillation from a teacher's K largest logits (agb_distill_topk_*) against its formula in 64 bits, and its refusals.

Tolerances.  u = 2^-24.  lse is a sum of `vocab` positive terms, each exp off by at most 2^-22 plus its argument's error: a thread adds
CHAIN terms at most one after the other, so log(sum) is off by (CHAIN + 64) * u, and by a few u of the magnitudes that are subtracted
(|z| / t, |lse|).  A probability carries that error relative to itself; the loss weighs such errors with p, which sums to one."""
import ctypes as C
import math

import pytest
import torch

from cgadimpl_b200 import _lib, build

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ops():
    from cgadimpl_b200 import ops as _ops

    yield _ops
    if torch.cuda.is_available():
        _ops.device_status()


def make(rows, vocab, k, dtype, seed=0, absent=0.0, idx_dtype=torch.int64, teacher_dtype=torch.float32, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def place(t):
        v = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:].view(t.shape)
        v.copy_(t)
        return v

    z = place((3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype))
    idx = torch.rand(rows, vocab, device="cuda", generator=g).argsort(-1)[:, :k].contiguous() if k <= vocab else torch.randint(
        0, vocab, (rows, k), device="cuda", generator=g)
    idx = torch.where(torch.rand(rows, idx.shape[1], device="cuda", generator=g) < absent, torch.full_like(idx, -1), idx)
    teacher = (3 * torch.randn(rows, idx.shape[1], device="cuda", generator=g)).to(teacher_dtype)
    gy = torch.randn(rows, device="cuda", generator=g)
    add = place(torch.randn(rows, vocab, device="cuda", generator=g).to(dtype))
    return z, idx.to(idx_dtype), teacher, gy, add


def reference(z, idx, teacher, gy, tau, add=None):
    """One row after the other, from the definition, in Python's terms."""
    z, teacher, gy, idx = z.double().cpu(), teacher.double().cpu(), gy.double().cpu(), idx.long().cpu()
    loss, lse, dz = [], [], []
    for r in range(z.shape[0]):
        pick = [(int(j), float(t) / tau) for j, t in zip(idx[r], teacher[r]) if 0 <= int(j) < z.shape[1] and float(t) > -math.inf]
        grad = torch.zeros(z.shape[1], dtype=torch.float64)
        if not pick:
            loss.append(0.0)
            lse.append(0.0)
        else:
            zr = z[r] / tau
            top = float(zr.max())
            row_lse = top + math.log(float(torch.exp(zr - top).sum()))
            ttop = max(t for _, t in pick)
            tlse = ttop + math.log(sum(math.exp(t - ttop) for _, t in pick))
            total = 0.0
            grad = torch.exp(zr - row_lse)
            for j, t in pick:
                p = math.exp(t - tlse)
                if p > 0:
                    total += p * ((t - tlse) - (float(zr[j]) - row_lse))
                grad[j] -= p
            grad = grad * float(gy[r]) * tau
            loss.append(tau * tau * total)
            lse.append(row_lse)
        dz.append(grad)
    dz = torch.stack(dz)
    if add is not None:
        dz = dz + add.double().cpu()
    return torch.tensor(loss, dtype=torch.float64), torch.tensor(lse, dtype=torch.float64), dz


def tolerances(z, teacher, gy, tau, ref, dtype, add=None):
    loss, lse, dz = ref
    zf, tf = z.double().cpu(), teacher.double().cpu()
    zmax = torch.where(zf.isfinite(), zf, 0).abs().max(-1).values / tau
    tmax = torch.where(tf.isfinite(), tf, 0).abs().max(-1).values / tau
    chain = z.shape[1] / 512 + 64
    lse_tol = (chain + 64) * U + 8 * U * (zmax + lse.abs())
    loss_tol = tau * tau * (lse_tol + 64 * U + 16 * U * (zmax + tmax + lse.abs() + 8)) + 8 * U * loss.abs()
    # a probability's relative error: the exponent's absolute one
    rel = (lse_tol + 16 * U * (zmax + lse.abs() + tmax + 8) + 64 * U)[:, None]
    g = (gy.double().cpu().abs() * tau)[:, None]
    zr = torch.exp(zf / tau - lse[:, None])
    pure = dz if add is None else dz - add.double().cpu()
    shares = (g * zr - pure * torch.sign(gy.double().cpu())[:, None]).abs()
    dz_tol = rel * (g * zr + shares) + half(dtype) * dz.abs() + 4 * U * dz.abs() + 2.0 ** -126
    if add is not None:
        dz_tol = dz_tol + 2 * U * add.double().cpu().abs()
    # a row of NaN is one that takes no part (elsewhere the tests look at NaN themselves): it has to be exactly what is wanted
    return loss_tol, lse_tol, torch.nan_to_num(dz_tol, nan=0.0)


def check(name, got, want, tol):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())}/{bad.numel()} off, worst {float((err - tol).max()):.3e} above its tolerance"


def run_case(ops, z, idx, teacher, gy, tau):
    ref = reference(z, idx, teacher, gy, tau)
    tol = tolerances(z, teacher, gy, tau, ref, z.dtype)
    loss, lse = ops.distill_topk_fwd(z, idx, teacher, tau)
    check("loss", loss, ref[0], tol[0])
    check("lse", lse, ref[1], tol[1])
    dz = ops.distill_topk_bwd(z, idx, teacher, lse, gy, tau)
    check("dz", dz, ref[2], tol[2])
    l2, s2, d2 = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, tau)
    check("loss (one pass)", l2, ref[0], tol[0])
    check("lse (one pass)", s2, ref[1], tol[1])
    check("dz (one pass)", d2, ref[2], tol[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (2, 2, 2), (3, 7, 3), (5, 100, 10), (4, 129, 129), (9, 1000, 1), (3, 4096, 64),
                                          (2, 10007, 33), (1, 50001, 20), (3, 32768, 1000), (2, 131072, 64), (1, 131071, 100),
                                          (400, 515, 8), (700, 2048, 16)])
def test_sizes(ops, rows, vocab, k, dtype):
    z, idx, teacher, gy, _ = make(rows, vocab, k, dtype, seed=vocab + k)
    run_case(ops, z, idx, teacher, gy, 1.0 if k % 2 else 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("teacher_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_types_and_temperatures(ops, dtype, idx_dtype, teacher_dtype, tau):
    z, idx, teacher, gy, _ = make(6, 3001, 17, dtype, seed=1, absent=0.3, idx_dtype=idx_dtype, teacher_dtype=teacher_dtype)
    run_case(ops, z, idx, teacher, gy, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_that_take_no_part(ops, dtype):
    z, idx, teacher, gy, _ = make(8, 2051, 12, dtype, seed=2)
    idx[0] = -1                                         # no teacher at all
    z[0] = float("nan")                                 # and a row that must not be looked at
    idx[1, 3:] = 2051                                   # beyond the vocabulary
    idx[2, :5] = -7
    idx[3, 0] = 2 ** 40                                 # beyond 32 bits
    teacher[4, 2:6] = -math.inf
    teacher[5] = -math.inf                              # nothing above -inf: an empty row
    idx[6, 1:] = idx[6, 0].item()                       # one column named twelve times
    idx[7, 6:] = idx[7, :6].clone()
    run_case(ops, z, idx, teacher, gy, 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_student_columns(ops, dtype):
    """A padded vocabulary: its last columns hold -inf or the type's lowest value; whole vectors and whole threads see nothing else."""
    for fill in (-math.inf, torch.finfo(dtype).min):
        z, idx, teacher, gy, _ = make(5, 40000, 9, dtype, seed=3)
        idx.remainder_(30000)
        z[:, 30000:] = fill
        z[1, :20000] = fill
        idx[1] = idx[1] % 10000 + 20000
        run_case(ops, z, idx, teacher, gy, 1.0)
    z, idx, teacher, gy, _ = make(3, 3000, 4, dtype, seed=4)
    z[:] = torch.finfo(dtype).min                       # all alike, however low: uniform
    loss, lse = ops.distill_topk_fwd(z, idx, teacher)
    assert bool(lse.isfinite().all())
    # lse = min + log(3000) rounds to min, so the loss is the teacher's negative entropy, as the formula in fp32 has it
    z[1, 5] = math.nan
    loss, lse, dz = ops.distill_topk_fwd_bwd(z, idx, teacher, gy)
    assert bool(loss[1].isnan()) and bool(dz[1].isnan().all()) and not bool(dz[[0, 2]].isnan().any())


@pytest.mark.gpu
def test_large_logits(ops):
    z, idx, teacher, gy, _ = make(4, 5000, 11, torch.float32, seed=5)
    run_case(ops, z * 300, idx, teacher * 300, gy, 1.0)
    run_case(ops, z + 5000, idx, teacher, gy, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shift", [(torch.float32, 1), (torch.float32, 3), (torch.bfloat16, 1), (torch.bfloat16, 5)])
@pytest.mark.parametrize("vocab", [1024, 4099, 20000])
def test_bases_off_the_vector_boundary(ops, vocab, dtype, shift):
    z, idx, teacher, gy, add = make(3, vocab, 8, dtype, seed=shift, shift=shift)
    run_case(ops, z, idx, teacher, gy, 1.0)
    ref = reference(z, idx, teacher, gy, 1.0, add)
    tol = tolerances(z, teacher, gy, 1.0, ref, dtype, add)
    for a in (add, add.clone()):                        # the addend (and dz) with and without z's phase
        _, _, dz = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, dz_add=a)
        check("dz + add", dz, ref[2], tol[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(2, 70001), (3, 8192), (500, 1001)])
def test_accumulation_and_in_place(ops, rows, vocab, dtype):
    z, idx, teacher, gy, add = make(rows, vocab, 13, dtype, seed=6, absent=0.2)
    idx[0] = -1
    ref = reference(z, idx, teacher, gy, 2.0, add)
    tol = tolerances(z, teacher, gy, 2.0, ref, dtype, add)
    _, lse = ops.distill_topk_fwd(z, idx, teacher, 2.0)
    buf = add.clone()
    check("dz += in place", ops.distill_topk_bwd(z, idx, teacher, lse, gy, 2.0, dz_add=buf, dz=buf), ref[2], tol[2])
    buf = add.clone()
    check("dz += in place (one pass)", ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0, dz_add=buf, dz=buf)[2], ref[2], tol[2])
    plain = ops.distill_topk_bwd(z, idx, teacher, lse, gy, 2.0)
    over = z.clone()
    assert torch.equal(ops.distill_topk_bwd(over, idx, teacher, lse, gy, 2.0, dz=over), plain)
    over = z.clone()
    l1, s1, d1 = ops.distill_topk_fwd_bwd(over, idx, teacher, gy, 2.0, dz=over)
    l2, s2, d2 = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0)
    assert torch.equal(l1, l2) and torch.equal(s1, s2) and torch.equal(d1, d2)


@pytest.mark.gpu
def test_gradient_against_differences(ops):
    """The sum of gy * loss moves by <dz, d> per unit along d (fp32, step 2^-5; error: the losses' rounding over the step and the third
    derivative's share, bounded by step^2 * sum|gy| * max|d|^3)."""
    z, idx, teacher, gy, _ = make(4, 900, 9, torch.float32, seed=7, absent=0.2)
    _, _, dz = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0)
    d = torch.randn(z.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    step = 2.0 ** -5

    def value(q):
        return float((ops.distill_topk_fwd(q, idx, teacher, 2.0)[0].double() * gy.double()).sum())

    diff = (value(z + step * d) - value(z - step * d)) / (2 * step)
    size = float(gy.double().abs().sum())
    noise = 4 * 300 * U * 12 * size / (2 * step) + step * step * size * float(d.abs().max()) ** 3
    assert abs(diff - float((dz.double() * d.double()).sum())) <= noise


@pytest.mark.gpu
def test_captured_and_replayed_and_on_another_stream(ops):
    z, idx, teacher, gy, _ = make(5, 30000, 16, torch.bfloat16, seed=9)
    want = ops.distill_topk_fwd_bwd(z, idx, teacher, gy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.distill_topk_fwd_bwd(z, idx, teacher, gy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    zs = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.distill_topk_fwd_bwd(zs, idx, teacher, gy)
    for scale in (1.0, 0.25):
        zs.copy_(z * scale)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, ops.distill_topk_fwd_bwd(zs, idx, teacher, gy)))


@pytest.mark.gpu
def test_wrapper_refuses_operands_that_do_not_fit(ops):
    z, idx, teacher, gy, _ = make(4, 64, 5, torch.float32)
    assert ops.distill_topk_fwd(z[:0], idx[:0], teacher[:0])[0].numel() == 0
    for bad in (lambda: ops.distill_topk_fwd(z.t(), idx, teacher), lambda: ops.distill_topk_fwd(z, idx[:, :3], teacher),
                lambda: ops.distill_topk_fwd(z, idx[:2].contiguous(), teacher[:2].contiguous()),
                lambda: ops.distill_topk_fwd(z, idx.cpu(), teacher), lambda: ops.distill_topk_bwd(z, idx, teacher, gy[:2], gy),
                lambda: ops.distill_topk_bwd(z, idx, teacher, gy, gy, dz_add=z.bfloat16())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.distill_topk_fwd(z.half(), idx, teacher), lambda: ops.distill_topk_fwd(z, idx.short(), teacher),
                lambda: ops.distill_topk_fwd(z, idx, teacher.half())):
        with pytest.raises(TypeError):
            bad()
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(_lib.AgbError):
            ops.distill_topk_fwd(z, idx, teacher, t)


def test_refusals_need_no_device():
    build.build()
    lib = _lib.lib()
    one, odd = C.c_void_p(0x1000), C.c_void_p(0x1002)
    fwd, bwd, both = lib.agb_distill_topk_fwd, lib.agb_distill_topk_bwd, lib.agb_distill_topk_fwd_bwd
    assert fwd(one, one, 1, one, 0, one, one, -1, 8, 2, 1.0, 0, None) == 1
    assert fwd(one, one, 1, one, 0, one, one, 4, 0, 2, 1.0, 0, None) == 1
    assert fwd(one, one, 1, one, 0, one, one, 4, 8, 0, 1.0, 0, None) == 1
    assert fwd(one, one, 1, one, 0, one, one, 4, 8, 1025, 1.0, 0, None) == 2
    assert fwd(one, one, 7, one, 0, one, one, 4, 8, 2, 1.0, 0, None) == 1
    assert fwd(one, one, 1, one, 2, one, one, 4, 8, 2, 1.0, 0, None) == 2
    assert fwd(one, one, 1, one, 0, one, one, 4, 8, 2, 1.0, 2, None) == 2
    for t in (0.0, -2.0, math.inf, math.nan, 1e-40):
        assert fwd(one, one, 1, one, 0, one, one, 4, 8, 2, t, 0, None) == 1
    assert fwd(None, one, 1, one, 0, one, one, 4, 8, 2, 1.0, 0, None) == 1
    assert fwd(one, C.c_void_p(0x1004), 1, one, 0, one, one, 4, 8, 2, 1.0, 0, None) == 3
    assert fwd(one, one, 1, one, 0, None, one, 4, 8, 2, 1.0, 0, None) == 1
    assert bwd(one, one, 1, one, 0, one, None, None, one, 4, 8, 2, 1.0, 0, None) == 1
    assert bwd(one, one, 1, one, 0, one, one, odd, one, 4, 8, 2, 1.0, 0, None) == 3
    assert both(one, one, 1, one, 0, one, None, one, one, None, 4, 8, 2, 1.0, 0, None) == 1
    assert fwd(None, None, 1, None, 0, None, None, 0, 8, 2, 1.0, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(300, 9000), (310, 40003), (150, 120001), (40, 400000)])
def test_more_rows_than_the_gpu_takes_at_once(ops, rows, vocab, dtype):
    """Rows in turn on the same CTAs, several slices and chunks each, some without entries, against the two separate calls and the formula."""
    z, idx, teacher, gy, add = make(rows, vocab, 7, dtype, seed=vocab, absent=0.3)
    idx[1::5] = -1
    z[1::5] = float("nan")
    loss, lse = ops.distill_topk_fwd(z, idx, teacher, 2.0)
    dz = ops.distill_topk_bwd(z, idx, teacher, lse, gy, 2.0)
    l2, s2, d2 = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0)
    pick = torch.tensor([0, 1, 2, rows // 2, rows - 2, rows - 1], device="cuda")
    ref = reference(z[pick], idx[pick], teacher[pick], gy[pick], 2.0)
    tol = tolerances(z[pick], teacher[pick], gy[pick], 2.0, ref, dtype)
    for l, s, d in ((loss, lse, dz), (l2, s2, d2)):
        check("loss", l[pick], ref[0], tol[0])
        check("lse", s[pick], ref[1], tol[1])
        check("dz", d[pick], ref[2], tol[2])
    # every row: the two ways differ by no more than both tolerances
    assert bool(((loss - l2).abs() <= 2 * tol[0].max() * (1 + loss.abs())).all())
    assert bool(((dz.float() - d2.float()).abs() <= 4 * half(dtype) * dz.float().abs() + 2.0 ** -14 * gy.abs()[:, None]).all())
    assert all(torch.equal(p, q) for p, q in zip((l2, s2, d2), ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0)))
    over, buf = z.clone(), add.clone()
    assert torch.equal(ops.distill_topk_fwd_bwd(over, idx, teacher, gy, 2.0, dz=over)[2], d2)
    got = ops.distill_topk_fwd_bwd(z, idx, teacher, gy, 2.0, dz_add=buf, dz=buf)[2]
    ref = reference(z[pick], idx[pick], teacher[pick], gy[pick], 2.0, add[pick])
    check("dz +=", got[pick], ref[2], tolerances(z[pick], teacher[pick], gy[pick], 2.0, ref, dtype, add[pick])[2])
