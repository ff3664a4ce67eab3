"""The operators at the end of a language model, as workloads: the last normalisation (layer normalisation with
weight and bias), the loss over the vocabulary taken straight from the hidden states (the logits are not kept), and
the distillation loss against the few largest logits of a teacher.

listed() and draw() describe cases, prepare() makes what a program has in hand before the call, run() makes one pass
(through the library where `own` is true, in elementary torch operations where it is not), work() counts what a pass
cannot do without and exact() is the same pass in 64 bits.
"""
import math

import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
ELEM = {"fp32": 4, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # One decode step of four sequences through the last norm: launch latency is all there is.
        {"name": "ln_fwd_bf16_4x4096", "op": "ln", "train": False, "rows": 4, "hidden": 4096, "dtype": "bf16", "beta": True},
        # A training step's norm at the size of this repository's 16-bit benchmark.
        {"name": "ln_train_bf16_16384x8192", "op": "ln", "train": True, "rows": 16384, "hidden": 8192, "dtype": "bf16", "beta": True},
        # The same in the reference's own type, without a bias.
        {"name": "ln_train_fp32_8192x4096", "op": "ln", "train": True, "rows": 8192, "hidden": 4096, "dtype": "fp32", "beta": False},
        # A width that no vector load divides and a ragged number of rows.
        {"name": "ln_train_bf16_4099x1001", "op": "ln", "train": True, "rows": 4099, "hidden": 1001, "dtype": "bf16", "beta": True},
        # Scoring a short continuation: reading the head's weight once is the work.
        {"name": "ce_loss_bf16_16x4096x32768", "op": "ce", "train": False, "rows": 16, "hidden": 4096, "vocab": 32768,
         "dtype": "bf16", "ignored": 0.0},
        # Evaluation (perplexity) of a batch over a large vocabulary.
        {"name": "ce_loss_bf16_2048x4096x131072", "op": "ce", "train": False, "rows": 2048, "hidden": 4096, "vocab": 131072,
         "dtype": "bf16", "ignored": 0.0},
        # A training step of the head; a quarter of the tokens (prompts, padding) takes no part in the loss.
        {"name": "ce_train_bf16_8192x4096x131072", "op": "ce", "train": True, "rows": 8192, "hidden": 4096, "vocab": 131072,
         "dtype": "bf16", "ignored": 0.25},
        # Full precision, a ragged batch and an odd vocabulary.
        {"name": "ce_train_fp32_1023x1024x50001", "op": "ce", "train": True, "rows": 1023, "hidden": 1024, "vocab": 50001,
         "dtype": "fp32", "ignored": 0.1},
        # A small model: every size odd.
        {"name": "ce_train_bf16_301x1001x10007", "op": "ce", "train": True, "rows": 301, "hidden": 1001, "vocab": 10007,
         "dtype": "bf16", "ignored": 0.1},
        # Scoring a few positions against a teacher: few rows, a long axis.
        {"name": "kd_loss_bf16_8x131072_k64", "op": "kd", "train": False, "rows": 8, "vocab": 131072, "k": 64, "dtype": "bf16",
         "teacher": "bf16", "temperature": 1.0, "absent": 0.0, "empty": 0.0},
        # A distillation step on a batch of logits.
        {"name": "kd_train_bf16_4096x131072_k64", "op": "kd", "train": True, "rows": 4096, "vocab": 131072, "k": 64, "dtype": "bf16",
         "teacher": "fp32", "temperature": 2.0, "absent": 0.1, "empty": 0.0},
        # Odd vocabulary, full precision, rows whose teacher kept nothing (padding).
        {"name": "kd_train_fp32_2047x50001_k20", "op": "kd", "train": True, "rows": 2047, "vocab": 50001, "k": 20, "dtype": "fp32",
         "teacher": "fp32", "temperature": 1.0, "absent": 0.2, "empty": 0.1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["ln", "ce", "kd"])
    dtype = rng.choice(["fp32", "bf16"])
    train = rng.random() < 0.7
    if op == "ln":
        hidden = _log_int(rng, 16, 16384)
        limit = 16384 * 8192 // (2 if dtype == "fp32" else 1)
        rows = _log_int(rng, 1, min(65536, limit // hidden))
        return {"op": op, "train": train, "rows": rows, "hidden": hidden, "dtype": dtype, "beta": rng.random() < 0.7}
    if op == "ce":
        hidden = _log_int(rng, 16, 8192)
        vocab = _log_int(rng, 100, 131072)
        limit = 8192 * 4096 * 131072 // (16 if dtype == "fp32" else 2)
        rows = _log_int(rng, 1, max(1, min(8192, limit // (hidden * vocab))))
        return {"op": op, "train": train, "rows": rows, "hidden": hidden, "vocab": vocab, "dtype": dtype,
                "ignored": rng.choice([0.0, 0.1, 0.5])}
    vocab = _log_int(rng, 100, 200000)
    limit = 4096 * 131072 // (2 if dtype == "fp32" else 1)
    rows = _log_int(rng, 1, min(8192, limit // vocab))
    return {"op": op, "train": train, "rows": rows, "vocab": vocab, "k": _log_int(rng, 1, 100), "dtype": dtype,
            "teacher": rng.choice(["fp32", dtype]), "temperature": rng.choice([1.0, 2.0, 4.0]),
            "absent": rng.choice([0.0, 0.2]), "empty": rng.choice([0.0, 0.1])}


def _without(rows, share, gen):
    """A truth value per row: true for int(share * rows) of them, spread at random."""
    return torch.rand(rows, device="cuda", generator=gen).argsort().argsort() < int(share * rows)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    rows, dt = case["rows"], DT[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "ln":
        hidden = case["hidden"]
        # residual streams have an offset and a few loud channels
        loud = 1.0 + 15.0 * (torch.rand(hidden, device="cuda", generator=gen) < 0.01).float()
        s["x"] = (normal(rows, hidden) * loud + 0.5).to(dt)
        s["gamma"] = (1.0 + 0.1 * normal(hidden)).to(dt)
        s["beta"] = (0.1 * normal(hidden)).to(dt) if case["beta"] else None
        s["gy"] = normal(rows, hidden).to(dt) if case["train"] else None
        return s
    if case["op"] == "ce":
        hidden, vocab = case["hidden"], case["vocab"]
        target = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        w = (normal(vocab, hidden) * (1.5 / math.sqrt(hidden))).to(dt)
        # a trained head: the hidden state leans towards its target's row
        s["h"] = (normal(rows, hidden) + 2.0 * w[target].float()).to(dt)
        s["w"] = w
        off = _without(rows, case["ignored"], gen)
        s["target"] = torch.where(off, torch.full_like(target, -100), target)
        # the gradient of a mean over the tokens that count
        s["gy"] = torch.full((rows,), 1.0 / max(1, rows - int(case["ignored"] * rows)), device="cuda")
        return s
    vocab, k = case["vocab"], min(case["k"], case["vocab"])
    z = 2.0 * normal(rows, vocab)
    s["z"] = z.to(dt)
    top = torch.topk(z + 0.7 * normal(rows, vocab), k, dim=-1)
    idx = top.indices
    idx = torch.where(torch.rand(rows, k, device="cuda", generator=gen) < case["absent"], torch.full_like(idx, -1), idx)
    s["idx"] = torch.where(_without(rows, case["empty"], gen)[:, None], torch.full_like(idx, -1), idx)
    s["teacher"] = top.values.to(DT[case["teacher"]])
    s["gy"] = torch.full((rows,), 1.0 / rows, device="cuda")
    return s


# ---------------------------------------------------------------- the formulas, in the type that they are given
def _ln(s, t):
    x, gamma = s["x"].to(t), s["gamma"].to(t)
    hidden = x.shape[-1]
    mean = x.mean(-1)
    xc = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1) + EPS)
    xhat = xc * rstd[:, None]
    y = xhat * gamma
    if s["beta"] is not None:
        y = y + s["beta"].to(t)
    out = [y, mean, rstd]
    if s["gy"] is not None:
        gy = s["gy"].to(t)
        g = gy * gamma
        dx = rstd[:, None] * (g - g.sum(-1, keepdim=True) / hidden - xhat * ((g * xhat).sum(-1, keepdim=True) / hidden))
        out += [dx, (gy * xhat).sum(0)]
        if s["beta"] is not None:
            out.append(gy.sum(0))
    return out


def _lse(z):
    m = z.max(-1).values
    return m + torch.log(torch.exp(z - m[:, None]).sum(-1))


def _ce(s, t):
    h, w, target = s["h"].to(t), s["w"].to(t), s["target"]
    on = (target >= 0) & (target < w.shape[0])
    at = torch.where(on, target, torch.zeros_like(target))[:, None]
    z = h @ w.T
    lse = _lse(z)
    zero = torch.zeros_like(lse)
    out = [torch.where(on, lse - z.gather(1, at)[:, 0], zero), torch.where(on, lse, zero)]
    if s["case"]["train"]:
        g = torch.exp(z - lse[:, None])
        g.scatter_add_(1, at, torch.full_like(at, -1, dtype=t))
        g = torch.where(on[:, None], g * s["gy"].to(t)[:, None], torch.zeros((), dtype=t, device=g.device))
        out += [g @ w, g.T @ h]
    return out


def _kd(s, t):
    tau = s["case"]["temperature"]
    z, tz, idx = s["z"].to(t) / tau, s["teacher"].to(t) / tau, s["idx"]
    there = (idx >= 0) & (idx < z.shape[1])
    on = there.any(-1)
    at = torch.where(there, idx, torch.zeros_like(idx))
    tz = torch.where(there, tz, torch.full_like(tz, -math.inf))
    top = torch.where(on, tz.max(-1).values, torch.zeros((), dtype=t, device=z.device))
    e = torch.exp(tz - top[:, None])
    total = torch.where(on, e.sum(-1), torch.ones((), dtype=t, device=z.device))
    p = e / total[:, None]
    log_p = tz - (top + torch.log(total))[:, None]
    lse = _lse(z)
    log_q = z.gather(1, at) - lse[:, None]
    zero = torch.zeros_like(lse)
    loss = tau * tau * torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(-1)
    out = [torch.where(on, loss, zero), torch.where(on, lse, zero)]
    if s["case"]["train"]:
        dz = torch.exp(z - lse[:, None])
        dz.scatter_add_(1, at, -p)
        out.append(torch.where(on, s["gy"].to(t) * tau, zero)[:, None] * dz)
    return out


def _rounded(s, out):
    """The outputs in the types that a user gets: those of the inputs' shape in the inputs' type, statistics, losses
    and the gradients of the norm's weight and bias in 32 bits."""
    case = s["case"]
    dt = DT[case["dtype"]]
    wide = {"ln": (1, 2, 4, 5), "ce": (0, 1), "kd": (0, 1)}[case["op"]]
    return [o.float() if i in wide else o.to(dt) for i, o in enumerate(out)]


def run(state):
    s, case = state, state["case"]
    if not own:
        return _rounded(s, {"ln": _ln, "ce": _ce, "kd": _kd}[case["op"]](s, torch.float32))
    from cgadimpl_b200 import ops

    if case["op"] == "ln":
        y, mean, rstd = ops.layernorm_affine_fwd(s["x"], s["gamma"], s["beta"], EPS)
        if not case["train"]:
            return [y, mean, rstd]
        dx, dgamma, dbeta = ops.layernorm_affine_bwd(s["x"], s["gamma"], mean, rstd, s["gy"], with_beta=s["beta"] is not None)
        return [y, mean, rstd, dx, dgamma] + ([] if dbeta is None else [dbeta])
    if case["op"] == "ce":
        loss, lse = ops.linear_ce_fwd(s["h"], s["w"], s["target"])
        if not case["train"]:
            return [loss, lse]
        dh, dw = ops.linear_ce_bwd(s["h"], s["w"], s["target"], lse, s["gy"])
        return [loss, lse, dh, dw]
    if not case["train"]:
        return list(ops.distill_topk_fwd(s["z"], s["idx"], s["teacher"], case["temperature"]))
    return list(ops.distill_topk_fwd_bwd(s["z"], s["idx"], s["teacher"], s["gy"], case["temperature"]))


def work(case):
    e, rows, train = ELEM[case["dtype"]], case["rows"], case["train"]
    if case["op"] == "ln":
        n, hidden = rows * case["hidden"], case["hidden"]
        small = 8 * rows + (2 if case["beta"] else 1) * hidden * (e + (4 if train else 0))
        return {"bytes": (4 if train else 2) * n * e + small, "flops": (19 if train else 8) * n}
    if case["op"] == "ce":
        on = rows - int(case["ignored"] * rows)
        hidden, vocab = case["hidden"], case["vocab"]
        # forward: the logits; backward: the logits again (they are not kept) and the products for both gradients
        product = 2 * on * hidden * vocab
        ends = (on + vocab) * hidden * e + rows * 16
        if train:
            ends += (rows + vocab) * hidden * e + rows * 4
        return {"bytes": ends, "flops": (4 if train else 1) * product}
    on = rows - int(case["empty"] * rows)
    n, k = on * case["vocab"], min(case["k"], case["vocab"])
    small = rows * 8 + rows * k * (8 + ELEM[case["teacher"]])
    return {"bytes": n * e + (rows * case["vocab"] * e + rows * 4 if train else 0) + small, "flops": (9 if train else 5) * n}


def exact(case, seed):
    s = prepare(case, seed)
    wide = torch.float64

    def pieces(n, width):
        step = max(1, (1 << 27) // max(1, width))
        return [(a, min(n, a + step)) for a in range(0, n, step)]

    rows = case["rows"]
    if case["op"] == "ln":
        gamma = s["gamma"].to(wide)
        y, mean, rstd, dx, dgamma, dbeta = [], [], [], [], 0.0, 0.0
        for a, b in pieces(rows, case["hidden"]):
            x = s["x"][a:b].to(wide)
            var, mu = torch.var_mean(x, dim=-1, correction=0)
            r = (var + EPS).rsqrt()
            hat = (x - mu[:, None]) * r[:, None]
            mean.append(mu)
            rstd.append(r)
            y.append(hat * gamma + (s["beta"].to(wide) if case["beta"] else 0.0))
            if case["train"]:
                gy = s["gy"][a:b].to(wide)
                # the Jacobian of the normalisation is (I - 1 1'/n - hat hat'/n) * rstd
                v = gy * gamma
                v = v - v.mean(-1, keepdim=True)
                dx.append((v - hat * (v * hat).mean(-1, keepdim=True)) * r[:, None])
                dgamma = dgamma + torch.einsum("rh,rh->h", gy, hat)
                dbeta = dbeta + gy.sum(0)
        out = [torch.cat(y), torch.cat(mean), torch.cat(rstd)]
        if case["train"]:
            out += [torch.cat(dx), dgamma] + ([dbeta] if case["beta"] else [])
        return out
    if case["op"] == "ce":
        w = s["w"].to(wide)
        vocab = case["vocab"]
        loss, lse, dh, dw = [], [], [], 0.0
        for a, b in pieces(rows, vocab):
            h, target = s["h"][a:b].to(wide), s["target"][a:b]
            counts = ((target >= 0) & (target < vocab)).to(wide)
            log_p = torch.log_softmax(h @ w.T, dim=-1)
            onehot = torch.zeros_like(log_p)
            onehot.scatter_(1, target.clamp(0, vocab - 1)[:, None], 1.0)
            z_at = (h * w[target.clamp(0, vocab - 1)]).sum(-1)
            nll = -(log_p * onehot).sum(-1)
            loss.append(nll * counts)
            lse.append((nll + z_at) * counts)
            if case["train"]:
                g = (log_p.exp_() - onehot) * (s["gy"][a:b].to(wide) * counts)[:, None]
                dh.append(g @ w)
                dw = dw + g.T @ h
        out = [torch.cat(loss), torch.cat(lse)]
        return out + [torch.cat(dh), dw] if case["train"] else out
    tau, vocab = case["temperature"], case["vocab"]
    loss, lse, dz = [], [], []
    for a, b in pieces(rows, vocab):
        z, tz, idx = s["z"][a:b].to(wide), s["teacher"][a:b].to(wide), s["idx"][a:b]
        there = (idx >= 0) & (idx < vocab)
        counts = there.any(-1).to(wide)
        p = torch.softmax(torch.where(there, tz / tau, torch.full_like(tz, -1e300)), dim=-1) * there.to(wide) * counts[:, None]
        log_q = torch.log_softmax(z / tau, dim=-1)
        full = torch.zeros_like(log_q).scatter_add_(1, idx.clamp(0, vocab - 1), p)
        cross = -(full * log_q).sum(-1)
        entropy = -torch.special.xlogy(p, p).sum(-1)
        loss.append(tau * tau * (cross - entropy))
        lse.append((z[:, 0] / tau - log_q[:, 0]) * counts)
        if case["train"]:
            dz.append((log_q.exp() * counts[:, None] - full) * (tau * s["gy"][a:b].to(wide))[:, None])
    out = [torch.cat(loss), torch.cat(lse)]
    return out + [torch.cat(dz)] if case["train"] else out
