"""Products with what follows them, forward and backward: the dense product with
bias, activation and residual, the expert products on ragged rows, and the
cross entropy over a large vocabulary.

``run`` computes each in its plain form from elementary torch operations where
``own`` is false, and through the package's entry points where it is true.
Sizes are those of the repository's own workloads (hidden 7168, expert width
2048, 256 experts, top-8, one rank of 8; the 8192 x 3584 projections; 4096
cubed) and generic smaller, larger and odd ones.  Inputs are drawn on the GPU
from the seed alone; ``exact`` gives the outputs in 64 bits from the
definitions.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
ZIPF = 1.1           # popularity of experts and of words: Zipf with this exponent
IGNORE = -100        # label of a token without a loss


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a small projection: a launch, all latency
        _lin("lin_token", 1, 2048, 2048, "silu", True, ""),
        # a decode batch through one rank's down-projection, added to the residual stream
        _lin("lin_decode", 32, 8192, 3584, "none", True, "bf16"),
        # a gathered batch through one rank's up-projection of a training step, which keeps the pre-activation
        _lin("lin_train", 16384, 8192, 3584, "gelu", True, "", pre=True),
        # an odd batch through odd sizes in columns of a wider matrix, onto a residual stream in float32
        _lin("lin_odd", 1003, 2811, 1501, "relu", True, "f32", pad=13),
        # gradient of a square projection with its activation
        _lin_grad("lin_grad", 4096, 4096, 4096, "silu", "bf16"),
        # a decode batch's rows (one or a few per expert) through one rank's experts
        _experts("experts_decode", "up", 64, 7168, 2048, 256, 8, 8, "bf16"),
        # a training batch through one rank's experts, which keeps the pre-activations
        _experts("experts_up", "up", 4096, 7168, 2048, 256, 8, 8, "bf16"),
        # gradients of the second product and of the activation in front of it
        _experts("experts_down_grad", "down_grad", 4096, 7168, 2048, 256, 8, 8, "bf16"),
        # gradients of the first product, ragged sizes, every expert here, weight gradients in float32
        _experts("experts_up_grad_ragged", "up_grad", 1000, 2056, 1384, 60, 1, 4, "f32"),
        # loss and gradients of a small model's step, odd vocabulary, a tenth of the labels ignored
        _vocab("vocab_small", 520, 1024, 5003, 0.1),
        # of an ordinary one
        _vocab("vocab_train", 2048, 2048, 32000, 0.0),
        # of a long batch over a large vocabulary
        _vocab("vocab_large", 4096, 4096, 131072, 0.05),
    ]


def _lin(name, M, K, N, act, bias, residual, pre=False, pad=0):
    """residual: its type, or ""; pre: whether the pre-activation is kept; pad: columns of A's rows behind K."""
    return {"name": name, "op": "lin", "M": M, "K": K, "N": N, "act": act, "bias": bias, "residual": residual,
            "pre": pre, "pad": pad}


def _lin_grad(name, M, K, N, act, grad, pad=0):
    """grad: type of B's gradient."""
    return {"name": name, "op": "lin_grad", "M": M, "K": K, "N": N, "act": act, "grad": grad, "pad": pad}


def _experts(name, op, T, H, I, E, ep, k, grad):
    return {"name": name, "op": op, "T": T, "H": H, "I": I, "E": E, "ep": ep, "k": k, "grad": grad}


def _vocab(name, T, H, V, ignored):
    return {"name": name, "op": "vocab", "T": T, "H": H, "V": V, "ignored": ignored}


def draw(rng):
    """One more case of the same ranges."""
    def spread(lo, hi, step=1):
        return step * max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step))

    op = rng.choice(["lin", "lin_grad", "up", "down_grad", "up_grad", "vocab"])
    step = rng.choice([1, 8, 64])
    if op == "lin":
        K, N = spread(64, 8192, step), spread(64, 8192, step)
        c = _lin("", min(spread(1, 16384), 16384 * 8192 * 3584 // (K * N)), K, N,
                 rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), rng.random() < 0.5,
                 rng.choice(["", "bf16", "f32"]), rng.random() < 0.3, rng.choice([0, 0, rng.randrange(1, 200)]))
    elif op == "lin_grad":
        act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        c = _lin_grad("", spread(128, 8192), spread(128, 8192, step), spread(128, 4096, step), act,
                      rng.choice(["bf16", "f32"]) if act in ("none", "relu") else "bf16",
                      rng.choice([0, 0, rng.randrange(1, 200)]))
    elif op == "vocab":
        T, H = spread(256, 4096), spread(256, 4096, rng.choice([1, 8, 64]))
        c = _vocab("", T, H, spread(1000, 131072, step), rng.choice([0.0, rng.uniform(0.02, 0.5)]))
    else:
        ep = rng.choice([1, 8])
        E = ep * spread(4, 48)
        c = _experts("", op, spread(1 if op == "up" else 64, 4096 if ep > 1 else 1024), spread(256, 7168, step),
                     spread(128, 2048, step), E, ep, min(E // ep, spread(1, 8)), rng.choice(["bf16", "f32"]))
    del c["name"]
    return c


# ------------------------------------------------------------------- inputs
def _generator(seed, part):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + part)


def _randn(shape, seed, part, scale, dtype=BF16):
    """N(0, scale^2), drawn in slices so that no large fp32 copy is held."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    g = _generator(seed, part)
    for piece in out.view(-1).split(1 << 27):
        piece.copy_(torch.randn(piece.numel(), generator=g, device=DEV).mul_(scale))
    return out


def _type(name):
    return F32 if name == "f32" else BF16


def _zipf(n, of):
    """Log popularity of n things, a property of the model: Zipf ranks dealt to them once."""
    return -ZIPF * torch.log(torch.randperm(n, generator=torch.Generator().manual_seed(of)).double() + 1.0)


def _counts(c, seed):
    """Rows of each local expert: each token takes its k best of log popularity and its own preference."""
    u = torch.rand((c["T"], c["E"]), generator=_generator(seed, 3), device=DEV).clamp_(1e-7, 1 - 1e-6)
    x = _zipf(c["E"], 6).to(DEV, F32) - torch.log(-torch.log(u))
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, : c["k"]]
    return torch.bincount(ids.flatten(), minlength=c["E"])[: c["E"] // c["ep"]].to(torch.int32)


def _capacity(c):
    """Rows of the buffers: more than a batch routes here."""
    rows = _expected(c)[0]
    return min(c["T"] * min(c["k"], c["E"] // c["ep"]), int(1.1 * rows + 8 * math.sqrt(rows)) + 64)


def _rows(c, counts, width, seed, part, scale):
    """Rows of all experts, one expert after another, in a buffer of zeros."""
    n = int(counts.sum())
    out = torch.zeros((_capacity(c), width), dtype=BF16, device=DEV)
    if n:
        out[:n] = _randn((n, width), seed, part, scale)
    return out


def _lin_inputs(c, seed):
    M, K, N = c["M"], c["K"], c["N"]
    s = {"a": _randn((M, K + c["pad"]), seed, 1, 1.0)[:, :K], "b": _randn((K, N), seed, 2, K ** -0.5)}
    if c["op"] == "lin":
        s["bias"] = _randn((N,), seed, 3, 0.5) if c["bias"] else None
        s["res"] = _randn((M, N), seed, 4, 1.0, _type(c["residual"])) if c["residual"] else None
    else:
        s["dc"] = _randn((M, N), seed, 5, 1.0 / M)
        s["pre"] = None if c["act"] == "none" else _randn((M, N), seed, 6, 1.0)
    return s


def _expert_inputs(c, seed):
    E, H, I = c["E"] // c["ep"], c["H"], c["I"]
    n = _counts(c, seed)
    s = {"counts": n}
    if c["op"] == "up":
        s["x"] = _rows(c, n, H, seed, 11, 1.0)
        s["w"] = _randn((E, H, 2 * I), seed, 12, H ** -0.5)
    elif c["op"] == "down_grad":
        s["dy"] = _rows(c, n, H, seed, 13, 1.0 / c["T"])
        s["act"] = _rows(c, n, I, seed, 14, 0.5)
        s["h"] = _rows(c, n, 2 * I, seed, 15, 1.0)
        s["w"] = _randn((E, I, H), seed, 16, I ** -0.5)
    else:
        s["dh"] = _rows(c, n, 2 * I, seed, 17, 1.0 / c["T"])
        s["x"] = _rows(c, n, H, seed, 11, 1.0)
        s["w"] = _randn((E, H, 2 * I), seed, 12, H ** -0.5)
    return s


def _vocab_inputs(c, seed):
    T, H, V = c["T"], c["H"], c["V"]
    x = _randn((T, H), seed, 21, 1.0)
    below = torch.cumsum(torch.softmax(_zipf(V, 7), 0), 0).to(DEV)
    u = torch.rand(T, generator=_generator(seed, 22), device=DEV, dtype=F64)
    labels = torch.searchsorted(below, u, right=True).clamp_(max=V - 1)
    if c["ignored"]:  # padding: what such a row holds is nobody's business
        gone = torch.rand(T, generator=_generator(seed, 23), device=DEV) < c["ignored"]
        labels[gone] = IGNORE
        x[gone] = float("nan")
    # logits of a deviation of about 2, as a model that has learned something has
    return {"x": x, "w": _randn((H, V), seed, 24, 2.0 * H ** -0.5), "labels": labels,
            "dloss": torch.full((T,), 1.0 / T, dtype=F32, device=DEV)}


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    if own:
        from mkernel_amd import ops
        s["ops"] = ops
    if c["op"] in ("lin", "lin_grad"):
        s.update(_lin_inputs(c, seed))
        if c["op"] == "lin" and c["pre"]:  # kept for the backward pass
            s["pre"] = torch.empty((c["M"], c["N"]), dtype=BF16, device=DEV)
    elif c["op"] == "vocab":
        s.update(_vocab_inputs(c, seed))
    else:
        s.update(_expert_inputs(c, seed))
        E, H, I, R = c["E"] // c["ep"], c["H"], c["I"], _capacity(c)
        # buffers that a step writes into: rows behind the routed ones stay as they are
        if c["op"] == "up":
            s["out"] = {"act": torch.zeros((R, I), dtype=BF16, device=DEV), "h": torch.zeros((R, 2 * I), dtype=BF16, device=DEV)}
        elif c["op"] == "down_grad":
            s["out"] = {"dh": torch.zeros((R, 2 * I), dtype=BF16, device=DEV),
                        "dw": torch.zeros((E, I, H), dtype=_type(c["grad"]), device=DEV)}
        else:
            s["out"] = {"dx": torch.zeros((R, H), dtype=BF16, device=DEV),
                        "dw": torch.zeros((E, H, 2 * I), dtype=_type(c["grad"]), device=DEV)}
        # where each routed row lies in a block of equal rows for every expert: the plan of a batched product
        n = s["counts"].long()
        e = torch.repeat_interleave(torch.arange(E, device=DEV), n)
        s["at"] = (e, torch.arange(e.numel(), device=DEV) - (torch.cumsum(n, 0) - n)[e])
        s["most"] = max(1, int(n.max()))
    return s


# ------------------------------------------------------------------- plain forms
def _act(x, act):
    if act == "relu":
        return torch.where(x < 0, 0.0, x)
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return x


def _act_slope(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * math.sqrt(2 / math.pi) * (1.0 + 3 * 0.044715 * x * x)
    s = 1.0 / (1.0 + torch.exp(-x))
    return s * (1.0 + x * (1.0 - s))


def _plain_lin(s):
    c = s["case"]
    x = s["a"].float() @ s["b"].float()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    y = _act(x, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = {"y": y.to(F32 if c["residual"] == "f32" else BF16)}
    if c["pre"]:
        s["pre"].copy_(x)
        out["pre"] = s["pre"]
    return out


def _plain_lin_grad(s):
    c = s["case"]
    d = s["dc"].float()
    if s["pre"] is not None:
        d = d * _act_slope(s["pre"].float(), c["act"])
    return {"da": (d @ s["b"].float().t()).to(BF16), "db": (s["a"].float().t() @ d).to(_type(c["grad"])),
            "dbias": d.sum(0)}


def _spread(s, rows):
    """Rows of the experts as equal blocks [E, most, width], zeros where an expert has fewer."""
    out = torch.zeros((s["counts"].numel(), s["most"], rows.shape[1]), dtype=F32, device=DEV)
    out[s["at"]] = rows[: s["at"][0].numel()].float()
    return out


def _plain_experts(s):
    c, o, n = s["case"], s["out"], s["at"][0].numel()
    w = s["w"].float()
    if c["op"] == "up":
        h = torch.bmm(_spread(s, s["x"]), w)[s["at"]]
        o["h"][:n] = h
        g, u = h[:, : c["I"]], h[:, c["I"]:]
        o["act"][:n] = g / (1.0 + torch.exp(-g)) * u
    elif c["op"] == "down_grad":
        dy = _spread(s, s["dy"])
        d = torch.bmm(dy, w.transpose(1, 2).contiguous())[s["at"]]
        h = s["h"][:n].float()
        g, u = h[:, : c["I"]], h[:, c["I"]:]
        sg = 1.0 / (1.0 + torch.exp(-g))
        o["dh"][:n, : c["I"]] = d * u * sg * (1.0 + g * (1.0 - sg))
        o["dh"][:n, c["I"]:] = d * g * sg
        o["dw"].copy_(torch.bmm(_spread(s, s["act"]).transpose(1, 2).contiguous(), dy))
    else:
        dh = _spread(s, s["dh"])
        o["dx"][:n] = torch.bmm(dh, w.transpose(1, 2).contiguous())[s["at"]]
        o["dw"].copy_(torch.bmm(_spread(s, s["x"]).transpose(1, 2).contiguous(), dh))
    return o


def _plain_vocab(s):
    live = s["labels"] >= 0
    x = torch.where(live[:, None], s["x"], 0.0).float()
    at = s["labels"].clamp(min=0)[:, None]
    w = s["w"].float()
    z = x @ w
    m = z.amax(1, keepdim=True)
    target = z.gather(1, at)
    e = torch.exp(z - m)
    lse = m + torch.log(e.sum(1, keepdim=True, dtype=F64)).float()
    d = torch.exp(z - lse)
    d.scatter_add_(1, at, torch.full_like(target, -1.0))
    d = d * torch.where(live, s["dloss"], 0.0)[:, None]
    return {"loss": torch.where(live, (lse - target)[:, 0], 0.0), "dx": (d @ w.t()).to(BF16), "dw": (x.t() @ d).to(BF16)}


# ------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "lin":
            return _plain_lin(s)
        if c["op"] == "lin_grad":
            return _plain_lin_grad(s)
        return _plain_vocab(s) if c["op"] == "vocab" else _plain_experts(s)
    ops = s["ops"]
    if c["op"] == "lin":
        y = ops.gemm_act(s["a"], s["b"], bias=s["bias"], act=c["act"], residual=s["res"], pre=s.get("pre"),
                         out_dtype=F32 if c["residual"] == "f32" else BF16)
        return {"y": y, "pre": s["pre"]} if c["pre"] else {"y": y}
    if c["op"] == "lin_grad":
        da, db, dbias = ops.gemm_act_backward(s["dc"], s["a"], s["b"], pre=s["pre"], act=c["act"],
                                              dB_dtype=_type(c["grad"]))
        return {"da": da, "db": db, "dbias": dbias}
    if c["op"] == "vocab":
        r = ops.vocab_loss(s["x"], s["w"], s["labels"], ignore_index=IGNORE)
        dx, dw = ops.vocab_loss_backward(s["x"], s["w"], s["labels"], r["lse"], s["dloss"], ignore_index=IGNORE)
        return {"loss": r["loss"], "dx": dx, "dw": dw}
    o, n = s["out"], s["counts"]
    if c["op"] == "up":
        ops.moe_ragged_gemm(s["x"], s["w"], n, mode=1, out=o["act"], h=o["h"])
    elif c["op"] == "down_grad":
        ops.moe_ragged_gemm_dgrad(s["dy"], s["w"], n, h=s["h"], out=o["dh"])
        ops.moe_ragged_gemm_wgrad(s["act"], s["dy"], n, out=o["dw"])
    else:
        ops.moe_ragged_gemm_dgrad(s["dh"], s["w"], n, out=o["dx"])
        ops.moe_ragged_gemm_wgrad(s["x"], s["dh"], n, out=o["dw"])
    return o


# ------------------------------------------------------------------- what it takes
def _expected(c):
    """(routed rows, local experts with a row) to expect of a batch: an expert is among a token's top-k with
    probability 1 - exp(-x p_e)."""
    p = torch.softmax(_zipf(c["E"], 6), 0)
    lo, hi = 0.0, 1e6
    for _ in range(200):
        x = 0.5 * (lo + hi)
        lo, hi = (x, hi) if float((1 - torch.exp(-x * p)).sum()) < c["k"] else (lo, x)
    hit = (1 - torch.exp(-x * p))[: c["E"] // c["ep"]]
    return max(1.0, float(c["T"] * hit.sum())), max(1.0, float((1 - (1 - hit) ** c["T"]).sum()))


def work(case):
    c = case
    if c["op"] == "lin":
        M, K, N = c["M"], c["K"], c["N"]
        res = {"": 0, "bf16": 2, "f32": 4}[c["residual"]]
        y = 4 if c["residual"] == "f32" else 2
        return {"bytes": 2 * (M * K + K * N) + M * N * (y + res + 2 * c["pre"]) + 2 * N * c["bias"], "flops": 2 * M * N * K}
    if c["op"] == "lin_grad":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": 2 * M * N * (1 if c["act"] == "none" else 2) + 4 * M * K + (2 + (4 if c["grad"] == "f32" else 2)) * K * N + 4 * N,
                "flops": 4 * M * N * K}
    if c["op"] == "vocab":
        T, H, V = c["T"], c["H"], c["V"]
        return {"bytes": 4 * T * H + 4 * H * V + 16 * T, "flops": 6 * T * H * V}
    rows, used = _expected(c)
    E, H, I = c["E"] // c["ep"], c["H"], c["I"]
    size = 4 if c["grad"] == "f32" else 2
    if c["op"] == "up":
        return {"bytes": 2 * rows * (H + 3 * I) + used * 4 * H * I, "flops": 4 * rows * H * I}
    if c["op"] == "down_grad":
        return {"bytes": 2 * rows * (H + 5 * I) + used * 2 * I * H + E * size * I * H, "flops": 4 * rows * H * I}
    return {"bytes": 2 * rows * (2 * I + 2 * H) + used * 4 * I * H + E * size * 2 * I * H, "flops": 8 * rows * H * I}


# ------------------------------------------------------------------- 64 bits
def _exact_act(x, act):
    """act(x) and its slope."""
    if act == "none":
        return x, torch.ones_like(x)
    if act == "relu":
        return x.clamp(min=0), (x > 0).to(F64)
    if act == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * (1 - s)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-x / math.sqrt(2.0))
        return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    # half of 1 + tanh(v) is sigmoid(2 v)
    s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
    return x * s, s + x * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * x * x)


def exact(case, seed):
    c = case
    if c["op"] in ("lin", "lin_grad"):
        s = _lin_inputs(c, seed)
        a, b = s["a"].to(F64), s["b"].to(F64)
        if c["op"] == "lin_grad":
            d = s["dc"].to(F64)
            if s["pre"] is not None:
                d = d * _exact_act(s["pre"].to(F64), c["act"])[1]
            return {"da": d @ b.t(), "db": a.t() @ d, "dbias": d.sum(0)}
        x = a @ b
        if s["bias"] is not None:
            x += s["bias"].to(F64)
        y = _exact_act(x, c["act"])[0]
        if s["res"] is not None:
            y = y + s["res"].to(F64)
        return {"y": y, "pre": x} if c["pre"] else {"y": y}
    if c["op"] == "vocab":
        s = _vocab_inputs(c, seed)
        T, H, V = c["T"], c["H"], c["V"]
        on = (s["labels"] != IGNORE).nonzero()[:, 0]
        x, at = s["x"][on].to(F64), s["labels"][on]
        w = s["w"].to(F64)
        logp = torch.log_softmax(x @ w, 1)
        here = torch.arange(on.numel(), device=DEV)
        loss = torch.zeros(T, dtype=F64, device=DEV)
        loss[on] = -logp[here, at]
        d = logp.exp_()
        d[here, at] -= 1
        d *= s["dloss"][on].to(F64)[:, None]
        dx = torch.zeros((T, H), dtype=F64, device=DEV)
        dx[on] = d @ w.t()
        return {"loss": loss, "dx": dx, "dw": x.t() @ d}
    s = _expert_inputs(c, seed)
    E, H, I = c["E"] // c["ep"], c["H"], c["I"]
    n = s["counts"].tolist()
    R = _capacity(c)
    if c["op"] == "up":
        o = {"act": torch.zeros((R, I), dtype=F64, device=DEV), "h": torch.zeros((R, 2 * I), dtype=F64, device=DEV)}
    elif c["op"] == "down_grad":
        o = {"dh": torch.zeros((R, 2 * I), dtype=F64, device=DEV), "dw": torch.zeros((E, I, H), dtype=F64, device=DEV)}
    else:
        o = {"dx": torch.zeros((R, H), dtype=F64, device=DEV), "dw": torch.zeros((E, H, 2 * I), dtype=F64, device=DEV)}
    lo = 0
    for e in range(E):
        hi = lo + n[e]
        if n[e]:
            w = s["w"][e].to(F64)
            if c["op"] == "up":
                h = s["x"][lo:hi].to(F64) @ w
                o["h"][lo:hi] = h
                o["act"][lo:hi] = _exact_act(h[:, :I], "silu")[0] * h[:, I:]
            elif c["op"] == "down_grad":
                dy = s["dy"][lo:hi].to(F64)
                d = dy @ w.t()
                h = s["h"][lo:hi].to(F64)
                a, slope = _exact_act(h[:, :I], "silu")
                o["dh"][lo:hi] = torch.cat([d * h[:, I:] * slope, d * a], 1)
                o["dw"][e] = s["act"][lo:hi].to(F64).t() @ dy
            else:
                dh = s["dh"][lo:hi].to(F64)
                o["dx"][lo:hi] = dh @ w.t()
                o["dw"][e] = s["x"][lo:hi].to(F64).t() @ dh
        lo = hi
    return o
