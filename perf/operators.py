"""Operators around the routed expert layer: the router with its balance loss
and gradient, the gradient of the weighted combine, and the products with 4-bit
weights that serve small batches.

``run`` computes each in its plain form from elementary torch operations where
``own`` is false, and through the package's entry points where it is true.
Sizes are those of the repository's own workloads (hidden 7168, expert width
2048, 256 experts, top-8, one rank of 8; the 8192 x 3584 projections) and
generic smaller and ragged ones.  Inputs are drawn on the GPU from the seed
alone; ``exact`` gives the outputs in 64 bits from the definitions.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
BLOCK = 128          # rows of an expert's padding block
ZIPF = 1.1           # popularity of the experts: Zipf with this exponent
COEF = 0.01          # weight of the balance loss in the training loss
INF = float("inf")


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token's routing in a decode step: a launch, all latency
        _route("route_token", 1, 256, 8, "f32", True, 0, 0.0),
        # a long prompt's routing from the logits that a bf16 GEMM gave, unnormalised gates
        _route("route_prefill", 16384, 256, 8, "bf16", False, 0, 0.0),
        # the router's part of a training step: gates, counts, balance loss, and the logits' gradient
        _train("router_train", 4096, 256, 8, "f32", True, 0, 0.0),
        # the same over a long ragged batch with padded tokens, few experts in the columns of a wider GEMM's output
        _train("router_train_long", 131001, 60, 4, "bf16", False, 196, 0.1),
        # gradient of the combine at one rank of eight: expert rows and gates
        _combine("combine_grad", 2048, 7168, 256, 8, 8, "f32"),
        # the same for a small ragged batch with every expert on this GPU
        _combine("combine_grad_ragged", 333, 2056, 60, 1, 4, "bf16"),
        # one token through a small projection of 4-bit weights: latency
        _w4("w4_token", 1, 2048, 2048, 128, False),
        # one token through one rank's up-projection
        _w4("w4_up", 1, 8192, 3584, 128, False),
        # a decode batch through one rank's down-projection, finer groups
        _w4("w4_batch", 64, 3584, 8192, 64, False),
        # a few drafted tokens, ragged sizes, the finest groups with zero points
        _w4("w4_ragged", 5, 5608, 2811, 32, True),
        # one token through a small routed layer, logits to output
        _moe("moe_w4_token", 1, 2048, 1024, 64, 1, 8, 128),
        # a decode batch through one rank's experts, logits to output
        _moe("moe_w4_decode", 64, 7168, 2048, 256, 8, 8, 128),
    ]


def _route(name, T, E, k, dtype, renorm, pad, masked):
    """pad: columns of the logits' rows behind the experts; masked: share of padded tokens."""
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "dtype": dtype, "renorm": renorm, "pad": pad,
            "masked": masked}


def _train(name, T, E, k, dtype, renorm, pad, masked):
    return dict(_route(name, T, E, k, dtype, renorm, pad, masked), op="train")


def _combine(name, T, H, E, ep, k, dtype):
    return {"name": name, "op": "combine", "T": T, "H": H, "E": E, "ep": ep, "k": k, "dtype": dtype}


def _w4(name, M, K, N, group, zeros):
    return {"name": name, "op": "w4", "M": M, "K": K, "N": N, "group": group, "zeros": zeros}


def _moe(name, T, H, I, E, ep, k, group):
    return {"name": name, "op": "moe", "T": T, "H": H, "I": I, "E": E, "ep": ep, "k": k, "group": group}


def draw(rng):
    """One more case of the same ranges."""
    def spread(lo, hi, step=1):
        return step * max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step))

    op = rng.choice(["route", "train", "combine", "w4", "w4", "moe"])
    if op in ("route", "train"):
        E = spread(8, 512)
        T = min(spread(1, 131072), (131072 if op == "train" else 16384) * 256 // max(E, 64))
        c = (_route if op == "route" else _train)(
            "", T, E, min(E, spread(1, 16)), rng.choice(["f32", "bf16"]), rng.random() < 0.5,
            rng.choice([0, 0, rng.randrange(1, 200)]), rng.choice([0.0, 0.0, rng.uniform(0.02, 0.6)]))
    elif op == "combine":
        ep = rng.choice([1, 4, 8])
        E = ep * spread(4, 32)
        c = _combine("", spread(1, 2048 if ep > 1 else 700), spread(256, 7168, 8), E, ep, min(E // ep, spread(1, 8)),
                     rng.choice(["f32", "bf16"]))
    elif op == "w4":
        zeros = rng.random() < 0.5
        c = _w4("", spread(1, 64), spread(256, 8192, 8), spread(64, 8192), rng.choice([32, 64, 128]), zeros)
    else:
        ep = rng.choice([1, 8])
        n_local = rng.choice([8, 16, 32])
        c = _moe("", spread(1, 64), spread(512, 7168, 8), spread(256, 2048, 16), n_local * ep, ep,
                 rng.choice([2, 4, 8]), rng.choice([64, 128]))
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


def _popularity(E):
    """Log popularity of the experts, a property of the model: Zipf ranks dealt to the experts once."""
    return -ZIPF * torch.log(torch.randperm(E, generator=torch.Generator().manual_seed(6)).double() + 1.0)


def _logits(c, seed):
    """Router logits [T, E] (a view of wider rows where the case has padding) and the mask of real tokens:
    log popularity of the experts plus each token's own preference."""
    T, E = c["T"], c["E"]
    u = torch.rand((T, E), generator=_generator(seed, 3), device=DEV).clamp_(1e-7, 1 - 1e-6)
    x = _popularity(E).to(DEV, F32) - torch.log(-torch.log(u))
    mask = None
    if c.get("masked"):
        mask = torch.rand(T, generator=_generator(seed, 4), device=DEV) >= c["masked"]
        x[~mask] = float("nan")  # what a padded token's row holds is nobody's business
    wide = torch.zeros((T, E + c.get("pad", 0)), dtype=F32 if c.get("dtype", "f32") == "f32" else BF16, device=DEV)
    wide[:, :E] = x
    return wide[:, :E], mask


def _capacity(c):
    """Padded rows of the worst routing of the batch."""
    return (c["T"] * c["k"] + c["E"] // c["ep"] * (BLOCK - 1) + BLOCK - 1) // BLOCK * BLOCK


def _codes(shape, group, seed, part, zeros=False):
    """4-bit codes [.., K, N] (one a byte), bf16 scales [.., ceil(K / group), N] and zero points, as a
    quantised checkpoint holds them; the weights they stand for have a deviation of about K ** -0.5."""
    *lead, K, N = shape
    groups = (*lead, (K + group - 1) // group, N)
    q = torch.randint(0, 16, shape, generator=_generator(seed, part), device=DEV, dtype=torch.uint8)
    s = torch.rand(groups, generator=_generator(seed, part + 1), device=DEV).add_(0.5).mul_(K ** -0.5 / 4.6).to(BF16)
    z = torch.randint(5, 11, groups, generator=_generator(seed, part + 2), device=DEV, dtype=torch.uint8) if zeros else None
    return q, s, z


def _choice(c, seed):
    """ids int32 and gates float32 [T, k] of a routed batch."""
    x, _ = _logits(c, seed)
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return ids[:, : c["k"]].to(torch.int32).contiguous(), torch.softmax(top[:, : c["k"]], dim=1).contiguous()


def _expert_rows(c, ids):
    """Where the routed rows of the local experts lie, expert by expert in blocks of BLOCK rows:
    (token, column of ids) of each row, -1 on padding rows."""
    n_local = c["E"] // c["ep"]
    where = []
    for e in range(n_local):
        at = (ids == e).nonzero()
        fill = (-at.shape[0]) % BLOCK
        where.append(at)
        where.append(torch.full((fill, 2), -1, dtype=at.dtype, device=DEV))
    return torch.cat(where)


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    op = c["op"]
    if own:
        from mkernel_amd import ops
        s["ops"] = ops
    if op in ("route", "train"):
        s["logits"], s["mask"] = _logits(c, seed)
        if op == "train":  # gradients of a mean over the tokens
            s["dgates"] = _randn((c["T"], c["k"]), seed, 5, 0.1 / c["T"], F32)
            s["dloss"] = torch.ones(1, dtype=F32, device=DEV)
    elif op == "combine":
        dt = F32 if c["dtype"] == "f32" else BF16
        s["dy"] = _randn((c["T"], c["H"]), seed, 1, 1.0 / c["T"], dt)
        s["ids"], s["gates"] = _choice(c, seed)
        s["where"] = _expert_rows(c, s["ids"])
        # buffers at the capacity, the row count on the device: rows behind the last block stay as they are
        s["ye"] = torch.zeros((_capacity(c), c["H"]), dtype=BF16, device=DEV)
        s["ye"][: s["where"].shape[0]] = _randn((s["where"].shape[0], c["H"]), seed, 2, 1.0)
        s["dye"] = torch.zeros_like(s["ye"])
        if own:  # the tables that the forward pass was run with
            s["t"] = s["ops"].moe_build_indices_dev(s["ids"], s["gates"].float(), 0, c["E"] // c["ep"], sync=False)
    elif op == "w4":
        s["x"] = _randn((c["M"], c["K"]), seed, 1, 1.0)
        s["w"] = _codes((c["K"], c["N"]), c["group"], seed, 10, c["zeros"])
        if own:
            s["packed"] = s["ops"].w4_pack(s["w"][0], s["w"][1], c["group"], zeros=s["w"][2])
    else:
        n_local, H, I = c["E"] // c["ep"], c["H"], c["I"]
        s["x"] = _randn((c["T"], H), seed, 1, 1.0)
        s["logits"], _ = _logits(c, seed)
        s["w1"] = _codes((n_local, H, 2 * I), c["group"], seed, 10)
        s["w2"] = _codes((n_local, I, H), c["group"], seed, 20)
        if own:
            s["p1"] = s["ops"].w4_pack(s["w1"][0], s["w1"][1], c["group"])
            s["p2"] = s["ops"].w4_pack(s["w2"][0], s["w2"][1], c["group"])
            s["act"] = torch.empty((_capacity(c), 2 * I), dtype=BF16, device=DEV)
            s["ye"] = torch.empty((_capacity(c), H), dtype=F32, device=DEV)
            s["y"] = torch.empty((c["T"], H), dtype=BF16, device=DEV)
    return s


# ------------------------------------------------------------------- plain forms
def _plain_route(c, logits, mask):
    """ids, gates, and the probabilities [T, E] with the rows that count."""
    x = logits.float()
    if mask is not None:
        x = torch.where(mask[:, None], x, -INF)
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top, ids = top[:, : c["k"]], ids[:, : c["k"]]
    live = top[:, :1] > -INF
    big = torch.where(live, top[:, :1], 0.0)
    e = torch.exp(x - big)
    p = e / torch.where(live, e.sum(1, keepdim=True), 1.0)
    chosen = top > -INF
    if c["renorm"]:
        g = torch.exp(top - big)
        g = g / torch.where(live, g.sum(1, keepdim=True), 1.0)
    else:
        g = p.gather(1, ids)
    ids = torch.where(chosen, ids, -1).to(torch.int32)
    return ids, torch.where(chosen, g, 0.0), p, live


def _plain_train(c, s):
    E, k = c["E"], c["k"]
    ids, gates, p, live = _plain_route(c, s["logits"], s["mask"])
    hit = torch.zeros((c["T"], E + 1), dtype=F32, device=DEV)
    hit.scatter_(1, torch.where(ids < 0, E, ids).long(), 1.0)
    hit = hit[:, :E]
    counts = hit.sum(0, dtype=F64)
    prob_sum = p.sum(0, dtype=F64)
    n = live.sum(dtype=F64)
    scale = COEF * E / (k * torch.clamp(n, min=1.0) ** 2)
    loss = scale * (counts * prob_sum).sum()
    # gates
    dg = torch.zeros((c["T"], E + 1), dtype=F32, device=DEV)
    dg.scatter_(1, torch.where(ids < 0, E, ids).long(), s["dgates"])
    dg = dg[:, :E]
    if c["renorm"]:
        g = p * hit
        g = g / torch.clamp(g.sum(1, keepdim=True), min=1e-30)
    else:
        g = p
    d = g * (dg - (g * dg).sum(1, keepdim=True))
    # balance
    cf = counts.float()
    d = d + (s["dloss"] * scale.float()) * p * (cf - (p * cf).sum(1, keepdim=True))
    d = torch.where(live, d, 0.0)
    return {"ids": ids, "gates": gates, "loss": loss.float().view(1), "counts": counts.to(torch.int32),
            "prob_sum": prob_sum.float(), "tokens": n.to(torch.int32).view(1), "dlogits": d.to(s["logits"].dtype)}


def _plain_weight(w, group):
    q, sc, z = w
    K = q.shape[-2]
    sc = sc.float().repeat_interleave(group, -2)[..., :K, :]
    z = 8.0 if z is None else z.float().repeat_interleave(group, -2)[..., :K, :]
    return (q.float() - z) * sc


def _plain_moe(c, s):
    ids, gates, _, _ = _plain_route(dict(c, renorm=True), s["logits"], None)
    x = s["x"].float()
    y = torch.zeros((c["T"], c["H"]), dtype=F32, device=DEV)
    for e in range(c["E"] // c["ep"]):
        h = x @ _plain_weight([v if v is None else v[e] for v in s["w1"]], c["group"])
        a = h[:, : c["I"]]
        a = a / (1.0 + torch.exp(-a)) * h[:, c["I"]:]
        g = (gates * (ids == e)).sum(1, keepdim=True)
        y += g * (a @ _plain_weight([v if v is None else v[e] for v in s["w2"]], c["group"]))
    return {"ids": ids, "gates": gates, "y": y.to(BF16)}


def _plain(s):
    c = s["case"]
    if c["op"] == "route":
        ids, gates, _, _ = _plain_route(c, s["logits"], s["mask"])
        return {"ids": ids, "gates": gates}
    if c["op"] == "train":
        return _plain_train(c, s)
    if c["op"] == "combine":
        t, j = s["where"][:, 0], s["where"][:, 1]
        real = t >= 0
        t, j = t.clamp(min=0), j.clamp(min=0)
        dy = s["dy"].float()[t]
        w = torch.where(real, s["gates"][t, j], 0.0)
        n = t.shape[0]
        dots = torch.where(real, (dy * s["ye"][:n].float()).sum(1), 0.0)
        dgates = torch.zeros((c["T"], c["k"]), dtype=F32, device=DEV)
        dgates.index_put_((t, j), dots, accumulate=True)
        s["dye"][:n] = w[:, None] * dy
        return {"dy_expert": s["dye"], "dgates": dgates}
    if c["op"] == "w4":
        return {"y": (s["x"].float() @ _plain_weight(s["w"], c["group"])).to(BF16)}
    return _plain_moe(c, s)


# ------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return _plain(s)
    c, ops = s["case"], s["ops"]
    if c["op"] == "route":
        ids, gates = ops.moe_route(s["logits"], c["k"], renorm=c["renorm"], token_mask=s["mask"])
        return {"ids": ids, "gates": gates}
    if c["op"] == "train":
        r = ops.moe_route_balance(s["logits"], c["k"], COEF, renorm=c["renorm"], token_mask=s["mask"])
        d = ops.moe_route_backward(s["logits"], r["ids"], dgates=s["dgates"], dloss=s["dloss"], counts=r["counts"],
                                   tokens=r["tokens"], coef=COEF, renorm=c["renorm"], token_mask=s["mask"])
        return {"ids": r["ids"], "gates": r["gates"], "loss": r["loss"], "counts": r["counts"],
                "prob_sum": r["prob_sum"], "tokens": r["tokens"], "dlogits": d}
    if c["op"] == "combine":
        t = s["t"]
        dy_expert, dgates = ops.moe_combine_backward(s["dy"], s["ye"], s["ids"], t["row_weight"], t["owner_offset"],
                                                     t["slot_to_row"], t["rb_rows"], 0, c["E"] // c["ep"],
                                                     dy_expert=s["dye"], sizes=t["sizes"])
        return {"dy_expert": dy_expert, "dgates": dgates}
    if c["op"] == "w4":
        return {"y": ops.gemm_w4(s["x"], s["packed"])}
    ids, gates = ops.moe_route(s["logits"], c["k"])
    t = ops.moe_build_indices_dev(ids, gates, 0, c["E"] // c["ep"], sync=False)
    ops.moe_ffn_combine_w4(s["x"], t["pull_indices"], t["row_weight"], t["owner_offset"], t["slot_to_row"], s["p1"],
                           s["p2"], s["act"], s["ye"], s["y"], t["rb_expert"], t["rb_rows"], sizes=t["sizes"])
    return {"ids": ids, "gates": gates, "y": s["y"]}


# ------------------------------------------------------------------- what it takes
def _expected(c):
    """(routed rows, local experts with a row, padded rows) to expect of a batch: an expert is among a
    token's top-k with probability 1 - exp(-x p_e)."""
    E, T = c["E"], c["T"]
    p = torch.softmax(_popularity(E), 0)
    lo, hi = 0.0, 1e6
    for _ in range(200):
        x = 0.5 * (lo + hi)
        lo, hi = (x, hi) if float((1 - torch.exp(-x * p)).sum()) < c["k"] else (lo, x)
    hit = (1 - torch.exp(-x * p))[: E // c["ep"]]
    rows = max(1.0, float(T * hit.sum()))
    used = max(1.0, float((1 - (1 - hit) ** T).sum()))
    return rows, used, sum(BLOCK * math.ceil(float(T * h) / BLOCK) for h in hit)


def work(case):
    c = case
    size = 2 if c.get("dtype") == "bf16" else 4
    if c["op"] in ("route", "train"):
        T, E, k = c["T"], c["E"], c["k"]
        read = T * E * size * (1 - c["masked"])
        b = read + T * k * 8 + (T if c["masked"] else 0)
        if c["op"] == "route":
            return {"bytes": b, "flops": 4 * T * E}
        return {"bytes": b + T * E * size + T * k * 4 + E * 8, "flops": 14 * T * E}
    if c["op"] == "combine":
        rows, _, padded = _expected(c)
        T, H = c["T"], c["H"]
        return {"bytes": min(T, rows) * H * size + rows * H * 2 + padded * H * 2 + T * c["k"] * 8,
                "flops": 3 * rows * H}

    def weights(K, N):
        groups = (K + c["group"] - 1) // c["group"]
        return K * N / 2 + groups * N * (3 if c.get("zeros") else 2)

    if c["op"] == "w4":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": weights(K, N) + 2 * M * (K + N), "flops": 2 * M * N * K}
    rows, used, _ = _expected(c)
    T, H, I = c["T"], c["H"], c["I"]
    return {"bytes": used * (weights(H, 2 * I) + weights(I, H)) + min(T, rows) * H * 2 + T * c["E"] * 4
            + T * c["k"] * 8 + T * H * 2, "flops": 6 * rows * H * I}


# ------------------------------------------------------------------- 64 bits
def _exact_choice(x, k):
    """The k largest of each row one after another, the lowest index among equals; -1 where only -inf is left."""
    T, E = x.shape
    left = x.clone()
    order = torch.arange(E, device=DEV)
    ids = torch.empty((T, k), dtype=torch.int64, device=DEV)
    for i in range(k):
        m = left.amax(1, keepdim=True)
        first = torch.where(left == m, order, E).amin(1)
        ids[:, i] = torch.where(m[:, 0] == -INF, -1, first)
        left.scatter_(1, first[:, None], -INF)
    return ids


def _softmax64(x):
    """Rows of -inf alone give zeros."""
    m = x.amax(1, keepdim=True)
    e = torch.where(m == -INF, 0.0, torch.exp(x - torch.where(m == -INF, 0.0, m)))
    return torch.nan_to_num(e / e.sum(1, keepdim=True), nan=0.0)


def _exact_route(c, seed):
    logits, mask = _logits(c, seed)
    x = logits.to(F64)
    if mask is not None:
        x[~mask] = -INF
    ids = _exact_choice(x, c["k"])
    p = _softmax64(x)
    got = ids >= 0
    pc = torch.where(got, p.gather(1, ids.clamp(min=0)), 0.0)
    gates = torch.nan_to_num(pc / pc.sum(1, keepdim=True), nan=0.0) if c["renorm"] else pc
    return ids, gates, p, got


def _weight64(w, e, group):
    q, sc, z = [v if v is None or e is None else v[e] for v in w]
    at = torch.arange(q.shape[0], device=DEV) // group
    return (q.to(F64) - (8 if z is None else z[at].to(F64))) * sc[at].to(F64)


def exact(case, seed):
    c = case
    if c["op"] == "route":
        ids, gates, _, _ = _exact_route(c, seed)
        return {"ids": ids.to(torch.int32), "gates": gates}
    if c["op"] == "train":
        T, E, k = c["T"], c["E"], c["k"]
        ids, gates, p, got = _exact_route(c, seed)
        dg = torch.where(got, _randn((T, k), seed, 5, 0.1 / T, F32).to(F64), 0.0)
        counts = torch.bincount(ids[got], minlength=E)
        n = int(got[:, 0].sum())
        scale = COEF * E / (k * max(n, 1) ** 2)
        f = counts.to(F64)
        total = p.sum(0)
        d = scale * p * (f[None] - (p @ f)[:, None])
        dot = (gates * dg).sum(1, keepdim=True)
        if c["renorm"]:
            d.scatter_add_(1, ids.clamp(min=0), torch.where(got, gates * (dg - dot), 0.0))
        else:
            d -= p * dot
            d.scatter_add_(1, ids.clamp(min=0), torch.where(got, gates * dg, 0.0))
        return {"ids": ids.to(torch.int32), "gates": gates, "loss": (scale * (f * total).sum()).view(1),
                "counts": counts.to(torch.int32), "prob_sum": total,
                "tokens": torch.full((1,), n, dtype=torch.int32, device=DEV), "dlogits": d}
    if c["op"] == "combine":
        dt = F32 if c["dtype"] == "f32" else BF16
        dy = _randn((c["T"], c["H"]), seed, 1, 1.0 / c["T"], dt)
        ids, gates = _choice(c, seed)
        rows = _expert_rows(c, ids)
        ye = _randn((rows.shape[0], c["H"]), seed, 2, 1.0)
        dye = torch.zeros((_capacity(c), c["H"]), dtype=F64, device=DEV)
        dgates = torch.zeros((c["T"], c["k"]), dtype=F64, device=DEV)
        r = (rows[:, 0] >= 0).nonzero()[:, 0]
        t, j = rows[r, 0], rows[r, 1]
        dye[r] = gates[t, j].to(F64)[:, None] * dy[t].to(F64)
        dgates[t, j] = (dy[t].to(F64) * ye[r].to(F64)).sum(1)
        return {"dy_expert": dye, "dgates": dgates}
    if c["op"] == "w4":
        x = _randn((c["M"], c["K"]), seed, 1, 1.0)
        w = _codes((c["K"], c["N"]), c["group"], seed, 10, c["zeros"])
        return {"y": x.to(F64) @ _weight64(w, None, c["group"])}
    ids, gates, _, _ = _exact_route(dict(c, renorm=True), seed)
    n_local, H, I = c["E"] // c["ep"], c["H"], c["I"]
    x = _randn((c["T"], H), seed, 1, 1.0).to(F64)
    w1 = _codes((n_local, H, 2 * I), c["group"], seed, 10)
    w2 = _codes((n_local, I, H), c["group"], seed, 20)
    y = torch.zeros((c["T"], H), dtype=F64, device=DEV)
    for e in range(n_local):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            h = x[t] @ _weight64(w1, e, c["group"])
            a = h[:, :I] * torch.sigmoid(h[:, :I]) * h[:, I:]
            y.index_add_(0, t, (a @ _weight64(w2, e, c["group"])) * gates[t, j][:, None])
    return {"ids": ids.to(torch.int32), "gates": gates, "y": y}
