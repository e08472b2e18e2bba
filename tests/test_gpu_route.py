"""The router (choices, gates, counts, balance loss), its gradient and the
combine's gradient, against plain 64-bit forms.

Tolerances (u = 2^-24, half an fp32 step): an exponential of x - max carries
1.3 |x - max| u from the rounding of its exponent and of the constant in it, at
most 37 u here (logits within 28 of the maximum), 2 u of its own; a sum of at
most 1024 positive terms, 16 per lane and 6 steps across, 22 u; quotient 1 u:
below 64 u = 2^-18 for a probability and for a gate.  A gradient adds at most as much once more per
product and sum, relative to the sum of its terms' magnitudes: 2^-17.  Sums
over tokens add their own roundings, at most (T / 4096 + 8) u in a lane."""
import numpy as np
import pytest
import torch

from mkernel_amd import capi, ops, workloads as wl

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
D = torch.float64


def _say(*a):
    print("[case]", *a, flush=True)


def _logits(T, E, dtype, seed, spread=4.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn((T, E + pad), generator=g).mul_(spread).clamp_(-14, 14).to(dtype)
    return wide


def _choose(x, k):
    """The k largest, ties to the lowest index, NaN largest; -1 where only -inf is left.  numpy, on the host."""
    x = x.double().numpy()
    key = np.where(np.isnan(x), np.inf, x)
    ids = np.full((x.shape[0], k), -1, dtype=np.int64)
    for t in range(x.shape[0]):
        order = sorted(range(x.shape[1]), key=lambda e: (not np.isnan(x[t, e]), -key[t, e], e))
        n = 0
        for e in order[:k]:
            if x[t, e] != -np.inf:
                ids[t, n] = e
                n += 1
    return torch.from_numpy(ids)


def _softmax(x):
    m = x.amax(1, keepdim=True)
    e = torch.where(x == -INF, torch.zeros_like(x), torch.exp(x - torch.where(m == -INF, torch.zeros_like(m), m)))
    return e / torch.where(m == -INF, torch.ones_like(m), e.sum(1, keepdim=True))


def _reference(x, k, renorm, mask, coef):
    """ids, gates, p, counts, n, loss in 64 bits."""
    x = x.to(D).clone()
    if mask is not None:
        x[~mask.bool()] = -INF
    ids = _choose(x, k)
    p = _softmax(x)
    on = ids >= 0
    g = torch.where(on, p.gather(1, ids.clamp(min=0)), torch.zeros(1, dtype=D))
    if renorm:
        g = torch.where(on, g / torch.where(on.any(1, keepdim=True), g.sum(1, keepdim=True), torch.ones(1, dtype=D)), g)
    E = x.shape[1]
    counts = torch.bincount(ids[on], minlength=E)
    n = int(on.any(1).sum())
    loss = coef * E / (k * max(n, 1) ** 2) * (counts.to(D) * p.sum(0)).sum()
    return ids, g, p, counts, n, loss


SIZES = [(1, 1, 1, 0), (1, 256, 8, 0), (3, 7, 7, 0), (5, 64, 6, 192), (64, 256, 8, 0), (17, 65, 1, 3), (130, 128, 32, 0),
         (129, 60, 4, 5), (33, 255, 9, 1), (40, 257, 16, 7), (20, 512, 10, 0), (9, 1000, 32, 24), (7, 1024, 8, 0),
         (1027, 16, 2, 0), (4099, 32, 4, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k,pad", SIZES)
def test_route_and_balance(dev, T, E, k, pad, renorm, dtype):
    _say("route", T, E, k, pad, renorm, dtype)
    wide = _logits(T, E, dtype, 3 * T + E, pad=pad)
    x = wide[:, :E]
    g = torch.Generator().manual_seed(1)
    for mask in (None, torch.rand(T, generator=g) < 0.7):
        if mask is not None:
            x = x.clone()
            x[~mask] = NAN
        ids, gates, p, counts, n, loss = _reference(x, k, renorm, mask, 0.25)
        d = wide.to(dev)[:, :E] if mask is None else torch.cat([x, x[:, :pad]], 1).to(dev)[:, :E]
        dm = None if mask is None else mask.to(dev)
        got = ops.moe_route(d, k, renorm=renorm, token_mask=dm)
        r = ops.moe_route_balance(d, k, 0.25, renorm=renorm, token_mask=None if dm is None else dm.to(torch.uint8))
        torch.cuda.synchronize()
        assert torch.equal(got[0].cpu().long(), ids)
        assert torch.allclose(got[1].cpu().to(D), gates, rtol=2 ** -18, atol=1e-37)
        assert torch.equal(r["ids"], got[0]) and torch.equal(r["gates"], got[1])
        assert torch.equal(r["counts"].cpu().long(), counts) and int(r["tokens"]) == n
        rtol = 2 ** -18 + (T / 4096 + 8) * 2 ** -24
        assert torch.allclose(r["prob_sum"].cpu().to(D), p.sum(0), rtol=rtol, atol=1e-37)
        assert abs(float(r["loss"]) - float(loss)) <= rtol * float(loss)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k", [(70001, 24, 3), (9001, 250, 8), (40000, 700, 2)])
def test_long_batches(dev, T, E, k, dtype):
    """Several tokens per wave, and as many workgroups as there may be."""
    _say("long", T, E, k, dtype)
    g = torch.Generator(device=dev).manual_seed(T)
    x = torch.randn((T, E), generator=g, device=dev).mul_(3).clamp_(-14, 14).to(dtype)
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    p = torch.softmax(x.to(D), 1)
    r = ops.moe_route_balance(x, k, 0.5)
    assert torch.equal(r["ids"].long(), ids[:, :k])
    assert torch.allclose(r["gates"].to(D), torch.softmax(top[:, :k].to(D), 1), rtol=2 ** -18, atol=0)
    counts = torch.bincount(ids[:, :k].reshape(-1), minlength=E)
    rtol = 2 ** -18 + (T / 4096 + 8) * 2 ** -24
    assert torch.equal(r["counts"].long(), counts) and int(r["tokens"]) == T
    assert torch.allclose(r["prob_sum"].to(D), p.sum(0), rtol=rtol, atol=0)
    loss = 0.5 * E / (k * T * T) * (counts.to(D) * p.sum(0)).sum()
    assert abs(float(r["loss"]) - float(loss)) <= rtol * float(loss)
    again = ops.moe_route_balance(x, k, 0.5)
    assert all(torch.equal(r[f], again[f]) for f in r)
    dg = torch.randn((T, k), generator=g, device=dev)
    d = ops.moe_route_backward(x, r["ids"], dgates=dg, counts=r["counts"], tokens=r["tokens"], coef=0.5)
    want, mag = _gradient(x.to(D).cpu(), ids[:, :k].cpu(), dg.cpu(), counts.cpu(), T, 0.5, 1.0, True)
    tol = 2 ** -17 * mag + 1e-37 + (2 ** -8 * want.abs() if dtype is torch.bfloat16 else 0)
    assert bool(((d.cpu().to(D) - want).abs() <= tol).all())


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_common_offsets(dev, dtype, renorm):
    """Logits around one far value per token, of both signs up to the type's largest: a softmax does not see it, and a
    token's results are the same bits whatever its neighbours are."""
    _say("offsets", dtype, renorm)
    E, k = 40, 6
    g = torch.Generator().manual_seed(12)
    offsets = [0.0, 3.0, -100.0, 1e3, -3e3, 1e5, -9e5, 1.1e6, -1e7, 1e8, 1e9, -1e12, 1e20, -1e30, 3e38, -3e38]
    x = torch.stack([(torch.randn(E, generator=g).clamp_(-3, 3) + o) for o in offsets]).to(dtype)
    x[::3, 5:9] = x[::3].amax(1, keepdim=True)
    x[3::4, 11] = -INF
    x[5::4, 12] = torch.finfo(dtype).min
    ids, want, p, counts, n, loss = _reference(x, k, renorm, None, 0.25)
    r = ops.moe_route_balance(x.to(dev), k, 0.25, renorm=renorm)
    assert torch.equal(r["ids"].cpu().long(), ids)
    # as in the docstring above, for |x - max| below 42 and with a second rounding of the exponent where the difference is
    # taken first: 2.3 x 42 u + 25 u
    got = r["gates"].cpu().to(D)
    near = want > 1e-18
    assert bool(((got - want).abs() <= 2 ** -17 * want)[near].all()) and bool((got[~near] <= 2e-18).all())
    assert bool(((r["prob_sum"].cpu().to(D) - p.sum(0)).abs() <= 2 ** -17 * p.sum(0) + 1e-16).all())
    dg = torch.randn((len(offsets), k), generator=g)
    kw = dict(coef=0.25, counts=r["counts"], tokens=r["tokens"], renorm=renorm)
    d = ops.moe_route_backward(x.to(dev), r["ids"], dgates=dg.to(dev), **kw)
    ref, mag = _gradient(x.to(D), ids, dg, counts, n, 0.25, 1.0, renorm)
    # a gate twice in a product, 122 u each, and 10 u of sums and products; gates below 1e-18 times gradients below 10
    tol = 2 ** -16 * mag + 1e-16 + (2 ** -8 * ref.abs() if dtype is torch.bfloat16 else 0)
    assert bool(((d.cpu().to(D) - ref).abs() <= tol).all())
    for t in range(len(offsets)):
        i, gate = ops.moe_route(x[t:t + 1].to(dev), k, renorm=renorm)
        assert torch.equal(i, r["ids"][t:t + 1]) and torch.equal(gate, r["gates"][t:t + 1])
        one = ops.moe_route_backward(x[t:t + 1].to(dev), i, dgates=dg[t:t + 1].to(dev), **kw)
        assert torch.equal(one, d[t:t + 1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_columns_of_a_wider_matrix(dev, dtype):
    """Logits, and their gradient, at column offsets and row strides of every alignment: nothing beside them is read or
    written. Sums over a token's experts go in another order where they are loaded in other pieces."""
    _say("columns", dtype)
    T, E, k = 37, 60, 4
    x = _logits(T, E, dtype, 4).to(dev)
    dg = torch.randn((T, k), generator=torch.Generator().manual_seed(3)).to(dev)
    r = ops.moe_route_balance(x, k, 0.5)
    kw = dict(dgates=dg, counts=r["counts"], tokens=r["tokens"], coef=0.5)
    want, mag = _gradient(x.to(D).cpu(), r["ids"].cpu().long(), dg.cpu(), r["counts"].cpu(), T, 0.5, 1.0, True)
    tol = 2 ** -17 * mag + 1e-37 + (2 ** -8 * want.abs() if dtype is torch.bfloat16 else 0)
    for first, width in ((0, 64), (1, 61), (2, 66), (4, 64), (3, 68), (4, 71), (8, 128)):
        wide = torch.full((T, width + first), float("nan"), dtype=dtype, device=dev)
        wide[:, first:first + E] = x
        view = wide[:, first:first + E]
        q = ops.moe_route_balance(view, k, 0.5)
        assert torch.equal(q["ids"], r["ids"]) and torch.equal(q["counts"], r["counts"])
        assert torch.allclose(q["gates"], r["gates"], rtol=2 ** -17, atol=0)  # 2^-18 each
        out = torch.full((T, width + first), 7.0, dtype=dtype, device=dev)
        got = ops.moe_route_backward(view, r["ids"], **kw, out=out[:, first:first + E])
        assert bool(((got.cpu().to(D) - want).abs() <= tol).all())
        out[:, first:first + E] = 7
        assert bool((out == 7).all())


def test_training_step(dev):
    """Router, index build, combine and their gradients together, as the router of a training step runs them, against
    64-bit automatic differentiation of sum(y G) + loss with the expert rows and the counts as constants."""
    _say("training step")
    T, E, k, H, e0, n_local, coef = 50, 24, 4, 64, 8, 12, 0.3
    logits = _logits(T, E, torch.float32, 6, spread=1.5)
    G = torch.randn((T, H), generator=torch.Generator().manual_seed(7)) * 0.1
    for renorm in (True, False):
        x = logits.to(dev)
        r = ops.moe_route_balance(x, k, coef, renorm=renorm)
        t = ops.moe_build_indices_dev(r["ids"], r["gates"], e0, n_local)
        ye = wl.randn_bf16((t["R_pad"], H), 8).to(dev)
        y = torch.empty((T, H), device=dev)
        ops.moe_combine(ye, t["row_weight"], t["owner_offset"], t["slot_to_row"], y)
        dye, dg = ops.moe_combine_backward(G.to(dev), ye, r["ids"], t["row_weight"], t["owner_offset"], t["slot_to_row"],
                                           t["rb_rows"], e0, n_local)
        d = ops.moe_route_backward(x, r["ids"], dgates=dg, counts=r["counts"], tokens=r["tokens"], coef=coef,
                                   renorm=renorm)
        # the same on the host
        z = logits.to(D).requires_grad_()
        ids = r["ids"].cpu().long()
        p = torch.softmax(z, 1)
        g = p.gather(1, ids)
        if renorm:
            g = g / g.sum(1, keepdim=True)
        rows = torch.zeros((T, k, H), dtype=D)
        at, row = {}, 0
        for e in range(n_local):
            mine = (ids == e0 + e).nonzero().tolist()
            at.update({(tt, j): row + i for i, (tt, j) in enumerate(mine)})
            row += (len(mine) + 127) // 128 * 128
        for (tt, j), i in at.items():
            rows[tt, j] = ye[i].cpu().to(D)
        rows.requires_grad_()
        out = (g[..., None] * rows).sum(1)
        f = torch.bincount(ids.reshape(-1), minlength=E).to(D)
        loss = coef * E / (k * T * T) * (f * p.sum(0)).sum()
        ((out * G.to(D)).sum() + loss).backward()
        # y: gates (2^-18, below 1 in sum), k products and sums. dlogits: 2^-17 of the terms g dg and g sum(g dg), each
        # at most the largest sum over the columns of |G y|, which also bounds the error of dg itself (64 sums of fp32
        # in pieces: below 2^-20 of it), and of the balance term, below 1
        assert torch.allclose(y.cpu().to(D), out.detach(), rtol=0, atol=2 ** -17 * float(rows.detach().abs().max()))
        most = float((rows.detach().abs() * G.to(D).abs()[:, None]).sum(2).max())
        assert abs(float(r["loss"]) - float(loss.detach())) <= 2 ** -17 * float(loss.detach())
        assert torch.allclose(d.cpu().to(D), z.grad, rtol=0, atol=2 ** -17 * (2 * most + 1))
        got = dye.cpu().to(D)
        for (tt, j), i in at.items():
            want = rows.grad[tt, j]
            # the gate's own rounding, 2^-18, and one of bf16
            assert bool(((got[i] - want).abs() <= (2 ** -8 + 2 ** -17) * want.abs()).all())
        rest = torch.ones(t["R_pad"], dtype=torch.bool)
        rest[list(at.values())] = False
        assert not got[rest].any()


@pytest.mark.parametrize("T", [0, 1])
def test_no_tokens(dev, T):
    """Nothing to route, or nothing that counts: no choice, sums and loss zero, no division by zero."""
    _say("no tokens", T)
    x = torch.full((T, 40), NAN, device=dev)
    mask = torch.zeros(T, dtype=torch.bool, device=dev)
    r = ops.moe_route_balance(x, 4, 1.0, token_mask=mask)
    assert r["ids"].shape == (T, 4) and bool((r["ids"] == -1).all()) and bool((r["gates"] == 0).all())
    assert not r["counts"].any() and not r["prob_sum"].any() and int(r["tokens"]) == 0 and float(r["loss"]) == 0
    d = ops.moe_route_backward(x, r["ids"], dgates=torch.ones((T, 4), device=dev), counts=r["counts"],
                               tokens=r["tokens"], coef=1.0, token_mask=mask)
    assert d.shape == (T, 40) and not d.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [6, 100, 300, 700])
def test_ties_signs_and_masked_experts(dev, E, dtype):
    """Equal logits go to the lowest expert (-0 equals 0); -inf is never chosen; a row of -inf alone
    does not count; the type's lowest value can be chosen; NaN ranks first and spreads over its row only."""
    _say("ties", E, dtype)
    k, low = 5, torch.finfo(dtype).min
    rows = [torch.zeros(E), torch.where(torch.arange(E) % 2 == 0, -0.0, 0.0), torch.full((E,), -INF),
            torch.full((E,), low), torch.full((E,), -INF), torch.arange(E).float() % 3, torch.full((E,), low),
            torch.full((E,), 2.0), torch.linspace(-1, 1, E), torch.linspace(1, -1, E)]
    rows[4][E - 2] = 1.5                       # one expert left
    rows[6][E // 2] = torch.finfo(dtype).max   # the difference to the others overflows
    rows[8][E - 3] = NAN
    rows[9][1] = INF
    x = torch.stack(rows).to(dtype)
    want = _choose(x, k)
    ids, gates = ops.moe_route(x.to(dev), k)
    r = ops.moe_route_balance(x[:8].to(dev), k, 1.0)
    full = ops.moe_route(x.to(dev), k, renorm=False)[1].cpu()
    ids, gates = ids.cpu().long(), gates.cpu()
    assert torch.equal(ids, want)
    assert ids[1].tolist() == list(range(5)) and ids[2].tolist() == [-1] * 5 and ids[4].tolist() == [E - 2] + [-1] * 4
    assert ids[8, 0] == E - 3 and ids[9, 0] == 1
    for g in (gates, full):
        assert torch.isfinite(g[:8]).all() and torch.isnan(g[8:]).all()
        assert not g[2].any() and g[4].tolist() == [1, 0, 0, 0, 0] and g[6].tolist() == [1, 0, 0, 0, 0]
    assert torch.allclose(gates[0].to(D), torch.full((5,), 0.2, dtype=D), rtol=2 ** -18, atol=0)
    assert torch.allclose(full[0].to(D), torch.full((5,), 1 / E, dtype=D), rtol=2 ** -18, atol=0)
    assert int(r["tokens"]) == 7 and int(r["counts"].sum()) == 6 * 5 + 1
    assert abs(float(r["prob_sum"].sum().double()) - 7) < 7 * 2 ** -17
    # the gradient of the same rows: finite, zero where nothing may flow, NaN in the NaN rows only
    d = ops.moe_route_backward(x.to(dev), ids.int().to(dev), dgates=torch.ones_like(gates).to(dev), counts=r["counts"],
                               tokens=r["tokens"], coef=1.0).float().cpu()
    assert torch.isfinite(d[:8]).all() and not d[2].any() and d[4][E - 2] == 0 and torch.isnan(d[8:]).all()


def _gradient(x, ids, dg, counts, n, coef, dloss, renorm):
    """The formula in 64 bits, and the sum of its terms' magnitudes."""
    p = _softmax(x)
    T, E = x.shape
    k = ids.shape[1]
    on = (ids >= 0) & (ids < E)
    at = ids.clamp(0, E - 1)
    zero = torch.zeros(1, dtype=D)
    dg = torch.where(on, dg.to(D), zero)
    d, mag = torch.zeros_like(x), torch.zeros_like(x)
    if renorm:
        xc = torch.where(on, x.gather(1, at), torch.full((1,), -INF, dtype=D))
        g = _softmax(xc)
        d.scatter_add_(1, at, torch.where(on, g * (dg - (g * dg).sum(1, keepdim=True)), zero))
        mag.scatter_add_(1, at, torch.where(on, g * (dg.abs() + (g * dg.abs()).sum(1, keepdim=True)), zero))
    else:
        g = torch.where(on, p.gather(1, at), zero)
        d -= p * (g * dg).sum(1, keepdim=True)
        mag += p * (g * dg.abs()).sum(1, keepdim=True)
        d.scatter_add_(1, at, torch.where(on, g * dg, zero))
        mag.scatter_add_(1, at, torch.where(on, g * dg.abs(), zero))
    if counts is not None and n:
        c = dloss * coef * E / (k * n * n)
        f = counts.to(D)
        s = (p * f).sum(1, keepdim=True)
        d += c * p * (f - s)
        mag += abs(c) * p * (f + s)
    return d, mag


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k,pad", SIZES)
def test_route_backward(dev, T, E, k, pad, renorm, dtype):
    _say("route backward", T, E, k, pad, renorm, dtype)
    wide = _logits(T, E, dtype, T + 7 * E, pad=pad)
    g = torch.Generator().manual_seed(2)
    mask = torch.rand(T, generator=g) < 0.8
    x = wide[:, :E].clone()
    if E > 4:
        x[:, 2] = -INF
    ids = _reference(x, k, renorm, mask, 1.0)[0]
    dg = torch.randn((T, k), generator=g)
    dg[ids < 0] = NAN  # nobody's gradient
    counts = torch.bincount(ids[ids >= 0], minlength=E) * 3  # as summed over three ranks
    n = 3 * int(mask.sum())
    to = lambda t: t.to(dev)
    whole = torch.cat([x, wide[:, E:]], 1).to(dev)
    xd, tokens = whole[:, :E], torch.tensor([n], dtype=torch.int32, device=dev)
    common = dict(renorm=renorm, token_mask=to(mask))
    both = dict(dgates=to(dg), counts=to(counts.int()), tokens=tokens, coef=0.5, dloss=torch.tensor([-1.5], device=dev))
    for parts in (both, {"dgates": both["dgates"]}, {k_: v for k_, v in both.items() if k_ != "dgates"}):
        got = ops.moe_route_backward(xd, to(ids.int()), **common, **parts)
        torch.cuda.synchronize()
        assert got.dtype == dtype and got.shape == (T, E)
        gates = dg if "dgates" in parts else torch.zeros_like(dg)
        want, mag = _gradient(x.to(D), ids, gates, counts if "counts" in parts else None, n, 0.5, -1.5, renorm)
        want[~mask], mag[~mask] = 0, 0
        tol = 2 ** -17 * mag + 1e-37 + (2 ** -8 * want.abs() if dtype is torch.bfloat16 else 0)
        assert bool(((got.cpu().to(D) - want).abs() <= tol).all())
    # in place, leaving the columns behind the experts alone
    behind = whole[:, E:].clone()
    first = ops.moe_route_backward(xd, to(ids.int()), **common, **both)
    out = ops.moe_route_backward(xd, to(ids.int()), **common, **both, out=xd)
    assert out.data_ptr() == xd.data_ptr() and torch.equal(out, first) and torch.equal(whole[:, E:], behind)


def test_backward_against_differences(dev):
    """The gradient of sum(gates * w) + loss by central differences of the 64-bit formula, with the counts held."""
    _say("differences")
    T, E, k = 6, 24, 4
    x = _logits(T, E, torch.float32, 5, spread=1.5).to(D)
    w = torch.randn((T, k), generator=torch.Generator().manual_seed(8))
    for renorm in (True, False):
        ids, _, _, counts, n, _ = _reference(x, k, renorm, None, 0.7)

        def value(y):
            p = _softmax(y)
            g = p.gather(1, ids)
            if renorm:
                g = g / g.sum(1, keepdim=True)
            return float((g * w.to(D)).sum() + 0.7 * E / (k * n * n) * (counts.to(D) * p.sum(0)).sum())

        got = ops.moe_route_backward(x.float().to(dev), ids.int().to(dev), dgates=w.to(dev), counts=counts.int().to(dev),
                                     tokens=torch.tensor([n], dtype=torch.int32, device=dev), coef=0.7, renorm=renorm)
        h = 1e-4
        for t in range(T):
            for e in range(E):
                a, b = x.clone(), x.clone()
                a[t, e] += h
                b[t, e] -= h
                # h^2 / 6 times a third derivative of a few units, and 2^-17 of magnitudes below 4
                assert abs(float(got[t, e]) - (value(a) - value(b)) / (2 * h)) < 1e-7 + 2 ** -15


def test_backward_odd_choices(dev):
    """Choices that the forward pass would not make: out of range (no gradient, nothing read or written there), the
    same expert twice (both count), experts at -inf, all of them left out."""
    _say("odd choices")
    E = 10
    x = _logits(5, E, torch.float32, 9)
    x[3, 4] = -INF
    ids = torch.tensor([[3, 3, 7], [1 << 30, -5, 2], [E, E, -1], [4, 4, 4], [0, 9, 0]])
    dg = torch.tensor([[1.0, 2.0, 3.0], [9.0, 9.0, 4.0], [5.0, 6.0, 7.0], [1.0, 1.0, 2.0], [1.0, -2.0, 0.5]])
    for renorm in (True, False):
        got = ops.moe_route_backward(x.to(dev), ids.int().to(dev), dgates=dg.to(dev), renorm=renorm).cpu().to(D)
        want, mag = _gradient(x.to(D), ids, dg, None, 0, 0, 0, renorm)
        want = torch.nan_to_num(want)
        assert bool(((got - want).abs() <= 2 ** -17 * torch.nan_to_num(mag) + 1e-37).all())


def _combine_case(dev, T, H, E, e0, n_local, k, dtype, seed, same=False):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else np.zeros((0, k), np.int32)
    if same:
        ids[:] = ids[:, :1]  # one expert k times
    gates = rng.random((T, k), dtype=np.float32)
    ids, gates = torch.from_numpy(ids), torch.from_numpy(gates)
    dy = torch.randn((T, H), generator=torch.Generator().manual_seed(seed)).to(dtype)
    return ids, gates, dy


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,E,e0,n_local,k,same", [
    (1, 8, 4, 0, 4, 2, False), (7, 2056, 40, 8, 16, 8, False), (300, 1032, 12, 0, 12, 3, False), (64, 7168, 256, 32, 32, 8, False),
    (5, 512, 40, 0, 40, 32, False), (9, 264, 6, 0, 6, 4, True), (50, 128, 64, 60, 4, 2, False)])
def test_combine_backward(dev, T, H, E, e0, n_local, k, same, dtype):
    _say("combine backward", T, H, E, e0, n_local, k, same, dtype)
    ids, gates, dy = _combine_case(dev, T, H, E, e0, n_local, k, dtype, T + H, same)
    idd, gd, dyd = ids.to(dev), gates.to(dev), dy.to(dev)
    t = ops.moe_build_indices_dev(idd, gd, e0, n_local)
    pull, w = t["pull_indices"].cpu(), t["row_weight"].cpu()
    ye = wl.randn_bf16((t["R_pad"], H), 5)
    a, dg = ops.moe_combine_backward(dyd, ye.to(dev), idd, t["row_weight"], t["owner_offset"], t["slot_to_row"],
                                     t["rb_rows"], e0, n_local)
    # a capacity, the row count on the device; rows behind it stay
    c = ops.moe_build_indices_dev(idd, gd, e0, n_local, sync=False)
    cap = c["pull_indices"].shape[0]
    yc = torch.zeros((cap, H), dtype=torch.bfloat16, device=dev)
    yc[:t["R_pad"]] = ye.to(dev)
    keep = torch.full((cap, H), 7.0, dtype=torch.bfloat16, device=dev)
    b, dg2 = ops.moe_combine_backward(dyd, yc, idd, c["row_weight"], c["owner_offset"], c["slot_to_row"], c["rb_rows"],
                                      e0, n_local, dy_expert=keep, sizes=c["sizes"])
    torch.cuda.synchronize()
    assert torch.equal(b[:t["R_pad"]], a) and bool((b[t["R_pad"]:] == 7).all()) and torch.equal(dg, dg2)
    # dy_expert: one fp32 product, one rounding: the same bits
    tok = pull[:, 2].clamp(min=0).long()
    want = torch.where((pull[:, 0] >= 0)[:, None], w[:, None] * dy.float()[tok], torch.zeros(1)).to(torch.bfloat16)
    assert torch.equal(a.cpu(), want)
    # dgates by the order of the rows of each expert
    ref, mag = torch.zeros((T, k), dtype=D), torch.zeros((T, k), dtype=D)
    row = 0
    for e in range(n_local):
        at = (ids == e0 + e).nonzero()
        for i, (tt, j) in enumerate(at.tolist()):
            v = dy[tt].to(D) * ye[row + i].to(D)
            ref[tt, j], mag[tt, j] = v.sum(), v.abs().sum()
        row += (at.shape[0] + 127) // 128 * 128
    # a lane's chain of at most H / 32 + 8 products and sums (each rounded), and 12 sums across
    assert bool(((dg.cpu().to(D) - ref).abs() <= (2 * (H / 32 + 8) + 12) * 2 ** -24 * mag).all())
    local = (ids >= e0) & (ids < e0 + n_local)
    assert not dg.cpu()[~local].any()


def test_combine_backward_in_place(dev):
    """dy_expert over y_expert, gates' gradient alone, tables with nonsense behind the routed rows, rows beyond the
    capacity of the given buffers, and two calls captured and replayed beside eager ones."""
    _say("combine backward in place")
    T, H, E, e0, n_local, k = 90, 520, 24, 4, 9, 5
    ids, gates, dy = _combine_case(dev, T, H, E, e0, n_local, k, torch.float32, 3, False)
    idd, gd, dyd = ids.to(dev), gates.to(dev), dy.to(dev)
    t = ops.moe_build_indices_dev(idd, gd, e0, n_local)
    tables = [t[n] for n in ("row_weight", "owner_offset", "slot_to_row", "rb_rows")]
    R = t["R_pad"]
    ye = wl.randn_bf16((R, H), 5).to(dev)
    a, dg = ops.moe_combine_backward(dyd, ye, idd, *tables, e0, n_local)
    over = ye.clone()
    b, dg2 = ops.moe_combine_backward(dyd, over, idd, *tables, e0, n_local, dy_expert=over)
    assert b.data_ptr() == over.data_ptr() and torch.equal(a, b) and torch.equal(dg, dg2)
    # a capacity whose tables hold nonsense where no row is
    c = ops.moe_build_indices_dev(idd, gd, e0, n_local, sync=False)
    cap = c["pull_indices"].shape[0]
    c["row_weight"][R:] = NAN
    c["rb_rows"][R // 128:] = -(1 << 30)
    c["slot_to_row"][int(c["sizes"][0]):] = 1 << 30
    wide = torch.full((cap, H), NAN, dtype=torch.bfloat16, device=dev)
    wide[:R] = ye
    keep = torch.full((cap, H), 7.0, dtype=torch.bfloat16, device=dev)
    tables_c = [c[n] for n in ("row_weight", "owner_offset", "slot_to_row", "rb_rows")]
    kw = dict(dy_expert=keep, sizes=c["sizes"])
    b, dg2 = ops.moe_combine_backward(dyd, wide, idd, *tables_c, e0, n_local, **kw)
    assert torch.equal(b[:R], a) and bool((b[R:] == 7).all()) and torch.equal(dg, dg2)
    # fewer rows than were routed: those behind them have no gradient and are not reached
    half = R // 256 * 128
    b, dg2 = ops.moe_combine_backward(dyd, ye[:half], idd, *tables, e0, n_local)
    assert torch.equal(b, a[:half])
    rows = torch.full((T, k), -1, dtype=torch.long)
    row = 0
    for e in range(n_local):
        at = (ids == e0 + e).nonzero()
        rows[at[:, 0], at[:, 1]] = row + torch.arange(at.shape[0])
        row += (at.shape[0] + 127) // 128 * 128
    assert torch.equal(dg2, torch.where((rows < half).to(dev), dg, torch.zeros(1, device=dev)))
    # captured
    graph, d = torch.cuda.CUDAGraph(), dyd.clone()
    with torch.cuda.graph(graph):
        one = ops.moe_combine_backward(d, ye, idd, *tables, e0, n_local)
        two = ops.moe_combine_backward(d.bfloat16(), ye, idd, *tables, e0, n_local)
    for rep in range(3):
        d.copy_(dyd if rep != 1 else 2 * dyd)
        graph.replay()
        torch.cuda.synchronize()
        want = [ops.moe_combine_backward(x, ye, idd, *tables, e0, n_local) for x in (d, d.bfloat16())]
        assert all(torch.equal(u, v) for i, j in zip((one, two), want) for u, v in zip(i, j)), rep


def test_gates_gradient_alone(dev):
    """The C entry without dy_expert and rb_rows: the same gates' gradient."""
    _say("combine backward, gates alone")
    T, H, E, e0, n_local, k = 33, 264, 10, 2, 5, 3
    ids, gates, dy = _combine_case(dev, T, H, E, e0, n_local, k, torch.bfloat16, 9, False)
    idd, dyd = ids.to(dev), dy.to(dev)
    t = ops.moe_build_indices_dev(idd, gates.to(dev), e0, n_local)
    ye = wl.randn_bf16((t["R_pad"], H), 5).to(dev)
    _, dg = ops.moe_combine_backward(dyd, ye, idd, t["row_weight"], t["owner_offset"], t["slot_to_row"], t["rb_rows"], e0,
                                     n_local)
    alone = torch.full((T, k), 7.0, device=dev)
    capi.call_values("mk_moe_combine_backward", capi.MoeCombineBackwardArgs, ops._stream(), dyd.data_ptr(), ye.data_ptr(),
                     idd.data_ptr(), t["row_weight"].data_ptr(), t["owner_offset"].data_ptr(),
                     t["slot_to_row"].data_ptr(), 0, 0, alone.data_ptr(), T, H, t["R_pad"], k, e0, n_local, 1, 0)
    assert torch.equal(alone, dg)


def test_past_32_bits(dev):
    """Logits and expert rows more than 2^31 elements into their buffers."""
    _say("offsets past 32 bits")
    T, E, k, ld = 60000, 40, 4, 40000
    assert (T - 1) * ld > 2**31
    wide = torch.empty((T, ld), dtype=torch.bfloat16, device=dev)
    x = _logits(T, E, torch.bfloat16, 3).to(dev)
    wide[:, 8:8 + E] = x
    view = wide[:, 8:8 + E]
    a, b = ops.moe_route_balance(view, k, 0.5), ops.moe_route_balance(x, k, 0.5)
    assert all(torch.equal(a[f], b[f]) for f in a)
    kw = dict(dgates=torch.randn((T, k), device=dev), counts=a["counts"], tokens=a["tokens"], coef=0.5)
    want = ops.moe_route_backward(x, b["ids"], **kw)
    ops.moe_route_backward(view, a["ids"], **kw, out=view)
    assert torch.equal(view, want)
    del wide, view
    # one token per expert: a padded row block each
    n, H = 2400, 7168
    assert n * 128 * H > 2**31
    ids = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().view(n, 1).to(dev)
    gates = torch.rand((n, 1), device=dev) + 0.5
    t = ops.moe_build_indices_dev(ids, gates, 0, n)
    assert t["R_pad"] == n * 128
    ye = torch.zeros((n * 128, H), dtype=torch.bfloat16, device=dev)
    rows = ids[:, 0].long() * 128
    ye[rows] = wl.randn_bf16((n, H), 2).to(dev)
    dy = wl.randn_bf16((n, H), 3).to(dev)
    dye, dg = ops.moe_combine_backward(dy, ye, ids, t["row_weight"], t["owner_offset"], t["slot_to_row"], t["rb_rows"], 0, n)
    assert torch.equal(dye[rows], (gates * dy.float()).to(torch.bfloat16))
    ref = (dy.to(D) * ye[rows].to(D))
    assert bool(((dg[:, 0].to(D) - ref.sum(1)).abs() <= (2 * (H / 32 + 8) + 12) * 2 ** -24 * ref.abs().sum(1)).all())
    dye[rows] = 0
    assert not dye.any()


def test_combine_backward_no_rows(dev):
    """A rank that no token was routed to, a batch of no tokens, and rows that another owner holds."""
    _say("combine backward without rows")
    ids = torch.zeros((6, 2), dtype=torch.int32, device=dev)
    gates = torch.ones((6, 2), device=dev)
    t = ops.moe_build_indices_dev(ids, gates, 5, 3)
    dy = torch.full((6, 64), NAN, device=dev)
    a, dg = ops.moe_combine_backward(dy, torch.empty((0, 64), dtype=torch.bfloat16, device=dev), ids, t["row_weight"],
                                     t["owner_offset"], t["slot_to_row"], t["rb_rows"], 5, 3)
    assert a.shape == (0, 64) and not dg.any()
    t = ops.moe_build_indices_dev(ids, gates, 0, 3)
    t["slot_to_row"].fill_(-1)
    ye = torch.zeros((t["R_pad"], 64), dtype=torch.bfloat16, device=dev)
    a, dg = ops.moe_combine_backward(dy, ye, ids, t["row_weight"], t["owner_offset"], t["slot_to_row"], t["rb_rows"], 0, 3)
    assert not dg.any() and not a[12:].any()
    none = ids[:0]
    a, dg = ops.moe_combine_backward(dy[:0], ye, none, t["row_weight"], torch.zeros(1, dtype=torch.int32, device=dev),
                                     t["slot_to_row"], t["rb_rows"], 0, 3)
    assert dg.shape == (0, 2)


def test_combine_backward_offsets_without_rows(dev):
    """Owner offsets of routed tokens, but no rows here: no table of rows is read, and dgates is 0."""
    _say("combine backward, offsets without rows")
    T, H, k = 6, 64, 2
    ids = torch.arange(T * k, dtype=torch.int32, device=dev).view(T, k) % 3
    t = ops.moe_build_indices_dev(ids, torch.ones((T, k), device=dev), 0, 3)
    dy = torch.ones((T, H), device=dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    assert none.data_ptr() == 0 and int(t["owner_offset"][-1]) == T * k
    a, dg = ops.moe_combine_backward(dy, torch.empty((0, H), dtype=torch.bfloat16, device=dev), ids, t["row_weight"][:0],
                                     t["owner_offset"], none, none, 0, 3, dgates=torch.full((T, k), NAN, device=dev))
    assert a.shape == (0, H) and not dg.any()
    # a capacity of one block, of which the device counts no row
    ye = torch.full((128, H), NAN, dtype=torch.bfloat16, device=dev)
    keep = torch.full((128, H), 7.0, dtype=torch.bfloat16, device=dev)
    _, dg = ops.moe_combine_backward(dy, ye, ids, torch.ones(128, device=dev), t["owner_offset"], t["slot_to_row"],
                                     torch.zeros(1, dtype=torch.int32, device=dev), 0, 3, dy_expert=keep,
                                     dgates=torch.full((T, k), NAN, device=dev),
                                     sizes=torch.zeros(2, dtype=torch.int64, device=dev))
    assert not dg.any() and bool((keep == 7).all())


def test_repeatable_on_other_streams_and_in_a_graph(dev):
    """Equal bits on another stream, beside another call, and in replays of a captured graph with new inputs."""
    _say("streams and graph")
    T, E, k = 3000, 60, 4
    xs = [_logits(T, E, torch.float32, s).to(dev) for s in range(3)]
    dg = torch.randn((T, k), device=dev)

    def step(x):
        r = ops.moe_route_balance(x, k, 0.1)
        d = ops.moe_route_backward(x, r["ids"], dgates=dg, counts=r["counts"], tokens=r["tokens"], coef=0.1)
        return [r["ids"], r["gates"], r["loss"], r["counts"], r["prob_sum"], r["tokens"], d]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(side, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(x))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for rep in range(4):
        x.copy_(xs[rep % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want[rep % 3])), rep
        step(xs[1])  # eager work between the replays
