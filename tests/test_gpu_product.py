"""Dense products with an epilogue, expert products on ragged rows and the
vocabulary loss, forward and backward, against their formulas in 64 bits.

Tolerances.  Inputs are exact bf16 values.  A sum of n products in fp32, in any
order, is off by at most n * 2^-24 * sum |products| (each addition rounds by half
a step of a partial sum that the sum of magnitudes bounds); an activation adds a
few fp32 steps of its argument and, for gelu, 1.5e-7 |x|; a result rounds once,
by half a step of its type: 2^-8 of its value in bf16, 2^-24 in fp32.  Where a
value goes through bf16 between two products (the gradient of a pre-activation
or of the logits), it is off by 2^-8 of itself, so the next sum by 2^-8 * sum
|products|."""
import math

import pytest
import torch

from mkernel_amd import ops
from mkernel_amd.capi import MkError

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def randn(*shape, seed=0, scale=1.0, dtype=BF16, pad=0, offset=0):
    """Normal values on the GPU; pad: columns behind each row, offset: elements in front of the first (a view)."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g, dtype=F32) * scale).to(dtype)
    if not pad and not offset:
        return x.cuda()
    *lead, rows, cols = x.shape if len(shape) > 1 else (1, *x.shape)
    wide = torch.full((offset + rows * (cols + pad),), float("nan"), dtype=dtype)
    view = wide[offset:].view(rows, cols + pad)[:, :cols]
    view.copy_(x.view(rows, cols))
    big = wide.cuda()
    v = big[offset:].view(rows, cols + pad)[:, :cols]
    return v if len(shape) > 1 else v[0]


def d(t):
    return t.detach().cpu().to(F64)


def act64(x, act):
    """act(x), its slope, and a bound of the slope's own slope."""
    if act == "none":
        return x, torch.ones_like(x)
    if act == "relu":
        return x.clamp(min=0), (x > 0).to(F64)
    if act == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * (1 - s)
    if act == "gelu":
        c = 0.5 * torch.erfc(-x / math.sqrt(2))
        return x * c, c + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (x + 0.044715 * x ** 3))
    return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)


def near(got, want, tol):
    got, tol = d(got), torch.as_tensor(tol, dtype=F64)
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, " \
                          f"worst {float((off / tol.clamp(min=1e-300)).max())} of the tolerance"


def act_tol(x, err):
    """What an error of the argument and the activation's own fp32 steps do: slopes are at most 1.13."""
    return 1.13 * err + 2.0 ** -20 * x.abs() + 1e-37


# ---------------------------------------------------------------- C = act(A @ B + bias) + residual
SHAPES = [(1, 1, 1), (1, 8, 8), (1, 2048, 2048), (2, 640, 24), (3, 72, 40), (7, 1000, 333), (31, 64, 129),
          (33, 100, 130), (64, 4096, 256), (129, 257, 255), (200, 31, 700), (256, 512, 256), (300, 1000, 520),
          (513, 96, 1025), (1100, 1544, 776)]


def _check_gemm_act(M, K, N, act, bias, residual, out_dtype, pre, pads=(0, 0, 0), offsets=(0, 0), seed=1):
    A = randn(M, K, seed=seed, pad=pads[0], offset=offsets[0])
    B = randn(K, N, seed=seed + 1, scale=max(K, 1) ** -0.5, pad=pads[1], offset=offsets[1])
    b = None if bias is None else randn(N, seed=seed + 2, dtype=bias)
    r = None if residual is None else randn(M, N, seed=seed + 3, dtype=residual, pad=pads[2])
    p = torch.empty(M, N, dtype=BF16, device="cuda") if pre else None
    got = ops.gemm_act(A, B, bias=b, act=act, residual=r, pre=p, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    x = d(A) @ d(B)
    mag = d(A).abs() @ d(B).abs()
    if b is not None:
        x, mag = x + d(b), mag + d(b).abs()
    err = (K + 2) * U * mag
    y = act64(x, act)[0]
    tol = act_tol(x, err)
    if r is not None:
        y, tol = y + d(r), tol + U * (y.abs() + d(r).abs())
    near(got, y, HALF[out_dtype] * (y.abs() + tol) + tol)
    if pre:
        near(p, x, HALF[BF16] * (x.abs() + err) + err)
    return got


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_gemm_act(shape, act):
    i = SHAPES.index(shape) + ACTS.index(act)
    _check_gemm_act(*shape, act, [None, BF16, F32][i % 3], [None, BF16, F32, None][i % 4], [BF16, F32][i % 2],
                    i % 3 == 1)


@pytest.mark.parametrize("pads,offsets", [((1, 0, 0), (0, 0)), ((0, 3, 5), (0, 0)), ((8, 16, 8), (0, 0)),
                                          ((0, 0, 0), (1, 0)), ((0, 0, 0), (0, 3)), ((7, 9, 1), (5, 2))], ids=str)
@pytest.mark.parametrize("shape", [(1, 96, 72), (37, 250, 131), (300, 512, 264)], ids=str)
def test_gemm_act_strides(shape, pads, offsets):
    """Columns of wider matrices (NaN behind each row) and first elements off a 16-byte boundary."""
    _check_gemm_act(*shape, "silu", BF16, F32, BF16, True, pads, offsets)


def test_gemm_act_without_a_sum():
    b, r = randn(24, seed=1), randn(5, 24, seed=2)
    got = ops.gemm_act(torch.empty(5, 0, dtype=BF16, device="cuda"), torch.empty(0, 24, dtype=BF16, device="cuda"),
                       bias=b, act="relu", residual=r, out_dtype=F32)
    assert torch.equal(got, b.float().clamp(min=0) + r.float())
    assert ops.gemm_act(randn(4, 8)[:0], randn(8, 16)).shape == (0, 16)
    assert ops.gemm_act(randn(4, 8), randn(8, 16)[:, :0]).shape == (4, 0)


def test_gemm_act_in_place_and_into_wider():
    A, B = randn(70, 200, seed=3), randn(200, 96, seed=4, scale=0.07)
    r = randn(70, 96, seed=5)
    want = ops.gemm_act(A, B, residual=r)
    stream = r.clone()
    assert ops.gemm_act(A, B, residual=stream, out=stream) is stream
    assert torch.equal(stream, want)
    wide = torch.full((70, 140), 7.0, dtype=BF16, device="cuda")
    ops.gemm_act(A, B, residual=r, out=wide[:, 20:116])
    assert torch.equal(wide[:, 20:116], want)
    assert (wide[:, :20] == 7).all() and (wide[:, 116:] == 7).all()


def test_gemm_act_what_is_not_finite():
    """NaN and infinities stay in their row, also behind the sum's last stage, and activations pass them on."""
    A, B = randn(40, 72, seed=6), randn(72, 33, seed=7)
    A[3, 71] = float("nan")
    A[5, 0] = float("inf")
    got = ops.gemm_act(A, B, act="relu", out_dtype=F32)
    assert got[3].isnan().all()
    assert torch.equal(got[5].isinf(), B[0] > 0) and (got[5][B[0] < 0] == 0).all()
    rest = [i for i in range(40) if i not in (3, 5)]
    assert got[rest].isfinite().all()


def test_gemm_act_far_arguments():
    """Every activation at arguments where its exponentials under- and overflow."""
    x = torch.tensor([-3e38, -1e4, -200.0, -88.0, -20.0, -5.0, -1e-30, 0.0, 1e-30, 5.0, 20.0, 88.0, 200.0, 1e4, 3e38])
    B = x.to(BF16).cuda()[None]
    A = torch.ones(1, 1, dtype=BF16, device="cuda")
    for act in ACTS:
        got = d(ops.gemm_act(A, B, act=act, out_dtype=F32))[0]
        xb = d(B)[0]
        want = xb.clamp(min=0) if act == "gelu_tanh" else act64(xb, act)[0]
        if act == "gelu_tanh":  # x^3 leaves fp32 (and its sum 64 bits' tanh) at the far ends, where the value is x or 0
            inner = xb.abs() < 1e3
            want[inner] = act64(xb, act)[0][inner]
        assert (got - want).abs().le(1e-5 * want.abs() + 2e-6).all(), (act, got, want)


def test_gemm_act_repeats_bit_for_bit():
    for M, K, N in [(1, 4096, 512), (16, 8192, 256), (300, 640, 520)]:
        A, B = randn(M, K, seed=8), randn(K, N, seed=9)
        first = ops.gemm_act(A, B)
        for _ in range(4):
            assert torch.equal(ops.gemm_act(A, B), first)


def test_gemm_act_agrees_with_gemm():
    A, B = randn(256, 512, seed=10), randn(512, 512, seed=11, scale=0.05)
    x = d(A) @ d(B)
    near(ops.gemm(A, B), x, 2.0 ** -8 * x.abs() + 514 * U * (d(A).abs() @ d(B).abs()))
    near(ops.gemm_act(A, B), d(ops.gemm(A, B)), 2.0 ** -7 * x.abs() + 1e-3)


# ---------------------------------------------------------------- gradients
def _check_backward(M, K, N, act, db_dtype, pads=(0, 0, 0, 0), accumulate=False, seed=20):
    dC = randn(M, N, seed=seed, pad=pads[0])
    A = randn(M, K, seed=seed + 1, pad=pads[1])
    B = randn(K, N, seed=seed + 2, scale=N ** -0.5, pad=pads[2])
    pre = None if act == "none" else randn(M, N, seed=seed + 3, pad=pads[3])
    dB = dbias = None
    if accumulate:
        dB, dbias = randn(K, N, seed=seed + 4, dtype=db_dtype), randn(N, seed=seed + 5, dtype=F32)
        dB0, db0 = d(dB), d(dbias)
    dA, dB, dbias = ops.gemm_act_backward(dC, A, B, pre=pre, act=act, dB=dB, dbias=dbias, dB_dtype=db_dtype,
                                          accumulate=accumulate)
    s = torch.ones(M, N, dtype=F64) if pre is None else act64(d(pre), act)[1]
    g = d(dC) * s
    # the slope's own steps: its parts are at most about 1 + |x|
    ge = (0 if act in ("none", "relu") else 2.0 ** -20 * (1 + d(pre).abs())) * d(dC).abs()
    gb = ge + (0 if act in ("none", "relu") else 2.0 ** -8 * (g.abs() + ge))
    want = g @ d(B).t()
    tol = (gb + N * U * g.abs()) @ d(B).abs().t()
    near(dA, want, 2.0 ** -8 * (want.abs() + tol) + tol)
    want = d(A).t() @ g
    tol = d(A).abs().t() @ (gb + (M + 1) * U * g.abs())
    if accumulate:
        want, tol = want + dB0, tol + U * (want.abs() + dB0.abs())
    near(dB, want, HALF[db_dtype] * (want.abs() + tol) + tol)
    want, tol = g.sum(0), (ge + (M + 2) * U * g.abs()).sum(0)
    if accumulate:
        want, tol = want + db0, tol + U * (want.abs() + db0.abs())
    near(dbias, want, tol + U * want.abs())


GRAD_SHAPES = [(1, 1, 1), (1, 64, 72), (2, 40, 8), (65, 130, 33), (128, 256, 128), (300, 264, 520), (700, 97, 101),
               (1030, 512, 256)]


@pytest.mark.parametrize("shape", GRAD_SHAPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_gemm_act_backward(shape, act):
    i = GRAD_SHAPES.index(shape) + ACTS.index(act)
    _check_backward(*shape, act, [BF16, F32][i % 2], accumulate=i % 3 == 0)


@pytest.mark.parametrize("pads", [(1, 0, 0, 0), (0, 5, 0, 0), (0, 0, 3, 0), (0, 0, 0, 2), (8, 8, 8, 8), (3, 1, 7, 5)], ids=str)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_gemm_act_backward_strides(pads, act):
    _check_backward(90, 120, 71, act, F32, pads)
    _check_backward(90, 120, 72, act, F32, pads)


def test_gemm_act_backward_parts_and_empty():
    dC, A, B = randn(64, 80, seed=1), randn(64, 48, seed=2), randn(48, 80, seed=3)
    full = ops.gemm_act_backward(dC, A, B)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)):
        got = ops.gemm_act_backward(dC, A, B, need_dA=bool(need[0]), need_dB=bool(need[1]), need_dbias=bool(need[2]))
        for g, f, n in zip(got, full, need):
            assert (g is None) == (not n) and (g is None or torch.equal(g, f))
    dA, dB, dbias = ops.gemm_act_backward(dC[:0], A[:0], B)
    assert dA.shape == (0, 48) and (dB == 0).all() and (dbias == 0).all()


def test_gemm_act_gradient_against_differences():
    """Along the gradient's own signs, against differences of the formula in 64 bits.  (Differences of the forward
    call itself need steps that bf16 inputs can take: 1/16 in each of 40 terms moves a pre-activation by about 2,
    where the third-order rest of the difference is as large as its first.)"""
    M, K, N, act = 24, 40, 56, "gelu_tanh"
    A, B, b = randn(M, K, seed=30), randn(K, N, seed=31, scale=K ** -0.5), randn(N, seed=32, dtype=F32)
    dC = randn(M, N, seed=33)
    pre = torch.empty(M, N, dtype=BF16, device="cuda")
    ops.gemm_act(A, B, bias=b, act=act, pre=pre)
    grads = ops.gemm_act_backward(dC, A, B, pre=pre, act=act, dB_dtype=F32)
    args = [d(A), d(B), d(b)]

    def value(a, w, c):
        return float((act64(a @ w + c, act)[0] * d(dC)).sum())

    x = args[0] @ args[1] + args[2]
    for i, grad in enumerate(grads):
        step = torch.sign(d(grad)) * 2.0 ** -14
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + step, args[i] - step
        slope, want = value(*hi) - value(*lo), float((d(grad) * (2 * step)).sum())
        # what a pre-activation moves by, times what its slope may be off by: pre is rounded (slopes' slopes are at
        # most 1.2), and so is dpre; then the result's own rounding, and 2^-14 for the rest of the difference
        move = 2 * ((step.abs() @ args[1].abs()) if i == 0 else args[0].abs() @ step.abs() if i == 1 else step.abs())
        off = float((d(dC).abs() * move * 2.0 ** -8 * (1.2 * x.abs() + 1.13)).sum()) + (2.0 ** -8 + 2.0 ** -14) * abs(want)
        assert abs(slope - want) <= off, (i, slope, want, off)
        assert off < 0.5 * abs(want)  # (so that another factor would be seen)


# ---------------------------------------------------------------- expert products on ragged rows
def _experts(counts, R, K, N, seed, scale=1.0, pad=0):
    E = len(counts)
    A = randn(R, K, seed=seed, pad=pad)
    n = 0
    rows = []
    for c in counts:
        c = max(c, 0)
        rows.append((min(n, R), min(n + c, R)))
        n += c
    A[min(n, R):] = float("nan")  # behind the last expert's rows
    W = randn(E, K, N, seed=seed + 1, scale=K ** -0.5)
    return A, W, torch.tensor(counts, dtype=torch.int32, device="cuda"), rows


COUNTS = [([5], 5), ([0], 3), ([1, 0, 2, 0], 9), ([130, 1, 0, 64, 257], 460), ([0, 0, 300], 300), ([40, -7, 50], 100),
          ([100, 100, 100], 150), ([3] * 100, 310), ([256, 512], 768)]
RAGGED = [(8, 16), (72, 64), (257, 130), (512, 256), (100, 1026)]


@pytest.mark.parametrize("counts,R", COUNTS, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("K,N", RAGGED)
@pytest.mark.parametrize("mode", [0, 1])
def test_moe_ragged_gemm(counts, R, K, N, mode):
    A, W, n, rows = _experts(counts, R, K, N, 40)
    out = torch.full((R, N // 2 if mode else N), 3.0, dtype=BF16, device="cuda")
    h = torch.full((R, N), 5.0, dtype=BF16, device="cuda") if mode else None
    assert ops.moe_ragged_gemm(A, W, n, mode=mode, out=out, h=h) is out
    for e, (lo, hi) in enumerate(rows):
        x = d(A[lo:hi]) @ d(W[e])
        err = (K + 2) * U * (d(A[lo:hi]).abs() @ d(W[e]).abs())
        if mode == 0:
            near(out[lo:hi], x, 2.0 ** -8 * (x.abs() + err) + err)
            continue
        near(h[lo:hi], x, 2.0 ** -8 * (x.abs() + err) + err)
        g, u = x[:, :N // 2], x[:, N // 2:]
        eg, eu = err[:, :N // 2], err[:, N // 2:]
        y = act64(g, "silu")[0] * u
        tol = act_tol(g, eg) * (u.abs() + eu) + g.abs() * eu + 2 * U * y.abs()
        near(out[lo:hi], y, 2.0 ** -8 * (y.abs() + tol) + tol)
    last = rows[-1][1]
    assert (out[last:] == 3).all() and (h is None or (h[last:] == 5).all())


@pytest.mark.parametrize("counts,R", COUNTS, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("K,N", RAGGED)
@pytest.mark.parametrize("swiglu", [False, True])
def test_moe_ragged_dgrad(counts, R, K, N, swiglu):
    dy, Wt, n, rows = _experts(counts, R, N, K, 50)
    W = Wt.transpose(1, 2).contiguous()
    h = randn(R, 2 * K, seed=52) if swiglu else None
    out = torch.full((R, 2 * K if swiglu else K), 3.0, dtype=BF16, device="cuda")
    ops.moe_ragged_gemm_dgrad(dy, W, n, h=h, out=out)
    for e, (lo, hi) in enumerate(rows):
        x = d(dy[lo:hi]) @ d(W[e]).t()
        err = (N + 2) * U * (d(dy[lo:hi]).abs() @ d(W[e]).abs().t())
        if not swiglu:
            near(out[lo:hi], x, 2.0 ** -8 * (x.abs() + err) + err)
            continue
        g, u = d(h[lo:hi, :K]), d(h[lo:hi, K:])
        a, slope = act64(g, "silu")
        for got, f, fe in ((out[lo:hi, :K], u * slope, 2.0 ** -20 * u.abs() * (1 + g.abs())),
                           (out[lo:hi, K:], a, 2.0 ** -20 * g.abs())):
            want = x * f
            tol = err * (f.abs() + fe) + x.abs() * fe + 4 * U * want.abs()
            near(got, want, 2.0 ** -8 * (want.abs() + tol) + tol)
    assert (out[rows[-1][1]:] == 3).all()
    if swiglu:  # in place of h
        h2 = h.clone()
        ops.moe_ragged_gemm_dgrad(dy, W, n, h=h2, out=h2)
        last = rows[-1][1]
        assert torch.equal(h2[:last], out[:last]) and torch.equal(h2[last:], h[last:])


@pytest.mark.parametrize("counts,R", COUNTS, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("K,N", RAGGED)
@pytest.mark.parametrize("dtype,accumulate", [(BF16, False), (F32, True)], ids=["bf16", "f32+"])
def test_moe_ragged_wgrad(counts, R, K, N, dtype, accumulate):
    A, _, n, rows = _experts(counts, R, K, N, 60)
    dy = randn(R, N, seed=62)
    dy[rows[-1][1]:] = float("inf")
    E = len(counts)
    out = randn(E, K, N, seed=63, dtype=dtype) if accumulate else torch.full((E, K, N), 9.0, dtype=dtype, device="cuda")
    before = d(out)
    ops.moe_ragged_gemm_wgrad(A, dy, n, out=out, accumulate=accumulate)
    for e, (lo, hi) in enumerate(rows):
        want = d(A[lo:hi]).t() @ d(dy[lo:hi])
        tol = (hi - lo + 1) * U * (d(A[lo:hi]).abs().t() @ d(dy[lo:hi]).abs())
        if accumulate:
            want, tol = want + before[e], tol + U * (want.abs() + before[e].abs())
        near(out[e], want, HALF[dtype] * (want.abs() + tol) + tol)


@pytest.mark.parametrize("pad", [1, 8])
def test_moe_ragged_strides(pad):
    counts, R, K, N = [33, 0, 90], 140, 96, 64
    A, W, n, rows = _experts(counts, R, K, N, 70, pad=pad)
    near(ops.moe_ragged_gemm(A, W, n)[:123], d(ops.moe_ragged_gemm(A.contiguous(), W, n)[:123]), 0)
    dy = randn(R, N, seed=72, pad=pad)
    near(ops.moe_ragged_gemm_dgrad(dy, W, n)[:123], d(ops.moe_ragged_gemm_dgrad(dy.contiguous(), W, n)[:123]), 0)
    near(ops.moe_ragged_gemm_wgrad(A, dy, n), d(ops.moe_ragged_gemm_wgrad(A.contiguous(), dy.contiguous(), n)), 0)


# ---------------------------------------------------------------- vocabulary loss
def _vocab64(x, W, labels, begin=0, ignore=-100):
    on = labels != ignore
    z = torch.where(on[:, None], d(x), 0.0) @ d(W)
    lse = torch.logsumexp(z, 1)
    at = labels - begin
    here = on & (at >= 0) & (at < W.shape[1])
    t = torch.where(here, z.gather(1, at.clamp(0, W.shape[1] - 1)[:, None])[:, 0], 0.0)
    mag = torch.where(on[:, None], d(x).abs(), 0.0) @ d(W).abs()
    return on, here, at, z, mag, torch.where(on, lse, 0.0), t


VOCAB = [(1, 8, 1), (1, 64, 1000), (3, 40, 17), (33, 100, 515), (64, 512, 4096), (130, 257, 1003), (300, 128, 2048),
         (520, 72, 777)]


def _check_vocab(T, H, V, labels, x, W, begin=0, ignore=-100, piece=0, dx_dtype=BF16, dw_dtype=BF16, accumulate=False):
    lab = labels.cuda()
    r = ops.vocab_loss(x, W, lab, vocab_begin=begin, ignore_index=ignore)
    on, here, at, z, mag, lse, t = _vocab64(x, W, labels.to(torch.int64), begin, ignore)
    err = (H + 2) * U * mag
    worst = torch.where(on, err.amax(1), 0.0)
    # each exponential: its argument's error, three steps of its own per unit of the argument; sums of V parts by
    # groups of 64, V / 64 of them
    span = (z.amax(1) - z.amin(1)).clamp(min=1)
    tol = worst + (64 + V / 64 + 4 * 8 + 3 * span.clamp(max=90)) * U + 4 * U * lse.abs()
    near(r["lse"], lse, torch.where(on, tol, 0.0))
    near(r["target"], t, torch.where(here, worst, 0.0))
    near(r["loss"], torch.where(on, lse - t, 0.0), torch.where(on, tol + worst + U * (lse.abs() + t.abs()), 0.0))
    dloss = randn(T, seed=90, dtype=F32)
    dloss[~on.cuda()] = float("nan")
    dW = randn(H, V, seed=91, dtype=dw_dtype) if accumulate else None
    before = d(dW) if accumulate else 0.0
    dx, dW = ops.vocab_loss_backward(x, W, lab, r["lse"], dloss, vocab_begin=begin, ignore_index=ignore, dW=dW,
                                     dx_dtype=dx_dtype, dW_dtype=dw_dtype, accumulate=accumulate, piece_columns=piece)
    p = torch.exp(z - lse[:, None])
    w = torch.where(on, d(dloss), 0.0)
    hot = torch.zeros(T, V, dtype=F64)
    hot[here.nonzero()[:, 0], at[here]] = 1.0
    dl = (p - hot) * w[:, None]
    # p is off by the errors of its exponent, then dl by its rounding
    pe = p * (err + tol[:, None] + 2 * (3 * (z - lse[:, None]).abs().clamp(max=90) + 2) * U) * w.abs()[:, None]
    # (exponentials and results below the smallest normal number, 2^-126, may be flushed to zero)
    tiny = 2.0 ** -126
    de = pe + 2.0 ** -8 * (dl.abs() + pe) + tiny * (1 + w.abs()[:, None])
    xs = torch.where(on[:, None], d(x), 0.0)
    want, n = dl @ d(W).t(), V + 8
    tol = (de + n * U * dl.abs()) @ d(W).abs().t()
    near(dx, want, HALF[dx_dtype] * (want.abs() + tol) + tol + tiny)
    want = xs.t() @ dl
    tol = xs.abs().t() @ (de + (T + 1) * U * dl.abs())
    if accumulate:
        want, tol = want + before, tol + U * (want.abs() + before.abs())
    near(dW, want, HALF[dw_dtype] * (want.abs() + tol) + tol + tiny)
    return r, dx, dW


def _labels(T, V, seed, begin=0, dtype=torch.int64):
    return (torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed)) + begin).to(dtype)


@pytest.mark.parametrize("T,H,V", VOCAB)
def test_vocab_loss(T, H, V):
    i = VOCAB.index((T, H, V))
    labels = _labels(T, V, 80, dtype=[torch.int64, torch.int32][i % 2])
    x, W = randn(T, H, seed=81), randn(H, V, seed=82, scale=2 * H ** -0.5)
    if T > 2:
        labels[::3] = -100
        x[::3] = float("nan")
        x[(T - 1) // 3 * 3] = float("inf")
    _check_vocab(T, H, V, labels, x, W, dx_dtype=[BF16, F32][i % 2], dw_dtype=[F32, BF16][i % 2],
                 accumulate=i % 3 == 0, piece=[0, 256, 512][i % 3])


@pytest.mark.parametrize("pads", [(3, 0), (0, 5), (8, 8), (1, 1)], ids=str)
def test_vocab_loss_strides(pads):
    T, H, V = 70, 96, 520
    _check_vocab(T, H, V, _labels(T, V, 83), randn(T, H, seed=84, pad=pads[0]),
                 randn(H, V, seed=85, scale=0.2, pad=pads[1]), piece=256)


def test_vocab_loss_all_ignored():
    x = torch.full((50, 64), float("nan"), dtype=BF16, device="cuda")
    _check_vocab(50, 64, 300, torch.full((50,), -1), x, randn(64, 300, seed=86), ignore=-1)
    r = ops.vocab_loss(x[:0], randn(64, 300), torch.empty(0, dtype=torch.int64, device="cuda"))
    assert r["loss"].shape == (0,)
    dx, dW = ops.vocab_loss_backward(x[:0], randn(64, 300), torch.empty(0, dtype=torch.int64, device="cuda"), r["lse"],
                                     r["lse"])
    assert dx.shape == (0, 64) and (dW == 0).all()


def test_vocab_loss_far_logits():
    """Logits of several hundreds: the running maximum keeps every exponential in range."""
    T, H, V = 40, 64, 900
    x, W = randn(T, H, seed=87, scale=16.0), randn(H, V, seed=88, scale=4.0)
    _check_vocab(T, H, V, _labels(T, V, 89), x, W)


def test_vocab_loss_shards():
    """Two ranks' halves of a vocabulary, joined, give the whole one's loss and gradients."""
    T, H, V, half = 60, 80, 1000, 480
    labels = _labels(T, V, 92)
    labels[7] = -100
    x, W = randn(T, H, seed=93), randn(H, V, seed=94, scale=0.3)
    parts = [(W[:, :half].contiguous(), 0), (W[:, half:].contiguous(), half)]
    r = [ops.vocab_loss(x, w, labels.cuda(), vocab_begin=b) for w, b in parts]
    for (w, b), q in zip(parts, r):
        _check_vocab(T, H, w.shape[1], labels, x, w, begin=b, dx_dtype=F32)
    lse = torch.logsumexp(torch.stack([q["lse"] for q in r]), 0)
    loss = lse - r[0]["target"] - r[1]["target"]
    whole = ops.vocab_loss(x, W, labels.cuda())
    on = (labels != -100).cuda()
    assert torch.allclose(loss[on], whole["loss"][on], rtol=0, atol=1e-4)
    dloss = torch.full((T,), 1.0 / T, device="cuda")
    dx, dW = ops.vocab_loss_backward(x, W, labels.cuda(), whole["lse"], dloss, dx_dtype=F32, dW_dtype=F32)
    g = [ops.vocab_loss_backward(x, w, labels.cuda(), torch.where(on, lse, 0.0), dloss, vocab_begin=b, dx_dtype=F32,
                                 dW_dtype=F32) for w, b in parts]
    # both round dl to bf16, from logits whose last bits may differ
    assert torch.allclose(g[0][0] + g[1][0], dx, rtol=0, atol=float(dx.abs().max()) * 2.0 ** -7)
    assert torch.allclose(torch.cat([g[0][1], g[1][1]], 1), dW, rtol=0, atol=float(dW.abs().max()) * 2.0 ** -7)


def test_vocab_loss_gradient_against_differences():
    """Along the gradient's own signs, against differences of the formula in 64 bits."""
    T, H, V = 20, 48, 300
    labels = _labels(T, V, 95)
    x, W = randn(T, H, seed=96), randn(H, V, seed=97, scale=0.3)
    dloss = randn(T, seed=98, dtype=F32)
    r = ops.vocab_loss(x, W, labels.cuda())
    grads = ops.vocab_loss_backward(x, W, labels.cuda(), r["lse"], dloss, dx_dtype=F32, dW_dtype=F32)
    args = [d(x), d(W)]

    def value(a, w):
        return float((-torch.log_softmax(a @ w, 1)[torch.arange(T), labels] * d(dloss)).sum())

    p = torch.softmax(args[0] @ args[1], 1)
    p[torch.arange(T), labels] -= 1
    dl = (p * d(dloss)[:, None]).abs()
    for i, grad in enumerate(grads):
        step = torch.sign(d(grad)) * 2.0 ** -14
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + step, args[i] - step
        slope, want = value(*hi) - value(*lo), float((d(grad) * (2 * step)).sum())
        # the logits' gradient is rounded to bf16; 2^-13 for fp32 and the rest of the difference
        move = 2 * ((step.abs() @ args[1].abs()) if i == 0 else args[0].abs() @ step.abs())
        off = float((dl * move).sum()) * 2.0 ** -8 + 2.0 ** -13 * abs(want)
        assert abs(slope - want) <= off, (i, slope, want, off)
        assert off < 0.5 * abs(want)  # (so that another factor would be seen)


def test_vocab_loss_pieces_of_laid_out_weights():
    """An odd vocabulary whose weights are laid out anew in several pieces, forward and back; labels in each."""
    T, H, V = 5, 4096, 33001
    labels = torch.tensor([0, 16383, 16384, 32768, 33000])
    _check_vocab(T, H, V, labels, randn(T, H, seed=99), randn(H, V, seed=100, scale=2 * H ** -0.5))


def test_vocab_loss_backward_of_ignored_tokens():
    """Zeros, whatever their rows, lse and dloss hold (a shard's joined lse of them is not 0)."""
    T, H, V = 40, 72, 333
    labels = _labels(T, V, 97)
    off = torch.arange(T) % 3 == 1
    labels[off] = -100
    x, W, labels, off = randn(T, H, seed=98), randn(H, V, seed=99, scale=0.3), labels.cuda(), off.cuda()
    lse = ops.vocab_loss(x, W, labels)["lse"]
    dloss = torch.full((T,), 0.25, device="cuda")
    want = ops.vocab_loss_backward(x, W, labels, lse, dloss, dx_dtype=F32, dW_dtype=F32)
    assert (want[0][off] == 0).all()
    for bad in (float("nan"), float("inf"), -float("inf"), 0.6931):
        got = ops.vocab_loss_backward(torch.where(off[:, None], bad, x.float()).to(BF16), W, labels,
                                      torch.where(off, bad, lse), torch.where(off, bad, dloss), dx_dtype=F32,
                                      dW_dtype=F32)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("every", [1.0 / 509, 1.0039, 1.0, 0.25 + 2.0 ** -10])
@pytest.mark.parametrize("piece", [0, 512])
def test_vocab_loss_backward_keeps_the_scale(every, piece):
    """One dloss for all tokens, whatever its significand: the gradients are not longer or shorter than they should be.
    The factor of the nearest multiple of the right gradient is off by the labels' entries of dl, -(1 - p) times a power
    of two, whose rounding is off by p at most where p < 2^-9 (to 1), by the other entries' roundings, random and of
    2^-9 each, over the root of their number, and by the sums' of at most 2^-14."""
    T, H, V = 509, 64, 4000
    labels = _labels(T, V, 100).cuda()
    x, W = randn(T, H, seed=101), randn(H, V, seed=102, scale=0.3 * H ** -0.5)
    lse = ops.vocab_loss(x, W, labels)["lse"]
    dloss = torch.full((T,), every, device="cuda")
    dx, dW = ops.vocab_loss_backward(x, W, labels, lse, dloss, dx_dtype=F32, dW_dtype=F32, piece_columns=piece)
    p = torch.softmax(d(x) @ d(W), 1)
    most = float(p.max())
    assert most < 2.0 ** -9
    p[torch.arange(T), labels.cpu()] -= 1
    dl = p * d(dloss)[:, None]
    for got, want in ((d(dx), dl @ d(W).t()), (d(dW), d(x).t() @ dl)):
        factor = float((got * want).sum() / (want * want).sum())
        assert abs(factor - 1) <= most + 2.0 ** -9 / T ** 0.5 + 2.0 ** -14, factor


def test_vocab_loss_backward_of_unlike_dloss():
    """Largest, smallest, infinite, NaN and zero dloss beside each other: each row of dx is its token's alone."""
    T, H, V = 24, 40, 300
    labels = _labels(T, V, 103).cuda()
    x, W = randn(T, H, seed=104), randn(H, V, seed=105, scale=0.3)
    lse = ops.vocab_loss(x, W, labels)["lse"]
    dloss = torch.tensor([1.5, 1e-30, 3e30, float("inf"), float("nan"), 0.0, -2.75, 1e-3] * 3, device="cuda")
    dx = d(ops.vocab_loss_backward(x, W, labels, lse, dloss, need_dW=False, dx_dtype=F32)[0])
    p = torch.softmax(d(x) @ d(W), 1)
    p[torch.arange(T), labels.cpu()] -= 1
    finite = torch.isfinite(dloss).cpu()
    dl = p * d(dloss)[:, None]
    tol = 2.0 ** -7 * dl.abs() @ d(W).abs().t()
    assert ((dx - dl @ d(W).t()).abs()[finite] <= tol[finite]).all()
    assert not torch.isfinite(dx[~finite]).any()
