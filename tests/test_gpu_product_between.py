"""Gradients whose dpre or dl go between the products in float32 (three bf16
parts, which hold all of its bits): as exact as fp32 sums of fp32 numbers.

Tolerances.  A slope is good to 2^-20 of (1 + |x|), its product with dC rounds by
2^-24; a sum of n products in fp32 is off by n * 2^-24 * sum |products|, of three
parts by that for each (the second is at most 2^-8 of the first, the third of the
second), and each of the three additions of sums by 2^-24 of them; a result rounds
once, by half a step of its type.  Parts below 2^-126 may be flushed to zero."""
import pytest
import torch

from mkernel_amd import ops
from mkernel_amd.capi import MkError
from test_gpu_product import BF16, F32, F64, HALF, U, _labels, _vocab64, act64, d, near, randn

pytestmark = pytest.mark.gpu
TINY = 2.0 ** -125
PARTS = 1 + 2.0 ** -7


def _backward(M, K, N, act, db_dtype, dpre, pads=(0, 0, 0, 0), accumulate=False, seed=120):
    dC, A = randn(M, N, seed=seed, pad=pads[0]), randn(M, K, seed=seed + 1, pad=pads[1])
    B, pre = randn(K, N, seed=seed + 2, scale=N ** -0.5, pad=pads[2]), randn(M, N, seed=seed + 3, pad=pads[3])
    dB = randn(K, N, seed=seed + 4, dtype=db_dtype) if accumulate else None
    dbias = randn(N, seed=seed + 5, dtype=F32) if accumulate else None
    old = (d(dB), d(dbias)) if accumulate else (0.0, 0.0)
    got = ops.gemm_act_backward(dC, A, B, pre=pre, act=act, dB=dB, dbias=dbias, dB_dtype=db_dtype, accumulate=accumulate,
                                dpre_dtype=dpre)
    g = d(dC) * act64(d(pre), act)[1]
    ge = 2.0 ** -20 * (1 + d(pre).abs()) * d(dC).abs() + U * g.abs()
    return dC, A, B, pre, g, ge, old, got


SHAPES = [(1, 1, 1), (1, 64, 72), (3, 40, 9), (65, 130, 33), (300, 264, 520), (700, 97, 101), (1030, 512, 256)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("db_dtype,dpre", [(F32, None), (F32, F32), (BF16, F32)], ids=["f32", "f32-f32", "bf16-f32"])
def test_gemm_act_backward(shape, act, accumulate, db_dtype, dpre):
    M, K, N = shape
    pads = [(0, 0, 0, 0), (3, 1, 7, 5)][(M + N) % 2]
    dC, A, B, pre, g, ge, (dB0, db0), (dA, dB, dbias) = _backward(M, K, N, act, db_dtype, dpre, pads, accumulate)
    want = g @ d(B).t()
    if dpre is F32:
        tol = (ge + PARTS * (N + 4) * U * g.abs() + TINY) @ d(B).abs().t() + TINY
        near(dA, want, HALF[BF16] * (want.abs() + tol) + tol)
    else:
        gb = ge + 2.0 ** -8 * (g.abs() + ge)
        tol = (gb + N * U * g.abs()) @ d(B).abs().t()
        near(dA, want, HALF[BF16] * (want.abs() + tol) + tol)
    want, tol = d(A).t() @ g, d(A).abs().t() @ (ge + PARTS * (M + 4) * U * g.abs() + TINY) + TINY
    if accumulate:
        want, tol = want + dB0, tol + 3 * U * (want.abs() + dB0.abs())
    near(dB, want, HALF[db_dtype] * (want.abs() + tol) + tol)
    want, tol = g.sum(0) + db0, (ge + (M + 2) * U * g.abs()).sum(0)
    near(dbias, want, tol + 2 * U * (want.abs() + (db0.abs() if accumulate else 0.0)))


def test_gemm_act_backward_choices():
    """bfloat16 for a float32 dB is one product of the rounded dpre; dA's own type decides for dA; relu has no rest."""
    M, K, N = 200, 96, 136
    dC, A, B, pre, *_ = _backward(M, K, N, "silu", BF16, BF16)
    one = ops.gemm_act_backward(dC, A, B, pre=pre, act="silu", dB_dtype=F32, dpre_dtype=BF16)
    by_type = ops.gemm_act_backward(dC, A, B, pre=pre, act="silu", dB_dtype=F32)
    low = ops.gemm_act_backward(dC, A, B, pre=pre, act="silu")
    assert torch.equal(one[0], low[0]) and torch.equal(by_type[0], low[0]) and torch.equal(one[1].to(BF16), low[1])
    assert not torch.equal(one[1], by_type[1])
    for act in ("none", "relu"):
        p = None if act == "none" else pre
        a, b = (ops.gemm_act_backward(dC, A, B, pre=p, act=act, dB_dtype=F32, dpre_dtype=t) for t in (BF16, F32))
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    with pytest.raises(ValueError, match="dpre_dtype"):
        ops.gemm_act_backward(dC, A, B, pre=pre, act="silu", dpre_dtype=torch.float16)


def test_gemm_act_backward_what_is_not_finite():
    """NaN and infinities stay in their row of dA and column of dB."""
    M, K, N = 40, 72, 33
    dC, A, B, pre = randn(M, N, seed=1), randn(M, K, seed=2), randn(K, N, seed=3), randn(M, N, seed=4)
    dC[3, 7], dC[5, 9] = float("nan"), float("inf")
    dA, dB, _ = ops.gemm_act_backward(dC, A, B, pre=pre, act="silu", dB_dtype=F32, dpre_dtype=F32)
    assert dA[3].isnan().all() and not dA[5].isfinite().any() and dB[:, 7].isnan().all() and dB[:, 9].isinf().all()
    rest = [i for i in range(M) if i not in (3, 5)]
    assert dA[rest].isfinite().all() and dB[:, [i for i in range(N) if i not in (7, 9)]].isfinite().all()


def test_gemm_act_backward_empty():
    pre, B = randn(0, 16, seed=1), randn(8, 16, seed=2)
    dA, dB, db = ops.gemm_act_backward(pre, randn(0, 8, seed=3), B, pre=pre, act="gelu", dB_dtype=F32, dpre_dtype=F32)
    assert dA.shape == (0, 8) and (dB == 0).all() and (db == 0).all()
    e = torch.empty(5, 0, dtype=BF16, device="cuda")
    dA, dB, db = ops.gemm_act_backward(e, randn(5, 8), B[:, :0], pre=e, act="gelu", dB_dtype=F32, dpre_dtype=F32)
    assert (dA == 0).all() and dB.shape == (8, 0) and db.shape == (0,)


# ---------------------------------------------------------------- vocabulary loss
def _check_vocab(T, H, V, x, W, labels, dloss, lse=None, begin=0, dx_dtype=F32, dw_dtype=F32, accumulate=False, piece=0, dl=None):
    lab = labels.cuda()
    on, here, at, z, mag, lse64, _ = _vocab64(x, W, labels, begin)
    if lse is None:
        lse = ops.vocab_loss(x, W, lab, vocab_begin=begin)["lse"]
    dW = randn(H, V, seed=130, dtype=dw_dtype) if accumulate else None
    before = d(dW) if accumulate else 0.0
    dx, dW = ops.vocab_loss_backward(x, W, lab, lse, dloss, vocab_begin=begin, dW=dW, dx_dtype=dx_dtype, dW_dtype=dw_dtype,
                                     accumulate=accumulate, piece_columns=piece, dl_dtype=dl)
    # of the lse that the call was given: its error is the forward call's
    far = torch.where(on[:, None], z - d(lse)[:, None], 0.0)
    p = torch.exp(far)
    w = torch.where(on, d(dloss), 0.0)[:, None]
    hot = torch.zeros(T, V, dtype=F64)
    hot[here.nonzero()[:, 0], at[here]] = 1.0
    g = (p - hot) * w
    # p by the error of its exponent, (the logit's, a rounding of the difference, and that of its product with log2 e)
    # and a step of its own; then the difference at the label, the division by the common scale and two products
    err = (H + 2) * U * mag
    ge = p * (err + (3 * far.abs().clamp(max=90) + 2) * U) * w.abs() + 4 * U * (g.abs() + hot * w.abs())
    tiny = TINY * (1 + w.abs())
    xs, w64 = torch.where(on[:, None], d(x), 0.0), d(W)
    want = g @ w64.t()
    n = 2.0 ** -8 * (g.abs() + ge) if dx_dtype is BF16 and dl is not F32 else 0.0
    tol = (ge + n + PARTS * (V + 24) * U * g.abs() + tiny) @ w64.abs().t() + TINY
    near(dx, want, HALF[dx_dtype] * (want.abs() + tol) + tol)
    want = xs.t() @ g
    n = 2.0 ** -8 * (g.abs() + ge) if dw_dtype is BF16 and dl is not F32 else 0.0
    tol = xs.abs().t() @ (ge + n + PARTS * (T + 4) * U * g.abs() + tiny) + TINY
    if accumulate:
        want, tol = want + before, tol + 3 * U * (want.abs() + before.abs())
    near(dW, want, HALF[dw_dtype] * (want.abs() + tol) + tol)
    return dx, dW


TYPES = [(F32, F32, None), (F32, BF16, None), (BF16, F32, None), (BF16, BF16, F32), (F32, F32, F32)]


@pytest.mark.parametrize("T,H,V,piece", [(1, 8, 1, 0), (3, 40, 17, 0), (33, 100, 515, 256), (64, 512, 2048, 512),
                                         (130, 257, 1003, 0), (300, 64, 777, 256)])
@pytest.mark.parametrize("dx_dtype,dw_dtype,dl", TYPES, ids=["f32-f32", "f32-bf16", "bf16-f32", "all", "f32-all"])
def test_vocab_loss_backward(T, H, V, piece, dx_dtype, dw_dtype, dl):
    labels = _labels(T, V, 131)
    x, W = randn(T, H, seed=132, pad=T % 2), randn(H, V, seed=133, scale=2 * H ** -0.5)
    if T > 2:
        labels[::3] = -100
        x[::3] = float("nan")
    dloss = randn(T, seed=134, dtype=F32)
    _check_vocab(T, H, V, x, W, labels, dloss, dx_dtype=dx_dtype, dw_dtype=dw_dtype, accumulate=T % 2 == 0, piece=piece, dl=dl)


def test_vocab_loss_backward_of_a_shard():
    T, H, V = 60, 80, 1000
    labels = _labels(T, V, 135)
    labels[7] = -100
    x, W = randn(T, H, seed=136), randn(H, V, seed=137, scale=0.3)
    lse, dloss = ops.vocab_loss(x, W, labels.cuda())["lse"], torch.full((T,), 1.0 / T, device="cuda")
    for lo, hi in ((0, 480), (480, V)):
        _check_vocab(T, H, hi - lo, x, W[:, lo:hi].contiguous(), labels, dloss, lse=lse, begin=lo, dw_dtype=BF16)


def test_vocab_loss_backward_of_distinct_dloss():
    """Three weights, a third of the tokens each: no group's labels are off by a common rounding."""
    T, H, V = 510, 64, 4000
    labels = _labels(T, V, 138)
    x, W = randn(T, H, seed=139), randn(H, V, seed=140, scale=0.3 * H ** -0.5)
    dloss = torch.tensor([1.0039, 1.0117, 1.9961], device="cuda").repeat(T // 3)
    _check_vocab(T, H, V, x, W, labels, dloss)
    _check_vocab(T, H, V, x, W, labels, dloss, piece=512, dx_dtype=BF16, dw_dtype=BF16, dl=F32)


def test_vocab_loss_backward_large():
    """256 x 256 and 128 x 128 tiles, three pieces: as exact as the product of float32 numbers (at sums of up to 8192,
    whose fp32 errors are 2^-14 at most and 2^-20 or so in the mean)."""
    T, H, V = 2100, 1030, 20005
    x, W = randn(T, H, seed=141), randn(H, V, seed=142, scale=2 * H ** -0.5)
    labels = _labels(T, V, 143).cuda()
    labels[::9] = -100
    dloss = torch.full((T,), 1.0 / T, device="cuda")
    lse = ops.vocab_loss(x, W, labels)["lse"]
    z = x.to(F64) @ W.to(F64)
    g = torch.exp(z - lse.to(F64)[:, None])
    on = labels >= 0
    g[on.nonzero()[:, 0], labels[on]] -= 1
    g *= torch.where(on, dloss, 0.0).to(F64)[:, None]
    want = g @ W.to(F64).t(), x.to(F64).t() @ g
    for types, most in ((dict(dx_dtype=F32, dW_dtype=F32), 2.0 ** -14), (dict(dl_dtype=F32), 2.0 ** -9),
                        (dict(dx_dtype=F32, dW_dtype=F32, dl_dtype=BF16), 2.0 ** -8)):
        got = ops.vocab_loss_backward(x, W, labels, lse, dloss, piece_columns=8192, **types)
        for a, b in zip(got, want):
            off = float((a.to(F64) - b).norm() / b.norm())
            assert off <= most, (types, off)


def test_vocab_loss_backward_choices():
    T, H, V = 100, 72, 600
    x, W, labels = randn(T, H, seed=144), randn(H, V, seed=145, scale=0.3), _labels(T, V, 146).cuda()
    lse, dloss = ops.vocab_loss(x, W, labels)["lse"], torch.full((T,), 1.0 / T, device="cuda")
    low = ops.vocab_loss_backward(x, W, labels, lse, dloss)
    one = ops.vocab_loss_backward(x, W, labels, lse, dloss, dx_dtype=F32, dW_dtype=F32, dl_dtype=BF16)
    mixed = ops.vocab_loss_backward(x, W, labels, lse, dloss, dW_dtype=F32)
    assert all(torch.equal(a.to(BF16), b) for a, b in zip(one, low))
    assert torch.equal(mixed[0], low[0]) and not torch.equal(mixed[1], one[1])
    with pytest.raises(ValueError, match="dl_dtype"):
        ops.vocab_loss_backward(x, W, labels, lse, dloss, dl_dtype=torch.float16)
    dx, dW = ops.vocab_loss_backward(x[:0], W, labels[:0], lse[:0], dloss[:0], dx_dtype=F32, dW_dtype=F32)
    assert dx.shape == (0, H) and (dW == 0).all()


def test_captured_calls_of_three_parts():
    """In a graph, replayed between eager calls of the same."""
    M, K, N = 200, 96, 136
    dC, A, B, pre, *_ = _backward(M, K, N, "silu", BF16, BF16)
    T, H, V = 100, 65, 600
    x, W, labels = randn(T, H, seed=147), randn(H, V, seed=148, scale=0.3), _labels(T, V, 149).cuda()
    lse, dloss = ops.vocab_loss(x, W, labels)["lse"], torch.full((T,), 1.0 / T, device="cuda")

    def calls():
        return [*ops.gemm_act_backward(dC, A, B, pre=pre, act="silu", dB_dtype=F32, dpre_dtype=F32),
                *ops.vocab_loss_backward(x, W, labels, lse, dloss, dx_dtype=F32, piece_columns=256, dl_dtype=F32)]

    want = calls()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = calls()
    for _ in range(5):
        for t in out:
            t.fill_(float("nan"))
        g.replay()
        eager = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(out, want, eager))
