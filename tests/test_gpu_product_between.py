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
from test_gpu_product import BF16, F32, F64, HALF, U, act64, d, near, randn

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
