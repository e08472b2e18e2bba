"""The products on tiles and cuts that the sizes of the other tests do not reach
(tests/test_product_tiles_host.py says which runs what): wide and tall tiles with
K in parts, and the vocabulary's epilogues on every tile, against 64 bits.

Tolerances as in test_gpu_product.py: n * 2^-24 * sum |products| for a sum of n
products, then half a step of the result's type; what goes through bf16 between
two products is off by 2^-8 of itself."""
import pytest
import torch

import test_gpu_product_large as large
from mkernel_amd import ops
from test_gpu_product_large import BF16, F32, F64, HALF, U, near, product, randn

pytestmark = pytest.mark.gpu

# M, K, N of the forward order, all of them cut: 64 x 128, the same behind whole rounds, 128 x 128, the same behind whole
FORWARD = [(33, 5631, 15478), (294, 7345, 13179), (970, 10143, 1003), (1538, 903, 10059)]
# K, M (the sum), N of dB: 128 x 128, 128 x 256 (64 x 64 where more follows than the plain result), 128 x 256 behind
# whole rounds (256 x 256), 64 x 128
RIGHT = [(66, 7590, 9140), (9906, 5521, 135), (13099, 1171, 1185), (282, 5516, 13615), (100, 6000, 3000)]
# T, H, V, columns of a piece (0: the library's choice, here all of them): statistics on 256 x 256 and logits' gradients
# on 256 x 256 and 128 x 128 (odd weights, laid out anew, and direct ones); 64 x 64, 128 x 128, 64 x 128 and 256 x 256
# in parts
VOCAB = [(2100, 1030, 32005, 8192), (2100, 1030, 32000, 8192), (100, 8192, 700, 0), (970, 10143, 1003, 0),
         (260, 8192, 1100, 0), (1219, 1722, 13145, 0)]


@pytest.mark.parametrize("M,K,N", FORWARD)
@pytest.mark.parametrize("plain", [True, False], ids=["plain", "all"])
def test_gemm_act(M, K, N, plain):
    large.test_gemm_act(M, K, N, plain)


@pytest.mark.parametrize("K,M,N", RIGHT)
@pytest.mark.parametrize("dtype,accumulate", [(BF16, False), (F32, False), (F32, True), (BF16, True)],
                         ids=["bf16", "f32", "f32+", "bf16+"])
def test_gemm_act_backward(K, M, N, dtype, accumulate):
    large.test_gemm_act_backward(K, M, N, dtype, accumulate)


@pytest.mark.parametrize("T,H,V,piece", VOCAB)
def test_vocab_loss(T, H, V, piece):
    """Labels on both sides of every piece's edges, the first and the last; ignored tokens whose rows are NaN."""
    x, W = randn(T, H, seed=18), randn(H, V, seed=19, scale=2 * H ** -0.5)
    labels = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(20), device="cuda")
    edges = [0, V - 1] + [c for e in range(piece, V, piece or V) for c in (e - 1, e) if e]
    labels[1:1 + len(edges)] = torch.tensor(edges, device="cuda")
    off = torch.zeros(T, dtype=torch.bool, device="cuda")
    off[::7] = True
    off[1:1 + len(edges)] = False
    labels[off] = -100
    x[off] = float("nan")
    on = ~off
    r = ops.vocab_loss(x, W, labels)
    xs = torch.where(on[:, None], x, torch.zeros_like(x))
    z, err = product(xs, W)
    lse = torch.logsumexp(z, 1)
    # the logits' error, V / 64 + 100 roundings of sums of exponentials, the logarithm's
    tol = err.amax(1) + (V / 64 + 200) * U + 4 * U * lse.abs()
    target = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    for name, want, t in (("lse", lse, tol), ("target", target, err.amax(1)),
                          ("loss", lse - target, tol + err.amax(1) + 2 * U * lse.abs())):
        near(r[name], torch.where(on, want, 0.0), torch.where(on, t, 0.0) + 1e-300)
    dloss = randn(T, seed=21, dtype=F32)
    dx, dW = ops.vocab_loss_backward(x, W, labels, r["lse"], dloss, piece_columns=piece)
    p = torch.exp(z - lse[:, None])
    w = torch.where(on, dloss.to(F64), 0.0)[:, None]
    pe = p * (err + tol[:, None] + (6 * (z - lse[:, None]).abs().clamp(max=90) + 4) * U) * w.abs()
    p.scatter_add_(1, labels.clamp(min=0)[:, None], torch.full((T, 1), -1.0, dtype=F64, device="cuda"))
    dl = p * w
    de = pe + 2.0 ** -8 * (dl.abs() + pe) + 2.0 ** -126 * (1 + w.abs())
    want, tol = dl @ W.to(F64).t(), (de + (V + 8) * U * dl.abs()) @ W.to(F64).abs().t()
    near(dx, want, HALF[BF16] * (want.abs() + tol) + tol + 1e-300)
    want, tol = xs.to(F64).t() @ dl, xs.to(F64).abs().t() @ (de + (T + 1) * U * dl.abs())
    near(dW, want, HALF[BF16] * (want.abs() + tol) + tol)


@pytest.mark.parametrize("T,H,V", [(3, 40, 17), (33, 100, 515), (130, 257, 1003), (600, 72, 9000), (2100, 64, 32000)])
def test_vocab_loss_of_infinite_logits(T, H, V):
    """log sum exp is inf where a logit is (the loss too, unless it is the label's own), and -inf where all are."""
    x, W = randn(T, H, seed=22), randn(H, V, seed=23)
    W[0], W[1] = W[0].abs() + 1, -(W[1].abs() + 1)
    W[2] = 1.0
    W[2, V // 2:] = -1.0
    labels = torch.arange(T, device="cuda") % (V // 2) + V // 2
    x[0, 0], x[1, 1], x[2, 2] = float("inf"), float("inf"), float("inf")  # all logits inf; all -inf; some of both
    r = ops.vocab_loss(x, W, labels)
    inf = float("inf")
    assert r["lse"][:3].tolist() == [inf, -inf, inf] and r["target"][:3].tolist() == [inf, -inf, -inf]
    assert r["loss"][:2].isnan().all() and r["loss"][2] == inf
    assert r["lse"][3:].isfinite().all() and r["loss"][3:].isfinite().all()
    rest = ops.vocab_loss(x[3:], W, labels[3:])["lse"] if T > 3 else None
    assert rest is None or torch.allclose(rest, r["lse"][3:], rtol=1e-5, atol=1e-5)


def test_vocab_loss_of_a_long_batch():
    """More tokens than 128 MB of dl have room for at 256 columns, the least that a piece has."""
    T, H, V = 300001, 24, 700
    x, W = randn(T, H, seed=24), randn(H, V, seed=25, scale=2 * H ** -0.5)
    labels = torch.arange(T, device="cuda") * 7919 % V
    labels[::5] = -100
    on = labels >= 0
    r = ops.vocab_loss(x, W, labels)
    z, err = product(x, W)
    lse = torch.logsumexp(z, 1)
    tol = err.amax(1) + (V / 64 + 200) * U + 4 * U * lse.abs()
    near(r["lse"], torch.where(on, lse, 0.0), torch.where(on, tol, 0.0) + 1e-300)
    dloss = torch.full((T,), 1.0 / T, device="cuda")
    dx, dW = ops.vocab_loss_backward(x, W, labels, r["lse"], dloss)
    p = torch.exp(z - lse[:, None])
    w = torch.where(on, dloss.to(F64), 0.0)[:, None]
    pe = p * (err + tol[:, None] + (6 * (z - lse[:, None]).abs().clamp(max=90) + 4) * U) * w
    p.scatter_add_(1, labels.clamp(min=0)[:, None], torch.full((T, 1), -1.0, dtype=F64, device="cuda"))
    dl = p * w
    de = pe + 2.0 ** -8 * (dl.abs() + pe) + 2.0 ** -126
    want, tol = dl @ W.to(F64).t(), (de + (V + 8) * U * dl.abs()) @ W.to(F64).abs().t()
    near(dx, want, HALF[BF16] * (want.abs() + tol) + tol + 1e-300)
    want, tol = x.to(F64).t() @ dl, x.to(F64).abs().t() @ (de + (T + 1) * U * dl.abs())
    near(dW, want, HALF[BF16] * (want.abs() + tol) + tol)
