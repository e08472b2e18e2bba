"""Which tile and cut the GPU tests' products run on, by epilogue: the host's
choice, compiled with the system C++ compiler."""
import test_gpu_product as small
import test_gpu_product_large as large
import test_gpu_product_tiles as tiles
from test_product_host import TILE32, TILE64, TILE64W, TILE128, TILE128W, TILE256, plans  # noqa: F401

CUT, WHOLE = True, False


def _vocab(plans, T, H, V, piece):
    """(tile, cut) of the statistics and of the logits' gradients."""
    piece = piece or V
    stats = plans(T, V, H)
    return ((stats[0], stats[1] > 1), {(t, s > 1) for t, s, _, _ in (plans(T, min(piece, V - c), H) for c in range(0, V, piece))})


def test_products_in_parts(plans):  # noqa: F811
    """Every tile with its K in parts: forward, and of weight gradients, plain and with more to follow."""
    for plain in (0, 1):
        got = {plans(M, N, K, plain=plain)[:2] + (plans(M, N, K, plain=plain)[3] > 0,) for M, K, N in small.SHAPES + large.FORWARD + tiles.FORWARD}
        cut = {(t, whole) for t, s, whole in got if s > 1}
        assert cut >= {(TILE32, False), (TILE64, False), (TILE64W, False), (TILE64W, True), (TILE128, False),
                       (TILE128, True), (TILE256, True)}
    for M, K, N in tiles.FORWARD:
        assert all(plans(M, N, K, plain=p)[1] > 1 for p in (0, 1))
    for plain, want in ((0, {TILE64, TILE64W, TILE128, TILE256}), (1, {TILE64W, TILE128, TILE128W})):
        right = [plans(K, N, M, right=1, plain=plain) for K, M, N in [(K, M, N) for M, K, N in small.GRAD_SHAPES] + large.RIGHT + tiles.RIGHT]
        assert {t for t, s, _, _ in right if s > 1} >= want
        if plain:  # 128 x 256: all of the result in parts, and behind whole rounds
            assert {w > 0 for t, s, _, w in right if t == TILE128W and s > 1} == {False, True}


def test_vocabulary(plans):  # noqa: F811
    """Both of the vocabulary's epilogues on every tile, whole and in parts."""
    cases = ([(T, H, V, 0) for T, H, V in small.VOCAB] + [(2048, 512, 9000, 0), (1500, 1001, 5003, 2048), (600, 256, 70000, 0)]
             + tiles.VOCAB)
    stats, grads = {s for s, _ in (_vocab(plans, *c) for c in cases)}, set().union(*(g for _, g in (_vocab(plans, *c) for c in cases)))
    for got in (stats, grads):
        assert got >= {(t, cut) for t in (TILE64, TILE64W, TILE128, TILE256) for cut in (CUT, WHOLE)} | {(TILE32, WHOLE)}
    T, H, V, piece = tiles.VOCAB[0]
    assert V % 8 and V % 256 and len(range(0, V, piece)) > 2  # laid out anew piece by piece, a last tile that is not full
