"""The products at sizes where every tile, a last round in parts and both kinds
of groups run (tests/test_product_host.py says which runs what), against 64 bits
on the GPU; streams, graphs and the expert layer's training step as it is used.

Tolerances as in test_gpu_product.py: n * 2^-24 * sum |products| for a sum of n
products, then half a step of the result's type."""
import pytest
import torch

from mkernel_amd import ops
from mkernel_amd.capi import MkError

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U}


def randn(*shape, seed=0, scale=1.0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)


def near(got, want, tol):
    off = (got.to(F64) - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, " \
                          f"worst {float((off / tol).max())} of the tolerance"


def product(a, b):
    """a @ b and the bound of its fp32 sums' error, in 64 bits."""
    a, b = a.to(F64), b.to(F64)
    return a @ b, (a.shape[1] + 2) * U * (a.abs() @ b.abs())


# M, K, N
FORWARD = [(4096, 264, 4096), (4100, 1001, 4099), (4608, 2048, 4608), (9000, 4104, 2100), (1100, 5000, 2050),
           (2500, 333, 700), (700, 3000, 600), (40, 4096, 600), (20, 4096, 600), (2, 1000, 16500), (1, 3001, 515)]


@pytest.mark.parametrize("M,K,N", FORWARD)
@pytest.mark.parametrize("plain", [True, False], ids=["plain", "all"])
def test_gemm_act(M, K, N, plain):
    A, B = randn(M, K, seed=1), randn(K, N, seed=2, scale=K ** -0.5)
    x, err = product(A, B)
    if plain:
        near(ops.gemm_act(A, B), x, HALF[BF16] * (x.abs() + err) + err)
        return
    bias, res = randn(N, seed=3), randn(M, N, seed=4, dtype=F32)
    pre = torch.empty(M, N, dtype=BF16, device="cuda")
    got = ops.gemm_act(A, B, bias=bias, act="silu", residual=res, pre=pre, out_dtype=F32)
    x, err = x + bias.to(F64), err + 2 * U * (x.abs() + bias.to(F64).abs())
    near(pre, x, HALF[BF16] * (x.abs() + err) + err)
    y = x * torch.sigmoid(x) + res.to(F64)
    tol = 1.13 * err + 2.0 ** -20 * x.abs() + 4 * U * (y.abs() + res.to(F64).abs()) + 1e-37
    near(got, y, tol)


# K, M (the sum), N: rows and columns of dB
RIGHT = [(4096, 300, 4096), (3000, 3000, 2000), (1000, 5000, 500), (700, 60, 3000), (4608, 3000, 4608), (200, 9000, 200)]


@pytest.mark.parametrize("K,M,N", RIGHT)
@pytest.mark.parametrize("dtype,accumulate", [(BF16, False), (F32, False), (F32, True), (BF16, True)],
                         ids=["bf16", "f32", "f32+", "bf16+"])
def test_gemm_act_backward(K, M, N, dtype, accumulate):
    dC, A, B = randn(M, N, seed=5), randn(M, K, seed=6), randn(K, N, seed=7, scale=N ** -0.5)
    old = randn(K, N, seed=8, dtype=dtype) if accumulate else None
    db0 = randn(N, seed=9, dtype=F32) if accumulate else None
    dA, dB, db = ops.gemm_act_backward(dC, A, B, dB=None if old is None else old.clone(),
                                       dbias=None if db0 is None else db0.clone(), dB_dtype=dtype, accumulate=accumulate)
    x, err = product(dC, B.t())
    near(dA, x, HALF[BF16] * (x.abs() + err) + err)
    x, err = product(A.t(), dC)
    s, serr = dC.to(F64).sum(0), (M + 2) * U * dC.to(F64).abs().sum(0)
    if accumulate:
        x, err = x + old.to(F64), err + U * (x.abs() + old.to(F64).abs())
        s, serr = s + db0.to(F64), serr + U * (s.abs() + db0.to(F64).abs())
    near(dB, x, HALF[dtype] * (x.abs() + err) + err)
    near(db, s, serr + U * s.abs())


def _groups(counts, R, K, seed):
    A = randn(R, K, seed=seed)
    ends = torch.tensor(counts).clamp(min=0).cumsum(0).clamp(max=R).tolist()
    rows = list(zip([0] + ends[:-1], ends))
    A[ends[-1]:] = float("nan")
    return A, torch.tensor(counts, dtype=torch.int32, device="cuda"), rows


# counts, R, K, N: rows tiles of 256 (whole, of up to 128 rows, halved over the XCDs), 128 and 64
RAGGED = [([1800, 3, 0, 900, 128, 129, 700], 4000, 1024, 2048), ([256, 255, 257, 0, 1, 511, 1200, 2600], 6000, 1000, 4096),
          ([300, 700, 0, 100, 200, 150], 1500, 512, 2048), ([20] * 70 + [900], 2400, 264, 520)]


@pytest.mark.parametrize("case", range(len(RAGGED)))
@pytest.mark.parametrize("mode", [0, 1])
def test_moe_ragged_gemm(case, mode):
    counts, R, K, N = RAGGED[case]
    A, n, rows = _groups(counts, R, K, 10)
    W = randn(len(counts), K, N, seed=11, scale=K ** -0.5)
    h = torch.full((R, N), 5.0, dtype=BF16, device="cuda") if mode else None
    out = torch.full((R, N // 2 if mode else N), 3.0, dtype=BF16, device="cuda")
    ops.moe_ragged_gemm(A, W, n, mode=mode, out=out, h=h)
    for e, (lo, hi) in enumerate(rows):
        x, err = product(A[lo:hi], W[e])
        if mode == 0:
            near(out[lo:hi], x, HALF[BF16] * (x.abs() + err) + err)
            continue
        near(h[lo:hi], x, HALF[BF16] * (x.abs() + err) + err)
        g, u, eg, eu = x[:, :N // 2], x[:, N // 2:], err[:, :N // 2], err[:, N // 2:]
        y = g * torch.sigmoid(g) * u
        tol = (1.13 * eg + 2.0 ** -20 * g.abs()) * (u.abs() + eu) + g.abs() * eu + 2 * U * y.abs()
        near(out[lo:hi], y, HALF[BF16] * (y.abs() + tol) + tol)
    last = rows[-1][1]
    assert (out[last:] == 3).all() and (h is None or (h[last:] == 5).all())


@pytest.mark.parametrize("case", range(len(RAGGED)))
@pytest.mark.parametrize("swiglu", [False, True])
def test_moe_ragged_dgrad(case, swiglu):
    counts, R, K, N = RAGGED[case]
    dy, n, rows = _groups(counts, R, N, 12)
    W = randn(len(counts), K, N, seed=13, scale=N ** -0.5)
    h = randn(R, 2 * K, seed=14) if swiglu else None
    out = torch.full((R, 2 * K if swiglu else K), 3.0, dtype=BF16, device="cuda")
    ops.moe_ragged_gemm_dgrad(dy, W, n, h=h, out=out)
    for e, (lo, hi) in enumerate(rows):
        x, err = product(dy[lo:hi], W[e].t())
        if not swiglu:
            near(out[lo:hi], x, HALF[BF16] * (x.abs() + err) + err)
            continue
        g, u = h[lo:hi, :K].to(F64), h[lo:hi, K:].to(F64)
        s = torch.sigmoid(g)
        for got, f, fe in ((out[lo:hi, :K], u * s * (1 + g * (1 - s)), 2.0 ** -20 * u.abs() * (1 + g.abs())),
                           (out[lo:hi, K:], g * s, 2.0 ** -20 * g.abs())):
            want = x * f
            tol = err * (f.abs() + fe) + x.abs() * fe + 4 * U * want.abs()
            near(got, want, HALF[BF16] * (want.abs() + tol) + tol)
    assert (out[rows[-1][1]:] == 3).all()


# counts, R, K, N of dW
RAGGED_W = [([400, 3, 0, 200, 17, 380], 1000, 2048, 4000), ([20, 0, 31, 64] * 5, 600, 1000, 520),
            ([700, 300, 1500, 500], 3000, 256, 256), ([5000, 0, 4000, 0], 9000, 2048, 2048), ([50, 60, 40, 0, 70, 80], 300, 100, 100)]


@pytest.mark.parametrize("case", range(len(RAGGED_W)))
@pytest.mark.parametrize("dtype,accumulate", [(BF16, False), (F32, False), (F32, True)], ids=["bf16", "f32", "f32+"])
def test_moe_ragged_wgrad(case, dtype, accumulate):
    counts, R, K, N = RAGGED_W[case]
    A, n, rows = _groups(counts, R, K, 15)
    dy = randn(R, N, seed=16)
    dy[rows[-1][1]:] = float("inf")
    old = randn(len(counts), K, N, seed=17, dtype=dtype) if accumulate else None
    out = old.clone() if accumulate else torch.full((len(counts), K, N), 9.0, dtype=dtype, device="cuda")
    ops.moe_ragged_gemm_wgrad(A, dy, n, out=out, accumulate=accumulate)
    for e, (lo, hi) in enumerate(rows):
        x, err = product(A[lo:hi].t(), dy[lo:hi])
        if accumulate:
            x, err = x + old[e].to(F64), err + U * (x.abs() + old[e].to(F64).abs())
        near(out[e], x, HALF[dtype] * (x.abs() + err) + err)


@pytest.mark.parametrize("T,H,V,piece", [(2048, 512, 9000, 0), (1500, 1001, 5003, 2048), (600, 256, 70000, 0)])
def test_vocab_loss(T, H, V, piece):
    x, W = randn(T, H, seed=18), randn(H, V, seed=19, scale=2 * H ** -0.5)
    labels = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(20), device="cuda")
    labels[::7] = -100
    x[::7] = float("nan")
    on = labels != -100
    r = ops.vocab_loss(x, W, labels)
    xs = torch.where(on[:, None], x, torch.zeros_like(x))
    z, err = product(xs, W)
    lse = torch.logsumexp(z, 1)
    # the logits' error, V / 64 + 100 roundings of sums of exponentials, the logarithm's
    tol = err.amax(1) + (V / 64 + 200) * U + 4 * U * lse.abs()
    target = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    for name, want, t in (("lse", lse, tol), ("target", target, err.amax(1)), ("loss", lse - target, tol + err.amax(1) + 2 * U * lse.abs())):
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


# ---------------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits():
    """Weights and results whose later elements lie 4 GiB and more behind the first: whatever is cut to 32 bits lands
    in the first part, which holds other values."""
    E, K, N = 5, 8192, 65536  # 5 GiB in all
    W = torch.zeros(E, K, N, dtype=BF16, device="cuda")
    W[4] = 1.0
    W[4, :, 1::2] = -1.0
    n = torch.tensor([0, 0, 3, 0, 5], dtype=torch.int32, device="cuda")
    A = torch.ones(8, K, dtype=BF16, device="cuda")
    out = ops.moe_ragged_gemm(A, W, n)
    assert (out[:3] == 0).all() and (out[3:, 0::2] == K).all() and (out[3:, 1::2] == -K).all()
    dA = ops.moe_ragged_gemm_dgrad(torch.ones(8, N, dtype=BF16, device="cuda"), W, n)
    assert (dA == 0).all()
    W[4] = 1.0
    dA = ops.moe_ragged_gemm_dgrad(torch.ones(8, N, dtype=BF16, device="cuda"), W, n)
    assert (dA[:3] == 0).all() and (dA[3:] == N).all()
    W.fill_(7.0)
    ops.moe_ragged_gemm_wgrad(A, torch.ones(8, N, dtype=BF16, device="cuda"), n, out=W)
    for e, v in enumerate([0, 0, 3, 0, 5]):
        assert (W[e] == v).all(), e
    del W, out, dA
    # one row block far behind the first, columns of a wider matrix
    M = 40000
    wide = torch.zeros(M, 60000, dtype=BF16, device="cuda")  # 4.5 GiB
    wide[-1, -64:] = 1.0
    B = torch.ones(64, 48, dtype=BF16, device="cuda")
    got = ops.gemm_act(wide[:, -64:], B)
    assert (got[-1] == 64).all() and (got[:-1] == 0).all()
    ops.gemm_act(torch.ones(M, 16, dtype=BF16, device="cuda"), torch.ones(16, 72, dtype=BF16, device="cuda"), out=wide[:, 59000:59072])
    assert (wide[:, 59000:59072] == 16).all() and (wide[:, :59000].amax() == 0) and (wide[:, 59072:-64].amax() == 0)


# ---------------------------------------------------------------- streams and graphs
def _calls():
    """Calls that cut K, lay operands out anew and use the workspace, with fixed inputs; each returns its results."""
    A, B = randn(20, 4096, seed=30), randn(4096, 600, seed=31)
    Ao, Bo = randn(70, 1001, seed=32), randn(1001, 333, seed=33)
    dC = randn(300, 520, seed=34)
    A2, B2, pre = randn(300, 264, seed=35), randn(264, 520, seed=36), randn(300, 520, seed=37)
    n = torch.tensor([5, 0, 70, 33], dtype=torch.int32, device="cuda")
    X, W = randn(120, 96, seed=38), randn(4, 96, 130, seed=39)
    x, V = randn(200, 65, seed=40), randn(65, 515, seed=41)
    labels = torch.randint(0, 515, (200,), generator=torch.Generator(device="cuda").manual_seed(42), device="cuda")
    dloss = randn(200, seed=43, dtype=F32)

    def vocab():
        r = ops.vocab_loss(x, V, labels)
        return [r["loss"], r["lse"], *ops.vocab_loss_backward(x, V, labels, r["lse"], dloss)]

    return [lambda: [ops.gemm_act(A, B, act="gelu")], lambda: [ops.gemm_act(Ao, Bo)],
            lambda: list(ops.gemm_act_backward(dC, A2, B2, pre=pre, act="silu")),
            lambda: [ops.moe_ragged_gemm(X, W, n)[:108], ops.moe_ragged_gemm_wgrad(X, ops.moe_ragged_gemm(X, W, n), n)], vocab]


def test_repeats_bit_for_bit_on_any_stream():
    calls = _calls()
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append([f() for f in calls])
        torch.cuda.synchronize()
        for g in got:
            for a, b in zip(g, want):
                assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_graphs_replay_beside_each_other_and_eager_calls():
    calls = _calls()
    want = [f() for f in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([f() for f in calls])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for r in range(6):
        for o in outs:
            for a in o:
                for t in a:
                    t.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        for got in (*outs, eager):
            for a, b in zip(got, want):
                assert all(torch.equal(u, v) for u, v in zip(a, b)), r


def test_other_current_device_and_refusals():
    A, B = randn(8, 64), randn(64, 32)
    for bad in (lambda: ops.gemm_act(A.float(), B), lambda: ops.gemm_act(A, B.cpu()), lambda: ops.gemm_act(A, B[:32]),
                lambda: ops.gemm_act(A, B, act="tanh"), lambda: ops.gemm_act(A, B, bias=B[0, :16]),
                lambda: ops.gemm_act(A, B, residual=randn(8, 33)), lambda: ops.gemm_act(A, B, out_dtype=torch.float16),
                lambda: ops.gemm_act(A, B.t()), lambda: ops.gemm_act(A[:, ::2], B[:32]),
                lambda: ops.gemm_act_backward(randn(8, 32), A, B, act="relu"),
                lambda: ops.gemm_act_backward(randn(8, 32), A, B, accumulate=True),
                lambda: ops.moe_ragged_gemm(A, randn(2, 64, 32), torch.tensor([1, 2], device="cuda")),
                lambda: ops.moe_ragged_gemm(A, randn(2, 64, 33), torch.zeros(2, dtype=torch.int32, device="cuda"), mode=1),
                lambda: ops.moe_ragged_gemm(A, randn(2, 64, 32), torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: ops.moe_ragged_gemm_wgrad(A, randn(7, 32), torch.zeros(2, dtype=torch.int32, device="cuda")),
                lambda: ops.vocab_loss(A, B, torch.zeros(8, device="cuda")),
                lambda: ops.vocab_loss(A, B, torch.zeros(7, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    labels, lse = torch.zeros(8, dtype=torch.int64, device="cuda"), torch.zeros(8, device="cuda")
    for bad in (lambda: ops.gemm_act(A, B, out=A[:, :32]), lambda: ops.gemm_act(A, B, pre=B[:8]),
                lambda: ops.gemm_act(A, B, residual=B[:8], out=B[1:9]),
                lambda: ops.vocab_loss_backward(A, B, labels, lse, lse, piece_columns=100),
                lambda: ops.vocab_loss_backward(A, B, labels, lse, lse, dx=A),
                lambda: ops.vocab_loss(A, B, labels, vocab_begin=-1)):
        with pytest.raises(MkError):
            bad()


def test_slopes_of_far_arguments():
    """dpre = act'(pre) at arguments whose powers leave fp32: 0 or 1 there, for every activation."""
    pre = torch.tensor([[-3e38, -1e30, -1e20, -1e10, -300.0, -40.0, 40.0, 300.0, 1e10, 1e20, 1e30, 3e38]]).to(BF16).cuda()
    n = pre.shape[1]
    one = torch.ones(1, n, dtype=BF16, device="cuda")
    want = (pre > 0).float()[0]
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        db = ops.gemm_act_backward(one, one[:, :1], torch.zeros(1, n, dtype=BF16, device="cuda"), pre, act)[2]
        # -40 e^-40 is the largest of what is not 0; at 1 a reciprocal (a step) and three roundings
        assert (db - want).abs().le(2e-16 + 5 * U * want).all(), (act, db)


def test_two_threads_on_one_stream():
    """Calls whose operands are laid out anew in the workspace, from two threads at once."""
    import threading
    A, B = randn(300, 2811), [randn(2811, 205, seed=s) for s in (1, 2)]
    want = [ops.gemm_act(A, b) for b in B]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def work(i):
        start.wait()
        for _ in range(200):
            got[i].append(ops.gemm_act(A, B[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert len(g) == 200 and all(torch.equal(x, w) for x in g)


# ---------------------------------------------------------------- a training step of the expert layer
@pytest.mark.parametrize("row_block", [1, 128])
def test_expert_layer_training_step(row_block):
    """Router with balance loss -> index build -> permute -> products -> combine -> projection -> vocabulary loss, and
    all the way back, against 64 bits and autograd of the formulas at the same rounded intermediate values' scale."""
    T, H, I, E, k, V = 192, 128, 96, 8, 2, 300
    x = randn(T, H, seed=50)
    router = randn(H, E, seed=51, scale=H ** -0.5)
    w1, w2 = randn(E, H, 2 * I, seed=52, scale=H ** -0.5), randn(E, I, H, seed=53, scale=I ** -0.5)
    proj, bias = randn(H, H, seed=54, scale=H ** -0.5), randn(H, seed=55, dtype=F32, scale=0.1)
    head = randn(H, V, seed=56, scale=H ** -0.5)
    labels = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(57), device="cuda")
    labels[5] = -100
    dloss = torch.full((T,), 1.0 / T, device="cuda")

    # forward
    logits = ops.gemm_act(x, router, out_dtype=F32)
    r = ops.moe_route_balance(logits, k, 0.01)
    t = ops.moe_build_indices_dev(r["ids"], r["gates"], 0, E, row_block=row_block)
    rows = ops.moe_permute(x, t["pull_indices"], torch.empty(t["R_pad"], H, dtype=BF16, device="cuda"))
    n = t["padded_tokens_per_expert"]
    h = torch.empty(t["R_pad"], 2 * I, dtype=BF16, device="cuda")
    act = ops.moe_ragged_gemm(rows, w1, n, mode=1, h=h)
    ye = ops.moe_ragged_gemm(act, w2, n)
    y = ops.moe_combine(ye, t["row_weight"], t["owner_offset"], t["slot_to_row"], torch.empty(T, H, dtype=BF16, device="cuda"))
    pre = torch.empty(T, H, dtype=BF16, device="cuda")
    z = ops.gemm_act(y, proj, bias=bias, act="gelu", residual=x, pre=pre)
    loss = ops.vocab_loss(z, head, labels)
    # back
    dz, dhead = ops.vocab_loss_backward(z, head, labels, loss["lse"], dloss)
    dy, dproj, dbias = ops.gemm_act_backward(dz, y, proj, pre=pre, act="gelu")
    if row_block == 128:
        rb = t["rb_rows"]
        R = t["R_pad"]
    else:  # every row is real: whole blocks of 128 for the combine's gradient
        R = -(-t["R_pad"] // 128) * 128
        rb = torch.full((R // 128,), 128, dtype=torch.int32, device="cuda")
    weight = torch.zeros(R, device="cuda")
    weight[:t["R_pad"]] = t["row_weight"]
    yep = torch.zeros(R, H, dtype=BF16, device="cuda")
    yep[:t["R_pad"]] = ye
    dye, dgates = ops.moe_combine_backward(dy, yep, r["ids"], weight, t["owner_offset"], t["slot_to_row"], rb, 0, E)
    dw2 = ops.moe_ragged_gemm_wgrad(act, dye[:t["R_pad"]], n, out_dtype=F32)
    dh = ops.moe_ragged_gemm_dgrad(dye[:t["R_pad"]], w2, n, h=h)
    dw1 = ops.moe_ragged_gemm_wgrad(rows, dh, n, out_dtype=F32)
    drows = ops.moe_ragged_gemm_dgrad(dh, w1, n)
    ones = torch.ones_like(t["row_weight"])
    dx = ops.moe_combine(drows, ones, t["owner_offset"], t["slot_to_row"], torch.empty(T, H, device="cuda"))
    dlogits = ops.moe_route_backward(logits, r["ids"], dgates=dgates, dloss=torch.ones(1, device="cuda"),
                                     counts=r["counts"], tokens=r["tokens"], coef=0.01)
    dxr, drouter, _ = ops.gemm_act_backward(dlogits.to(BF16), x, router, need_dbias=False, dB_dtype=F32)

    # the same in 64 bits
    p = [v.detach().to(F64).requires_grad_() for v in (x, router, w1, w2, proj, bias, head)]
    X, Rt, W1, W2, P, Bs, Hd = p
    lg = X @ Rt
    ids = r["ids"].long()
    g = torch.softmax(lg.gather(1, ids), 1)
    Y = torch.zeros(T, H, dtype=F64, device="cuda")
    for e in range(E):
        tok, j = (ids == e).nonzero(as_tuple=True)
        a = X[tok] @ W1[e]
        Y = Y.index_add(0, tok, (torch.nn.functional.silu(a[:, :I]) * a[:, I:]) @ W2[e] * g[tok, j][:, None])
    Z = torch.nn.functional.gelu(Y @ P + Bs) + X
    L = torch.nn.functional.cross_entropy(Z @ Hd, labels, reduction="none", ignore_index=-100)
    probs = torch.softmax(lg, 1)
    f = torch.bincount(ids.flatten(), minlength=E).to(F64)
    total = (L * dloss).sum() + 0.01 * E / (k * T ** 2) * (f * probs.sum(0)).sum()
    grads = torch.autograd.grad(total, p)
    # each value went through bf16 a few times on its way, so it is off by a few times 2^-9 of the whole in the mean
    def rel(a, b):
        return float((a.to(F64) - b).norm() / b.norm())
    assert rel(loss["loss"], L.detach()) < 0.01 and loss["loss"][5] == 0
    for name, got, want in (("head", dhead, grads[6]), ("proj", dproj, grads[4]), ("bias", dbias, grads[5]),
                            ("w2", dw2, grads[3]), ("w1", dw1, grads[2]), ("router", drouter, grads[1]),
                            ("x", dx.to(F64) + dxr + dz, grads[0])):
        assert rel(got, want) < 0.03, (name, rel(got, want))
