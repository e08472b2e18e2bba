"""Products with 4-bit weights, dense and for routed experts, against 64-bit
plain forms.

Two kinds of input.  Whole numbers and scales that are powers of two make every
product and sum exact in fp32 (a group's sum stays below 128 * 3 * 143 * 2 <
2^24), so the result is the exact one rounded once: equal bits, whatever the
order of the sums.  Normal inputs: one rounding to bf16 (2^-8 of the value), and
fp32 roundings of a group's sums, at most 2 per product of magnitude up to 143
|x| s (the code's offset included) on a chain of a group's 2 * 128 products, and
one per group and wave sum."""
import numpy as np
import pytest
import torch

from mkernel_amd import capi, ops, workloads as wl

pytestmark = pytest.mark.gpu
D = torch.float64


def _say(*a):
    print("[case]", *a, flush=True)


def _weights(shape, group, seed, zeros, exact):
    g = torch.Generator().manual_seed(seed)
    *lead, K, N = shape
    gs = (*lead, (K + group - 1) // group, N)
    codes = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8)
    if exact:
        scales = 2.0 ** torch.randint(-3, 1, gs, generator=g)
    else:
        scales = (torch.rand(gs, generator=g) + 0.5) * K ** -0.5 / 4.6
    z = torch.randint(0, 16, gs, generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales.to(torch.bfloat16), z


def _dense(codes, scales, z, group):
    at = torch.arange(codes.shape[-2]) // group
    zz = 8.0 if z is None else z[..., at, :].to(D)
    return (codes.to(D) - zz) * scales[..., at, :].to(D)


def _pack(dev, w, group):
    return ops.w4_pack(w[0].to(dev), w[1].to(dev), group, zeros=None if w[2] is None else w[2].to(dev))


def _whole(shape, seed):
    return torch.randint(-3, 4, shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _bound(x, w, group, want):
    """2^-8 of the value, and 256 + ceil(K / 128) + 8 fp32 roundings of the sum of |x| 143 s."""
    s = w[1][..., torch.arange(w[0].shape[-2]) // group, :].to(D)
    mag = x.to(D).abs() @ (143.0 * s)
    n = 256 + (w[0].shape[-2] + 127) // 128 + 8
    return 2.0 ** -8 * want.abs() + n * 2.0 ** -24 * mag + 1e-37


SHAPES = [(1, 8, 1), (1, 128, 16), (1, 2048, 2048), (2, 136, 17), (5, 5608, 2811), (16, 1024, 100), (17, 264, 33),
          (33, 96, 50), (48, 520, 2064), (64, 3584, 512), (65, 1032, 70), (130, 384, 40), (1, 8192, 3584), (3, 16384, 64),
          (0, 64, 64), (4, 136, 50), (5, 264, 6168), (20, 136, 3090), (16, 392, 4090),
          (16, 136, 8210), (40, 1032, 1370), (33, 264, 8200),
          (130, 136, 4090), (17, 1032, 16400), (1000, 40, 300)]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gemm_exact(dev, M, K, N, group, zeros):
    _say("gemm_w4 exact", M, K, N, group, zeros)
    w = _weights((K, N), group, K + N, zeros, True)
    x = _whole((M, K), M)
    want = (x.to(D) @ _dense(*w, group)).float().to(torch.bfloat16)
    p = _pack(dev, w, group)
    assert torch.equal(ops.gemm_w4(x.to(dev), p).cpu(), want)
    # rows of wider matrices; what lies beside the result stays
    wide = torch.full((M, K + 24), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 8:8 + K] = x.to(dev)
    out = torch.full((M, N + 5), 3.0, dtype=torch.bfloat16, device=dev)
    if M > 1:
        got = ops.gemm_w4(wide[:, 8:8 + K], p, out=out[:, :N])
        assert torch.equal(got.cpu(), want) and bool((out[:, N:] == 3).all())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(1, 512, 200), (3, 256, 50), (5, 264, 40), (16, 512, 2064), (40, 256, 8210)])
def test_small_beside_large(dev, M, K, N, group, zeros):
    """Half of x odd numbers up to 3, half multiples of 32 up to 6144, all positive: a group's partial sums of
    x (16 + code) and x (16 + zero), codes and zeros up to 15, are whole numbers up to 31 * 64 * (6144 + 3) < 2^24,
    so nothing is rounded in fp32 and nothing of the small x may be missing from a float32 result; so the total,
    15 * 256 * 6147 at most in a sum over 512 rows, of codes that lie around the zero point."""
    _say("small beside large", M, K, N, group, zeros)
    g = torch.Generator().manual_seed(M + N)
    codes, scales, z = _weights((K, N), group, K + N, zeros, True)
    scales = torch.ones_like(scales)
    if zeros:
        z = torch.randint(6, 10, z.shape, generator=g, dtype=torch.uint8)
    x = 32.0 * torch.randint(160, 193, (M, K), generator=g)
    x[:, 1::2] = 2.0 * torch.randint(0, 2, (M, K // 2), generator=g) + 1
    assert torch.equal(x.to(torch.bfloat16).float(), x)
    w = _dense(codes, scales, z, group)
    for g0 in range(0, K, group):  # (the running total over groups)
        assert float((x[:, :g0 + group].to(D) @ w[:g0 + group]).abs().max()) < 2 ** 24
    want = x.to(D) @ w
    out = torch.empty((M, N), device=dev)
    ops.gemm_w4(x.to(torch.bfloat16).to(dev), _pack(dev, (codes, scales, z), group), out=out)
    assert torch.equal(out.cpu().to(D), want)
    E = 3  # the experts' product: one expert's rows, and the halves of a pair (the large and the small numbers)
    p = ops.w4_pack(*(t.expand(E, *t.shape).contiguous().to(dev) for t in (codes, scales)), group,
                    zeros=None if z is None else z.expand(E, *z.shape).contiguous().to(dev))
    A = torch.zeros((128, K))
    A[:M] = x
    one, rows = torch.tensor([1], dtype=torch.int32, device=dev), torch.tensor([M], dtype=torch.int32, device=dev)
    small = torch.zeros_like(A)
    small[:, 1::2] = A[:, 1::2]
    for a in (A, torch.cat([A - small, small], 1)):
        y = torch.zeros((128, N), device=dev)
        ops.moe_grouped_gemm_w4(a.to(torch.bfloat16).to(dev), p, y, one, rows)
        assert torch.equal(y[:M].cpu().to(D), want)


@pytest.mark.parametrize("M,K,N,group,zeros", [(1, 8192, 3584, 128, False), (1, 2048, 2048, 32, True), (7, 5608, 2811, 32, True),
                                               (64, 3584, 8192, 64, False), (16, 7168, 4096, 128, True), (100, 1000, 300, 64, False)])
def test_gemm_normal(dev, M, K, N, group, zeros):
    _say("gemm_w4 normal", M, K, N, group, zeros)
    w = _weights((K, N), group, 1, zeros, False)
    x = wl.randn_bf16((M, K), 2)
    want = x.to(D) @ _dense(*w, group)
    p = _pack(dev, w, group)
    got = ops.gemm_w4(x.to(dev), p)
    err = (got.cpu().to(D) - want).abs()
    assert bool((err <= _bound(x, w, group, want)).all())
    assert float(err.norm() / want.norm()) < 2.0 ** -8  # one rounding's norm, the fp32 sums' far below
    # a batch's rows do not depend on each other, nor a row on the batch's size (within a tile height)
    again = ops.gemm_w4(x.to(dev), p, out=torch.empty((M, N), device=dev))
    assert torch.equal(got, again.to(torch.bfloat16))
    x[0] = float("nan")
    bad = ops.gemm_w4(x.to(dev), p)
    assert torch.isnan(bad[0]).all() and torch.equal(bad[1:], got[1:])


@pytest.mark.parametrize("shape", [(200, 33), (3, 128, 48), (7, 64)])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize(dev, shape, group):
    """Scales and codes by the definition, bit by bit; the values within half a step of the weights."""
    _say("quantize", shape, group)
    W = wl.randn_bf16(shape, 3)
    W[..., 0] = 0
    codes, scales = (t.cpu() for t in ops.w4_quantize(W.to(dev), group))
    K = shape[-2]
    at = torch.arange(K) // group
    for g in range((K + group - 1) // group):
        most = W[..., at == g, :].float().abs().amax(-2)
        assert torch.equal(scales[..., g, :], (most / 7).to(torch.bfloat16))
    s = scales[..., at, :].float()
    q = torch.where(s > 0, W.float() / s, torch.zeros(1)).round().clamp(-8, 7) + 8
    assert torch.equal(codes.float(), q)
    # half a step of the code; the largest magnitudes lie up to 7 (1 + 2^-8) steps out
    back = (codes.float() - 8) * s
    assert bool(((back - W.float()).abs() <= s * (0.5 + 7 * 2 ** -8)).all())
    if len(shape) == 2 and K % 8 == 0:
        x = wl.randn_bf16((4, K), 4)
        want = x.to(D) @ back.to(D)
        got = ops.gemm_w4(x.to(dev), ops.w4_pack(codes.to(dev), scales.to(dev), group)).cpu().to(D)
        assert bool(((got - want).abs() <= _bound(x, (codes, scales), group, want)).all())


def test_quantize_not_finite(dev):
    """A NaN makes its group's scale NaN, an infinity infinite; no other group's codes or scales change, and the
    weights they stand for are NaN and infinite where they were."""
    _say("quantize NaN and infinities")
    K, N, group = 136, 40, 64
    W = wl.randn_bf16((K, N), 3)
    codes, scales = ops.w4_quantize(W.to(dev), group)
    bad = W.clone()
    bad[3, 5], bad[70, 6], bad[71, 6], bad[135, 7], bad[0, 8] = (float(v) for v in ("nan", "inf", "-inf", "-inf", "nan"))
    bad[1, 8] = float("inf")
    c2, s2 = ops.w4_quantize(bad.to(dev), group)
    hit = torch.zeros((3, N), dtype=torch.bool)
    hit[0, 5] = hit[1, 6] = hit[2, 7] = hit[0, 8] = True
    rows = hit[torch.arange(K) // group].to(dev)
    assert torch.equal(c2[~rows], codes[~rows]) and torch.equal(s2[~hit.to(dev)], scales[~hit.to(dev)])
    back = (c2.float() - 8) * s2.float()[torch.arange(K, device=dev) // group]
    back = back.cpu()
    assert back[:64, 5].isnan().all() and back[:64, 8].isnan().all() and torch.isinf(s2[[1, 2], [6, 7]]).all()
    assert back[70, 6] == float("inf") and back[71, 6] == -float("inf") and back[135, 7] == -float("inf")
    # through a product: whole columns are not finite, others as they were
    x = wl.randn_bf16((3, K), 4).to(dev)
    got, want = ops.gemm_w4(x, ops.w4_pack(c2, s2, group)), ops.gemm_w4(x, ops.w4_pack(codes, scales, group))
    cols = hit.any(0).to(dev)
    assert not torch.isfinite(got[:, cols]).any() and torch.equal(got[:, ~cols], want[:, ~cols])


def _tables(dev, counts, E):
    """Tables of experts with these row counts, in 128-row blocks."""
    blocks = [(c + 127) // 128 for c in counts]
    rb_expert = torch.tensor([e for e in range(E) for _ in range(blocks[e])], dtype=torch.int32)
    rb_rows = torch.tensor([min(128, counts[e] - 128 * b) for e in range(E) for b in range(blocks[e])], dtype=torch.int32)
    return rb_expert.to(dev), rb_rows.to(dev)


@pytest.mark.parametrize("counts", [[1, 0, 3], [0, 0, 0], [16, 17, 64, 65], [128, 1, 129, 300], [2] * 7])
@pytest.mark.parametrize("K,N,mode,group,zeros", [(128, 64, 0, 128, False), (264, 96, 1, 32, False), (520, 50, 0, 64, True),
                                                  (1024, 544, 1, 128, True)])
def test_grouped(dev, counts, K, N, mode, group, zeros):
    _say("grouped_w4", counts, K, N, mode, group, zeros)
    E = len(counts)
    w = _weights((E, K, N), group, 5, zeros, True)
    p = _pack(dev, w, group)
    rb_expert, rb_rows = _tables(dev, counts, E)
    R, width = 128 * rb_expert.shape[0], N // 2 if mode else N
    A = _whole((R, K), 6)
    real = torch.zeros(R, dtype=torch.bool)
    for b, n in enumerate(rb_rows.tolist()):
        real[128 * b:128 * b + n] = True
    Ad = A.clone()
    Ad[~real] = float("nan")
    out = torch.full((R + 128, width), 7.0, dtype=torch.bfloat16, device=dev)
    ops.moe_grouped_gemm_w4(Ad.to(dev), p, out[:R], rb_expert, rb_rows, mode=mode)
    got = out.cpu()
    assert bool((got[R:] == 7).all()) and bool((got[:R][~real] == 7).all())
    dense = _dense(*w, group)
    for b in range(R // 128):
        rows = slice(128 * b, 128 * b + int(rb_rows[b]))
        h = A[rows].to(D) @ dense[int(rb_expert[b])]
        if mode == 0:
            assert torch.equal(got[rows], h.float().to(torch.bfloat16)), b
        else:
            want = torch.nn.functional.silu(h[:, :width]) * h[:, width:]
            # one rounding, and 8 fp32 roundings of the SwiGLU (of exact sums)
            assert torch.allclose(got[rows].to(D), want, rtol=2 ** -8 + 2 ** -20, atol=1e-30), b
    # fp32 and pairs: the same sums; a pair's halves add up to them, and are read as such
    for kind in (torch.float32, "pair"):
        wide = torch.full((R, width * (2 if kind == "pair" else 1)), 7.0, device=dev,
                          dtype=torch.bfloat16 if kind == "pair" else kind)
        ops.moe_grouped_gemm_w4(Ad.to(dev), p, wide, rb_expert, rb_rows, mode=mode)
        back = wide.float().view(R, 2 if kind == "pair" else 1, width)
        assert bool((back[~real.to(dev)] == 7).all())
        back, rounded = back[real.to(dev)], out[:R][real.to(dev)]
        if kind == "pair":
            assert torch.equal(back[:, 0], rounded.float())
            pairs, full = back.double().sum(1), whole[real.to(dev)].double()
            # 2^-8 of 2^-8; the smallest bf16 step is 2^-133, half of it what the second rounding may be off by at least
            assert bool(((pairs - full).abs() <= 2.0 ** -16 * full.abs() + 2.0 ** -134).all())
            if width % 8 == 0:
                w2 = _weights((E, width, 48), group, 9, zeros, True)
                y = torch.empty((R, 48), device=dev)
                ops.moe_grouped_gemm_w4(wide, _pack(dev, w2, group), y, rb_expert, rb_rows)
                d2 = _dense(*w2, group)
                for b in range(R // 128):
                    rows = slice(128 * b, 128 * b + int(rb_rows[b]))
                    x = wide[rows].cpu().view(-1, 2, width)
                    ref = x.to(D).sum(1) @ d2[int(rb_expert[b])]
                    mag = x.to(D).abs().sum(1) @ (143.0 * w2[1][int(rb_expert[b]), torch.arange(width) // group].to(D))
                    # as _bound, with twice the products
                    assert bool(((y[rows].cpu().to(D) - ref).abs() <= (512 + width / 128 + 8) * 2.0 ** -24 * mag).all())
        else:
            whole = wide
            assert torch.equal(back[:, 0].to(torch.bfloat16), rounded)
    # rows of a token buffer through a pull table, the row count on the device, blocks behind it and bad experts skipped
    tokens = _whole((40, K), 7)
    pick = torch.randint(0, 40, (R,), generator=torch.Generator().manual_seed(8))
    pull = torch.stack([torch.zeros(R, dtype=torch.int64), torch.zeros(R, dtype=torch.int64), pick], 1)
    pull[~real] = -1
    direct = torch.full((R, width), 7.0, dtype=torch.bfloat16, device=dev)
    ops.moe_grouped_gemm_w4(tokens[pick].to(dev), p, direct, rb_expert, rb_rows, mode=mode)
    bad = torch.tensor([E, -1], dtype=torch.int32, device=dev)
    more_pull = torch.cat([pull, torch.zeros((256, 3), dtype=torch.int64)]).int().to(dev)
    more = torch.full((R + 256, width), 7.0, dtype=torch.bfloat16, device=dev)
    ops.moe_grouped_gemm_w4(tokens.to(dev), p, more, torch.cat([rb_expert, bad]),
                            torch.cat([rb_rows, torch.full((2,), 128, dtype=torch.int32, device=dev)]), mode=mode,
                            gather_pull=more_pull, sizes=torch.tensor([R, R + 128], dtype=torch.int64, device=dev))
    assert torch.equal(more[:R], direct) and bool((more[R:] == 7).all())


def _layer(dev, T, H, I, E, e0, n_local, k, group, seed, zeros=False):
    g = torch.Generator().manual_seed(seed)
    x = wl.randn_bf16((T, H), seed)
    logits = torch.randn((T, E), generator=g)
    w1, w2 = _weights((n_local, H, 2 * I), group, seed + 1, zeros, False), _weights((n_local, I, H), group, seed + 2, zeros, False)
    return x, logits, w1, w2


def _run_layer(dev, x, logits, p1, p2, e0, n_local, k, out, bufs=None):
    """Logits to layer output, as a decode step runs it."""
    ids, gates = ops.moe_route(logits, k)
    t = ops.moe_build_indices_dev(ids, gates, e0, n_local, sync=False)
    cap = t["pull_indices"].shape[0]
    act = torch.full((cap, 2 * p2.K), float("nan"), dtype=torch.bfloat16, device=dev)
    ye = torch.full((cap, p1.K), float("nan"), device=dev)
    y = torch.empty(x.shape, dtype=out, device=dev)
    ops.moe_ffn_combine_w4(x, t["pull_indices"], t["row_weight"], t["owner_offset"], t["slot_to_row"], p1, p2, act, ye,
                           y, t["rb_expert"], t["rb_rows"], sizes=t["sizes"])
    return y, ids, gates


@pytest.mark.parametrize("T,H,I,E,e0,n_local,k,group,zeros,out", [
    (1, 512, 128, 16, 0, 16, 4, 128, False, torch.bfloat16), (5, 264, 48, 8, 2, 4, 2, 32, True, torch.float32),
    (64, 1024, 256, 64, 8, 8, 8, 64, False, torch.bfloat16), (300, 256, 112, 4, 0, 4, 2, 128, False, torch.float32),
    (3, 512, 128, 16, 12, 4, 1, 128, False, torch.bfloat16)])
def test_layer_from_logits(dev, T, H, I, E, e0, n_local, k, group, zeros, out):
    """Router, index build and 4-bit expert layer together, in 64 bits: one rounding to bf16 (of a bf16
    output), the activation held to 2^-16 of its value, and the fp32 sums."""
    _say("layer", T, H, I, E, e0, n_local, k, group, zeros, out)
    x, logits, w1, w2 = _layer(dev, T, H, I, E, e0, n_local, k, group, 11, zeros)
    p1, p2 = _pack(dev, w1, group), _pack(dev, w2, group)
    y, ids, gates = _run_layer(dev, x.to(dev), logits.to(dev), p1, p2, e0, n_local, k, out)
    ids, gates = ids.cpu(), gates.cpu()
    d1, d2 = _dense(*w1, group), _dense(*w2, group)
    ref, mag = torch.zeros((T, H), dtype=D), torch.zeros((T, H), dtype=D)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j]) - e0
            if 0 <= e < n_local:
                h = x[t].to(D) @ d1[e]
                a = torch.nn.functional.silu(h[:I]) * h[I:]
                ref[t] += gates[t, j].to(D) * (a @ d2[e])
                mag[t] += gates[t, j].to(D) * (a.abs() @ d2[e].abs())
    got = y.cpu().to(D)
    # the fp32 sums of either product: `n` roundings (see _bound) of 143 s |x| where mag counts |q - z| s |x|, which
    # is 4 on average: 36 times as much, and as much again of the first product's passed on through the second
    n = 256 + (max(H, I) + 127) // 128 + 8
    tol = (2 * 36 * n * 2.0 ** -24 + 2.0 ** -16) * mag + (2.0 ** -8 * ref.abs() if out is torch.bfloat16 else 0) + 1e-30
    assert bool(((got - ref).abs() <= tol).all())
    assert not got[mag.sum(1) == 0].any()
    if mag.any():
        assert float((got - ref).norm() / ref.norm()) < (2.0 ** -8 if out is torch.bfloat16 else 2.0 ** -15)


def test_layer_graph_and_streams(dev):
    """The decode step captured and replayed with new tokens, eager steps between; two streams at once."""
    _say("layer graph")
    T, H, I, E, k = 24, 512, 128, 32, 4
    x, logits, w1, w2 = _layer(dev, T, H, I, E, 0, E, k, 128, 21)
    p1, p2 = _pack(dev, w1, 128), _pack(dev, w2, 128)
    data = [(wl.randn_bf16((T, H), s).to(dev), torch.randn((T, E), generator=torch.Generator().manual_seed(s)).to(dev))
            for s in range(3)]
    want = [_run_layer(dev, a, b, p1, p2, 0, E, k, torch.bfloat16) for a, b in data]
    torch.cuda.synchronize()
    sx, sl = data[0][0].clone(), data[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run_layer(dev, sx, sl, p1, p2, 0, E, k, torch.bfloat16)
    for rep in range(4):
        sx.copy_(data[rep % 3][0])
        sl.copy_(data[rep % 3][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want[rep % 3])), rep
        _run_layer(dev, *data[1], p1, p2, 0, E, k, torch.bfloat16)
    got = []
    for (a, b) in data[:2]:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_run_layer(dev, a, b, p1, p2, 0, E, k, torch.bfloat16))
    torch.cuda.synchronize()
    for u, v in zip(got, want):
        assert all(torch.equal(i, j) for i, j in zip(u, v))


def test_many_blocks(dev):
    """More row blocks than a workgroup lists, a few rows in each (none in some), and rows at a block's end only."""
    _say("many blocks")
    E, K, N, B = 3, 96, 40, 700
    w = _weights((E, K, N), 32, 1, False, True)
    p = _pack(dev, w, 32)
    g = torch.Generator().manual_seed(4)
    rb_expert = torch.randint(0, E, (B,), generator=g)
    rb_rows = torch.randint(0, 20, (B,), generator=g)
    rb_rows[::97] = 128
    A = _whole((B * 128, K), 5)
    out = torch.full((B * 128, N), 7.0, dtype=torch.bfloat16, device=dev)
    ops.moe_grouped_gemm_w4(A.to(dev), p, out, rb_expert.int().to(dev), rb_rows.int().to(dev))
    got, dense = out.cpu(), _dense(*w, 32)
    for b in range(B):
        n = int(rb_rows[b])
        rows = slice(128 * b, 128 * b + n)
        assert torch.equal(got[rows], (A[rows].to(D) @ dense[int(rb_expert[b])]).float().to(torch.bfloat16)), b
        assert bool((got[128 * b + n:128 * b + 128] == 7).all()), b
    # the same with the row count on the device, below what is listed and above
    for rows in (128 * 300, 128 * 600):
        part = torch.full_like(out, 7.0)
        ops.moe_grouped_gemm_w4(A.to(dev), p, part, rb_expert.int().to(dev), rb_rows.int().to(dev),
                                sizes=torch.tensor([1, rows], dtype=torch.int64, device=dev))
        assert torch.equal(part[:rows], out[:rows]) and bool((part[rows:] == 7).all())


def test_every_row_real_and_several_sources(dev):
    """No rb_rows: all 128 rows of a block, as rb_rows of 128 gives them, for single values and pairs; tokens of several
    sources through the pull table, entries outside them read as zeros."""
    _say("whole blocks, sources")
    E, K, N, B = 3, 264, 96, 4
    w = _weights((E, K, N), 32, 1, True, True)
    p = _pack(dev, w, 32)
    rb_expert = torch.tensor([2, 0, 1, 0], dtype=torch.int32, device=dev)
    full = torch.full((B,), 128, dtype=torch.int32, device=dev)
    A = _whole((B * 128, K), 5).to(dev)
    for mode, a in ((0, A), (1, A), (0, torch.cat([A, A * 2 ** -9], 1))):
        width = N // 2 if mode else N
        got, want = (torch.full((B * 128, width), 7.0, device=dev) for _ in range(2))
        ops.moe_grouped_gemm_w4(a, p, got, rb_expert, mode=mode)
        ops.moe_grouped_gemm_w4(a, p, want, rb_expert, full, mode=mode)
        assert torch.equal(got, want)
        if mode == 0:
            x = a.cpu().to(D).view(B, 128, -1, K).sum(2)
            dense = _dense(*w, 32)
            ref = torch.cat([x[b] @ dense[int(rb_expert[b])] for b in range(B)])
            assert torch.equal(got.cpu(), ref.float())
    tokens = _whole((6 * 20, K), 7).to(dev)  # 3 nodes of 2 devices with 20 tokens each
    g = torch.Generator().manual_seed(3)
    R = B * 128
    pull = torch.stack([torch.randint(0, 3, (R,), generator=g), torch.randint(0, 2, (R,), generator=g),
                        torch.randint(0, 20, (R,), generator=g)], 1)
    at = (pull[:, 0] * 2 + pull[:, 1]) * 20 + pull[:, 2]
    rows = tokens.cpu()[at]
    pull[7] = torch.tensor([9, 0, 0])      # past the buffer
    pull[200] = torch.tensor([-1, -1, -1])  # a padding row
    rows[7] = rows[200] = 0
    got, want = (torch.full((R, N), 7.0, device=dev) for _ in range(2))
    ops.moe_grouped_gemm_w4(tokens, p, got, rb_expert, gather_pull=pull.int().to(dev), tokens_per_src=20, devs_per_node=2)
    ops.moe_grouped_gemm_w4(rows.to(dev), p, want, rb_expert)
    assert torch.equal(got, want)


def test_layer_with_host_sizes(dev):
    """Tables trimmed on the host: the bits of the device's row count; without rb_rows, padding rows as zeros."""
    _say("layer, host sizes")
    T, H, I, E, k = 40, 264, 48, 10, 3
    x, logits, w1, w2 = _layer(dev, T, H, I, E, 0, E, k, 64, 5)
    p1, p2 = _pack(dev, w1, 64), _pack(dev, w2, 64)
    want, ids, gates = _run_layer(dev, x.to(dev), logits.to(dev), p1, p2, 0, E, k, torch.float32)
    t = ops.moe_build_indices_dev(ids, gates, 0, E)
    R = t["R_pad"]
    for rb_rows in (t["rb_rows"], None):
        act = torch.full((R, 2 * I), float("nan"), dtype=torch.bfloat16, device=dev)
        ye = torch.full((R, H), float("nan"), device=dev)
        y = torch.empty((T, H), device=dev)
        ops.moe_ffn_combine_w4(x.to(dev), t["pull_indices"], t["row_weight"], t["owner_offset"], t["slot_to_row"], p1, p2,
                               act, ye, y, t["rb_expert"], rb_rows)
        if rb_rows is not None:
            assert torch.equal(y, want)
        else:  # other passes of the same rows: other sums of the same terms, an activation within 2^-16 of each
            assert float((y - want).norm() / want.norm()) < 2.0 ** -15


def test_past_32_bits(dev):
    """Packed weights of more than 4 GiB: the last experts' are the same as packed alone.  Rows of x and of the result
    more than 2^31 elements into their buffers."""
    _say("offsets past 32 bits")
    E, K, N, group = 36, 16384, 16384, 128
    g = torch.Generator(device=dev).manual_seed(5)
    codes = torch.randint(0, 16, (E, K, N), generator=g, dtype=torch.uint8, device=dev)
    scales = 2.0 ** torch.randint(-3, 1, (E, K // group, N), generator=g, device=dev).to(torch.bfloat16)
    p = ops.w4_pack(codes, scales, group)
    assert p.packed.numel() > 2**32
    x = _whole((256, K), 6).to(dev)
    rb_expert, rb_rows = torch.tensor([E - 1, 1], dtype=torch.int32, device=dev), torch.tensor([3, 2], dtype=torch.int32, device=dev)
    out = torch.zeros((256, N), device=dev)
    ops.moe_grouped_gemm_w4(x, p, out, rb_expert, rb_rows)
    for e, rows in ((E - 1, slice(0, 3)), (1, slice(128, 130))):
        one = ops.w4_pack(codes[e], scales[e], group)
        assert torch.equal(out[rows], ops.gemm_w4(x[rows], one, out=torch.empty((rows.stop - rows.start, N), device=dev)))
    del codes, p
    # strided rows
    M, K, N, ld = 70, 256, 96, 1 << 24
    w = _pack(dev, _weights((K, N), 64, 1, False, True), 64)
    wide = torch.empty((M, ld), dtype=torch.bfloat16, device=dev)
    assert (M - 1) * ld < 2**31 < 2 * (M - 1) * ld
    wide[:, :K] = _whole((M, K), 2).to(dev)
    assert torch.equal(ops.gemm_w4(wide[:, :K], w), ops.gemm_w4(wide[:, :K].contiguous(), w))
    far = torch.empty((M, 1 << 25), dtype=torch.bfloat16, device=dev)
    assert (M - 1) * (1 << 25) > 2**31
    assert torch.equal(ops.gemm_w4(wide[:, :K], w, out=far[:, :N]), ops.gemm_w4(wide[:, :K].contiguous(), w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_at_odd_places(dev, dtype):
    """Results that start at any element: columns from an odd one on, rows behind an odd width, for both products
    and for a pair; what lies beside them stays."""
    _say("outputs at odd places", dtype)
    for M, K, N in ((1, 136, 33), (5, 264, 2811), (40, 136, 8211)):
        w = _weights((K, N), 64, M, True, True)
        p, x = _pack(dev, w, 64), _whole((M, K), 1).to(dev)
        want = ops.gemm_w4(x, p, out=torch.empty((M, N), dtype=dtype, device=dev))
        for out in (torch.full((M, N + 3), 7.0, dtype=dtype, device=dev)[:, 1:N + 1],
                    torch.full((M + 2, N), 7.0, dtype=dtype, device=dev)[1:M + 1]):
            assert out.data_ptr() % 16
            assert torch.equal(ops.gemm_w4(x, p, out=out), want)
            whole = out._base if out._base is not None else out
            assert int((whole != 7).sum()) == int((want != 7).sum())
    K, N = 136, 96
    w = _weights((1, K, N), 64, 5, False, True)
    p, x = _pack(dev, w, 64), _whole((128, K), 1).to(dev)
    rb = torch.zeros(1, dtype=torch.int32, device=dev)
    for width in (N,) if dtype is torch.float32 else (N, 2 * N):
        want = ops.moe_grouped_gemm_w4(x, p, torch.empty((128, width), dtype=dtype, device=dev), rb)
        flat = torch.full((128 * width + 2,), 7.0, dtype=dtype, device=dev)
        got = ops.moe_grouped_gemm_w4(x, p, flat[1:-1].view(128, width), rb)
        assert got.data_ptr() % 16 and torch.equal(got, want) and bool((flat[[0, -1]] == 7).all())


def test_result_beside_its_input(dev):
    """Results in the same memory as their input but apart from it: other columns of the same rows, the rows
    behind; the layer's output over its tokens.  In place is refused."""
    _say("results beside inputs")
    M, K, N = 40, 264, 100
    w = _weights((K, N), 64, 3, True, True)
    p, x = _pack(dev, w, 64), _whole((M, K), 1).to(dev)
    want = ops.gemm_w4(x, p)
    for first in (True, False):  # out before or behind x in a row
        rows = torch.full((M, 400), 7.0, dtype=torch.bfloat16, device=dev)
        a, out = (rows[:, 104:104 + K], rows[:, 1:101]) if first else (rows[:, :K], rows[:, K:K + N])
        a.copy_(x)
        assert torch.equal(ops.gemm_w4(a, p, out=out), want) and torch.equal(a, x)
    flat = torch.full((M * K + M * N,), 7.0, dtype=torch.bfloat16, device=dev)
    flat[:M * K] = x.view(-1)
    assert torch.equal(ops.gemm_w4(flat[:M * K].view(M, K), p, out=flat[M * K:].view(M, N)), want)
    square = _pack(dev, _weights((K, K), 64, 4, False, True), 64)
    with pytest.raises(capi.MkError, match="overlaps"):
        ops.gemm_w4(x, square, out=x)
    T, H, I, E = 9, 64, 32, 4
    xs, logits, w1, w2 = _layer(dev, T, H, I, E, 0, E, 2, 32, 5)
    p1, p2, xd = _pack(dev, w1, 32), _pack(dev, w2, 32), xs.to(dev)
    want, ids, gates = _run_layer(dev, xd, logits.to(dev), p1, p2, 0, E, 2, torch.bfloat16)
    t = ops.moe_build_indices_dev(ids, gates, 0, E)
    args = xd, t["pull_indices"], t["row_weight"], t["owner_offset"], t["slot_to_row"], p1, p2
    act = torch.empty((t["R_pad"], 2 * I), dtype=torch.bfloat16, device=dev)
    ye = torch.empty((t["R_pad"], H), device=dev)
    with pytest.raises(capi.MkError, match="overlap"):
        ops.moe_ffn_combine_w4(*args, act, ye, ye.view(torch.bfloat16).view(-1)[:T * H].view(T, H), t["rb_expert"],
                               t["rb_rows"])
    assert torch.equal(ops.moe_ffn_combine_w4(*args, act, ye, xd, t["rb_expert"], t["rb_rows"]), want)


def test_no_tokens(dev):
    _say("layer without tokens, product without rows")
    w1, w2 = _weights((2, 64, 64), 32, 1, False, False), _weights((2, 32, 64), 32, 2, False, False)
    p1, p2 = _pack(dev, w1, 32), _pack(dev, w2, 32)
    e = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device=dev)
    bf = torch.bfloat16
    y = ops.moe_ffn_combine_w4(e(0, 64, t=bf), e(128, 3), e(128, t=torch.float32), e(1), e(1), p1, p2, e(128, 64, t=bf),
                               e(128, 64, t=torch.float32), e(0, 64, t=bf), e(1), e(1))
    assert y.shape == (0, 64)
    # no rows routed here: zeros, whatever the scratch holds
    nan = torch.full((0, 64), float("nan"), device=dev)
    y = torch.full((3, 64), 5.0, device=dev)
    ops.moe_ffn_combine_w4(torch.ones((3, 64), dtype=bf, device=dev), e(0, 3), e(0, t=torch.float32), e(4), e(1), p1, p2,
                           e(0, 64, t=bf), nan, y, e(0), e(0))
    assert not y.any()


def test_layer_rows_behind_the_buffers(dev):
    """Owner offsets of a routed batch with fewer rows than were routed, and with none: what has no row adds
    nothing, and no table of rows is read where there are no rows."""
    _say("layer, slots without rows")
    T, H, I, bf = 6, 64, 32, torch.bfloat16
    w1, w2 = _weights((2, H, 2 * I), 32, 1, False, False), _weights((2, I, H), 32, 2, False, False)
    ids = torch.tensor([[0, 1]] * T, dtype=torch.int32, device=dev)
    gates = torch.full((T, 2), 0.5, device=dev)
    x = wl.randn_bf16((T, H), 3).to(dev)
    both, first = ops.moe_build_indices_dev(ids, gates, 0, 2), ops.moe_build_indices_dev(ids, gates, 0, 1)
    assert both["R_pad"] == 256 and first["R_pad"] == 128

    def layer(t, rows, n):
        y = torch.full((T, H), float("nan"), device=dev)
        ye = torch.full((256, H), float("nan"), device=dev)  # (behind the rows: what may not be read)
        pack = lambda w: _pack(dev, (w[0][:n], w[1][:n], None), 32)
        ops.moe_ffn_combine_w4(x, t["pull_indices"][:rows], t["row_weight"][:rows], t["owner_offset"],
                               t["slot_to_row"] if rows else t["slot_to_row"][:0].clone(), pack(w1), pack(w2),
                               torch.empty((rows, 2 * I), dtype=bf, device=dev), ye[:rows], y, t["rb_expert"][:rows // 128],
                               t["rb_rows"][:rows // 128])
        return y

    assert torch.equal(layer(both, 128, 2), layer(first, 128, 1))
    assert not layer(both, 0, 2).any()


def test_weights_as_a_tensor(dev):
    """Packed weights stored and loaded; only the low four bits of a code count; a wrong size is refused."""
    _say("packed tensor")
    w = _weights((200, 50), 64, 3, True, True)
    p = _pack(dev, w, 64)
    again = ops.w4_pack((w[0] + 16 * (w[0] % 5)).to(dev), w[1].to(dev), 64, zeros=(w[2] + 32).to(dev))
    assert torch.equal(p.packed, again.packed)
    loaded = ops.W4Weights(p.packed.cpu().to(dev), 200, 50, 64, zeros=True)
    x = _whole((3, 200), 1).to(dev)
    assert torch.equal(ops.gemm_w4(x, loaded), ops.gemm_w4(x, p))
    for bad in ((p.packed, 200, 50, 64), (p.packed, 200, 50, 32, 1, True), (p.packed[:-16], 200, 50, 64, 1, True),
                (p.packed, 200, 50, 48, 1, True), (p.packed.cpu(), 200, 50, 64, 1, True), (p.packed, 0, 50, 64, 1, True)):
        with pytest.raises(ValueError):
            ops.W4Weights(*bad)


def test_python_refusals(dev):
    _say("refusals")
    codes = torch.zeros((64, 32), dtype=torch.uint8, device=dev)
    scales = torch.ones((2, 32), dtype=torch.bfloat16, device=dev)
    p = ops.w4_pack(codes, scales, 32)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device=dev)
    two = ops.w4_pack(codes.repeat(2, 1, 1), scales.repeat(2, 1, 1), 32)
    rb = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.zeros((128, 32), dtype=torch.bfloat16, device=dev)
    for call in (lambda: ops.w4_pack(codes, scales, 48), lambda: ops.w4_pack(codes, scales[:1], 32),
                 lambda: ops.w4_pack(codes.t(), scales, 32), lambda: ops.w4_pack(codes, scales.float(), 32),
                 lambda: ops.w4_pack(codes[:0], scales[:0], 32), lambda: ops.gemm_w4(x[:, :56], p),
                 lambda: ops.gemm_w4(x.t().contiguous().t(), p), lambda: ops.gemm_w4(x, two), lambda: ops.gemm_w4(x.float(), p),
                 lambda: ops.gemm_w4(x, p, out=out[:2, :31]), lambda: ops.gemm_w4(x.expand(2, 64)[:1].expand(4, 64), p),
                 lambda: ops.moe_grouped_gemm_w4(x, two, out, rb), lambda: ops.moe_grouped_gemm_w4(out, two, out, rb)):
        with pytest.raises(ValueError):
            call()
    logits = torch.zeros((3, 8), device=dev)
    ids = torch.zeros((3, 2), dtype=torch.int32, device=dev)
    for call in (lambda: ops.moe_route(logits, 9), lambda: ops.moe_route(logits, 0), lambda: ops.moe_route(logits.t(), 1),
                 lambda: ops.moe_route(logits.half(), 1), lambda: ops.moe_route(logits, 1, token_mask=ids[:, 0]),
                 lambda: ops.moe_route_balance(logits, 1, float("inf")), lambda: ops.moe_route_balance(logits, 1, 1e39),
                 lambda: ops.moe_route_backward(logits, ids), lambda: ops.moe_route_backward(logits, ids, counts=ids[0]),
                 lambda: ops.moe_route_backward(logits, ids, dgates=torch.zeros((2, 2), device=dev))):
        with pytest.raises((ValueError, OverflowError)):
            call()
