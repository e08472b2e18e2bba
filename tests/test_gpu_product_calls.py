"""How the products' entry points keep what lies between their launches: the
small workspaces of threads and streams, and what a graph's capture records."""
import ctypes
import threading

import pytest
import torch

from mkernel_amd import capi, ops
from test_gpu_product_large import randn

pytestmark = pytest.mark.gpu


def _gemm_act_bytes(A, B, out) -> int:
    M, K = A.shape
    N = B.shape[1]
    return capi.workspace_bytes("mk_gemm_act", capi.GemmActArgs, A.data_ptr(), B.data_ptr(), out.data_ptr(), 0, 0, 0, M, N, K,
                                K, N, N, 0, 0, 0, 1, 0, 0)


def test_two_threads_share_no_small_workspace():
    """Two threads' calls on one stream whose operands are laid out anew in the small workspace: a launch of one may
    come between two of the other."""
    A, B = randn(300, 1501), [randn(1501, 205, seed=s) for s in (1, 2)]
    want = [ops.gemm_act(A, b) for b in B]
    assert all(0 < _gemm_act_bytes(A, b, w) <= ops._SPACE for b, w in zip(B, want))  # (larger ones are each call's own)
    torch.cuda.synchronize()
    got, at, start = [[], []], [None, None], threading.Barrier(2)

    def work(i):
        start.wait()
        for _ in range(300):
            got[i].append(ops.gemm_act(A, B[i]))
        at[i] = ops._space(A.device.index, torch.cuda.current_stream().cuda_stream)
        start.wait()  # (a thread's workspace goes with it)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert len(g) == 300 and all(torch.equal(x, w) for x in g)
    assert len({*at, ops._space(A.device.index, torch.cuda.current_stream().cuda_stream)}) == 3


def _nodes(call):
    """Nodes of a captured call, and the graph with its results."""
    hip = ctypes.CDLL("libamdhip64.so")
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        out = call()
    n = ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(ctypes.c_void_p(g.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    g.instantiate()
    return n.value, g, out


def test_captured_calls_record_no_tickets_they_do_not_touch():
    """A product whose K is not cut is one node, with a fill of the tickets in front of it where it is."""
    one = randn(1, 2048, seed=5), randn(2048, 2048, seed=6), randn(2048, seed=7)
    some = randn(256, 96, seed=8), randn(96, 512, seed=9)
    cut = randn(20, 4096, seed=10), randn(4096, 600, seed=11)
    x, V = randn(200, 64, seed=12), randn(64, 520, seed=13)
    labels = torch.arange(200, device="cuda")
    dloss = torch.full((200,), 0.005, device="cuda")
    lse = ops.vocab_loss(x, V, labels)["lse"]
    calls = [(1, lambda: [ops.gemm_act(one[0], one[1], bias=one[2], act="silu")]), (1, lambda: [ops.gemm_act(*some)]),
             (2, lambda: [ops.gemm_act(*cut)]),
             (2, lambda: list(ops.vocab_loss(x, V, labels).values())),  # statistics, their join
             (4, lambda: list(ops.vocab_loss_backward(x, V, labels, lse, dloss)))]  # rows of x, dl, dx, dW
    for want, call in calls:
        eager = call()
        n, g, out = _nodes(call)
        assert n == want, (want, n)
        for _ in range(4):
            for t in out:
                t.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_vocab_loss_workspace_holds_the_tiles_statistics():
    """8 bytes a token for each column tile that the launch has, 256 wide for a large batch, and no more.  (Addresses
    are not read for the question.)"""
    T, H, V, at = 32768, 512, 131072, 1 << 40
    n = capi.workspace_bytes("mk_vocab_loss", capi.VocabLossArgs, at, 2 * at, 3 * at, 4 * at, 5 * at, 6 * at, T, H, V, H, V, 0,
                             -100, 1)
    assert n == T * V // 256 * 8


def test_small_workspaces_are_given_back():
    A, B = randn(300, 1501), randn(1501, 205, seed=1)
    want = ops.gemm_act(A, B)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(ops.gemm_act(A, B), want)
    torch.cuda.synchronize()
    sets = len(ops._spaces.of)
    before = torch.cuda.memory_allocated()
    ops.release_split_workspaces()
    assert sets >= 2 and before - torch.cuda.memory_allocated() >= sets * ops._SPACE
    for _ in range(2):
        assert torch.equal(ops.gemm_act(A, B), want)  # (tickets are zeroed anew)
