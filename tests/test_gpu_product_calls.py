"""How the products' entry points keep what lies between their launches: the
small workspaces of threads and streams, and what a graph's capture records."""
import threading

import torch
import pytest

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
