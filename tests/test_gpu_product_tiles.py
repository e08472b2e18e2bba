"""The products on tiles and cuts that the sizes of the other tests do not reach
(tests/test_product_tiles_host.py says which runs what): wide and tall tiles with
K in parts, against 64 bits.

Tolerances as in test_gpu_product.py: n * 2^-24 * sum |products| for a sum of n
products, then half a step of the result's type."""
import pytest

import test_gpu_product_large as large
from test_gpu_product_large import BF16, F32

pytestmark = pytest.mark.gpu

# M, K, N of the forward order, all of them cut: 64 x 128, the same behind whole rounds, 128 x 128, the same behind whole
FORWARD = [(33, 5631, 15478), (294, 7345, 13179), (970, 10143, 1003), (1538, 903, 10059)]
# K, M (the sum), N of dB: 128 x 128, 128 x 256 (64 x 64 where more follows than the plain result), 128 x 256 behind
# whole rounds (256 x 256), 64 x 128
RIGHT = [(66, 7590, 9140), (9906, 5521, 135), (13099, 1171, 1185), (282, 5516, 13615), (100, 6000, 3000)]


@pytest.mark.parametrize("M,K,N", FORWARD)
@pytest.mark.parametrize("plain", [True, False], ids=["plain", "all"])
def test_gemm_act(M, K, N, plain):
    large.test_gemm_act(M, K, N, plain)


@pytest.mark.parametrize("K,M,N", RIGHT)
@pytest.mark.parametrize("dtype,accumulate", [(BF16, False), (F32, False), (F32, True), (BF16, True)],
                         ids=["bf16", "f32", "f32+", "bf16+"])
def test_gemm_act_backward(K, M, N, dtype, accumulate):
    large.test_gemm_act_backward(K, M, N, dtype, accumulate)
