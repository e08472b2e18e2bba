"""CPU-side checks of the questions about workspaces and tickets."""
import ctypes as C

import pytest

from mkernel_amd import capi
from test_product_host import _args


@pytest.mark.parametrize("name", capi._CUT_PRODUCTS)
def test_ticket_words_of_refused_calls(name):
    ask = getattr(capi.lib(), name + "_ticket_words")
    assert ask(None) < 0
    a = _args(name, dict(M=-1) if "gemm" in name else dict(T=-1))
    assert ask(C.byref(a)) < 0
    assert "sizes" in capi.lib().mk_last_error_string().decode()
