"""Refusals of how numbers between two products are held (CPU)."""
import ctypes as C

import pytest

from mkernel_amd import capi
from test_product_host import EINVAL, _args


@pytest.mark.parametrize("name", ["mk_gemm_act_backward", "mk_vocab_loss_backward"])
@pytest.mark.parametrize("between", [-1, 3, 99])
def test_refusals(name, between):
    L, a = capi.lib(), _args(name, dict(between=between))
    assert getattr(L, name)(C.byref(a), None) == EINVAL
    assert "between" in L.mk_last_error_string().decode()


def test_values_match_header():
    from test_product_host import ROOT
    text = (ROOT / "include" / "mk.h").read_text()
    for name, v in capi.BETWEEN.items():
        assert f"#define MK_BETWEEN_{name.upper()} {v}" in text
