"""CPU-side checks of the router, combine-gradient and 4-bit entry points:
struct layouts against the header, sizes, and every refusal (a negative code
before any device call: a device call here would give a positive one)."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from mkernel_amd import capi, ops

ROOT = Path(__file__).resolve().parent.parent

STRUCTS = {"mk_moe_route_args": capi.MoeRouteArgs, "mk_moe_route_backward_args": capi.MoeRouteBackwardArgs,
           "mk_moe_combine_backward_args": capi.MoeCombineBackwardArgs, "mk_w4_weights": capi.W4WeightsC,
           "mk_w4_pack_args": capi.W4PackArgs, "mk_w4_quantize_args": capi.W4QuantizeArgs,
           "mk_gemm_w4_args": capi.GemmW4Args, "mk_moe_grouped_gemm_w4_args": capi.MoeGroupedGemmW4Args,
           "mk_moe_ffn_w4_args": capi.MoeFfnW4Args}
ENTRIES = {"mk_moe_route": capi.MoeRouteArgs, "mk_moe_route_backward": capi.MoeRouteBackwardArgs,
           "mk_moe_combine_backward": capi.MoeCombineBackwardArgs, "mk_w4_pack": capi.W4PackArgs,
           "mk_w4_quantize": capi.W4QuantizeArgs, "mk_gemm_w4": capi.GemmW4Args,
           "mk_moe_grouped_gemm_w4": capi.MoeGroupedGemmW4Args, "mk_moe_ffn_combine_w4": capi.MoeFfnW4Args}


def test_struct_layouts_match_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "mk.h"}"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0; }"]))
    subprocess.run([cc, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in out.split("\n") if l}
    for cname, cls in STRUCTS.items():
        assert got[cname, "size"] == C.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert got[cname, f] == getattr(cls, f).offset, (cname, f)


@pytest.mark.parametrize("cls", list(STRUCTS.values()), ids=list(STRUCTS))
def test_packed_values_match_the_struct(cls):
    """call_values' byte block (nested weights' values in their place) is the struct's."""
    def leaves(c, base=0):
        for f, t in c._fields_:
            off = base + getattr(c, f).offset
            if isinstance(t, type) and issubclass(t, C.Structure):
                yield from leaves(t, off)
            else:
                yield off, t
    fields = list(leaves(cls))
    values = [i + 3 for i in range(len(fields))]
    block = capi._packer(cls)(*values)
    assert len(block) == C.sizeof(cls)
    for (off, t), v in zip(fields, values):
        assert (t.from_buffer_copy(block, off).value or 0) == v


@pytest.mark.parametrize("name", sorted(ENTRIES))
def test_missing_arguments(name):
    fn, L = getattr(capi.lib(), name), capi.lib()
    assert fn(None, None) < 0 and name.encode() in L.mk_last_error_string()
    assert fn(C.byref(ENTRIES[name]()), None) < 0, L.mk_last_error_string()


_BUF = (C.c_char * 4096)()
P = (C.addressof(_BUF) + 255) // 256 * 256  # never read: every call below is refused
EINVAL, ESHAPE = -1, -2


def _refused(name, args, code, match):
    L = capi.lib()
    assert getattr(L, name)(C.byref(args), None) == code
    assert match in L.mk_last_error_string().decode(), L.mk_last_error_string()


def _args(cls, base, change):
    a = cls()
    for k, v in {**base, **change}.items():
        setattr(a, k, v)
    return a


ROUTE = dict(logits=P, topk_ids=P, gates=P, num_tokens=4, ld=64, num_experts=64, topk=8)
BALANCE = dict(counts=P, prob_sum=P, tokens=P, loss=P, workspace=P, workspace_bytes=1 << 30)


@pytest.mark.parametrize("change,code,match", [
    (dict(num_tokens=-1), EINVAL, "sizes"), (dict(num_experts=0), EINVAL, "sizes"), (dict(topk=0), EINVAL, "sizes"),
    (dict(logits_dtype=2), EINVAL, "logits_dtype"), (dict(num_experts=1025, ld=1025), ESHAPE, "1024"),
    (dict(topk=33), ESHAPE, "topk"), (dict(num_experts=4, topk=5), ESHAPE, "topk"), (dict(ld=63), ESHAPE, "ld"),
    (dict(num_tokens=1 << 30), ESHAPE, "32-bit"), (dict(logits=0), EINVAL, "null"), (dict(gates=0), EINVAL, "null"),
    (dict(BALANCE, loss=0), EINVAL, "counts needs"), (dict(BALANCE, workspace=0), EINVAL, "counts needs"),
    (dict(BALANCE, workspace=P + 8), EINVAL, "aligned"), (dict(BALANCE, workspace_bytes=8), EINVAL, "smaller")])
def test_route_refusals(change, code, match):
    _refused("mk_moe_route", _args(capi.MoeRouteArgs, ROUTE, change), code, match)


BACK = dict(logits=P, topk_ids=P, dgates=P, dlogits=P, num_tokens=4, ld=64, ld_out=64, num_experts=64, topk=8)


@pytest.mark.parametrize("change,code,match", [
    (dict(topk=33), ESHAPE, "topk"), (dict(ld_out=63), ESHAPE, "ld_out"), (dict(dgates=0), EINVAL, "dgates or counts"),
    (dict(counts=P), EINVAL, "tokens"), (dict(topk_ids=0), EINVAL, "null"), (dict(dlogits=0), EINVAL, "null"),
    (dict(logits_dtype=-1), EINVAL, "logits_dtype")])
def test_route_backward_refusals(change, code, match):
    _refused("mk_moe_route_backward", _args(capi.MoeRouteBackwardArgs, BACK, change), code, match)


@pytest.mark.parametrize("change", [
    dict(dlogits=P + 4), dict(dlogits=P + 255), dict(ld_out=68), dict(dlogits=P + 256, ld_out=65),
    dict(ld=128, ld_out=128, dlogits=P + 252), dict(ld=128, ld_out=128, dlogits=P + 260), dict(dlogits=P - 4),
    dict(dlogits=P + 4 * 255), dict(num_tokens=1, dlogits=P + 4), dict(ld=128, ld_out=128, dlogits=P + 508)])
def test_route_backward_overlap(change):
    """An output that shares elements with the logits and is not the logits."""
    _refused("mk_moe_route_backward", _args(capi.MoeRouteBackwardArgs, BACK, change), EINVAL, "overlaps")


COMBINE = dict(dy=P, y_expert=P, topk_ids=P, row_weight=P, owner_offset=P, slot_to_row=P, rb_rows=P, dy_expert=P,
               dgates=P, num_tokens=4, H=64, R_pad=128, topk=2, expert_begin=0, n_local=4)


@pytest.mark.parametrize("change,code,match", [
    (dict(H=12), ESHAPE, "H"), (dict(R_pad=100), ESHAPE, "R_pad"), (dict(topk=33), ESHAPE, "topk"),
    (dict(n_local=0), EINVAL, "sizes"), (dict(expert_begin=-1), EINVAL, "sizes"), (dict(dy_dtype=3), EINVAL, "dy_dtype"),
    (dict(dy=0), EINVAL, "null"), (dict(slot_to_row=0), EINVAL, "null"), (dict(rb_rows=0), EINVAL, "null"),
    (dict(dy=P + 8), EINVAL, "aligned"), (dict(num_tokens=1 << 31), ESHAPE, "rows")])
def test_combine_backward_refusals(change, code, match):
    _refused("mk_moe_combine_backward", _args(capi.MoeCombineBackwardArgs, COMBINE, change), code, match)


@pytest.mark.parametrize("change", [
    dict(dy_expert=P + 128 * 128 - 16), dict(dy_expert=P + 16), dict(dy_expert=P - 16), dict(dy=P + (1 << 20), dy_expert=P + (1 << 20)),
    dict(dy=P + (1 << 20), dy_expert=P + (1 << 20) + 4 * 256 - 16),
    dict(dy=P + (1 << 20), dy_expert=P + (1 << 20) + 4 * 128 - 16, dy_dtype=1), dict(dy=P, dy_expert=P)])
def test_combine_backward_overlap(change):
    """dy_expert over a part of y_expert, or over dy (4 tokens of 64 columns)."""
    _refused("mk_moe_combine_backward", _args(capi.MoeCombineBackwardArgs, COMBINE, change), EINVAL, "overlaps")


def _weights(**change):
    return _args(capi.W4WeightsC, dict(packed=P, K=256, N=64, group=128, num_experts=1), change)


@pytest.mark.parametrize("change,code,match", [
    (dict(packed=0), EINVAL, "null"), (dict(group=48), EINVAL, "group"), (dict(K=0), ESHAPE, "sizes"),
    (dict(N=1 << 25), ESHAPE, "sizes"), (dict(packed=P + 2), EINVAL, "aligned")])
def test_weight_refusals(change, code, match):
    w = _weights(**change)
    _refused("mk_gemm_w4", _args(capi.GemmW4Args, dict(A=P, C=P, M=1, lda=256, ldc=64, W=w), {}), code, match)
    _refused("mk_w4_pack", _args(capi.W4PackArgs, dict(codes=P, scales=P, out=w), {}), code, match)


GEMM = dict(A=P, C=P, M=1, lda=256, ldc=64, out_type=1)


@pytest.mark.parametrize("weights,change,code,match", [
    ({}, dict(M=-1), ESHAPE, "M must"), ({}, dict(M=(1 << 20) + 1), ESHAPE, "M must"), (dict(K=252), {}, ESHAPE, "K must"),
    ({}, dict(lda=248), ESHAPE, "lda"), ({}, dict(lda=260), ESHAPE, "lda"), ({}, dict(ldc=63), ESHAPE, "lda"),
    (dict(num_experts=2), {}, EINVAL, "matrices"), ({}, dict(out_type=2), EINVAL, "out_type"),
    ({}, dict(lda=1 << 25), ESHAPE, "lda"), ({}, dict(A=0), EINVAL, "null"), ({}, dict(A=P + 2), EINVAL, "aligned")])
def test_gemm_w4_refusals(weights, change, code, match):
    _refused("mk_gemm_w4", _args(capi.GemmW4Args, dict(GEMM, W=_weights(**weights)), change), code, match)


@pytest.mark.parametrize("out_type,off", [(0, 2), (0, 1), (1, 1), (2, 1)])
def test_w4_outputs_are_aligned_to_their_elements(out_type, off):
    if out_type < 2:
        _refused("mk_gemm_w4", _args(capi.GemmW4Args, dict(GEMM, W=_weights(), C=P + off, out_type=out_type), {}), EINVAL,
                 "elements")
    _refused("mk_moe_grouped_gemm_w4", _args(capi.MoeGroupedGemmW4Args,
                                             dict(GROUPED, W=_weights(), out=P + off, out_type=out_type), {}), EINVAL, "elements")


@pytest.mark.parametrize("change", [dict(act=P + 4), dict(y_expert=P + 4), dict(tokens=P + 8)])
def test_ffn_w4_scratch_alignment(change):
    a = dict(FFN, w1=_weights(K=256, N=64), w2=_weights(K=32, N=256))
    _refused("mk_moe_ffn_combine_w4", _args(capi.MoeFfnW4Args, a, change), EINVAL, "16-byte")


# A is 4 rows of 512 bytes, C 4 rows of 64 columns
@pytest.mark.parametrize("change", [
    dict(C=P), dict(C=P + 1024), dict(C=P + 4 * 512 - 2), dict(C=P - 3 * 128 - 126), dict(C=P + 512, ldc=256),
    dict(lda=512, ldc=512, C=P + 510), dict(lda=512, ldc=512, C=P + 1024 - 126), dict(lda=512, ldc=256, out_type=0, C=P + 800),
    dict(M=1, C=P + 510)])
def test_gemm_w4_overlap(change):
    """A result that shares elements with A, which other workgroups may still read."""
    _refused("mk_gemm_w4", _args(capi.GemmW4Args, dict(GEMM, M=4, W=_weights()), change), EINVAL, "overlaps")


def test_expert_products_overlap():
    far = P + (1 << 30)  # never read
    for change in (dict(out=P), dict(out=P + 128 * 512 - 2), dict(out=P - 128 * 128 + 2), dict(PULL, n_src_rows=2, out=P + 1022)):
        _refused("mk_moe_grouped_gemm_w4", _args(capi.MoeGroupedGemmW4Args, dict(GROUPED, W=_weights()), change), EINVAL,
                 "overlaps")
    for change in (dict(act=P), dict(act=P + 496), dict(act=far, y_expert=far), dict(act=far, y_expert=far + 128 * 128 - 16),
                   dict(act=far, y_expert=far - 128 * 1024 + 16), dict(act=far, y_expert=2 * far, y_out=2 * far + 1024)):
        a = dict(FFN, w1=_weights(K=256, N=64), w2=_weights(K=32, N=256))
        _refused("mk_moe_ffn_combine_w4", _args(capi.MoeFfnW4Args, a, change), EINVAL, "overlap")


def test_pack_refusals():
    _refused("mk_w4_pack", _args(capi.W4PackArgs, dict(codes=P, scales=P, zeros=P, out=_weights()), {}), EINVAL, "one side")
    _refused("mk_w4_quantize", _args(capi.W4QuantizeArgs, dict(W=P, codes=P, scales=P, K=8, N=8, group=16, num_experts=1),
                                     {}), EINVAL, "group")


GROUPED = dict(A=P, out=P, rb_expert=P, R_pad=128, mode=0, a_parts=1, out_type=1)
PULL = dict(gather_pull=P, n_src_rows=1, tokens_per_src=1, devs_per_node=1)


@pytest.mark.parametrize("weights,change,code,match", [
    ({}, dict(mode=2), EINVAL, "mode"), ({}, dict(R_pad=64), ESHAPE, "R_pad"), ({}, dict(rb_expert=0), EINVAL, "null"),
    (dict(N=48), dict(mode=1), ESHAPE, "SwiGLU"), ({}, dict(gather_pull=P), EINVAL, "gather_pull"),
    ({}, dict(PULL, a_parts=2), EINVAL, "gather_pull"), ({}, dict(PULL, n_src_rows=1 << 22), EINVAL, "2 GiB"),
    ({}, dict(a_parts=0), EINVAL, "a_parts"), ({}, dict(out_type=3), EINVAL, "out_type"),
    ({}, dict(R_pad=1 << 22), ESHAPE, "R_pad"), (dict(K=100), {}, ESHAPE, "K must")])
def test_grouped_w4_refusals(weights, change, code, match):
    _refused("mk_moe_grouped_gemm_w4", _args(capi.MoeGroupedGemmW4Args, dict(GROUPED, W=_weights(**weights)), change),
             code, match)


FFN = dict(tokens=P, pull_indices=P, rb_expert=P, row_weight=P, owner_offset=P, slot_to_row=P, act=P, y_expert=P,
           y_out=P, num_tokens=1, n_src_rows=1, R_pad=128, tokens_per_src=1, devs_per_node=1)


@pytest.mark.parametrize("w2,change,code,match", [
    (dict(K=64), {}, ESHAPE, "w1 must"), (dict(num_experts=3), {}, ESHAPE, "w1 must"), ({}, dict(act=0), EINVAL, "null"),
    ({}, dict(out_dtype=2), EINVAL, "out_dtype"), ({}, dict(num_tokens=-1), ESHAPE, "num_tokens"),
    ({}, dict(y_out=P + 4), EINVAL, "aligned"), ({}, dict(tokens_per_src=0), EINVAL, "gather_pull")])
def test_ffn_w4_refusals(w2, change, code, match):
    a = dict(FFN, w1=_weights(K=256, N=64), w2=_weights(**dict(dict(K=32, N=256), **w2)))
    _refused("mk_moe_ffn_combine_w4", _args(capi.MoeFfnW4Args, a, change), code, match)


def test_sizes():
    L = capi.lib()
    assert L.mk_w4_packed_bytes(256, 64, 1, 128, 0) == 256 * 64 // 2 + 2 * 64 * 2
    # whole blocks of 128 rows by two tiles of 16 columns; a byte per zero point
    assert L.mk_w4_packed_bytes(129, 33, 3, 32, 1) == 3 * (256 * 64 // 2 + 8 * 64 * 3)
    assert L.mk_w4_packed_bytes(0, 64, 1, 128, 0) < 0 and L.mk_w4_packed_bytes(64, 64, 1, 16, 0) < 0
    # more weights than any memory holds: no byte count that wraps round
    assert L.mk_w4_packed_bytes(1 << 24, 1 << 24, 65536, 128, 0) < 0 and L.mk_w4_packed_bytes(1 << 20, 1 << 20, 2, 32, 1) < 0
    assert L.mk_w4_packed_bytes(1 << 20, 1 << 20, 1, 128, 0) == (1 << 39) + (1 << 34)
    assert L.mk_moe_route_workspace_bytes(-1, 8) < 0 and L.mk_moe_route_workspace_bytes(1, 1025) < 0
    assert L.mk_moe_route_workspace_bytes(0, 8) > 0
    # bounded however long the batch is
    assert L.mk_moe_route_workspace_bytes(1 << 30, 256) == L.mk_moe_route_workspace_bytes(1 << 20, 256)


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 8)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: ops.moe_route(x, 2), lambda: ops.moe_route_balance(x, 2, 0.1),
                 lambda: ops.moe_route_backward(x, ids, dgates=torch.zeros(4, 2)),
                 lambda: ops.w4_pack(torch.zeros(8, 8, dtype=torch.uint8), x, 32),
                 lambda: ops.w4_quantize(x.bfloat16(), 32), lambda: ops.gemm_w4(x.bfloat16(), None),
                 lambda: ops.moe_combine_backward(x, x, ids, x, ids, ids, ids, 0, 1)):
        with pytest.raises(ValueError):
            call()
