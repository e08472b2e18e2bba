"""CPU-side checks of the products' entry points: struct layouts against the
header, every refusal (a negative code before any device call), and the host's
choice of tile and cut, compiled with the system C++ compiler, so that the GPU
tests' shapes run on every tile."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import test_gpu_product as small
import test_gpu_product_large as large
from mkernel_amd import capi, ops

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"mk_gemm_act": capi.GemmActArgs, "mk_gemm_act_backward": capi.GemmActBackwardArgs,
           "mk_moe_ragged_gemm": capi.MoeRaggedGemmArgs, "mk_moe_ragged_dgrad": capi.MoeRaggedDgradArgs,
           "mk_moe_ragged_wgrad": capi.MoeRaggedWgradArgs, "mk_vocab_loss": capi.VocabLossArgs,
           "mk_vocab_loss_backward": capi.VocabLossBackwardArgs}
_BUF = (C.c_char * 4096)()
P = (C.addressof(_BUF) + 255) // 256 * 256  # never read: every call below is refused
FAR = P + (1 << 40)
EINVAL, ESHAPE, EWORKSPACE = -1, -2, -5


def test_struct_layouts_match_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "mk.h"}"', "int main(void) {",
             '  printf("tickets 0 %d\\n", MK_PRODUCT_TICKETS);', '  printf("workspace 0 %d\\n", MK_EWORKSPACE);']
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}_args));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}_args, {f}));' for f, _ in cls._fields_]
    for a, v in capi.ACTS.items():
        lines.append(f'  printf("act {a} %d\\n", MK_ACT_{a.upper()});')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0; }"]))
    subprocess.run([cc, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in out.split("\n") if l}
    for name, cls in STRUCTS.items():
        assert got[name, "size"] == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert got[name, f] == getattr(cls, f).offset, (name, f)
    assert got["tickets", "0"] == capi.PRODUCT_TICKETS and got["workspace", "0"] == capi.EWORKSPACE
    for a, v in capi.ACTS.items():
        assert got["act", a] == v


BASE = {
    "mk_gemm_act": dict(A=P, B=FAR, C=2 * FAR, M=4, N=32, K=64, lda=64, ldb=32, ldc=32, ldr=32, ldp=32, c_type=1,
                        bias_type=1, residual_type=1, tickets=P),
    "mk_gemm_act_backward": dict(dC=P, A=FAR, B=2 * FAR, pre=3 * FAR, dA=4 * FAR, dB=5 * FAR, dbias=6 * FAR, M=4, N=32,
                                 K=64, lddc=32, lda=64, ldb=32, ldp=32, ldda=64, lddb=32, act=4, db_type=1, tickets=P),
    "mk_moe_ragged_gemm": dict(A=P, W=FAR, counts=P, out=2 * FAR, R=8, K=64, N=32, lda=64, ldo=32, ldh=32, num_experts=4),
    "mk_moe_ragged_dgrad": dict(dy=P, W=FAR, counts=P, out=2 * FAR, R=8, K=64, N=32, lddy=32, ldh=128, ldo=128, num_experts=4),
    "mk_moe_ragged_wgrad": dict(A=P, dy=FAR, counts=P, dW=2 * FAR, R=8, K=64, N=32, lda=64, lddy=32, num_experts=4, dw_type=1),
    "mk_vocab_loss": dict(x=P, W=FAR, labels=2 * FAR, lse=3 * FAR, target=4 * FAR, loss=5 * FAR, T=4, H=64, V=100, ldx=64,
                          ldw=100, ignore_index=-100, labels_type=1, tickets=P),
    "mk_vocab_loss_backward": dict(x=P, W=FAR, labels=2 * FAR, lse=3 * FAR, dloss=4 * FAR, dx=5 * FAR, dW=6 * FAR, T=4,
                                   H=64, V=100, ldx=64, ldw=100, lddx=64, lddw=100, ignore_index=-100, labels_type=1,
                                   dx_type=1, dw_type=1, tickets=P),
}

REFUSALS = [
    ("mk_gemm_act", dict(M=-1), ESHAPE, "sizes"), ("mk_gemm_act", dict(N=1 << 22), ESHAPE, "sizes"),
    ("mk_gemm_act", dict(act=5), EINVAL, "act"), ("mk_gemm_act", dict(act=-1), EINVAL, "act"),
    ("mk_gemm_act", dict(c_type=2), EINVAL, "types"), ("mk_gemm_act", dict(lda=63), ESHAPE, "rows of A"),
    ("mk_gemm_act", dict(ldb=1 << 22), ESHAPE, "rows of B"), ("mk_gemm_act", dict(A=0), EINVAL, "A is null"),
    ("mk_gemm_act", dict(C=0), EINVAL, "C is null"), ("mk_gemm_act", dict(A=P + 1), EINVAL, "aligned"),
    ("mk_gemm_act", dict(bias=P + 2, bias_type=0), EINVAL, "aligned"), ("mk_gemm_act", dict(tickets=0), EINVAL, "tickets"),
    ("mk_gemm_act", dict(C=P), EINVAL, "C overlaps A"), ("mk_gemm_act", dict(C=FAR + 8), EINVAL, "C overlaps B"),
    ("mk_gemm_act", dict(pre=2 * FAR), EINVAL, "pre overlaps C"), ("mk_gemm_act", dict(pre=P + 2), EINVAL, "pre overlaps A"),
    ("mk_gemm_act", dict(residual=2 * FAR + 2), EINVAL, "C overlaps residual"),
    ("mk_gemm_act", dict(residual=2 * FAR, ldr=40), EINVAL, "C overlaps residual"),
    ("mk_gemm_act", dict(residual=2 * FAR, residual_type=0), EINVAL, "C overlaps residual"),
    ("mk_gemm_act", dict(bias=2 * FAR), EINVAL, "C overlaps bias"), ("mk_gemm_act", dict(residual=P + 1024, ldr=31), ESHAPE, "residual"),
    ("mk_gemm_act_backward", dict(pre=0), EINVAL, "pre is null"), ("mk_gemm_act_backward", dict(dA=0, dB=0, dbias=0), EINVAL, "must be set"),
    ("mk_gemm_act_backward", dict(dA=P), EINVAL, "dA overlaps dC"), ("mk_gemm_act_backward", dict(dB=4 * FAR), EINVAL, "dB overlaps dA"),
    ("mk_gemm_act_backward", dict(dbias=5 * FAR + 4), EINVAL, "dbias overlaps dB"),
    ("mk_gemm_act_backward", dict(db_type=3), EINVAL, "db_type"), ("mk_gemm_act_backward", dict(A=0), EINVAL, "A is null"),
    ("mk_gemm_act_backward", dict(dB=3 * FAR), EINVAL, "dB overlaps pre"), ("mk_gemm_act_backward", dict(act=9), EINVAL, "act"),
    ("mk_moe_ragged_gemm", dict(mode=2), EINVAL, "mode"), ("mk_moe_ragged_gemm", dict(mode=1, N=33, ldo=33), ESHAPE, "even"),
    ("mk_moe_ragged_gemm", dict(h=P), EINVAL, "mode 1"), ("mk_moe_ragged_gemm", dict(num_experts=1025), ESHAPE, "experts"),
    ("mk_moe_ragged_gemm", dict(num_experts=0), ESHAPE, "experts"), ("mk_moe_ragged_gemm", dict(counts=0), EINVAL, "counts"),
    ("mk_moe_ragged_gemm", dict(K=0), ESHAPE, "K and N"), ("mk_moe_ragged_gemm", dict(R=-1), ESHAPE, "sizes"),
    ("mk_moe_ragged_gemm", dict(out=P), EINVAL, "out overlaps A"), ("mk_moe_ragged_gemm", dict(out=FAR + 64 * 64 * 3), EINVAL, "out overlaps W"),
    ("mk_moe_ragged_gemm", dict(mode=1, h=2 * FAR), EINVAL, "h overlaps out"),
    ("mk_moe_ragged_dgrad", dict(out=P), EINVAL, "out overlaps dy"), ("mk_moe_ragged_dgrad", dict(h=2 * FAR + 2), EINVAL, "out overlaps h"),
    ("mk_moe_ragged_dgrad", dict(h=2 * FAR, ldh=130), EINVAL, "out overlaps h"), ("mk_moe_ragged_dgrad", dict(ldo=63), ESHAPE, "out"),
    ("mk_moe_ragged_wgrad", dict(dW=P), EINVAL, "dW overlaps A"), ("mk_moe_ragged_wgrad", dict(dw_type=2), EINVAL, "dw_type"),
    ("mk_moe_ragged_wgrad", dict(dy=0), EINVAL, "dy is null"),
    ("mk_vocab_loss", dict(V=0), ESHAPE, "H and V"), ("mk_vocab_loss", dict(vocab_begin=-1), EINVAL, "vocab_begin"),
    ("mk_vocab_loss", dict(labels_type=2), EINVAL, "labels_type"), ("mk_vocab_loss", dict(labels=0), EINVAL, "null"),
    ("mk_vocab_loss", dict(labels=P + 4), EINVAL, "labels"), ("mk_vocab_loss", dict(lse=P), EINVAL, "lse overlaps x"),
    ("mk_vocab_loss", dict(loss=3 * FAR + 4), EINVAL, "loss overlaps lse"), ("mk_vocab_loss", dict(T=(1 << 21) + 1), ESHAPE, "tokens"),
    ("mk_vocab_loss_backward", dict(piece_columns=100), EINVAL, "piece_columns"),
    ("mk_vocab_loss_backward", dict(piece_columns=-256), EINVAL, "piece_columns"),
    ("mk_vocab_loss_backward", dict(dx=0, dW=0), EINVAL, "must be set"), ("mk_vocab_loss_backward", dict(dloss=0), EINVAL, "dloss"),
    ("mk_vocab_loss_backward", dict(dx=P), EINVAL, "dx overlaps x"), ("mk_vocab_loss_backward", dict(dW=FAR), EINVAL, "dW overlaps W"),
    ("mk_vocab_loss_backward", dict(dx_type=5), EINVAL, "types"), ("mk_vocab_loss_backward", dict(lddw=99), ESHAPE, "dW"),
]


def _args(name, change):
    a = STRUCTS[name]()
    for k, v in {**BASE[name], **change}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("name,change,code,match", REFUSALS, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refusals(name, change, code, match):
    L, a = capi.lib(), _args(name, change)
    assert getattr(L, name)(C.byref(a), None) == code, L.mk_last_error_string()
    assert match in L.mk_last_error_string().decode(), L.mk_last_error_string()
    if "tickets" not in change:
        assert getattr(L, name + "_workspace_bytes")(C.byref(a)) < 0


@pytest.mark.parametrize("name", list(STRUCTS))
def test_missing_arguments(name):
    L = capi.lib()
    assert getattr(L, name)(None, None) < 0 and getattr(L, name + "_workspace_bytes")(None) < 0


def test_host_tensors_are_refused():
    a = torch.zeros(4, 8, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.gemm_act(a, a.t().contiguous()), lambda: ops.gemm_act_backward(a, a, a),
                 lambda: ops.moe_ragged_gemm(a, torch.zeros(2, 8, 4, dtype=torch.bfloat16), n),
                 lambda: ops.moe_ragged_gemm_dgrad(a, torch.zeros(2, 4, 8, dtype=torch.bfloat16), n),
                 lambda: ops.moe_ragged_gemm_wgrad(a, a, n), lambda: ops.vocab_loss(a, a.t().contiguous(), n),
                 lambda: ops.vocab_loss_backward(a, a.t().contiguous(), n, a, a)):
        with pytest.raises(ValueError, match="device tensor"):
            call()


PROG = r"""
#include "mk_product_plan.h"
extern "C" {
// out: tile, parts along K, tiles, tiles that are whole
void plan(int64_t M, int64_t cols, int64_t K, int64_t groups, int ragged, int right, int plain, int cut, int64_t* out) {
  const mk::ProductPlan p = mk::plan_product(M, cols, K, groups, ragged, right, plain, cut, 256);
  out[0] = p.tile; out[1] = p.split; out[2] = p.tiles; out[3] = p.whole;
}
int few(int64_t M, int64_t N, int64_t K, int aligned) { return mk::product_few_rows(M, N, K, aligned); }
int shape(int i, int k) { return k == 0 ? mk::kProductShapes[i].bm : k == 1 ? mk::kProductShapes[i].bn : mk::kProductShapes[i].per_cu; }
}
"""
TILE32, TILE64, TILE64W, TILE128, TILE256, TILE128W = range(6)


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(PROG)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT / 'mkernel_amd' / 'csrc'}", str(d / "p.cpp"),
                    "-o", str(d / "p.so")], check=True)
    L = C.CDLL(str(d / "p.so"))
    L.plan.argtypes = [C.c_int64] * 4 + [C.c_int] * 4 + [C.c_void_p]
    L.few.argtypes = [C.c_int64] * 3 + [C.c_int]

    def plan(M, cols, K, groups=1, ragged=0, right=0, plain=1, cut=1):
        out = (C.c_int64 * 4)()
        L.plan(M, cols, K, groups, ragged, right, plain, cut, out)
        return tuple(out)
    plan.few, plan.shape = L.few, L.shape
    return plan


def test_the_gpu_tests_run_every_tile(plans):
    """Dense, ragged and gradient shapes of the GPU tests, whole and in parts."""
    dense = {plans(M, N, K)[:2] for M, K, N in small.SHAPES + large.FORWARD}
    assert {t for t, _ in dense} == {TILE32, TILE64, TILE64W, TILE128, TILE256}
    assert {t for t, s in dense if s > 1} >= {TILE32, TILE64, TILE256}
    for M, K, N in large.FORWARD:
        t, s, tiles, whole = plans(M, N, K)
        assert whole == tiles if s == 1 else whole < tiles
    assert any(0 < plans(M, N, K)[3] < plans(M, N, K)[2] for M, K, N in large.FORWARD)  # a last round in parts
    right = {plans(K, N, M, right=1, plain=p)[0] for K, M, N in large.RIGHT for p in (0, 1)}
    assert right >= {TILE64, TILE64W, TILE256, TILE128W}
    ragged = {plans(R, N, K, len(c), 1, cut=0)[0] for c, R, K, N in large.RAGGED}
    assert ragged >= {TILE64W, TILE256}
    right = {plans(K, N, R, len(c), 2, 1, p, 0)[0] for c, R, K, N in large.RAGGED_W for p in (0, 1)}
    assert right >= {TILE64, TILE64W, TILE256, TILE128W}
    assert plans.few(1, 515, 3001, 0) and plans.few(2, 16500, 1000, 1) and plans.few(1, 2048, 2048, 1)


def test_plans_hold_for_any_size(plans):
    """Tiles cover the result, parts fit the tickets and the chip's slots, and only what may be cut is."""
    import random
    rng = random.Random(3)
    for _ in range(4000):
        M, N, K = (int(2 ** rng.uniform(0, 17)) for _ in range(3))
        ragged, cut, right, plain = rng.choice([0, 0, 1, 2]), rng.randrange(2), rng.randrange(2), rng.randrange(2)
        groups = rng.randrange(1, 200) if ragged else 1
        t, s, tiles, whole = plans(M, N, K, groups, ragged, right, plain, cut)
        bm, bn, per_cu = (plans.shape(t, k) for k in range(3))
        assert 0 <= t <= TILE128W and (t != TILE128W or (right and plain)) and (t != TILE32 or not (right or ragged))
        if ragged == 0:
            assert tiles == -(-M // bm) * -(-N // bn)
        assert s == 1 or (cut and not ragged)
        if s > 1:
            assert 0 < tiles - whole <= 256 and (tiles - whole) * s <= per_cu * 256 and s <= 16 and K >= 128 * s - 15
        else:
            assert whole == tiles


@pytest.mark.parametrize("name,out", [("mk_moe_ragged_gemm", "out"), ("mk_moe_ragged_dgrad", "out"), ("mk_moe_ragged_wgrad", "dW")])
def test_results_over_the_counts_are_refused(name, out):
    """Workgroups read the counts while others store results already."""
    for at, what in ((7 * FAR, "overlaps counts"), (7 * FAR + 14, "overlaps counts"), (7 * FAR + 2, "counts must be aligned")):
        a = _args(name, {"counts": at if "aligned" in what else 7 * FAR, out: 8 * FAR if "aligned" in what else at})
        assert getattr(capi.lib(), name)(C.byref(a), None) == EINVAL
        assert what in capi.lib().mk_last_error_string().decode()


@pytest.mark.parametrize("name,rows", [("mk_gemm_act", "M"), ("mk_gemm_act_backward", "M"), ("mk_moe_ragged_gemm", "R"),
                                       ("mk_moe_ragged_dgrad", "R"), ("mk_moe_ragged_wgrad", "R")])
def test_rows_beyond_a_launch_are_refused(name, rows):
    """More rows than a kernel that has 64 threads for each can be launched for."""
    a = _args(name, {rows: (1 << 25) + 1})
    assert getattr(capi.lib(), name)(C.byref(a), None) == ESHAPE
    assert "sizes" in capi.lib().mk_last_error_string().decode()
