"""Torch-tensor front end of libmk (device memory and streams come from torch;
every computation runs in libmk's HIP kernels through the C-ABI).

All functions launch on torch's current HIP stream and return immediately.
Shape/argument problems raise :class:`mkernel_amd.capi.MkError`.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import itertools
import math
import threading

import numpy as np
import torch

from . import capi
from .capi import (AgGemmArgs, GemmActArgs, GemmActBackwardArgs, GemmAr2Args, GemmArArgs, GemmArgs, GemmRsArgs,
                   GemmW4Args, MoeCombineArgs, MoeCombineBackwardArgs, MoeFfnArgs, MoeFfnW4Args, MoeGroupedGemmArgs,
                   MoeGroupedGemmW4Args, MoeIndex, MoeIndexDevArgs, MoePermuteArgs, MoeRaggedDgradArgs,
                   MoeRaggedGemmArgs, MoeRaggedWgradArgs, MoeRouteArgs, MoeRouteBackwardArgs, VocabLossArgs,
                   VocabLossBackwardArgs, W4PackArgs, W4QuantizeArgs)


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


# current_stream(i).cuda_stream without the Stream object, where torch has these
# (they are not part of its public interface)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_capturing = torch.cuda.is_current_stream_capturing
_device_index = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream() -> int:
    if not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_device_index())


def _bf16(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 device tensor")


def cu_count() -> int:
    return int(capi.lib().mk_device_cu_count())


_split_ws: dict = {}


def split_workspace(device=None, stream=None) -> torch.Tensor:
    """The K-split workspace the GEMM entry points use by default: one per
    (device, stream), mk_query_workspace_bytes() bytes, zero-filled once
    (every launch leaves it zeroed).  Launches on one stream are ordered, so
    they can share it; launches on different streams get different ones.
    ``stream``: a torch stream, default the current stream of the device.
    Graph capture runs on a stream of its own: fetch the workspace before
    capturing and pass it as ``split_ws``; one first created inside the
    capture has its zero-fill recorded into the graph (about 11 us per
    replay on MI355X).  Every distinct (device, stream handle) keeps its
    workspace (mk_query_workspace_bytes() bytes, ~67 MB on 256 CUs) until
    the process exits or release_split_workspaces() is called; a stream
    created later with a recycled handle reuses that entry, which is safe
    because each launch leaves the workspace zeroed."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
    key = (dev, (torch.cuda.current_stream(dev) if stream is None else stream).cuda_stream)
    ws = _split_ws.get(key)
    if ws is None:
        n = int(capi.lib().mk_query_workspace_bytes(0, 0, 0, 0))
        if n < 0:
            raise capi.MkError("mk_query_workspace_bytes", n, capi.lib().mk_last_error_string().decode())
        ws = torch.zeros(n, dtype=torch.uint8, device=dev)
        _split_ws[key] = ws
    return ws


def release_split_workspaces() -> None:
    """Free every cached default K-split workspace, and the calling thread's
    tickets and small workspaces of the products (after synchronizing every
    device that has one, so no queued launch still uses them)."""
    for dev in {k[0] for k in _split_ws} | {torch.device("cuda", k[0]) for k in _spaces.of}:
        torch.cuda.synchronize(dev)
    _split_ws.clear()
    _spaces.of.clear()


def _ws(split_ws, device) -> tuple:
    """(pointer, bytes) of the K-split workspace: the default one of the
    device's current stream, an explicit tensor, or none at all when
    split_ws is False."""
    if split_ws is False:
        return 0, 0
    if split_ws is None or split_ws is True:
        i = device.index
        ws = _split_ws.get((device, _raw_stream(i))) if i is not None and device.type == "cuda" else None
        if ws is None:
            ws = split_workspace(device)
    else:
        ws = split_ws
    return ws.data_ptr(), ws.numel() * ws.element_size()


def gemm(A: torch.Tensor, B: torch.Tensor, out: torch.Tensor | None = None, num_cus: int = 0,
         tile_m: int = 0, waves: int = 0, split_ws=None) -> torch.Tensor:
    """C = A @ B (bf16 in, fp32 accumulate, bf16 out).  split_ws: None = the
    default per-device K-split workspace, False = no K-split, or a tensor."""
    _bf16(A, "A"); _bf16(B, "B")
    M, K = A.shape
    N = B.shape[1]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=A.device)
    _bf16(out, "C")
    capi.call_values("mk_gemm", GemmArgs, _stream(), A.data_ptr(), B.data_ptr(), out.data_ptr(), M, N, K, K, N, N,
                     num_cus, tile_m, waves, *_ws(split_ws, A.device))
    return out


def ag_gemm(A_shards, A_full, B, C_out, flags, stage_order, epoch: int, gated: bool = True,
            num_producers: int = -1, num_cus: int = 0, spin_limit: int = 0, error_word=None,
            stage_counters=None, split_ws=None, epoch_ptr=None, n_present: int = 0) -> torch.Tensor:
    """Flag-gated AllGather+GEMM; see include/mk.h mk_ag_gemm.  epoch_ptr: an
    optional uint32 device word read for the epoch instead of `epoch`
    (advanced by epoch_advance, e.g. inside a recorded graph).  num_producers
    -1 (default) stages cooperatively, the two halves of the grid taking
    turns to copy ahead; -2 stages cooperatively with every workgroup copying
    an even share before every round; -3 .. -6 run a staging kernel of
    (-2 - num_producers) one-wave workgroups per CU beside the GEMM on a
    side stream (the wave-specialised producer role).  All of them need
    stage_counters (int32 [M/128], zeroed once).  n_present: the first n_present blocks of
    stage_order are already in A_full (published, not copied)."""
    _bf16(A_full, "A_full"); _bf16(B, "B"); _bf16(C_out, "C")
    M, K = A_full.shape
    N = B.shape[1]
    capi.call_values("mk_ag_gemm", AgGemmArgs, _stream(), _ptr(A_shards), _ptr(A_full), _ptr(B), _ptr(C_out), M, N, K,
                     _ptr(flags), _ptr(stage_order), epoch, int(gated), num_producers, num_cus, spin_limit,
                     _ptr(error_word), _ptr(stage_counters), *_ws(split_ws, A_full.device),
                     _ptr(epoch_ptr), n_present)
    return C_out


def gemm_rs(A, B, workspace, output, peer_src, peer_recv, world: int, rank: int, flags, stage_order, epoch: int,
            gated: bool = True, num_producers: int = -1, num_cus: int = 0, spin_limit: int = 0,
            error_word=None, stage_counters=None, split_ws=None, epoch_ptr=None) -> torch.Tensor:
    """GEMM with the reduce-scatter fold in the epilogue; see mk_gemm_rs.
    epoch_ptr: as in ag_gemm."""
    _bf16(A, "A"); _bf16(B, "B")
    M, K = A.shape
    N = B.shape[1]
    capi.call_values("mk_gemm_rs", GemmRsArgs, _stream(), _ptr(A), _ptr(B), _ptr(workspace), _ptr(output),
                     _ptr(peer_src), _ptr(peer_recv), M, N, K, world, rank, _ptr(flags), _ptr(stage_order), epoch,
                     int(gated), num_producers, num_cus, spin_limit, _ptr(error_word), _ptr(stage_counters),
                     *_ws(split_ws, A.device), _ptr(epoch_ptr))
    return output


def gemm_ar(A, B, C_final, peer_src, peer_recv, world: int, flags, stage_order, epoch: int, gated: bool = True,
            num_producers: int = -1, num_cus: int = 0, spin_limit: int = 0, error_word=None, stage_counters=None,
            done_flags=None, split_ws=None, epoch_ptr=None) -> torch.Tensor:
    """GEMM + all-reduce at one rank's share (mk_gemm_ar): C_final = A @ B +
    sum of the world-1 staged peer partials [world-1, M, N], fp32 adds."""
    _bf16(A, "A"); _bf16(B, "B"); _bf16(C_final, "C_final")
    M, K = A.shape
    N = B.shape[1]
    capi.call_values("mk_gemm_ar", GemmArArgs, _stream(), _ptr(A), _ptr(B), _ptr(C_final), _ptr(peer_src),
                     _ptr(peer_recv), M, N, K, world, _ptr(flags), _ptr(stage_order), epoch, int(gated), num_producers,
                     num_cus, spin_limit, _ptr(error_word), _ptr(stage_counters), _ptr(done_flags),
                     *_ws(split_ws, A.device), _ptr(epoch_ptr))
    return C_final


def gemm_ar_two_shot(A, B, C_final, sends, peer_src, peer_recv, peer_reduced, world: int, rank: int, flags,
                     stage_order, epoch: int, gated: bool = True, num_producers: int = -1, num_cus: int = 0,
                     spin_limit: int = 0, error_word=None, stage_counters=None, done_flags=None, split_ws=None,
                     epoch_ptr=None) -> torch.Tensor:
    """GEMM + all-reduce at one rank's share, two-shot (mk_gemm_ar_two_shot):
    this rank's slice of C_final = A @ B + the world-1 staged peer partials
    of that slice ([world-1, M/world, N]); the other slices are the peers'
    reduced rows ``peer_reduced`` ([world-1, M/world, N], slice order
    without ``rank``), staged in; ``sends`` gets this rank's partial rows of
    the other slices.  flags / stage_counters / stage_order cover
    2*(world-1)*(M/world)/128 blocks (partials first, then reduced rows)."""
    _bf16(A, "A"); _bf16(B, "B"); _bf16(C_final, "C_final"); _bf16(sends, "sends")
    M, K = A.shape
    N = B.shape[1]
    capi.call_values("mk_gemm_ar_two_shot", GemmAr2Args, _stream(), _ptr(A), _ptr(B), _ptr(C_final), _ptr(sends),
                     _ptr(peer_src), _ptr(peer_recv), _ptr(peer_reduced), M, N, K, world, rank, _ptr(flags),
                     _ptr(stage_order), epoch, int(gated), num_producers, num_cus, spin_limit, _ptr(error_word),
                     _ptr(stage_counters), _ptr(done_flags), *_ws(split_ws, A.device), _ptr(epoch_ptr))
    return C_final


def epoch_advance(epoch_word: torch.Tensor) -> torch.Tensor:
    """*epoch_word += 1 on the current stream, skipping 0 (mk_epoch_advance);
    epoch_word: a one-element int32/uint32 device tensor."""
    if not epoch_word.is_cuda or epoch_word.numel() != 1 or epoch_word.element_size() != 4:
        raise ValueError("epoch_word must be a one-element 32-bit device tensor")
    capi.check("mk_epoch_advance", capi.lib().mk_epoch_advance(_ptr(epoch_word), C.c_void_p(_stream() or None)))
    return epoch_word


def moe_build_indices(topk_ids: np.ndarray, gates: np.ndarray, e0: int, n_local: int,
                      row_block: int = capi.ROW_BLOCK) -> dict:
    """Host-side routing index build (libmk C++); returns numpy arrays."""
    ids = np.ascontiguousarray(topk_ids, dtype=np.int32)
    g = np.ascontiguousarray(gates, dtype=np.float32)
    T, k = ids.shape
    L = capi.lib()
    R, Rp = C.c_int64(), C.c_int64()
    p = lambda a: a.ctypes.data_as(C.c_void_p)
    capi.check("mk_moe_index_sizes", L.mk_moe_index_sizes(p(ids), T, k, e0, n_local, row_block, C.byref(R), C.byref(Rp)))
    R, Rp = R.value, Rp.value
    o = {
        "padded_tokens_per_expert": np.zeros(n_local, np.int32),
        "local_rb_per_expert": np.zeros(n_local, np.int32),
        "pull_indices": np.zeros((Rp, 3), np.int32),
        "row_expert": np.zeros(Rp, np.int32),
        "rb_expert": np.zeros(Rp // row_block, np.int32),
        "rb_rows": np.zeros(Rp // row_block, np.int32),
        "row_weight": np.zeros(Rp, np.float32),
        "owner_offset": np.zeros(T + 1, np.int32),
        "row_to_slot": np.zeros(Rp, np.int32),
        "row_to_owner": np.zeros(Rp, np.int32),
        "slot_to_row": np.zeros(max(R, 1), np.int32),
    }
    idx = MoeIndex(*[p(o[f]) for f, _ in MoeIndex._fields_])
    capi.check("mk_moe_build_indices", L.mk_moe_build_indices(p(ids), p(g), T, k, e0, n_local, row_block, C.byref(idx)))
    o["slot_to_row"] = o["slot_to_row"][:R]
    o["R"], o["R_pad"] = R, Rp
    return o


_INDEX_TABLES = ("padded_tokens_per_expert", "local_rb_per_expert", "pull_indices", "row_expert", "rb_expert",
                 "rb_rows", "row_weight", "owner_offset", "row_to_slot", "row_to_owner", "slot_to_row")


def moe_build_indices_dev(topk_ids: torch.Tensor, gates: torch.Tensor, e0: int, n_local: int,
                          row_block: int = capi.ROW_BLOCK, sync: bool = True) -> dict:
    """Routing index build on the GPU (mk_moe_build_indices_dev) from device
    top-k ids (int32) and gates (float32) [T, k].  Tables are allocated at
    the worst-case capacity; with sync=True the sizes are read back and the
    returned tensors are views trimmed to R / R_pad rows (the same dict
    layout as moe_build_indices, as device tensors).  With sync=False nothing
    is read back: the tables stay at their capacity and "sizes" holds the
    device int64 {R, R_pad} for moe_ffn_combine(..., sizes=...).
    All tables are pieces of one buffer, which holds the build's workspace too
    and lives as long as any of them (about 32 bytes per row of the capacity;
    clone() a table to keep or store it alone).  The tables by row
    (pull_indices, row_expert, row_weight, row_to_slot, row_to_owner,
    slot_to_row) start at multiples of 512 bytes where row_block is a multiple
    of 128, the others at multiples of 4."""
    if topk_ids.dtype != torch.int32 or gates.dtype != torch.float32 or not topk_ids.is_cuda:
        raise ValueError("topk_ids must be int32 and gates float32 device tensors")
    ids = topk_ids.contiguous()
    g = gates.contiguous()
    T, k = ids.shape
    dev = ids.device
    # worst case, rounded to whole row blocks so the capacity is a valid
    # row count for the grouped GEMMs
    cap = (T * k + n_local * (row_block - 1) + row_block - 1) // row_block * row_block
    wsb = int(capi.lib().mk_moe_index_workspace_bytes(T, k, n_local))
    # one allocation for the tables and the workspace: 13 took most of the call.  Behind the sizes' 512 bytes the
    # row tables: whole row blocks, so that each starts where an allocation might
    nb = (cap + row_block - 1) // row_block
    parts = (4, 124, 3 * cap, cap, cap, cap, cap, max(cap, 1), n_local, n_local, nb, nb, T + 1, max(wsb, 4) // 4)
    buf = torch.empty(sum(parts), dtype=torch.int32, device=dev)
    # ("unsafe": pieces that autograd does not know as views, which tables need not be; 4.1 us with views, so 2.9)
    sizes, _, pull, row_expert, weight, to_slot, to_owner, to_row, padded, local_rb, rb_expert, rb_rows, offset, _ = \
        torch.unsafe_split_with_sizes(buf, parts)
    t = dict(zip(_INDEX_TABLES, (padded, local_rb, pull.view(cap, 3), row_expert, rb_expert, rb_rows,
                                 weight.view(torch.float32), offset, to_slot, to_owner, to_row)))
    sizes = sizes.view(torch.int64)  # both words are written by the build
    at, _, a_pull, a_expert, a_weight, a_slot, a_owner, a_row, a_padded, a_local, a_rb, a_rows, a_offset, ws = \
        itertools.accumulate((4 * n for n in parts[:-1]), initial=buf.data_ptr())
    capi.call_values("mk_moe_build_indices_dev", MoeIndexDevArgs, _stream(), ids.data_ptr(), g.data_ptr(), T, k, e0,
                     n_local, row_block, cap, ws, wsb, at, a_padded, a_local, a_pull, a_expert, a_rb, a_rows, a_weight,
                     a_offset, a_slot, a_owner, a_row)
    if not sync:
        t["sizes"] = sizes
        return t
    R, Rp = (int(v) for v in sizes.cpu())
    for f in ("pull_indices", "row_expert", "row_weight", "row_to_slot", "row_to_owner"):
        t[f] = t[f][:Rp]
    t["rb_expert"] = t["rb_expert"][:Rp // row_block]
    t["rb_rows"] = t["rb_rows"][:Rp // row_block]
    t["slot_to_row"] = t["slot_to_row"][:R]
    t["R"], t["R_pad"] = R, Rp
    return t


def moe_permute(tokens, pull, post, tokens_per_src: int | None = None, devs_per_node: int = 1, sizes=None):
    """sizes: optional device int64 {R, R_pad}; post's rows are then a
    capacity and rows past R_pad are skipped."""
    _bf16(tokens, "tokens"); _bf16(post, "post_tokens")
    R_pad, H = post.shape
    tps = tokens.shape[0] if tokens_per_src is None else tokens_per_src
    capi.call_values("mk_moe_permute", MoePermuteArgs, _stream(), _ptr(tokens), _ptr(pull), _ptr(post), R_pad, H,
                     tokens.shape[0], tps, devs_per_node, _ptr(sizes))
    return post


def moe_grouped_gemm(A, W, out, rb_expert=None, padded_tokens_per_expert=None, mode: int = 0, num_cus: int = 0,
                     rb_rows=None, split_ws=None, gather_pull=None, tokens_per_src: int | None = None,
                     devs_per_node: int = 1, tile_n: int = 0, sizes=None):
    """mode 0: out = A @ W[e]; mode 1: out = silu(h[:, :I]) * h[:, I:], h = A @ W[e].
    tile_n: output tile width 256 or 512 (0: the library's choice).  sizes:
    optional device int64 {R, R_pad}; the row count is then a capacity and
    row tiles past R_pad are not computed."""
    _bf16(A, "A"); _bf16(W, "W"); _bf16(out, "out")
    # with gather_pull, A is the token buffer and the rows come from the pull table
    R_pad = gather_pull.shape[0] if gather_pull is not None else A.shape[0]
    K = A.shape[1]
    E, _, Nw = W.shape
    tps = A.shape[0] if tokens_per_src is None else tokens_per_src
    capi.call_values("mk_moe_grouped_gemm", MoeGroupedGemmArgs, _stream(), _ptr(A), _ptr(W), _ptr(out),
                     _ptr(rb_expert), _ptr(padded_tokens_per_expert), _ptr(rb_rows), R_pad, K, Nw, E, mode, num_cus,
                     *_ws(split_ws, A.device), _ptr(gather_pull), A.shape[0], tps, devs_per_node, tile_n, _ptr(sizes))
    return out


def moe_tile_rows(pull, rb_rows):
    """rb_rows[b] = real rows in row block b (from the pull table)."""
    capi.check("mk_moe_tile_rows", capi.lib().mk_moe_tile_rows(_ptr(pull), pull.shape[0], _ptr(rb_rows),
                                                               C.c_void_p(_stream() or None)))
    return rb_rows


def moe_invert_slots(row_to_slot, row_to_owner, slot_to_row, owner: int = 0, error_word=None):
    """slot_to_row[:] = -1, then slot_to_row[row_to_slot[r]] = r for the rows
    of `owner` (mk_moe_invert_slots); slots past slot_to_row's length set
    bit 1 of error_word."""
    capi.check("mk_moe_invert_slots", capi.lib().mk_moe_invert_slots(
        _ptr(row_to_slot), _ptr(row_to_owner), row_to_slot.numel(), owner, slot_to_row.numel(), _ptr(slot_to_row),
        _ptr(error_word), C.c_void_p(_stream() or None)))
    return slot_to_row


def moe_combine(y_expert, row_weight, owner_offset, slot_to_row, y_out):
    _bf16(y_expert, "y_expert")
    T, H = y_out.shape
    od = 0 if y_out.dtype == torch.float32 else 1
    if od == 1 and y_out.dtype != torch.bfloat16:
        raise ValueError("y_out must be float32 or bfloat16")
    capi.call_values("mk_moe_combine", MoeCombineArgs, _stream(), _ptr(y_expert), _ptr(row_weight), _ptr(owner_offset),
                     _ptr(slot_to_row), _ptr(y_out), T, H, od)
    return y_out


def moe_ffn_combine(tokens, pull, row_weight, owner_offset, slot_to_row, w1, w2, post, act, y_expert, y_out,
                    rb_expert=None, padded_tokens_per_expert=None, tokens_per_src: int | None = None,
                    devs_per_node: int = 1, num_cus: int = 0, rb_rows=None, split_ws=None,
                    fuse_dispatch: bool = False, tile_n: int = 0, sizes=None):
    """permute -> grouped GEMM1 + SwiGLU -> grouped GEMM2 -> combine.  With
    fuse_dispatch, GEMM1 reads the token rows through the pull table itself
    (no permute kernel, post may be None and is not written).  sizes: the
    device {R, R_pad} of moe_build_indices_dev(sync=False); the tables and
    buffers are then at their capacity and nothing is read back to the host
    (the call can be recorded in a CUDA/HIP graph)."""
    T, H = y_out.shape
    E, _, I2 = w1.shape
    R_pad = pull.shape[0]
    od = 0 if y_out.dtype == torch.float32 else 1
    tps = tokens.shape[0] if tokens_per_src is None else tokens_per_src
    capi.call_values("mk_moe_ffn_combine", MoeFfnArgs, _stream(), _ptr(tokens), _ptr(pull), _ptr(rb_expert),
                     _ptr(padded_tokens_per_expert), _ptr(rb_rows), _ptr(row_weight), _ptr(owner_offset),
                     _ptr(slot_to_row), _ptr(w1), _ptr(w2), _ptr(post), _ptr(act), _ptr(y_expert), _ptr(y_out), T,
                     tokens.shape[0], R_pad, H, I2 // 2, E, tps, devs_per_node, od, num_cus,
                     *_ws(split_ws, tokens.device), int(fuse_dispatch), tile_n, _ptr(sizes))
    return y_out


# ------------------------------------------------------------------- router
def _tensor(t, name: str, dtypes, shape=None, dim=None, rows=False, device=None) -> None:
    """Checks one device tensor: type, shape (None: any size) and layout
    (contiguous, or with `rows` a matrix whose rows are), on `device`."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor of type {' or '.join(str(d)[6:] for d in dtypes)}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and w != n for w, n in zip(shape, t.shape))):
        raise ValueError(f"{name} must have shape {tuple('any' if w is None else w for w in shape)}, not {tuple(t.shape)}")
    if rows:
        if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{name} must be a matrix with contiguous rows that do not overlap")
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _is(t, dtype, shape, device) -> bool:
    """The usual case of _tensor, in a third of its time."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device
            and t.is_contiguous())


def _vector(t, name: str, device) -> None:
    """An int32 table of any length."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.dim() == 1 and t.device == device
            and t.is_contiguous()):
        _tensor(t, name, _I32, dim=1, device=device)


def _ld(t: torch.Tensor) -> int:
    """Row stride; of a matrix of one row, its width."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _on(device):
    """The device as the current one for a launch, where it is not that already."""
    return contextlib.nullcontext() if device.index == _device_index() else torch.cuda.device(device)


_LOGITS = (torch.float32, torch.bfloat16)
_F32, _BF16, _I32, _U8 = (torch.float32,), (torch.bfloat16,), (torch.int32,), (torch.uint8,)


_NO_BALANCE = (0, 0, 0, 0, 0.0, 0, 0)


def _route_inputs(logits, topk, token_mask):
    if not (isinstance(logits, torch.Tensor) and logits.dtype in _LOGITS and logits.is_cuda and logits.dim() == 2
            and logits.is_contiguous()):
        _tensor(logits, "logits", _LOGITS, rows=True)
    T, E = logits.shape
    if not 1 <= topk <= E:
        raise ValueError(f"topk must be 1 .. {E}")
    if token_mask is not None and not _is(token_mask, torch.bool, (T,), logits.device):
        _tensor(token_mask, "token_mask", (torch.bool, torch.uint8), (T,), device=logits.device)
    return T, E, logits.device


def _coef(coef) -> float:
    coef = float(coef)
    if not math.isfinite(C.c_float(coef).value):
        raise ValueError("coef must be finite in fp32")
    return coef


def moe_route(logits: torch.Tensor, topk: int, renorm: bool = True, token_mask: torch.Tensor | None = None) -> tuple:
    """Top-k choice and gates of the router (mk_moe_route): (ids int32, gates
    float32), both [T, topk], as moe_build_indices_dev takes them.  logits:
    float32 or bfloat16 [T, E], rows contiguous (columns of a wider matrix are
    fine).  Choices come in falling order, ties to the lowest expert; -inf is
    never chosen (id -1, gate 0 in the places left).  gates: softmax over the
    chosen logits, or with renorm=False the chosen entries of the softmax over
    all.  token_mask (bool or uint8 [T]): tokens where it is 0 get ids -1.
    Nothing is recorded for autograd: moe_route_backward is called by hand."""
    return _route(logits, topk, renorm, token_mask, None)[:2]


def moe_route_balance(logits: torch.Tensor, topk: int, coef: float, renorm: bool = True,
                      token_mask: torch.Tensor | None = None) -> dict:
    """moe_route for training: ids and gates, and of the same pass "counts"
    (int32 [E], choices of each expert), "prob_sum" (float32 [E], sum of its
    probabilities over the tokens), "tokens" (int32 [1], tokens that count) and
    "loss" (float32 [1]) = coef * E / (topk * tokens^2) * sum(counts * prob_sum).
    Bitwise repeatable.  moe_route_backward has the gradient."""
    ids, gates, loss, counts, prob_sum, tokens = _route(logits, topk, renorm, token_mask, _coef(coef))
    return {"ids": ids, "gates": gates, "loss": loss, "counts": counts, "prob_sum": prob_sum, "tokens": tokens}


def _route(logits, topk, renorm, token_mask, coef):
    T, E, dev = _route_inputs(logits, topk, token_mask)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return _route(logits, topk, renorm, token_mask, coef)
    ids = torch.empty(T, topk, dtype=torch.int32, device=dev)
    gates = torch.empty_like(ids, dtype=torch.float32)
    out, balance = (ids, gates), _NO_BALANCE
    if coef is not None:
        # loss, prob_sum, counts and tokens in one tensor; the workspace in another (it holds nothing between calls)
        sums = torch.empty(2 * E + 2, dtype=torch.int32, device=dev)
        n = capi.lib().mk_moe_route_workspace_bytes(T, E)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
        at = sums.data_ptr()
        balance = (at + 4 + 4 * E, at + 4, at + 4 + 8 * E, at, coef, ws.data_ptr(), n)
        loss, prob_sum, counts, tokens = torch.unsafe_split_with_sizes(sums, (1, E, E, 1))
        out += (loss.view(torch.float32), counts, prob_sum.view(torch.float32), tokens)
    capi.call_values("mk_moe_route", MoeRouteArgs, _raw_stream(dev.index), logits.data_ptr(),
                     0 if token_mask is None else token_mask.data_ptr(), ids.data_ptr(), gates.data_ptr(), T,
                     logits.stride(0) if T > 1 else E, E, topk, logits.dtype is torch.bfloat16, bool(renorm), *balance)
    return out


def moe_route_backward(logits: torch.Tensor, ids: torch.Tensor, dgates: torch.Tensor | None = None,
                       dloss: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                       tokens: torch.Tensor | None = None, coef: float = 0.0, renorm: bool = True,
                       token_mask: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of the logits (mk_moe_route_backward), in their type: the
    gates' part from dgates (float32 [T, topk]), the balance loss's part from
    counts and tokens (as moe_route_balance gave them, or summed over ranks),
    coef and dloss (one float32 on the device; None: 1).  Either part may be
    left out.  ids, renorm and token_mask as in the forward call.  out: where
    to write it; the logits themselves may be given, but no other tensor that
    shares elements with them."""
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError("ids must be an int32 device tensor [T, topk]")
    topk = ids.shape[1]
    T, E, dev = _route_inputs(logits, topk, token_mask)
    if not _is(ids, torch.int32, (T, topk), dev):
        _tensor(ids, "ids", _I32, (T, topk), device=dev)
    if dgates is None and counts is None:
        raise ValueError("dgates or counts must be given")
    if dgates is not None and not _is(dgates, torch.float32, (T, topk), dev):
        _tensor(dgates, "dgates", _F32, (T, topk), device=dev)
    if counts is not None:
        if not _is(counts, torch.int32, (E,), dev):
            _tensor(counts, "counts", _I32, (E,), device=dev)
        if not _is(tokens, torch.int32, (1,), dev):
            if tokens is None:
                raise ValueError("counts needs tokens")
            _tensor(tokens, "tokens", _I32, device=dev)
            if tokens.numel() != 1:
                raise ValueError("tokens must hold one number")
    if dloss is not None and not _is(dloss, torch.float32, (1,), dev):
        _tensor(dloss, "dloss", _F32, device=dev)
        if dloss.numel() != 1:
            raise ValueError("dloss must hold one number")
    if out is not None:
        _tensor(out, "out", (logits.dtype,), (T, E), rows=True, device=dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_route_backward(logits, ids, dgates, dloss, counts, tokens, coef, renorm, token_mask, out)
    if out is None:
        out = logits.new_empty(T, E)
    capi.call_values("mk_moe_route_backward", MoeRouteBackwardArgs, _raw_stream(dev.index), logits.data_ptr(), _ptr(token_mask),
                     ids.data_ptr(), _ptr(dgates), _ptr(dloss), _ptr(counts), _ptr(tokens), out.data_ptr(), T,
                     _ld(logits), _ld(out), E, topk, logits.dtype is torch.bfloat16, bool(renorm), _coef(coef))
    return out


def moe_combine_backward(dy: torch.Tensor, y_expert: torch.Tensor, ids: torch.Tensor, row_weight: torch.Tensor,
                         owner_offset: torch.Tensor, slot_to_row: torch.Tensor, rb_rows: torch.Tensor, e0: int,
                         n_local: int, dy_expert: torch.Tensor | None = None, dgates: torch.Tensor | None = None,
                         sizes: torch.Tensor | None = None) -> tuple:
    """Gradient of moe_combine (mk_moe_combine_backward): (dy_expert bf16
    [R_pad, H], dgates float32 [T, topk]) from dy ([T, H], the type of the
    combine's output), with the tables of moe_build_indices(_dev)(ids, ...,
    e0, n_local) at row_block 128.  dgates is 0 for experts of other ranks.
    With sizes (moe_build_indices_dev(sync=False)) the rows are a capacity and
    those behind the routed ones are left as they are.  dy_expert may be
    y_expert itself, but shares no other memory with y_expert or dy."""
    _tensor(dy, "dy", _LOGITS, dim=2)
    dev = dy.device
    T, H = dy.shape
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_combine_backward(dy, y_expert, ids, row_weight, owner_offset, slot_to_row, rb_rows, e0, n_local,
                                        dy_expert, dgates, sizes)
    _tensor(y_expert, "y_expert", _BF16, (None, H), device=dev)
    R_pad = y_expert.shape[0]
    _tensor(ids, "ids", _I32, (T, None), device=dev)
    k = ids.shape[1]
    if not _is(row_weight, torch.float32, (R_pad,), dev):
        _tensor(row_weight, "row_weight", _F32, dim=1, device=dev)
    if not _is(owner_offset, torch.int32, (T + 1,), dev):
        _tensor(owner_offset, "owner_offset", _I32, (T + 1,), device=dev)
    _vector(slot_to_row, "slot_to_row", dev)
    _vector(rb_rows, "rb_rows", dev)
    if row_weight.shape[0] < R_pad or rb_rows.shape[0] * capi.ROW_BLOCK < R_pad:
        raise ValueError("row_weight and rb_rows must cover the rows of y_expert")
    if not (0 <= e0 < 2**31 and 0 < n_local < 2**31):
        raise ValueError("experts e0 .. e0 + n_local must be numbers of 32 bits")
    if sizes is not None and not _is(sizes, torch.int64, (2,), dev):
        _tensor(sizes, "sizes", (torch.int64,), (2,), device=dev)
    if dy_expert is None:
        dy_expert = torch.empty_like(y_expert)
    elif not _is(dy_expert, torch.bfloat16, (R_pad, H), dev):
        _tensor(dy_expert, "dy_expert", _BF16, (R_pad, H), device=dev)
    if dgates is None:
        dgates = torch.empty_like(ids, dtype=torch.float32)
    elif not _is(dgates, torch.float32, (T, k), dev):
        _tensor(dgates, "dgates", _F32, (T, k), device=dev)
    capi.call_values("mk_moe_combine_backward", MoeCombineBackwardArgs, _raw_stream(dev.index), dy.data_ptr(),
                     y_expert.data_ptr(), ids.data_ptr(), row_weight.data_ptr(), owner_offset.data_ptr(),
                     slot_to_row.data_ptr(), rb_rows.data_ptr(), dy_expert.data_ptr(), dgates.data_ptr(), T, H,
                     R_pad, k, e0, n_local, dy.dtype is torch.bfloat16, _ptr(sizes))
    return dy_expert, dgates


# ------------------------------------------------------------------- 4-bit weights
class W4Weights:
    """4-bit weights laid out by w4_pack: ``experts`` matrices [K, N], values
    (code - zero) * scale per ``group`` rows of K, in one uint8 tensor
    ``packed`` that may be stored and made W4Weights again."""
    __slots__ = ("packed", "K", "N", "group", "experts", "zeros")

    def __init__(self, packed: torch.Tensor, K: int, N: int, group: int, experts: int = 1, zeros: bool = False):
        _tensor(packed, "packed", _U8, dim=1)
        n = capi.lib().mk_w4_packed_bytes(K, N, experts, group, bool(zeros))
        if n < 0:
            raise ValueError(f"no 4-bit weights of {experts} x {K} x {N} in groups of {group}")
        if packed.numel() != n:
            raise ValueError(f"packed holds {packed.numel()} bytes, {experts} x {K} x {N} takes {n}")
        self.packed, self.K, self.N, self.group, self.experts, self.zeros = packed, K, N, group, experts, bool(zeros)

    def _values(self) -> tuple:
        return self.packed.data_ptr(), self.K, self.N, self.group, self.experts, self.zeros


def _groups(K: int, group: int) -> int:
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    return (K + group - 1) // group


def _matrices(t, name, dtypes):
    _tensor(t, name, dtypes)
    if t.dim() not in (2, 3) or 0 in t.shape:
        raise ValueError(f"{name} must be [K, N] or [E, K, N], not empty")
    return (1, *t.shape) if t.dim() == 2 else tuple(t.shape)


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, group: int, zeros: torch.Tensor | None = None) -> W4Weights:
    """Lays 4-bit weights out for gemm_w4 and the expert products (mk_w4_pack;
    once, when a model is loaded).  codes: uint8 [K, N] or [E, K, N], one code
    0 .. 15 a byte; scales: bf16 [.., ceil(K / group), N] (fp16 scales have to be
    rounded to it, which takes three of their bits); zeros: uint8 of the scales'
    shape, or None (8)."""
    E, K, N = _matrices(codes, "codes", _U8)
    shape = (*codes.shape[:-2], _groups(K, group), N)
    _tensor(scales, "scales", _BF16, shape, device=codes.device)
    if zeros is not None:
        _tensor(zeros, "zeros", _U8, shape, device=codes.device)
    dev = codes.device
    n = capi.lib().mk_w4_packed_bytes(K, N, E, group, zeros is not None)
    with _on(dev):
        w = W4Weights(torch.empty(max(n, 0), dtype=torch.uint8, device=dev), K, N, group, E, zeros is not None)
        capi.call_values("mk_w4_pack", W4PackArgs, _stream(), codes.data_ptr(), scales.data_ptr(), _ptr(zeros),
                         *w._values())
    return w


def w4_quantize(W: torch.Tensor, group: int) -> tuple:
    """(codes, scales) of bf16 weights [K, N] or [E, K, N] for w4_pack
    (mk_w4_quantize): per group scale = bf16(largest magnitude / 7), code =
    round(w / scale) + 8."""
    E, K, N = _matrices(W, "W", _BF16)
    dev = W.device
    with _on(dev):
        codes = torch.empty(W.shape, dtype=torch.uint8, device=dev)
        scales = torch.empty((*W.shape[:-2], _groups(K, group), N), dtype=torch.bfloat16, device=dev)
        capi.call_values("mk_w4_quantize", W4QuantizeArgs, _stream(), W.data_ptr(), codes.data_ptr(),
                         scales.data_ptr(), K, N, group, E)
    return codes, scales


def _w4(W, name, device, experts=None) -> None:
    if not isinstance(W, W4Weights):
        raise ValueError(f"{name} must be W4Weights (w4_pack)")
    if W.packed.device != device:
        raise ValueError(f"{name} is on {W.packed.device}, not on {device}")
    if experts is not None and W.experts != experts:
        raise ValueError(f"{name} holds {W.experts} matrices, not {experts}")


def gemm_w4(A: torch.Tensor, W: W4Weights, out: torch.Tensor | None = None) -> torch.Tensor:
    """C = A @ w for few rows (mk_gemm_w4): A bf16 [M, K], w 4-bit weights of
    w4_pack; fp32 sums of exact products, scaled group by group in fp32; out
    bf16 (what is made where none is given) or float32.  K a multiple of 8, any
    M and N; rows of A (a multiple of 8 elements apart, the first 16-byte
    aligned) and of out need only be contiguous each; out may not overlap A.  The weights are expanded for
    every 16 or 32 rows: beyond about 128 rows gemm with bf16 weights is faster
    (1024 x 3584 x 8192: 108 us and 55)."""
    if not (isinstance(A, torch.Tensor) and A.dtype is torch.bfloat16 and A.is_cuda and A.dim() == 2
            and A.is_contiguous()):
        _tensor(A, "A", _BF16, rows=True)
    dev = A.device
    if type(W) is not W4Weights or W.experts != 1 or W.packed.device != dev:
        _w4(W, "W", dev, 1)
    M, K = A.shape
    N = W.N
    if K != W.K:
        raise ValueError(f"A has {K} columns, the weights {W.K} rows")
    if out is not None:
        _tensor(out, "out", _LOGITS, (M, N), rows=True, device=dev)
    index = dev.index
    if index != _device_index():
        with torch.cuda.device(dev):
            return gemm_w4(A, W, out)
    if out is None:
        out, ldc, bf16 = A.new_empty(M, N), N, True
    else:
        ldc, bf16 = _ld(out), out.dtype is torch.bfloat16
    capi.call_values("mk_gemm_w4", GemmW4Args, _raw_stream(index), A.data_ptr(), out.data_ptr(), *W._values(), M,
                     A.stride(0) if M > 1 else K, ldc, bf16)
    return out


def _block_tables(rb_expert, rb_rows, R_pad, sizes, dev):
    n = R_pad // capi.ROW_BLOCK
    if R_pad % capi.ROW_BLOCK:
        raise ValueError(f"the tables' rows must be a multiple of {capi.ROW_BLOCK}")
    for t, name in ((rb_expert, "rb_expert"), (rb_rows, "rb_rows")):
        if (t is None and name == "rb_rows") or _is(t, torch.int32, (n,), dev):
            continue
        _tensor(t, name, _I32, dim=1, device=dev)
        if t.shape[0] < n:
            raise ValueError(f"{name} must cover the rows")
    if sizes is not None and not _is(sizes, torch.int64, (2,), dev):
        _tensor(sizes, "sizes", (torch.int64,), (2,), device=dev)


def moe_grouped_gemm_w4(A: torch.Tensor, W: W4Weights, out: torch.Tensor, rb_expert: torch.Tensor,
                        rb_rows: torch.Tensor | None = None, mode: int = 0,
                        gather_pull: torch.Tensor | None = None, tokens_per_src: int | None = None,
                        devs_per_node: int = 1, sizes: torch.Tensor | None = None) -> torch.Tensor:
    """moe_grouped_gemm with 4-bit expert weights (mk_moe_grouped_gemm_w4), for
    the few rows per expert of a decode batch.  mode 0: out = A @ w[e]; mode 1:
    out = silu(h[:, :I]) * h[:, I:], h = A @ w[e].  Only the real rows (rb_rows)
    of the 128-row blocks are computed and written.  out is float32, bfloat16 or,
    with twice the columns, a bfloat16 pair: the rounded values and behind them
    what the rounding left; A may hold such pairs ([R_pad, 2 K])."""
    _tensor(A, "A", _BF16, dim=2)
    dev = A.device
    _w4(W, "W", dev)
    if mode not in (0, 1):
        raise ValueError("mode must be 0 or 1")
    R_pad = A.shape[0] if gather_pull is None else gather_pull.shape[0]
    parts = 2 if gather_pull is None and A.shape[1] == 2 * W.K else 1
    if A.shape[1] != W.K * parts:
        raise ValueError(f"A has {A.shape[1]} columns, the weights {W.K} rows")
    width = W.N // 2 if mode else W.N
    _tensor(out, "out", _LOGITS, (R_pad, None), device=dev)
    pair = out.dtype == torch.bfloat16 and out.shape[1] == 2 * width
    if out.shape[1] != width and not pair:
        raise ValueError(f"out has {out.shape[1]} columns, not {width}")
    _block_tables(rb_expert, rb_rows, R_pad, sizes, dev)
    if gather_pull is not None:
        _tensor(gather_pull, "gather_pull", _I32, (R_pad, 3), device=dev)
    tps = A.shape[0] if tokens_per_src is None else tokens_per_src
    with _on(dev):
        capi.call_values("mk_moe_grouped_gemm_w4", MoeGroupedGemmW4Args, _stream(), A.data_ptr(), *W._values(),
                         out.data_ptr(), rb_expert.data_ptr(), _ptr(rb_rows), R_pad, mode, parts,
                         2 if pair else int(out.dtype == torch.bfloat16), _ptr(gather_pull), A.shape[0], tps,
                         devs_per_node, _ptr(sizes))
    return out


def moe_ffn_combine_w4(tokens: torch.Tensor, pull: torch.Tensor, row_weight: torch.Tensor, owner_offset: torch.Tensor,
                       slot_to_row: torch.Tensor, w1: W4Weights, w2: W4Weights, act: torch.Tensor,
                       y_expert: torch.Tensor, y_out: torch.Tensor, rb_expert: torch.Tensor,
                       rb_rows: torch.Tensor | None = None, tokens_per_src: int | None = None, devs_per_node: int = 1,
                       sizes: torch.Tensor | None = None) -> torch.Tensor:
    """moe_ffn_combine with 4-bit expert weights w1 [E, H, 2I] and w2 [E, I, H]
    (mk_moe_ffn_combine_w4), for decode batches: grouped GEMM1 + SwiGLU (reads
    the tokens through the pull table) -> grouped GEMM2 -> combine.  act
    (bfloat16 [R_pad, 2 I]: rounded values and what the rounding left, 17 bits
    together) and y_expert (float32 [R_pad, H]) are scratch; y_out is bfloat16 or
    float32 and may be the tokens' memory; sizes as in moe_ffn_combine.  Codes are
    expanded for every 16 rows of an expert (8 in the second product): beyond
    about 1000 tokens (7168 / 2048, 32 of 256 experts) the bf16 layer is faster."""
    if not (isinstance(tokens, torch.Tensor) and tokens.dtype is torch.bfloat16 and tokens.is_cuda
            and tokens.dim() == 2 and tokens.is_contiguous()):
        _tensor(tokens, "tokens", _BF16, dim=2)
    dev = tokens.device
    _w4(w1, "w1", dev)
    _w4(w2, "w2", dev, w1.experts)
    n, H = tokens.shape
    I = w2.K
    if w1.N != 2 * I or w2.N != H or w1.K != H:
        raise ValueError("w1 must be [E, H, 2I], w2 [E, I, H] and tokens [n, H]")
    if not (isinstance(pull, torch.Tensor) and _is(pull, torch.int32, (*pull.shape[:1], 3), dev)):
        _tensor(pull, "pull", _I32, (None, 3), device=dev)
    R_pad = pull.shape[0]
    if not _is(act, torch.bfloat16, (R_pad, 2 * I), dev):
        _tensor(act, "act", _BF16, (R_pad, 2 * I), device=dev)
    if not _is(y_expert, torch.float32, (R_pad, H), dev):
        _tensor(y_expert, "y_expert", _F32, (R_pad, H), device=dev)
    _tensor(y_out, "y_out", _LOGITS, (None, H), device=dev)
    T = y_out.shape[0]
    if T == 0 and n == 0:
        return y_out
    if not _is(row_weight, torch.float32, (R_pad,), dev):
        _tensor(row_weight, "row_weight", _F32, dim=1, device=dev)
        if row_weight.shape[0] < R_pad:
            raise ValueError("row_weight must cover the rows")
    if not _is(owner_offset, torch.int32, (T + 1,), dev):
        _tensor(owner_offset, "owner_offset", _I32, (T + 1,), device=dev)
    _vector(slot_to_row, "slot_to_row", dev)
    _block_tables(rb_expert, rb_rows, R_pad, sizes, dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_ffn_combine_w4(tokens, pull, row_weight, owner_offset, slot_to_row, w1, w2, act, y_expert,
                                      y_out, rb_expert, rb_rows, tokens_per_src, devs_per_node, sizes)
    capi.call_values("mk_moe_ffn_combine_w4", MoeFfnW4Args, _raw_stream(dev.index), tokens.data_ptr(), pull.data_ptr(),
                     rb_expert.data_ptr(), _ptr(rb_rows), row_weight.data_ptr(), owner_offset.data_ptr(),
                     slot_to_row.data_ptr(), *w1._values(), *w2._values(), act.data_ptr(), y_expert.data_ptr(),
                     y_out.data_ptr(), T, n, R_pad, n if tokens_per_src is None else tokens_per_src, devs_per_node,
                     y_out.dtype is torch.bfloat16, _ptr(sizes))
    return y_out


# ------------------------------------------------------------------- products with what follows them
# Tickets (zeroed words by which the parts of a product's K meet, left zeroed by every launch) and behind them a small
# workspace: one set per thread, device and stream, whose launches are ordered (the launches of two threads' calls on
# one stream may come between each other).  They go with their thread, or by release_split_workspaces.
_SPACE = 4 << 20
_UNTOUCHED = 16  # in place of tickets that a call does not touch


class _Spaces(threading.local):
    def __init__(self):
        self.of = {}


_spaces = _Spaces()


def _space(index: int, stream: int) -> int:
    t = _spaces.of.get((index, stream))
    if t is None:
        n = capi.PRODUCT_TICKETS * 4
        t = torch.empty(n + _SPACE, dtype=torch.uint8, device=torch.device("cuda", index))
        t[:n].zero_()
        _spaces.of[index, stream] = t
    return t.data_ptr()


def _product(fn: str, cls, device, cut: bool, *values) -> None:
    """Calls an entry point whose arguments end with a workspace (and, with
    cut, tickets): the stream's small one where that is enough, else memory of
    its own, which the caching allocator reuses in stream order.  Inside a
    graph's capture both are the graph's (torch keeps what it allocates there
    for it), the tickets' zeros recorded with it where the call touches them:
    graphs may then run beside each other and beside eager calls."""
    index = device.index
    stream = _raw_stream(index)
    if _capturing():
        # (tickets that are not touched: any address)
        words = capi.ticket_words(fn, cls, *values) if cut else 0
        at = torch.zeros(words, dtype=torch.int32, device=device) if words else None
        tickets = (at.data_ptr() if words else _UNTOUCHED,) if cut else ()
    else:
        at = _space(index, stream)
        tickets = (at,) if cut else ()
        if capi.call_with_workspace(fn, cls, stream, *values, at + capi.PRODUCT_TICKETS * 4, _SPACE, *tickets):
            return
    n = capi.workspace_bytes(fn, cls, *values)
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    capi.call_values(fn, cls, stream, *values, ws.data_ptr(), n, *tickets)


def _rows(t, name: str, dtypes, shape, device) -> None:
    """A matrix with contiguous rows, any distance apart."""
    if not (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.shape == shape and t.device == device
            and t.is_contiguous()):
        _tensor(t, name, dtypes, shape, rows=True, device=device)


def _matrix(t, name: str) -> tuple:
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.bfloat16 and t.is_cuda and t.dim() == 2
            and t.is_contiguous()):
        _tensor(t, name, _BF16, rows=True)
    return t.shape


def _act(act: str) -> int:
    if act not in capi.ACTS:
        raise ValueError(f"act must be one of {', '.join(capi.ACTS)}")
    return capi.ACTS[act]


def _between(dtype, name: str) -> int:
    """How a number between two products is held (MK_BETWEEN_*)."""
    if dtype not in (None, *_LOGITS):
        raise ValueError(f"{name} must be torch.bfloat16, torch.float32 or None")
    return capi.BETWEEN["result" if dtype is None else "bf16" if dtype is torch.bfloat16 else "fp32"]


def _result(out, name: str, dtype, shape, device):
    """out, checked, or a new tensor of that type."""
    if out is None:
        if dtype not in _LOGITS:
            raise ValueError(f"{name} is float32 or bfloat16")
        return torch.empty(shape, dtype=dtype, device=device)
    _rows(out, name, _LOGITS, shape, device)
    return out


def _code(t) -> int:
    return int(t is not None and t.dtype is torch.bfloat16)


def gemm_act(A: torch.Tensor, B: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
             residual: torch.Tensor | None = None, out: torch.Tensor | None = None, pre: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out = act(A @ B + bias) + residual in one pass (mk_gemm_act): A bf16
    [M, K], B bf16 [K, N], fp32 sums, one rounding.  Any sizes, from one row on;
    rows need only be contiguous each (operands whose rows do not start at
    16-byte boundaries are laid out anew first, which costs a copy).  act: none,
    relu, gelu, gelu_tanh or silu.  bias [N] and residual [M, N]: bfloat16 or
    float32; out: bfloat16 or float32 (out_dtype where none is given), may be the
    residual itself, overlaps nothing else.  pre (bf16 [M, N]) receives A @ B +
    bias for gemm_act_backward.  Where nothing follows a bfloat16 product of whole
    tiles, gemm is as fast or faster.  Nothing is recorded for autograd."""
    M, K = _matrix(A, "A")
    dev = A.device
    if _matrix(B, "B")[0] != K or B.device != dev:
        raise ValueError(f"B must be [{K}, N] on {dev}")
    N = B.shape[1]
    code = _act(act)
    if bias is not None and not (_is(bias, torch.bfloat16, (N,), dev) or _is(bias, torch.float32, (N,), dev)):
        _tensor(bias, "bias", _LOGITS, (N,), device=dev)
    if residual is not None:
        _rows(residual, "residual", _LOGITS, (M, N), dev)
    if pre is not None:
        _rows(pre, "pre", _BF16, (M, N), dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return gemm_act(A, B, bias, act, residual, out, pre, out_dtype)
    out = _result(out, "out", out_dtype, (M, N), dev)
    if out.numel() == 0:
        return out
    _product("mk_gemm_act", GemmActArgs, dev, True, A.data_ptr(), B.data_ptr(), out.data_ptr(), _ptr(bias),
             _ptr(residual), _ptr(pre), M, N, K, _ld(A), _ld(B), _ld(out), 0 if residual is None else _ld(residual),
             0 if pre is None else _ld(pre), code, _code(out), _code(bias), _code(residual))
    return out


def gemm_act_backward(dC: torch.Tensor, A: torch.Tensor, B: torch.Tensor, pre: torch.Tensor | None = None,
                      act: str = "none", need_dA: bool = True, need_dB: bool = True, need_dbias: bool = True,
                      dA: torch.Tensor | None = None, dB: torch.Tensor | None = None,
                      dbias: torch.Tensor | None = None, dB_dtype: torch.dtype = torch.bfloat16,
                      accumulate: bool = False, dpre_dtype: torch.dtype | None = None) -> tuple:
    """Gradients of gemm_act (mk_gemm_act_backward): (dA bf16, dB bfloat16 or
    float32, dbias float32), None for what is not needed; the residual's is dC
    itself (bf16 [M, N]).  pre: what the forward call kept, needed with an
    activation.  dpre_dtype: how dpre = dC * act'(pre) goes into the products of dA
    and dB; in bfloat16, one product each, they are off by up to 2^-8 of each
    element of it, in float32 by nothing, which takes three products each.  None:
    float32 for a float32 dB, else bfloat16.  (dbias takes dpre as it is; without an
    activation it is dC, with relu bfloat16 holds it.)  accumulate: dB and dbias,
    which are then given, are added to."""
    M, N = _matrix(dC, "dC")
    dev = dC.device
    K = _matrix(A, "A")[1]
    if A.shape[0] != M or A.device != dev or _matrix(B, "B") != (K, N) or B.device != dev:
        raise ValueError(f"A must be [{M}, K] and B [K, {N}] on {dev}")
    code = _act(act)
    between = _between(dpre_dtype, "dpre_dtype")
    if code:
        if pre is None:
            raise ValueError("pre is needed with an activation")
        _rows(pre, "pre", _BF16, (M, N), dev)
    if not (need_dA or need_dB or need_dbias):
        return None, None, None
    if accumulate and ((need_dB and dB is None) or (need_dbias and dbias is None)):
        raise ValueError("accumulate needs dB and dbias")
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return gemm_act_backward(dC, A, B, pre, act, need_dA, need_dB, need_dbias, dA, dB, dbias, dB_dtype,
                                     accumulate, dpre_dtype)
    if need_dA and dA is not None:
        _rows(dA, "dA", _BF16, (M, K), dev)
    dA = _result(dA, "dA", torch.bfloat16, (M, K), dev) if need_dA else None
    dB = _result(dB, "dB", dB_dtype, (K, N), dev) if need_dB else None
    if not need_dbias:
        dbias = None
    elif dbias is None:
        dbias = torch.empty(N, dtype=torch.float32, device=dev)
    elif not _is(dbias, torch.float32, (N,), dev):
        _tensor(dbias, "dbias", _F32, (N,), device=dev)
    _product("mk_gemm_act_backward", GemmActBackwardArgs, dev, True, dC.data_ptr(), A.data_ptr(), B.data_ptr(),
             _ptr(pre) if code else 0, _ptr(dA), _ptr(dB), _ptr(dbias), M, N, K, _ld(dC), _ld(A), _ld(B),
             _ld(pre) if code else 0, 0 if dA is None else _ld(dA), 0 if dB is None else _ld(dB), code, _code(dB),
             bool(accumulate), between)
    return dA, dB, dbias


def _experts(W, counts, device) -> tuple:
    if not (isinstance(W, torch.Tensor) and W.dtype is torch.bfloat16 and W.device == device and W.dim() == 3
            and W.is_contiguous()):
        _tensor(W, "W", _BF16, dim=3, device=device)
    if not _is(counts, torch.int32, (W.shape[0],), device):
        _tensor(counts, "counts", _I32, (W.shape[0],), device=device)
    return W.shape


def moe_ragged_gemm(A: torch.Tensor, W: torch.Tensor, counts: torch.Tensor, mode: int = 0,
                    out: torch.Tensor | None = None, h: torch.Tensor | None = None) -> torch.Tensor:
    """Expert products on ragged rows (mk_moe_ragged_gemm): A bf16 [R, K] holds
    counts[e] rows for expert e, one expert behind the other (counts int32 [E] on
    the device, e.g. padded_tokens_per_expert of moe_build_indices_dev, at
    row_block 1 or any other; nothing is read back), W bf16 [E, K, N].
    mode 0: out = A @ W[e] (bf16 [R, N]); mode 1: out = silu(g) * u with (g | u) =
    A @ W[e] (bf16 [R, N / 2]), and h (bf16 [R, N]) receives (g | u) for the
    backward pass.  Any sizes.  Rows behind the experts' are not written (new
    results hold whatever was there), and nothing that they hold is in a result."""
    R, K = _matrix(A, "A")
    dev = A.device
    if _experts(W, counts, dev)[1] != K:
        raise ValueError(f"W must be [E, {K}, N]")
    E, _, N = W.shape
    if mode not in (0, 1) or (mode == 1 and N % 2):
        raise ValueError("mode must be 0, or 1 with an even N")
    if h is not None:
        if mode == 0:
            raise ValueError("h belongs to mode 1")
        _rows(h, "h", _BF16, (R, N), dev)
    shape = (R, N // 2 if mode else N)
    if out is not None:
        _rows(out, "out", _BF16, shape, dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_ragged_gemm(A, W, counts, mode, out, h)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    _product("mk_moe_ragged_gemm", MoeRaggedGemmArgs, dev, False, A.data_ptr(), W.data_ptr(), counts.data_ptr(),
             out.data_ptr(), _ptr(h), R, K, N, _ld(A), _ld(out), 0 if h is None else _ld(h), E, mode)
    return out


def moe_ragged_gemm_dgrad(dy: torch.Tensor, W: torch.Tensor, counts: torch.Tensor, h: torch.Tensor | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of moe_ragged_gemm's rows (mk_moe_ragged_dgrad): dA = dy @ W[e]^T
    (bf16 [R, K]).  With h (bf16 [R, 2K], as mode 1 kept it in front of this
    product): the gradient of h itself, bf16 [R, 2K], in the same pass; out may
    then be h."""
    R, N = _matrix(dy, "dy")
    dev = dy.device
    if _experts(W, counts, dev)[2] != N:
        raise ValueError(f"W must be [E, K, {N}]")
    E, K, _ = W.shape
    shape = (R, 2 * K if h is not None else K)
    if h is not None:
        _rows(h, "h", _BF16, shape, dev)
    if out is not None:
        _rows(out, "out", _BF16, shape, dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_ragged_gemm_dgrad(dy, W, counts, h, out)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    _product("mk_moe_ragged_dgrad", MoeRaggedDgradArgs, dev, False, dy.data_ptr(), W.data_ptr(), counts.data_ptr(),
             _ptr(h), out.data_ptr(), R, K, N, _ld(dy), 0 if h is None else _ld(h), _ld(out), E)
    return out


def moe_ragged_gemm_wgrad(A: torch.Tensor, dy: torch.Tensor, counts: torch.Tensor, out: torch.Tensor | None = None,
                          out_dtype: torch.dtype = torch.bfloat16, accumulate: bool = False) -> torch.Tensor:
    """Gradient of moe_ragged_gemm's weights (mk_moe_ragged_wgrad): dW[e] = A_e^T
    @ dy_e, bfloat16 or float32 [E, K, N]; zeros for an expert without rows.
    accumulate: out is added to."""
    R, K = _matrix(A, "A")
    dev = A.device
    if _matrix(dy, "dy")[0] != R or dy.device != dev:
        raise ValueError(f"dy must be [{R}, N] on {dev}")
    N = dy.shape[1]
    if not (isinstance(counts, torch.Tensor) and counts.dim() == 1 and _is(counts, torch.int32, counts.shape, dev)):
        _tensor(counts, "counts", _I32, dim=1, device=dev)
    E = counts.shape[0]
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
    else:
        _tensor(out, "out", _LOGITS, (E, K, N), device=dev)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return moe_ragged_gemm_wgrad(A, dy, counts, out, out_dtype, accumulate)
    if out is None:
        if out_dtype not in _LOGITS:
            raise ValueError("out is float32 or bfloat16")
        out = torch.empty((E, K, N), dtype=out_dtype, device=dev)
    _product("mk_moe_ragged_wgrad", MoeRaggedWgradArgs, dev, False, A.data_ptr(), dy.data_ptr(), counts.data_ptr(),
             out.data_ptr(), R, K, N, _ld(A), _ld(dy), E, _code(out), bool(accumulate))
    return out


def _vocab(x, W, labels) -> tuple:
    T, H = _matrix(x, "x")
    dev = x.device
    if _matrix(W, "W")[0] != H or W.device != dev:
        raise ValueError(f"W must be [{H}, V] on {dev}")
    if not (_is(labels, torch.int64, (T,), dev) or _is(labels, torch.int32, (T,), dev)):
        _tensor(labels, "labels", (torch.int32, torch.int64), (T,), device=dev)
    return T, H, W.shape[1], dev, labels.dtype is torch.int64


def vocab_loss(x: torch.Tensor, W: torch.Tensor, labels: torch.Tensor, vocab_begin: int = 0,
               ignore_index: int = -100) -> dict:
    """Cross entropy of the logits x @ W, which are never stored (mk_vocab_loss):
    x bf16 [T, H], W bf16 [H, V], labels int32 or int64 [T].  Returns float32 [T]
    "lse" = log sum exp of the logits, "target" = the label's logit and "loss" =
    lse - target; all 0 for tokens whose label is ignore_index, whatever their
    rows of x hold.  One rank's shard of a vocabulary: W holds the columns from
    vocab_begin on, and target is 0 where another rank has the label; the ranks'
    lse are joined by torch.logsumexp, their targets by a sum, and the loss is
    the difference (ignored tokens, whose zeros join to the logarithm of the
    ranks' number, are set to 0 by the caller; the backward pass gives them zeros
    whatever their lse and dloss are)."""
    T, H, V, dev, wide = _vocab(x, W, labels)
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return vocab_loss(x, W, labels, vocab_begin, ignore_index)
    lse, target, loss = torch.empty((3, T), dtype=torch.float32, device=dev).unbind(0)
    _product("mk_vocab_loss", VocabLossArgs, dev, True, x.data_ptr(), W.data_ptr(), labels.data_ptr(), lse.data_ptr(),
             target.data_ptr(), loss.data_ptr(), T, H, V, _ld(x), _ld(W), vocab_begin, ignore_index, wide)
    return {"loss": loss, "lse": lse, "target": target}


def vocab_loss_backward(x: torch.Tensor, W: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor,
                        dloss: torch.Tensor, vocab_begin: int = 0, ignore_index: int = -100, need_dx: bool = True,
                        need_dW: bool = True, dx: torch.Tensor | None = None, dW: torch.Tensor | None = None,
                        dx_dtype: torch.dtype = torch.bfloat16, dW_dtype: torch.dtype = torch.bfloat16,
                        accumulate: bool = False, piece_columns: int = 0,
                        dl_dtype: torch.dtype | None = None) -> tuple:
    """Gradients of vocab_loss's loss (mk_vocab_loss_backward): (dx [T, H], dW
    [H, V]), bfloat16 or float32, None for what is not needed, from dloss
    (float32 [T]) and lse (of a shard: the joined one).  The logits are computed
    anew, a piece of the vocabulary at a time (piece_columns, a multiple of 256;
    0: as many as keep the piece's gradient of the logits in bfloat16 at 128 MB or
    less, at least 256).  dl_dtype:
    how that gradient goes into the products of dx and dW.  In bfloat16, one
    product each, each element is off by up to 2^-8 of itself (without the
    significand of the largest dloss, which the sums take back, so that a mean's
    equal dloss leaves no common rounding; of several distinct dloss the others
    keep one each, at their labels); in float32 by nothing, which takes three
    products each.  None: float32 for a float32 result, bfloat16 for a bfloat16
    one.  A shard's dx is its part of a sum over the ranks (dx_dtype=torch.float32
    for that).  accumulate: dW, which is then given, is added to."""
    T, H, V, dev, wide = _vocab(x, W, labels)
    for t, name in ((lse, "lse"), (dloss, "dloss")):
        if not _is(t, torch.float32, (T,), dev):
            _tensor(t, name, _F32, (T,), device=dev)
    between = _between(dl_dtype, "dl_dtype")
    if not (need_dx or need_dW):
        return None, None
    if accumulate and need_dW and dW is None:
        raise ValueError("accumulate needs dW")
    if dev.index != _device_index():
        with torch.cuda.device(dev):
            return vocab_loss_backward(x, W, labels, lse, dloss, vocab_begin, ignore_index, need_dx, need_dW, dx, dW,
                                       dx_dtype, dW_dtype, accumulate, piece_columns, dl_dtype)
    dx = _result(dx, "dx", dx_dtype, (T, H), dev) if need_dx else None
    dW = _result(dW, "dW", dW_dtype, (H, V), dev) if need_dW else None
    _product("mk_vocab_loss_backward", VocabLossBackwardArgs, dev, True, x.data_ptr(), W.data_ptr(), labels.data_ptr(),
             lse.data_ptr(), dloss.data_ptr(), _ptr(dx), _ptr(dW), T, H, V, _ld(x), _ld(W),
             0 if dx is None else _ld(dx), 0 if dW is None else _ld(dW), vocab_begin, ignore_index, piece_columns,
             wide, _code(dx), _code(dW), bool(accumulate), between)
    return dx, dW


def probe_mfma_ceiling(iters: int = 20000, num_wg: int = 0, reps: int = 3) -> dict:
    """MFMA throughput ceiling of the current device under sustained load
    (mk_probe_mfma_ceiling): one 8-wave workgroup per CU issuing independent
    32x32x16 bf16 MFMAs on random operands, no memory traffic.  Returns the
    median TFLOP/s over `reps` launches (HIP events on the launch stream) and
    the engine clock those launches ran at (shader cycles / 100 MHz ticks)."""
    L = capi.lib()
    n_wg = num_wg or cu_count()
    threads = int(L.mk_probe_threads())
    sink = torch.empty(n_wg * threads, dtype=torch.float32, device="cuda")
    clocks = torch.zeros(n_wg * 2, dtype=torch.int64, device="cuda")
    flops = float(n_wg) * (threads // 64) * iters * 16 * 2 * 32 * 32 * 16
    s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    capi.check("mk_probe_mfma_ceiling", L.mk_probe_mfma_ceiling(iters // 10, n_wg, _ptr(sink), _ptr(clocks), _stream()))
    res = []
    for _ in range(reps):
        s.record()
        capi.check("mk_probe_mfma_ceiling", L.mk_probe_mfma_ceiling(iters, n_wg, _ptr(sink), _ptr(clocks), _stream()))
        e.record()
        torch.cuda.synchronize()
        ck = clocks.view(n_wg, 2).cpu().double()
        ghz = float((ck[:, 0] / ck[:, 1]).median()) * 0.1
        res.append((s.elapsed_time(e), ghz))
    ms, ghz = sorted(res)[len(res) // 2]
    return {"tflops": flops / ms / 1e9, "sclk_ghz": ghz, "workgroups": n_wg, "us": ms * 1e3,
            "finite": bool(torch.isfinite(sink).all())}
