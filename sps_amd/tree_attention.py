"""Attention of drafted tokens over a sequence's KV cache, and the append of those that were accepted.

``tree_attention`` verifies up to 64 drafted tokens of every sequence in one call: a tree (each draft names its parent),
a chain, or one token, the single-token step of models whose scores are changed (``biased_attention``'s cap and biases
by distance). It stands beside ``masked_kv_attention`` and takes the same ``KVSegment``s. ``commit_drafts`` appends the
path to the last accepted draft to a segment's cache, in place of ``fused_sps_kv_update``'s one token. Both run in
libsps_attn.so (``sps_tree_attention``, ``sps_commit_drafts``); there is no CPU path.

A draft's parent is -1 (it follows the cached sequence's last token) or the index of an earlier draft. Any other value
marks padding: such a row, and what descends from it, is no draft; it sees nothing, no draft sees it and its output is 0.
"""

from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch
from torch import Tensor

from . import _native as N
from .biased_attention import change_struct, check_change
from .decode_attention import _DECODE_HEAD_DIMS, _KV_DTYPES, _segment_scan_len, KVSegment

MAX_DRAFTS = 64
_INDEX_DTYPES = {torch.int32: N.DTYPE_I32, torch.int64: N.DTYPE_I64}


@functools.lru_cache(maxsize=256)
def _tree_ws_bytes(b: int, h: int, d: int, t: int, scans: tuple) -> int:
    return int(N.lib().sps_tree_workspace_bytes(b, h, d, t, len(scans), N.i64_const(scans)))


def _rows16(t: Tensor) -> bool:
    """Unit last stride and 16-byte aligned rows, read in place by the kernels."""
    size = t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for s in t.stride()[:-1])


def _drafts(name: str, t: Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> Tensor:
    if not t.is_cuda or t.device != device:
        raise RuntimeError(f"{name} must be on the GPU of the caches ({device}), got {t.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} as the caches, got {t.dtype}")
    return t if _rows16(t) and t.stride(1) >= 0 else t.contiguous()


def _indices(name: str, t: Optional[Tensor], shape: tuple, device: torch.device) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dtype not in _INDEX_DTYPES:
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if tuple(t.shape) != shape or t.device != device:
        raise ValueError(f"{name} must be {list(shape)} on {device}, got {list(t.shape)} on {t.device}")
    return t.contiguous()


def _check_segment(seg: KVSegment, b: int, h: int, d: int, dtype: torch.dtype, device: torch.device) -> None:
    for name, t in (("keys", seg.k), ("values", seg.v)):
        if t.device != device:
            raise RuntimeError(f"segment {name} must be on {device}, got {t.device}")
        if t.dim() != 4 or t.shape != seg.k.shape or (t.shape[0], t.shape[1], t.shape[3]) != (b, h, d):
            raise ValueError(f"segment {name} must be [{b}, {h}, storage, {d}], got {list(t.shape)}")
        if t.dtype != dtype:
            raise TypeError(f"segment {name} must be {dtype}, got {t.dtype}")
        if t.numel() and (not _rows16(t) or t.stride(2) < 0):
            raise ValueError(f"segment {name} need a unit last stride and 16-byte aligned rows")
    if seg.lengths.dtype not in _INDEX_DTYPES:
        raise TypeError(f"segment lengths must be int32 or int64, got {seg.lengths.dtype}")
    if tuple(seg.lengths.shape) not in ((b,), (b, h)) or seg.lengths.device != device:
        raise ValueError(f"segment lengths must be [{b}] or [{b}, {h}] on {device}, got {list(seg.lengths.shape)} on "
                         f"{seg.lengths.device}")


def tree_attention(
    q_BxTxHxD: Tensor,
    segments: list[KVSegment],
    *,
    draft_k_BxTxHxD: Tensor,
    draft_v_BxTxHxD: Tensor,
    parents_BxT: Optional[Tensor] = None,
    sm_scale: Optional[float] = None,
    softcap: Optional[float] = None,
    slopes: Optional[Tensor] = None,
    bias_table: Optional[Tensor] = None,
    max_distance: int = 128,
) -> Tensor:
    """Attention of T (1 to 64) drafts per sequence; returns [B, T, H, D] in the queries' dtype (bf16 or f16).

    Each draft sees every live key of the (at most 3) segments, its ancestors among the drafts and itself.
    ``parents_BxT``: [B, T] int32/int64, None for a chain (draft i follows draft i - 1). Segments, queries and drafts
    share one dtype; segments need not be contiguous. ``sm_scale``: 1 / sqrt(D) by default. ``softcap``, ``slopes``,
    ``bias_table``, ``max_distance``: as in ``biased_attention``; positions run through the segments' live keys in
    their order, and a draft's position is their number plus its depth. A draft's non-finite value row reaches every draft of
    its sequence, whose weight of it may be 0; dead and padding rows reach none. Forward only (no gradients)."""
    if not torch.compiler.is_compiling():
        # Ordinary eager calls run in native code; None: the general path below.
        out = N.binding().tree_attention(q_BxTxHxD, segments, draft_k_BxTxHxD, draft_v_BxTxHxD, parents_BxT, sm_scale,
                                         softcap, slopes, bias_table, max_distance)
        if out is not None:
            return out
    return _tree_attention(q_BxTxHxD, segments, draft_k_BxTxHxD, draft_v_BxTxHxD, parents_BxT, sm_scale, softcap, slopes,
                           bias_table, max_distance)


@torch.compiler.disable  # compiled models call it as it is: a launch, and views of memory that is updated in place
def _tree_attention(q_BxTxHxD, segments, draft_k_BxTxHxD, draft_v_BxTxHxD, parents_BxT, sm_scale, softcap, slopes,
                    bias_table, max_distance) -> Tensor:
    if not q_BxTxHxD.is_cuda:
        raise RuntimeError("sps_amd tree_attention runs on the GPU only (got a CPU tensor)")
    if q_BxTxHxD.dim() != 4:
        raise ValueError(f"queries must be [B, T, H, D], got {list(q_BxTxHxD.shape)}")
    b, t, h, d = shape = tuple(q_BxTxHxD.shape)
    device, dtype = q_BxTxHxD.device, q_BxTxHxD.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"tree_attention takes bfloat16 and float16, got {dtype}")
    if not 1 <= t <= MAX_DRAFTS:
        raise ValueError(f"tree_attention takes 1 to {MAX_DRAFTS} drafts, got {t}")
    if d not in _DECODE_HEAD_DIMS:
        raise ValueError(f"tree_attention is built for head_dim in {_DECODE_HEAD_DIMS}, got {d}")
    if len(segments) > 3:
        raise ValueError(f"tree_attention takes at most 3 segments, got {len(segments)}")
    read = [q_BxTxHxD, draft_k_BxTxHxD, draft_v_BxTxHxD, *(x for sg in segments for x in (sg.k, sg.v))]
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (*read, bias_table)):
        raise RuntimeError("tree_attention has no backward: call it under torch.no_grad() or on detached tensors")
    q = _drafts("queries", q_BxTxHxD, shape, dtype, device)
    dk = _drafts("draft keys", draft_k_BxTxHxD, shape, dtype, device)
    dv = _drafts("draft values", draft_v_BxTxHxD, shape, dtype, device)
    parents = _indices("parents", parents_BxT, (b, t), device)
    for seg in segments:
        _check_segment(seg, b, h, d, dtype, device)
    cap = check_change(softcap, slopes, bias_table, max_distance, h, device)
    slopes = slopes.contiguous() if slopes is not None else None
    scans = tuple(_segment_scan_len(sg) for sg in segments)
    lens = [sg.lengths.contiguous() for sg in segments]
    with torch.cuda.device(device):
        out = torch.empty(shape, dtype=dtype, device=device)
        ws = torch.empty(_tree_ws_bytes(b, h, d, t, scans), dtype=torch.uint8, device=device)
        change = change_struct(cap, slopes, bias_table, int(max_distance))
        N.check("sps_tree_attention", N.lib().sps_tree_attention(
            b, h, d, t, _KV_DTYPES[dtype], q.data_ptr(), N.i64_const(q.stride()[:3]), len(segments),
            N.ptr_const(tuple(sg.k.data_ptr() for sg in segments)),
            N.i64_const(tuple(x for sg in segments for x in sg.k.stride()[:3])),
            N.ptr_const(tuple(sg.v.data_ptr() for sg in segments)),
            N.i64_const(tuple(x for sg in segments for x in sg.v.stride()[:3])),
            N.ptr_const(tuple(x.data_ptr() for x in lens)), N.i32_const(tuple(_INDEX_DTYPES[x.dtype] for x in lens)),
            N.i32_const(tuple(int(x.dim() == 2) for x in lens)), N.i64_const(scans),
            dk.data_ptr(), N.i64_const(dk.stride()[:3]), dv.data_ptr(), N.i64_const(dv.stride()[:3]),
            parents.data_ptr() if parents is not None else None,
            _INDEX_DTYPES[parents.dtype] if parents is not None else N.DTYPE_I32, t,
            d ** -0.5 if sm_scale is None else float(sm_scale), C.byref(change), out.data_ptr(), ws.data_ptr(),
            ws.numel(), torch.cuda.current_stream(device).cuda_stream))
    return out


def commit_drafts(
    segment: KVSegment,
    draft_k_BxTxHxD: Tensor,
    draft_v_BxTxHxD: Tensor,
    last_B: Tensor,
    *,
    parents_BxT: Optional[Tensor] = None,
) -> None:
    """Appends each sequence's accepted drafts to ``segment`` (k, v and lengths are updated in place).

    ``last_B``: [B] int32/int64, the last accepted draft of each sequence; the path from its root to it is appended in
    order, and the lengths ([B] or [B, H]) advance by the rows stored. Rows past the storage are dropped and
    the length stops there. Nothing happens where ``last_B`` names no draft (-1, out of range, padding) or
    a length is negative or already at the end. Drafts have the caches' dtype (bf16, f16 or fp32) and memory outside
    the caches'; caches and lengths are no expanded views."""
    if not torch.compiler.is_compiling() and N.binding().commit_drafts(segment, draft_k_BxTxHxD, draft_v_BxTxHxD, last_B,
                                                                       parents_BxT):
        return
    _commit_drafts(segment, draft_k_BxTxHxD, draft_v_BxTxHxD, last_B, parents_BxT)


@torch.compiler.disable
def _commit_drafts(segment, draft_k_BxTxHxD, draft_v_BxTxHxD, last_B, parents_BxT) -> None:
    if not segment.k.is_cuda:
        raise RuntimeError("sps_amd commit_drafts runs on the GPU only (got a CPU tensor)")
    if draft_k_BxTxHxD.dim() != 4:
        raise ValueError(f"draft keys must be [B, T, H, D], got {list(draft_k_BxTxHxD.shape)}")
    b, t, h, d = shape = tuple(draft_k_BxTxHxD.shape)
    device, dtype = segment.k.device, segment.k.dtype
    if dtype not in _KV_DTYPES:
        raise TypeError(f"commit_drafts takes bfloat16, float16 and float32 caches, got {dtype}")
    if not 1 <= t <= MAX_DRAFTS:
        raise ValueError(f"commit_drafts takes 1 to {MAX_DRAFTS} drafts, got {t}")
    if d not in _DECODE_HEAD_DIMS:
        raise ValueError(f"commit_drafts is built for head_dim in {_DECODE_HEAD_DIMS}, got {d}")
    _check_segment(segment, b, h, d, dtype, device)
    dk = _drafts("draft keys", draft_k_BxTxHxD, shape, dtype, device)
    dv = _drafts("draft values", draft_v_BxTxHxD, shape, dtype, device)
    parents = _indices("parents", parents_BxT, (b, t), device)
    last = _indices("last_B", last_B, (b,), device)
    if last is None:
        raise TypeError("last_B is required")
    per_head = segment.lengths.dim() == 2
    with torch.cuda.device(device):
        N.check("sps_commit_drafts", N.lib().sps_commit_drafts(
            b, h, d, t, _KV_DTYPES[dtype], segment.k.data_ptr(), segment.v.data_ptr(),
            N.i64_const((*segment.k.stride()[:3], *segment.v.stride()[:3])), segment.k.shape[2],
            segment.lengths.data_ptr(), _INDEX_DTYPES[segment.lengths.dtype], int(per_head),
            N.i64_const(segment.lengths.stride() if per_head else (segment.lengths.stride(0), 0)),
            dk.data_ptr(), N.i64_const(dk.stride()[:3]), dv.data_ptr(), N.i64_const(dv.stride()[:3]),
            parents.data_ptr() if parents is not None else None,
            _INDEX_DTYPES[parents.dtype] if parents is not None else N.DTYPE_I32, t,
            last.data_ptr(), _INDEX_DTYPES[last.dtype], torch.cuda.current_stream(device).cuda_stream))
