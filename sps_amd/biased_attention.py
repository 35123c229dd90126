"""Document-masked causal attention with changed scores: a tanh cap, a bias by distance, a visible prefix.

``biased_attention`` stands beside ``full_attention`` for models whose scores are not the plain scaled products.
For a query at position q, a key at position k and head h, with x = sm_scale * (q . k) and the distance
n = max(q - k, 0), the softmax is taken over

    s = softcap * tanh(x / softcap) - slopes[h] * n + bias_table[bucket(n), h]

(each part only where its argument is given), over the keys with k <= q or k < prefix_len[b], and of the query's
document. ``bias_buckets`` gives bucket(n). Forward and backward run in libsps_attn.so (``sps_biased_fwd``,
``sps_biased_bwd``); there is no CPU path.

Gradients go to q, k, v and the bias table; the slopes are constants. With O the output, dO its gradient, P the
weights and Delta = rowsum(O * dO): dS = P (dO V^T - Delta), dTable[j, h] the sum of dS over all pairs of bucket j,
and dS * (1 - tanh^2) * sm_scale the gradient of the products. Sums are fp32; P and dS are rounded to the inputs' type
for their products, and Delta comes from the rounded O, as in ``full_attention``, so a table in fp32 gets a gradient
with the relative error of that rounding, not of fp32. Results do not depend on timing.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native as N
from .attention import _alloc_like_bnhd, _docs_args, _dtype_code, _kernel_view, _strides, _stream, _validate, _ws_args

_TABLE_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16, torch.float32: N.DTYPE_F32}
MIN_CAP, MAX_CAP = 2.0 ** -10, 2.0 ** 20
_LEN_DTYPES = {torch.int32: N.DTYPE_I32, torch.int64: N.DTYPE_I64}


def bias_buckets(distances: int, num_buckets: int, max_distance: int = 128) -> Tensor:
    """[distances] int64 (CPU): the bucket of each distance 0 .. distances - 1.

    With e = num_buckets // 2, distances below e have a bucket each; a greater distance n has
    min(num_buckets - 1, e + floor((num_buckets - e) * log(n / e) / log(max_distance / e))), borders that are whole
    numbers counted exactly. 2 <= num_buckets <= 256 and num_buckets // 2 < max_distance <= 512."""
    if distances < 0:
        raise ValueError(f"distances must not be negative, got {distances}")
    out = (C.c_int * max(distances, 1))()
    N.check("sps_bias_buckets", N.lib().sps_bias_buckets(int(num_buckets), int(max_distance), int(distances), out))
    return torch.tensor(out[:distances], dtype=torch.int64)


def check_change(softcap: Optional[float], slopes: Optional[Tensor], bias_table: Optional[Tensor], max_distance: int,
                 n_head: int, device: torch.device) -> float:
    """Validates the score changes of a call with ``n_head`` heads; returns the cap (0 for none)."""
    if softcap is not None and not MIN_CAP <= softcap <= MAX_CAP:
        raise ValueError(f"softcap must be None or in [2^-10, 2^20], got {softcap}")
    if slopes is not None:
        if slopes.dtype != torch.float32:
            raise TypeError(f"slopes must be float32, got {slopes.dtype}")
        if slopes.shape != (n_head,) or slopes.device != device:
            raise ValueError(f"slopes must be [{n_head}] on {device}, got {tuple(slopes.shape)} on {slopes.device}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise ValueError("slopes are constants: they get no gradient")
    if bias_table is not None:
        if bias_table.dtype not in _TABLE_DTYPES:
            raise TypeError(f"bias_table must be bfloat16, float16 or float32, got {bias_table.dtype}")
        if bias_table.dim() != 2 or bias_table.shape[1] != n_head or bias_table.device != device:
            raise ValueError(f"bias_table must be [num_buckets, {n_head}] on {device}, got {tuple(bias_table.shape)} on "
                             f"{bias_table.device}")
        nb = bias_table.shape[0]
        if not 2 <= nb <= 256 or not nb // 2 < int(max_distance) <= 512:
            raise ValueError(f"num_buckets must be in [2, 256] and max_distance in (num_buckets // 2, 512], got {nb} "
                             f"and {max_distance}")
    return float(softcap) if softcap is not None else 0.0


def change_struct(softcap: float, slopes: Optional[Tensor], bias_table: Optional[Tensor], max_distance: int):
    """The C structure of checked score changes (it points into the tensors, which the caller keeps)."""
    c = N.ScoreChange()
    c.softcap = softcap
    c.slopes = slopes.data_ptr() if slopes is not None else None
    if bias_table is not None:
        c.bias_table = bias_table.data_ptr()
        c.table_dtype = _TABLE_DTYPES[bias_table.dtype]
        c.table_strides[0], c.table_strides[1] = bias_table.stride()
        c.num_buckets, c.max_distance = bias_table.shape[0], max_distance
    return c


def _prefix_args(prefix: Optional[Tensor]):
    return (prefix.data_ptr(), _LEN_DTYPES[prefix.dtype]) if prefix is not None else (None, N.DTYPE_I32)


def _workspace(q: Tensor, has_docs: bool, backward: bool, buckets: int) -> Optional[Tensor]:
    b, h, n, _ = q.shape
    nbytes = N.lib().sps_biased_workspace_bytes(b, h, n, int(has_docs), int(backward), buckets)
    return torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None


# The attention as torch.library custom ops, as full_attention's: a compiled model traces it without a graph break,
# the forward's workspace hands the document row layout to the backward, which writes its own scratch into it (and
# only that), so both ops are declared pure.
@torch.library.custom_op("sps_amd::biased_attention_fwd", mutates_args=())
def _fwd_op(q: Tensor, k: Tensor, v: Tensor, docs: Optional[Tensor], prefix: Optional[Tensor], slopes: Optional[Tensor],
            table: Optional[Tensor], sm_scale: float, softcap: float, max_distance: int,
            backward_buckets: int) -> Tuple[Tensor, Tensor, Tensor]:
    # backward_buckets: -1 where no backward follows, else the buckets of the table whose gradient it forms (0: none).
    with torch.cuda.device(q.device):
        q, k, v = _kernel_view(q), _kernel_view(k), _kernel_view(v)
        if slopes is not None:
            slopes = slopes.contiguous()
        if prefix is not None:
            prefix = prefix.contiguous()
        b, h, n, d = q.shape
        o = _alloc_like_bnhd(q)
        lse = torch.empty((b, h, n), dtype=torch.float32, device=q.device)
        keep = backward_buckets >= 0 and docs is not None
        ws = _workspace(q, docs is not None, keep, max(backward_buckets, 0))
        change = change_struct(softcap, slopes, table, max_distance)
        N.check("sps_biased_fwd", N.lib().sps_biased_fwd(
            b, h, n, d, _dtype_code(q), q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
            o.data_ptr(), _strides(o), lse.data_ptr(), *_docs_args(docs), *_prefix_args(prefix), sm_scale,
            C.byref(change), *_ws_args(ws), _stream(q)))
    return o, lse, ws if keep else torch.empty((0,), dtype=torch.uint8, device=q.device)


@_fwd_op.register_fake
def _(q, k, v, docs, prefix, slopes, table, sm_scale, softcap, max_distance, backward_buckets):
    b, h, n, d = q.shape
    nbytes = 0
    if backward_buckets >= 0 and docs is not None:
        nbytes = int(N.lib().sps_biased_workspace_bytes(int(b), int(h), int(n), 1, 1, backward_buckets))
    return (q.new_empty((b, n, h, d)).transpose(1, 2), q.new_empty((b, h, n), dtype=torch.float32),
            q.new_empty((nbytes,), dtype=torch.uint8))


@torch.library.custom_op("sps_amd::biased_attention_bwd", mutates_args=())
def _bwd_op(do: Tensor, q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, docs: Optional[Tensor],
            prefix: Optional[Tensor], slopes: Optional[Tensor], table: Optional[Tensor], ws: Tensor, sm_scale: float,
            softcap: float, max_distance: int, backward_buckets: int) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    with torch.cuda.device(q.device):
        do, q, k, v = _kernel_view(do), _kernel_view(q), _kernel_view(k), _kernel_view(v)
        if slopes is not None:
            slopes = slopes.contiguous()
        if prefix is not None:
            prefix = prefix.contiguous()
        b, h, n, d = q.shape
        dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
        reuse = docs is not None and ws.numel() > 0
        if not reuse:
            ws = _workspace(q, docs is not None, True, backward_buckets)
        dtable = torch.empty((backward_buckets, h), dtype=table.dtype if table is not None else torch.float32,
                             device=q.device)
        change = change_struct(softcap, slopes, table, max_distance)
        N.check("sps_biased_bwd", N.lib().sps_biased_bwd(
            b, h, n, d, _dtype_code(q), q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
            o.data_ptr(), _strides(o), do.data_ptr(), _strides(do), lse.data_ptr(), dq.data_ptr(), _strides(dq),
            dk.data_ptr(), _strides(dk), dv.data_ptr(), _strides(dv), dtable.data_ptr() if backward_buckets else None,
            *_docs_args(docs), *_prefix_args(prefix), sm_scale, C.byref(change), int(reuse), *_ws_args(ws), _stream(q)))
    return dq, dk, dv, dtable


@_bwd_op.register_fake
def _(do, q, k, v, o, lse, docs, prefix, slopes, table, ws, sm_scale, softcap, max_distance, backward_buckets):
    dtable = q.new_empty((backward_buckets, q.shape[1]), dtype=table.dtype if table is not None else torch.float32)
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), dtable


def _setup_context(ctx, inputs, output):
    q, k, v, docs, prefix, slopes, table, sm_scale, softcap, max_distance, buckets = inputs
    o, lse, ws = output
    ctx.save_for_backward(q, k, v, o, lse, docs, prefix, slopes, table, ws)
    ctx.params = (float(sm_scale), float(softcap), int(max_distance), int(buckets))


def _backward(ctx, do, _dlse, _dws):
    q, k, v, o, lse, docs, prefix, slopes, table, ws = ctx.saved_tensors
    sm_scale, softcap, max_distance, buckets = ctx.params
    dq, dk, dv, dtable = torch.ops.sps_amd.biased_attention_bwd(
        do, q, k, v, o, lse, docs, prefix, slopes, table, ws, sm_scale, softcap, max_distance, max(buckets, 0))
    return dq, dk, dv, None, None, None, dtable if buckets > 0 else None, None, None, None, None


_fwd_op.register_autograd(_backward, setup_context=_setup_context)


def biased_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    sm_scale: float,
    *,
    softcap: Optional[float] = None,
    slopes: Optional[Tensor] = None,
    bias_table: Optional[Tensor] = None,
    max_distance: int = 128,
    documents_idx_BxT: Optional[Tensor] = None,
    prefix_len_B: Optional[Tensor] = None,
) -> Tensor:
    """Document-masked causal attention with changed scores. q, k, v: [B, H, T, D] bf16/f16, D in 16 .. 256 as
    ``full_attention``; returns [B, H, T, D] (in [B, T, H, D] memory order).

    ``softcap``: scores are capped to (-softcap, softcap) by a tanh, in fp32: 2^-10 to 2^20, and an error of the scores
    of some 2^-22 softcap, so a great cap is better left out. ``slopes``: [H] fp32, the scores lose
    slopes[h] times the distance; no gradient. ``bias_table``: [num_buckets, H] bf16/f16/fp32, added by distance bucket
    (``bias_buckets``); entries below -16384 (-inf, the types' lowest values) hide their pairs.
    ``documents_idx_BxT``: [B, T] ids as in ``full_attention``. ``prefix_len_B``: [B] int32/int64, the leading
    positions of each row (pads included) that every query of the row sees, later ones too, within its document; a
    key ahead of its query has distance 0. Queries that see no key yield 0. As in ``full_attention``, a non-finite value row can reach
    the outputs of other queries of its 32-query tile, whose weight of it is 0."""
    if not torch.compiler.is_compiling():
        # Ordinary eager calls run in native code from here on; None: the general path below.
        o = N.binding().biased_attention(q, k, v, sm_scale, softcap, slopes, bias_table, max_distance, documents_idx_BxT,
                                         prefix_len_B)
        if o is not None:
            return o
    _validate(q, k, v, N.FAMILY_FULL, documents_idx_BxT)
    cap = check_change(softcap, slopes, bias_table, max_distance, q.shape[1], q.device)
    if k.device != q.device or v.device != q.device:
        raise RuntimeError("q, k and v must be on one device")
    if documents_idx_BxT is not None and documents_idx_BxT.device != q.device:
        raise RuntimeError("documents_idx_BxT must be on the queries' device")
    if prefix_len_B is not None:
        if prefix_len_B.dtype not in _LEN_DTYPES:
            raise TypeError(f"prefix_len_B must be int32 or int64, got {prefix_len_B.dtype}")
        if prefix_len_B.shape != (q.shape[0],) or prefix_len_B.device != q.device:
            raise ValueError(f"prefix_len_B must be [{q.shape[0]}] on {q.device}, got {tuple(prefix_len_B.shape)} on "
                             f"{prefix_len_B.device}")
    buckets = -1
    if torch.is_grad_enabled():
        table_grad = bias_table is not None and bias_table.requires_grad
        if table_grad or any(t.requires_grad for t in (q, k, v)):
            buckets = bias_table.shape[0] if table_grad else 0
    o, _, _ = torch.ops.sps_amd.biased_attention_fwd(
        q, k, v, documents_idx_BxT, prefix_len_B, slopes, bias_table, float(sm_scale), cap, int(max_distance), buckets)
    return o
