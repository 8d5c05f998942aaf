"""Packed attention as an operator on torch tensors (mi_attention_dev, mi_attention_backward_dev): whole sequences of different
lengths back to back, or a padded batch under a key mask; causal or not; grouped key / value heads; a relative position bias
learned by buckets.  The formulas and the limits stand in include/mi355rag.h.  Everything numeric runs in
rag_amd/lib/libmi355rag.so on an MI355X; there is no CPU fallback.

    out = packed_attention(q, k, v, offsets, causal=True)              # q [tokens][heads][head_dim], k / v [tokens][kv_heads][head_dim]
    out = packed_attention(q, k, v, key_mask=mask, bias_table=table)   # q [batch][length][heads][head_dim] ..., mask [batch][length]
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

from . import _capi
from ._capi import AttentionConfig, AttentionRows


def _dtype_code(t):
    import torch
    code = {torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_F16}.get(t.dtype)
    if code is None:
        raise ValueError(f"packed_attention: bfloat16 or float16 tensors, got {t.dtype}")
    return code


def _rows(name: str, t, like, heads: Optional[int] = None) -> AttentionRows:
    """A [tokens][heads][head_dim] or [batch][length][heads][head_dim] tensor as mi_attention_rows (views are fine while head_dim is
    adjacent and a batch's rows are evenly spaced)."""
    if t.device != like.device or t.dtype != like.dtype:
        raise ValueError(f"packed_attention: {name} is {t.dtype} on {t.device}, q is {like.dtype} on {like.device}")
    if t.dim() != like.dim() or t.shape[:-2] != like.shape[:-2] or t.shape[-1] != like.shape[-1] or (heads and t.shape[-2] != heads):
        raise ValueError(f"packed_attention: {name} has shape {tuple(t.shape)}, q {tuple(like.shape)}")
    s, z = t.stride(), t.shape
    if z[-1] > 1 and s[-1] != 1:
        raise ValueError(f"packed_attention: the head_dim elements of {name} must be adjacent (strides {s})")
    if t.dim() == 4 and z[0] > 1 and z[1] > 0 and s[0] != z[1] * s[1] and t.numel():
        raise ValueError(f"packed_attention: the rows of {name} must be evenly spaced over the batch (strides {s})")
    # the stride of an axis of one entry is never used; what torch reports for it is arbitrary
    return AttentionRows(t.data_ptr(), s[-3] if z[-3] > 1 else (s[0] if t.dim() == 4 and z[0] > 1 else z[-2] * z[-1]),
                         s[-2] if z[-2] > 1 else z[-1])


def _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional):
    """(config, tokens, nseq, offsets, key_mask, bias_table as pointers, keeping what they point to alive) after the checks."""
    import torch
    if not q.is_cuda or q.dim() not in (3, 4):
        raise ValueError("packed_attention: q must be a [tokens][heads][head_dim] or [batch][length][heads][head_dim] tensor on the GPU")
    dtype = _dtype_code(q)
    heads, hd = q.shape[-2], q.shape[-1]
    if k.dim() != q.dim() or v.shape != k.shape:
        raise ValueError(f"packed_attention: shapes of q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    tokens = q.shape[0] if q.dim() == 3 else q.shape[0] * q.shape[1]
    if q.dim() == 3:
        if offsets is None:
            raise ValueError("packed_attention: packed rows need offsets (int32 [sequences + 1]); a padded batch is 4-dimensional")
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous() or offsets.device != q.device:
            raise ValueError("packed_attention: offsets must be a contiguous int32 [sequences + 1] tensor on the device of q")
        nseq = offsets.shape[0] - 1
    else:
        if offsets is not None:
            raise ValueError("packed_attention: a padded batch (4-dimensional q) takes no offsets")
        nseq = q.shape[0] if tokens else 0
    if key_mask is not None:
        if key_mask.dtype != torch.int32 or key_mask.shape != q.shape[:-2] or not key_mask.is_contiguous() or key_mask.device != q.device:
            raise ValueError(f"packed_attention: key_mask must be a contiguous int32 {list(q.shape[:-2])} tensor on the device of q")
    buckets = 0
    if bias_table is not None:
        if bias_table.dtype != torch.float32 or bias_table.dim() != 2 or bias_table.shape[1] != heads or not bias_table.is_contiguous() or bias_table.device != q.device:
            raise ValueError(f"packed_attention: bias_table must be a contiguous float32 [num_buckets][{heads}] tensor on the device of q")
        buckets = bias_table.shape[0]
        if buckets == 0:
            raise ValueError("packed_attention: bias_table has no buckets")
    if scale is None:
        scale = 1.0 / math.sqrt(hd) if hd else 1.0
    cfg = AttentionConfig(heads, k.shape[-2], hd, dtype, int(bool(causal)), 1, float(scale), buckets, int(max_distance), int(bool(bidirectional)))
    p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())          # noqa: E731
    return cfg, tokens, nseq, p(offsets), p(key_mask), p(bias_table)


def relative_position_buckets(rel, num_buckets: int, max_distance: int = 128, bidirectional: bool = True):
    """The bucket of each relative position key - query (any integer array; host computation): row of the bias table it adds."""
    import numpy as np
    rel = np.ascontiguousarray(rel, dtype=np.int64)
    out = np.empty(rel.shape, dtype=np.int32)
    p = lambda a: a.ctypes.data_as(ctypes.c_void_p)          # noqa: E731
    _capi.check(_capi.load().mi_attention_buckets(int(num_buckets), int(max_distance), int(bool(bidirectional)), rel.size, p(rel), p(out)))
    return out


def packed_attention(q, k, v, offsets=None, *, causal: bool = False, scale: Optional[float] = None, key_mask=None,
                     bias_table=None, max_distance: int = 128, bidirectional: Optional[bool] = None, return_lse: bool = False):
    """softmax(scale * q k^T + bias) v over the rows of each sequence.

    q [tokens][heads][head_dim], k, v [tokens][kv_heads][head_dim], bfloat16 or float16, with offsets (int32 [sequences + 1], rising
    from 0: sequence i is rows offsets[i] .. offsets[i + 1]); or [batch][length][...] without offsets.  Views are taken as they
    are (slices of one QKV tensor).  key_mask (int32, the leading shape of q): rows that are 0 are no keys.  scale: default
    head_dim ** -0.5.  bias_table (float32 [num_buckets][heads]) adds bias_table[bucket(key - query)]; bidirectional: buckets for
    both directions (default: not causal).  Rows that attend nothing, and rows behind the last sequence, are 0.

    return_lse: also the float32 [heads][tokens] log-sum-exp of each row's scores, which packed_attention_backward takes.  Runs on
    the current stream of q's device."""
    import torch
    if bidirectional is None:
        bidirectional = not causal
    cfg, tokens, nseq, off, mask, table = _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional)
    rows = [_rows("q", q, q), _rows("k", k, q), _rows("v", v, q)]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[-2], tokens), dtype=torch.float32, device=q.device) if return_lse else None
    _capi.check(_capi.load().mi_attention_dev(_capi.get_ctx(q.device.index), cfg, tokens, nseq, off, mask, rows[0], rows[1], rows[2], table,
                                              _rows("out", out, q), lse.data_ptr() if return_lse else None, _capi.stream_arg(q.device)))
    return (out, lse) if return_lse else out


def packed_attention_backward(dout, q, k, v, out, lse, offsets=None, *, causal: bool = False, scale: Optional[float] = None, key_mask=None,
                              bias_table=None, max_distance: int = 128, bidirectional: Optional[bool] = None):
    """Gradients of sum(dout * packed_attention(q, k, v, ...)): (dq, dk, dv, dbias_table), the last None without a bias_table.

    out and lse are what packed_attention(..., return_lse=True) gave for the same arguments.  dk and dv sum over the query heads of
    a key head; rows behind the last sequence have gradient 0.  A repeated call gives the same bits."""
    import torch
    if bidirectional is None:
        bidirectional = not causal
    cfg, tokens, nseq, off, mask, table = _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional)
    heads = q.shape[-2]
    if lse.dtype != torch.float32 or tuple(lse.shape) != (heads, tokens) or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError(f"packed_attention_backward: lse must be the contiguous float32 [{heads}][{tokens}] tensor of the forward pass")
    rows = [_rows("q", q, q), _rows("k", k, q), _rows("v", v, q), _rows("out", out, q, heads), _rows("dout", dout, q, heads)]
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    dtable = torch.empty_like(bias_table) if bias_table is not None else None
    lib, need = _capi.load(), ctypes.c_size_t()
    _capi.check(lib.mi_attention_backward_workspace(cfg, tokens, nseq, int(offsets is not None), ctypes.byref(need)))
    work = torch.empty(max(need.value, 1), dtype=torch.uint8, device=q.device)
    _capi.check(lib.mi_attention_backward_dev(_capi.get_ctx(q.device.index), cfg, tokens, nseq, off, mask, rows[0], rows[1], rows[2], table, rows[3],
                                              lse.data_ptr(), rows[4], _rows("dq", dq, q), _rows("dk", dk, q), _rows("dv", dv, q),
                                              dtable.data_ptr() if dtable is not None else None, work.data_ptr(), work.numel(), _capi.stream_arg(q.device)))
    return dq, dk, dv, dtable
