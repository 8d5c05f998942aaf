"""Packed attention as an operator on torch tensors (mi_attention_dev, mi_attention_backward_dev): whole sequences of different
lengths back to back, or a padded batch under a key mask; causal or not; grouped key / value heads; a relative position bias
learned by buckets (a finite bias counts as at most 4096 in size, here and in the gradients).  The formulas and the limits stand in
include/mi355rag.h.  Everything numeric runs in
rag_amd/lib/libmi355rag.so on an MI355X; there is no CPU fallback.

    out = packed_attention(q, k, v, offsets, causal=True)              # q [tokens][heads][head_dim], k / v [tokens][kv_heads][head_dim]
    out = packed_attention(q, k, v, key_mask=mask, bias_table=table)   # q [batch][length][heads][head_dim] ..., mask [batch][length]
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

from . import _capi
from ._capi import AttentionConfig, AttentionRows


_F32 = _I32 = _CODES = _empty_like = _grad_enabled = _forward_ad = _modes = _modes_before = _trace = None


def _types():
    global _F32, _I32, _CODES, _empty_like, _grad_enabled, _forward_ad, _modes, _modes_before, _trace
    import torch
    import torch.autograd.forward_ad
    _grad_enabled, _forward_ad = torch.is_grad_enabled, torch.autograd.forward_ad
    # whether a dispatch mode or a trace may be on at all, in tenths of a microsecond; where torch has no such name, the whole check
    always = lambda: 1                                       # noqa: E731
    _modes = getattr(torch._C, "_len_torch_dispatch_stack", always)
    _modes_before = getattr(torch._ops, "_len_torch_dispatch_stack_pre_dispatch", always)
    _trace = getattr(torch._C, "_get_tracing_state", always)
    _empty_like = torch.empty_like
    _F32, _I32, _CODES = torch.float32, torch.int32, {torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_F16}
    return _CODES


def _rows(name: str, t, shape, dtype, device) -> AttentionRows:
    """A [tokens][heads][head_dim] or [batch][length][heads][head_dim] tensor as mi_attention_rows (views are fine while head_dim is
    adjacent and a batch's rows are evenly spaced)."""
    if t.dtype is not dtype or t.device != device:
        raise ValueError(f"packed_attention: {name} is {t.dtype} on {t.device}, q is {dtype} on {device}")
    if t.shape != shape:
        raise ValueError(f"packed_attention: {name} has shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    z = shape
    if t.is_contiguous():
        hd = z[-1]
        return AttentionRows(t.data_ptr(), z[-2] * hd, hd)
    s = t.stride()
    if z[-1] > 1 and s[-1] != 1:
        raise ValueError(f"packed_attention: the head_dim elements of {name} must be adjacent (strides {s})")
    if len(z) == 4 and z[0] > 1 and z[1] > 1 and s[0] != z[1] * s[1] and t.numel():
        raise ValueError(f"packed_attention: the rows of {name} must be evenly spaced over the batch (strides {s})")
    # the stride of an axis of one entry is never used; what torch reports for it is arbitrary
    return AttentionRows(t.data_ptr(), s[-3] if z[-3] > 1 else (s[0] if len(z) == 4 and z[0] > 1 else z[-2] * z[-1]),
                         s[-2] if z[-2] > 1 else z[-1])


def _own_rows(t, heads, hd) -> AttentionRows:
    """... of a contiguous tensor made here, or q itself: nothing to check."""
    return AttentionRows(t.data_ptr(), heads * hd, hd)


def _like(t):
    """A new contiguous tensor of t's shape (empty_like is the shorter call, but would keep the strides of a permuted tensor)."""
    return _empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


@functools.lru_cache(maxsize=256)
def _config(heads, kv_heads, hd, dtype, causal, scale, buckets, max_distance, bidirectional):
    if scale is None:
        scale = 1.0 / math.sqrt(hd) if hd else 1.0
    return AttentionConfig(heads, kv_heads, hd, dtype, int(causal), 1, scale, buckets, max_distance, int(bidirectional))


@functools.lru_cache(maxsize=256)
def _workspace(heads, kv_heads, hd, buckets, max_distance, bidirectional, tokens, nseq, packed) -> int:
    """Words of workspace of the backward pass."""
    cfg = AttentionConfig(heads, kv_heads, hd, _capi.DTYPE_BF16, 0, 1, 1.0, buckets, max_distance, bidirectional)
    need = ctypes.c_size_t()
    _capi.check(_capi.load().mi_attention_backward_workspace(cfg, tokens, nseq, packed, ctypes.byref(need)))
    return (max(need.value, 4) + 3) // 4


def _numbers(causal, scale, max_distance, bidirectional):
    """As plain numbers.  Tensors and arrays of one element are numbers too, as they stand at the call: what is kept by their identity
    (the cache of _config, an autograd node) would not see them change."""
    return bool(causal), None if scale is None else float(scale), int(max_distance), None if bidirectional is None else bool(bidirectional)


def _seen_whole(*tensors) -> None:
    """Refuses what would see a call without its kernels.  A trace (make_fx, torch.jit.trace) would hold the allocation of the result and
    nothing that fills it.  Tensors that carry a forward-mode tangent do not require a gradient: the kernels would run on their values
    alone and the result's derivative would be zero.  (Dispatch modes that only watch are left alone.)"""
    if _CODES is None:
        _types()
    if _modes() or _trace() is not None or _modes_before():
        import torch
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if torch.jit.is_tracing() or get_proxy_mode() is not None:
            raise RuntimeError("packed_attention: under a trace (make_fx, torch.jit.trace), which would not record the kernels")
    if getattr(_forward_ad, "_current_level", 0) < 0:        # no such level is open
        return
    import torch
    if any(isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("packed_attention: no forward-mode derivatives (torch.autograd.forward_ad); reverse mode has them")


def _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional):
    """(config, tokens, nseq, addresses of offsets, key_mask, bias_table) after the checks."""
    causal, scale, max_distance, bidirectional = _numbers(causal, scale, max_distance, bidirectional)
    z, device = q.shape, q.device
    if not q.is_cuda or len(z) not in (3, 4):
        raise ValueError("packed_attention: q must be a [tokens][heads][head_dim] or [batch][length][heads][head_dim] tensor on the GPU")
    code = (_CODES or _types()).get(q.dtype)
    if code is None:
        raise ValueError(f"packed_attention: bfloat16 or float16 tensors, got {q.dtype}")
    heads, hd = z[-2], z[-1]
    zk = k.shape
    if len(zk) != len(z) or zk[:-2] != z[:-2] or zk[-1] != hd:
        raise ValueError(f"packed_attention: shapes of q {tuple(z)} and k {tuple(zk)}")
    off = mask = table = None
    if len(z) == 3:
        tokens = z[0]
        if offsets is None:
            raise ValueError("packed_attention: packed rows need offsets (int32 [sequences + 1]); a padded batch is 4-dimensional")
        if offsets.dtype != _I32 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous() or offsets.device != device:
            raise ValueError("packed_attention: offsets must be a contiguous int32 [sequences + 1] tensor on the device of q")
        nseq, off = offsets.shape[0] - 1, offsets.data_ptr()
    else:
        if offsets is not None:
            raise ValueError("packed_attention: a padded batch (4-dimensional q) takes no offsets")
        tokens = z[0] * z[1]
        nseq = z[0] if tokens else 0
    if key_mask is not None:
        if key_mask.dtype != _I32 or key_mask.shape != z[:-2] or not key_mask.is_contiguous() or key_mask.device != device:
            raise ValueError(f"packed_attention: key_mask must be a contiguous int32 {list(z[:-2])} tensor on the device of q")
        mask = key_mask.data_ptr()
    buckets = 0
    if bias_table is not None:
        zt = bias_table.shape
        if bias_table.dtype != _F32 or len(zt) != 2 or zt[1] != heads or zt[0] == 0 or not bias_table.is_contiguous() or bias_table.device != device:
            raise ValueError(f"packed_attention: bias_table must be a contiguous float32 [num_buckets][{heads}] tensor on the device of q")
        buckets, table = zt[0], bias_table.data_ptr()
    if bidirectional is None:
        bidirectional = not causal
    return _config(heads, zk[-2], hd, code, causal, scale, buckets, max_distance, bidirectional), tokens, nseq, off, mask, table


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
    """softmax(scale * q k^T + bias) v over the rows of each sequence, bias being the table's value or, where a finite one is larger in
    size, 4096 with its sign.

    q [tokens][heads][head_dim], k, v [tokens][kv_heads][head_dim], bfloat16 or float16, with offsets (int32 [sequences + 1], rising
    from 0: sequence i is rows offsets[i] .. offsets[i + 1]); or [batch][length][...] without offsets.  Views are taken as they
    are (slices of one QKV tensor).  key_mask (int32, the leading shape of q): rows that are 0 are no keys.  scale: a number (not
    differentiated), default head_dim ** -0.5.  bias_table (float32 [num_buckets][heads]) adds
    bias_table[bucket(key - query)]; bidirectional: buckets for both directions (default: not causal).  Rows that attend nothing, and
    rows behind the last sequence, are 0.

    return_lse: also the float32 [heads][tokens] log-sum-exp of each row's scores, which packed_attention_backward takes.  Runs on
    the current stream of q's device.

    Differentiable once in q, k, v and bias_table under torch.autograd (out; lse is not), in reverse mode: tensors with forward-mode
    tangents are refused, and so is a call under make_fx or torch.jit.trace.  A step that is captured into a graph calls
    packed_attention_backward itself: a captured backward pass of autograd may wait for streams outside the capture."""
    _seen_whole(q, k, v, bias_table, scale)
    if getattr(scale, "requires_grad", False) and _grad_enabled():
        raise ValueError("packed_attention: scale is a number and has no gradient here; multiply q by what is to be learned")
    if (q.requires_grad or k.requires_grad or v.requires_grad or (bias_table is not None and bias_table.requires_grad)) and _grad_enabled():
        causal, scale, max_distance, bidirectional = _numbers(causal, scale, max_distance, bidirectional)
        out, lse = _function().apply(q, k, v, bias_table, offsets, key_mask, causal, scale, max_distance, bidirectional)
    else:
        out, lse = _forward(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional, return_lse)
    return (out, lse) if return_lse else out


def _forward(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional, with_lse):
    cfg, tokens, nseq, off, mask, table = _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional)
    z, zk, dtype, device = q.shape, k.shape, q.dtype, q.device
    own = q.is_contiguous()
    out = _empty_like(q) if own else _like(q)
    lse = q.new_empty((z[-2], tokens), dtype=_F32) if with_lse else None
    _capi.check(_capi.load().mi_attention_dev(_capi.get_ctx(device.index), cfg, tokens, nseq, off, mask,
                                              _own_rows(q, z[-2], z[-1]) if own else _rows("q", q, z, dtype, device),
                                              _rows("k", k, zk, dtype, device), _rows("v", v, zk, dtype, device), table, _own_rows(out, z[-2], z[-1]),
                                              lse.data_ptr() if with_lse else None, _capi.stream_arg(device)))
    return out, lse


def _not_captured(device) -> None:
    import torch
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("packed_attention: autograd under graph capture; call packed_attention(..., return_lse=True) on detached "
                               "tensors and packed_attention_backward")


@functools.lru_cache(maxsize=1)
def _function():
    """The autograd node (made on first use: importing this module does not import torch)."""
    import torch
    from torch.autograd.function import once_differentiable

    class PackedAttention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, bias_table, offsets, key_mask, causal, scale, max_distance, bidirectional):
            if q.is_cuda:
                _not_captured(q.device)
            out, lse = _forward(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional, True)
            ctx.save_for_backward(q, k, v, bias_table, offsets, key_mask, out, lse)
            ctx.form = {"causal": causal, "scale": scale, "max_distance": max_distance, "bidirectional": bidirectional}
            ctx.mark_non_differentiable(lse)
            return out, lse

        @staticmethod
        @once_differentiable
        def backward(ctx, dout, _):
            q, k, v, bias_table, offsets, key_mask, out, lse = ctx.saved_tensors
            _not_captured(q.device)
            if not dout.is_contiguous() or dout.data_ptr() % 16:       # autograd hands over expanded scalars, too
                dout = dout.clone(memory_format=torch.contiguous_format)
            grads = packed_attention_backward(dout, q, k, v, out, lse, offsets, key_mask=key_mask, bias_table=bias_table, **ctx.form)
            return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 6

    return PackedAttention


def packed_attention_backward(dout, q, k, v, out, lse, offsets=None, *, causal: bool = False, scale: Optional[float] = None, key_mask=None,
                              bias_table=None, max_distance: int = 128, bidirectional: Optional[bool] = None):
    """Gradients of sum(dout * packed_attention(q, k, v, ...)): (dq, dk, dv, dbias_table), the last None without a bias_table.

    out and lse are what packed_attention(..., return_lse=True) gave for the same arguments.  dk and dv sum over the query heads of
    a key head; rows behind the last sequence have gradient 0.  dbias_table is the gradient in the bias as it counts: the bound of
    4096 passes it through.  A repeated call gives the same bits."""
    _seen_whole(dout, q, k, v, out, lse, bias_table, scale)
    cfg, tokens, nseq, off, mask, table = _setup(q, k, v, offsets, causal, scale, key_mask, bias_table, max_distance, bidirectional)
    z, zk, dtype, device = q.shape, k.shape, q.dtype, q.device
    heads = z[-2]
    if lse.dtype != _F32 or tuple(lse.shape) != (heads, tokens) or not lse.is_contiguous() or lse.device != device:
        raise ValueError(f"packed_attention_backward: lse must be the contiguous float32 [{heads}][{tokens}] tensor of the forward pass")
    rows = (_own_rows(q, heads, z[-1]) if q.is_contiguous() else _rows("q", q, z, dtype, device), _rows("k", k, zk, dtype, device),
            _rows("v", v, zk, dtype, device), _rows("out", out, z, dtype, device), _rows("dout", dout, z, dtype, device))
    dq, dk, dv = _like(q), _like(k), _like(v)
    dtable = _like(bias_table) if bias_table is not None else None
    work = q.new_empty(_workspace(heads, zk[-2], z[-1], cfg.num_buckets, cfg.max_distance, cfg.bidirectional, tokens, nseq, offsets is not None), dtype=_F32)
    _capi.check(_capi.load().mi_attention_backward_dev(_capi.get_ctx(device.index), cfg, tokens, nseq, off, mask, rows[0], rows[1], rows[2], table, rows[3],
                                              lse.data_ptr(), rows[4], _own_rows(dq, heads, z[-1]), _own_rows(dk, zk[-2], z[-1]),
                                              _own_rows(dv, zk[-2], z[-1]), dtable.data_ptr() if dtable is not None else None, work.data_ptr(),
                                              work.numel() * 4, _capi.stream_arg(device)))
    return dq, dk, dv, dtable
