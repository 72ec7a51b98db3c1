"""Rotary positions on queries and keys, in front of any attention call of this package.

``rotary_embedding`` turns pairs of every row by the angles of the row's token, with one position per token or with several (time, height and
width of images and video), and differentiates through autograd; ``rotary_embedding_`` does so in place, for serving. The
reference has no such operator: its models bring their own.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _cabi
from .ops import _check, _stream_ptr

__all__ = ["rotary_embedding", "rotary_embedding_"]


def _sections(sections: Optional[Sequence[int]], positions, query, pairs: int):
    """(sections, whether positions have an axis dimension)"""
    if sections is None:
        return (pairs,), False
    sections = tuple(int(n) for n in sections)
    _check(1 <= len(sections) <= 4 and min(sections) >= 0 and sum(sections) == pairs,
           f"sections must be one to four numbers of pairs that add up to rotary_dim / 2 = {pairs} (got {sections})")
    return sections, True


def _check_inputs(query, key, positions, inv_freq):
    _check(query.dim() in (3, 4), "query must be packed [tokens, heads, head_dim] or [batch, heads, seq_len, head_dim]")
    for name, t in (("query", query), ("key", key)):
        if t is None:
            continue
        _check(t.is_cuda, f"{name} must be on a CUDA device (this path has no CPU fallback)")
        _check(t.dtype in (torch.bfloat16, torch.float16) and t.dtype == query.dtype, "query and key must be bf16 or fp16, both the same")
        _check(t.stride(-1) == 1, f"{name} must have a contiguous last dimension")
        _check(t.dim() == query.dim() and t.device == query.device and t.size(-1) == query.size(-1), "query and key must agree in dimensions, device and head_dim")
        if t.dim() == 3:
            _check(t.size(0) == query.size(0), "query and key must have the same tokens")
        else:
            _check(t.size(0) == query.size(0) and t.size(2) == query.size(2), "query and key must have the same batch and length")
    _check(inv_freq.dim() == 1 and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous() and inv_freq.device == query.device,
           "inv_freq must be a contiguous fp32 vector of rotary_dim / 2 frequencies on the device of query")
    _check(positions.dtype in (torch.int32, torch.int64) and positions.device == query.device, "positions must be int32 or int64, on the device of query")


def _position_strides(positions, query, axes: int, with_axes: bool):
    """(axis, batch, row) strides of positions: [axes,] tokens, or [axes,] [batch or 1,] length."""
    sizes = (query.size(0),) if query.dim() == 3 else (query.size(0), query.size(2))
    dims, stride = list(positions.shape), list(positions.stride())
    axis = 0
    if with_axes:
        _check(positions.dim() >= 1 and dims[0] == axes, f"positions must have {axes} axes in front (got shape {tuple(positions.shape)})")
        axis, dims, stride = stride[0], dims[1:], stride[1:]
    want = "[axes, ...]" if with_axes else ""
    if query.dim() == 3:
        _check(dims == [sizes[0]], f"positions must be {want}[tokens] (got shape {tuple(positions.shape)})")
        return axis, 0, stride[0]
    if len(dims) == 1:
        dims, stride = [1] + dims, [0] + stride
    _check(len(dims) == 2 and dims[0] in (1, sizes[0]) and dims[1] == sizes[1],
           f"positions must be {want}[length] or {want}[batch, length] (got shape {tuple(positions.shape)})")
    return axis, 0 if dims[0] == 1 else stride[0], stride[1]


def _strides(t):
    """(batch, head, row) strides of a packed or dense tensor"""
    return (0, t.stride(1), t.stride(0)) if t.dim() == 3 else (t.stride(0), t.stride(1), t.stride(2))


def _new_like(t):
    if t.dim() == 3:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    B, H, L, D = t.shape
    return torch.empty((B, L, H, D), dtype=t.dtype, device=t.device).transpose(1, 2)


def _rotate(query, key, positions, inv_freq, sections, interleaved, scaling, inverse, in_place):
    _check_inputs(query, key, positions, inv_freq)
    pairs = inv_freq.numel()
    sections, with_axes = _sections(sections, positions, query, pairs)
    pos = _position_strides(positions, query, len(sections), with_axes)
    tensors = (query,) if key is None else (query, key)
    outs = tensors if in_place else tuple(_new_like(t) for t in tensors)
    if query.numel() == 0:
        return outs[0], None if key is None else outs[1]
    p = _cabi.RotaryParams()
    for name, t, out in zip(("q", "k"), tensors, outs):
        setattr(p, name, t.data_ptr())
        setattr(p, name + "_out", out.data_ptr())
        for prefix, x in ((name, t), (name + "o", out)):
            for field, s in zip(("batch", "head", "row"), _strides(x)):
                setattr(p, f"{prefix}_{field}_stride", s)
    p.positions, p.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    p.batch, p.length = (1, query.size(0)) if query.dim() == 3 else (query.size(0), query.size(2))
    p.heads_q, p.heads_k = query.size(1), 0 if key is None else key.size(1)
    p.head_dim, p.rotary_dim, p.axes = query.size(-1), 2 * pairs, len(sections)
    p.sections[:len(sections)] = sections
    p.interleaved, p.inverse, p.positions_64 = int(interleaved), int(inverse), int(positions.dtype == torch.int64)
    p.dtype = _cabi.DTYPE_F16 if query.dtype == torch.float16 else _cabi.DTYPE_BF16
    p.scaling = scaling
    p.pos_axis_stride, p.pos_batch_stride, p.pos_row_stride = pos
    lib = _cabi.load()
    with torch.cuda.device(query.device):
        _cabi.check(lib.sdpa_b200_rotary(ctypes.byref(p), _stream_ptr(query.device)), "sdpa_b200_rotary")
    return outs[0], None if key is None else outs[1]


def rotary_embedding(query, key, positions, inv_freq, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                     scaling: float = 1.0):
    """(query, key) with the first ``2 * len(inv_freq)`` elements of every row turned; ``key`` may be None.

    query / key are packed [tokens, heads, head_dim] or [batch, heads, seq_len, head_dim] (any strides with a unit head_dim stride), bf16 or
    fp16. positions (int32 or int64) are [tokens], respectively [seq_len] or [batch, seq_len]. With ``sections`` they have one more dimension in
    front, an axis per section, and the pairs of section a turn by the positions of axis a. Pair j is (j, j + rotary_dim / 2), or
    (2j, 2j + 1) with ``interleaved``, its angle position * inv_freq[j]; cosine and sine are multiplied by ``scaling``.
    """
    return _rotate(query, key, positions, inv_freq, sections, interleaved, scaling, False, False)


def rotary_embedding_(query, key, positions, inv_freq, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                      scaling: float = 1.0):
    """``rotary_embedding`` in place, for tensors that need no gradient."""
    return _rotate(query, key, positions, inv_freq, sections, interleaved, scaling, False, True)
