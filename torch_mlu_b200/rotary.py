"""Rotary positions on queries and keys, in front of any attention call of this package.

``rotary_embedding`` turns pairs of every row by the angles of the row's token, with one position per token or with several (time, height and
width of images and video), and differentiates through autograd; ``rotary_embedding_`` does so in place, for serving. The
reference has no such operator: its models bring their own.
"""
from __future__ import annotations

from typing import Optional, Sequence

from . import torch_glue

__all__ = ["rotary_embedding", "rotary_embedding_"]


def rotary_embedding(query, key, positions, inv_freq, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                     scaling: float = 1.0):
    """(query, key) with the first ``2 * len(inv_freq)`` elements of every row turned; ``key`` may be None.

    query / key are packed [tokens, heads, head_dim] or [batch, heads, seq_len, head_dim] (any strides with a unit head_dim stride), bf16 or
    fp16. positions (int32 or int64) are [tokens], respectively [seq_len] or [batch, seq_len]. With ``sections`` they have one more dimension in
    front, an axis per section, and the pairs of section a turn by the positions of axis a. Pair j is (j, j + rotary_dim / 2), or
    (2j, 2j + 1) with ``interleaved``, its angle position * inv_freq[j]; cosine and sine are multiplied by ``scaling``.
    inv_freq is fp32; the angle is formed in 64 bits. rotary_dim is a multiple of 16, strides are multiples of 8 elements.
    """
    calls = torch_glue.calls or torch_glue.load()
    return calls.rotary(query, key, positions, inv_freq, sections, interleaved, scaling, False)


def rotary_embedding_(query, key, positions, inv_freq, *, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                      scaling: float = 1.0):
    """``rotary_embedding`` in place, for tensors that need no gradient and share no elements."""
    calls = torch_glue.calls or torch_glue.load()
    return calls.rotary(query, key, positions, inv_freq, sections, interleaved, scaling, True)
