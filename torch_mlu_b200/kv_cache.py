"""The 8-bit paged cache of a serving loop and the attention over it.

Keys and values of all requests live in blocks of ``block_size`` tokens: codes [num_blocks, heads_kv, block_size, head_dim]
(torch.float8_e4m3fn or torch.int8) and one fp32 scale per block and head, [num_blocks, heads_kv]; an element is code * scale. ``block_table``
[requests, max_blocks] (int32) names the blocks of each request, in order. A step of a serving loop is

    step = plan_step(lens, new_tokens, block_table, ring, ring_state, block_size=64, num_tokens=T)     # once
    rotary.rotary_embedding_(q, k, step.positions, inv_freq)                                            # in every layer
    store(k, v, step.slots, key_cache, value_cache, key_scale, value_scale)
    out, lse = attention(q, key_cache, value_cache, key_scale, value_scale, block_table, step.seq_lens, step.cu_seqlens, max_q, max_k)

None of it reads anything back to the host. The reference has no paged cache.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import torch_glue

__all__ = ["plan_step", "store", "attention", "StepPlan", "BLOCK_SIZES"]

BLOCK_SIZES = (16, 32, 64, 128)


def _calls():
    return torch_glue.calls or torch_glue.load()


class StepPlan(NamedTuple):
    """What plan_step returns, all int32 on the device."""

    seq_lens: torch.Tensor    # [requests]: tokens of each, the new ones among them
    cu_seqlens: torch.Tensor  # [requests + 1]: offsets of each request's new tokens
    positions: torch.Tensor   # [num_tokens]: position of each new token in its request, 0 behind the last
    slots: torch.Tensor       # [num_tokens]: its place in the cache, block * block_size + place in the block; -1 behind the last
    ring_state: torch.Tensor  # [3]: where the free blocks begin in the ring, how many there are, why the step was refused (0: it was not)


def plan_step(cached_lens, new_tokens, block_table, ring, ring_state, *, block_size: int, num_tokens: int, in_place: bool = False) -> StepPlan:
    """Blocks, positions and slots of a serving step, from the lengths of the requests.

    ``new_tokens[i]`` tokens are added to request i, which has ``cached_lens[i]``; a negative number takes tokens back (all of them when the request
    has ended). Blocks that a request needs are taken from the front of ``ring``, those that it gives back are put at its end:
    ring [num_blocks] holds ``ring_state[1]`` free block numbers from index ``ring_state[0]`` on, modulo its size. ``block_table`` and ``ring`` are
    written; entries of the table behind a request's last block mean nothing. ``num_tokens`` is at least the number of new tokens.

    All or nothing: a step that does not fit changes nothing and comes back without new tokens, and ``ring_state[2]`` of the result says why: the
    number of blocks that were lacking, or -1 - i for the first request i whose length would be negative or pass the table, or whose
    tokens would pass ``num_tokens``. With ``in_place`` the new lengths and state are written into cached_lens and ring_state themselves
    (a captured graph can then be replayed step after step); else they are new tensors.
    """
    return StepPlan(*_calls().plan_step(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens, in_place))


def store(key, value, slots, key_cache, value_cache, key_scale, value_scale) -> None:
    """Put the keys and values of a step ([tokens, heads_kv, head_dim], any strides with a unit head_dim stride) into the cache, at ``slots``
    ([tokens], from plan_step; a token with a negative slot is left out).

    Every block and head that gets tokens has its scale raised to the smallest power of two at which the largest of them is a code (448 for
    e4m3, 127 for int8), unless it is as large already; tokens that the block holds are rounded again to a scale that has grown. A block
    whose first place is written starts anew. The tokens of a block stand next to each other, with rising slots, as plan_step gives them (fewer than 32
    that are left out may stand between them). A NaN or
    infinite element becomes a NaN of e4m3; in an int8 cache it makes the block's scale NaN until the block starts anew.
    """
    _calls().cache_store(key, value, slots, key_cache, value_cache, key_scale, value_scale)


def attention(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens=None, max_seqlen_q: int = 1,
              max_seqlen_k: Optional[int] = None, *, is_causal: bool = True, scale: Optional[float] = None):
    """(output [tokens, heads_q, head_dim], logsumexp [heads_q, tokens] fp32) of the step's queries over the cache.

    query is packed [tokens, heads_q, head_dim]; request i owns rows cu_seqlens[i] to cu_seqlens[i + 1] - 1, its last tokens, and sees the
    ``seq_lens[i]`` tokens that the blocks of ``block_table[i]`` hold, up to its own with ``is_causal`` (bottom-right aligned). Without cu_seqlens every
    request has one row. ``max_seqlen_q`` and ``max_seqlen_k`` are at least the most rows and the longest request; without max_seqlen_k it is what
    the table holds. Few rows per request stream the codes; with many (chunks of prompts) they are brought to 16 bits in the workspace, which takes
    4 * requests * max_seqlen_k * heads_kv * head_dim bytes, and the prefill kernel runs.

    A row without a visible key gets 0 and a logsumexp of +inf, rows outside every request are left unwritten, and a block number outside the
    cache makes the rows that see it NaN (their logsumexp +inf, as that of all NaN rows in this package).
    """
    return _calls().cache_attention(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens, max_seqlen_q, max_seqlen_k,
                                    is_causal, scale)
