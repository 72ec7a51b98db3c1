"""The 8-bit paged cache of a serving loop and the attention over it.

Keys and values of all requests live in blocks of ``block_size`` tokens: codes [num_blocks, heads_kv, block_size, head_dim]
(torch.float8_e4m3fn or torch.int8) and one fp32 scale per block and head, [num_blocks, heads_kv]; an element is code * scale. ``block_table``
[requests, max_blocks] (int32) names the blocks of each request, in order. A step of a serving loop is

    step = plan_step(lens, new_tokens, block_table, ring, ring_state, block_size=64, num_tokens=T)     # once
    rotary.rotary_embedding_(q, k, step.positions, inv_freq)                                            # in every layer
    store(k, v, step.slots, key_cache, value_cache, key_scale, value_scale)
    out, lse = attention(q, key_cache, value_cache, key_scale, value_scale, block_table, step.seq_lens, step.cu_seqlens, max_q, max_k)

None of it reads anything back to the host. ``PagedCache`` keeps the tensors and makes these calls. The reference has no paged cache.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import rotary, torch_glue

__all__ = ["plan_step", "store", "attention", "StepPlan", "PagedCache", "BLOCK_SIZES"]

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
    written; entries of the table behind a request's last block mean nothing. ``num_tokens`` is at least the number of new tokens, and at least 1.

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
    that are left out may stand between them; a block that came up again behind another would be worked on twice at a time). A NaN or
    infinite element becomes a NaN of e4m3; in an int8 cache it makes the block's scale NaN until the block starts anew. There is no gradient.
    """
    _calls().cache_store(key, value, slots, key_cache, value_cache, key_scale, value_scale)


def attention(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens=None, max_seqlen_q: int = 1,
              max_seqlen_k: Optional[int] = None, *, is_causal: bool = True, scale: Optional[float] = None):
    """(output [tokens, heads_q, head_dim], logsumexp [heads_q, tokens] fp32) of the step's queries over the cache.

    query is packed [tokens, heads_q, head_dim]; request i owns rows cu_seqlens[i] to cu_seqlens[i + 1] - 1, its last tokens, and sees the
    ``seq_lens[i]`` tokens that the blocks of ``block_table[i]`` hold, up to its own with ``is_causal`` (bottom-right aligned). Without cu_seqlens every
    request has one row. ``max_seqlen_q`` and ``max_seqlen_k`` are at least the most rows and the longest request; without max_seqlen_k it is what
    the table holds. Few rows per request stream the codes; with many (chunks of prompts) they are brought to 16 bits in the workspace and the prefill
    kernel runs: 4 * max_seqlen_k * heads_kv * head_dim bytes a request, for as many requests at a time as fit 4 GiB (where not even one does, the codes are streamed). That is exact with scales that are powers of two, as store gives
    them; with others every element is rounded once. Elements beyond the largest number of query's type are that number there (fp16: 65504, of which the code may be 65536),
    and fp16 queries over a cache that was filled from bf16 lose what fp16 cannot hold, below 2^-24.

    There is no gradient. A row without a visible key gets 0 and a logsumexp of +inf, rows outside every request are left unwritten, and a block number outside the
    cache makes the rows that see it NaN (their logsumexp +inf, as that of all NaN rows in this package), a length that passes the table's row all rows of its request.
    A key that is NaN reaches the rows that see it, a value any row of its request and kv head (in an int8 cache, whose block has the scale NaN then: the block's keys, the block's values).
    """
    return _calls().cache_attention(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens, max_seqlen_q, max_seqlen_k,
                                    is_causal, scale)


class PagedCache:
    """The cache of a model's layers and its bookkeeping, for up to ``max_requests`` requests of up to ``max_blocks`` blocks each.

        cache = PagedCache(layers, num_blocks, heads_kv, head_dim, max_requests, max_blocks)
        cache.step(new_tokens, num_tokens)                          # int32 [max_requests] on the device
        for layer in range(layers):
            out, lse = cache.attend(layer, q, k, v, max_seqlen_q, max_seqlen_k, inv_freq=inv_freq)

    A row of the table is a request; one that gets no new tokens takes no part in the step, and one that gives all of its tokens back (minus its length) is
    free for another. Lengths and free blocks are kept on the device and written in place, so that a captured step can be replayed.
    """

    def __init__(self, layers: int, num_blocks: int, heads_kv: int, head_dim: int, max_requests: int, max_blocks: int, *, block_size: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise RuntimeError(f"the caches must both be float8_e4m3fn or int8 (got {dtype})")
        if block_size not in BLOCK_SIZES:
            raise RuntimeError(f"block_size must be 16, 32, 64 or 128 (got {block_size})")
        shape = (layers, num_blocks, heads_kv, block_size, head_dim)
        ints = dict(dtype=torch.int32, device=device)
        self.block_size = block_size
        self.key_cache, self.value_cache = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.key_scale, self.value_scale = (torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        self.block_table = torch.full((max_requests, max_blocks), -1, **ints)
        self.lens = torch.zeros(max_requests, **ints)
        self.ring = torch.arange(num_blocks, **ints)
        self.ring_state = torch.tensor([0, num_blocks, 0], **ints)
        self.plan: Optional[StepPlan] = None

    def step(self, new_tokens, num_tokens: int) -> StepPlan:
        """plan_step in place: lengths, blocks and free blocks move on by ``new_tokens``."""
        self.plan = plan_step(self.lens, new_tokens, self.block_table, self.ring, self.ring_state, block_size=self.block_size, num_tokens=num_tokens,
                              in_place=True)
        return self.plan

    def refused(self) -> int:
        """Why the last step changed nothing, or 0: see plan_step. Waits for the device."""
        return int(self.ring_state[2])

    def attend(self, layer: int, query, key, value, max_seqlen_q: int = 1, max_seqlen_k: Optional[int] = None, *, inv_freq=None, positions=None,
               sections=None, interleaved: bool = False, is_causal: bool = True, scale: Optional[float] = None):
        """(output, logsumexp) of one layer for the tokens of the last step: keys and values ([tokens, heads_kv, head_dim]) go into the cache, then the queries
        ([tokens, heads_q, head_dim]) see it. With ``inv_freq`` queries and keys are turned first, in place, by the step's positions or by those given
        (see rotary.rotary_embedding)."""
        if self.plan is None:
            raise RuntimeError("PagedCache.attend: call step() first")
        if inv_freq is not None:
            rotary.rotary_embedding_(query, key, self.plan.positions if positions is None else positions, inv_freq, sections=sections, interleaved=interleaved)
        caches = (self.key_cache[layer], self.value_cache[layer], self.key_scale[layer], self.value_scale[layer])
        store(key, value, self.plan.slots, *caches)
        return attention(query, *caches, self.block_table, self.plan.seq_lens, self.plan.cu_seqlens, max_seqlen_q, max_seqlen_k, is_causal=is_causal, scale=scale)
