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

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _cabi
from .ops import _Workspace, _check, _stream_ptr, calculate_scale

__all__ = ["plan_step", "store", "attention", "StepPlan", "BLOCK_SIZES"]

BLOCK_SIZES = (16, 32, 64, 128)
_CODES = {torch.float8_e4m3fn: _cabi.CODE_E4M3, torch.int8: _cabi.CODE_INT8}


class StepPlan(NamedTuple):
    """What plan_step returns, all int32 on the device."""

    seq_lens: torch.Tensor    # [requests]: tokens of each, the new ones among them
    cu_seqlens: torch.Tensor  # [requests + 1]: offsets of each request's new tokens
    positions: torch.Tensor   # [num_tokens]: position of each new token in its request, 0 behind the last
    slots: torch.Tensor       # [num_tokens]: its place in the cache, block * block_size + place in the block; -1 behind the last
    ring_state: torch.Tensor  # [3]: where the free blocks begin in the ring, how many there are, why the step was refused (0: it was not)


def _words(device, **tensors):
    for name, t in tensors.items():
        _check(t.is_cuda and t.device == device and t.dtype == torch.int32, f"{name} must be an int32 tensor on the device of the others")
        _check(t.is_contiguous(), f"{name} must be contiguous")


def _table(block_table, device):
    _check(block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.is_cuda and block_table.device == device
           and block_table.stride(1) == 1, "block_table must be int32 [requests, max_blocks] with contiguous rows, on the device of the others")


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
    device = cached_lens.device
    _words(device, cached_lens=cached_lens, new_tokens=new_tokens, ring=ring, ring_state=ring_state)
    _table(block_table, device)
    B = block_table.size(0)
    _check(tuple(cached_lens.shape) == (B,) and tuple(new_tokens.shape) == (B,) and ring.dim() == 1 and tuple(ring_state.shape) == (3,),
           "cached_lens and new_tokens must be [requests], ring [num_blocks], ring_state [3]")
    new = lambda n: torch.empty(n, dtype=torch.int32, device=device)
    step = StepPlan(cached_lens if in_place else new(B), new(B + 1), new(num_tokens), new(num_tokens), ring_state if in_place else new(3))
    p = _cabi.PlanParams()
    p.cached_lens, p.new_tokens, p.block_table, p.ring, p.ring_state = (t.data_ptr() for t in (cached_lens, new_tokens, block_table, ring, ring_state))
    p.seq_lens, p.cu_seqlens, p.positions, p.slots, p.next_state = (t.data_ptr() for t in step)
    p.table_stride = block_table.stride(0)
    p.batch, p.max_blocks, p.num_blocks, p.block_size, p.num_tokens = B, block_table.size(1), ring.numel(), block_size, num_tokens
    with torch.cuda.device(device):
        _cabi.check(_cabi.load().sdpa_b200_plan_step(ctypes.byref(p), _stream_ptr(device)), "sdpa_b200_plan_step")
    return step


def _cache_params(x, key_cache, value_cache, key_scale, value_scale) -> _cabi.CacheParams:
    _check(x.is_cuda, "Input tensor must be on a CUDA device (this path has no CPU fallback)")
    _check(x.dtype in (torch.bfloat16, torch.float16), f"16-bit tensors must be fp16 or bf16 (got {x.dtype})")
    _check(key_cache.dim() == 4 and key_cache.shape == value_cache.shape, "key_cache and value_cache must both be [num_blocks, heads_kv, block_size, head_dim]")
    _check(key_cache.dtype in _CODES and value_cache.dtype == key_cache.dtype, "the caches must both be float8_e4m3fn or int8")
    N, H, S, D = key_cache.shape
    _check(x.size(-1) == D, "the caches must have the head_dim of the other tensors")
    for t in (key_cache, value_cache):
        _check(t.device == x.device and t.stride(3) == 1, "the caches must have a contiguous last dimension, on the device of the other tensors")
    for t in (key_scale, value_scale):
        _check(t.dtype == torch.float32 and tuple(t.shape) == (N, H) and t.is_contiguous() and t.device == x.device,
               "key_scale and value_scale must be contiguous fp32 [num_blocks, heads_kv] on the device of the other tensors")
    p = _cabi.CacheParams()
    p.k_cache, p.v_cache, p.k_scale, p.v_scale = (t.data_ptr() for t in (key_cache, value_cache, key_scale, value_scale))
    p.k_block_stride, p.k_head_stride, p.k_row_stride = key_cache.stride()[:3]
    p.v_block_stride, p.v_head_stride, p.v_row_stride = value_cache.stride()[:3]
    p.num_blocks, p.heads_kv, p.block_size, p.head_dim = N, H, S, D
    p.code = _CODES[key_cache.dtype]
    p.dtype = _cabi.DTYPE_F16 if x.dtype == torch.float16 else _cabi.DTYPE_BF16
    return p


def store(key, value, slots, key_cache, value_cache, key_scale, value_scale) -> None:
    """Put the keys and values of a step ([tokens, heads_kv, head_dim], any strides with a unit head_dim stride) into the cache, at ``slots``
    ([tokens], from plan_step; a token with a negative slot is left out).

    Every block and head that gets tokens has its scale raised to the smallest power of two at which the largest of them is a code (448 for
    e4m3, 127 for int8), unless it is as large already; tokens that the block holds are rounded again to a scale that has grown. A block
    whose first place is written starts anew. The tokens of a block stand next to each other, with rising slots, as plan_step gives them (fewer than 32
    that are left out may stand between them). A NaN or
    infinite element becomes a NaN of e4m3; in an int8 cache it makes the block's scale NaN until the block starts anew.
    """
    _check(key.dim() == 3 and key.shape == value.shape, "key and value must both be [tokens, heads_kv, head_dim]")
    _check(key.dtype == value.dtype and key.device == value.device and key.stride(2) == 1 and value.stride(2) == 1,
           "key and value must have the same dtype and device, and a contiguous last dimension")
    p = _cache_params(key, key_cache, value_cache, key_scale, value_scale)
    _check(key.size(1) == key_cache.size(1), "the caches must have the heads of key and value")
    _words(key.device, slots=slots)
    _check(tuple(slots.shape) == (key.size(0),), "slots must be [tokens]")
    if key.size(0) == 0:
        return
    p.key, p.value, p.slots, p.num_tokens = key.data_ptr(), value.data_ptr(), slots.data_ptr(), key.size(0)
    p.key_row_stride, p.key_head_stride = key.stride()[:2]
    p.value_row_stride, p.value_head_stride = value.stride()[:2]
    with torch.cuda.device(key.device):
        _cabi.check(_cabi.load().sdpa_b200_cache_store(ctypes.byref(p), _stream_ptr(key.device)), "sdpa_b200_cache_store")


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
    _check(query.dim() == 3 and query.stride(2) == 1, "query must be [tokens, heads_q, head_dim] with a contiguous last dimension")
    p = _cache_params(query, key_cache, value_cache, key_scale, value_scale)
    device = query.device
    _table(block_table, device)
    B = block_table.size(0)
    _words(device, seq_lens=seq_lens, **({} if cu_seqlens is None else {"cu_seqlens": cu_seqlens}))
    _check(tuple(seq_lens.shape) == (B,), "seq_lens must be [requests]")
    _check(cu_seqlens is None or tuple(cu_seqlens.shape) == (B + 1,), "cu_seqlens must have requests + 1 entries")
    out = torch.empty(query.shape, dtype=query.dtype, device=device)
    lse = torch.empty((query.size(1), query.size(0)), dtype=torch.float32, device=device)
    if query.numel() == 0:
        return out, lse
    p.q, p.out, p.lse = query.data_ptr(), out.data_ptr(), lse.data_ptr()
    p.q_row_stride, p.q_head_stride = query.stride()[:2]
    p.o_row_stride, p.o_head_stride = out.stride()[:2]
    p.block_table, p.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
    p.cu_seqlens_q = None if cu_seqlens is None else cu_seqlens.data_ptr()
    p.table_stride, p.max_blocks = block_table.stride(0), block_table.size(1)
    p.batch, p.total_q, p.heads_q = B, query.size(0), query.size(1)
    p.max_seqlen_q = int(max_seqlen_q)
    p.max_seqlen_k = block_table.size(1) * key_cache.size(2) if max_seqlen_k is None else int(max_seqlen_k)
    p.is_causal = int(bool(is_causal))
    p.softmax_scale = calculate_scale(query, scale)
    lib = _cabi.load()
    with torch.cuda.device(device):
        p.device_status = _Workspace.status_word(device).data_ptr()
        need = ctypes.c_size_t(0)
        _cabi.check(lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(need)), "workspace query")
        ws = torch.empty(need.value, dtype=torch.uint8, device=device)
        _cabi.check(lib.sdpa_b200_cache_attention(ctypes.byref(p), ws.data_ptr(), need.value, _stream_ptr(device)), "sdpa_b200_cache_attention")
    return out, lse
