"""The 4-bit paged cache without a GPU: argument checks through the C ABI, and the restatements against plain arithmetic."""
import ctypes
import math

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache_cpu import _cache, _set
from torch_mlu_b200 import _cabi, kv_cache


@pytest.fixture(scope="module")
def native_lib():
    return _cabi.load()


def _cache4():
    p = _cache()
    p.code = _cabi.CODE_INT4
    p.k_scale = p.v_scale = 1 << 13
    for x in ("k", "v"):
        for f, stride in zip(("row", "head", "block"), (p.head_dim // 2, p.head_dim // 2 * p.block_size, p.head_dim // 2 * p.block_size * p.heads_kv)):
            setattr(p, f"{x}_{f}_stride", stride)
    p.key_out = p.value_out = p.cu_seqlens_k = 1 << 14
    return p


REFUSED = [
    ("cache_store", _set(head_dim=96), _cabi.UNSUPPORTED, "4-bit cache is built for head_dim 64 and 128"),
    ("cache_store", _set(k_row_stride=48), _cabi.INVALID_ARG, "at least head_dim / 2"),
    ("cache_store", _set(v_block_stride=(1 << 40)), _cabi.INVALID_ARG, "multiples of 16 bytes"),
    ("cache_store", _set(k_scale=(1 << 13) + 8), _cabi.INVALID_ARG, "16-byte aligned"),
    ("cache_store", _set(slots=0), _cabi.INVALID_ARG, "slots"),
    ("cache_store", _set(num_tokens=(1 << 31) - 1), _cabi.INVALID_ARG, "too many tokens"),
    ("cache_attention", _set(v_scale=0), _cabi.INVALID_ARG, "k_scale and v_scale"),
    ("cache_attention", _set(heads_q=7), _cabi.INVALID_ARG, "must divide number of heads in query"),
    ("cache_load", _set(code=3), _cabi.UNSUPPORTED, "e4m3 or int8, or int4"),
    ("cache_load", _set(num_tokens=0), _cabi.INVALID_ARG, "must be positive"),
    ("cache_load", _set(num_tokens=(1 << 31) - 1), _cabi.UNSUPPORTED, "too many rows"),
    ("cache_load", _set(batch=0), _cabi.INVALID_ARG, "must be positive"),
    ("cache_load", _set(table_stride=3), _cabi.INVALID_ARG, "must hold max_blocks"),
    ("cache_load", _set(block_table=0), _cabi.INVALID_ARG, "must be given"),
    ("cache_load", _set(cu_seqlens_k=0), _cabi.INVALID_ARG, "must be given"),
    ("cache_load", _set(first=4098), _cabi.INVALID_ARG, "4-byte aligned"),
    ("cache_load", _set(value_out=4112), _cabi.INVALID_ARG, "value_out must be a 32-byte aligned"),
    ("cache_load", _set(key_out=0), _cabi.INVALID_ARG, "key_out must be a 32-byte aligned"),
]


@pytest.mark.parametrize("call,change,status,needle", REFUSED)
def test_refusals(native_lib, call, change, status, needle):
    p = _cache4()
    change(p)
    if call == "cache_attention":
        got = native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, 1 << 30, None)
    else:
        got = getattr(native_lib, "sdpa_b200_" + call)(ctypes.byref(p), None)
    assert got == status and needle in native_lib.sdpa_b200_last_error().decode(), native_lib.sdpa_b200_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU answer")
def test_valid_calls_refuse_without_a_gpu(native_lib):
    for code in (_cabi.CODE_INT4, _cabi.CODE_E4M3):
        p = _cache4() if code == _cabi.CODE_INT4 else _cache()
        p.key_out = p.value_out = p.cu_seqlens_k = 1 << 14
        for call in ("cache_store", "cache_load"):
            assert getattr(native_lib, "sdpa_b200_" + call)(ctypes.byref(p), None) == _cabi.NO_DEVICE
        assert native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, 1 << 30, None) == _cabi.NO_DEVICE
    assert native_lib.sdpa_b200_cache_load(None, None) == _cabi.INVALID_ARG


def test_host_tensors_are_refused():
    cache, scale, ints = torch.zeros(3, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 16, 2, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv_cache.load(cache, cache, scale, scale, ints.view(2, 2), ints[:3], 4)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv_cache.store(torch.zeros(4, 2, 64).bfloat16(), torch.zeros(4, 2, 64).bfloat16(), ints, cache, cache, scale, scale)


def test_paged_cache_of_four_bits():
    cache = kv_cache.PagedCache(3, 10, 2, 128, 4, 5, block_size=32, dtype=torch.uint8, device="cpu")
    assert cache.key_cache.shape == (3, 10, 2, 32, 64) and cache.value_scale.shape == (3, 10, 2, 32, 4) and cache.key_scale.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="multiple of 32"):
        kv_cache.PagedCache(1, 4, 2, 72, 1, 4, dtype=torch.uint8, device="cpu")


def test_numbers_of_a_byte():
    assert orc.numbers4(torch.tensor([[0x00, 0x7f, 0x8f, 0x91]], dtype=torch.uint8)).tolist() == [[0, 0, -1, 7, -1, -8, 1, -7]]


def test_scales_and_codes_of_the_restatement():
    """The least scale of five bits whose 7 covers the group, by trying them all; codes by trying all numbers, the even one of two as near."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(6, 2, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (6, 2, 1), generator=g).float())).bfloat16()
    x[5, 0, :14], x[5, 0, 20], x[5, 0, 14:20] = torch.arange(-13, 14, 2) / 2.0, 7.0, 0.0
    x[5, 0, 21:32] = 0.0
    codes, scales = torch.zeros(1, 2, 16, 32, dtype=torch.uint8), torch.zeros(1, 2, 16, 2, dtype=torch.bfloat16)
    values, scales = orc.store4(x, torch.arange(6), codes, scales)
    every = sorted(m * 2.0 ** e for m in range(16, 32) for e in range(-104, 60))
    for t in range(6):
        for h in range(2):
            for n in range(2):
                part = x[t, h, 32 * n:32 * n + 32].double().tolist()
                scale = next(s for s in every if s >= 2.0 ** -100 and 7 * s >= max(map(abs, part)))
                assert float(scales[0, h, t, n]) == scale
                want = [min(range(-7, 8), key=lambda c: (abs(v - c * scale), c % 2)) for v in part]
                assert values[0, h, t, 32 * n:32 * n + 32].tolist() == want
    assert values[0, 0, 5, :14].tolist() == [-6, -6, -4, -4, -2, -2, 0, 0, 2, 2, 4, 4, 6, 6] and math.isclose(float(scales[0, 0, 5, 0]), 1.0)
