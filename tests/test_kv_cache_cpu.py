"""The serving operators' boundary on the CPU: struct layouts, refusals by status code and message, no device touched."""
import ctypes
import os
import subprocess

import pytest
import torch

from torch_mlu_b200 import _cabi, kv_cache, rotary

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sdpa_b200.h")


@pytest.mark.parametrize("struct,name", [(_cabi.RotaryParams, "sdpa_b200_rotary_params"), (_cabi.PlanParams, "sdpa_b200_plan_params"),
                                         (_cabi.CacheParams, "sdpa_b200_cache_params")])
def test_structs_match_the_header(tmp_path, struct, name):
    fields = [f[0] for f in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({name}));']
                             + [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "layout")], check=True)
    vals = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert vals == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def _rotary():
    p = _cabi.RotaryParams()
    p.q = p.k = p.q_out = p.k_out = p.positions = p.inv_freq = 4096
    p.batch, p.length, p.heads_q, p.heads_k, p.head_dim, p.rotary_dim, p.axes = 2, 7, 4, 2, 128, 128, 1
    p.sections[0] = 64
    for x in ("q", "k", "qo", "ko"):
        for i, f in enumerate(("batch", "head", "row")):
            setattr(p, f"{x}_{f}_stride", 128 * (i + 1))
    p.scaling = 1.0
    return p


def _plan():
    p = _cabi.PlanParams()
    for f, _ in p._fields_[:10]:
        setattr(p, f, 4096)
    p.table_stride, p.batch, p.max_blocks, p.num_blocks, p.block_size, p.num_tokens = 8, 3, 8, 100, 64, 5
    return p


def _cache():
    p = _cabi.CacheParams()
    p.k_cache = p.v_cache = p.k_scale = p.v_scale = p.key = p.value = p.slots = p.q = p.out = p.lse = p.block_table = p.seq_lens = p.cu_seqlens_q = 4096
    p.num_blocks, p.block_size, p.heads_kv, p.head_dim = 10, 64, 2, 128
    for x in "kv":
        setattr(p, f"{x}_block_stride", 2 * 64 * 128)
        setattr(p, f"{x}_head_stride", 64 * 128)
        setattr(p, f"{x}_row_stride", 128)
    p.key_row_stride = p.value_row_stride = 256
    p.key_head_stride = p.value_head_stride = p.q_head_stride = p.o_head_stride = 128
    p.num_tokens, p.batch, p.heads_q, p.total_q = 5, 3, 8, 5
    p.q_row_stride = p.o_row_stride = 1024
    p.table_stride = p.max_blocks = 4
    p.max_seqlen_q, p.max_seqlen_k, p.softmax_scale, p.is_causal = 2, 200, 0.1, 1
    return p


def _set(**values):
    def change(p):
        for f, v in values.items():
            setattr(p, f, v)
    return change


def _sections(*values):
    def change(p):
        p.axes = len(values)
        p.sections[:len(values)] = values
    return change


REFUSED = [
    ("rotary", _rotary, _set(dtype=2), _cabi.UNSUPPORTED, "bf16 or f16"),
    ("rotary", _rotary, _set(length=0), _cabi.INVALID_ARG, "must be positive"),
    ("rotary", _rotary, _set(head_dim=130), _cabi.INVALID_ARG, "multiple of 8"),
    ("rotary", _rotary, _set(head_dim=264), _cabi.INVALID_ARG, "at most 256"),
    ("rotary", _rotary, _set(rotary_dim=40), _cabi.INVALID_ARG, "multiple of 16"),
    ("rotary", _rotary, _set(rotary_dim=144), _cabi.INVALID_ARG, "at most head_dim"),
    ("rotary", _rotary, _set(axes=5), _cabi.INVALID_ARG, "one to four axes"),
    ("rotary", _rotary, _sections(32, 33), _cabi.INVALID_ARG, "add up to"),
    ("rotary", _rotary, _sections(-1, 65), _cabi.INVALID_ARG, "add up to"),
    ("rotary", _rotary, _set(positions=0), _cabi.INVALID_ARG, "must be given"),
    ("rotary", _rotary, _set(k=0), _cabi.INVALID_ARG, "k is NULL"),
    ("rotary", _rotary, _set(q=4098), _cabi.INVALID_ARG, "16-byte aligned"),
    ("rotary", _rotary, _set(k_row_stride=100), _cabi.INVALID_ARG, "multiples of 8"),
    ("rotary", _rotary, _set(qo_row_stride=0), _cabi.INVALID_ARG, "those of the result positive"),
    ("plan_step", _plan, _set(slots=0), _cabi.INVALID_ARG, "NULL"),
    ("plan_step", _plan, _set(ring=4097), _cabi.INVALID_ARG, "4-byte aligned"),
    ("plan_step", _plan, _set(batch=0), _cabi.INVALID_ARG, "must be positive"),
    ("plan_step", _plan, _set(batch=16385), _cabi.INVALID_ARG, "1 to 16384"),
    ("plan_step", _plan, _set(num_tokens=0), _cabi.INVALID_ARG, "must be positive"),
    ("plan_step", _plan, _set(table_stride=7), _cabi.INVALID_ARG, "must hold max_blocks"),
    ("plan_step", _plan, _set(block_size=48), _cabi.INVALID_ARG, "16, 32, 64 or 128"),
    ("plan_step", _plan, _set(num_blocks=1 << 26), _cabi.INVALID_ARG, "32 bits"),
    ("cache_store", _cache, _set(code=2), _cabi.UNSUPPORTED, "e4m3 or int8"),
    ("cache_store", _cache, _set(dtype=2), _cabi.UNSUPPORTED, "bf16 or f16"),
    ("cache_store", _cache, _set(head_dim=96), _cabi.UNSUPPORTED, "head_dim 64 and 128"),
    ("cache_store", _cache, _set(block_size=8), _cabi.INVALID_ARG, "16, 32, 64 or 128"),
    ("cache_store", _cache, _set(num_blocks=1 << 25), _cabi.INVALID_ARG, "below 2^31"),
    ("cache_store", _cache, _set(v_cache=4104), _cabi.INVALID_ARG, "v_cache must be a 16-byte aligned"),
    ("cache_store", _cache, _set(k_row_stride=120), _cabi.INVALID_ARG, "multiples of 16 bytes"),
    ("cache_store", _cache, _set(k_head_stride=64), _cabi.INVALID_ARG, "at least head_dim"),
    ("cache_store", _cache, _set(v_scale=0), _cabi.INVALID_ARG, "k_scale and v_scale"),
    ("cache_store", _cache, _set(num_tokens=0), _cabi.INVALID_ARG, "num_tokens must be positive"),
    ("cache_store", _cache, _set(slots=0), _cabi.INVALID_ARG, "slots"),
    ("cache_store", _cache, _set(value=4100), _cabi.INVALID_ARG, "value must be a 16-byte aligned"),
    ("cache_store", _cache, _set(key_head_stride=4), _cabi.INVALID_ARG, "multiples of 8"),
    ("cache_attention", _cache, _set(heads_q=7), _cabi.INVALID_ARG, "must divide number of heads in query"),
    ("cache_attention", _cache, _set(max_seqlen_k=0), _cabi.INVALID_ARG, "sequence lengths must be positive"),
    ("cache_attention", _cache, _set(cu_seqlens_q=0), _cabi.INVALID_ARG, "one row of q per request"),
    ("cache_attention", _cache, _set(softmax_scale=0.0), _cabi.INVALID_ARG, "softmax_scale"),
    ("cache_attention", _cache, _set(q=4104), _cabi.INVALID_ARG, "q must be a 16-byte aligned"),
    ("cache_attention", _cache, _set(o_row_stride=4), _cabi.INVALID_ARG, "positive multiples of 8"),
    ("cache_attention", _cache, _set(seq_lens=0), _cabi.INVALID_ARG, "seq_lens must be given"),
    ("cache_attention", _cache, _set(table_stride=3), _cabi.INVALID_ARG, "must hold max_blocks"),
    ("cache_attention", _cache, _set(device_status=4098), _cabi.INVALID_ARG, "device_status"),
]


@pytest.mark.parametrize("call,make,change,status,needle", REFUSED)
def test_refusals(native_lib, call, make, change, status, needle):
    p = make()
    change(p)
    if call == "cache_attention":
        got = native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, 1 << 30, None)
        assert native_lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(ctypes.c_size_t())) == status
    else:
        got = getattr(native_lib, "sdpa_b200_" + call)(ctypes.byref(p), None)
    assert got == status and needle in native_lib.sdpa_b200_last_error().decode(), native_lib.sdpa_b200_last_error()


@pytest.mark.parametrize("change", [_set(positions=4098), _set(positions=4100, positions_64=1), _set(inv_freq=4097)])
def test_rotary_refuses_unaligned_positions(native_lib, change):
    p = _rotary()
    change(p)
    assert native_lib.sdpa_b200_rotary(ctypes.byref(p), None) == _cabi.INVALID_ARG and "aligned to their elements" in native_lib.sdpa_b200_last_error().decode()


def test_workspaces(native_lib):
    """Few rows: parts for two CTAs per SM, whatever the lengths are. Many rows: 16-bit keys and values, every request's filled up to 128. Too small a one is refused."""
    n = ctypes.c_size_t(0)
    size = lambda p: native_lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) or n.value
    p = _cache()
    few = size(p)
    p.max_seqlen_k, p.batch = 100000, 1
    assert size(p) == few
    p = _cache()
    p.max_seqlen_q = p.total_q = 200
    many = size(p)
    assert many >= 256 + 2 * 3 * 256 * 2 * 128 * 2
    for p, need in ((_cache(), few), (p, many)):
        assert native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, need - 1, None) == _cabi.INVALID_ARG
        assert native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4100, need, None) == _cabi.INVALID_ARG
    assert native_lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), None) == _cabi.INVALID_ARG
    for call in ("rotary", "plan_step", "cache_store"):
        assert getattr(native_lib, "sdpa_b200_" + call)(None, None) == _cabi.INVALID_ARG
    assert native_lib.sdpa_b200_cache_attention(None, 4096, 1 << 20, None) == _cabi.INVALID_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU answer")
def test_valid_calls_refuse_without_a_gpu(native_lib):
    assert native_lib.sdpa_b200_rotary(ctypes.byref(_rotary()), None) == _cabi.NO_DEVICE
    assert native_lib.sdpa_b200_plan_step(ctypes.byref(_plan()), None) == _cabi.NO_DEVICE
    assert native_lib.sdpa_b200_cache_store(ctypes.byref(_cache()), None) == _cabi.NO_DEVICE
    assert native_lib.sdpa_b200_cache_attention(ctypes.byref(_cache()), 4096, 1 << 30, None) == _cabi.NO_DEVICE


def test_host_tensors_are_refused():
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    ints = torch.zeros(4, dtype=torch.int32)
    cache, scale = torch.zeros(3, 2, 64, 128, dtype=torch.int8), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="CUDA device"):
        rotary.rotary_embedding(q, q, ints, torch.zeros(64))
    with pytest.raises(RuntimeError, match="int32 tensor on the device|CUDA"):
        kv_cache.plan_step(ints, ints, ints.view(4, 1), ints, ints[:3], block_size=16, num_tokens=4)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv_cache.store(q, q, ints, cache, cache, scale, scale)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv_cache.attention(q, cache, cache, scale, scale, ints.view(4, 1), ints)
