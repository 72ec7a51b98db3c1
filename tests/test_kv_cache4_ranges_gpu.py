"""The ends of the 4-bit cache's ranges, against the restatements in 64 bits: scales of V that are 0, all small or large, or different from group to group. Tolerances and helpers as in
test_kv_cache4_gpu.py; each dimension is held to the mean of its own values' magnitudes, so that small ones decide where nothing else stands."""
import io

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache4_gpu import INT4, _batch4, _cache4, _compare, _same
from test_kv_cache_gpu import E4M3, INT8, _cache, _ints, _run
from torch_mlu_b200 import kv_cache, ops

pytestmark = pytest.mark.gpu
LENS = [700, 333, 130]


def _moved(dev, rows, dim, block, by, seed):
    """Three requests; with few rows 40 times as many, so that a CTA has several tiles of a unit one after another."""
    times, heads = (40, (16, 8)) if rows < 10 else (1, (8, 2))
    b = _batch4(dev, LENS * times, [rows, min(rows, 40), 1] * times, *heads, dim, block, torch.bfloat16, seed=seed)
    b[4][:] = (b[4].double() * 2.0 ** by).bfloat16()
    return b


def _compare_products(out, lse, b, many):
    """_compare, where scales differ so much that a weight times a scale has no bits left in f16: none below 2^-24, where the row's largest such product is 2^13 or more. So up to 2^-38 of the
    largest scale for every token, times codes of up to 8."""
    want = orc.attention(*b)[0]
    lost = 2.0 ** -38 * 8 * int(b[6].max()) * float(b[4].nan_to_num(0).max())
    _compare(torch.where((out.double() - want).abs() <= lost, want, out.double()), lse, b, many=many)


@pytest.mark.parametrize("rows", [1, 3, 9, 30, 600])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 64)])
@pytest.mark.parametrize("by", [-94, -80, -60, -40, 0, 18, 22, 60, 100])
def test_scales_of_values_that_are_all_small_or_large(cuda_device, by, dim, block, rows):
    b = _moved(cuda_device, rows, dim, block, by, rows)
    _compare(*_run(b), b, many=rows > 500)
    assert ops.device_status() == 0


@pytest.mark.parametrize("rows", [1, 3, 9, 30])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 64)])
def test_largest_values(cuda_device, dim, block, rows):
    """Values of up to 2^127, in units of which the streaming kernel's sums are held. (Where many rows are brought to 16 bits they are sums of 700 weights of up to 2^8 times values, in fp32: 2^127 *
    700 * 2^8 does not fit it, and is no case there.)"""
    b = _moved(cuda_device, rows, dim, block, 126, rows)
    _compare(*_run(b), b)


@pytest.mark.parametrize("rows", [1, 3, 9, 30, 600])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 64)])
@pytest.mark.parametrize("by", [-80, -60, -40, -30, 0, 15, 18, 22, 60, 100])
@pytest.mark.parametrize("zero", [0.0, 2.0 ** -100])
def test_tokens_without_values(cuda_device, zero, by, dim, block, rows):
    """Tokens whose scales of V are 0, or what the store gives zeros: whole blocks in front, in the middle and at the end, and single ones between the others. They have weights and nothing else."""
    b = _moved(cuda_device, rows, dim, block, by, rows + 1)
    for i, n in enumerate(b[6].tolist()):
        mine = b[5][i, :-(-n // block)].long()
        whole = 128 // block  # of blocks
        b[4][mine[:whole] if i % 3 != 1 else mine[-whole:]] = zero
        if i % 3 == 0:
            b[4][mine[3 * whole:4 * whole]] = zero
        b[4][mine, :, 5::7] = zero
        b[4][mine[-1], :, n % block or block:] = float("nan")
    _compare_products(*_run(b), b, rows > 500)
    assert ops.device_status() == 0


@pytest.mark.parametrize("rows", [1, 3, 30])
def test_a_head_without_values(cuda_device, rows):
    b = _moved(cuda_device, rows, 128, 16, 0, rows)
    b[4][:, 1] = 0.0
    out, lse = _run(b)
    _compare(out, lse, b)
    group = b[0].shape[1] // b[1].shape[1]
    assert bool((out[:, group:2 * group] == 0).all())


@pytest.mark.parametrize("rows", [1, 9, 600])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("by", [(0, -9), (0, -12), (0, 19), (0, 22), (-30, 12), (0, -45), (30, -45)])
def test_blocks_of_other_scales(cuda_device, by, dim, rows):
    """Every second block's scales of V are moved one way, the others another: both ways that a step may go, in turn."""
    b = _moved(cuda_device, rows, dim, 64, 0, rows)
    b[4][::2] = (b[4][::2].double() * 2.0 ** by[0]).bfloat16()
    b[4][1::2] = (b[4][1::2].double() * 2.0 ** by[1]).bfloat16()
    _compare_products(*_run(b), b, rows > 500)


@pytest.mark.parametrize("rows", [1, 3, 9, 30, 600])
@pytest.mark.parametrize("dim,group", [(64, 0), (128, 3), (128, 1)])
@pytest.mark.parametrize("by", [-12, -16])
def test_a_group_of_small_values(cuda_device, by, dim, group, rows):
    """32 dimensions whose values are 2^-12 or 2^-16 of the others' for every token. Streamed, a weight times a scale has no bits below 2^-24 in f16, where the row's largest such product is 2^13 or
    more: up to 2^-38 of the largest scale for every token, times codes of up to 8."""
    b = _moved(cuda_device, rows, dim, 16, 0, rows)
    b[4][..., group] = (b[4][..., group].double() * 2.0 ** by).bfloat16()
    out, lse = _run(b)
    _compare(out, lse, b, many=rows > 500)  # (not loose: the sums' 2^-10 is of each dimension's own values)
    if rows <= 500:
        want, _, size, _ = orc.attention(*b)
        mine = slice(32 * group, 32 * group + 32)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2e-4) * size + 2.0 ** -38 * 8 * max(LENS) * float(b[4].nan_to_num(0).max())
        assert bool(((out.double() - want).abs() <= tol)[..., mine].all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_stored_zeros(cuda_device, dim, dtype):
    """Through the store: tokens of zero values, prompts that begin with them, a head that has nothing else."""
    heads, block, n = 2, 16, 500
    g = torch.Generator(device=cuda_device).manual_seed(dim)
    k, v = (torch.randn(n, heads, dim, generator=g, device=cuda_device).to(dtype) for _ in range(2))
    v[:40], v[100::9], v[200:300, 0], v[:, 1, 32:64] = 0, 0, 0, 0
    blocks = -(-n // block)
    kc, ks = _cache4(cuda_device, blocks, heads, block, dim, 1)
    vc, vs = _cache4(cuda_device, blocks, heads, block, dim, 2)
    slots = torch.randperm(blocks, generator=torch.Generator().manual_seed(1))
    slots = torch.tensor([int(slots[t // block]) * block + t % block for t in range(n)])
    want = orc.store4(v, slots, vc, vs)
    kv_cache.store(k, v, slots.int().to(cuda_device), kc, vc, ks, vs)
    _same(vc, vs, *want)
    table = (slots[::block] // block).int()[None].to(cuda_device)
    for rows in (1, 2, 25):
        q = torch.randn(rows, 4 * heads, dim, generator=g, device=cuda_device).to(dtype)
        b = (q, kc, vc, ks, vs, table, _ints(cuda_device, [n]), _ints(cuda_device, [0, rows]))
        out, lse = _run(b)
        _compare(out, lse, b)
        assert bool((out[:, 4:, 32:64] == 0).all())


# ---------------------------------------------------------------------------------------------- load
@pytest.mark.parametrize("code", [INT4, E4M3])
def test_what_is_loaded_has_memory_of_its_own(cuda_device, code):
    """Keys are kept, saved and changed without the values, and the other way round."""
    heads, dim, block = 2, 64, 16
    (kc, ks), (vc, vs) = (_cache4(cuda_device, 6, heads, block, dim, i) if code == INT4 else _cache(cuda_device, 6, heads, block, dim, code, i) for i in (1, 2))
    args = kc, vc, ks, vs, _ints(cuda_device, [[3, 1, 2]]), _ints(cuda_device, [0, 45]), 45
    key, value = kv_cache.load(*args)
    again = kv_cache.load(*args)
    for x in (key, value):
        assert x.is_contiguous() and x.storage_offset() == 0 and x.untyped_storage().nbytes() == x.numel() * 2
        with io.BytesIO() as f:
            torch.save(x, f)
            assert len(f.getvalue()) < x.numel() * 2 + 4096
    key.zero_()
    assert torch.equal(value, again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
def test_load_with_scales_of_all_their_bits(cuda_device, code, dtype):
    """Scales that store does not write (8 significant bits of bf16, 24 of fp32), elements below fp16's normal numbers: a product in 32 bits, rounded to 16. With 4-bit codes that product is
    exact."""
    heads, dim, block, n = 3, 128, 16, 300
    g = torch.Generator(device=cuda_device).manual_seed(1)
    caches, scales, want = [], [], []
    for i in (1, 2):
        c, s = _cache4(cuda_device, 20, heads, block, dim, i) if code == INT4 else _cache(cuda_device, 20, heads, block, dim, code, i)
        s = ((1 + torch.rand(s.shape, generator=g, device=cuda_device)) * torch.exp2(torch.randint(-30, 3, s.shape, generator=g, device=cuda_device).float())).to(s.dtype)
        x = orc.numbers4(c).float() * s.float().repeat_interleave(32, -1) if code == INT4 else c.float() * s[:, :, None, None]
        if code == INT4:
            assert torch.equal(x.double(), orc.elements(c, s))
        caches.append(c), scales.append(s)
        largest = torch.finfo(dtype).max
        want.append(x.clamp(-largest, largest).transpose(1, 2).flatten(0, 1)[:n].to(dtype))
    got = kv_cache.load(*caches, *scales, torch.arange(20, dtype=torch.int32, device=cuda_device)[None], _ints(cuda_device, [0, n]), n, dtype=dtype)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
