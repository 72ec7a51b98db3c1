"""The 4-bit paged cache, and reading caches back, against restatements in 64 bits (oracle/cache_oracle.py).

Codes, scales and what is read back have to be equal. Attention, few rows: a weight is rounded to f16 twice (half a step is 2^-11), with what is left of V's scale and before, the result to its
type; exponentials and scores in 32 bits are covered by 1e-4 of the weights, as in test_kv_cache_gpu.py, to which the scores of 4-bit codes add what their accumulators lose: those hold up to 16
* 2^-24 sum |q| in the products' unit, and two steps of 32 dimensions round to 2^-23 of that, times the scale of K. Many rows: keys and values are exact in 16 bits, weights and result are rounded to the type, with 2^-10 for either where a call may take both paths."""
import ctypes
import math

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache_gpu import E4M3, INT8, _cache, _ints, _run
from torch_mlu_b200 import _cabi, kv_cache, ops

pytestmark = pytest.mark.gpu
INT4 = torch.uint8


def _cache4(dev, blocks, heads, block, dim, seed, block_first=True):
    """Random codes, and scales of five bits between 2^-5 and 2^-2."""
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = torch.randint(0, 256, (blocks, heads, block, dim // 2), generator=g, device=dev, dtype=INT4)
    if not block_first:  # the memory order [blocks, block, heads, dim]
        codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
    size = (blocks, heads, block, dim // 32)
    scales = torch.exp2(torch.randint(-5, -2, size, generator=g, device=dev).float()) * torch.randint(16, 32, size, generator=g, device=dev) / 16
    return codes, scales.bfloat16()


def _same(codes, scales, want_numbers, want_scales):
    assert torch.equal(scales.cpu().double().nan_to_num(1e30), want_scales.nan_to_num(1e30))
    assert torch.equal(orc.numbers4(codes.cpu()).double(), want_numbers)


def _batch4(dev, lens, rows, hq, hkv, dim, block, dtype, seed=0, poison=True, block_first=True, spare=2):
    """Queries, cache, table and lengths. What stands behind a request's last token has NaN for scales, and so have free blocks."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    blocks = sum(pages) + spare
    (kc, ks), (vc, vs) = (_cache4(dev, blocks, hkv, block, dim, seed + i, block_first) for i in (1, 2))
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(pages + [1]) + 3), 1 << 30, dtype=torch.int32)
    for i, n in enumerate(pages):
        mine = [order.pop() for _ in range(n)]
        table[i, :n] = torch.tensor(mine, dtype=torch.int32)
        if poison and n and lens[i] % block:
            ks[mine[-1], :, lens[i] % block:] = math.nan
            vs[mine[-1], :, lens[i] % block:] = math.nan
    if poison:
        ks[order], vs[order] = math.nan, math.nan
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], hq, dim, generator=g, device=dev).to(dtype)
    return q, kc, vc, ks, vs, table.to(dev), _ints(dev, lens), _ints(dev, cu)


def _compare(out, lse, b, causal=True, scale=None, many=False):
    q, kc, vc, ks, vs, table, lens, cu = b
    want, want_lse, size, most = orc.attention(q, kc, vc, ks, vs, table, lens, cu, causal, scale)
    half = torch.finfo(q.dtype).eps / 2
    assert float(most.nan_to_num(0).max()) < 60
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    # the scores' own error: [heads, tokens]
    lost = 2.0 ** -23 * 2 * 16 * scale * q.double().abs().sum(-1).t() * float(ks.nan_to_num(0, 0, 0).abs().max())
    tol = half * want.abs() + ((max(half, 2.0 ** -10) if many else 2.0 ** -10) + 1e-4 + lost.t()[..., None]) * size + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    longest = int(lens.max())
    if many and q.dtype == torch.float16:
        # the prefill kernel keeps weights in units of one that is no larger than the row's largest: those below 2^-14 are subnormal, off by up to 2^-25 whatever they are, and the row's sum is at
        # least 1. So up to 2^-25 of every value that the row sees
        tol = tol + 2.0 ** -25 * longest * 8 * float(vs.nan_to_num(0, 0, 0).abs().max())
    off = (out.double() - want).abs()
    ok = (off <= tol) | (out.isnan() & want.isnan())
    assert bool(ok.all()), (int((~ok).sum()), float((off - tol).nan_to_num(0).max()))
    ltol = 2.0 ** -24 * (longest / 128 * 9 + 40) + 2.0 ** -21 * most.clamp_min(1) + 2.0 ** -23 * want_lse.abs() + lost
    loff = (lse.double() - want_lse).abs()
    lok = (loff <= ltol) | ((lse == math.inf) & (want_lse.isnan() | want_lse.isinf()))
    assert bool(lok.all()), (int((~lok).sum()), float((loff - ltol).nan_to_num(0).max()))


# ---------------------------------------------------------------------------------------------- store
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,block,dim,lens", [(8, 64, 128, [(0, 1), (5, 1), (63, 1), (64, 1), (200, 1)]), (4, 16, 64, [(3, 40), (16, 16), (15, 2), (0, 77)]),
                                                  (1, 128, 128, [(100, 300), (0, 128), (127, 1)]), (3, 32, 64, [(31, 33), (1, 0), (7, 9)])])
def test_store(cuda_device, dtype, heads, block, dim, lens):
    g = torch.Generator(device=cuda_device).manual_seed(block)
    pages = [-(-(c + n) // block) for c, n in lens]
    order = torch.randperm(sum(pages) + 3, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in pages]
    slots = [tables[i][p // block] * block + p % block for i, (c, n) in enumerate(lens) for p in range(c, c + n)]
    slots = slots[:2] + [-1] + slots[2:] + [-1, -5]  # padding
    base = torch.randn(len(slots), 2 * heads + 3, dim, generator=g, device=cuda_device) * torch.exp2(torch.randint(-4, 5, (len(slots), 1, 1), generator=g, device=cuda_device))
    base = base.to(dtype)
    k, v = base[:, :heads], base[:, heads + 3:]
    kc, ks = _cache4(cuda_device, sum(pages) + 3, heads, block, dim, 5)
    vc, vs = _cache4(cuda_device, sum(pages) + 3, heads, block, dim, 6, block_first=False)
    want = orc.store4(k, torch.tensor(slots), kc, ks), orc.store4(v, torch.tensor(slots), vc, vs)
    kv_cache.store(k, v, _ints(cuda_device, slots), kc, vc, ks, vs)
    _same(kc, ks, *want[0])
    _same(vc, vs, *want[1])


@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 64), (3000, 7, 128), (1500, 5, 64)])
def test_store_in_any_order(cuda_device, tokens, heads, dim):
    """Tokens that go to places in no order, as of blocks that many requests share; a thread has one row or several."""
    g = torch.Generator(device=cuda_device).manual_seed(tokens)
    blocks = tokens // 16 + 2
    slots = torch.randperm(blocks * 16, generator=torch.Generator().manual_seed(2))[:tokens]
    k, v = torch.randn(2, tokens, heads, dim, generator=g, device=cuda_device).bfloat16()
    kc, ks = _cache4(cuda_device, blocks, heads, 16, dim, 5)
    vc, vs = _cache4(cuda_device, blocks, heads, 16, dim, 6)
    want = orc.store4(k, slots, kc, ks), orc.store4(v, slots, vc, vs)
    kv_cache.store(k, v, slots.int().to(cuda_device), kc, vc, ks, vs)
    _same(kc, ks, *want[0])
    _same(vc, vs, *want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_store_of_unusual_values(cuda_device, dtype):
    """Zeros, the type's largest and smallest values, elements at the border of a scale and halfway between codes, NaN and infinities, the same slot twice in a row, a slot behind the cache."""
    heads, block, dim = 2, 16, 64
    k = torch.zeros(40, heads, dim, dtype=torch.float64)
    k[1] = torch.finfo(dtype).max
    k[2] = torch.finfo(dtype).tiny
    k[3, :, 3], k[4, :, 3], k[5, :, 3] = 7.0, 7.03125, 7 * 31 / 16
    k[6, 0, 7], k[6, 1, 40], k[7, 0, 0] = math.nan, math.inf, -math.inf
    k[8], k[9] = 1.0, 2.0
    k[10, :, :15] = torch.arange(-7, 8) / 1.0
    k[11, :, :14] = torch.arange(-13, 14, 2) / 2.0  # halfway between codes of scale 1
    k[11, :, 20] = 7.0
    for i in range(12, 28):  # the same for every five-bit scale
        s = (i + 4) / 16
        k[i, :, :14] = torch.arange(-13, 14, 2) / 2.0 * s
        k[i, :, 20] = 7 * s
        k[i, :, 32:46] = torch.arange(-13, 14, 2) / 2.0 * s * 1.0078125
        k[i, :, 50] = -7 * s
    k[28:] = torch.randn(12, heads, dim, generator=torch.Generator().manual_seed(3)).double()
    k = k.to(dtype).to(cuda_device)
    slots = list(range(40))
    slots[8] = slots[9]
    slots[39] = 1 << 30
    kc, ks = _cache4(cuda_device, 3, heads, block, dim, 1)
    vc, vs = kc.clone(), ks.clone()
    want = orc.store4(k, torch.tensor(slots), kc, ks)
    kv_cache.store(k, k.clone(), _ints(cuda_device, slots), kc, vc, ks, vs)
    _same(kc, ks, *want)
    _same(vc, vs, *want)
    assert float(ks[0, 0, 0, 0]) == 2.0 ** -100


# ---------------------------------------------------------------------------------------------- load
def _equal(x, y):
    return bool(((x == y) | (x.isnan() & y.isnan())).all())


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,block,parts,spare", [
    (8, 128, 64, [(0, 301)], 0), (2, 64, 16, [(3, 1), (0, 0), (15, 2), (700, 333), (0, 0), (0, 0), (31, 65)], 7), (1, 128, 128, [(5, 0)] * 40 + [(127, 130)] + [(0, 0)] * 300, 1),
    (3, 64, 32, [(i % 50, i % 3) for i in range(600)], 90), (5, 128, 16, [(0, 0)], 33)])
def test_load(cuda_device, heads, dim, block, parts, spare, dtype, code):
    """Stretches that begin and end anywhere, requests that give none, rows of no request behind the last."""
    pages = [-(-(a + n) // block) for a, n in parts]
    blocks = sum(pages) + 2
    (kc, ks), (vc, vs) = (_cache4(cuda_device, blocks, heads, block, dim, i) if code == INT4 else _cache(cuda_device, blocks, heads, block, dim, code, i, i == 1) for i in (1, 2))
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(3)).tolist()
    table = torch.full((len(parts), max(pages) + 2), -1, dtype=torch.int32)
    for i, n in enumerate(pages):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    cu = torch.tensor([0] + [n for _, n in parts]).cumsum(0)
    total, first = int(cu[-1]) + spare, torch.tensor([a for a, _ in parts])
    args = kc, vc, ks, vs, table.to(cuda_device), cu.int().to(cuda_device), total
    got = kv_cache.load(*args, first.int().to(cuda_device), dtype=dtype)
    want = orc.load(kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table, cu, total, first)
    for x, y in zip(got, want):
        assert x.shape == (total, heads, dim) and x.dtype == dtype
        assert _equal(x.cpu(), y.float().to(dtype))
    if not any(a for a, _ in parts):
        for x, y in zip(kv_cache.load(*args, dtype=dtype), got):
            assert _equal(x, y)


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
def test_load_of_what_is_no_number(cuda_device, code):
    """Blocks outside the cache, tokens behind the table's row and in front of 0, scales that are NaN or infinite, elements beyond fp16's largest, offsets that do not begin at 0."""
    heads, dim, block = 2, 64, 16
    (kc, ks), (vc, vs) = (_cache4(cuda_device, 6, heads, block, dim, i) if code == INT4 else _cache(cuda_device, 6, heads, block, dim, code, i) for i in (1, 2))
    ks[1], vs[2], ks[3] = math.inf, math.nan, 3e5 if code == INT4 else 3e3
    table = torch.tensor([[0, 1, 2, 3], [4, 6, -1, 1 << 30], [5, 5, 5, 5]], dtype=torch.int32)
    cu, first = torch.tensor([3, 67, 131, 151]), torch.tensor([0, 0, 50])
    got = kv_cache.load(kc, vc, ks, vs, table.to(cuda_device), cu.int().to(cuda_device), 160, first.int().to(cuda_device), dtype=torch.float16)
    want = orc.load(kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table, cu, 160, first)
    for x, y in zip(got, want):
        y = y.clamp(-65504, 65504).float().half()
        assert _equal(x.cpu(), y)
        assert bool((x[:3] == 0).all()) and bool((x[151:] == 0).all()) and bool(x[85:131].isnan().all()) and bool(x[145:151].isnan().all())
    minus = kv_cache.load(kc, vc, ks, vs, table.to(cuda_device), cu.int().to(cuda_device), 160, _ints(cuda_device, [-1, -(1 << 31), (1 << 31) - 1]))
    assert bool(minus[0][3].isnan().all()) and bool((minus[0][4, 0, 0].cpu() == want[0][3, 0, 0].bfloat16())) and bool(minus[1][67:151].isnan().all())


def test_load_of_offsets_that_do_not_fit(cuda_device):
    """Offsets that fall, are negative or leave the outputs: nothing is written outside of them (bytes around the outputs are checked through the C ABI)."""
    heads, dim, block, rows = 2, 128, 16, 50
    (kc, ks), (vc, vs) = (_cache4(cuda_device, 6, heads, block, dim, i) for i in (1, 2))
    table = _ints(cuda_device, [[0, 1, 2, 3], [4, 5, 0, 1]])
    lib = _cabi.load()
    for cu in ([0, 70, 140], [-9, 20, 45], [40, 10, 60], [0, 1 << 30, -5], [60, 70, 80], [0, 0, 0]):
        whole = torch.full((2, rows + 20, heads, dim), 7.0, device=cuda_device).bfloat16()
        p = _params(kc, vc, ks, vs, torch.bfloat16)
        offsets = _ints(cuda_device, cu)
        p.block_table, p.table_stride, p.max_blocks, p.batch, p.cu_seqlens_k, p.num_tokens = table.data_ptr(), 4, 4, 2, offsets.data_ptr(), rows
        p.key_out, p.value_out = whole[0, 10:].data_ptr(), whole[1, 10:].data_ptr()
        assert lib.sdpa_b200_cache_load(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert bool((whole[:, :10] == 7).all()) and bool((whole[:, -10:] == 7).all())
        if cu[0] >= rows or cu == [0, 0, 0]:
            assert bool((whole[:, 10:-10] == 0).all())


def _params(kc, vc, ks, vs, dtype):
    p = _cabi.CacheParams()
    p.k_cache, p.v_cache, p.k_scale, p.v_scale = (x.data_ptr() for x in (kc, vc, ks, vs))
    for x, c in (("k", kc), ("v", vc)):
        for f, stride in zip(("block", "head", "row"), c.stride()):
            setattr(p, f"{x}_{f}_stride", stride)
    p.num_blocks, p.heads_kv, p.block_size, p.head_dim = kc.shape
    p.head_dim *= 2
    p.code, p.dtype = _cabi.CODE_INT4, _cabi.DTYPE_BF16 if dtype == torch.bfloat16 else _cabi.DTYPE_F16
    return p


# ---------------------------------------------------------------------------------------------- attention
ONE_ROW = [
    ([1000], 32, 8, 128, 64), ([1], 8, 8, 64, 16), ([1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], 8, 2, 128, 16),
    ([40, 0, 300, 0, 0, 5], 4, 1, 64, 32), ([9000, 3, 777, 128], 16, 16, 128, 128), ([33000], 8, 1, 128, 64), ([513, 300, 2000] * 20, 16, 4, 64, 64),
    ([100, 200, 300], 48, 4, 128, 32), ([100, 200, 300], 40, 2, 64, 64), ([64] * 150, 3, 3, 128, 16), ([20000], 8, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hkv,dim,block", ONE_ROW)
def test_one_row_each(cuda_device, lens, hq, hkv, dim, block, dtype):
    b = _batch4(cuda_device, lens, [1] * len(lens), hq, hkv, dim, block, dtype, seed=len(lens))
    _compare(*_run(b), b)
    # the same without offsets, and with the table's own bound on lengths
    _compare(*kv_cache.attention(*b[:7]), b)
    assert ops.device_status() == 0


SOME_ROWS = [
    ([1000, 300, 77], [4, 4, 4], 32, 8, 128, 64), ([50, 4, 3, 2, 0, 900], [4, 4, 4, 4, 2, 0], 16, 4, 64, 16), ([129, 500], [1, 9], 8, 1, 128, 32),
    ([2000, 1999, 64], [8, 3, 1], 64, 8, 128, 64), ([700, 90], [31, 64], 4, 4, 64, 128), ([5000], [20], 12, 12, 128, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,rows,hq,hkv,dim,block", SOME_ROWS)
def test_some_rows_each(cuda_device, lens, rows, hq, hkv, dim, block, dtype, causal):
    b = _batch4(cuda_device, lens, rows, hq, hkv, dim, block, dtype, seed=rows[0])
    _compare(*_run(b, is_causal=causal, scale=0.05), b, causal, 0.05)


@pytest.mark.parametrize("rows,hq,hkv,dim,dtype", [(1, 16, 8, 128, torch.bfloat16), (1, 32, 8, 64, torch.float16), (3, 32, 8, 128, torch.bfloat16), (5, 32, 8, 128, torch.float16),
                                                   (9, 64, 8, 128, torch.bfloat16)])
def test_many_units_to_a_share(cuda_device, rows, hq, hkv, dim, dtype):
    """Shares of many tiles and several units each: short requests, some empty, one long."""
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 1700 if dim == 64 else 900, (160,), generator=g).tolist()
    lens[3], lens[7], lens[40], lens[159] = 0, 1, 7000, 129
    b = _batch4(cuda_device, lens, [rows if i % 5 else 1 for i in range(160)], hq, hkv, dim, 16, dtype, seed=rows)
    _compare(*_run(b), b)
    assert ops.device_status() == 0


@pytest.mark.parametrize("lens,rows,hq,hkv,dim,dtype", [
    ([1000], 1, 32, 8, 128, torch.bfloat16), ([4000, 130, 0, 1], 1, 16, 4, 64, torch.float16), ([257, 128, 3, 900, 1024], 4, 8, 2, 128, torch.bfloat16),
    ([129, 256, 64, 255] * 4, 1, 32, 8, 128, torch.float16), ([2, 5000], 2, 32, 4, 128, torch.bfloat16), ([300] * 8, 16, 4, 4, 64, torch.float16)])
def test_few_short_units(cuda_device, lens, rows, hq, hkv, dim, dtype):
    """Units that clusters of CTAs take, of every size, and the same calls with a bound on lengths at which they are shared out by tiles."""
    b = _batch4(cuda_device, lens, [min(rows, n) if i % 3 == 2 else rows for i, n in enumerate(lens)], hq, hkv, dim, 16, dtype, seed=len(lens))
    for most in (max(lens), 1 << 20):
        for causal in (True, False):
            _compare(*_run(b, max_k=most, is_causal=causal), b, causal)
    assert ops.device_status() == 0


MANY_ROWS = [
    ([700, 600], [513, 520], 8, 2, 128, 64), ([1300, 130, 64], [600, 1, 0], 4, 4, 64, 16), ([300, 1000], [299, 300], 16, 2, 128, 128), ([520], [530], 1, 1, 64, 32),
    ([500, 0, 300], [490, 3, 300], 32, 2, 64, 16), ([257, 129, 128], [300, 129, 256], 32, 4, 64, 64), ([1000], [1000], 64, 8, 128, 32),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,rows,hq,hkv,dim,block", MANY_ROWS)
def test_many_rows_each(cuda_device, lens, rows, hq, hkv, dim, block, dtype, causal):
    b = _batch4(cuda_device, lens, rows, hq, hkv, dim, block, dtype, seed=rows[0])
    _compare(*_run(b, is_causal=causal), b, causal, many=True)
    assert ops.device_status() == 0


@pytest.mark.parametrize("rows", [1, 3, 30, 600])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_it(cuda_device, rows):
    """NaN and infinite scales of K and of V, a block outside the cache: the rows that see the token are NaN, the others are as without it; on both paths."""
    lens, each = [700, 300], [rows, min(rows, 40)]
    b = list(_batch4(cuda_device, lens, each, 8, 2, 128, 16, torch.bfloat16, seed=rows))
    table = b[5].cpu()
    at = lambda i, token: (int(table[i, token // 16]), slice(None), token % 16)
    b[3][at(0, 699)][:, 1], b[4][at(0, 690)][0, 3] = math.inf, math.nan
    b[4][at(1, 299)][:, 0] = -math.inf
    if rows > 100:  # a key and a value in the middle of the new tokens
        b[3][at(0, 400)][1, 2], b[4][at(0, 300)][0, 1] = math.nan, math.inf
    out, lse = _run(b)
    want = orc.attention(*b)[0]
    assert torch.equal(out.isnan(), want.isnan()) and 0 < int(out.isnan().sum()) and bool((lse == math.inf)[want.isnan().all(-1).t()].all())
    _compare(out, lse, tuple(b), many=rows > 500)
    b[5][1, 5] = b[1].shape[0]
    out, lse = _run(b)
    assert bool(out[each[0]:].isnan().all()) and torch.equal(out.isnan(), orc.attention(*b)[0].isnan())


@pytest.mark.parametrize("rows", [1, 20, 600])
def test_longer_than_the_table(cuda_device, rows):
    b = list(_batch4(cuda_device, [300, 200], [rows, 1], 4, 2, 64, 16, torch.float16))
    b[5] = b[5][:, :15].contiguous()
    out, lse = _run(b, max_k=300)
    assert bool(out[:rows].isnan().all()) and bool((lse[:, :rows] == math.inf).all())
    tail = (b[0][rows:], *b[1:5], b[5][1:], b[6][1:], _ints(cuda_device, [0, 1]))
    _compare(out[rows:], lse[:, rows:], tail)


@pytest.mark.parametrize("rows", [1, 4, 600])
def test_negative_zero_and_least_scales(cuda_device, rows):
    b = list(_batch4(cuda_device, [600, 64], [rows, 1], 4, 2, 64, 16, torch.bfloat16, seed=1))
    first = b[5][0, :37].long()
    b[3][first[1]] *= -1.0
    b[4][first[2]] *= -1.0
    b[4][first[3], :, :, 0] = 0.0
    b[4][first[4]] = 0.0
    b[3][first[5]] = 0.0
    b[4][first[6]] = 2.0 ** -100
    b[4][first[7], :, 3:9, 1] *= 2.0 ** -12
    _compare(*_run(b), tuple(b), many=rows > 500)


def test_values_far_apart(cuda_device):
    """Scales of V between 2^-90 and 2^120 whose keys weigh as much as the others once their scores are low enough: sums hold either. And queries of bf16's whole range."""
    b = list(_batch4(cuda_device, [400, 64], [1, 1], 4, 2, 64, 16, torch.bfloat16, seed=2))
    first = b[5][0, :25].long()
    b[4][first[3]] *= 2.0 ** 60
    b[4][first[9]] *= 2.0 ** 118
    b[4][first[12]] *= 2.0 ** -85
    out, lse = _run(b)
    want, want_lse, size, _ = orc.attention(*b)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2e-3 * size).all()) and bool(((lse.double() - want_lse).abs() < 1e-4).all())
    # the same sums where the far values weigh nothing: their keys' scores are 2^7 and more below the others'
    b = list(_batch4(cuda_device, [400, 64], [1, 1], 4, 2, 64, 16, torch.bfloat16, seed=3))
    b[1][first[9]], b[3][first[9]] = 0x99, 40.0  # codes of -7
    b[0] = b[0].abs()
    b[4][first[9]] *= 2.0 ** 110
    out, lse = _run(b)
    want, want_lse, size, most = orc.attention(*b)
    assert bool(((lse.double() - want_lse).abs() <= 2.0 ** -18 * most + 1e-4).all())
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2e-3 * size)[want.isfinite()].all())
    for up in (1e30, 1e36):
        b = list(_batch4(cuda_device, [400, 64], [1, 1], 4, 2, 64, 16, torch.bfloat16, seed=4))
        scaled = [b[0] * up, *b[1:3], (b[3].double() / (b[0] * up).double().div(b[0].double()).nanmedian()).bfloat16(), *b[4:]]
        out, lse = _run(scaled)
        want, _, size, _ = orc.attention(*scaled)
        assert bool(out.isfinite().all()) and bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2e-3 * size).all())


@pytest.mark.parametrize("rows", [1, 560, 1100])
def test_layouts(cuda_device, rows):
    """A cache whose blocks hold all heads of a token side by side, table rows and queries that are slices, against the plain ones: the same bits."""
    a = _batch4(cuda_device, [600, 700], [rows, 2], 8, 4, 128, 64, torch.bfloat16)
    q, kc, vc, ks, vs, table, sl, cu = a
    turn = lambda c: c.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.randn(q.shape[0], 20, 128, device=cuda_device).bfloat16()
    wide[:, 4:12] = q
    table2 = torch.full((2, table.size(1) + 5), -7, dtype=torch.int32, device=cuda_device)
    table2[:, :table.size(1)] = table
    one, two = _run(a), _run((wide[:, 4:12], turn(kc), turn(vc), ks, vs, table2[:, :table.size(1)], sl, cu))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    offsets = _ints(cuda_device, [0, 600, 1300])
    for x, y in zip(kv_cache.load(kc, vc, ks, vs, table, offsets, 1300), kv_cache.load(turn(kc), turn(vc), ks, vs, table2[:, :table.size(1)], offsets, 1300)):
        assert torch.equal(x, y)


def test_rows_outside_every_request_are_left(cuda_device):
    """Offsets that begin behind the first row and end in front of the last, and offsets that leave q; the outputs are read through the C ABI into buffers of a known filling."""
    lib = _cabi.load()
    for rows, many in (([1, 2], False), ([530, 2], True), ([1600, 2], True)):
        q, kc, vc, ks, vs, table, lens, cu = _batch4(cuda_device, [600, 64], rows, 4, 2, 64, 32, torch.bfloat16)
        pad = torch.full((3, 4, 64), math.nan, dtype=q.dtype, device=cuda_device)
        q2, cu2 = torch.cat([pad, q, pad]), cu + 3
        out, lse = torch.full_like(q2, 7.0), torch.full((4, q2.shape[0]), 7.0, device=cuda_device)
        p = _params(kc, vc, ks, vs, torch.bfloat16)
        p.q, p.out, p.lse, p.block_table, p.seq_lens, p.cu_seqlens_q = (t.data_ptr() for t in (q2, out, lse, table, lens, cu2))
        p.q_row_stride = p.o_row_stride = 256
        p.q_head_stride = p.o_head_stride = 64
        p.table_stride, p.max_blocks, p.batch, p.total_q, p.heads_q = table.stride(0), table.size(1), 2, q2.shape[0], 4
        p.max_seqlen_q, p.max_seqlen_k, p.is_causal, p.softmax_scale = max(rows), 600, 1, 0.125
        n = ctypes.c_size_t(0)
        assert lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
        ws = torch.full((n.value,), 255, dtype=torch.uint8, device=cuda_device)
        assert lib.sdpa_b200_cache_attention(ctypes.byref(p), ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert int(ws[:4].view(torch.int32)) == 0
        assert bool((out[:3] == 7).all()) and bool((out[-3:] == 7).all()) and bool((lse[:, :3] == 7).all()) and bool((lse[:, -3:] == 7).all())
        _compare(out[3:-3], lse[:, 3:-3], (q, kc, vc, ks, vs, table, lens, cu), many=many)


def test_offsets_past_32_bits(cuda_device):
    """A cache of 4.6 GB each for keys and values: blocks at both ends, through all three operators."""
    blocks, hkv, block, dim = 70400, 8, 128, 128
    assert blocks * hkv * block * dim // 2 > 1 << 32
    kc, vc = (torch.empty(blocks, hkv, block, dim // 2, dtype=INT4, device=cuda_device) for _ in range(2))
    ks, vs = (torch.full((blocks, hkv, block, dim // 32), 0.03, device=cuda_device, dtype=torch.bfloat16) for _ in range(2))
    mine = [blocks - 1, 0, blocks - 2, 66000]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for c in (kc, vc):
        c[mine] = torch.randint(0, 256, (4, hkv, block, dim // 2), generator=g, device=cuda_device, dtype=INT4)
    table = _ints(cuda_device, [mine])
    for rows in (1, 400):
        q = torch.randn(rows, 16, dim, generator=g, device=cuda_device).half()
        b = (q, kc, vc, ks, vs, table, _ints(cuda_device, [500]), _ints(cuda_device, [0, rows]))
        small = (q, kc[mine], vc[mine], ks[mine], vs[mine], _ints(cuda_device, [[0, 1, 2, 3]]), b[6], b[7])
        one, two = _run(b), _run(small)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    for x, y in zip(kv_cache.load(kc, vc, ks, vs, table, _ints(cuda_device, [0, 512]), 512), kv_cache.load(*small[1:6], _ints(cuda_device, [0, 512]), 512)):
        assert torch.equal(x, y)
    k = torch.randn(3, hkv, dim, generator=g, device=cuda_device).half()
    a, s = kc[mine].clone(), ks[mine].clone()
    want = orc.store4(k, torch.tensor([5, 6, 7]), a, s)
    kv_cache.store(k, k, _ints(cuda_device, [(blocks - 1) * block + i for i in (5, 6, 7)]), kc, vc, ks, vs)
    _same(kc[mine], ks[mine], *want)


@pytest.mark.parametrize("rows", [1, 3, 530, 1100])
def test_captured_and_replayed(cuda_device, rows):
    """One captured call of attention and load, replayed with other lengths, tables and queries; and two graphs that run side by side."""
    lens = [600, 900]
    a = _batch4(cuda_device, lens, [rows, 1], 8, 2, 128, 16, torch.bfloat16, poison=False)
    offsets = _ints(cuda_device, [0, 600, 1500])
    _run(a), kv_cache.load(*a[1:6], offsets, 1510)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((_run(a, max_q=max(rows, 1), max_k=1000), kv_cache.load(*a[1:6], offsets, 1510)))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in (lens, [590, 60], [601, 1]):
        a[6].copy_(_ints(cuda_device, n))
        offsets.copy_(_ints(cuda_device, [0, n[0], sum(n)]))
        a[0].normal_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = kv_cache.load(*a[1:6], offsets, 1510)
        for (out, lse), read in outs:
            _compare(out, lse, a, many=rows > 500)
            assert torch.equal(read[0], want[0]) and torch.equal(read[1], want[1])


def test_calls_on_two_streams_at_once(cuda_device):
    calls = [_batch4(cuda_device, [3000, 50, 700], [1, r, 2], 16, 4, 128, 32, torch.float16, seed=r) for r in (1, 3, 4, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        outs = []
        for s, b in zip(streams, calls):
            with torch.cuda.stream(s):
                outs.append(kv_cache.attention(*b, 4, 3000))
    torch.cuda.synchronize()
    for (out, lse), b in zip(outs, calls):
        _compare(out, lse, b)


def test_refusals(cuda_device):
    q, kc, vc, ks, vs, table, lens, cu = _batch4(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, torch.float16)
    k, slots = torch.zeros(2, 2, 64, device=cuda_device, dtype=torch.float16), _ints(cuda_device, [0, 1])
    for args, text in [((q.float(), kc, vc, ks, vs, table, lens), "fp16 or bf16"), ((q, kc, vc.view(torch.int8), ks, vs, table, lens), "uint8 with a scale"),
                       ((q, kc, vc, ks.float(), vs, table, lens), "4-bit caches must be contiguous bf16"), ((q, kc, vc, ks, vs[..., :1], table, lens), "4-bit caches must be contiguous bf16"),
                       ((q, kc, vc, ks.transpose(1, 2).contiguous().transpose(1, 2), vs, table, lens), "4-bit caches must be contiguous bf16"),
                       ((torch.cat([q, q], -1), kc, vc, ks, vs, table, lens), "head_dim"), ((q[:, :3], kc, vc, ks, vs, table, lens), "must divide"),
                       ((q, kc, vc, ks.cpu(), vs, table, lens), "CUDA")]:
        with pytest.raises(RuntimeError, match=text):
            kv_cache.attention(*args)
    with pytest.raises(RuntimeError, match="has no gradient"):
        kv_cache.attention(q.clone().requires_grad_(), kc, vc, ks, vs, table, lens)
    with pytest.raises(RuntimeError, match="keeps no gradient"):
        kv_cache.store(k.clone().requires_grad_(), k, slots, kc, vc, ks, vs)
    for caches in ((kc, kc, ks, vs), (kc, vc, ks, ks)):
        with pytest.raises(RuntimeError, match="of their own"):
            kv_cache.store(k, k, slots, *caches)
    for args, text in [((kc, vc, ks, vs, table, cu[:2], 5), "requests \\+ 1"), ((kc, vc, ks, vs, table, cu, -1), "negative"), ((kc, vc, ks, vs, table, cu, 5, lens[:1]), "first must be"),
                       ((kc, vc, ks, vs, table, cu.long(), 5), "cu_seqlens must be an int32"), ((kc, vc, ks, vs, table, cu, 1 << 31), "32 bits"),
                       ((kc, vc[:-1], ks, vs, table, cu, 5), "both be")]:
        with pytest.raises(RuntimeError, match=text):
            kv_cache.load(*args)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        kv_cache.load(kc, vc, ks, vs, table, cu, 5, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="no gradient"):
        kv_cache.load(kc, vc, ks.clone().requires_grad_(), vs, table, cu, 5)
    assert kv_cache.load(kc, vc, ks, vs, table, cu, 0)[0].shape == (0, 2, 64)
    with pytest.raises(RuntimeError, match="uint8 for 4-bit"):
        kv_cache.PagedCache(1, 4, 2, 64, 1, 4, dtype=torch.int32, device=cuda_device)


def test_operators_are_registered(cuda_device):
    """Through b200_sdpa, and seen by a tracer."""
    from torch.fx.experimental.proxy_tensor import make_fx
    b = _batch4(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, torch.float16)
    offsets = _ints(cuda_device, [0, 100, 190])
    args = (*b[1:6], offsets, 190, None, torch.float16)
    one, two = torch.ops.b200_sdpa.cache_load(*args), kv_cache.load(*args[:-2], dtype=torch.float16)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    traced = make_fx(lambda table: kv_cache.load(*b[1:5], table, offsets, 190)[0] + 1)(b[5])
    assert any("cache_load" in str(n.target) for n in traced.graph.nodes)
    assert torch.equal(traced(b[5]), kv_cache.load(*b[1:6], offsets, 190)[0] + 1)


# ---------------------------------------------------------------------------------------------- all of it together
@pytest.mark.parametrize("dtype,dim,block,captured", [(torch.bfloat16, 64, 16, False), (torch.float16, 128, 32, False), (torch.bfloat16, 128, 64, True)])
def test_serving_loop(cuda_device, dtype, dim, block, captured):
    """Requests come, grow and end over some steps of two layers. Every step's cache and results are held to the restatements, and what is read back gives the attention of the dense operators."""
    layers, hq, hkv, requests, most, tokens = 2, 8, 2, 5, 12, 150
    cache = kv_cache.PagedCache(layers, 40 * 64 // block, hkv, dim, requests, most * 64 // block, block_size=block, dtype=INT4, device=cuda_device)
    g = torch.Generator().manual_seed(block)
    inv_freq = (1e4 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().to(cuda_device)
    held = [0] * requests
    q, k, v = (torch.zeros(tokens, h, dim, dtype=dtype, device=cuda_device) for h in (hq, hkv, hkv))
    news = torch.zeros(requests, dtype=torch.int32, device=cuda_device)

    def step():
        plan = cache.step(news, tokens)
        return plan, [(x, *cache.attend(i, *x, 64, most * 64, inv_freq=inv_freq)) for i in range(layers) for x in [(q * (i + 1), k * (i + 1), v * (1 + 0.5 * i))]]

    graph = None
    for it in range(20):
        new = []
        for c in held:
            r = float(torch.rand((), generator=g))
            new.append(int(40 * r * 2) if c == 0 and r < 0.6 else 0 if c == 0 else -c if r < 0.08 or c > 600 else -min(c - 1, 3) if r < 0.2 else 1 if r < 0.9 else 60)
        while sum(max(n, 0) for n in new) > tokens:
            new[max(range(requests), key=lambda i: new[i])] //= 2
        live = sum(max(n, 0) for n in new)
        news.copy_(torch.tensor(new, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        k[live:], v[live:] = math.nan, math.inf  # behind the last token there may be anything
        before = [[t.clone() for t in (cache.key_cache[i], cache.key_scale[i], cache.value_cache[i], cache.value_scale[i])] for i in range(layers)]
        if captured:
            if graph is None:
                keep = [t.clone() for t in (cache.lens, cache.block_table, cache.ring, cache.ring_state)]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                side.synchronize()
                for t, old in zip((cache.lens, cache.block_table, cache.ring, cache.ring_state), keep):
                    t.copy_(old)
                for i in range(layers):
                    for t, old in zip((cache.key_cache[i], cache.key_scale[i], cache.value_cache[i], cache.value_scale[i]), before[i]):
                        t.copy_(old)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    plan, got = step()
            graph.replay()
        else:
            plan, got = step()
        held = [c + n for c, n in zip(held, new)]
        assert cache.lens.tolist() == held and cache.refused() == 0
        for i, ((qi, ki, vi), out, lse) in enumerate(got):
            kc0, ks0, vc0, vs0 = before[i]
            _same(cache.key_cache[i], cache.key_scale[i], *orc.store4(ki, plan.slots, kc0, ks0))
            _same(cache.value_cache[i], cache.value_scale[i], *orc.store4(vi, plan.slots, vc0, vs0))
            if live:
                b = (qi[:live], cache.key_cache[i], cache.value_cache[i], cache.key_scale[i], cache.value_scale[i], cache.block_table, plan.seq_lens, plan.cu_seqlens)
                _compare(out[:live], lse[:, :live], b, many=True)
                # the same rows from what is read back, through the varlen operator
                total = sum(held)
                rk, rv = cache.load(i, total + 3, dtype=dtype)
                cu_k = torch.tensor([0, *held]).cumsum(0).int().to(cuda_device)
                again = ops._flash_attention_forward(qi[:live], rk, rv, plan.cu_seqlens, cu_k, max(new), max(held), 0.0, True, False)
                _compare(again[0], again[1], b, many=True)
    assert ops.device_status() == 0
