"""The 8-bit paged cache against request-by-request restatements in 64 bits (oracle/cache_oracle.py).

Bookkeeping, codes and scales have to be equal. Attention, few rows: P is rounded to f16 (2^-11 of each weight), the result to its type
(half a step: 2^-8 bf16, 2^-11 f16); exponentials and scores in 32 bits add 2^-22 of the weight and of |score| (at most 60 here, which 1e-4 of the weights covers).
Many rows: P is rounded to the 16-bit type, twice half a step with the result. The logsumexp is a sum of at most 33000 weights, in 32 bits, in chains of
length / 128 * 9 additions and 40 merges: 2^-24 each, and 2^-21 of the largest |score|."""
import math

import pytest
import torch

from oracle import cache_oracle as orc
from torch_mlu_b200 import kv_cache, ops

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


# ---------------------------------------------------------------------------------------------- plan_step
def _plan_state(dev, cached, block, width, free, seed=0, blocks=None):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-c // block) for c in cached]
    blocks = blocks or sum(pages) + free
    order = torch.randperm(blocks, generator=g).tolist()
    table = [[-1] * width for _ in cached]
    for row, n in zip(table, pages):
        row[:n] = [order.pop() for _ in range(n)]
    first = int(torch.randint(blocks, (1,), generator=g))
    ring = [-1] * blocks
    for i, b in enumerate(order[:free]):
        ring[(first + i) % blocks] = b
    return table, ring, [first, min(free, len(order)), 0]


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("requests,block,tokens,free", [(1, 64, 1, 3), (64, 64, 64, 20), (5, 16, 777, 200), (300, 32, 5000, 400), (1030, 16, 9000, 900),
                                                        (2, 128, 20000, 400)])
def test_plan_step(cuda_device, requests, block, tokens, free):
    g = torch.Generator().manual_seed(requests)
    cached = torch.randint(0, 900, (requests,), generator=g).tolist()
    new = [min(int(x), max(1, tokens // requests)) for x in torch.randint(0, 2 * max(1, tokens // requests) + 1, (requests,), generator=g)]
    for i in range(0, requests, 7):
        if requests > 6:
            new[i] = -cached[i] if i % 2 else -(cached[i] // 3)
    width = -(-(max(cached) + max(new)) // block) + 1
    need = sum(max(0, -(-(c + n) // block) - -(-c // block)) for c, n in zip(cached, new))
    for spare in (free, 0, -1):  # ample, just enough, one too few
        table, ring, state = _plan_state(cuda_device, cached, block, width, max(need + spare, 0), requests)
        total = max(1, sum(max(n, 0) for n in new) + (5 if spare > 0 else 0))
        want = orc.plan_step(cached, new, table, ring, state, block, total)
        if spare < 0 and need > 0:
            assert want[4][2] == 1
        t, r = _ints(cuda_device, table), _ints(cuda_device, ring)
        step = kv_cache.plan_step(_ints(cuda_device, cached), _ints(cuda_device, new), t, r, _ints(cuda_device, state), block_size=block, num_tokens=total)
        got = [x.tolist() for x in (step.seq_lens, step.cu_seqlens, step.positions, step.slots, step.ring_state, t, r)]
        for name, a, b in zip(("seq_lens", "cu_seqlens", "positions", "slots", "state", "table", "ring"), got, want):
            assert a == b, (name, spare)


def test_plan_step_refuses_what_does_not_fit(cuda_device):
    """A negative length, a request longer than its table row, too many tokens: nothing changes, and the state names the first such request."""
    cached, block = [10, 100, 20], 16
    table, ring, state = _plan_state(cuda_device, cached, block, 7, 20)
    for new, tokens, code in (([1, 1, -21], 8, -3), ([1, 13, 1], 100, -2), ([5, 4, 1], 8, -2), ([1, 2**31 - 200, 1], 8, -2), ([-11, 1, -50], 8, -1)):
        t, r, c, s = (_ints(cuda_device, x) for x in (table, ring, cached, state))
        step = kv_cache.plan_step(c, _ints(cuda_device, new), t, r, s, block_size=block, num_tokens=tokens)
        assert step.ring_state.tolist() == [state[0], state[1], code]
        assert step.seq_lens.tolist() == cached and step.cu_seqlens.tolist() == [0] * 4 and step.slots.tolist() == [-1] * tokens
        assert t.tolist() == table and r.tolist() == ring


def test_plan_steps_in_place_and_replayed(cuda_device):
    """A captured step, replayed: requests grow over blocks, the ring runs round, ended requests give their blocks back."""
    block, width, blocks, requests = 16, 6, 14, 3
    cached, table, state = [0] * requests, [[-1] * width for _ in range(requests)], [9, blocks, 0]
    ring = [(5 * i) % blocks for i in range(blocks)]
    lens, t, r, s, new = (_ints(cuda_device, x) for x in (cached, table, ring, state, [1] * requests))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kv_cache.plan_step(lens.clone(), new, t.clone(), r.clone(), s.clone(), block_size=block, num_tokens=40)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step = kv_cache.plan_step(lens, new, t, r, s, block_size=block, num_tokens=40, in_place=True)
    g = torch.Generator().manual_seed(3)
    for it in range(40):
        n = [-c if c > 70 else int(x) for c, x in zip(cached, torch.randint(1, 13, (requests,), generator=g))]
        want = orc.plan_step(cached, n, table, ring, state, block, 40)
        new.copy_(_ints(cuda_device, n))
        graph.replay()
        assert step.seq_lens.data_ptr() == lens.data_ptr()
        got = [x.tolist() for x in (lens, step.cu_seqlens, step.positions, step.slots, s, t, r)]
        assert got == list(want), it
        cached, state, table, ring = want[0], want[4], want[5], want[6]


# ---------------------------------------------------------------------------------------------- store
def _cache(dev, blocks, heads, block, dim, code, seed, block_first=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(blocks, heads, block, dim, generator=g, device=dev) * (127 if code == INT8 else 448) / 5
    codes = x.round().clamp(-127, 127).to(code) if code == INT8 else x.to(code)
    if not block_first:  # the memory order [blocks, block, heads, dim]
        codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
    scales = torch.exp2(torch.randint(-9, -3, (blocks, heads), generator=g, device=dev).float())
    return codes, scales


def _same_cache(codes, scales, want_values, want_scales, touched=None):
    assert torch.equal(scales.cpu().double().nan_to_num(1e30), want_scales.nan_to_num(1e30))
    got, want = codes.cpu().float().double(), want_values
    ok = (got == want) | (got.isnan() & want.isnan()) | want_scales.isnan()[:, :, None, None]
    assert bool(ok.all()), int((~ok).sum())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,block,dim,lens", [(8, 64, 128, [(0, 1), (5, 1), (63, 1), (64, 1), (200, 1)]), (4, 16, 64, [(3, 40), (16, 16), (15, 2), (0, 77)]),
                                                  (1, 128, 128, [(100, 300), (0, 128), (127, 1)]), (3, 32, 64, [(31, 33), (1, 0), (7, 9)])])
def test_store(cuda_device, code, dtype, heads, block, dim, lens):
    g = torch.Generator(device=cuda_device).manual_seed(block)
    pages = [-(-(c + n) // block) for c, n in lens]
    order = torch.randperm(sum(pages) + 3, generator=torch.Generator().manual_seed(1)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in pages]
    slots = [tables[i][p // block] * block + p % block for i, (c, n) in enumerate(lens) for p in range(c, c + n)]
    slots = slots[:2] + [-1] + slots[2:] + [-1, -5]  # padding
    base = torch.randn(len(slots), 2 * heads + 3, dim, generator=g, device=cuda_device) * torch.exp2(torch.randint(-4, 5, (len(slots), 1, 1), generator=g, device=cuda_device))
    base = base.to(dtype)
    k, v = base[:, :heads], base[:, heads + 3:]
    kc, ks = _cache(cuda_device, sum(pages) + 3, heads, block, dim, code, 5)
    vc, vs = _cache(cuda_device, sum(pages) + 3, heads, block, dim, code, 6, block_first=False)
    want = orc.store(k, torch.tensor(slots), kc, ks), orc.store(v, torch.tensor(slots), vc, vs)
    kv_cache.store(k, v, _ints(cuda_device, slots), kc, vc, ks, vs)
    _same_cache(kc, ks, *want[0])
    _same_cache(vc, vs, *want[1])


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_store_of_unusual_values(cuda_device, code):
    """Zeros, the type's largest values, elements right at the border of a scale, NaN and infinities, the same slot twice in a row, scales that are no powers of two,
    slots behind the cache."""
    heads, block, dim = 2, 16, 64
    k = torch.zeros(14, heads, dim, dtype=torch.bfloat16, device=cuda_device)
    k[1] = 3.3895e38
    k[2, :, 3] = 448.0
    k[3, :, 3] = 450.0
    k[4, :, 5] = 127.0
    k[5, :, 5] = 127.5
    k[6, 0, 7], k[6, 1, 7] = math.nan, math.inf
    k[7, 0, 9] = -math.inf
    k[8], k[9] = 1.0, 2.0
    k[10], k[11] = 1e-38, 5.0
    k[12], k[13] = 7.0, 9.0
    # a block each for tokens 0..5; a NaN in a block that goes on; the same place twice; a block that goes on from a scale of 0.3; behind the cache
    slots = [0, 16, 32, 48, 64, 80, 96 + 3, 96 + 4, 112, 112, 128, 144 + 7, 10 * 16, 1 << 30]
    kc, ks = _cache(cuda_device, 10, heads, block, dim, code, 1)
    ks[9] = 0.3
    ks[6, 1] = 2.0 ** 20
    vc, vs = kc.clone(), ks.clone()
    want = orc.store(k, torch.tensor(slots), kc, ks)
    kv_cache.store(k, k.clone(), _ints(cuda_device, slots), kc, vc, ks, vs)
    _same_cache(kc, ks, *want)
    _same_cache(vc, vs, *want)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_store_token_by_token(cuda_device, code):
    """A block that fills up one token at a time, elements growing: scales rise, earlier tokens are rounded again each time."""
    heads, block, dim, g = 2, 16, 128, torch.Generator(device=cuda_device).manual_seed(9)
    kc, ks = _cache(cuda_device, 3, heads, block, dim, code, 1)
    vc, vs = _cache(cuda_device, 3, heads, block, dim, code, 2)
    want = (kc.cpu().float().double(), ks.cpu().double()), (vc.cpu().float().double(), vs.cpu().double())
    for i in range(20):
        k = (torch.randn(1, heads, dim, generator=g, device=cuda_device) * 1.4 ** i).bfloat16()
        v = (torch.randn(1, heads, dim, generator=g, device=cuda_device) * 1.4 ** (20 - i)).bfloat16()
        slot = 16 + i if i < 16 else i - 16
        want = [orc.store(x, torch.tensor([slot]), c.to(code), s) for x, (c, s) in zip((k, v), want)]
        kv_cache.store(k, v, _ints(cuda_device, [slot]), kc, vc, ks, vs)
        _same_cache(kc, ks, *want[0])
        _same_cache(vc, vs, *want[1])


@pytest.mark.parametrize("seed,block,tokens,most_left_out", [(0, 16, 1500, 31), (1, 32, 1500, 31), (2, 64, 2500, 3), (3, 128, 2500, 31), (4, 16, 40, 31), (5, 64, 300, 2), (6, 128, 5000, 0)])
def test_store_runs_of_any_shape(cuda_device, seed, block, tokens, most_left_out):
    """Runs of a block that begin and end anywhere, with tokens left out in them (-1, or behind the cache) and between them."""
    heads, dim, g = 2, 64, torch.Generator().manual_seed(seed)
    draw = lambda lo, hi: int(torch.randint(lo, hi + 1, (), generator=g))
    slots, blocks = [-1] * draw(0, 40), 0
    left_out = lambda n: slots.extend([-1 if draw(0, 1) else 1 << 29] * n)
    while len(slots) < tokens:
        place = draw(0, block - 1) if draw(0, 2) == 0 else 0
        count = min(draw(1, block) if draw(0, 2) else block, block - place)
        slot = blocks * block + place
        for i in range(count):
            if i and draw(0, 9) == 0:
                left_out(draw(0, most_left_out))
            slots.append(slot + i)
        blocks += 1
        if draw(0, 5) == 0:
            left_out(draw(0, 100))
    perm = torch.randperm(blocks, generator=g).tolist()
    slots = [perm[s // block] * block + s % block if 0 <= s < blocks * block else s for s in slots]
    k = torch.randn(len(slots), 2 * heads, dim, generator=torch.Generator(device=cuda_device).manual_seed(seed), device=cuda_device).bfloat16()
    kc, ks = _cache(cuda_device, blocks, heads, block, dim, E4M3, 5)
    vc, vs = _cache(cuda_device, blocks, heads, block, dim, E4M3, 6)
    want = orc.store(k[:, :heads], torch.tensor(slots), kc, ks), orc.store(k[:, heads:], torch.tensor(slots), vc, vs)
    kv_cache.store(k[:, :heads], k[:, heads:], _ints(cuda_device, slots), kc, vc, ks, vs)
    _same_cache(kc, ks, *want[0])
    _same_cache(vc, vs, *want[1])


# ---------------------------------------------------------------------------------------------- attention
def _batch(dev, lens, rows, hq, hkv, dim, block, code, dtype, seed=0, powers=True, poison=True, block_first=True, spare=2):
    """Queries, cache, table and lengths. What stands behind a request's last token is NaN (e4m3) or the largest code, free blocks have NaN scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    blocks = sum(pages) + spare
    kc, _ = _cache(dev, blocks, hkv, block, dim, code, seed + 1, block_first)
    vc, _ = _cache(dev, blocks, hkv, block, dim, code, seed + 2, block_first)
    unit = 5.0 / (127 if code == INT8 else 448)
    ks, vs = (torch.exp2(torch.randint(-1, 2, (blocks, hkv), generator=g, device=dev).float()) * 2.0 ** round(math.log2(unit)) for _ in range(2))
    if not powers:
        ks, vs = ks * (1 + torch.rand(blocks, hkv, generator=g, device=dev)), vs * (1 + torch.rand(blocks, hkv, generator=g, device=dev))
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(pages + [1]) + 3), 1 << 30, dtype=torch.int32)
    bad = math.nan if code == E4M3 else 127
    for i, n in enumerate(pages):
        mine = [order.pop() for _ in range(n)]
        table[i, :n] = torch.tensor(mine, dtype=torch.int32)
        if poison and n and lens[i] % block:
            kc[mine[-1], :, lens[i] % block:] = torch.tensor(bad, device=dev).to(code)
            vc[mine[-1], :, lens[i] % block:] = torch.tensor(bad, device=dev).to(code)
    if poison:
        ks[order], vs[order] = math.nan, math.nan
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], hq, dim, generator=g, device=dev).to(dtype)
    return q, kc, vc, ks, vs, table.to(dev), _ints(dev, lens), _ints(dev, cu)


def _compare(out, lse, b, causal=True, scale=None, many=False, cu=None):
    q, kc, vc, ks, vs, table, lens, cu_q = b
    want, want_lse, size, most = orc.attention(q, kc, vc, ks, vs, table, lens, cu_q if cu is None else cu, causal, scale)
    half = torch.finfo(q.dtype).eps / 2
    assert float(most.nan_to_num(0).max()) < 60
    tol = half * want.abs() + ((half if many else 2.0 ** -11) + 1e-4) * size + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    off = (out.double() - want).abs()
    ok = (off <= tol) | (out.isnan() & want.isnan())
    assert bool(ok.all()), (int((~ok).sum()), float((off - tol).nan_to_num(0).max()))
    longest = int(lens.max())
    ltol = 2.0 ** -24 * (longest / 128 * 9 + 40) + 2.0 ** -21 * most.clamp_min(1) + 2.0 ** -23 * want_lse.abs()
    loff = (lse.double() - want_lse).abs()
    lok = (loff <= ltol) | ((lse == math.inf) & (want_lse.isnan() | want_lse.isinf()))  # a NaN row has a logsumexp of +inf in all kernels here
    assert bool(lok.all()), (int((~lok).sum()), float((loff - ltol).nan_to_num(0).max()))


def _run(b, max_q=None, max_k=None, **kw):
    q, kc, vc, ks, vs, table, lens, cu = b
    max_q = max_q or max(1, int((cu[1:] - cu[:-1]).max()))
    return kv_cache.attention(q, kc, vc, ks, vs, table, lens, cu, max_q, max_k or max(1, int(lens.max())), **kw)


ONE_ROW = [
    ([1000], 32, 8, 128, 64), ([1], 8, 8, 64, 16), ([1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], 8, 2, 128, 16),
    ([40, 0, 300, 0, 0, 5], 4, 1, 64, 32), ([9000, 3, 777, 128], 16, 16, 128, 128), ([33000], 8, 1, 128, 64), ([513, 300, 2000] * 20, 16, 4, 64, 64),
    ([100, 200, 300], 48, 4, 128, 32), ([100, 200, 300], 40, 2, 64, 64), ([64] * 150, 3, 3, 128, 16),
]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hkv,dim,block", ONE_ROW)
def test_one_row_each(cuda_device, lens, hq, hkv, dim, block, dtype, code):
    b = _batch(cuda_device, lens, [1] * len(lens), hq, hkv, dim, block, code, dtype, seed=len(lens), powers=len(lens) % 2 == 0)
    _compare(*_run(b), b)
    # the same without offsets, and with the table's own bound on lengths
    out, lse = kv_cache.attention(*b[:7])
    _compare(out, lse, b)
    assert ops.device_status() == 0


SOME_ROWS = [
    ([1000, 300, 77], [4, 4, 4], 32, 8, 128, 64), ([50, 4, 3, 2, 0, 900], [4, 4, 4, 4, 2, 0], 16, 4, 64, 16), ([129, 500], [1, 9], 8, 1, 128, 32),
    ([2000, 1999, 64], [8, 3, 1], 64, 8, 128, 64), ([700, 90], [31, 64], 4, 4, 64, 128), ([5000], [20], 12, 12, 128, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("code,dtype", [(E4M3, torch.bfloat16), (INT8, torch.float16), (INT8, torch.bfloat16)])
@pytest.mark.parametrize("lens,rows,hq,hkv,dim,block", SOME_ROWS)
def test_some_rows_each(cuda_device, lens, rows, hq, hkv, dim, block, code, dtype, causal):
    b = _batch(cuda_device, lens, rows, hq, hkv, dim, block, code, dtype, seed=rows[0], powers=False)
    _compare(*_run(b, is_causal=causal, scale=0.05), b, causal, 0.05)


@pytest.mark.parametrize("rows,hq,hkv,dim,code,dtype", [(1, 16, 8, 128, E4M3, torch.bfloat16), (1, 32, 8, 64, INT8, torch.float16), (3, 32, 8, 128, INT8, torch.bfloat16),
                                                        (5, 32, 8, 128, E4M3, torch.float16), (9, 64, 8, 128, E4M3, torch.bfloat16)])
def test_many_units_to_a_share(cuda_device, rows, hq, hkv, dim, code, dtype):
    """Shares of many tiles and several units each, which count the hand-overs between units: short requests, some empty, one long."""
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 1700 if dim == 64 else 900, (160,), generator=g).tolist()
    lens[3], lens[7], lens[40], lens[159] = 0, 1, 7000, 129
    b = _batch(cuda_device, lens, [rows if i % 5 else 1 for i in range(160)], hq, hkv, dim, 16, code, dtype, seed=rows)
    _compare(*_run(b), b)
    assert ops.device_status() == 0


@pytest.mark.parametrize("lens,rows,hq,hkv,dim,code,dtype", [
    ([1000], 1, 32, 8, 128, E4M3, torch.bfloat16), ([4000, 130, 0, 1], 1, 16, 4, 64, INT8, torch.float16), ([257, 128, 3, 900, 1024], 4, 8, 2, 128, INT8, torch.bfloat16),
    ([129, 256, 64, 255] * 4, 1, 32, 8, 128, E4M3, torch.float16), ([2, 5000], 2, 32, 4, 128, E4M3, torch.bfloat16), ([300] * 8, 16, 4, 4, 64, E4M3, torch.float16)])
def test_few_short_units(cuda_device, lens, rows, hq, hkv, dim, code, dtype):
    """Units that clusters of CTAs take, of every size, and the same calls with a bound on lengths at which they are shared out by tiles."""
    b = _batch(cuda_device, lens, [min(rows, n) if i % 3 == 2 else rows for i, n in enumerate(lens)], hq, hkv, dim, 16, code, dtype, seed=len(lens), powers=False)
    for most in (max(lens), 1 << 20):
        for causal in (True, False):
            _compare(*_run(b, max_k=most, is_causal=causal), b, causal)
    assert ops.device_status() == 0


MANY_ROWS = [
    ([700, 600], [513, 520], 8, 2, 128, 64), ([1300, 130, 64], [600, 1, 0], 4, 4, 64, 16), ([300, 1000], [299, 300], 16, 2, 128, 128), ([520], [530], 1, 1, 64, 32),
    ([500, 0, 300], [490, 3, 300], 32, 2, 64, 16), ([257, 129, 128], [300, 129, 256], 32, 4, 64, 64), ([1000], [1000], 64, 8, 128, 32),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("code,dtype", [(E4M3, torch.bfloat16), (INT8, torch.float16)])
@pytest.mark.parametrize("lens,rows,hq,hkv,dim,block", MANY_ROWS)
def test_many_rows_each(cuda_device, lens, rows, hq, hkv, dim, block, code, dtype, causal):
    b = _batch(cuda_device, lens, rows, hq, hkv, dim, block, code, dtype, seed=rows[0])
    _compare(*_run(b, is_causal=causal), b, causal, many=True)
    assert ops.device_status() == 0


def test_both_paths_are_taken(cuda_device):
    """Many rows of many heads go through 16-bit copies in the workspace, which is then large; few do not, however long the table is."""
    torch.cuda.synchronize()
    used = []
    for rows, hq in (([1000], 64), ([2], 64)):
        b = _batch(cuda_device, [20000], rows, hq, 8, 128, 64, E4M3, torch.bfloat16)
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        _run(b)
        used.append(torch.cuda.max_memory_allocated() - before)
    copies = 2 * 20096 * 8 * 128 * 2
    assert used[0] > copies > 3 * used[1]


@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 600, 1], [3, 1100, 1]])
def test_a_bad_block_spoils_its_own_request_only(cuda_device, rows):
    b = list(_batch(cuda_device, [700, 650, 70], rows, 8, 2, 128, 16, E4M3, torch.bfloat16))
    b[5][1, 20] = (-1, 10 ** 6)[rows[0] == 1]
    out, lse = _run(b)
    mine = slice(rows[0], rows[0] + rows[1])
    # causal: rows whose last visible token stands in front of page 20 do not see it
    sees = torch.arange(650 - rows[1], 650, device=cuda_device) >= 320
    assert bool(out[mine][sees].isnan().all()) and bool((lse[:, mine][:, sees] == math.inf).all())
    _compare(out, lse, b, many=max(rows) > 500)


def test_a_request_longer_than_its_table_is_nan(cuda_device):
    b = list(_batch(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, INT8, torch.float16))
    b[6][0] = 100000
    out, lse = _run(b, max_k=128)
    assert bool(out[0].isnan().all()) and not bool(out[1].isnan().any())
    # all of its rows, also those that stand in front of the last
    b = list(_batch(cuda_device, [100, 90], [5, 2], 4, 2, 64, 16, E4M3, torch.bfloat16))
    b[6][0] = b[5].size(1) * 16 + 1
    out, lse = _run(b, max_k=400)
    assert bool(out[:5].isnan().all()) and not bool(out[5:].isnan().any())


def test_inference_mode(cuda_device):
    """Tensors made under torch.inference_mode, as a server makes them."""
    b = _batch(cuda_device, [100, 90], [5, 2], 4, 2, 64, 16, INT8, torch.bfloat16)
    want = _run(b)
    with torch.inference_mode():
        c = tuple(t.clone() for t in b)
        out, lse = _run(c)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        k = torch.randn(3, 2, 64, device=cuda_device).bfloat16()
        kv_cache.store(k, k, _ints(cuda_device, [0, 1, 2]), c[1], c[2], c[3], c[4])
        step = kv_cache.plan_step(c[6], torch.ones_like(c[6]), c[5], torch.arange(8, device=cuda_device).int(), _ints(cuda_device, [0, 8, 0]), block_size=16, num_tokens=4)
        assert step.seq_lens.tolist() == [101, 91] and step.positions.tolist() == [100, 90, 0, 0]


def test_gradients_are_refused(cuda_device):
    b = list(_batch(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, INT8, torch.float16))
    b[0].requires_grad_()
    with pytest.raises(RuntimeError, match="has no gradient"):
        _run(b)
    with torch.no_grad():
        assert not _run(b)[0].requires_grad


def test_store_refuses_gradients_and_shared_caches(cuda_device):
    k = torch.randn(2, 2, 64, device=cuda_device).bfloat16()
    kc, ks = _cache(cuda_device, 3, 2, 16, 64, E4M3, 1)
    vc, vs = _cache(cuda_device, 3, 2, 16, 64, E4M3, 2)
    before, slots = [x.clone() for x in (kc.view(torch.int8), ks)], _ints(cuda_device, [0, 1])
    for key, value in ((k.clone().requires_grad_(), k), (k, k.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="keeps no gradient"):
            kv_cache.store(key, value, slots, kc, vc, ks, vs)
    with pytest.raises(RuntimeError, match="of their own"):
        kv_cache.store(k, k, slots, kc, kc, ks, vs)
    with pytest.raises(RuntimeError, match="of their own"):
        kv_cache.store(k, k, slots, kc, vc, ks, ks)
    assert torch.equal(kc.view(torch.int8), before[0]) and torch.equal(ks, before[1])
    with torch.no_grad():
        kv_cache.store(k.clone().requires_grad_(), k, slots, kc, vc, ks, vs)
    assert not torch.equal(kc.view(torch.int8), before[0])


def test_rows_outside_every_request_are_left(cuda_device):
    """Offsets that begin behind the first row and end in front of the last; the outputs are read through the C ABI into buffers of a known filling."""
    import ctypes
    from torch_mlu_b200 import _cabi
    for rows, many in (([1, 2], False), ([530, 2], True), ([1600, 2], True)):
        q, kc, vc, ks, vs, table, lens, cu = _batch(cuda_device, [600, 64], rows, 4, 2, 64, 32, INT8, torch.bfloat16)
        pad = torch.full((3, 4, 64), math.nan, dtype=q.dtype, device=cuda_device)
        q2, cu2 = torch.cat([pad, q, pad]), cu + 3
        out = torch.full_like(q2, 7.0)
        lse = torch.full((4, q2.shape[0]), 7.0, device=cuda_device)
        p = _cabi.CacheParams()
        p.k_cache, p.v_cache, p.k_scale, p.v_scale = (x.data_ptr() for x in (kc, vc, ks, vs))
        for x, c in (("k", kc), ("v", vc)):
            for f, stride in zip(("block", "head", "row"), c.stride()):
                setattr(p, f"{x}_{f}_stride", stride)
        p.num_blocks, p.heads_kv, p.block_size, p.head_dim = kc.shape
        p.code, p.dtype = _cabi.CODE_INT8, _cabi.DTYPE_BF16
        p.q, p.out, p.lse, p.block_table, p.seq_lens, p.cu_seqlens_q = (t.data_ptr() for t in (q2, out, lse, table, lens, cu2))
        p.q_row_stride = p.o_row_stride = 256
        p.q_head_stride = p.o_head_stride = 64
        p.table_stride, p.max_blocks, p.batch, p.total_q, p.heads_q = table.stride(0), table.size(1), 2, q2.shape[0], 4
        p.max_seqlen_q, p.max_seqlen_k, p.is_causal, p.softmax_scale = max(rows), 600, 1, 0.125
        n = ctypes.c_size_t(0)
        lib = _cabi.load()
        assert lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
        ws = torch.full((n.value,), 255, dtype=torch.uint8, device=cuda_device)  # NaN everywhere; and no device_status: the workspace's first word is used
        assert lib.sdpa_b200_cache_attention(ctypes.byref(p), ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert int(ws[:4].view(torch.int32)) == 0
        assert bool((out[:3] == 7).all()) and bool((out[-3:] == 7).all()) and bool((lse[:, :3] == 7).all()) and bool((lse[:, -3:] == 7).all())
        _compare(out[3:-3], lse[:, 3:-3], (q, kc, vc, ks, vs, table, lens, cu), many=many)


@pytest.mark.parametrize("rows", [1, 560, 1100])
def test_layouts(cuda_device, rows):
    """A cache whose blocks hold all heads of a token side by side, table rows and queries that are slices, against the plain ones: the same bits."""
    lens, each = [600, 700], [rows, 2]
    a = _batch(cuda_device, lens, each, 8, 4, 128, 64, E4M3, torch.bfloat16)
    q, kc, vc, ks, vs, table, sl, cu = a
    turn = lambda c: c.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.randn(q.shape[0], 20, 128, device=cuda_device).bfloat16()
    wide[:, 4:12] = q
    table2 = torch.full((2, table.size(1) + 5), -7, dtype=torch.int32, device=cuda_device)
    table2[:, :table.size(1)] = table
    one, two = _run(a), _run((wide[:, 4:12], turn(kc), turn(vc), ks, vs, table2[:, :table.size(1)], sl, cu))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_scales_of_zero_and_values_far_apart(cuda_device):
    """A block of zeros with the least scale, blocks of V that differ by 2^40, queries of bf16's whole range."""
    b = list(_batch(cuda_device, [200, 64], [1, 1], 4, 2, 64, 16, INT8, torch.bfloat16))
    first = b[5][0, :12].long()
    b[1][first[2]] = 0
    b[2][first[2]] = 0
    b[3][first[2]] = b[4][first[2]] = 2.0 ** -100
    b[4][first[5]] = 0.0
    b[4][first[6]] *= 2.0 ** -20
    b[4][first[7]] *= 2.0 ** 20
    b[0][0] *= 1e-3
    _compare(*_run(b), b)
    b[0][1] = b[0][1] * 1e30
    b[3] *= 1e-30
    out, lse = _run(b)
    want = orc.attention(*b)[0]
    assert bool(((out[1].double() - want[1]).abs() <= 2.0 ** -8 * want[1].abs() + 1e-3 * want[1].abs().amax()).all())


def test_offsets_past_32_bits(cuda_device):
    """A cache of 4.6 GB each for keys and values: blocks at both ends."""
    blocks, hkv, block, dim = 35200, 8, 128, 128
    assert blocks * hkv * block * dim > 1 << 32
    kc, vc = (torch.empty(blocks, hkv, block, dim, dtype=INT8, device=cuda_device) for _ in range(2))
    ks, vs = (torch.full((blocks, hkv), 0.03, device=cuda_device) for _ in range(2))
    mine = [blocks - 1, 0, blocks - 2, 33000]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for c in (kc, vc):
        c[mine] = torch.randint(-127, 128, (4, hkv, block, dim), generator=g, device=cuda_device, dtype=INT8)
    table = _ints(cuda_device, [mine])
    for rows in (1, 400):
        q = torch.randn(rows, 16, dim, generator=g, device=cuda_device).half()
        b = (q, kc, vc, ks, vs, table, _ints(cuda_device, [500]), _ints(cuda_device, [0, rows]))
        small = (q, kc[mine], vc[mine], ks[mine], vs[mine], _ints(cuda_device, [[0, 1, 2, 3]]), b[6], b[7])
        one, two = _run(b), _run(small)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    k = torch.randn(3, hkv, dim, generator=g, device=cuda_device).half()
    slots = _ints(cuda_device, [(blocks - 1) * block + i for i in (5, 6, 7)])
    a, s = kc[mine].clone(), ks[mine].clone()
    want = orc.store(k, torch.tensor([5, 6, 7]), a, s)
    kv_cache.store(k, k, slots, kc, vc, ks, vs)
    _same_cache(kc[mine], ks[mine], *want)


@pytest.mark.parametrize("rows", [1, 3, 530, 1100])
def test_captured_and_replayed(cuda_device, rows):
    """One captured call, replayed with other lengths, tables and queries; and two graphs that run side by side."""
    lens = [600, 900]
    a = _batch(cuda_device, lens, [rows, 1], 8, 2, 128, 16, E4M3, torch.bfloat16, poison=False)
    _run(a)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(a, max_q=max(rows, 1), max_k=1000))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in (lens, [590, 60], [601, 1]):
        a[6].copy_(_ints(cuda_device, n))
        a[0].normal_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for out, lse in outs:
            _compare(out, lse, a, many=rows > 500)


def test_calls_on_two_streams_at_once(cuda_device):
    calls = [_batch(cuda_device, [3000, 50, 700], [1, r, 2], 16, 4, 128, 32, INT8, torch.float16, seed=r) for r in (1, 3, 4, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    outs = []
    for _ in range(4):
        outs = []
        for s, b in zip(streams, calls):
            with torch.cuda.stream(s):
                outs.append(kv_cache.attention(*b, 4, 3000))
    torch.cuda.synchronize()
    for (out, lse), b in zip(outs, calls):
        _compare(out, lse, b)


def test_refusals(cuda_device):
    q, kc, vc, ks, vs, table, lens, cu = _batch(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, INT8, torch.float16)
    k = torch.zeros(2, 2, 64, device=cuda_device, dtype=torch.float16)
    slots = _ints(cuda_device, [0, 1])
    for args, text in [((q.float(), kc, vc, ks, vs, table, lens), "fp16 or bf16"), ((q, kc.view(torch.uint8), vc.view(torch.uint8), ks, vs, table, lens), "float8_e4m3fn or int8"),
                       ((q, kc, vc[:-1], ks, vs, table, lens), "both be"), ((q, kc, vc, ks.double(), vs, table, lens), "key_scale and value_scale"),
                       ((q, kc, vc, ks, vs, table.long(), lens), "block_table"), ((q, kc, vc, ks, vs, table, lens[:1]), "seq_lens must be"),
                       ((q, kc, vc, ks, vs, table, lens, cu[:2]), "requests \\+ 1"), ((q[:, :3], kc, vc, ks, vs, table, lens), "must divide"),
                       ((q[:1], kc, vc, ks, vs, table, lens), "one row of q per request"), ((q[..., :32], kc, vc, ks, vs, table, lens), "head_dim"),
                       ((q, kc, vc, ks, vs, table, lens, cu, 0, 100), "must be positive"), ((q, kc[..., :32], vc[..., :32], ks, vs, table, lens), "head_dim"),
                       ((q, kc.cpu(), vc.cpu(), ks, vs, table, lens), "device")]:
        with pytest.raises(RuntimeError, match=text):
            kv_cache.attention(*args)
    for args, text in [((k, k[:1], slots, kc, vc, ks, vs), "both be"), ((k, k, slots.long(), kc, vc, ks, vs), "slots must be an int32"),
                       ((k, k, slots[:1], kc, vc, ks, vs), r"slots must be \[tokens\]"), ((k[:, :1], k[:, :1], slots, kc, vc, ks, vs), "heads of key"),
                       ((k, k.bfloat16(), slots, kc, vc, ks, vs), "same dtype")]:
        with pytest.raises(RuntimeError, match=text):
            kv_cache.store(*args)
    with pytest.raises(RuntimeError, match="16, 32, 64 or 128"):
        kv_cache.plan_step(lens, lens, table, slots, _ints(cuda_device, [0, 2, 0]), block_size=24, num_tokens=4)
    with pytest.raises(RuntimeError, match="ring_state"):
        kv_cache.plan_step(lens, lens, table, slots, slots, block_size=16, num_tokens=4)


# ---------------------------------------------------------------------------------------------- all of it together
@pytest.mark.parametrize("code,dtype,block,captured", [(E4M3, torch.bfloat16, 16, False), (INT8, torch.float16, 32, False), (E4M3, torch.bfloat16, 64, True)])
def test_serving_loop(cuda_device, code, dtype, block, captured):
    """Requests come, grow and end over some thirty steps of two layers: prompts, decode steps, padded token counts, dropped tokens, blocks that change hands. Every
    step's codes, scales and results are held to the restatements, on a cache that the restatements keep for themselves."""
    layers, hq, hkv, dim, requests, most = 2, 8, 2, 64, 5, 12
    cache = kv_cache.PagedCache(layers, 40 * 64 // block, hkv, dim, requests, most * 64 // block, block_size=block, dtype=code, device=cuda_device)
    g = torch.Generator().manual_seed(block)
    inv_freq = (1e4 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().to(cuda_device)
    state = [[0] * requests, [list(r) for r in cache.block_table.tolist()], cache.ring.tolist(), cache.ring_state.tolist()]
    mirror = [[(c[i].cpu().float().nan_to_num(0).double(), s[i].cpu().double()) for c, s in ((cache.key_cache, cache.key_scale), (cache.value_cache, cache.value_scale))]
              for i in range(layers)]
    tokens = 150
    q, k, v = (torch.zeros(tokens, h, dim, dtype=dtype, device=cuda_device) for h in (hq, hkv, hkv))
    news = torch.zeros(requests, dtype=torch.int32, device=cuda_device)

    def step():
        plan = cache.step(news, tokens)
        got = []
        for i in range(layers):
            qi, ki, vi = q * (i + 1), k * (i + 1), v * (1 + 0.5 * i)
            out, lse = cache.attend(i, qi, ki, vi, 64, most * 64, inv_freq=inv_freq)
            got.append((qi, ki, vi, out, lse))
        return plan, got

    graph = None
    for it in range(30):
        new = []
        for c in state[0]:
            r = float(torch.rand((), generator=g))
            new.append(int(40 * r * 2) if c == 0 and r < 0.6 else 0 if c == 0 else -c if r < 0.08 or c > 600 else -min(c - 1, 3) if r < 0.2 else 1 if r < 0.9 else 60)
        while sum(max(n, 0) for n in new) > tokens:
            new[max(range(requests), key=lambda i: new[i])] //= 2
        want = orc.plan_step(state[0], new, state[1], state[2], state[3], block, tokens)
        news.copy_(torch.tensor(new, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        k[want[1][-1]:] = math.nan  # behind the last token there may be anything
        v[want[1][-1]:] = math.inf
        if not captured:
            plan, got = step()
        else:
            if graph is None:
                keep = [t.clone() for t in (cache.lens, cache.block_table, cache.ring, cache.ring_state, cache.key_cache, cache.value_cache, cache.key_scale, cache.value_scale)]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                side.synchronize()
                for t, old in zip((cache.lens, cache.block_table, cache.ring, cache.ring_state, cache.key_cache, cache.value_cache, cache.key_scale, cache.value_scale), keep):
                    t.copy_(old)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    plan, got = step()
            graph.replay()
        torch.cuda.synchronize()
        assert [x.tolist() for x in (plan.seq_lens, plan.cu_seqlens, plan.positions, plan.slots, plan.ring_state, cache.block_table, cache.ring)] == list(want), it
        assert cache.refused() == want[4][2]
        state = [want[0], want[5], want[6], want[4]]
        for i, (qi, ki, vi, out, lse) in enumerate(got):
            for which, (x, c, s) in enumerate(((ki, cache.key_cache[i], cache.key_scale[i]), (vi, cache.value_cache[i], cache.value_scale[i]))):
                values, scales = mirror[i][which]
                mirror[i][which] = orc.store(x, plan.slots, values.to(code), scales)
                used = torch.zeros(values.shape[0], values.shape[2], dtype=torch.bool)
                for row, n in zip(state[1], state[0]):
                    for p in range(n):
                        used[row[p // block], p % block] = True
                got_codes = c.cpu().float().double()
                same = (got_codes == mirror[i][which][0]) | (got_codes.isnan() & mirror[i][which][0].isnan())
                assert bool((same | ~used[:, None, :, None]).all()), (it, i, which)
                touched = used.any(1)
                assert torch.equal(s.cpu().double()[touched], mirror[i][which][1][touched])
            live = want[1][-1]
            if live:
                b = (qi[:live], cache.key_cache[i], cache.value_cache[i], cache.key_scale[i], cache.value_scale[i], cache.block_table, plan.seq_lens, plan.cu_seqlens)
                _compare(out[:live], lse[:, :live], b)
    assert ops.device_status() == 0
