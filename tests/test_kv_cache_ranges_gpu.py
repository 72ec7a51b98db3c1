"""The ends of the serving operators' ranges: long lists, the types' largest values, lengths and bounds that do not fit, against the restatements in 64 bits.
Tolerances as in test_kv_cache_gpu.py, from which the helpers come."""
import ctypes
import math

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache_gpu import E4M3, INT8, _batch, _cache, _compare, _ints, _run, _same_cache
from torch_mlu_b200 import _cabi, kv_cache, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,at", [(2048, 700), (16384, 16383)])
def test_one_long_chunk_among_many_requests(cuda_device, requests, at):
    """The chunk has nearly all tiles of the list, more than an equal part of 32 bits for each request."""
    lens, rows = [5 + i % 60 for i in range(requests)], [1] * requests
    lens[at], rows[at] = 20000, 3000
    b = _batch(cuda_device, lens, rows, 16, 8, 64, 128, INT8, torch.bfloat16, poison=False)
    _compare(*_run(b), b)
    assert ops.device_status() == 0


def test_a_list_that_takes_several_launches(cuda_device):
    """Tables so wide that the tiles of all requests at their longest would not be counted in 32 bits."""
    requests, heads, block = 70, 128, 128
    for rows in (1, 2):
        lens = [1 + 37 * i % 300 for i in range(requests)]
        b = list(_batch(cuda_device, lens, [rows] * requests, heads, heads, 64, block, E4M3, torch.bfloat16, poison=False))
        wide = torch.full((requests, 1 << 19), -1, dtype=torch.int32, device=cuda_device)
        wide[:, :b[5].size(1)] = b[5]
        b[5] = wide
        before = _cabi.launch_count()
        out, lse = _run(b) if rows > 1 else kv_cache.attention(*b[:7], max_seqlen_k=max(lens))
        launched = _cabi.launch_count() - before
        b[5] = wide[:, :8]
        _compare(out, lse, b)
        before = _cabi.launch_count()
        again = _run(b) if rows > 1 else kv_cache.attention(*b[:7], max_seqlen_k=max(lens))
        assert launched == 2 * (_cabi.launch_count() - before)
        # which CTAs share a unit differs, and so the order of the sums
        _compare(*again, b)


def _gathers(b, max_q=None, max_k=None, **kw):
    """Whether a call brings keys and values to 16 bits in its workspace, by the size of that (without copies it is one of four, for parts of 8 to 64 rows); and its results."""
    q, kc, vc, ks, vs, table, lens, cu = b
    max_q = max_q or max(1, int((cu[1:] - cu[:-1]).max()))
    max_k = max_k or max(1, int(lens.max()))
    p = _cabi.CacheParams()
    p.k_cache, p.v_cache, p.k_scale, p.v_scale = (x.data_ptr() for x in (kc, vc, ks, vs))
    for x, c in (("k", kc), ("v", vc)):
        for f, stride in zip(("block", "head", "row"), c.stride()):
            setattr(p, f"{x}_{f}_stride", stride)
    p.num_blocks, p.heads_kv, p.block_size, p.head_dim = kc.shape
    p.code, p.dtype = _cabi.CODE_INT8 if kc.dtype == INT8 else _cabi.CODE_E4M3, _cabi.DTYPE_F16 if q.dtype == torch.float16 else _cabi.DTYPE_BF16
    p.q = p.out = p.lse = q.data_ptr()  # (only asked for sizes)
    p.block_table, p.seq_lens, p.cu_seqlens_q = (t.data_ptr() for t in (table, lens, cu))
    p.q_row_stride, p.q_head_stride, _ = p.o_row_stride, p.o_head_stride, _ = q.stride()
    p.table_stride, p.max_blocks, p.batch, p.total_q, p.heads_q = table.stride(0), table.size(1), table.size(0), q.shape[0], q.shape[1]
    p.max_seqlen_q, p.max_seqlen_k, p.is_causal, p.softmax_scale = max_q, max_k, 1, 0.1
    n = ctypes.c_size_t(0)
    assert _cabi.load().sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
    parts = [256 + -(-320 * (2 * rows * (kc.shape[3] + 1) * 4 + 24) // 256) * 256 for rows in (8, 16, 32, 64)]
    return (n.value not in parts, *_run(b, max_q, max_k, **kw))


@pytest.mark.parametrize("code,values", [(E4M3, (63488.0, 64000.0, 65504.0)), (INT8, (65024.0, 65280.0, 65504.0))])
@pytest.mark.parametrize("rows", [2, 1000])
def test_f16_elements_whose_codes_are_65536(cuda_device, rows, code, values):
    """On both paths. The keys' large elements meet queries of 2^-10: a score has 8 to 11 of each. Where they are clamped to 65504 it is off by 2^-11 of that, 2^-11 * 11.4 * 3 for
    the three of a key at most, and a weight by twice as much of itself; a value by 2^-11 of itself; the logsumexp by as much as a score."""
    n, hq, hkv, dim, block = 1300, 64, 8, 128, 64
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    k, v = (torch.randn(n, hkv, dim, generator=g, device=cuda_device).half() for _ in range(2))
    for i, x in enumerate(values):
        k[i::7, :, i] = x * (1 if i % 2 else -1)
        v[i::11, i % hkv, i::5] = x
    kc, ks = _cache(cuda_device, 24, hkv, block, dim, code, 1)
    vc, vs = _cache(cuda_device, 24, hkv, block, dim, code, 2)
    pages = torch.randperm(24, generator=torch.Generator().manual_seed(1))[:-(-n // block)]
    slots = _ints(cuda_device, [int(pages[t // block]) * block + t % block for t in range(n)])
    want = orc.store(k, slots, kc, ks), orc.store(v, slots, vc, vs)
    kv_cache.store(k, v, slots, kc, vc, ks, vs)
    _same_cache(kc, ks, *want[0])
    _same_cache(vc, vs, *want[1])
    for c, scale in ((kc, ks), (vc, vs)):  # (the last block has more than the tokens)
        largest = float((c[pages[:-1]].float() * scale[pages[:-1]][..., None, None]).abs().max())
        assert largest == 65536
    q = torch.randn(rows, hq, dim, generator=g, device=cuda_device).half()
    q[..., :3] = 2.0 ** -10 * q[..., :3].sign()
    b = (q, kc, vc, ks, vs, _ints(cuda_device, [pages.tolist()]), _ints(cuda_device, [n]), _ints(cuda_device, [0, rows]))
    gathers, out, lse = _gathers(b)
    assert gathers == (rows == 1000)
    ref, ref_lse, size, most = orc.attention(*b)
    clamped = gathers * 2.0 ** -11
    score = clamped * 65536 * 2.0 ** -10 * 3 * dim ** -0.5
    # v is up to 65536 in few places, so that the result stays below 65504
    assert float(ref.abs().max()) < 60000 and bool(out.isfinite().all())
    tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 1e-4 + clamped + 2 * score) * size
    assert bool(((out.double() - ref).abs() <= tol).all()), float(((out.double() - ref).abs() - tol).max())
    ltol = 2.0 ** -24 * (n / 128 * 9 + 40) + 2.0 ** -21 * most.clamp_min(1) + 2.0 ** -23 * ref_lse.abs() + score
    assert bool(((lse.double() - ref_lse).abs() <= ltol).all())


def test_f16_queries_over_a_cache_of_bf16_elements(cuda_device):
    """Values beyond f16's range count as 65504 where they are brought to 16 bits, and as they are where they are not; NaN stays what it is."""
    n, dim, block = 1100, 64, 64
    for rows, hq in ((1, 4), (1000, 64)):
        b = list(_batch(cuda_device, [n, 64], [rows, 1], hq, 2, dim, block, E4M3, torch.float16, poison=False))
        b[2] = (torch.ones_like(b[2], dtype=torch.float32) * 256).to(E4M3)
        b[4] = torch.full_like(b[4], 2.0 ** 9)  # 131072 everywhere
        gathers, out, lse = _gathers(b)
        assert gathers == (rows == 1000)
        # 131072 does not fit the result and is +inf. A mean of numbers that are all 65504, with weights rounded to f16, is off by up to (2^-11 + 1e-4) * 65504 = 38.6: 65465 to
        # 65543, of which the nearest f16 numbers are 65472 and, from 65520 on, +inf
        assert bool((out >= (65472 if gathers else math.inf)).all()) and bool(lse.isfinite().all()) and bool(out.isfinite().any()) == gathers
        b[2][int(b[5][0, 3]), 0, 5] = torch.tensor(math.nan, device=cuda_device).to(E4M3)
        out, lse = _run(b)
        assert bool(out[:rows, :hq // 2].isnan().any()) and not bool(out[rows:].isnan().any())


@pytest.mark.parametrize("rows,dim,width,max_k", [(1, 128, 8, None), (1, 64, 16, None), (3, 128, 8, 128), (1, 128, 90, None), (5, 64, 90, 1440), (1100, 128, 90, None), (1100, 64, 90, 1440),
                                                  (1500, 128, 90, None), (1500, 128, 90, 1000)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_request_longer_than_its_table(cuda_device, rows, dim, width, max_k, causal):
    """All of its rows are NaN, on both paths, whatever the bound on lengths, also where the call has no more tiles than requests, or the request more rows than the table tokens;
    the requests beside it are as they would be."""
    lens, each = [90, 60, 100, 128, 70], [2, 1, rows, 1, 3] if rows > 1 else [1] * 5
    hq, hkv = (64, 8) if rows > 500 else (8, 2)
    if width * 16 >= 1300:
        lens = [1000, 60, 700, 900, 1300]
    for length in (width * 16 + 1, 10 ** 9, 2 ** 31 - 1):
        b = list(_batch(cuda_device, lens, each, hq, hkv, dim, 16, E4M3, torch.bfloat16, seed=rows))
        table = torch.full((5, width), -5, dtype=torch.int32, device=cuda_device)
        n = min(width, b[5].size(1))
        table[:, :n] = b[5][:, :n]
        b[5] = table
        lens_given = b[6].clone()
        lens_given[2] = length
        q, kc, vc, ks, vs, _, _, cu = b
        kw = dict(is_causal=causal)
        out, lse = kv_cache.attention(q, kc, vc, ks, vs, table, lens_given, cu, max(each), max_k, **kw) if rows > 1 else kv_cache.attention(q, kc, vc, ks, vs, table, lens_given, max_seqlen_k=max_k, **kw)
        lo, hi = int(cu[2]), int(cu[3])
        assert bool(out[lo:hi].isnan().all()) and bool((lse[:, lo:hi] == math.inf).all())
        out[lo:hi], lse[:, lo:hi] = 0, math.inf  # as of a request without tokens
        b[6] = b[6].clone()
        b[6][2] = 0
        _compare(out, lse, b, causal, many=rows > 500)
    assert ops.device_status() == 0


def test_requests_gathered_in_several_launches(cuda_device):
    """A bound on lengths at which the 16-bit copies of all requests would take 9.7 GB: they are made for a few at a time, and where those of one would take more than 4 GiB not at
    all; rows outside every request stay as they are."""
    lens, rows = [1300, 300, 1, 0, 700, 1500, 1024, 64, 900], [1000, 300, 1, 2, 700, 1, 1024, 40, 900]
    b = _batch(cuda_device, lens, rows, 64, 8, 128, 64, E4M3, torch.bfloat16)
    for bound, many in ((1500, True), (1 << 18, True), ((1 << 20) + 1, False)):
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        gathers, out, lse = _gathers(b, max_k=bound)
        assert gathers == many and torch.cuda.max_memory_allocated() < 9 << 30
        _compare(out, lse, b, many=many)
    # replayed from a graph, on a workspace that is full of NaN
    keep = _run(b, max_k=1500)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = _run(b, max_q=1024, max_k=1 << 18)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    _compare(out, lse, b, many=True)
    assert torch.equal(out[:1000], keep[0][:1000])  # the same tiles, whoever is beside them
    assert ops.device_status() == 0


def _far_apart(b, exponents, block):
    """Scales of V by the place of a block in its request: 2^e for the exponents in turn, None: a block of zeros with the least scale. Scores are of N(0,1) queries and keys."""
    q, kc, vc, ks, vs, table, lens, cu = b
    if kc.dtype == E4M3:  # drawn codes beyond 448 are NaN, which is not what is looked at here
        for c in (kc, vc):
            c.copy_(c.float().nan_to_num(448.0).to(E4M3))
    for i, n in enumerate(lens.tolist()):
        for page in range(-(-n // block)):
            at, e = int(table[i, page]), exponents[page % len(exponents)]
            if e is None:
                vc[at] = torch.zeros((), device=vc.device).to(vc.dtype)
                vs[at] = 2.0 ** -100
            else:
                vs[at] = 2.0 ** e
    return b


def _compare_far(out, lse, b, causal):
    """As _compare; a score carries log2 of V's scale, up to 127, in 32 bits, and so does the running maximum: each off by 2^-18, of the logsumexp (times ln 2) 2^-17 together."""
    want, want_lse, size, most = orc.attention(*b[:7], b[7], causal)
    half = torch.finfo(b[0].dtype).eps / 2
    assert float(most.max()) < 60
    tol = half * want.abs() + (2.0 ** -11 + 1e-4) * size
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), (int((off > tol).sum()), float((off / size.clamp_min(1e-300)).max()))
    ltol = 2.0 ** -24 * (int(b[6].max()) / 128 * 9 + 40) + 2.0 ** -21 * most.clamp_min(1) + 2.0 ** -23 * want_lse.abs() + 2.0 ** -17
    assert bool(((lse.double() - want_lse).abs() <= ltol).all()), float((lse.double() - want_lse).abs().max())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("exponents", [(100,), (119,), (96, 110), (None, 60), (60, None), (None, None, None, 100, -20), (110, None, 0, -90), (-90, -60, 20, 70)])
@pytest.mark.parametrize("lens,rows,hq,hkv,dim", [([300], 1, 8, 2, 64), ([1000, 77, 640], 1, 32, 8, 128), ([700, 65, 900], 3, 16, 4, 64), ([500, 400], 12, 8, 2, 128), ([3000] * 40, 1, 16, 4, 128)])
def test_values_of_the_whole_range_of_bf16(cuda_device, lens, rows, hq, hkv, dim, exponents, code):
    """Values of up to 2^127, beside blocks of zeros and small ones: every key has its weight, whatever the scales of V are."""
    b = list(_batch(cuda_device, lens, [rows] * len(lens), hq, hkv, dim, 16, code, torch.bfloat16, seed=len(lens), poison=False))
    top = 119 if code == E4M3 else 120
    if code == E4M3:  # codes of up to 448
        b[2] = (b[2].float() / 4).to(E4M3)
    else:
        b[2] = b[2] // 4
    b = _far_apart(b, [e if e is None else min(e, top - 2) for e in exponents], 16)
    for causal in (True, False):
        _compare_far(*_run(b, is_causal=causal), b, causal)
        _compare_far(*_run(b, max_k=1 << 20, is_causal=causal), b, causal)  # by shares of the list where clusters would take the units


def test_stored_values_of_the_whole_range_of_bf16(cuda_device):
    """Through the store, whose scales go from 2^-100 to 2^119, and on both paths. (The prefill kernel sums weights times values in 32 bits before it divides by the sum of the
    weights, as for any value: 600 of 2^124 would not fit.)"""
    n, dim, block = 600, 128, 64
    for rows, hq in ((1, 16), (500, 64)):
        g = torch.Generator(device=cuda_device).manual_seed(rows)
        k, v = (torch.randn(n, 8, dim, generator=g, device=cuda_device).bfloat16() for _ in range(2))
        v *= 2.0 ** (122 if rows == 1 else 110)
        v[64:128] = 0
        kc, ks = _cache(cuda_device, 12, 8, block, dim, E4M3, 1)
        vc, vs = _cache(cuda_device, 12, 8, block, dim, E4M3, 2)
        table = _ints(cuda_device, [[3, 1, 4, 7, 5, 9, 2, 6, 11, 0]])
        kv_cache.store(k, v, _ints(cuda_device, [int(table[0, t // block]) * block + t % block for t in range(n)]), kc, vc, ks, vs)
        assert float(vs[1].max()) == 2.0 ** -100 and float(vs[3].max()) >= 2.0 ** (115 if rows == 1 else 103)
        q = torch.randn(rows, hq, dim, generator=g, device=cuda_device).bfloat16()
        b = (q, kc, vc, ks, vs, table, _ints(cuda_device, [n]), _ints(cuda_device, [0, rows]))
        gathers, out, lse = _gathers(b)
        assert gathers == (rows == 500)
        if gathers:
            _compare(out, lse, b, many=True)
        else:
            _compare_far(out, lse, b, True)


@pytest.mark.parametrize("rows,hq", [(1, 16), (500, 64)])
def test_scales_that_no_element_can_have(cuda_device, rows, hq):
    """Infinite ones of K and V, NaN, and negative ones of V: the rows that see their blocks are NaN on both paths, those of other requests as they are."""
    for which, value in ((3, math.inf), (3, -math.inf), (3, math.nan), (4, math.inf), (4, math.nan), (4, -1.0), (4, -math.inf)):
        b = list(_batch(cuda_device, [600, 200], [rows, 1], hq, 8, 128, 64, INT8, torch.bfloat16, poison=False))
        want = _run(b)
        b[which][int(b[5][0, 0])] = value
        gathers, out, lse = _gathers(b)
        assert gathers == (rows == 500)
        assert bool(out[:rows].isnan().all()), (which, value)
        assert which == 4 or bool((lse[:, :rows] == math.inf).all())  # (the logsumexp has no part of V)
        assert torch.equal(out[rows:], want[0][rows:]) and torch.equal(lse[:, rows:], want[1][:, rows:])


def test_plan_of_the_most_tokens(cuda_device):
    """2^30 tokens in a step, the most that are counted: with twice as many the second request is the one that does not fit, however many blocks there are."""
    most, width, blocks = 1 << 30, 1 << 23, (1 << 24) - 1
    table = torch.full((2, width), -1, dtype=torch.int32, device=cuda_device)
    ring = torch.arange(blocks, dtype=torch.int32, device=cuda_device)
    state, none = _ints(cuda_device, [0, blocks, 0]), _ints(cuda_device, [0, 0])
    plan = lambda new: kv_cache.plan_step(none, _ints(cuda_device, new), table, ring, state, block_size=128, num_tokens=most)
    step = plan([most, most])
    assert step.ring_state.tolist() == [0, blocks, -2] and step.seq_lens.tolist() == [0, 0] and step.cu_seqlens.tolist() == [0, 0, 0]
    assert int(step.slots[-1]) == -1 and int(table[0, 0]) == -1
    del step
    step = plan([most - 5, 5])
    assert step.ring_state.tolist() == [width + 1, blocks - width - 1, 0] and step.cu_seqlens.tolist() == [0, most - 5, most]
    assert step.positions[-7:].tolist() == [most - 7, most - 6, 0, 1, 2, 3, 4] and step.slots[-5:].tolist() == [width * 128 + i for i in range(5)]
    assert int(step.slots[most - 6]) == most - 6 and int(table[1, 0]) == width


@pytest.mark.parametrize("rows,bound,dim", [(20, 4, 64), (9, 2, 128), (100, 30, 128)])
def test_more_rows_than_the_bound_says(cuda_device, rows, bound, dim):
    """Those behind the bound may stay unwritten; those in front of it, and other requests, are as they should be."""
    b = _batch(cuda_device, [900, 400, 70], [2, rows, 1], 8, 2, dim, 32, INT8, torch.float16)
    for max_k in (900, 1 << 20):
        out, lse = _run(b, max_q=bound, max_k=max_k)
        whole, whole_lse = _run(b)
        for i in range(2 + bound, 2 + rows):
            out[i], lse[:, i] = whole[i], whole_lse[:, i]
        _compare(out, lse, b)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("rows,hq", [(4, 8), (600, 64)])
def test_nan_among_the_last_drafted_tokens(cuda_device, code, rows, hq):
    """What a key, or a value, that is no number reaches: the rows that see the key; of a value any row of its request; in int8, which marks the block's scale, the same of the
    block's keys and values. Other requests are as they are, and so are the request's other kv heads."""
    for which in (0, 1):
        lens = [640, 500]
        b = list(_batch(cuda_device, lens, [rows, 3], hq, 2 if rows < 100 else 8, 128, 64, code, torch.bfloat16, poison=False))
        if code == E4M3:
            for c in (b[1], b[2]):
                c.copy_(c.float().nan_to_num(448.0).to(E4M3))
        hkv = b[1].shape[1]
        want = _run(b)
        k, v = (torch.randn(2, hkv, 128, device=cuda_device).bfloat16() * 1e-3 for _ in range(2))
        block = int(b[5][0, 9])
        (k, v)[which][1, 0, 7] = math.nan
        kv_cache.store(k, v, _ints(cuda_device, [block * 64 + 62, block * 64 + 63]), *b[1:5])  # the last two tokens of the first request
        out, lse = _run(b)
        group = hq // hkv
        other = slice(group, None)
        assert bool(out[:, other].isfinite().all()) and torch.equal(out[rows:], want[0][rows:]) and torch.equal(lse[:, rows:], want[1][:, rows:])
        assert bool(out[rows - 1, :group].isnan().any())  # the last row sees it
        if which == 0:
            sees = torch.arange(640 - rows, 640, device=cuda_device) >= (639 if code == E4M3 else 576)
            assert bool(out[:rows, :group][sees].isnan().all()) and bool(out[:rows, :group][~sees].isfinite().all())


@pytest.mark.parametrize("rows,hq,hkv", [(3, 8, 2), (40, 16, 2), (1000, 64, 8)])
def test_offsets_that_leave_q(cuda_device, rows, hq, hkv):
    """A step's offsets beside fewer rows of q, or offsets of less than 0: nothing is written outside out and lse, and requests whose rows are all there are as they should be."""
    dim = 64
    b = _batch(cuda_device, [1100, 300, 200, 70], [rows, 2, rows // 2 + 1, 1], hq, hkv, dim, 32, INT8, torch.bfloat16)
    q, kc, vc, ks, vs, table, lens, cu = b
    for shift, total in ((0, int(cu[3]) - 1), (0, int(cu[2])), (-1, int(cu[4])), (-(1 << 30), int(cu[4])), (5, int(cu[4])), (1 << 30, int(cu[4]))):
        given = cu + shift
        guard = 4096
        out_all = torch.full((2 * guard + total * hq * dim,), 7.0, dtype=q.dtype, device=cuda_device)
        lse_all = torch.full((2 * guard + hq * total,), 7.0, device=cuda_device)
        out, lse = out_all[guard:-guard].view(total, hq, dim), lse_all[guard:-guard].view(hq, total)
        p = _cabi.CacheParams()
        p.k_cache, p.v_cache, p.k_scale, p.v_scale = (x.data_ptr() for x in (kc, vc, ks, vs))
        for x, c in (("k", kc), ("v", vc)):
            for f, stride in zip(("block", "head", "row"), c.stride()):
                setattr(p, f"{x}_{f}_stride", stride)
        p.num_blocks, p.heads_kv, p.block_size, p.head_dim = kc.shape
        p.code, p.dtype = _cabi.CODE_INT8, _cabi.DTYPE_BF16
        part = q[:total].contiguous()
        p.q, p.out, p.lse, p.block_table, p.seq_lens, p.cu_seqlens_q = (t.data_ptr() for t in (part, out, lse, table, lens, given))
        p.q_row_stride = p.o_row_stride = hq * dim
        p.q_head_stride = p.o_head_stride = dim
        p.table_stride, p.max_blocks, p.batch, p.total_q, p.heads_q = table.stride(0), table.size(1), 4, total, hq
        p.max_seqlen_q, p.max_seqlen_k, p.is_causal, p.softmax_scale = max(2, rows), 1100, 1, 0.125
        n = ctypes.c_size_t(0)
        lib = _cabi.load()
        assert lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
        ws = torch.full((n.value,), 255, dtype=torch.uint8, device=cuda_device)
        assert lib.sdpa_b200_cache_attention(ctypes.byref(p), ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        for x in (out_all, lse_all):
            assert bool((x[:guard] == 7).all()) and bool((x[-guard:] == 7).all())
        if shift == 0:  # those whose rows are all there
            end = int(cu[2])
            _compare(out[:end], lse[:, :end], (q[:end], kc, vc, ks, vs, table[:2], lens[:2], cu[:3]), many=rows > 500)
    assert ops.device_status() == 0
