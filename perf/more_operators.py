"""Performance cases of the 4-bit paged cache: writing it, attention over it, and reading caches of 4 and 8 bits back.

A case is a dict of plain values. ``kind`` says which public call it makes:

* ``store``   a step's keys and values into the 4-bit cache: ``kv_cache.store``
* ``attend``  attention of a step's queries over the 4-bit cache: ``kv_cache.attention``
* ``load``    stretches of requests out of a cache as packed 16-bit keys and values: ``kv_cache.load``

A 4-bit cache holds whole numbers from -8 to 7, two in a byte, the even element in the low half, and a bf16 scale for every 32 elements of a token and head;
an element is its number times its scale. ``kv_cache.store`` takes the smallest scale of five significant bits, 2^-100 at least, at which the largest of the 32
elements is no more than 7, and rounds to the nearest number, ties to even.

Where ``own`` is false the operators are computed in elementary torch operations instead. Keys and values are N(0,1) with channels of their own size and a few
large ones, as projections have them. Codes are compared as the bytes that hold them: they have to be equal.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
BITS = {"int4": 4, "e4m3": 8, "int8": 8}
LARGEST = {"int4": 7.0, "e4m3": 448.0, "int8": 127.0}
GROUP = 32  # elements that share a scale in a 4-bit cache
LEAST_EXPONENT = -100  # of a scale: that of zeros


def listed():
    return [
        # one token of each of 64 requests into one layer's cache: nothing but latency
        dict(name="store4_decode_b64", kind="store", requests=64, cached=4096, new=1, heads_q=32, heads_kv=8, head_dim=128, block=64, dtype="bf16",
             lens_seed=1),
        # four prompts, 8192 tokens together
        dict(name="store4_prompts_t8192", kind="store", requests=4, cached=0, new=2048, heads_q=32, heads_kv=8, head_dim=128, block=64, dtype="bf16",
             lens_seed=2),
        # chunks that begin and end inside small blocks, a small model's heads
        dict(name="store4_chunks_d64_f16", kind="store", requests=23, cached=1000, new=111, heads_q=16, heads_kv=4, head_dim=64, block=16, dtype="f16",
             lens_seed=3),
        # one interactive request, early in its answer
        dict(name="attend4_b1_l1000", kind="attend", requests=1, lo=1000, hi=1000, new=1, heads_q=32, heads_kv=8, head_dim=128, block=64, dtype="bf16",
             lens_seed=4),
        # eight long requests
        dict(name="attend4_b8_l32768", kind="attend", requests=8, lo=32768, hi=32768, new=1, heads_q=32, heads_kv=8, head_dim=128, block=128, dtype="bf16",
             lens_seed=5),
        # a full serving batch whose requests are between 2 K and 32 K tokens long
        dict(name="attend4_b64_l2048_32768", kind="attend", requests=64, lo=2048, hi=32768, new=1, heads_q=32, heads_kv=8, head_dim=128, block=64,
             dtype="bf16", lens_seed=6),
        # four drafted tokens per request are checked at once, in a small model
        dict(name="attend4_draft4_b16_d64", kind="attend", requests=16, lo=300, hi=9000, new=4, heads_q=16, heads_kv=4, head_dim=64, block=16, dtype="f16",
             lens_seed=7),
        # the next 512 tokens of two prompts whose first 7680 are in the cache
        dict(name="attend4_chunk512_of_8192", kind="attend", requests=2, lo=8192, hi=8192, new=512, heads_q=32, heads_kv=8, head_dim=128, block=64,
             dtype="bf16", lens_seed=8),
        # a short prefix that requests share, for a model's dense attention
        dict(name="load4_b1_l301", kind="load", requests=1, lo=301, hi=301, first=0, spare=0, heads_kv=8, head_dim=128, block=64, dtype="bf16", code="int4",
             lens_seed=9),
        # what the requests of a batch have in the cache, for another machine or for a gradient
        dict(name="load4_b16_l8192", kind="load", requests=16, lo=4096, hi=8192, first=0, spare=100, heads_kv=8, head_dim=128, block=64, dtype="bf16",
             code="int4", lens_seed=10),
        # stretches that begin inside small blocks, a small model's heads
        dict(name="load8_b23_d64_f16_int8", kind="load", requests=23, lo=1, hi=1500, first=1000, spare=7, heads_kv=4, head_dim=64, block=16, dtype="f16",
             code="int8", lens_seed=11),
        dict(name="load8_b8_l8192_e4m3", kind="load", requests=8, lo=8192, hi=8192, first=0, spare=0, heads_kv=8, head_dim=128, block=64, dtype="bf16",
             code="e4m3", lens_seed=12),
    ]


# The largest cost of a drawn case of each kind, in bytes and operations: about that of the largest listed one.
MOST_BYTES = {"store": 4.2e7, "attend": 1.1e9, "load": 5.0e8}
MOST_FLOPS = {"store": 1e12, "attend": 1.3e11, "load": 1e12}


def _log_int(rng, lo, hi):
    """An integer between lo and hi, evenly spread over the logarithm: mostly odd ones, some multiples of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.25 and n >= 64:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    while True:
        kind = rng.choice(["store", "attend", "attend", "attend", "load", "load"])
        heads_q, heads_kv = rng.choice([(32, 8), (32, 8), (16, 16), (16, 4), (64, 8), (8, 1), (12, 12)])
        cache = dict(heads_kv=heads_kv, head_dim=rng.choice([128, 128, 64]), block=rng.choice([16, 32, 64, 64, 128]), dtype=rng.choice(["bf16", "bf16", "f16"]),
                     lens_seed=rng.randrange(10000))
        if kind == "store":
            case = dict(kind=kind, requests=_log_int(rng, 1, 128), cached=rng.choice([0, 100, 1000, 3000]), new=_log_int(rng, 1, 2048), heads_q=heads_q, **cache)
        elif kind == "attend":
            lo = _log_int(rng, 16, 16384)
            new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1024)])
            case = dict(kind=kind, requests=_log_int(rng, 1, 64), lo=max(lo, new), hi=0, new=new, heads_q=heads_q, **cache)
            case["hi"] = _log_int(rng, case["lo"], 32768)
        else:
            lo = _log_int(rng, 1, 8192)
            case = dict(kind=kind, requests=_log_int(rng, 1, 64), lo=lo, hi=_log_int(rng, lo, 16384), first=rng.choice([0, 0, 100, 4000]),
                        spare=rng.choice([0, 0, 1, 500]), code=rng.choice(["int4", "int4", "e4m3", "int8"]), **cache)
        w = work(case)
        if w["bytes"] <= MOST_BYTES[kind] and w["flops"] <= MOST_FLOPS[kind]:
            return case


# ---- lengths: by the case alone, since the work goes by them
def _store_lengths(case):
    """(cached, new) of each request."""
    r = random.Random(case["lens_seed"])
    return [(r.randint(case["cached"] // 2, case["cached"]), case["new"] if case["new"] == 1 else r.randint(max(1, case["new"] * 3 // 4), case["new"] * 5 // 4))
            for _ in range(case["requests"])]


def _attend_lengths(case):
    """(length in the cache, queries) of each request."""
    r = random.Random(case["lens_seed"])
    return [(r.randint(case["lo"], case["hi"]), case["new"] if case["new"] < 9 or case["lo"] == case["hi"] else r.randint(max(1, case["new"] * 3 // 4), case["new"]))
            for _ in range(case["requests"])]


def _load_lengths(case):
    """(first token, tokens) of each request; one in eight of a larger batch gives none."""
    r = random.Random(case["lens_seed"])
    got = [(r.randint(0, case["first"]), r.randint(case["lo"], case["hi"])) for _ in range(case["requests"])]
    return [(a, 0 if i % 8 == 5 else n) for i, (a, n) in enumerate(got)]


def _pages(n, block):
    return -(-n // block)


# ---- inputs
def _randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _channels(gen, heads, dim):
    """Sizes of the channels of keys or values: within a factor of two of one, and one in sixteen eight times as large."""
    size = torch.exp2(torch.rand(heads, dim, generator=gen, device="cuda") * 2 - 1)
    return torch.where(torch.rand(heads, dim, generator=gen, device="cuda") < 1 / 16, size * 8, size)


def _five_bits_up(x):
    """The smallest number of five significant bits that is no smaller than x, 2^LEAST_EXPONENT at least."""
    part, exponent = torch.frexp(x.clamp_min(2.0 ** LEAST_EXPONENT))
    return torch.ldexp(torch.ceil(part * 32) / 32, exponent)


def _scales4(x):
    """Scales [..., dim / 32] of x [..., dim], in 64 bits."""
    largest = x.abs().unflatten(-1, (-1, GROUP)).amax(-1).double()
    return _five_bits_up(largest / torch.full_like(largest[..., :1], LARGEST["int4"]))


def _bytes4(x, scale):
    """The codes of x [..., dim], two in a byte."""
    codes = (x.float().unflatten(-1, (-1, GROUP)) / scale.float()[..., None]).round().to(torch.int8).flatten(-2).view(torch.uint8) & 15
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _numbers4(codes):
    """The whole numbers that bytes [..., dim / 2] hold: [..., dim] int8."""
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return (both ^ 8).view(torch.int8) - 8


def _filled_cache(gen, blocks, case, code):
    """Codes and scales of a cache in use."""
    heads, block, dim = case["heads_kv"], case["block"], case["head_dim"]
    four = code == "int4"
    dtype = {"int4": torch.uint8, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[code]
    codes = torch.empty(blocks, heads, block, dim // 2 if four else dim, dtype=dtype, device="cuda")
    scales = torch.empty((blocks, heads, block, dim // GROUP) if four else (blocks, heads), dtype=torch.bfloat16 if four else torch.float32, device="cuda")
    channels = _channels(gen, heads, dim)
    step = max(1, (1 << 26) // (heads * block * dim))
    for at in range(0, blocks, step):
        x = _randn(gen, torch.bfloat16, min(step, blocks - at), heads, block, dim) * channels[:, None].bfloat16()
        if four:
            scale = _scales4(x)
            scales[at:at + step] = scale
            codes[at:at + step] = _bytes4(x, scale)
            continue
        part, exponent = torch.frexp(x.abs().amax((2, 3)).float())
        top, top_exponent = math.frexp(LARGEST[code])
        scale = torch.ldexp(torch.ones_like(part), exponent - top_exponent + (part > top).int())
        x = x.float() / scale[:, :, None, None]
        scales[at:at + step] = scale
        codes[at:at + step] = x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)
    return codes, scales


def _block_table(gen, lens, block, spare):
    """A table of blocks in no order, -1 behind each request's last one, and the number of blocks."""
    pages = [_pages(n, block) for n in lens]
    total, width = sum(pages), max(max(pages), 1) + 2
    order = torch.randperm(total + spare, generator=gen, device="cuda").int()
    at = torch.arange(width, device="cuda")[None]
    start = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device="cuda")[:, None]
    mine = at < torch.tensor(pages, device="cuda")[:, None]
    return torch.where(mine, order[torch.where(mine, start + at, 0)], -1).int().contiguous(), total + spare


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    kind, block, dim, hkv = case["kind"], case["block"], case["head_dim"], case["heads_kv"]
    code = case.get("code", "int4")
    if kind == "store":
        lens = _store_lengths(case)
        hq = case["heads_q"]
        table, blocks = _block_table(gen, [c + n for c, n in lens], block, 8)
        at = [(i, c + j) for i, (c, n) in enumerate(lens) for j in range(n)]
        row, pos = _ints([a for a, _ in at]).long(), _ints([p for _, p in at]).long()
        s["slots"] = (table[row, pos // block] * block + pos % block).int()
        # keys and values as one projection writes them: beside the queries of the same token
        qkv = _randn(gen, DTYPES[case["dtype"]], len(at), hq + 2 * hkv, dim)
        qkv[:, hq:] *= _channels(gen, 2 * hkv, dim).to(qkv.dtype)
        s["key"], s["value"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    elif kind == "attend":
        lens = _attend_lengths(case)
        s["table"], blocks = _block_table(gen, [n for n, _ in lens], block, 8)
        s["seq_lens"] = _ints([n for n, _ in lens])
        ends = [sum(q for _, q in lens[:i]) for i in range(len(lens) + 1)]
        s["cu_seqlens"] = _ints(ends)
        s["max_q"], s["max_k"] = max(q for _, q in lens), max(n for n, _ in lens)
        s["query"] = _randn(gen, DTYPES[case["dtype"]], ends[-1], case["heads_q"], dim)
    else:
        lens = _load_lengths(case)
        s["table"], blocks = _block_table(gen, [a + n for a, n in lens], block, 8)
        ends = [sum(n for _, n in lens[:i]) for i in range(len(lens) + 1)]
        s["cu_seqlens"], s["firsts"] = _ints(ends), _ints([a for a, _ in lens])
        s["tokens"] = ends[-1] + case["spare"]
    s["key_cache"], s["key_scale"] = _filled_cache(gen, blocks, case, code)
    s["value_cache"], s["value_scale"] = _filled_cache(gen, blocks, case, code)
    return s


# ---- one pass
def run(s):
    return {"store": _run_store, "attend": _run_attend, "load": _run_load}[s["kind"]](s)


def _caches(s):
    return s["key_cache"], s["value_cache"], s["key_scale"], s["value_scale"]


def _run_store(s):
    if own:
        from torch_mlu_b200 import kv_cache
        kv_cache.store(s["key"], s["value"], s["slots"], *_caches(s))
        return _caches(s)
    slots = s["slots"].long()
    at = slots // s["block"], slice(None), slots % s["block"]
    for x, codes, scales in ((s["key"], s["key_cache"], s["key_scale"]), (s["value"], s["value_cache"], s["value_scale"])):
        scale = _scales4(x)
        scales[at] = scale.to(scales.dtype)
        codes[at] = _bytes4(x, scale)
    return _caches(s)


def _run_attend(s):
    if own:
        from torch_mlu_b200 import kv_cache
        return kv_cache.attention(s["query"], *_caches(s), s["table"], s["seq_lens"], s["cu_seqlens"], s["max_q"], s["max_k"])
    q, cu, lens = s["query"], s["cu_seqlens"].long(), s["seq_lens"].long()
    requests, hkv, block, dim = s["table"].shape[0], s["heads_kv"], s["block"], s["head_dim"]
    group, pages = s["heads_q"] // hkv, _pages(s["max_k"], s["block"])
    blocks = s["table"][:, :pages].long().clamp_min(0)

    def gathered(codes, scale):
        x = _numbers4(codes[blocks]).unflatten(-1, (-1, GROUP)) * scale[blocks].float()[..., None]
        return x.flatten(-2).transpose(1, 2).reshape(requests, hkv, pages * block, dim)

    i, j = torch.arange(s["max_q"], device=q.device), torch.arange(pages * block, device=q.device)
    count = cu[1:] - cu[:-1]
    rows = q[(cu[:-1, None] + i).clamp_max(q.shape[0] - 1)].float()
    rows = rows.view(requests, s["max_q"], hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(requests, hkv, group * s["max_q"], dim)
    scores = (rows @ gathered(s["key_cache"], s["key_scale"]).transpose(2, 3)) * dim ** -0.5
    seen = j <= (i[:, None] + (lens - count)[:, None, None])
    scores = scores.view(requests, hkv, group, s["max_q"], -1).masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = (weights / total).view(requests, hkv, group * s["max_q"], -1) @ gathered(s["value_cache"], s["value_scale"])
    lse = (top + total.log())[..., 0]
    t = torch.arange(q.shape[0], device=q.device)
    row = torch.searchsorted(cu[1:], t, right=True)
    out = out.view(requests, hkv * group, s["max_q"], dim)[row, :, t - cu[row]]
    return out.to(q.dtype), lse.view(requests, hkv * group, s["max_q"])[row, :, t - cu[row]].t().contiguous()


def _run_load(s):
    dtype = DTYPES[s["dtype"]]
    if own:
        from torch_mlu_b200 import kv_cache
        return kv_cache.load(*_caches(s), s["table"], s["cu_seqlens"], s["tokens"], s["firsts"], dtype=dtype)
    cu = s["cu_seqlens"].long()
    t = torch.arange(s["tokens"], device=cu.device)
    live = t < cu[-1]
    row = torch.searchsorted(cu[1:], t, right=True).clamp_max(cu.numel() - 2)
    position = torch.where(live, s["firsts"][row] + t - cu[row], 0)
    block, place = s["table"][row, position // s["block"]].long().clamp_min(0), position % s["block"]
    outs = []
    for codes, scale in ((s["key_cache"], s["key_scale"]), (s["value_cache"], s["value_scale"])):
        x = codes.view(torch.uint8)[block, :, place]
        if s["code"] == "int4":
            x = (_numbers4(x).unflatten(-1, (-1, GROUP)) * scale[block, :, place].float()[..., None]).flatten(-2)
        else:
            x = x.view(codes.dtype).float() * scale[block][..., None]
        outs.append(torch.where(live[:, None, None], x, 0).to(dtype))
    return tuple(outs)


# ---- what a pass cannot do without
def _token_bytes(case, code):
    """Of a token's keys and values in the cache: codes, and the scales of 4-bit ones."""
    elements = 2 * case["heads_kv"] * case["head_dim"]
    return elements * BITS[code] // 8 + (elements // GROUP * 2 if code == "int4" else 0)


def work(case):
    kind, code = case["kind"], case.get("code", "int4")
    if kind == "store":
        tokens = sum(n for _, n in _store_lengths(case))
        return {"bytes": tokens * (4 * case["heads_kv"] * case["head_dim"] + _token_bytes(case, code) + 4), "flops": 0}
    if kind == "attend":
        lens = _attend_lengths(case)
        rows = sum(q for _, q in lens) * case["heads_q"]
        pairs = sum(q * (n - q) + q * (q + 1) // 2 for n, q in lens) * case["heads_q"]
        return {"bytes": sum(n * _token_bytes(case, code) + 4 * _pages(n, case["block"]) for n, _ in lens) + 4 * rows * case["head_dim"] + 4 * rows,
                "flops": 4 * pairs * case["head_dim"]}
    lens = _load_lengths(case)
    tokens, pages = sum(n for _, n in lens), sum(_pages(a + n, case["block"]) - a // case["block"] for a, n in lens)
    scales = 0 if code == "int4" else 8 * case["heads_kv"] * pages
    return {"bytes": tokens * _token_bytes(case, code) + scales + 4 * pages + 4 * (tokens + case["spare"]) * case["heads_kv"] * case["head_dim"], "flops": 0}


# ---- the definitions in 64 bits
def exact(case, seed):
    return {"store": _exact_store, "attend": _exact_attend, "load": _exact_load}[case["kind"]](prepare(case, seed))


def _exact_store(s):
    numbers = torch.arange(-7, 8, device="cuda", dtype=torch.float64)
    outs = []
    for x, codes, scales in ((s["key"], s["key_cache"], s["key_scale"]), (s["value"], s["value_cache"], s["value_scale"])):
        for lo in range(0, x.shape[0], 256):
            part, slots = x[lo:lo + 256].double(), s["slots"][lo:lo + 256].long()
            part = part.reshape(*part.shape[:2], -1, GROUP)
            # five significant bits: m * 2^e with m from 16 to 31; 7 of them hold the largest element
            largest = part.abs().amax(-1)
            unit = torch.exp2(torch.floor(torch.log2((largest / 7).clamp_min(2.0 ** LEAST_EXPONENT))) - 5)
            scale = torch.full_like(largest, math.inf)
            for m in list(range(64, 31, -2)) + list(range(31, 15, -1)):  # of twice the unit, of the unit: the logarithm may be off by one
                fits = 7 * m * unit >= largest
                scale = torch.where(fits & (m * unit >= 2.0 ** LEAST_EXPONENT), m * unit, scale)
            # the nearest number, the even one of two as near
            off = (part[..., None] - numbers * scale[..., None, None]).abs() / scale[..., None, None] + (numbers % 2) * 2.0 ** -40
            number = off.argmin(-1) - 7
            number = number.reshape(*number.shape[:2], -1) % 16
            block, place = slots // s["block"], slots % s["block"]
            codes[block, :, place] = (number[..., 0::2] + 16 * number[..., 1::2]).to(torch.uint8)
            scales[block, :, place] = scale.to(scales.dtype)
        outs.append((codes, scales))
    return outs[0][0], outs[1][0], outs[0][1].double(), outs[1][1].double()


def _elements(codes, scale, code, block, place):
    """Tokens `place` of blocks `block`, [tokens, heads, dim] in 64 bits."""
    x = codes.view(torch.uint8)[block, :, place]
    if code != "int4":
        return x.view(codes.dtype).double() * scale[block].double()[..., None]
    low, high = x.long() % 16, x.long() // 16
    x = torch.empty(*x.shape[:2], 2 * x.shape[2], dtype=torch.float64, device=x.device)
    x[..., 0::2], x[..., 1::2] = torch.where(low > 7, low - 16, low).double(), torch.where(high > 7, high - 16, high).double()
    return x * scale[block, :, place].double().repeat_interleave(GROUP, -1)


def _exact_attend(s):
    q, group = s["query"], s["heads_q"] // s["heads_kv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(s["heads_q"], q.shape[0], dtype=torch.float64, device=q.device)
    cu, lens = s["cu_seqlens"].tolist(), s["seq_lens"].tolist()
    for b, n in enumerate(lens):
        at = torch.arange(n, device=q.device)
        block, place = s["table"][b, at // s["block"]].long(), at % s["block"]
        k, v = (_elements(c, a, "int4", block, place) for c, a in ((s["key_cache"], s["key_scale"]), (s["value_cache"], s["value_scale"])))
        x = q[cu[b]:cu[b + 1]].double()
        m = x.shape[0]
        for h in range(s["heads_kv"]):
            for lo in range(0, m, 64):
                rows = x[lo:lo + 64, h * group:(h + 1) * group]
                logits = torch.einsum("mgd,nd->gmn", rows, k[:, h]) / math.sqrt(s["head_dim"])
                logits[:, at[None] > torch.arange(lo, min(m, lo + 64), device=q.device)[:, None] + n - m] = -math.inf
                out[cu[b] + lo:cu[b] + lo + rows.shape[0], h * group:(h + 1) * group] = torch.einsum("gmn,nd->mgd", torch.softmax(logits, -1), v[:, h])
                lse[h * group:(h + 1) * group, cu[b] + lo:cu[b] + lo + rows.shape[0]] = torch.logsumexp(logits, -1)
    return out, lse


def _exact_load(s):
    outs = [torch.zeros(s["tokens"], s["heads_kv"], s["head_dim"], dtype=torch.float64, device="cuda") for _ in range(2)]
    cu, firsts = s["cu_seqlens"].tolist(), s["firsts"].tolist()
    for b, first in enumerate(firsts):
        at = torch.arange(first, first + cu[b + 1] - cu[b], device="cuda")
        block, place = s["table"][b, at // s["block"]].long(), at % s["block"]
        for x, codes, scale in zip(outs, (s["key_cache"], s["value_cache"]), (s["key_scale"], s["value_scale"])):
            x[cu[b]:cu[b + 1]] = _elements(codes, scale, s["code"], block, place)
    return tuple(outs)
