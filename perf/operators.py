"""Performance cases of the serving operators: block bookkeeping, the 8-bit paged cache and the attention over it, rotary positions.

A case is a dict of plain values. ``kind`` says which public call it makes:

* ``plan``    block tables, positions and slots of one serving step: ``kv_cache.plan_step``
* ``store``   the step's keys and values into the 8-bit cache: ``kv_cache.store``
* ``attend``  attention of the step's queries over the cache: ``kv_cache.attention``
* ``rotary``  rotary positions on queries and keys: ``rotary.rotary_embedding``, with its gradients where ``train`` is set

Where ``own`` is false the operators are computed in elementary torch operations instead. Keys and values are N(0,1) with channels of their
own size and a few large ones, as projections have them; the cache's scales are powers of two, as ``kv_cache.store`` chooses them.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST_CODE = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXPONENT = -100  # of a scale: that of a block of zeros


def listed():
    return [
        # the next token of a full serving batch: nothing but latency
        dict(name="plan_decode_b64", kind="plan", requests=64, longest=32768, prompts=0, ended=0, block=64, tokens=64, lens_seed=1),
        # a step that takes in prompts (chunks of them) beside 192 decoding requests and gives the blocks of ended ones back
        dict(name="plan_mixed_b256_t16384", kind="plan", requests=256, longest=8192, prompts=40, ended=24, block=16, tokens=16384, lens_seed=2),
        # one token of each of 64 requests into one layer's cache
        dict(name="store_decode_b64", kind="store", requests=64, cached=4096, new=1, heads_q=32, heads_kv=8, head_dim=128, block=64,
             dtype="bf16", code="e4m3", lens_seed=3),
        # four prompts, 8192 tokens together
        dict(name="store_prompts_t8192", kind="store", requests=4, cached=0, new=2048, heads_q=32, heads_kv=8, head_dim=128, block=64,
             dtype="bf16", code="e4m3", lens_seed=4),
        # chunks that begin and end inside small blocks, a small model's heads, int8
        dict(name="store_chunks_d64_int8", kind="store", requests=23, cached=1000, new=111, heads_q=16, heads_kv=4, head_dim=64, block=16,
             dtype="f16", code="int8", lens_seed=5),
        # one interactive request, early in its answer
        dict(name="attend_b1_l1000", kind="attend", requests=1, lo=1000, hi=1000, new=1, heads_q=32, heads_kv=8, head_dim=128, block=64,
             dtype="bf16", code="e4m3", lens_seed=6),
        # a full serving batch whose requests are between 2 K and 32 K tokens long
        dict(name="attend_b64_l2048_32768", kind="attend", requests=64, lo=2048, hi=32768, new=1, heads_q=32, heads_kv=8, head_dim=128,
             block=64, dtype="bf16", code="e4m3", lens_seed=7),
        # four drafted tokens per request are checked at once; a small model in int8
        dict(name="attend_draft4_b16_d64_int8", kind="attend", requests=16, lo=300, hi=9000, new=4, heads_q=16, heads_kv=4, head_dim=64,
             block=16, dtype="f16", code="int8", lens_seed=8),
        # the next 512 tokens of two prompts whose first 7680 are in the cache
        dict(name="attend_chunk512_of_8192", kind="attend", requests=2, lo=8192, hi=8192, new=512, heads_q=32, heads_kv=8, head_dim=128,
             block=64, dtype="bf16", code="e4m3", lens_seed=9),
        # the next token of 64 requests
        dict(name="rotary_decode_b64", kind="rotary", packed=True, batch=1, length=64, heads_q=32, heads_kv=8, head_dim=128, rotary_dim=128,
             axes=1, interleaved=False, train=False, far=32768, dtype="bf16"),
        # a packed prompt of text, images and video: time, height and width
        dict(name="rotary_video_t16384", kind="rotary", packed=True, batch=1, length=16384, heads_q=32, heads_kv=8, head_dim=128,
             rotary_dim=128, axes=3, interleaved=False, train=False, far=100000, dtype="bf16"),
        # the benchmark's training workload: queries and keys as its projections give them, and their gradients
        dict(name="rotary_train_b8_h16_l2048", kind="rotary", packed=False, batch=8, length=2048, heads_q=16, heads_kv=16, head_dim=128,
             rotary_dim=128, axes=1, interleaved=False, train=True, far=0, dtype="bf16"),
    ]


# The largest cost of a drawn case of each kind, in bytes and operations: about that of the largest listed one.
MOST_BYTES = {"plan": 1e6, "store": 6e7, "attend": 2.0e9, "rotary": 5.5e8}
MOST_FLOPS = {"plan": 1e12, "store": 1e12, "attend": 1.3e11, "rotary": 1e12}


def _log_int(rng, lo, hi):
    """An integer between lo and hi, evenly spread over the logarithm: mostly odd ones, some multiples of 64."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.25 and n >= 64:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    while True:
        kind = rng.choice(["plan", "store", "attend", "attend", "attend", "rotary", "rotary"])
        heads_q, heads_kv = rng.choice([(32, 8), (32, 8), (16, 16), (16, 4), (64, 8), (8, 1), (12, 12)])
        seed = rng.randrange(10000)
        block = rng.choice([16, 32, 64, 64, 128])
        cache = dict(heads_q=heads_q, heads_kv=heads_kv, head_dim=rng.choice([128, 128, 64]), block=block, dtype=rng.choice(["bf16", "bf16", "f16"]),
                     code=rng.choice(["e4m3", "e4m3", "int8"]), lens_seed=seed)
        if kind == "plan":
            requests = _log_int(rng, 1, 1024)
            case = dict(kind=kind, requests=requests, longest=_log_int(rng, 256, 32768), prompts=rng.randint(0, requests // 4),
                        ended=rng.randint(0, requests // 4), block=block, tokens=0, lens_seed=seed)
            case["tokens"] = sum(max(0, n) for _, n in _plan_lengths(case)) + rng.choice([0, 0, 5, 200])
            if not 0 < case["tokens"] <= 65536:
                continue
        elif kind == "store":
            case = dict(kind=kind, requests=_log_int(rng, 1, 128), cached=rng.choice([0, 100, 1000, 3000]), new=_log_int(rng, 1, 2048), **cache)
        elif kind == "attend":
            lo = _log_int(rng, 16, 16384)
            new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1024)])
            case = dict(kind=kind, requests=_log_int(rng, 1, 64), lo=max(lo, new), hi=0, new=new, **cache)
            case["hi"] = _log_int(rng, case["lo"], 32768)
        else:
            train = rng.random() < 0.5
            head_dim, rotary_dim = rng.choice([(128, 128), (128, 128), (64, 64), (80, 80), (128, 64), (256, 64), (96, 96)])
            packed = not train or rng.random() < 0.5
            case = dict(kind=kind, packed=packed, batch=1 if packed else _log_int(rng, 1, 16), length=_log_int(rng, 1, 16384), heads_q=heads_q,
                        heads_kv=heads_kv, head_dim=head_dim, rotary_dim=rotary_dim, axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.3,
                        train=train, far=rng.choice([0, 5000, 1000000]), dtype=rng.choice(["bf16", "bf16", "f16"]))
        w = work(case)
        if w["bytes"] <= MOST_BYTES[kind] and w["flops"] <= MOST_FLOPS[kind]:
            return case


# ---- lengths: by the case alone, since the work goes by them
def _plan_lengths(case):
    """(cached, new) of each request: prompts bring many tokens, ended requests give all of theirs back, some decoding ones drop drafted tokens."""
    r = random.Random(case["lens_seed"])
    got = []
    for i in range(case["requests"]):
        n = r.randint(1, case["longest"])
        if i < case["prompts"]:
            got.append((0 if r.random() < 0.5 else n // 2, r.randint(1, min(700, case["longest"]))))
        elif i < case["prompts"] + case["ended"]:
            got.append((n, -n))
        else:
            got.append((n, -min(n - 1, r.randint(1, 5)) if r.random() < 0.05 and case["prompts"] else 1))
    r.shuffle(got)
    return got


def _store_lengths(case):
    """(cached, new) of each request."""
    r = random.Random(case["lens_seed"])
    return [(r.randint(case["cached"] // 2, case["cached"]), case["new"] if case["new"] == 1 else r.randint(max(1, case["new"] * 3 // 4), case["new"] * 5 // 4))
            for _ in range(case["requests"])]


def _attend_lengths(case):
    """(length in the cache, queries) of each request."""
    r = random.Random(case["lens_seed"])
    return [(r.randint(case["lo"], case["hi"]), case["new"] if case["new"] < 9 else r.randint(max(1, case["new"] * 3 // 4), case["new"]) if case["lo"] < case["hi"] else case["new"])
            for _ in range(case["requests"])]


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


def _scale_for(largest, code):
    """The smallest power of two by which values up to `largest` become codes."""
    part, exponent = torch.frexp(largest)
    top, top_exponent = math.frexp(LARGEST_CODE[code])
    return torch.ldexp(torch.ones_like(largest), (exponent - top_exponent + (part > top).int()).clamp_min(LEAST_EXPONENT))


def _codes(x, code):
    """Values in units of the scale, as codes: rounded to the nearest, ties to even."""
    if code == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.to(torch.float8_e4m3fn)


def _filled_cache(gen, blocks, case):
    """Codes [blocks, heads, block, dim] and scales [blocks, heads] of a cache in use."""
    heads, block, dim = case["heads_kv"], case["block"], case["head_dim"]
    codes = torch.empty(blocks, heads, block, dim, dtype=CODES[case["code"]], device="cuda")
    scales = torch.empty(blocks, heads, dtype=torch.float32, device="cuda")
    channels = _channels(gen, heads, dim)
    step = max(1, (1 << 27) // (heads * block * dim))
    for at in range(0, blocks, step):
        x = _randn(gen, torch.bfloat16, min(step, blocks - at), heads, block, dim) * channels[:, None].bfloat16()
        scales[at:at + step] = _scale_for(x.abs().amax((2, 3)).float(), case["code"])
        codes[at:at + step] = _codes(x.float() / scales[at:at + step, :, None, None], case["code"])
    return codes, scales


def _block_table(gen, lens, block, spare):
    """A table of blocks in no order, -1 behind each request's last one, and the free blocks."""
    pages = [_pages(n, block) for n in lens]
    total, width = sum(pages), max(max(pages), 1) + 2
    blocks = total + spare
    order = torch.randperm(blocks, generator=gen, device="cuda").int()
    at = torch.arange(width, device="cuda")[None]
    start = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device="cuda")[:, None]
    mine = at < torch.tensor(pages, device="cuda")[:, None]
    table = torch.where(mine, order[torch.where(mine, start + at, 0)], -1)
    return table.int().contiguous(), order[total:], blocks


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    kind = case["kind"]
    if kind == "plan":
        lens = _plan_lengths(case)
        width = _pages(max(c + max(n, 0) for c, n in lens), case["block"])
        need = sum(max(0, _pages(c + n, case["block"]) - _pages(c, case["block"])) for c, n in lens)
        table, free, blocks = _block_table(gen, [c for c, _ in lens], case["block"], need + 100)
        s["table"] = torch.full((len(lens), max(width, table.shape[1])), -1, dtype=torch.int32, device="cuda")
        s["table"][:, :table.shape[1]] = table
        # the free blocks stand in a ring, somewhere
        first = random.Random(seed).randrange(blocks)
        s["ring"] = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
        s["ring"][(torch.arange(free.numel(), device="cuda") + first) % blocks] = free
        s["ring_state"] = _ints([first, free.numel(), 0])
        s["cached"], s["new_tokens"] = _ints([c for c, _ in lens]), _ints([n for _, n in lens])
    elif kind == "store":
        lens = _store_lengths(case)
        hq, hkv, dim, block = case["heads_q"], case["heads_kv"], case["head_dim"], case["block"]
        table, _, blocks = _block_table(gen, [c + n for c, n in lens], block, 8)
        at = [(i, c + j) for i, (c, n) in enumerate(lens) for j in range(n)]
        row, pos = _ints([a for a, _ in at]).long(), _ints([p for _, p in at]).long()
        s["slots"] = (table[row, pos // block] * block + pos % block).int()
        s["key_cache"], s["key_scale"] = _filled_cache(gen, blocks, case)
        s["value_cache"], s["value_scale"] = _filled_cache(gen, blocks, case)
        # keys and values as one projection writes them: beside the queries of the same token
        qkv = _randn(gen, DTYPES[case["dtype"]], len(at), hq + 2 * hkv, dim)
        qkv[:, hq:] *= _channels(gen, 2 * hkv, dim).to(qkv.dtype)
        s["key"], s["value"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["most_runs"] = sum(_pages(c + n, block) - c // block for c, n in lens)
    elif kind == "attend":
        lens = _attend_lengths(case)
        s["table"], _, blocks = _block_table(gen, [n for n, _ in lens], case["block"], 8)
        s["key_cache"], s["key_scale"] = _filled_cache(gen, blocks, case)
        s["value_cache"], s["value_scale"] = _filled_cache(gen, blocks, case)
        s["seq_lens"] = _ints([n for n, _ in lens])
        ends = [sum(q for _, q in lens[:i]) for i in range(len(lens) + 1)]
        s["cu_seqlens"] = _ints(ends)
        s["max_q"], s["max_k"] = max(q for _, q in lens), max(n for n, _ in lens)
        s["query"] = _randn(gen, DTYPES[case["dtype"]], ends[-1], case["heads_q"], case["head_dim"])
    else:
        dt, b, n, dim, half = DTYPES[case["dtype"]], case["batch"], case["length"], case["head_dim"], case["rotary_dim"] // 2
        theta = 1e6 if case["axes"] > 1 else 1e4
        s["inv_freq"] = (theta ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()
        shapes = [(n, h, dim) if case["packed"] else (b, n, h, dim) for h in (case["heads_q"], case["heads_kv"])]
        made = [_randn(gen, dt, *shape) for shape in (shapes * 2 if case["train"] else shapes)]
        s["made"] = [t if case["packed"] else t.transpose(1, 2) for t in made]
        for t in s["made"][:2]:
            t.requires_grad_(case["train"])
        base = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device="cuda", dtype=torch.int32)
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        if case["packed"] and case["axes"] == 1 and not case["train"]:  # a step of a serving batch: every token at a place of its own
            pos = torch.randint(0, case["far"] + n + 1, (1, n), generator=gen, device="cuda", dtype=torch.int32)
        else:
            pos = base + at
        if case["axes"] == 3:  # frames of 16 x 16 patches behind the text so far
            pos = torch.stack([base + at // 256, base + at // 16 % 16, base + at % 16])
        s["positions"] = (pos[..., 0, :] if case["packed"] else pos).contiguous()
        s["sections"] = _sections(half, case["axes"])
    return s


def _sections(half, axes):
    """How many pairs turn by each axis: a quarter by time, the rest by height and width."""
    if axes == 1:
        return None
    t, h = half // 4, (half - half // 4 + 1) // 2
    return (t, h, half - t - h)


# ---- one pass
def run(s):
    return {"plan": _run_plan, "store": _run_store, "attend": _run_attend, "rotary": _run_rotary}[s["kind"]](s)


def _run_plan(s):
    if own:
        from torch_mlu_b200 import kv_cache
        step = kv_cache.plan_step(s["cached"], s["new_tokens"], s["table"], s["ring"], s["ring_state"], block_size=s["block"], num_tokens=s["tokens"])
        return step.seq_lens, step.cu_seqlens, step.positions, step.slots, step.ring_state, s["table"], s["ring"]
    block, total = s["block"], s["tokens"]
    table, ring, cached, new = s["table"], s["ring"], s["cached"].long(), s["new_tokens"].long()
    requests, width = table.shape
    first, count = s["ring_state"][0].long(), s["ring_state"][1].long()
    lens = cached + new
    had, has = (cached + block - 1) // block, (lens + block - 1) // block
    need, freed = (has - had).clamp_min(0), (had - has).clamp_min(0)
    ends = new.clamp_min(0).cumsum(0)
    # a request that does not fit, or too few blocks: nothing changes but the third word of the state
    bad = (lens < 0) | (has > width) | (ends > total)
    lacking = (need.sum() - count).clamp_min(0)
    refused = torch.where(bad.any(), -1 - bad.int().argmax(), lacking)
    fine = refused == 0
    # new blocks into the table, blocks given back into the ring
    page = torch.arange(width, device=table.device)
    j = page - had[:, None]
    given = ring[(first + (need.cumsum(0) - need)[:, None] + j.clamp_min(0)) % ring.numel()]
    back = page - has[:, None]
    at = (first + count + (freed.cumsum(0) - freed)[:, None] + back.clamp_min(0)) % ring.numel()
    gives = fine & (back >= 0) & (page < had[:, None])
    into = torch.cat([ring, ring[:1]])
    into[torch.where(gives, at, ring.numel())] = table
    table.copy_(torch.where(fine & (j >= 0) & (page < has[:, None]), given, table))
    ring.copy_(into[:-1])
    # each token's place
    t = torch.arange(total, device=table.device)
    row = torch.searchsorted(ends, t, right=True).clamp_max(requests - 1)
    live = fine & (t < ends[-1])
    position = torch.where(live, cached[row] + t - (ends[row] - new[row]), 0)
    slot = table[row, (position // block).clamp_max(width - 1)] * block + position % block
    taken = torch.where(fine, need.sum(), 0)
    state = torch.stack([(first + taken) % ring.numel(), count - taken + torch.where(fine, freed.sum(), 0), refused])
    cu = torch.cat([torch.zeros_like(ends[:1]), torch.where(fine, ends, 0)])
    return (torch.where(fine, lens, cached).int(), cu.int(), position.int(), torch.where(live, slot, -1).int(), state.int(), table, ring)


def _run_store(s):
    if own:
        from torch_mlu_b200 import kv_cache
        kv_cache.store(s["key"], s["value"], s["slots"], s["key_cache"], s["value_cache"], s["key_scale"], s["value_scale"])
    else:
        slots = s["slots"].long()
        block, place = slots // s["block"], slots % s["block"]
        # one token of each block that is written to
        starts = torch.cat([torch.ones_like(block[:1]), (block[1:] != block[:-1]).long()])
        one = torch.nonzero_static(starts, size=s["most_runs"], fill_value=0)[:, 0]
        touched = block[one]
        blocks = s["key_cache"].shape[0]
        earlier = torch.full((blocks,), s["block"], device=slots.device).scatter_reduce(0, block, place, "amin")[touched]
        for x, cache, scale in ((s["key"], s["key_cache"], s["key_scale"]), (s["value"], s["value_cache"], s["value_scale"])):
            largest = torch.zeros_like(scale).index_reduce(0, block, x.abs().amax(-1).float(), "amax")[touched]
            before = scale[touched]
            now = torch.maximum(torch.where(earlier[:, None] > 0, before, 0), _scale_for(largest, s["code"]))
            kept = cache.view(torch.uint8)[touched].view(cache.dtype)
            again = _codes(kept.float() * before[..., None, None] / now[..., None, None], s["code"]).view(torch.uint8)
            old = torch.arange(s["block"], device=slots.device) < earlier[:, None]
            kept = torch.where((old[:, None] & (now > before)[..., None])[..., None], again, kept.view(torch.uint8))
            cache.view(torch.uint8)[touched] = kept
            scale[touched] = now
            codes = _codes(x.float() / scale[block][..., None], s["code"])
            cache.view(torch.uint8)[block, :, place] = codes.view(torch.uint8)
    return s["key_cache"], s["value_cache"], s["key_scale"], s["value_scale"]


def _run_attend(s):
    if own:
        from torch_mlu_b200 import kv_cache
        return kv_cache.attention(s["query"], s["key_cache"], s["value_cache"], s["key_scale"], s["value_scale"], s["table"], s["seq_lens"],
                                  s["cu_seqlens"], s["max_q"], s["max_k"])
    q, cu, lens = s["query"], s["cu_seqlens"].long(), s["seq_lens"].long()
    requests, hkv, block, dim = s["table"].shape[0], s["heads_kv"], s["block"], s["head_dim"]
    group, pages = s["heads_q"] // hkv, _pages(s["max_k"], s["block"])
    blocks = s["table"][:, :pages].long().clamp_min(0)

    def gathered(cache, scale):
        x = cache.view(torch.uint8)[blocks].view(cache.dtype).float() * scale[blocks][..., None, None]
        return x.transpose(1, 2).reshape(requests, hkv, pages * block, dim)

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


def _run_rotary(s):
    q, k = s["made"][:2]
    if own:
        from torch_mlu_b200 import rotary
        q2, k2 = rotary.rotary_embedding(q, k, s["positions"], s["inv_freq"], sections=s["sections"], interleaved=s["interleaved"])
        if not s["train"]:
            return q2, k2
        return q2.detach(), k2.detach(), *torch.autograd.grad((q2, k2), (q, k), s["made"][2:4])
    half = s["rotary_dim"] // 2
    pos = s["positions"].double()
    if s["sections"] is not None:  # the axis of each pair
        axis = torch.arange(len(s["sections"]), device=pos.device).repeat_interleave(torch.tensor(s["sections"], device=pos.device), output_size=half)
        pos = pos[axis].movedim(0, -1)
    else:
        pos = pos[..., None]
    angle = pos * s["inv_freq"].double()
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)  # the same for all heads

    def turned(x, sin):
        y = x.detach().float()
        pair = y[..., :2 * half].unflatten(-1, (half, 2) if s["interleaved"] else (2, half))
        a, b = pair.unbind(-1 if s["interleaved"] else -2)
        pair = torch.stack([a * cos - b * sin, a * sin + b * cos], -1 if s["interleaved"] else -2)
        return torch.cat([pair.flatten(-2), y[..., 2 * half:]], -1).to(x.dtype)

    outs = turned(q, sin), turned(k, sin)
    if s["train"]:
        outs += tuple(turned(g, -sin) for g in s["made"][2:4])
    return outs


# ---- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "plan":
        lens = _plan_lengths(case)
        moved = sum(abs(_pages(c + n, case["block"]) - _pages(c, case["block"])) for c, n in lens)
        touched = sum(c % case["block"] != 0 and n > 0 for c, n in lens)
        return {"bytes": 16 * len(lens) + 8 * moved + 4 * touched + 8 * case["tokens"] + 24, "flops": 0}
    if kind == "store":
        lens = _store_lengths(case)
        tokens, runs = sum(n for _, n in lens), sum(_pages(c + n, case["block"]) - c // case["block"] for c, n in lens)
        # two bytes read and one written per element of keys and values; a scale of each block that is written to, slots
        return {"bytes": 6 * tokens * case["heads_kv"] * case["head_dim"] + 16 * runs * case["heads_kv"] + 4 * tokens, "flops": 0}
    if kind == "attend":
        lens = _attend_lengths(case)
        cached, rows = sum(n for n, _ in lens) * case["heads_kv"], sum(q for _, q in lens) * case["heads_q"]
        pairs = sum(q * (n - q) + q * (q + 1) // 2 for n, q in lens) * case["heads_q"]
        pages = sum(_pages(n, case["block"]) for n, _ in lens)
        return {"bytes": 2 * cached * case["head_dim"] + pages * (8 * case["heads_kv"] + 4) + 4 * rows * case["head_dim"] + 4 * rows,
                "flops": 4 * pairs * case["head_dim"]}
    rows = case["batch"] * case["length"] * (case["heads_q"] + case["heads_kv"])
    return {"bytes": rows * case["head_dim"] * (8 if case["train"] else 4) + 4 * case["batch"] * case["length"] * case["axes"], "flops": 0}


# ---- the definitions in 64 bits
def exact(case, seed):
    return {"plan": lambda s: None, "store": _exact_store, "attend": _exact_attend, "rotary": _exact_rotary}[case["kind"]](prepare(case, seed))


def _nearest(x, code):
    """The code's value nearest to x, which is in units of the scale, in 64 bits: a multiple of the step at its size."""
    if code == "int8":
        return torch.clamp(torch.round(x), -127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.clamp(torch.round(x / step) * step, -448, 448)


def _exact_store(s):
    slots, size, code = s["slots"].tolist(), s["block"], s["code"]
    runs = []
    for t, slot in enumerate(slots):
        if runs and slots[t - 1] // size == slot // size:
            runs[-1][2] = t + 1
        else:
            runs.append([slot // size, t, t + 1])
    if len(runs) > 20000:
        return None
    outs = []
    for x, codes, scales in ((s["key"], s["key_cache"], s["key_scale"]), (s["value"], s["value_cache"], s["value_scale"])):
        values, x = codes.float(), x.double()  # a code's value is exact in 32 bits
        for block, lo, hi in runs:
            place = slots[lo] % size
            most = x[lo:hi].abs().amax((0, 2))
            need = torch.exp2(torch.floor(torch.log2(most.clamp_min(2.0 ** (LEAST_EXPONENT + 10)))) - 10)  # too small, unless at the least
            for _ in range(6):
                need = torch.where(need * LARGEST_CODE[code] < most, need * 2, need)
            old = scales[block].double() * (place > 0)
            now = torch.maximum(old, need)
            if place:
                kept = values[block, :, :place].double()
                values[block, :, :place] = torch.where((now > old)[:, None, None], _nearest(kept * (old / now)[:, None, None], code), kept).float()
            values[block, :, place:place + hi - lo] = _nearest(x[lo:hi].transpose(0, 1) / now[:, None, None], code).float()
            scales[block] = now.float()
        outs.append((values.to(codes.dtype), scales))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]


def _exact_attend(s):
    q, group = s["query"], s["heads_q"] // s["heads_kv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(s["heads_q"], q.shape[0], dtype=torch.float64, device=q.device)
    cu, lens = s["cu_seqlens"].tolist(), s["seq_lens"].tolist()
    for b, n in enumerate(lens):
        blocks = s["table"][b, :_pages(n, s["block"])].long()
        k, v = ((c.view(torch.uint8)[blocks].view(c.dtype).double() * a[blocks].double()[:, :, None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
                for c, a in ((s["key_cache"], s["key_scale"]), (s["value_cache"], s["value_scale"])))
        x = q[cu[b]:cu[b + 1]].double()
        m = x.shape[0]
        for h in range(s["heads_kv"]):
            for lo in range(0, m, 64):
                rows = x[lo:lo + 64, h * group:(h + 1) * group]
                logits = torch.einsum("mgd,nd->gmn", rows, k[h]) / math.sqrt(s["head_dim"])
                hidden = torch.arange(n, device=q.device)[None] > torch.arange(lo, min(m, lo + 64), device=q.device)[:, None] + n - m
                logits[:, hidden] = -math.inf
                out[cu[b] + lo:cu[b] + lo + rows.shape[0], h * group:(h + 1) * group] = torch.einsum("gmn,nd->mgd", torch.softmax(logits, -1), v[h])
                lse[h * group:(h + 1) * group, cu[b] + lo:cu[b] + lo + rows.shape[0]] = torch.logsumexp(logits, -1)
    return out, lse


def _exact_rotary(s):
    half, pos = s["rotary_dim"] // 2, s["positions"].double()
    parts = s["sections"] or (half,)
    pos = pos if s["sections"] is not None else pos[None]
    at, angles = 0, []
    for a, n in enumerate(parts):
        angles.append(pos[a][..., None] * s["inv_freq"][at:at + n].double())
        at += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=pos.device), torch.cat(angles, -1)).unsqueeze(1)

    def turned(x, turn):
        x = x.detach().double()
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        z = torch.complex(head[..., 0::2], head[..., 1::2]) if s["interleaved"] else torch.complex(head[..., :half], head[..., half:])
        z = z * turn
        head = torch.view_as_real(z).flatten(-2) if s["interleaved"] else torch.cat([z.real, z.imag], -1)
        return torch.cat([head, rest], -1)

    outs = [turned(x, turn) for x in s["made"][:2]] + [turned(x, turn.conj()) for x in s["made"][2:4]]
    return tuple(outs)
