"""Plain restatements, in 64 bits and request by request, of the serving operators: bookkeeping of a step, the 8-bit paged cache, attention over it,
rotary positions. Test infrastructure only."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def plan_step(cached, new, table, ring, state, block_size, num_tokens):
    """(seq_lens, cu_seqlens, positions, slots, state, table, ring) as lists; the arguments are lists, left as they are."""
    table, ring = [list(r) for r in table], list(ring)
    pages = lambda n: -(-n // block_size)
    first, count, _ = state
    tokens = refused = need = 0
    for i, (c, n) in enumerate(zip(cached, new)):
        tokens += max(n, 0)
        if c + n < 0 or pages(c + n) > len(table[i]) or tokens > num_tokens:
            refused = -1 - i
            break
        need += max(0, pages(c + n) - pages(c))
    if refused == 0 and need > count:
        refused = need - count
    if refused:
        return list(cached), [0] * (len(cached) + 1), [0] * num_tokens, [-1] * num_tokens, [first, count, refused], table, ring
    at, end = first, first + count
    lens, cu, positions, slots, taken, freed = [], [0], [], [], 0, 0
    old = list(ring)
    for i, (c, n) in enumerate(zip(cached, new)):
        for page in range(pages(c), pages(c + n)):
            table[i][page] = old[at % len(ring)]
            at, taken = at + 1, taken + 1
        for page in range(pages(c + n), pages(c)):
            ring[end % len(ring)] = table[i][page]
            end, freed = end + 1, freed + 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[i][p // block_size] * block_size + p % block_size)
        lens.append(c + n)
        cu.append(len(positions))
    rest = num_tokens - len(positions)
    return lens, cu, positions + [0] * rest, slots + [-1] * rest, [at % len(ring), count - taken + freed, 0], table, ring


def scale_for(largest, dtype):
    """The smallest power of two, at least 2^-100, at which `largest` is a code."""
    scale = 2.0 ** -100
    while scale * LARGEST[dtype] < largest:
        scale *= 2
    return scale


def nearest(x, dtype):
    """The nearest values that codes have, ties to even, of x in units of the scale (fp64)."""
    if dtype == torch.int8:
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.where(x.isfinite(), (torch.round(x / step) * step).clamp(-448, 448), torch.full_like(x, math.nan))


def store(x, slots, codes, scales):
    """(values [blocks, heads, block, dim] in units of the scale, scales), fp64, after tokens x [tokens, heads, dim] went to `slots`."""
    dtype, size = codes.dtype, codes.shape[2]
    values, scales, x = codes.cpu().float().double(), scales.cpu().double().clone(), x.cpu().double()
    placed = [t for t, slot in enumerate(slots.tolist()) if 0 <= slot < codes.shape[0] * size]
    slots, x = slots[placed].tolist(), x[placed]
    t = 0
    while t < len(slots):
        block, end = slots[t] // size, t + 1
        while end < len(slots) and slots[end] // size == block:
            end += 1
        place = slots[t] % size
        for h in range(codes.shape[1]):
            part = x[t:end, h]
            finite = part[part.isfinite()].abs()
            need = scale_for(float(finite.max()) if finite.numel() else 0.0, dtype)
            old = float(scales[block, h])
            now = need
            if place > 0:
                now = old if math.isnan(old) or old >= need else need
                if now != old and not math.isnan(old):
                    values[block, h, :place] = nearest(values[block, h, :place] * old / now, dtype)
            if dtype == torch.int8 and not bool(part.isfinite().all()):
                now = math.nan
            scales[block, h] = now
            for i in range(t, end):
                values[block, h, slots[i] % size] = nearest(x[i, h] / now, dtype) if not math.isnan(now) else 0.0
        t = end
    return values, scales


def attention(q, key_cache, value_cache, key_scale, value_scale, table, seq_lens, cu, causal=True, scale=None):
    """(out [tokens, heads, dim], lse [heads, tokens], mean |v| by the weights [tokens, heads, dim], largest |score| [heads, tokens]) in 64 bits; NaN where nothing is written."""
    T, Hq, D = q.shape
    H, S = key_cache.shape[1], key_cache.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    size = out.clone()
    lse = torch.full((Hq, T), math.nan, dtype=torch.float64, device=q.device)
    most = torch.zeros_like(lse)
    for b, n in enumerate(seq_lens.tolist()):
        lo, hi = (int(cu[b]), int(cu[b + 1])) if cu is not None else (b, b + 1)
        if lo == hi:
            continue
        ids = table[b, :-(-n // S)].long()
        bad = (ids < 0) | (ids >= key_cache.shape[0])
        ids = torch.where(bad, 0, ids)
        # a block outside the cache: its scores are NaN, its values 0
        whole = lambda c, s, spoilt: torch.where(bad[:, None, None, None], spoilt, c.view(torch.uint8)[ids].view(c.dtype).double() * s[ids].double()[:, :, None, None]
                                                 ).permute(1, 0, 2, 3).reshape(H, -1, D)[:, :n]
        k, v = whole(key_cache, key_scale, math.nan), whole(value_cache, value_scale, 0.0)
        rows = q[lo:hi].double().permute(1, 0, 2).reshape(H, Hq // H, hi - lo, D)
        s = torch.einsum("hgmd,hnd->hgmn", rows, k) * scale
        seen = torch.ones(hi - lo, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(n, device=q.device)[None] <= torch.arange(hi - lo, device=q.device)[:, None] + n - (hi - lo)
        s = torch.where(seen, s, -math.inf)
        empty = ~seen.any(-1)
        top = s.amax(-1, keepdim=True) if n else torch.zeros(*s.shape[:-1], 1, dtype=s.dtype, device=s.device)
        w = torch.exp(s - torch.where(top == -math.inf, 0, top))
        total = w.sum(-1, keepdim=True)
        p = torch.where(empty[:, None], 0, w / total)
        out[lo:hi] = torch.einsum("hgmn,hnd->hgmd", p, v).reshape(Hq, hi - lo, D).transpose(0, 1)
        size[lo:hi] = torch.einsum("hgmn,hnd->hgmd", p, v.abs()).reshape(Hq, hi - lo, D).transpose(0, 1)
        lse[:, lo:hi] = torch.where(empty, math.inf, (top + total.log())[..., 0]).reshape(Hq, hi - lo)
        if n:
            most[:, lo:hi] = torch.where(seen, s.abs(), 0).amax(-1).reshape(Hq, hi - lo)
    return out, lse, size, most


def rotary(x, positions, inv_freq, sections=None, interleaved=False, scaling=1.0, inverse=False):
    """x [..., heads, rows, dim] or packed [rows, heads, dim], in 64 bits. positions [axes, ...] with sections, else [...]."""
    half = inv_freq.numel()
    pos = positions.double()
    pos = pos if sections is not None else pos[None]
    axis = torch.tensor([a for a, n in enumerate(sections or (half,)) for _ in range(n)], device=x.device)
    angle = pos[axis].movedim(0, -1) * inv_freq.double()  # [tokens, half] or [(batch,) length, half]
    c, s = angle.cos() * scaling, angle.sin() * scaling * (-1 if inverse else 1)
    if x.dim() == 3:
        c, s = c[:, None], s[:, None]
    else:
        c, s = (c[:, None], s[:, None]) if c.dim() == 3 else (c[None, None], s[None, None])
    y = x.double().clone()
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    first, second = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = first, second
    else:
        y[..., :half], y[..., half:2 * half] = first, second
    return y
