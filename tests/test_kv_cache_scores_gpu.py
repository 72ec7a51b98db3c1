"""Attention over the paged cache at softmax scales from 32 bits' smallest number to near its largest, and so at scores of any size, against the restatement in 64 bits.

Where all scores of a row are near 0 the tolerances are those of the other files. Where they are large, the row's largest score stands so far above the others that theirs weigh
nothing, which is asserted: a score is a sum of head_dim products in 32 bits, off by up to 2^-20 of the sum of the products' magnitudes (an addition rounds by 2^-24 of what it has, there are 128,
codes of 4 bits add 2^-19 of sum |q| times the scale of K: 16 * 2^-24 in each of two steps of 16 dimensions). The row is then the one value, rounded to its type, its weight and the sum off by no
more than one f16 rounding each (2^-11), and the logsumexp the score itself."""
import math

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache4_gpu import INT4, _batch4
from test_kv_cache4_gpu import _compare as _compare4
from test_kv_cache_gpu import E4M3, INT8, _batch, _compare, _run
from torch_mlu_b200 import ops

pytestmark = pytest.mark.gpu


def _any_batch(dev, lens, rows, dim, code, seed, hq=8, hkv=2, block=16, dtype=torch.bfloat16):
    if code == INT4:
        return _batch4(dev, lens, rows, hq, hkv, dim, block, dtype, seed=seed)
    return _batch(dev, lens, rows, hq, hkv, dim, block, code, dtype, seed=seed)


def _zero_some(b, rows):
    """Rows of zeros and of ones among the queries."""
    q = b[0]
    q[::3] = 0
    q[1::3, ::2] = 1
    return b


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [1e-45, 1e-38, 1e-12])
def test_scales_at_which_all_scores_vanish(cuda_device, scale, dim, rows, code):
    b = _zero_some(_any_batch(cuda_device, [700, 45, 130], [rows, min(rows, 40), 1], dim, code, rows), rows)
    (_compare4 if code == INT4 else _compare)(*_run(b, scale=scale), b, True, scale, many=rows > 500)
    assert ops.device_status() == 0


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
@pytest.mark.parametrize("scale", [2.0 ** 13, 2.0 ** 118, 1e36, 2.9e38])
def test_rows_of_zeros_at_any_scale(cuda_device, scale, rows, code):
    """Their scores are 0 whatever the scale."""
    b = _any_batch(cuda_device, [700, 45, 130], [rows, min(rows, 40), 1], 128, code, rows)
    b[0][:] = 0
    (_compare4 if code == INT4 else _compare)(*_run(b, scale=scale), b, True, scale, many=rows > 500)
    assert ops.device_status() == 0


def _one_key(out, lse, b, scale):
    q, kc, vc, ks, vs, table, lens, cu = b
    hq, dim, hkv, block = q.shape[1], q.shape[2], kc.shape[1], kc.shape[2]
    decided, lo = 0, 0
    for i, n in enumerate(lens.tolist()):
        hi = int(cu[i + 1])
        ids = table[i, :-(-n // block)].long()
        flat = lambda c, s: orc.elements(c.view(torch.uint8)[ids].view(c.dtype), s[ids]).permute(1, 0, 2, 3).reshape(hkv, -1, dim)[:, :n].repeat_interleave(hq // hkv, 0)
        k, v = flat(kc, ks), flat(vc, vs)
        rows = q[lo:hi].double().transpose(0, 1)  # [heads, rows, dim]
        s = torch.einsum("hmd,hnd->hmn", rows, k) * scale
        error = torch.einsum("hmd,hnd->hmn", rows.abs(), k.abs()) * scale * 2.0 ** -20
        if kc.dtype == INT4:
            error = error + rows.abs().sum(-1, keepdim=True) * scale * 2.0 ** -19 * float(ks.nan_to_num(0, 0, 0).abs().max())
        seen = torch.arange(n, device=q.device)[None] <= torch.arange(hi - lo, device=q.device)[:, None] + n - (hi - lo)
        s = torch.where(seen, s, -math.inf)
        top, at = s.max(-1, keepdim=True)
        others = torch.where(torch.arange(n, device=q.device) == at, -math.inf, s + error).amax(-1)
        clear = (top - error.gather(-1, at))[..., 0] > others + 40  # [heads, rows]
        decided += int(clear.sum())
        want = torch.stack([v[h, at[h, :, 0]] for h in range(hq)])  # [heads, rows, dim]
        got = out[lo:hi].transpose(0, 1).double()
        tol = (torch.finfo(q.dtype).eps / 2 + 2.0 ** -10) * want.abs()
        assert bool((((got - want).abs() <= tol).all(-1) | ~clear).all()), (i, float(((got - want).abs() - tol).nan_to_num(1e9).max()))
        assert bool(got.isfinite().all())
        ltol = error.gather(-1, at)[..., 0] + 2.0 ** -22 * top[..., 0].abs()
        assert bool((((lse[:, lo:hi].double() - top[..., 0]).abs() <= ltol) | ~clear).all())
        lo = hi
    assert decided > 0.8 * out.shape[0] * hq


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
@pytest.mark.parametrize("scale", [2.0 ** 19, 2.0 ** 20, 2.0 ** 21, 2.0 ** 22, 2.0 ** 24, 1e18, 1e36])
def test_scores_of_any_size(cuda_device, scale, rows, code):
    """Queries of ones and of random numbers, whose scores are 2^20 and more: a weight is a power of two of their difference, in which a rounding of the score counts by whole steps."""
    b = _any_batch(cuda_device, [700, 45, 130], [rows, min(rows, 40), 1], 128, code, rows + 1)
    b[0][::2] = 1
    _one_key(*_run(b, scale=scale), b, scale)
    if code != INT4:  # scales of V above 1, whose sums are formed on their own
        b[4][:] *= 2.0 ** 12
        _one_key(*_run(b, scale=scale), b, scale)
    assert ops.device_status() == 0


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
@pytest.mark.parametrize("dim,by", [(64, -100), (128, -60), (128, 60), (64, 100)])
def test_small_queries_over_large_keys(cuda_device, dim, by, rows, code):
    """Queries times a power of two over keys divided by it: the same scores, and the same tolerances."""
    b = _any_batch(cuda_device, [700, 45, 130], [rows, min(rows, 40), 1], dim, code, rows + 2)
    b = ((b[0].double() * 2.0 ** by).bfloat16(), *b[1:3], (b[3].double() * 2.0 ** -by).to(b[3].dtype), *b[4:])
    (_compare4 if code == INT4 else _compare)(*_run(b), b, many=rows > 500)
    assert ops.device_status() == 0


@pytest.mark.parametrize("code", [INT4, E4M3])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
def test_the_same_call_gives_the_same_bits(cuda_device, rows, code):
    b = _any_batch(cuda_device, [5000, 45, 1300] * 4, [rows, min(rows, 40), 1] * 4, 128, code, rows)
    out, lse = _run(b)
    for _ in range(5):
        again = _run(b)
        assert torch.equal(out.view(torch.int16), again[0].view(torch.int16)) and torch.equal(lse, again[1])


@pytest.mark.parametrize("code", [INT4, E4M3, INT8])
@pytest.mark.parametrize("rows", [1, 3, 30, 600])
@pytest.mark.parametrize("dim", [64, 128])
def test_queries_that_are_no_numbers(cuda_device, dim, rows, code):
    """A NaN or an infinity in one head of a row makes that row and head NaN; those beside it in the same unit are as they would be."""
    b = _any_batch(cuda_device, [700, 45, 130], [rows, min(rows, 40), 1], dim, code, rows + 3)
    last = b[0].shape[0] - 1
    b[0][0, 1, 5], b[0][last, 2, dim - 1], b[0][rows // 2, 6, 0] = math.nan, math.inf, -math.inf
    out, lse = _run(b)
    want = orc.attention(*b)[0]
    assert torch.equal(out.isnan(), want.isnan()) and int(out.isnan().all(-1).sum()) == 3 and int(out.isnan().any(-1).sum()) == 3
    at = out.isnan().any(-1)
    b[0][at], out[at] = 0, 0
    rest = orc.attention(*b)
    out[at], lse.t()[at] = rest[0][at].to(out.dtype), rest[1].t()[at].float()
    (_compare4 if code == INT4 else _compare)(out, lse, b, many=rows > 500)
