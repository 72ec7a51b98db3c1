"""The ends of the serving operators' ranges: long lists, the types' largest values, lengths and bounds that do not fit, against the restatements in 64 bits.
Tolerances as in test_kv_cache_gpu.py, from which the helpers come."""
import math

import pytest
import torch

from oracle import cache_oracle as orc
from test_kv_cache_gpu import E4M3, INT8, _batch, _cache, _compare, _ints, _run, _same_cache
from torch_mlu_b200 import kv_cache, ops

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
    from torch_mlu_b200 import _cabi
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
