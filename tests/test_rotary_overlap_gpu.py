"""Rotary positions in place on slices of one tensor: those that share elements are refused, those that do not are turned as each alone."""
import pytest
import torch

from test_rotary_gpu import _freq
from torch_mlu_b200 import rotary

pytestmark = pytest.mark.gpu


def _slices(base, dense):
    """(query, key, whether they share elements) of [tokens, 12 heads, 64] or [2, 12 heads, tokens, 64] in three memory orders."""
    at = (lambda lo, hi, step=1: base[:, lo:hi:step])
    yield at(0, 6), at(6, 8), False
    yield at(0, 6), at(5, 8), True
    yield at(6, 12), at(0, 6), False
    yield at(6, 12), at(0, 7), True
    yield at(0, 12), at(3, 4), True
    yield at(0, 12, 2), at(1, 12, 2), False  # heads in turn
    yield at(0, 12, 2), at(2, 12, 2), True
    yield at(2, 3), at(2, 3), True
    if not dense:  # rows that begin 8 elements behind those of a head
        yield at(0, 6), base.as_strided((base.shape[0], 2, 64), (base.stride(0), base.stride(1), 1), 5 * 64 + 8), True
        yield at(0, 6), base.as_strided((base.shape[0], 2, 64), (base.stride(0), base.stride(1), 1), 6 * 64), False


@pytest.mark.parametrize("layout", ["packed", "heads", "tokens"])
def test_slices_of_one_tensor(cuda_device, layout):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    base = torch.randn(*((9, 12, 64) if layout == "packed" else (2, 12, 9, 64) if layout == "heads" else (2, 9, 12, 64)), generator=g, device=cuda_device).half()
    pos, f = torch.arange(9, device=cuda_device) * 7, _freq(32, cuda_device)
    view = (lambda x: x.transpose(1, 2)) if layout == "tokens" else (lambda x: x)
    for i in range(8 if layout != "packed" else 10):
        work = base.clone()
        q, k, shared = list(_slices(view(work), layout != "packed"))[i]
        if shared:
            with pytest.raises(RuntimeError, match="share some"):
                rotary.rotary_embedding_(q, k, pos, f)
            assert torch.equal(work, base)
        else:
            want = rotary.rotary_embedding(q, k, pos, f)
            rotary.rotary_embedding_(q, k, pos, f)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1]), i


def test_shifted_by_a_token(cuda_device):
    base = torch.randn(10, 4, 64, device=cuda_device).half()
    pos, f = torch.arange(9, device=cuda_device), _freq(32, cuda_device)
    with pytest.raises(RuntimeError, match="share some"):
        rotary.rotary_embedding_(base[:9], base[1:], pos, f)
    rotary.rotary_embedding_(base[:5], base[5:], pos[:5], f)
    wide = torch.randn(2, 9, 4, 64, device=cuda_device).half()
    with pytest.raises(RuntimeError, match="share some"):
        rotary.rotary_embedding_(wide[:1].transpose(1, 2), wide.view(18, 4, 64)[8:17][None].transpose(1, 2), pos, f)
    rotary.rotary_embedding_(wide[:1].transpose(1, 2), wide[1:].transpose(1, 2), pos, f)
