"""Rotary positions against the formula in 64 bits: layouts, axes, both pairings, partial rows, far positions, gradients, in place.

Tolerance: the result is rounded once, half a step of its type (2^-8 of the value in bf16, 2^-11 in f16, half of f16's least step below its smallest
normal number), and computed in 32 bits before: the reduced angle (at most pi) is off by 2^-24 * pi, cosine and sine by 2^-23, two products and a sum by
2^-24 each of |x| + |y|: less than 6e-7 * (|x| + |y|) * scaling together."""
import pytest
import torch

from oracle import cache_oracle as orc
from torch_mlu_b200 import rotary

pytestmark = pytest.mark.gpu


def _check(got, x, positions, inv_freq, what, scaling=1.0, **kw):
    assert got.shape == x.shape and got.dtype == x.dtype
    want = orc.rotary(x, positions, inv_freq, scaling=scaling, **kw)
    size = orc.rotary(x.abs(), torch.zeros_like(positions), inv_freq, **{**kw, "inverse": False})  # |x|; the partner's is at most the row's largest
    part = x.abs().double().amax(-1, keepdim=True) + size
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 6e-7 * part * abs(scaling) + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (what, float((off - tol).max()))


def _freq(half, dev, theta=1e4):
    return (theta ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)).float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot,interleaved", [(1, 32, 8, 128, 128, False), (64, 32, 8, 128, 128, False), (33, 8, 1, 128, 64, True),
                                                              (2500, 4, 2, 64, 64, True), (7, 3, 3, 80, 80, False), (2049, 2, 1, 256, 256, False),
                                                              (5, 12, 4, 96, 16, True), (19, 5, 0, 72, 32, False)])
def test_packed(cuda_device, dtype, tokens, hq, hk, dim, rot, interleaved):
    g = torch.Generator(device=cuda_device).manual_seed(tokens)
    q = torch.randn(tokens, hq, dim, generator=g, device=cuda_device).to(dtype)
    k = torch.randn(tokens, hk, dim, generator=g, device=cuda_device).to(dtype) if hk else None
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device=cuda_device, dtype=torch.int32)
    f = _freq(rot // 2, cuda_device)
    a, b = rotary.rotary_embedding(q, k, pos, f, interleaved=interleaved)
    _check(a, q, pos, f, "q", interleaved=interleaved)
    if hk:
        _check(b, k, pos, f, "k", interleaved=interleaved)
    else:
        assert b is None


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(16, 24, 24), (0, 64), (1, 2, 3, 58), (64,)])
def test_axes(cuda_device, sections, interleaved):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    q = torch.randn(2, 6, 50, 128, generator=g, device=cuda_device).bfloat16()
    k = torch.randn(2, 2, 50, 128, generator=g, device=cuda_device).bfloat16()
    pos = torch.randint(-3, 100000, (len(sections), 2, 50), generator=g, device=cuda_device)  # int64
    f = _freq(64, cuda_device, 1e6)
    a, b = rotary.rotary_embedding(q, k, pos, f, sections=sections, interleaved=interleaved, scaling=0.75)
    _check(a, q, pos, f, "q", scaling=0.75, sections=sections, interleaved=interleaved)
    _check(b, k, pos, f, "k", scaling=0.75, sections=sections, interleaved=interleaved)
    # a position for all batches, and positions of any strides
    a, _ = rotary.rotary_embedding(q, k, pos[:, :1], f, sections=sections)
    _check(a, q, pos[:, :1].expand(-1, 2, -1), f, "broadcast", sections=sections)
    turned = pos.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    assert torch.equal(rotary.rotary_embedding(q, k, turned, f, sections=sections)[0], rotary.rotary_embedding(q, k, pos, f, sections=sections)[0])


def test_layouts_and_one_position_row(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(2)
    pos, f = torch.arange(37, device=cuda_device, dtype=torch.int32), _freq(32, cuda_device)
    base = torch.randn(3, 37, 2 * 8 + 4, 64, generator=g, device=cuda_device).half()
    q, k = base[:, :, :8].transpose(1, 2), base[:, :, 16:].transpose(1, 2)  # slices of a projection, [batch, heads, length, dim]
    for x, y in ((q, k), (q.contiguous(), k.contiguous()), (q[:1].expand(3, -1, -1, -1), k[:, :1].expand(-1, 4, -1, -1))):
        a, b = rotary.rotary_embedding(x, y, pos, f)
        _check(a, x, pos, f, "q")
        _check(b, y, pos, f, "k")
    packed = rotary.rotary_embedding(base[1, :, :8], base[1, :, 16:], pos, f)
    assert torch.equal(packed[0], rotary.rotary_embedding(q, k, pos, f)[0][1].transpose(0, 1))
    empty = rotary.rotary_embedding(base[1, :0, :8], base[1, :0, 16:], pos[:0], f)
    assert empty[0].shape == (0, 8, 64) and empty[1].shape == (0, 4, 64)


def test_in_place_touches_its_rows_only(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    base = torch.randn(21, 12, 128, generator=g, device=cuda_device).bfloat16()
    pos, f = torch.arange(21, device=cuda_device), _freq(32, cuda_device)
    want = rotary.rotary_embedding(base[:, :6], base[:, 8:10], pos, f)
    work = base.clone()
    q, k = rotary.rotary_embedding_(work[:, :6], work[:, 8:10], pos, f)
    assert q.data_ptr() == work.data_ptr()
    assert torch.equal(work[:, :6], want[0]) and torch.equal(work[:, 8:10], want[1])
    assert torch.equal(work[:, 6:8], base[:, 6:8]) and torch.equal(work[:, 10:], base[:, 10:])


def test_refusals(cuda_device):
    q, f = torch.zeros(4, 2, 128, device=cuda_device, dtype=torch.bfloat16), _freq(64, cuda_device)
    pos = torch.zeros(4, device=cuda_device, dtype=torch.int32)
    call = rotary.rotary_embedding
    for args, kw, text in [((q.float(), None, pos, f), {}, "bf16 or fp16"), ((q, q.half(), pos, f), {}, "both the same"), ((q, q[:3], pos, f), {}, "same tokens"),
                           ((q, q, pos.float(), f), {}, "int32 or int64"), ((q, q, pos[:3], f), {}, r"positions must be \[tokens\]"),
                           ((q, q, pos, f.double()), {}, "inv_freq"), ((q, q, pos, f), {"sections": (32, 31)}, "sections"),
                           ((q, q, pos[None].expand(2, -1), f), {"sections": (20, 20, 24)}, "3 axes"), ((q[..., ::2], None, pos, f), {}, "contiguous last"),
                           ((q, q, pos, f[:20]), {}, "multiple of 16"), ((q[:, :, :64], q, pos, f[:32]), {}, "agree")]:
        with pytest.raises(RuntimeError, match=text):
            call(*args, **kw)


@pytest.mark.parametrize("layout", ["packed", "dense"])
@pytest.mark.parametrize("interleaved,rot", [(False, 128), (True, 64)])
def test_gradients(cuda_device, layout, interleaved, rot):
    """Against the formula (the gradient is the turn backwards) and against differences of the 64-bit forward, which is linear: <dy, f(e)> for a unit
    vector e is exact but for the rounding of the result, half a step."""
    g = torch.Generator(device=cuda_device).manual_seed(4)
    shapes = [(30, h, 128) if layout == "packed" else (2, h, 15, 128) for h in (6, 2)]
    q, k, dq, dk = (torch.randn(*s, generator=g, device=cuda_device).bfloat16() for s in shapes * 2)
    tokens = (30,) if layout == "packed" else (2, 15)
    pos = torch.randint(0, 50000, (2,) + tokens, generator=g, device=cuda_device)
    f, sections = _freq(rot // 2, cuda_device), (rot // 8, rot // 2 - rot // 8)
    q.requires_grad_()
    k.requires_grad_()
    kw = dict(sections=sections, interleaved=interleaved, scaling=1.5)
    a, b = rotary.rotary_embedding(q, k, pos, f, **kw)
    assert a.requires_grad and b.requires_grad
    gq, gk = torch.autograd.grad((a, b), (q, k), (dq, dk), retain_graph=True)
    for got, d in ((gq, dq), (gk, dk)):
        _check(got, d, pos, f, "gradient", inverse=True, **kw)
    for at in [(0, 0, 0), (3, 1, 5), (29, 5, 127)] if layout == "packed" else [(0, 0, 0, 0), (1, 5, 14, 63), (1, 0, 7, 127)]:
        e = torch.zeros(shapes[0], dtype=torch.float64, device=cuda_device)
        e[at] = 1
        want = float((orc.rotary(e, pos, f, **kw) * dq.double()).sum())
        assert abs(float(gq[at]) - want) <= 2.0 ** -8 * abs(want) + 6e-7 * 1.5 * 2 * float(dq.double().abs().max())
    # one of the two alone; a gradient that is expanded, and one whose rows the kernel cannot read
    only, = torch.autograd.grad(b, k, dk, retain_graph=True)
    assert torch.equal(only, gk)
    only, = torch.autograd.grad((a, b), q, (dq, dk), retain_graph=True)
    assert torch.equal(only, gq)
    one = torch.ones((), device=cuda_device, dtype=torch.bfloat16).expand(shapes[0])
    got, = torch.autograd.grad(a, q, one, retain_graph=True)
    _check(got, one, pos, f, "expanded", inverse=True, **kw)
    odd = torch.randn(*shapes[0][:-1], 129, generator=g, device=cuda_device).bfloat16()[..., 1:]
    got, = torch.autograd.grad(a, q, odd, retain_graph=True)
    _check(got, odd, pos, f, "odd rows", inverse=True, **kw)


def test_second_derivative_and_shared_inputs(cuda_device):
    """The backward is differentiable itself; a leaf used by both and an input expanded over heads get the sum of their gradients."""
    pos, f = torch.arange(9, device=cuda_device), _freq(32, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(9, 1, 64, generator=g, device=cuda_device).half().requires_grad_()
    v = torch.randn(9, 4, 64, generator=g, device=cuda_device).half().requires_grad_()
    y, _ = rotary.rotary_embedding(x.expand(-1, 4, -1), None, pos, f)
    gx, = torch.autograd.grad(y, x, v, create_graph=True)
    want = orc.rotary(v, pos, f, inverse=True).sum(1, keepdim=True)
    assert bool(((gx.double() - want).abs() <= 2.0 ** -11 * (want.abs() + 4 * 4) + 1e-5).all())  # four rounded rows, then their sum in f16, twice
    w = torch.randn(9, 1, 64, generator=g, device=cuda_device).half()
    gv, = torch.autograd.grad(gx, v, w)
    want = orc.rotary(w, pos, f)
    assert bool(((gv.double() - want).abs() <= 2.0 ** -11 * want.abs() + 1e-5).all())
    a, b = rotary.rotary_embedding(x, x, pos, f)
    g1, = torch.autograd.grad((a, b), x, (w, w))
    _check(g1 / 2, w, pos, f, "shared", inverse=True)


def test_learned_frequencies_are_refused(cuda_device):
    pos, f = torch.arange(9, device=cuda_device), _freq(32, cuda_device).requires_grad_()
    x = torch.randn(9, 2, 64, device=cuda_device).half()
    with pytest.raises(RuntimeError, match="no gradient of inv_freq"):
        rotary.rotary_embedding(x, None, pos, f)
    with torch.no_grad():
        assert torch.equal(rotary.rotary_embedding(x, None, pos, f)[0], rotary.rotary_embedding(x, None, pos, f.detach())[0])


def test_autograd_refuses_what_it_would_get_wrong(cuda_device):
    pos, f = torch.arange(9, device=cuda_device), _freq(32, cuda_device)
    x = torch.randn(9, 2, 64, device=cuda_device).half()
    with pytest.raises(RuntimeError, match="no gradient: use rotary_embedding"):
        rotary.rotary_embedding_(x.clone().requires_grad_(), None, pos, f)
    with pytest.raises(RuntimeError, match="elements of their own"):
        rotary.rotary_embedding_(x[:, :1].expand(-1, 2, -1), None, pos, f)
    with pytest.raises(RuntimeError, match="the same memory"):
        rotary.rotary_embedding_(x, x, pos, f)
    with torch.inference_mode():
        y = x.clone()
        want = rotary.rotary_embedding(x, None, pos, f)[0]
        assert torch.equal(rotary.rotary_embedding_(y, None, pos, f)[0], want)
    with pytest.raises(RuntimeError, match="ordinary tensor"):
        torch.func.grad(lambda t: rotary.rotary_embedding(t, None, pos, f)[0].float().sum())(x)
    # a tensor saved for a backward pass and then turned in place is noticed
    y = (x.clone().requires_grad_() * 2)
    z = y * y
    with torch.no_grad():
        rotary.rotary_embedding_(y, None, pos, f)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_captured_training_step(cuda_device):
    """Forward and backward into a graph, replayed on new data, while an eager graph of the same values lives. The captured step has a leaf of its own over
    them: torch ties a leaf's gradient node to the stream that first used it, and a capture cannot wait for the default stream, whatever the operator."""
    pos, f = torch.arange(40, device=cuda_device), _freq(64, cuda_device)
    q = torch.randn(40, 4, 128, device=cuda_device).bfloat16().requires_grad_()
    d = torch.randn(40, 4, 128, device=cuda_device).bfloat16()
    leaf = q.detach().requires_grad_()
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, leaf, d)))(rotary.rotary_embedding(leaf, None, pos, f)[0])
    alive = rotary.rotary_embedding(q, None, pos, f)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gq = step()
    for _ in range(2):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            d.copy_(torch.randn_like(d))
            pos += 1000
        graph.replay()
        torch.cuda.synchronize()
        _check(y, q.detach(), pos, f, "replayed")
        _check(gq, d, pos, f, "replayed gradient", inverse=True)
    del alive
