"""The serving operators and rotary positions under tracers, dispatch modes and functional transforms: what records a call records the operator, not its results as constants."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from test_kv_cache_gpu import E4M3, INT8, _batch, _cache, _ints, _run
from test_rotary_gpu import _freq
from torch_mlu_b200 import kv_cache, rotary

pytestmark = pytest.mark.gpu


def _nodes(traced):
    return [str(n.target) for n in traced.graph.nodes if n.op == "call_function"]


def _inputs(dev, seed, tokens=33, grad=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, k = (torch.randn(tokens, h, 128, generator=g, device=dev).bfloat16().requires_grad_(grad) for h in (4, 2))
    return q, k, torch.randint(0, 9000, (tokens,), generator=g, device=dev)


class _Log(torch.utils._python_dispatch.TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("with_key", [True, False])
@pytest.mark.parametrize("how", ["make_fx", "jit"])
def test_traced_rotary_positions(cuda_device, how, with_key):
    f = _freq(64, cuda_device)

    def turn(q, k, pos):
        a, b = rotary.rotary_embedding(q, k if with_key else None, pos, f, scaling=0.5)
        return a if b is None else (a, b)

    traced = make_fx(turn)(*_inputs(cuda_device, 1)) if how == "make_fx" else torch.jit.trace(turn, _inputs(cuda_device, 1), check_trace=False)
    if how == "make_fx":
        assert _nodes(traced).count("b200_sdpa.rotary_embedding.default") == 1
    other = _inputs(cuda_device, 2)
    for a, b in zip(traced(*other), turn(*other)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("how", ["make_fx", "jit"])
def test_traced_rotary_positions_in_place_and_with_axes(cuda_device, how):
    f = _freq(64, cuda_device)

    def turn(q, k, pos):
        q, k = q.clone(), k.clone()
        pos = torch.stack([pos, pos + 1, pos * 2])
        rotary.rotary_embedding_(q, k, pos, f, sections=(16, 24, 24), interleaved=True)
        return q, k

    traced = make_fx(turn)(*_inputs(cuda_device, 1)) if how == "make_fx" else torch.jit.trace(turn, _inputs(cuda_device, 1), check_trace=False)
    other = _inputs(cuda_device, 2)
    for a, b in zip(traced(*other), turn(*other)):
        assert torch.equal(a, b)


def test_make_fx_records_the_gradient(cuda_device):
    """Forward, backward and the backward's own gradient."""
    f = _freq(64, cuda_device)

    def step(q, k, pos):
        a, b = rotary.rotary_embedding(q, k, pos, f)
        gq, gk = torch.autograd.grad((a, b), (q, k), (a * 2, b * b), create_graph=True)
        return a, b, gq, gk, torch.autograd.grad(gq, q, a)[0]

    traced = make_fx(step)(*_inputs(cuda_device, 1, grad=True))
    assert _nodes(traced).count("b200_sdpa.rotary_embedding.default") >= 3
    other = _inputs(cuda_device, 2, grad=True)
    for a, b in zip(traced(*other), step(*other)):
        assert torch.equal(a, b)


def test_a_traced_gradient_runs_again(cuda_device):
    """torch.jit.trace of a call whose inputs need gradients: the traced program differentiates as the call does."""
    f = _freq(64, cuda_device)
    turn = lambda q, k, pos: rotary.rotary_embedding(q, k, pos, f)
    traced = torch.jit.trace(turn, _inputs(cuda_device, 1, grad=True), check_trace=False)
    q, k, pos = _inputs(cuda_device, 2, grad=True)
    grads = [torch.autograd.grad(fn(q, k, pos), (q, k), (q.detach(), k.detach())) for fn in (traced, turn)]
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("how", ["make_fx", "jit"])
def test_a_traced_serving_step(cuda_device, how):
    """Bookkeeping in place and not, store and attention, run again on other tokens, lengths and caches."""
    blocks, heads, block, dim, requests, tokens = 12, 2, 16, 64, 2, 24

    def state(seed):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        kc, ks = _cache(cuda_device, blocks, heads, block, dim, INT8, seed)
        vc, vs = _cache(cuda_device, blocks, heads, block, dim, INT8, seed + 1)
        q, k, v = (torch.randn(tokens, h, dim, generator=g, device=cuda_device).half() for h in (4, heads, heads))
        return (q, k, v, _ints(cuda_device, [seed, 20 - seed]), _ints(cuda_device, [0, 0]), torch.full((requests, 4), -1, dtype=torch.int32, device=cuda_device),
                torch.arange(blocks, dtype=torch.int32, device=cuda_device), _ints(cuda_device, [seed, blocks, 0]), kc, vc, ks, vs)

    def step(q, k, v, new, lens, table, ring, ring_state, kc, vc, ks, vs):
        plan = kv_cache.plan_step(lens, new, table, ring, ring_state, block_size=block, num_tokens=tokens)
        again = kv_cache.plan_step(plan.seq_lens, new * 0, table, ring, plan.ring_state, block_size=block, num_tokens=tokens, in_place=True)
        kv_cache.store(k, v, plan.slots, kc, vc, ks, vs)
        out, lse = kv_cache.attention(q, kc, vc, ks, vs, table, again.seq_lens, plan.cu_seqlens, 20, 64)
        live = torch.arange(tokens, device=q.device) < plan.cu_seqlens[-1]
        return (torch.where(live[:, None, None], out, 0), torch.where(live, lse, 0), *plan, *again, table, ring, kc, vc, ks, vs)

    traced = make_fx(step)(*state(3)) if how == "make_fx" else torch.jit.trace(step, state(3), check_trace=False)
    if how == "make_fx":
        nodes = _nodes(traced)
        for name in ("plan_step", "plan_step_", "cache_store_", "cache_attention"):
            assert f"b200_sdpa.{name}.default" in nodes
    for a, b in zip(traced(*state(7)), step(*state(7))):
        assert torch.equal(a.view(torch.int8) if a.dtype == E4M3 else a, b.view(torch.int8) if b.dtype == E4M3 else b)


def test_dispatch_modes_see_a_serving_step(cuda_device):
    def serve(log=None):
        cache = kv_cache.PagedCache(1, 8, 2, 64, 2, 4, block_size=16, device=cuda_device)
        g = torch.Generator(device=cuda_device).manual_seed(1)
        q, k, v = (torch.randn(9, h, 64, generator=g, device=cuda_device).bfloat16() for h in (4, 2, 2))
        new = _ints(cuda_device, [5, 4])
        if log is None:
            cache.step(new, 9)
            return cache.attend(0, q, k, v, 5, 64, inv_freq=_freq(32, cuda_device))
        f = _freq(32, cuda_device)
        with log:
            cache.step(new, 9)
            return cache.attend(0, q, k, v, 5, 64, inv_freq=f)

    log = _Log()
    for a, b in zip(serve(log), serve()):
        assert torch.equal(a, b)
    for name in ("plan_step_", "rotary_embedding_", "cache_store_", "cache_attention"):
        assert log.seen.count(f"b200_sdpa.{name}.default") == 1, log.seen


def test_dispatch_modes_see_the_gradient(cuda_device):
    f = _freq(64, cuda_device)
    q, k, pos = _inputs(cuda_device, 1, grad=True)
    a, b = rotary.rotary_embedding(q, k, pos, f)
    want = torch.autograd.grad((a, b), (q, k), (q.detach(), k.detach()), retain_graph=True)
    with _Log() as log:
        got = torch.autograd.grad((a, b), (q, k), (q.detach(), k.detach()))
    assert log.seen.count("b200_sdpa.rotary_embedding.default") == 1
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_registered_operators_are_the_calls(cuda_device):
    """torch.ops.b200_sdpa: the same results and checks; under autocast, inference mode and below autograd too."""
    f = _freq(64, cuda_device)
    q, k, pos = _inputs(cuda_device, 1, grad=True)
    want = rotary.rotary_embedding(q, k, pos, f)
    got = torch.ops.b200_sdpa.rotary_embedding(q, k, pos, f, None, False, 1.0, False)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and got[0].requires_grad
    back = torch.ops.b200_sdpa.rotary_embedding(got[0], None, pos, f, None, False, 1.0, True)
    assert len(back) == 1 and float((back[0] - q).abs().max()) < 0.1
    with torch.autocast("cuda", torch.float16):
        assert all(torch.equal(x, y) for x, y in zip(rotary.rotary_embedding(q, k, pos, f), want))
    with torch.inference_mode():
        assert all(torch.equal(x, y) for x, y in zip(rotary.rotary_embedding(q, k, pos, f), want))
    with torch._C._AutoDispatchBelowAutograd():
        below = rotary.rotary_embedding(q, k, pos, f)
    assert not below[0].requires_grad and torch.equal(below[0], want[0])
    with pytest.raises(RuntimeError, match="no gradient of inv_freq"):
        torch.ops.b200_sdpa.rotary_embedding(q, k, pos, f.clone().requires_grad_(), None, False, 1.0, False)
    b = _batch(cuda_device, [100, 90], [5, 2], 4, 2, 64, 16, INT8, torch.bfloat16)
    one, two = _run(b), torch.ops.b200_sdpa.cache_attention(*b, 5, 100, True, None)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    with pytest.raises(RuntimeError, match="has no gradient"):
        torch.ops.b200_sdpa.cache_attention(b[0].clone().requires_grad_(), *b[1:], 5, 100, True, None)


def test_functional_transforms_are_refused(cuda_device):
    q, kc, vc, ks, vs, table, lens, cu = _batch(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, INT8, torch.float16)
    k = torch.zeros(2, 2, 64, device=cuda_device, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ordinary tensor"):
        torch.func.grad(lambda t: kv_cache.attention(t, kc, vc, ks, vs, table, lens)[0].float().sum())(q)
    with pytest.raises(RuntimeError, match="ordinary tensor"):
        torch.func.vmap(lambda t: kv_cache.attention(t, kc, vc, ks, vs, table, lens)[0])(torch.stack([q, q]))
    with pytest.raises(RuntimeError, match="ordinary tensor"):
        torch.func.functionalize(lambda t: kv_cache.store(t, k, lens * 0, kc, vc, ks, vs))(k)
    with pytest.raises(RuntimeError, match="ordinary tensor"):
        torch.func.vmap(lambda t: kv_cache.plan_step(lens, t, table, lens, _ints(cuda_device, [0, 0, 0]), block_size=16, num_tokens=4).slots)(torch.stack([lens, lens]))


def test_what_would_be_left_out_of_a_derivative_is_refused(cuda_device):
    """Scales and caches that need gradients, and tangents of any argument."""
    import torch.autograd.forward_ad as fwAD
    q, kc, vc, ks, vs, table, lens, cu = _batch(cuda_device, [100, 90], [1, 1], 4, 2, 64, 16, E4M3, torch.bfloat16, poison=False)
    k, slots, f, pos = torch.ones(2, 2, 64, device=cuda_device, dtype=torch.bfloat16), _ints(cuda_device, [0, 1]), _freq(32, cuda_device), _ints(cuda_device, [3, 4])
    attend = lambda *a: kv_cache.attention(*a, table, lens)
    store = lambda *a: kv_cache.store(a[0], a[1], slots, *a[2:])
    before = [x.clone() for x in (kc.view(torch.int8), vc.view(torch.int8), ks, vs)]
    for call, args, text in ((attend, (q, kc, vc, ks, vs), "has no gradient"), (store, (k, k.clone(), kc, vc, ks, vs), "keeps no gradient")):
        for i, x in enumerate(args):
            if x.dtype == E4M3:
                continue
            with pytest.raises(RuntimeError, match=text):
                call(*(y.detach().requires_grad_() if j == i else y for j, y in enumerate(args)))
            with torch.no_grad():
                call(*(y.detach().clone().requires_grad_() if j == i else y.clone() for j, y in enumerate(args)))
            with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(*(fwAD.make_dual(y, torch.ones_like(y)) if j == i else y for j, y in enumerate(args)))
    for call in (rotary.rotary_embedding, rotary.rotary_embedding_):
        for i in (0, 1, 3):
            args = [q.clone(), k.clone(), pos, f]
            with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                args[i] = fwAD.make_dual(args[i], torch.ones_like(args[i]))
                call(*args)
    assert all(torch.equal(x, y) for x, y in zip(before, (kc.view(torch.int8), vc.view(torch.int8), ks, vs)))
