"""Norm and attention under what has to see their custom ops: compilation, dispatch modes, batches of output gradients, vmap,
forward-mode differentiation, views with the negative bit, saved tensors of another layout."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.ops.add(str(func))
        return func(*args, **(kwargs or {}))


def _randn(*shape, dt=torch.bfloat16, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dt)


def _attention(dt=torch.bfloat16):
    leaves = [_randn(90, h, 64, dt=dt, seed=h + i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    cu = torch.tensor([0, 40, 90], device=DEV, dtype=torch.int32)
    return (lambda *t: cp.causal_attention(*t, cu)), leaves


def _norm(dt=torch.bfloat16):
    leaves = [_randn(30, 96, dt=dt).requires_grad_(), _randn(96, dt=torch.float32, seed=1).requires_grad_(),
              _randn(96, dt=torch.float32, seed=2).requires_grad_(), _randn(30, 96, dt=dt, seed=3).requires_grad_()]
    return (lambda x, w, b, r: cp.layer_norm(x, w, b, residual=r)), leaves


def _plain_norm(dt=torch.bfloat16):
    f, leaves = _norm(dt)
    return (lambda x, w, b: cp.layer_norm(x, w, b)), leaves[:3]


OPS = [_attention, _norm, _plain_norm]


def _outs(y):
    return list(y) if isinstance(y, tuple) else [y]


@gpu
@pytest.mark.parametrize("make", OPS)
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls(make, backend):
    f, leaves = make()
    outs = _outs(f(*leaves))
    dys = [_randn(*o.shape, seed=9 + i) for i, o in enumerate(outs)]
    want = outs + list(torch.autograd.grad(outs, leaves, dys))
    g = torch.compile(f, fullgraph=True, backend=backend)
    got = _outs(g(*leaves))
    got += list(torch.autograd.grad(got, leaves, dys))
    cp.check_device_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(_outs(g(*leaves)), want))


@gpu
def test_compiled_decode():
    q, k, v = _randn(3, 4, 64), _randn(3, 70, 2, 64, seed=1), _randn(3, 70, 2, 64, seed=2)
    n = torch.tensor([70, 0, 13], device=DEV, dtype=torch.int32)
    got = torch.compile(cp.decode_attention, fullgraph=True, backend="aot_eager")(q, k, v, n)
    assert torch.equal(got, cp.decode_attention(q, k, v, n))


@gpu
@pytest.mark.parametrize("make", OPS)
def test_backward_of_an_ordinary_forward_by_other_means(make):
    """A dispatch mode around the backward sees the custom op; a batch of output gradients is taken one by one."""
    f, leaves = make()
    outs = _outs(f(*leaves))
    dys = [_randn(3, *o.shape, seed=9 + i) for i, o in enumerate(outs)]
    plain = [torch.autograd.grad(outs, leaves, [d[i] for d in dys], retain_graph=True) for i in range(3)]
    mode = _Seen()
    with mode:
        seen = torch.autograd.grad(outs, leaves, [d[0] for d in dys], retain_graph=True)
    assert any("_backward" in o and "prism_b200" in o for o in mode.ops)
    batched = torch.autograd.grad(outs, leaves, dys, is_grads_batched=True)
    cp.check_device_status()
    for i, b in enumerate(batched):
        assert torch.equal(seen[i], plain[0][i]) and torch.equal(b, torch.stack([p[i] for p in plain]))


@gpu
@pytest.mark.parametrize("make", OPS)
def test_dispatch_modes_see_the_whole_call(make):
    f, leaves = make()
    outs = _outs(f(*leaves))
    dys = [_randn(*o.shape, seed=9 + i) for i, o in enumerate(outs)]
    want = outs + list(torch.autograd.grad(outs, leaves, dys))
    mode = _Seen()
    with mode:
        got = _outs(f(*leaves))
        got += list(torch.autograd.grad(got, leaves, dys))
    assert sum("prism_b200" in o for o in mode.ops) == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_vmap():
    """One call for each entry of the mapped dimension."""
    q, k, v = (_randn(3, 50, h, 64, seed=h) for h in (4, 2, 2))
    got = torch.func.vmap(cp.causal_attention)(q, k, v)
    assert torch.equal(got, torch.stack([cp.causal_attention(*t) for t in zip(q, k, v)]))
    x, w = _randn(3, 20, 48), _randn(48)
    y, s = torch.func.vmap(lambda a, b: cp.layer_norm(a, w, None, residual=b))(x, x.flip(0))
    want = [cp.layer_norm(a, w, None, residual=b) for a, b in zip(x, x.flip(0))]
    assert torch.equal(y, torch.stack([t[0] for t in want])) and torch.equal(s, torch.stack([t[1] for t in want]))
    assert torch.equal(torch.func.vmap(lambda a: cp.layer_norm(a, w))(x), cp.layer_norm(x, w))
    cache = _randn(3, 2, 40, 2, 64)
    n = torch.tensor([[40, 3], [0, 1], [17, 40]], device=DEV, dtype=torch.int32)
    qd = _randn(3, 2, 4, 64)
    got = torch.func.vmap(cp.decode_attention)(qd, cache, cache, n)
    assert torch.equal(got, torch.stack([cp.decode_attention(a, b, b, c) for a, b, c in zip(qd, cache, n)]))
    cp.check_device_status()


def _decode():
    n = torch.tensor([70, 0, 13], device=DEV, dtype=torch.int32)
    return (lambda q, k, v: cp.decode_attention(q, k, v, n)), [_randn(3, 4, 64), _randn(3, 70, 2, 64, seed=1), _randn(3, 70, 2, 64, seed=2)]


@gpu
@pytest.mark.parametrize("make", [*OPS, _decode])
def test_tangents_are_refused_not_dropped(make):
    """No forward-mode formula exists: an error, not a derivative of zero; inputs without tangents pass, also inside a level."""
    f, leaves = make()
    leaves = [t.detach() for t in leaves]
    want = _outs(f(*leaves))
    fw = torch.autograd.forward_ad
    for i in range(len(leaves)):
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(*[fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(leaves)])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: f(*leaves[:i], t, *leaves[i + 1:]), (leaves[i],), (torch.ones_like(leaves[i]),))
    with fw.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(_outs(f(*leaves)), want))


@gpu
@pytest.mark.parametrize("make", OPS)
def test_no_second_derivative(make):
    f, leaves = make()
    y = _outs(f(*leaves))[0]
    g, = torch.autograd.grad((y.float() ** 2).sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().pow(2).sum().backward()


@gpu
@pytest.mark.parametrize("make", OPS)
@pytest.mark.parametrize("grad", [False, True])
def test_views_with_the_negative_bit(make, grad):
    f, leaves = make()
    leaves = [t.requires_grad_(grad) for t in leaves]
    want = _outs(f(*leaves))
    flipped = [torch._neg_view(-t.detach()).requires_grad_(grad) for t in leaves]
    assert flipped[0].is_neg()
    got = _outs(f(*flipped))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if grad:
        dys = [_randn(*o.shape, seed=9 + i) for i, o in enumerate(want)]
        neg = [torch._neg_view(-d) for d in dys]
        for a, b in zip(torch.autograd.grad(want, leaves, dys, retain_graph=True), torch.autograd.grad(want, leaves, neg)):
            assert torch.equal(a, b)
    cp.check_device_status()


@gpu
@pytest.mark.parametrize("make", OPS)
@pytest.mark.parametrize("hooks", [(lambda t: torch.stack((t, t), -1), lambda s: s[..., 0]),
                                   (lambda t: torch.cat((t.reshape(-1)[:1], t.reshape(-1))), None)])
def test_saved_tensors_of_another_layout(make, hooks):
    """Hooks that hand back every second element of a wider buffer, and one element behind a buffer's start."""
    pack, unpack = hooks
    if unpack is None:
        pack, unpack = lambda t, p=pack: (p(t), t.shape), lambda s: s[0][1:].view(s[1])
    f, leaves = make()
    outs = _outs(f(*leaves))
    dys = [_randn(*o.shape, seed=9 + i) for i, o in enumerate(outs)]
    want = torch.autograd.grad(outs, leaves, dys)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        outs = _outs(f(*leaves))
    got = torch.autograd.grad(outs, leaves, dys)
    cp.check_device_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
