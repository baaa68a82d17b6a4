"""GPU: the conditioning operators under compiled autograd, checkpointing, vmap, functional gradients, forward-mode
tangents, subclasses and modes in the backward: what has to see the registered op does, with its results."""
from __future__ import annotations

import pytest
import torch
import torch._dynamo.compiled_autograd
import torch.autograd.forward_ad as fw
import torch.utils.checkpoint
from torch.utils._python_dispatch import TorchDispatchMode

from sihc_hip import cross_attention, embedding_lookup, group_norm_act

pytestmark = pytest.mark.gpu
NAMES = ["embed", "norm", "attend", "attend_bf16"]


def calls(name):
    """(the public call, its differentiable arguments)"""
    g = torch.Generator().manual_seed(1)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    if name == "embed":
        ids = torch.randint(0, 50, (4, 9), generator=g).cuda()
        return (lambda t: embedding_lookup(t, ids, 2.0, 3, validate=False)), [normal(50, 24)]
    if name == "norm":
        return (lambda *t: group_norm_act(*t, 4)), [normal(2, 5, 5, 24), normal(24), normal(24)]
    dtype = torch.bfloat16 if name.endswith("bf16") else torch.float32
    n = torch.tensor([30, 7], dtype=torch.int32, device="cuda")
    return ((lambda *t: cross_attention(*t, n, validate=False)),
            [normal(2, 11, 4, 40, dtype=dtype), normal(2, 30, 2, 40, dtype=dtype), normal(2, 30, 2, 40, dtype=dtype)])


def leaves_of(values):
    return [v.clone().requires_grad_() for v in values]


def grads_of(call, values):
    leaves = leaves_of(values)
    out = call(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]


def equal(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_compiled_autograd(name):
    call, values = calls(name)
    want, leaves = grads_of(call, values), leaves_of(values)
    out = call(*leaves)
    torch._dynamo.reset()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="eager")):
        torch.autograd.backward(out, torch.ones_like(out))
    assert equal([out.detach(), *(t.grad for t in leaves)], want)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_checkpointing(name, reentrant):
    call, values = calls(name)
    want = grads_of(call, values)
    leaves = leaves_of(values)
    out = torch.utils.checkpoint.checkpoint(call, *leaves, use_reentrant=reentrant)
    torch.autograd.backward(out, torch.ones_like(out))
    assert equal([out.detach(), *(t.grad for t in leaves)], want)


@pytest.mark.parametrize("name", NAMES)
def test_vmap(name):
    call, values = calls(name)
    with torch.no_grad():
        want = [call(factor * values[0], *values[1:]) for factor in (1, 2)]
        got = torch.func.vmap(lambda t: call(t, *values[1:]))(torch.stack([values[0], 2 * values[0]]))
    assert equal(list(got), want)


@pytest.mark.parametrize("name", NAMES)
def test_functional_gradients_are_refused(name):
    """torch.func has no rule for the registered gradients of custom ops, here as for every op of the package."""
    call, values = calls(name)
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.grad(lambda t: call(t, *values[1:]).float().sum())(values[0])


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_not_dropped_silently_in_a_native_call(name):
    """A forward-mode tangent reaches the registered op, which has no rule for it: the value is right, or it raises."""
    call, values = calls(name)
    with torch.no_grad():
        want = call(*values)
    with fw.dual_level():
        try:
            out = call(fw.make_dual(values[0], torch.ones_like(values[0])), *values[1:])
        except (RuntimeError, NotImplementedError):
            return
        assert torch.equal(fw.unpack_dual(out).primal, want)


@pytest.mark.parametrize("name", NAMES)
def test_modes_in_the_backward_subclasses_and_parameters(name):
    call, values = calls(name)
    want, seen = grads_of(call, values), []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves = leaves_of(values)
    out = call(*leaves)
    with Log():
        got = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert any("sihc" in s and "backward" in s for s in seen) and equal(list(got), want[1:])

    class Sub(torch.Tensor):
        pass

    with torch.no_grad():
        out = call(values[0].as_subclass(Sub), *values[1:])
        assert isinstance(out, Sub) and torch.equal(out.as_subclass(torch.Tensor), want[0])
        assert torch.equal(call(torch.nn.Parameter(values[0]), *values[1:]), want[0])


@pytest.mark.parametrize("name", NAMES[1:])  # (the embedding's gradient reads its ids alone)
def test_saved_tensors_changed_in_place_are_noticed(name):
    call, values = calls(name)
    leaves = [v.clone().requires_grad_() for v in values]
    moved = [v * 1.0 for v in leaves]
    out = call(*moved)
    with torch.no_grad():
        moved[0].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))
