"""GPU: the native dispatch of the conditioning operators gives the registered ops' results and
gradients bit for bit, and leaves to them whatever has to see the op."""
from __future__ import annotations

import pytest
import torch
from torch.library import CustomOpDef
from torch.utils._python_dispatch import TorchDispatchMode

from sihc_hip import _native, conditioning

pytestmark = pytest.mark.gpu


def cases():
    g = torch.Generator().manual_seed(0)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    ids = torch.randint(0, 50, (4, 9), generator=g).cuda()
    kv = normal(2, 30, 2, 2, 40, dtype=torch.bfloat16)
    n = torch.tensor([30, 7], dtype=torch.int32).cuda()
    yield conditioning._embedding_lookup, [normal(50, 24)], (ids, 2.0, 3)
    yield conditioning._embedding_lookup, [normal(50, 24, dtype=torch.bfloat16)], (ids.int(), 2, -1)
    yield conditioning._group_norm_act, [normal(2, 5, 5, 24, dtype=torch.bfloat16), normal(24), normal(24)], (4, 1e-6, "silu")
    yield conditioning._group_norm_act, [normal(2, 25, 24), normal(24), normal(24)], (4, 1e-6, "none")
    yield conditioning._cross_attention, [normal(2, 11, 4, 40, dtype=torch.bfloat16), kv[:, :, 0], kv[:, :, 1]], (n, 0.2, True)
    yield conditioning._cross_attention, [normal(2, 11, 4, 40), normal(2, 3, 2, 40), normal(2, 3, 2, 40)], (None, 0.2, True)


def passed(op, leaves, rest, call):
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = call(*leaves, *rest)
    first = out[0] if isinstance(out, tuple) else out
    grads = torch.autograd.grad(first, leaves, torch.ones_like(first))
    return [t.detach() for t in (out if isinstance(out, tuple) else (out,))] + list(grads)


def test_same_bits_as_the_registered_ops(monkeypatch):
    for op, leaves, rest in cases():
        taken = []
        load = op._sihc_load
        monkeypatch.setattr(op, "_sihc_entry", None)
        monkeypatch.setattr(op, "_sihc_load", lambda: (lambda e: lambda *a: taken.append(e(*a)) or taken[-1])(load()))
        native = passed(op, leaves, rest, op)
        assert taken and taken[0] is not NotImplemented, op
        plain = passed(op, leaves, rest, lambda *a: CustomOpDef.__call__(op, *a))
        assert len(native) == len(plain) and all(torch.equal(a, b) for a, b in zip(native, plain)), op
        with torch.no_grad():  # (train=True: all outputs are filled)
            again = op(*leaves, *rest)
        again = again if isinstance(again, tuple) else (again,)
        assert all(torch.equal(a, b) for a, b in zip(again, native))
        monkeypatch.undo()


def test_stats_carry_no_gradient_and_unused_inputs_none():
    x = torch.randn(2, 4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda")
    y, stats = conditioning._group_norm_act(x, w, w, 2, 1e-6, "silu")
    assert y.requires_grad and not stats.requires_grad
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape  # (only x asks for a gradient)
    q = torch.randn(1, 2, 1, 8, device="cuda", requires_grad=True)
    out, stats, low = conditioning._cross_attention(q, q.detach(), q.detach(), None, 1.0, True)
    assert out.requires_grad and not stats.requires_grad and not low.requires_grad
    # a call that is not to be differentiated keeps nothing, and says so when it is
    out, stats, low = conditioning._cross_attention(q.detach(), q.detach(), q.detach(), None, 1.0, False)
    assert not out.requires_grad and not stats.numel() and not low.numel()


def test_modes_hooks_and_bad_arguments_reach_the_registered_ops():
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for op, leaves, rest in cases():
        seen.clear()
        with Watch():
            op(*leaves, *rest)
        assert any(op._qualname.replace("::", ".") in name for name in seen), (op, seen)
        with pytest.raises((ValueError, RuntimeError)):
            op(*[t.double() for t in leaves], *rest)

        def shrink(t):  # an unpack hook that gives back something else: refused, never launched
            return t[..., :1] if t.ndim > 1 else t

        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, shrink):
            with pytest.raises((ValueError, RuntimeError)):
                passed(op, leaves, rest, op)


def test_entries_are_the_modules_own():
    for name, op in (("embedding_lookup", conditioning._embedding_lookup),
                     ("group_norm_act", conditioning._group_norm_act),
                     ("cross_attention", conditioning._cross_attention)):
        assert _native.module().entry(name, op._qualname) is not None
