"""GPU: forward-mode tangents are refused by the body operators' calls and backward passes, on the native path and on
the registered ops; what carries none keeps its native call."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.library import CustomOpDef

from sihc_hip import body

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).cuda()


def calls():
    w, head = normal(16, 16, seed=1), normal(4, seed=2)
    at, key = torch.arange(8, dtype=torch.int32, device="cuda").reshape(8, 1), torch.tensor([3], device="cuda")
    other = normal(3, 8, 4, 4, seed=3)
    return {
        "linear": (body._linear_act, lambda x: (x, w, None, "silu", None, None)),
        "heads": (body._qk_norm_rotary, lambda x: (x.view(3, 8, 4, 4), other, head, head, at, [4], 1e4, 1e-6)),
        "rotary": (body._axis_rotary, lambda x: (x.view(3, 8, 4, 4), at, [4], 1e4, False)),
        "dropout": (body._dropout, lambda x: (x, 0.4, key, 2, None)),
    }


def first(out):
    return out[0] if isinstance(out, tuple) else out


NAMES = ["linear", "heads", "rotary", "dropout"]


@pytest.mark.parametrize("name", NAMES)
def test_calls(name):
    op, arguments = calls()[name]
    x = normal(3, 8, 16)
    want = first(op(*arguments(x)))
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        assert torch.equal(first(op(*arguments(x))), want)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            op(*arguments(dual))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: first(op(*arguments(t))), (x,), (torch.ones_like(x),))
    assert torch.equal(first(op(*arguments(x))), want)


@pytest.mark.parametrize("registered", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_backward_passes(name, registered):
    op, arguments = calls()[name]
    x = normal(3, 8, 16).requires_grad_()
    out = first(CustomOpDef.__call__(op, *arguments(x)) if registered else op(*arguments(x)))
    (want,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
    with fw.dual_level():
        (got,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, x, fw.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    (got,) = torch.autograd.grad(out, x, torch.ones_like(out))
    assert torch.equal(got, want)


def test_a_batch_of_gradients_still_passes():
    op, arguments = calls()["rotary"]
    x = normal(3, 8, 16).requires_grad_()
    out = op(*arguments(x))
    ups = torch.stack([torch.ones_like(out), 2 * torch.ones_like(out)])
    (got,) = torch.autograd.grad(out, x, ups, is_grads_batched=True, retain_graph=True)
    for up, g in zip(ups, got):
        assert torch.equal(torch.autograd.grad(out, x, up, retain_graph=True)[0], g)
