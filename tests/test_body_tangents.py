"""CPU: the body operators have no forward-mode derivative, and refuse a tangent instead of dropping it."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from sihc_hip import body

X, W, HEAD = torch.randn(3, 8, 16), torch.randn(16, 16), torch.randn(4)
AT, SEED = torch.arange(8, dtype=torch.int32).reshape(8, 1), torch.tensor([3])
CALLS = {
    "linear": lambda x: body.linear_act(x, W, None, "silu"),
    "linear weight": lambda x: body.linear_act(X, x[0, :8, :].reshape(8, 16), None, "silu"),
    "linear residual": lambda x: body.linear_act(X, W, residual=x),
    "linear of a part": lambda x: body._linear_act(x, W, None, "silu", None, None),
    "keywords": lambda x: body._linear_act_result(x=x, weight=W, bias=None, act="none", gate=None, residual=None),
    "heads": lambda x: body.qk_norm_rotary(X.view(3, 8, 4, 4), x.view(3, 8, 4, 4), HEAD, HEAD, AT, (4,)),
    "rotary": lambda x: body.axis_rotary(x.view(3, 8, 4, 4), AT, (4,)),
    "dropout": lambda x: body.dropout(x, 0.4, SEED, 2),
    "dropout residual": lambda x: body.dropout(X, 0.4, SEED, 2, x),
}
refused = pytest.raises(NotImplementedError, match="forward-mode")


@pytest.mark.parametrize("name", CALLS)
def test_dual_tensors(name):
    with fw.dual_level(), refused:
        CALLS[name](fw.make_dual(X, torch.ones_like(X)))
    with fw.dual_level(), torch.no_grad(), refused:
        CALLS[name](fw.make_dual(X, torch.ones_like(X)))


@pytest.mark.parametrize("name", CALLS)
def test_functional_transforms(name):
    call = CALLS[name]
    ones = torch.ones_like(X)
    with refused:
        torch.func.jvp(call, (X,), (ones,))
    with refused:
        torch.func.jacfwd(call)(X)
    with refused:  # a batch of tangents
        torch.func.vmap(lambda t: torch.func.jvp(call, (X,), (t,)))(torch.stack([ones, ones]))
    with refused:  # a batch inside the differentiated function
        torch.func.jvp(lambda a: torch.func.vmap(lambda b: call(b))(torch.stack([a, a])), (X,), (ones,))
    with refused:  # the outer of two directions
        torch.func.jvp(lambda a: torch.func.jvp(lambda b: (call(a), b)[1], (X,), (ones,))[1], (X,), (ones,))


@pytest.mark.parametrize("name", CALLS)
def test_what_has_no_tangent_is_not_refused(name):
    """These calls come as far as the check of the device."""
    call = CALLS[name]
    device = pytest.raises(ValueError, match="CUDA device")
    with device:
        call(X)
    with fw.dual_level():
        fw.make_dual(X.clone(), torch.ones_like(X))
        with device:
            call(X)
    with device:
        torch.func.jvp(lambda a: (call(X), a)[1], (X,), (torch.ones_like(X),))
    with device:
        torch.func.jvp(lambda a: (call(a.detach()), a)[1], (X,), (torch.ones_like(X),))


@pytest.mark.parametrize("name", ["linear", "heads", "rotary", "dropout"])
def test_compiled(name):
    def both(x):
        return torch.func.jvp(CALLS[name], (x,), (torch.ones_like(x),))

    torch._dynamo.reset()
    with pytest.raises(Exception, match="forward-mode"):
        torch.compile(both, backend="aot_eager")(X)
