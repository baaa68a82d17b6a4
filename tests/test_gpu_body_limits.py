"""GPU: sizes at the documented limits of the body operators, with small rows so that they fit the card."""
from __future__ import annotations

import pytest
import torch

from helpers import announce
from sihc_hip import body

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,inner,outer,act", [(2 ** 30, 1, 1, "none"), (2 ** 29 + 5, 3, 2, "swiglu"), (2 ** 26 + 1, 8, 300, "swiglu")],
                         ids=str)
def test_as_many_rows_as_fit(rows, inner, outer, act):
    """A product whose cheapest tiles are more than a launch takes has others."""
    wide = 2 * outer if act == "swiglu" else outer
    if torch.cuda.mem_get_info()[0] < rows * (inner + outer) * 4 + (8 << 30):
        pytest.skip("needs more memory")
    announce(f"linear_act of {rows} rows of {inner} to {outer} {act} fp32")
    x = torch.zeros(rows, inner, device="cuda", dtype=F32)
    g = torch.Generator().manual_seed(0)
    w, b, tail = (torch.randn(*s, generator=g).cuda() for s in ((wide, inner), (wide,), (500, inner)))
    x[-500:] = tail
    y = body.linear_act(x, w, b, act)
    few = x[:70].contiguous(), x[-500:].contiguous()
    h = [(v.double() @ w.double().t() + b.double()) for v in few]
    want = [v if act == "none" else torch.nn.functional.silu(v[:, :outer]) * v[:, outer:] for v in h]
    for got, exact in ((y[:70], want[0]), (y[-500:], want[1])):
        assert float((got.double() - exact).abs().max()) <= 2.0 ** -16 * float(exact.abs().max())
    del y


def test_as_many_tokens_as_a_launch_takes():
    """The most tokens of heads of which a wave takes one token."""
    heads, dim = 129, 2
    tokens = (2 ** 26 - 4)
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    announce(f"axis_rotary of {tokens} tokens")
    x = torch.ones(1, 1, heads, dim, device="cuda", dtype=BF16).expand(1, tokens, heads, dim)
    at = torch.zeros(tokens, 1, device="cuda", dtype=torch.int32)
    at[-1] = 7
    y = body.axis_rotary(x, at, (2,))
    assert torch.equal(y[:, :1000], x[:, :1000]) and torch.equal(y[:, -1000:-1], x[:, -1000:-1])
    c, s = torch.tensor(7.0, dtype=torch.float64).cos(), torch.tensor(7.0, dtype=torch.float64).sin()
    last = y[0, -1].double().cpu()
    want = torch.stack([c - s, c + s]).expand(heads, dim)
    assert ((last - want).abs() <= torch.finfo(BF16).eps / 2 * want.abs() * 1.001 + 2.0 ** -20).all()
    with pytest.raises(ValueError, match="at most 67108860 tokens"):
        body.axis_rotary(x[:, :1].expand(1, tokens + 1, heads, dim), torch.zeros(tokens + 1, 1, device="cuda", dtype=torch.int32), (2,))
