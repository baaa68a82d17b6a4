"""GPU: sizes at the documented limits of the body operators, with small rows so that they fit the card."""
from __future__ import annotations

import pytest
import torch

from helpers import announce
from sihc_hip import body

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


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
