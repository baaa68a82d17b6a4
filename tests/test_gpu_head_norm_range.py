"""GPU: norms of heads over the whole range of the type, where neither the squares of the values nor the
reciprocal of their root fit fp32."""
from __future__ import annotations

import pytest
import torch

import body_reference as R
from helpers import announce
from sihc_hip import body

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
AXES = (2,)


def values(kind, dim, dtype):
    g = torch.Generator().manual_seed(dim)
    shape = (2, 3, 5, dim)
    sign = torch.randint(0, 2, shape, generator=g) * 2 - 1
    if kind == "subnormal":  # multiples of fp32's (bf16's) least value
        return (torch.randint(1, 100, shape, generator=g) * sign * (2.0 ** -149 if dtype == F32 else 2.0 ** -133)).to(dtype)
    if kind == "spread":
        return (torch.rand(shape, generator=g) * 3.3e38 * sign).to(dtype)
    return (torch.full(shape, kind) * sign).to(dtype)


# (kind, the size that the output's gradient has so that dx, its size over the values', is a normal number)
SIZES = [(2.0 ** 127, 2.0 ** 30), (2.0 ** 126, 2.0 ** 30), (3.2e38, 2.0 ** 30), ("spread", 2.0 ** 30), (2.0 ** 62.5, 1.0),
         (2.0 ** -46, 1.0), (2.0 ** -100, 2.0 ** -20), ("subnormal", 2.0 ** -40)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 128, 256])
@pytest.mark.parametrize("kind,size", SIZES, ids=str)
def test_heads_of_any_size(kind, size, dim, dtype):
    announce(f"qk_norm_rotary of {kind} {dim} {dtype}")
    x = values(kind, dim, dtype).cuda()
    x[:, 1, ::2] = values(1.0, dim, dtype)[:, 1, ::2].cuda()  # beside heads of size 1
    w = torch.linspace(0.5, 1.5, dim, device="cuda")
    at = torch.arange(3, dtype=torch.int32, device="cuda").reshape(3, 1)
    grad = (torch.randn(x.shape, generator=torch.Generator().manual_seed(1)) * size).to(dtype).cuda()
    for heads in (5, 1):
        lx, lw = x[:, :, :heads].contiguous().requires_grad_(), w.clone().requires_grad_()
        g = grad[:, :, :heads].contiguous()
        out, _ = body.qk_norm_rotary(lx, lx.detach(), lw, w, at, AXES, 1e4, 0.0)
        dx, dw = torch.autograd.grad(out, (lx, lw), g)
        want = R.heads(lx.cpu(), w.cpu(), at.cpu(), AXES, 1e4, 0.0, g.cpu())
        R.check(out, *want[0], f"result of {kind}, {dim} channels")
        # (a value below the least normal one is rounded to a multiple of the type's least, by half of it)
        least = 2.0 ** -134 if dtype == BF16 else 2.0 ** -150
        R.check(dx, want[1][0], want[1][1] + 1.01 * least, f"gradient of {kind}, {dim} channels")
        R.check(dw, *want[2], f"gradient of the weight, {kind}, {dim} channels")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_that_one_wave_shares(dtype):
    """Many heads (a token a wave) and few (several tokens a wave) give the largest values the same result."""
    x = values(2.0 ** 127, 64, dtype)[:, :, :1].expand(2, 3, 40, 64).contiguous().cuda()
    w = torch.ones(64, device="cuda")
    at = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    many = body.qk_norm_rotary(x, x, w, w, at, AXES, 1e4, 1e-6)[0]
    few = body.qk_norm_rotary(x[:, :, :1], x[:, :, :1], w, w, at, AXES, 1e4, 1e-6)[0]
    assert torch.equal(many[:, :, :1], few)
    assert float((few.double().abs() - 1).abs().max()) <= 8 * R.F32  # (a root of one step, and exact products)
