"""GPU: channels of a head past the axes of a rotation stay as they are, whatever is in them."""
from __future__ import annotations

import pytest
import torch

from helpers import announce
from sihc_hip import body

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
# heads, key heads, channels, axes: lanes that turn all, some and none of their channels, and an odd last one;
# many heads (a token a wave) and few
CASES = [(2, 1, 64, (16, 20)), (24, 12, 64, (16, 20)), (3, 3, 67, (22, 20, 22)), (40, 40, 67, (22, 20, 22)),
         (2, 2, 5, ()), (3, 1, 130, (64, 6)), (16, 16, 72, (36, 36)), (200, 100, 7, (2, 2))]


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def same(a, b):
    """The same values, any NaN for a NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def positions(count):
    return (torch.arange(9 * count, dtype=torch.int32).reshape(9, count) - 4).cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotation(case, dtype):
    heads, _, dim, axes = case
    announce(f"axis_rotary {case} {dtype}")
    at, turned = positions(len(axes)), sum(axes)
    x, grad = normal(2, 9, heads, dim).to(dtype), normal(2, 9, heads, dim, seed=1).to(dtype)
    want = body.axis_rotary(x.cuda(), at, axes)
    for bad in (INF, -INF, NAN):
        for channel in {turned, dim - 1, (turned + dim) // 2}:
            if channel == dim:
                continue  # (nothing is past the axes)
            worse = x.clone()
            if channel >= turned:
                worse[:, ::2, :, channel] = bad
            lx = worse.cuda().requires_grad_()
            y = body.axis_rotary(lx, at, axes)
            assert same(y[..., turned:].cpu(), worse[..., turned:])  # the tail is a copy
            assert torch.equal(y[..., :turned], want[..., :turned])
            up = grad.clone()
            if channel >= turned:
                up[:, ::2, :, channel] = bad
            (dx,) = torch.autograd.grad(y, lx, up.cuda())
            (clean,) = torch.autograd.grad(body.axis_rotary(lx, at, axes), lx, grad.cuda())
            assert same(dx[..., turned:].cpu(), up[..., turned:])
            assert torch.equal(dx[..., :turned], clean[..., :turned])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_norm(case, dtype):
    """An infinite value past the axes: its own result is inf / inf, the head's others are finite / inf. A weight
    or a gradient that is not finite there reaches no other channel's result."""
    heads, kv_heads, dim, axes = case
    announce(f"qk_norm_rotary {case} {dtype}")
    at, turned = positions(len(axes)), sum(axes)
    if turned == dim:
        return
    q, k = normal(2, 9, heads, dim).to(dtype), normal(2, 9, kv_heads, dim, seed=1).to(dtype)
    w = 1 + 0.1 * normal(dim, seed=2)
    for channel in {turned, dim - 1, (turned + dim) // 2}:
        bad = q.clone()
        bad[1, 3, :, channel] = INF
        got, other = body.qk_norm_rotary(bad.cuda(), k.cuda(), w.cuda(), w.cuda(), at, axes)
        want, _ = body.qk_norm_rotary(q.cuda(), k.cuda(), w.cuda(), w.cuda(), at, axes)
        want = want.clone()
        want[1, 3] = 0
        want[1, 3, :, channel] = NAN
        assert same(got, want), channel
        rest = [c for c in range(dim) if c != channel]
        worse = w.clone()
        worse[channel] = NAN
        want, _ = body.qk_norm_rotary(q.cuda(), k.cuda(), w.cuda(), w.cuda(), at, axes)
        got, _ = body.qk_norm_rotary(q.cuda(), k.cuda(), worse.cuda(), w.cuda(), at, axes)
        assert torch.equal(got[..., rest], want[..., rest]) and got[..., channel].isnan().all()
        # the weights' gradients are sums over heads of one channel's own terms
        grad = normal(2, 9, heads, dim, seed=3).to(dtype)
        sums = []
        for value in (1.0, NAN):
            up = grad.clone()
            up[0, 0, 0, channel] = value
            lw = w.cuda().requires_grad_()
            y, _ = body.qk_norm_rotary(q.cuda(), k.cuda(), lw, w.cuda(), at, axes)
            sums.append(torch.autograd.grad(y, lw, up.cuda())[0])
        assert torch.equal(sums[0][rest], sums[1][rest]) and sums[1][channel].isnan()
