"""GPU: group norm where a few values are far from the rest.

Bounds: fp32 1e-5 in relative L2, as for ordinary inputs. A value D deviations away puts D^2 into its
group's sum of squares, so sums that are taken about anything but an outlier lose no digits to it: a
thread's 32 terms carry at most 32 * 2^-24 = 2e-6 of it."""
from __future__ import annotations

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip import group_norm_act
from test_gpu_conditioning import norm_oracle, normal

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# slices of a block, and images in whole rows: 4.7 MB in 32 groups, one group of all, rows of odd width
@pytest.mark.parametrize("far", [100.0, 3e2, 3e3, 3e4])
@pytest.mark.parametrize("pixels,channels,groups", [(256, 64, 4), (1024, 1152, 32), (16384, 128, 4), (40000, 33, 1)])
def test_group_norm_keeps_its_digits_beside_an_outlier(pixels, channels, groups, far):
    announce(f"group norm of {pixels}x{channels} in {groups} groups, the first value of each {far:g} deviations away")
    x = normal((2, pixels, channels), F32, 40)
    x[:, 0, ::channels // groups] = far
    x.requires_grad_()
    w, b = normal((channels,), F32, 41, mean=1.0, std=0.2).requires_grad_(), normal((channels,), F32, 42).requires_grad_()
    grad = normal(x.shape, F32, 43)
    for act in ("none", "silu"):
        y = group_norm_act(x, w, b, groups, 1e-6, act)
        got = (y, *torch.autograd.grad(y, (x, w, b), grad))
        for name, g, e in zip(("y", "dx", "dw", "db"), got, norm_oracle(x, w, b, groups, 1e-6, act, grad)):
            assert rel_l2(g.cpu(), e) <= 1e-5, (act, name)
    # the other values, which are small beside the outliers, by themselves and group by group
    one, zero = torch.ones_like(w), torch.zeros_like(w)
    y, want = (t.detach().double().cpu().reshape(2, pixels, groups, -1)[:, 1:]
               for t in (group_norm_act(x, one, zero, groups, 1e-6, "none"),
                         norm_oracle(x, one, zero, groups, 1e-6, "none", grad)[0]))
    assert float(((y - want).square().sum((1, 3)) / want.square().sum((1, 3))).sqrt().max()) <= 1e-5


# a mean of about 8 deviations is where the variance is taken again, about the mean; images and groups on both sides of
# that line, in blocks of one group, of several, and of many
@pytest.mark.parametrize("batch,pixels,channels,groups", [(600, 64, 128, 32), (600, 256, 128, 16), (300, 100, 64, 64),
                                                          (8, 256, 64, 2)])
def test_group_norm_of_means_about_eight_deviations(batch, pixels, channels, groups):
    announce(f"group norm {batch}x{pixels}x{channels} in {groups} groups, means about 8 deviations")
    mean = normal((batch, 1, groups, 1), F32, 48, mean=8.0, std=0.2).repeat_interleave(channels // groups, 3)
    x = (normal((batch, pixels, channels), F32, 49) + mean.reshape(batch, 1, channels)).to(BF16).requires_grad_()
    w, b = normal((channels,), BF16, 50, mean=1.0).requires_grad_(), normal((channels,), BF16, 51).requires_grad_()
    grad = normal(x.shape, BF16, 52)
    y = group_norm_act(x, w, b, groups)
    got = (y, *torch.autograd.grad(y, (x, w, b), grad))
    for name, g, e in zip(("y", "dx", "dw", "db"), got, norm_oracle(x, w, b, groups, 1e-6, "silu", grad)):
        assert rel_l2(g.cpu(), e) <= 3.3e-3, name
    assert torch.equal(group_norm_act(x, w, b, groups), y)


# a deviation whose square passes fp32: the variance is infinite, its reciprocal root zero, and y = act(bias)
@pytest.mark.parametrize("pixels,channels,groups", [(256, 36, 1), (16384, 36, 1), (1024, 1152, 32)])
@pytest.mark.parametrize("half", [False, True], ids=["two", "half"])
def test_group_norm_of_squares_past_fp32(pixels, channels, groups, half):
    announce(f"group norm of {pixels}x{channels} in {groups} groups, squares past fp32")
    x = normal((1, pixels, channels), F32, 44)
    if half:
        x[:, torch.arange(pixels, device="cuda") % 32 > 15] = 5e19
    else:
        x[:, 0, 1::channels // groups], x[:, 1, 5::channels // groups] = -2e19, 2e19
    x.requires_grad_()
    w, b = normal((channels,), F32, 45, mean=1.0).requires_grad_(), normal((channels,), F32, 46).requires_grad_()
    grad = normal(x.shape, F32, 47)
    y = group_norm_act(x, w, b, groups)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), grad)
    bias = b.detach().double().requires_grad_()
    want = torch.nn.functional.silu(bias).expand(x.shape)
    assert rel_l2(y, want) <= 1e-6
    assert not dx.any() and not dw.any()
    assert rel_l2(db, torch.autograd.grad(want, bias, grad.double())[0]) <= 1e-5
