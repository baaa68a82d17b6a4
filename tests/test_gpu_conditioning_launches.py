"""GPU: sizes that take more threads than one launch has (2^32 in a dimension): millions of images of a few
pixels, and of table rows of one channel."""
from __future__ import annotations

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip import embedding_lookup, group_norm_act

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def test_group_norm_of_more_small_images_than_a_launch_takes():
    """One slice of 256 threads each. In bf16: the weight gradient is a chain of millions of fp32 sums."""
    shape, groups = (2**24 + 5, 2, 2), 1
    announce(f"group norm of {shape} in {groups} groups")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=gen).requires_grad_()
    w = torch.empty(shape[-1], dtype=BF16, device="cuda").normal_(1.0, 0.2, generator=gen).requires_grad_()
    b = torch.empty(shape[-1], dtype=BF16, device="cuda").normal_(generator=gen).requires_grad_()
    grad = torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=gen)
    y = group_norm_act(x, w, b, groups, 1e-5, "none")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), grad)
    axes = tuple(range(1, len(shape)))
    sums = torch.zeros(2, shape[-1], dtype=torch.float64, device="cuda")
    step = 1 << 20
    for i in range(0, shape[0], step):
        v, g = x.detach()[i:i + step].float(), grad[i:i + step].float()
        centred = v - v.mean(axes, keepdim=True)
        r = (centred.square().mean(axes, keepdim=True) + 1e-5).rsqrt()
        h = centred * r
        wg = g * w.detach().float()
        want = r * (wg - wg.mean(axes, keepdim=True) - h * (wg * h).mean(axes, keepdim=True))
        if i == 0 or i + step >= shape[0] or (i // step) % 4 == 3:  # (both ends, and where one launch ends)
            assert rel_l2(y[i:i + step], h * w.detach().float() + b.detach().float()) <= 3.3e-3
            assert rel_l2(dx[i:i + step], want) <= 3.3e-3
        sums += torch.stack([(g * h).flatten(0, -2).sum(0, dtype=torch.float64), g.flatten(0, -2).sum(0, dtype=torch.float64)])
    assert rel_l2(dw, sums[0]) <= 3.3e-3 and rel_l2(db, sums[1]) <= 3.3e-3


def test_group_norm_of_more_chunks_than_a_launch_takes():
    """Images in whole rows, 34 GB of them: the ends of both launches are what they are by themselves."""
    announce("group norm of 16,385 images of 4096 x 255")
    x = torch.zeros(16385, 4096, 255, dtype=BF16, device="cuda")
    some = [0, 16381, 16382, 16383, 16384]
    gen = torch.Generator(device="cuda").manual_seed(2)
    few = torch.empty(len(some), 4096, 255, dtype=BF16, device="cuda").normal_(generator=gen)
    for i, v in zip(some, few):
        x[i] = v
    w = torch.empty(255, dtype=F32, device="cuda").normal_(1.0, 0.2, generator=gen).requires_grad_()
    b = torch.empty(255, dtype=F32, device="cuda").normal_(generator=gen).requires_grad_()
    x.requires_grad_(), few.requires_grad_()
    want = group_norm_act(few, w, b, 5)
    y = group_norm_act(x, w, b, 5)
    assert torch.equal(y[some], want)
    del y
    y = group_norm_act(x, w, b, 5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), x.detach())
    dx0, dw0, db0 = torch.autograd.grad(want, (few, w, b), few.detach())
    assert torch.equal(dx[some], dx0) and not dx[1:100].any()
    assert rel_l2(dw, dw0) <= 1e-5 and rel_l2(db, db0) <= 1e-5


def test_embedding_gradient_of_more_rows_than_a_launch_takes():
    rows = 2**27 + 11
    announce(f"embedding of {rows} rows of one channel")
    table = torch.zeros(rows, 1, dtype=BF16, device="cuda").requires_grad_()
    ids = torch.tensor([0, 5, rows - 1, rows - 1, 2**27 - 8, 2**27 - 1, 2**27, rows - 2], device="cuda")
    grad = torch.tensor([[1.0], [2], [3], [4], [5], [6], [7], [8]], dtype=BF16, device="cuda")
    (dt,) = torch.autograd.grad(embedding_lookup(table, ids, 2.0), table, grad)
    want = {0: 2.0, 5: 4.0, rows - 1: 14.0, 2**27 - 8: 10.0, 2**27 - 1: 12.0, 2**27: 14.0, rows - 2: 16.0}
    assert {int(i): float(dt[i, 0]) for i in dt.flatten().nonzero().flatten()} == want
