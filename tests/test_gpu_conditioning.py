"""GPU: embedding lookup, cross attention and group norm against their definitions in 64 bits.

Tolerances. fp32: relative L2 and largest error over the largest value at most 1e-5 (assert_parity).
bf16: one rounding of a result is at most 2^-8 of it, an rms of 2^-8 / sqrt(3) = 2.3e-3 at worst;
results that are products of operands rounded once more on the way (probabilities, score
gradients) carry two such errors, so relative L2 at most 5e-3, and 3.3e-3 for the others (one
rounding beside fp32 noise). Exact zeros and bits are asked for where the definition gives them.
"""
from __future__ import annotations

import math

import pytest
import torch

from helpers import announce, assert_parity, rel_l2
from sihc_hip import conditioning as C
from sihc_hip import cross_attention, embedding_lookup, group_norm_act

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
TYPES = [BF16, F32]


def near(actual, expected, dtype, what, bound):
    expected = expected.detach()
    if not expected.numel():
        assert actual.shape == expected.shape
        return
    assert_parity(actual, expected, dtype, what=what, kind="chained")
    if dtype == BF16 and float(expected.double().norm()) > 0:
        assert rel_l2(actual.cpu(), expected.cpu()) <= bound, what


def normal(shape, dtype, seed, mean=0.0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (mean + std * torch.randn(shape, generator=g, dtype=torch.float64)).to(dtype).cuda()


# ------------------------------------------------------------------------- embedding lookup
def embed_oracle(table, ids, scale, padding, grad):
    t, i = table.detach().double().cpu(), ids.long().cpu().flatten()
    out = (t[i] * scale).reshape(*ids.shape, t.shape[1])
    rows = grad.double().cpu().reshape(len(i), t.shape[1]) * scale
    if padding is not None:
        rows = rows * (i != padding % t.shape[0])[:, None]
    return out, torch.zeros_like(t).index_add_(0, i, rows)


# rows, channels, ids' shape, one row's share of the ids: both kernels of the gradient, one, two and
# three passes of the sort (11, 1000, 40000 and 1.1e6 rows), tiles and chunks with tails, rows of one
# channel, odd widths, a run through many chunks and one that ends at a chunk's edge
EMBED = [
    (1, 8, (5,), 0.0), (7, 1, (1,), 0.0), (11, 67, (3, 9), 0.5), (1001, 1152, (256,), 0.0),
    (1000, 130, (1024,), 0.3), (1000, 130, (1025,), 0.3), (1023, 64, (2, 1024), 0.0), (40000, 96, (4096,), 0.9),
    (5, 3, (3001,), 0.0), (3, 520, (6, 700), 0.0), (1100000, 8, (5000,), 0.2), (50, 1155, (2080,), 1.0), (17, 24, (0,), 0.0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,channels,shape,share", EMBED)
def test_embedding(rows, channels, shape, share, dtype):
    announce(f"embedding rows={rows} C={channels} ids={shape} share={share} {dtype}")
    g = torch.Generator().manual_seed(rows + channels)
    ids = torch.randint(0, rows, shape, generator=g)
    ids = torch.where(torch.rand(shape, generator=g) < share, rows // 2, ids)
    for id_type, padding in ((torch.int32, None), (torch.int64, rows // 2 - rows if rows > 4 else None)):
        table = normal((rows, channels), dtype, 1).requires_grad_()
        grad = normal((*shape, channels), dtype, 2)
        out = embedding_lookup(table, ids.to(id_type).cuda(), 3.5, padding)
        (dt,) = torch.autograd.grad(out, table, grad)
        want, dwant = embed_oracle(table, ids, 3.5, padding, grad)
        near(out, want, dtype, "out", 3.3e-3)
        near(dt, dwant, dtype, "table", 3.3e-3)
        assert not dt[dwant.cuda().abs().sum(1) == 0].any()
        again = torch.autograd.grad(embedding_lookup(table, ids.to(id_type).cuda(), 3.5, padding), table, grad)[0]
        assert torch.equal(dt, again), "identical inputs must give identical bits"


def test_embedding_out_of_range_ids_select_the_last_row_without_validation():
    table = normal((9, 16), F32, 3).requires_grad_()
    ids = torch.tensor([0, 9, -1, 2**31 - 1, 8], dtype=torch.int32, device="cuda")
    out = embedding_lookup(table, ids, 2.0, validate=False)
    assert torch.equal(out[1:], (table * 2.0)[[8, 8, 8, 8]])
    (dt,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert torch.equal(dt[8], torch.full((16,), 8.0, device="cuda")) and not dt[1:8].any()
    with pytest.raises(ValueError, match="ids must lie"):
        embedding_lookup(table, ids)


def test_embedding_scalar_ids_and_strided_gradient():
    table = normal((9, 16), F32, 4).requires_grad_()
    out = embedding_lookup(table, torch.tensor(3, device="cuda"))
    assert torch.equal(out, table[3])
    ids = torch.tensor([[1, 2], [2, 3]], device="cuda")
    (dt,) = torch.autograd.grad(embedding_lookup(table, ids).sum((0, 2)).sum(), table)  # an expanded gradient
    assert torch.equal(dt[:, 0].cpu(), torch.tensor([0.0, 1, 2, 1, 0, 0, 0, 0, 0]))


# ------------------------------------------------------------------------ group norm and act
def norm_oracle(x, w, b, groups, eps, act, grad):
    xd, wd, bd = (t.detach().double().cpu().requires_grad_() for t in (x, w, b))
    flat = xd.reshape(x.shape[0], math.prod(x.shape[1:-1]), groups, x.shape[-1] // groups)
    mean = flat.mean((1, 3), keepdim=True)
    var = (flat - mean).square().mean((1, 3), keepdim=True)
    u = ((flat - mean) / (var + eps).sqrt()).reshape(x.shape) * wd + bd
    y = u * torch.sigmoid(u) if act == "silu" else u
    return (y.detach(), *torch.autograd.grad(y, (xd, wd, bd), grad.double().cpu()))


# batch, pixels, channels, groups: one pixel, one channel a group, groups of odd, of 4-, 8- and
# 16-byte vectors, several groups a block, one group of all, a slice in chunks (128 x 128 pixels), and
# the sizes around the registers' limit
NORM = [
    (2, (1,), 8, 8), (1, (3, 3), 4, 1), (3, (7, 7), 136, 8), (2, (16, 16), 64, 32), (2, (32, 32), 1152, 32),
    (1, (64, 64), 72, 2), (1, (128, 128), 36, 1), (2, (50, 41), 34, 2), (2, (28, 28), 96, 4), (1, (5,), 1152, 1),
    (4, (2, 3, 5), 40, 4), (1, (16385,), 8, 1), (0, (4, 4), 8, 2), (1, (97, 61), 2, 1), (1, (90, 90), 9, 9),
]


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("batch,pixels,channels,groups", NORM)
def test_group_norm(batch, pixels, channels, groups, dtype, act):
    announce(f"group norm {batch}x{pixels}x{channels} groups={groups} {dtype} {act}")
    wide = F32 if act == "none" else dtype  # fp32 weights beside a bf16 input
    x = normal((batch, *pixels, channels), dtype, 5, mean=0.7).requires_grad_()
    w, b = normal((channels,), wide, 6, mean=1.0, std=0.3).requires_grad_(), normal((channels,), wide, 7).requires_grad_()
    grad = normal(x.shape, dtype, 8)
    y = group_norm_act(x, w, b, groups, 1e-5, act)
    got = torch.autograd.grad(y, (x, w, b), grad)
    want = norm_oracle(x, w, b, groups, 1e-5, act, grad)
    near(y, want[0], dtype, "y", 3.3e-3)
    if batch and math.prod(pixels) * (channels // groups) == 1:  # one element a group: y = act(bias), dx = 0
        assert float(got[0].float().abs().max()) <= 1e-5
    else:
        near(got[0], want[1], dtype, "dx", 3.3e-3)
    for g, e, name in zip(got[1:], want[2:], ("dw", "db")):
        near(g, e, wide, name, 3.3e-3)
    again = torch.autograd.grad(group_norm_act(x, w, b, groups, 1e-5, act), (x, w, b), grad)
    assert all(torch.equal(p, q) for p, q in zip(got, again)), "identical inputs must give identical bits"


def test_group_norm_keeps_its_digits_under_a_large_mean_and_large_values():
    # a mean of 1000 deviations: fp32 inputs carry 2^-24 of 1000, so 6e-5 of a deviation at most
    x = normal((2, 33, 33, 24), F32, 9, mean=1000.0)
    w, b = torch.ones(24, device="cuda"), torch.zeros(24, device="cuda")
    y = group_norm_act(x, w, b, 3, 1e-6, "none")
    want = norm_oracle(x, w, b, 3, 1e-6, "none", torch.zeros_like(x))[0]
    assert float((y.cpu().double() - want).abs().max()) <= 3e-4
    # values whose exponentials overflow: silu is u above and 0 below
    y = group_norm_act(normal((1, 64, 8), F32, 10), w[:8] * 1e6, b[:8], 1, 1e-6, "silu")
    assert torch.isfinite(y).all()


def test_group_norm_nan_stays_in_its_image_and_group():
    x = normal((3, 8, 8, 64), BF16, 11)
    x[1, 2, 3, 17] = float("nan")
    y = group_norm_act(x, torch.ones(64, device="cuda", dtype=BF16), torch.zeros(64, device="cuda", dtype=BF16), 4)
    bad = torch.isnan(y)
    assert bad[1, :, :, 16:32].all() and int(bad.sum()) == 64 * 16


# ----------------------------------------------------------------------------- cross attention
def attention_oracle(q, k, v, lengths, scale, grad):
    outs = []
    each = q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        n = k.shape[1] if lengths is None else int(lengths[b])
        qd, kd, vd = (t[b].detach().double().cpu().requires_grad_() for t in (q, k, v))
        kk, vv = (t[:n].repeat_interleave(each, 1).transpose(0, 1) for t in (kd, vd))
        p = torch.softmax(qd.transpose(0, 1) @ kk.transpose(1, 2) * scale, -1)
        out = (p @ vv).transpose(0, 1) if n else qd * 0.0
        grads = (torch.autograd.grad(out, (qd, kd, vd), grad[b].double().cpu()) if n else
                 [torch.zeros_like(t) for t in (qd, kd, vd)])
        outs.append((out.detach(), *grads))
    return [torch.stack(t) for t in zip(*outs)]


# batch, queries, keys, heads, key heads, channels, lengths: one query, one key, no key, odd sizes, every
# width of the compiled heads and the ones beside them, pieces of 64 keys with tails, shared heads
ATTEND = [
    (1, 1, 1, 1, 1, 1, None), (2, 1, 300, 8, 2, 128, (300, 17)), (3, 33, 65, 2, 1, 40, (65, 0, 1)),
    (2, 256, 77, 4, 4, 72, (77, 9)), (1, 130, 129, 3, 3, 64, (128,)), (2, 31, 64, 6, 2, 33, (64, 63)),
    (1, 70, 200, 2, 2, 96, None), (2, 5, 97, 5, 5, 97, (96, 97)), (1, 17, 33, 4, 1, 7, (32,)), (2, 4, 0, 2, 2, 16, (0, 0)),
    (1, 129, 1023, 1, 1, 80, (1000,)), (4, 2, 40, 2, 1, 32, (0, 0, 0, 0)), (1, 257, 321, 2, 2, 127, (320,)),
    (1, 3, 5000, 4, 2, 64, (4999,)),
]


def attention_inputs(batch, queries, keys, heads, shared, dim, lengths, dtype):
    q = normal((batch, queries, heads, dim), dtype, 12).requires_grad_()
    k = normal((batch, keys, shared, dim), dtype, 13).requires_grad_()
    v = normal((batch, keys, shared, dim), dtype, 14, mean=0.2).requires_grad_()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return q, k, v, n, normal((batch, queries, heads, dim), dtype, 15)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_cross_attention(case, dtype):
    announce(f"cross attention {case} {dtype}")
    q, k, v, n, grad = attention_inputs(*case, dtype)
    out = cross_attention(q, k, v, n)
    got = torch.autograd.grad(out, (q, k, v), grad)
    want = attention_oracle(q, k, v, n, 1 / math.sqrt(q.shape[3]), grad)
    near(out, want[0], dtype, "out", 5e-3)
    if case[2] == 1:  # one key: P = 1 whatever q and k, so their gradients are rounding noise about 0
        assert float(got[0].float().abs().max()) <= 1e-2 and float(got[1].float().abs().max()) <= 1e-2
        near(got[2], want[3], dtype, "dv", 5e-3)
    else:
        for g, e, name in zip(got, want[1:], ("dq", "dk", "dv")):
            near(g, e, dtype, name, 5e-3)
    if n is not None:
        for b, length in enumerate(case[6]):
            assert not got[1][b, length:].any() and not got[2][b, length:].any()
            if length == 0:
                assert not out[b].any() and not got[0][b].any()
    again = torch.autograd.grad(cross_attention(q, k, v, n), (q, k, v), grad)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "identical inputs must give identical bits"
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, n), out)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp32"])
def test_cross_attention_ignores_what_lies_past_the_lengths(dtype):
    q, k, v, n, grad = attention_inputs(3, 40, 150, 4, 2, 72, (150, 64, 3), dtype)
    out = cross_attention(q, k, v, n)
    want = (out, *torch.autograd.grad(out, (q, k, v), grad))
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        kb, vb = k.detach().clone(), v.detach().clone()
        for b, length in enumerate((150, 64, 3)):
            kb[b, length:] = bad
            vb[b, length:] = bad
        kb.requires_grad_(), vb.requires_grad_()
        out = cross_attention(q, kb, vb, n)
        got = (out, *torch.autograd.grad(out, (q, kb, vb), grad))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_cross_attention_large_and_negative_scores():
    # scores of thousands: the probabilities are those of the largest score, without overflow
    q, k, v, n, grad = attention_inputs(1, 65, 130, 2, 2, 64, (129,), F32)
    for scale in (40.0, -40.0, 0.0):
        out = cross_attention(q, k, v, n, scale)
        got = (out, *torch.autograd.grad(out, (q, k, v), grad))
        assert all(torch.isfinite(t).all() for t in got)
        want = attention_oracle(q, k, v, n, scale, grad)
        # a score of 1000 carries 2^-24 of itself, and the probabilities as much relatively
        assert float((out.detach().double().cpu() - want[0]).abs().max()) <= 2e-3 * float(want[0].abs().max())


def test_cross_attention_strides_broadcasts_and_streams():
    kv = normal((2, 90, 2, 3, 40), BF16, 16)
    q = normal((2, 3, 50, 40), BF16, 17).transpose(1, 2)  # heads before tokens
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = cross_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(cross_attention(q, k, v), want)
    shifted = torch.empty(k.numel() + 1, dtype=BF16, device="cuda")[1:].view(k.shape).copy_(k)  # 2-byte aligned
    assert torch.equal(cross_attention(q, shifted, v), want)
    # states shared by the whole batch: one row, expanded; its gradient is the batch's sum
    one = normal((1, 90, 3, 40), F32, 18).requires_grad_()
    many = one.detach().expand(4, -1, -1, -1).contiguous().requires_grad_()
    qf, grad = normal((4, 20, 3, 40), F32, 19), normal((4, 20, 3, 40), F32, 20)
    got = torch.autograd.grad(cross_attention(qf, one.expand(4, -1, -1, -1), one.expand(4, -1, -1, -1)), one, grad)[0]
    want = torch.autograd.grad(cross_attention(qf, many, many), many, grad)[0].sum(0, keepdim=True)
    assert_parity(got, want, F32, what="broadcast states")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = cross_attention(qf, many, many)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(late, cross_attention(qf, many, many))


# ----------------------------------------------------------------------- gradients by differences
def directional(f, inputs, seeds, h=2e-3):
    """(f(x + h d) - f(x - h d)) / 2h and <grad, d> for random directions d, in fp32."""
    loss = f(*inputs)
    grads = torch.autograd.grad(loss, inputs)
    for i, (x, g) in enumerate(zip(inputs, grads)):
        d = normal(tuple(x.shape), F32, seeds + i)
        ends = [f(*(t.detach() + s * h * d if j == i else t.detach() for j, t in enumerate(inputs))) for s in (1, -1)]
        slope = float((ends[0] - ends[1]).double()) / (2 * h)
        # third derivatives times h^2, and 2^-24 of the summed terms over h
        yield slope, float((g.double() * d.double()).sum()), float(g.double().norm())


def test_gradients_follow_differences():
    q, k, v, n, grad = attention_inputs(2, 9, 21, 4, 2, 24, (21, 5), F32)
    table, ids = normal((12, 20), F32, 21).requires_grad_(), torch.arange(30, device="cuda") % 7
    eg = normal((30, 20), F32, 22)
    x = normal((2, 6, 6, 24), F32, 23).requires_grad_()
    w, b = normal((24,), F32, 24).requires_grad_(), normal((24,), F32, 25).requires_grad_()
    xg = normal((2, 6, 6, 24), F32, 26)
    for f, inputs in (
        (lambda *t: (cross_attention(*t, n).double() * grad).sum(), (q, k, v)),
        (lambda t: (embedding_lookup(t, ids, 2.0).double() * eg).sum(), (table,)),
        (lambda *t: (group_norm_act(*t, 4).double() * xg).sum(), (x, w, b)),
    ):
        for slope, inner, size in directional(f, inputs, 40):
            assert abs(slope - inner) <= 5e-3 * size, (slope, inner, size)


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    table, ids = normal((5, 8), F32, 30), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: embedding_lookup(table.t(), ids), lambda: embedding_lookup(table.double(), ids),
                lambda: embedding_lookup(table, ids.float()), lambda: embedding_lookup(table, ids.cpu()),
                lambda: embedding_lookup(table, ids, 1.0, 5), lambda: embedding_lookup(table[0], ids),
                lambda: embedding_lookup(table, ids + 5), lambda: embedding_lookup(table, ids - 1),
                lambda: embedding_lookup(table.half(), ids, validate=False)):
        with pytest.raises(ValueError):
            bad()
    x, w = normal((2, 4, 4, 8), BF16, 31), normal((8,), BF16, 32)
    for bad in (lambda: group_norm_act(x, w, w, 3), lambda: group_norm_act(x, w, w, 0),
                lambda: group_norm_act(x.transpose(1, 3), w, w, 2), lambda: group_norm_act(x, w[:4], w, 2),
                lambda: group_norm_act(x, w, w.float(), 2), lambda: group_norm_act(x, w, w, 2, 1e-6, "relu"),
                lambda: group_norm_act(x.float(), w, w, 2), lambda: group_norm_act(x, w.cpu(), w.cpu(), 2),
                lambda: group_norm_act(x[0, 0, 0], w, w, 2)):
        with pytest.raises(ValueError):
            bad()
    q, k, v, n, _ = attention_inputs(2, 4, 6, 4, 2, 16, (6, 2), BF16)
    for bad in (lambda: cross_attention(q, k[:1], v[:1]), lambda: cross_attention(q, k, v[:, :5]),
                lambda: cross_attention(q[:, :, :3], k, v), lambda: cross_attention(q, k.float(), v.float()),
                lambda: cross_attention(q, k, v, n.long()), lambda: cross_attention(q, k, v, n[:1]),
                lambda: cross_attention(q, k, v, n + 1), lambda: cross_attention(q, k, v, n - 3),
                lambda: cross_attention(q, k, v, n.cpu()), lambda: cross_attention(q[0], k[0], v[0]),
                lambda: cross_attention(q[..., ::2], k[..., ::2], v[..., ::2]),
                lambda: cross_attention(q.repeat(1, 1, 1, 9), k.repeat(1, 1, 1, 9), v.repeat(1, 1, 1, 9))):
        with pytest.raises(ValueError):
            bad()
    # lengths that were not checked are clamped
    assert torch.equal(cross_attention(q, k, v, n + 100, validate=False), cross_attention(q, k, v))
    assert not cross_attention(q, k, v, n - 100, validate=False).any()
    assert C.__all__ == ["embedding_lookup", "cross_attention", "group_norm_act"]
