"""GPU: the conditioning operators at offsets past 32 bits, in captured graphs, under torch.compile and
over many drawn sizes.

Bounds as in test_gpu_conditioning.py: 1e-5 for fp32, 5e-3 in relative L2 for bf16 attention, 3.3e-3
for the other operators; 1.5 times those for drawn sizes, whose smallest outputs are a handful of
numbers and so not an average of roundings."""
from __future__ import annotations

import math
import random

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip import cross_attention, embedding_lookup, group_norm_act
from test_gpu_conditioning import attention_oracle, embed_oracle, norm_oracle, normal

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def test_embedding_of_a_table_past_32_bits():
    rows, channels = 1_900_000, 1152  # 2.19e9 elements
    announce("embedding of 2.19e9 elements")
    table = torch.zeros(rows, channels, dtype=BF16, device="cuda")
    table[-1], table[rows // 2] = 3.0, 2.0
    table.requires_grad_()
    for count in (7, 3000):  # both kernels of the gradient
        ids = torch.full((count,), rows - 1, dtype=torch.int64, device="cuda")
        ids[0], ids[1] = rows // 2, 0
        out = embedding_lookup(table, ids, 2.0)
        assert torch.equal(out[:, 5].cpu().float(), torch.tensor([4.0, 0.0] + [6.0] * (count - 2)))
        (dt,) = torch.autograd.grad(out, table, torch.ones_like(out))
        assert torch.equal(dt[-1].float(), torch.full((channels,), 2.0 * (count - 2), device="cuda").to(BF16).float())
        assert float(dt[rows // 2, 1151]) == 2.0 and float(dt[0, 0]) == 2.0
        assert int(torch.count_nonzero(dt[:1 << 20])) == 2 * channels and not dt[rows - 5:rows - 1].any()
        del dt, out


def test_group_norm_of_a_tensor_past_32_bits():
    announce("group norm of 2.2e9 elements")
    x = torch.zeros(131, 128, 128, 1024, dtype=BF16, device="cuda")
    x[-1].normal_()
    w, b = normal((1024,), BF16, 1), normal((1024,), BF16, 2)
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, w, b)[-1], group_norm_act(x[-1:].clone(), w, b)[0])


@pytest.mark.parametrize("stride", [(1 << 31) + 64, 1 << 25], ids=["batch", "token"])
def test_cross_attention_of_states_past_32_bits(stride):
    announce(f"cross attention with a stride of {stride} elements")
    buffer = torch.empty((1 << 31) + (1 << 29), dtype=BF16, device="cuda")
    shape, steps = ((2, 66, 2, 64), (stride, 128, 64, 1)) if stride > 1 << 30 else ((1, 66, 2, 64), (0, stride, 64, 1))
    k = buffer.as_strided(shape, steps).normal_()
    q = normal((shape[0], 40, 4, 64), BF16, 3)
    assert torch.equal(cross_attention(q, k, k), cross_attention(q, k.contiguous(), k.contiguous()))
    leaves = [t.detach().requires_grad_() for t in (q, k, k)]
    packed = [t.detach().contiguous().requires_grad_() for t in (q, k, k)]
    grad = normal(q.shape, BF16, 4)
    for a, b in zip(torch.autograd.grad(cross_attention(*leaves), leaves, grad),
                    torch.autograd.grad(cross_attention(*packed), packed, grad)):
        assert torch.equal(a, b)


def passes():
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 900, (3000,), generator=g).cuda()
    n = torch.tensor([300, 0, 77], dtype=torch.int32, device="cuda")
    yield (lambda t: embedding_lookup(t, ids, 2.0, 3, validate=False)), [normal((900, 72), BF16, 6)]
    yield (lambda t: embedding_lookup(t, ids[:50], 2.0, validate=False)), [normal((900, 72), F32, 6)]
    yield (lambda *t: group_norm_act(*t, 4)), [normal((2, 20, 20, 96), BF16, 7), normal((96,), BF16, 8), normal((96,), BF16, 9)]
    yield (lambda *t: group_norm_act(*t, 1)), [normal((1, 128, 128, 36), F32, 7), normal((36,), F32, 8), normal((36,), F32, 9)]
    yield (lambda *t: cross_attention(*t, n, validate=False)), [normal((3, 5, 4, 64), BF16, 10), normal((3, 300, 2, 64), BF16, 11),
                                                                normal((3, 300, 2, 64), BF16, 12)]
    yield (lambda *t: cross_attention(*t, n, validate=False)), [normal((3, 300, 4, 40), F32, 10), normal((3, 300, 2, 40), F32, 11),
                                                                normal((3, 300, 2, 40), F32, 12)]


@pytest.mark.parametrize("which", range(6))
def test_captured_graphs_replay_the_eager_results(which):
    call, values = list(passes())[which]
    leaves = [v.clone().requires_grad_() for v in values]

    def step():
        out = call(*leaves)
        return (out, *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        with torch.no_grad():
            for leaf, v in zip(leaves, values):
                leaf.copy_(v * (1.0 + 0.25 * turn))
        graph.replay()
        torch.cuda.synchronize()
        want = step()  # eager, between the replays
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


@pytest.mark.parametrize("which", range(6))
def test_compiled_calls_equal_eager_ones(which):
    call, values = list(passes())[which]
    torch._dynamo.reset()
    compiled = torch.compile(lambda *t: call(*t) * 2, fullgraph=True)
    results = []
    for f in (lambda *t: call(*t) * 2, compiled):
        leaves = [v.clone().requires_grad_() for v in values]
        out = f(*leaves)
        results.append([out, *torch.autograd.grad(out, leaves, torch.ones_like(out))])
    for a, b in zip(*results):
        assert rel_l2(a, b) <= (1e-5 if a.dtype == F32 else 5e-3)


def test_drawn_sizes():
    rng = random.Random(11)
    for turn in range(60):
        dtype = rng.choice((BF16, F32))
        b, groups = rng.randint(1, 4), rng.choice((1, 2, 3, 8))
        width, edge = rng.choice((1, 2, 5, 8, 12, 33)), rng.choice((1, 2, 9, 16, 41, 70))
        announce(f"norm {turn}: {b}x{edge}x{edge}x{groups * width} / {groups} {dtype}")
        x = normal((b, edge, edge, groups * width), dtype, turn, mean=rng.choice((0.0, 30.0)) if dtype == BF16 else 0.5).requires_grad_()
        w, c = (normal((groups * width,), dtype, turn + s, mean=1.0).requires_grad_() for s in (100, 200))
        grad = normal(x.shape, dtype, turn + 300)
        y = group_norm_act(x, w, c, groups)
        got, want = (y, *torch.autograd.grad(y, (x, w, c), grad)), norm_oracle(x, w, c, groups, 1e-6, "silu", grad)
        for name, g, e in zip(("y", "dx", "dw", "db"), got, want):
            if name == "dx" and edge * edge * width < 4:
                continue  # (differences of a few equal numbers: rounding noise about 0)
            assert rel_l2(g.cpu(), e) <= 1.5 * (3.3e-3 if dtype == BF16 else 1e-5), name
    for turn in range(60):
        dtype = rng.choice((BF16, F32))
        b, shared, each = rng.randint(1, 5), rng.choice((1, 2, 3)), rng.choice((1, 2, 4))
        queries, keys, dim = rng.choice((1, 7, 64, 130, 300)), rng.choice((2, 31, 64, 65, 200, 700)), rng.choice((8, 24, 40, 63, 72, 96, 128))
        lengths = torch.tensor([rng.choice((0, 2, keys // 2 + 1, keys)) for _ in range(b)], dtype=torch.int32, device="cuda")
        announce(f"attention {turn}: {b}x{queries} over {keys} ({lengths.tolist()}), {shared}x{each} heads of {dim} {dtype}")
        q = normal((b, queries, shared * each, dim), dtype, turn).requires_grad_()
        k, v = (normal((b, keys, shared, dim), dtype, turn + s).requires_grad_() for s in (400, 500))
        grad = normal(q.shape, dtype, turn + 600)
        out = cross_attention(q, k, v, lengths)
        got = (out, *torch.autograd.grad(out, (q, k, v), grad))
        for g, e in zip(got, attention_oracle(q, k, v, lengths, 1 / math.sqrt(dim), grad)):
            assert torch.equal(g.cpu() == 0, e.to(dtype) == 0) if not e.any() else rel_l2(g.cpu(), e) <= 1.5 * (5e-3 if dtype == BF16 else 1e-5)
    for turn in range(40):
        dtype = rng.choice((BF16, F32))
        rows, channels, count = rng.choice((1, 60, 1500, 70000)), rng.choice((1, 7, 64, 264)), rng.choice((3, 900, 1030, 9000))
        announce(f"embedding {turn}: {rows}x{channels}, {count} ids {dtype}")
        skew = rng.choice((1.0, 6.0))
        g = torch.Generator().manual_seed(turn)
        ids = (rows * torch.rand(count, generator=g).pow(skew)).long().clamp_(max=rows - 1)
        padding = rng.choice((None, 0, rows - 1))
        table, grad = normal((rows, channels), dtype, turn).requires_grad_(), normal((count, channels), dtype, turn + 1)
        out = embedding_lookup(table, ids.cuda(), 1.5, padding)
        (dt,) = torch.autograd.grad(out, table, grad)
        want, dwant = embed_oracle(table, ids, 1.5, padding, grad)
        assert rel_l2(out.cpu(), want) <= 1.5 * (3.3e-3 if dtype == BF16 else 1e-5)
        assert rel_l2(dt.cpu(), dwant) <= 1.5 * (3.3e-3 if dtype == BF16 else 1e-5) if dwant.any() else not dt.any()


# batches that leave a block many groups: 16 of one channel and 4 waves, 32 and 16 waves, 64, and a prime number
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("batch,pixels,channels,groups", [
    (300, 16, 32, 32), (600, 9, 64, 64), (600, 200, 32, 32), (520, 5, 97, 97), (300, 30, 128, 32), (1100, 40, 64, 64)])
def test_group_norm_of_many_narrow_groups(batch, pixels, channels, groups, dtype):
    announce(f"group norm {batch}x{pixels}x{channels} groups={groups} {dtype}")
    x = normal((batch, pixels, channels), dtype, 31, mean=0.4).requires_grad_()
    w, b = normal((channels,), dtype, 32, mean=1.0, std=0.3).requires_grad_(), normal((channels,), dtype, 33).requires_grad_()
    grad = normal(x.shape, dtype, 34)
    y = group_norm_act(x, w, b, groups, 1e-5, "silu")
    got = (y, *torch.autograd.grad(y, (x, w, b), grad))
    for g, e, name in zip(got, norm_oracle(x, w, b, groups, 1e-5, "silu", grad), ("y", "dx", "dw", "db")):
        assert rel_l2(g.cpu(), e) <= (1e-5 if dtype is F32 else 3.3e-3), name
