"""GPU: every variant that the conditioning operators choose by size, against 64 bits, at small widths.

Each test names the kernels that its sizes are for and looks for them in a profile of the call, so that a line that
moves between two variants does not take one of them out of the tests. Bounds as in test_gpu_conditioning.py."""
from __future__ import annotations

import math

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip import cross_attention, embedding_lookup, group_norm_act
from test_gpu_conditioning import attention_oracle, embed_oracle, norm_oracle, normal

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])


def profiled(call):
    """(call(), the names of the kernels that it launched)."""
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU, torch.profiler.ProfilerActivity.CUDA]) as prof:
        out = call()
        torch.cuda.synchronize()
    return out, [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]


def launched(names, *wanted):
    for want in wanted:
        assert any(want in name for name in names), (want, names)


# ------------------------------------------------------------------------- embedding lookup
# rows, tokens, the kernels of the sort: chunks of 32 tokens past 16,384, 16 keys a thread past 65,536, the scan by one
# block past 262,144; one to three passes; half of the tokens select one row, whose run passes more than 16 chunks
@TYPES
@pytest.mark.parametrize("rows,tokens,channels,kernels", [
    (900, 16384, 40, ("k_embed_grad<", ", 8>", "k_sort_count<", ", 4>")),
    (900, 16385, 40, (", 32>", "k_sort_scatter<", ", 4>")),
    (30000, 32771, 24, (", 32>", ", 4>")),
    (30000, 65537, 17, (", 32>", "k_sort_count<", ", 16>")),
    (1100000, 70001, 8, (", 32>", ", 16>")),
    (5000, 270007, 16, (", 32>", ", 16>", "k_sort_scan")),
])
def test_embedding_gradient_of_many_tokens(rows, tokens, channels, kernels, dtype):
    announce(f"embedding of {tokens} tokens, {rows} rows of {channels} channels {dtype}")
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(0, rows, (tokens,), generator=g)
    ids = torch.where(torch.rand(tokens, generator=g) < 0.5, rows // 3, ids)
    for id_type, padding in ((torch.int32, None), (torch.int64, rows // 3), (torch.int64, int(ids[7]))):
        table = normal((rows, channels), dtype, 1).requires_grad_()
        grad, at = normal((tokens, channels), dtype, 2), ids.to(id_type).cuda()
        out = embedding_lookup(table, at, 1.5, padding)
        (dt,), names = profiled(lambda: torch.autograd.grad(out, table, grad, retain_graph=True))
        launched(names, *kernels)
        want, dwant = embed_oracle(table, ids, 1.5, padding, grad)
        assert rel_l2(out.cpu(), want) <= (3.3e-3 if dtype == BF16 else 1e-5)
        assert rel_l2(dt.cpu(), dwant) <= (3.3e-3 if dtype == BF16 else 1e-5)
        assert torch.equal((dt == 0).all(1).cpu(), (dwant == 0).all(1))
        assert torch.equal(torch.autograd.grad(out, table, grad)[0], dt), "identical inputs must give identical bits"


# ------------------------------------------------------------------------ group norm and act
# forward blocks of 512 threads: 512 slices, of one group or two, vectors of 16 bytes and of 8, and each compiled
# count of them; pixels in several widths, the last one short: odd channels, vectors of 8 and of 4, one group a width
@pytest.mark.parametrize("batch,pixels,channels,groups,dtype,kernel", [
    (512, 400, 72, 1, BF16, ", 8, 8, 512>"), (256, 1024, 96, 4, BF16, ", 8, 14, 512>"), (512, 1000, 72, 1, BF16, ", 8, 20, 512>"),
    (520, 500, 72, 2, BF16, ", 4, 20, 512>"), (512, 700, 36, 1, F32, ", 4, 14, 512>"), (513, 500, 24, 2, F32, ", 512>"),
    (2, 400, 1155, 5, BF16, "k_norm_moments<"), (2, 400, 1155, 5, F32, "k_norm_apply<"), (2, 150, 4128, 3, BF16, "k_norm_moments<"),
    (3, 200, 2080, 5, F32, "k_norm_moments<"), (1, 400, 4100, 41, F32, "k_norm_moments<"), (2, 130, 12288, 3, BF16, "k_norm_moments<"),
])
@pytest.mark.parametrize("act", ["silu", "none"])
def test_group_norm_variants(batch, pixels, channels, groups, dtype, kernel, act):
    announce(f"group norm {batch}x{pixels}x{channels} in {groups} groups {dtype} {act}")
    wide = F32 if act == "none" else dtype
    x = normal((batch, pixels, channels), dtype, 5, mean=0.7).requires_grad_()
    w, b = normal((channels,), wide, 6, mean=1.0, std=0.3).requires_grad_(), normal((channels,), wide, 7).requires_grad_()
    grad = normal(x.shape, dtype, 8)
    y, names = profiled(lambda: group_norm_act(x, w, b, groups, 1e-5, act))
    launched(names, kernel)
    got = torch.autograd.grad(y, (x, w, b), grad)
    for name, g, e in zip(("y", "dx", "dw", "db"), (y, *got), norm_oracle(x, w, b, groups, 1e-5, act, grad)):
        assert rel_l2(g.cpu(), e) <= (3.3e-3 if g.dtype == BF16 else 3.3e-3 if dtype == BF16 and name == "dx" else 1e-5), name
    again = torch.autograd.grad(group_norm_act(x, w, b, groups, 1e-5, act), (x, w, b), grad)
    assert all(torch.equal(p, q) for p, q in zip(got, again)), "identical inputs must give identical bits"


# ----------------------------------------------------------------------------- cross attention
# key heads in clusters of two and four on an XCD: whole rounds of 8 clusters, and what is left of them; several tiles a
# head and more than eight (which are not clustered); parts of the keys beside the clusters
@TYPES
@pytest.mark.parametrize("batch,queries,keys,heads,shared", [
    (128, 5, 33, 2, 2), (67, 40, 70, 4, 4), (129, 3, 20, 4, 4), (128, 1, 300, 2, 2), (32, 300, 65, 16, 8), (33, 70, 50, 32, 16),
    (65, 20, 90, 12, 6),
])
def test_cross_attention_in_clusters_of_heads(batch, queries, keys, heads, shared, dtype):
    announce(f"cross attention {batch}x{queries} over {keys}, {heads} heads over {shared} {dtype}")
    g = torch.Generator().manual_seed(batch + keys)
    lengths = torch.randint(0, keys + 1, (batch,), generator=g, dtype=torch.int32)
    lengths[1], lengths[2] = 0, keys
    q = normal((batch, queries, heads, 16), dtype, 12).requires_grad_()
    k, v = (normal((batch, keys, shared, 16), dtype, s).requires_grad_() for s in (13, 14))
    grad = normal(q.shape, dtype, 15)
    out = cross_attention(q, k, v, lengths.cuda())
    got = (out, *torch.autograd.grad(out, (q, k, v), grad))
    for name, a, e in zip(("out", "dq", "dk", "dv"), got, attention_oracle(q, k, v, lengths, 1 / math.sqrt(16), grad)):
        assert rel_l2(a.cpu(), e) <= (5e-3 if dtype == BF16 else 1e-5), name
        # each batch row by itself: a row in another's place would be lost in a mean over all
        for i in range(batch):
            if lengths[i] == 0:
                assert not a[i].any(), (name, i)
            elif lengths[i] == 1 and name in ("dq", "dk"):  # P = 1: rounding noise about 0, but on the keys past it
                assert float(a[i].float().abs().max()) <= 1e-2 and not (name == "dk" and a[i, 1:].any()), (name, i)
            else:
                assert rel_l2(a[i].cpu(), e[i]) <= (5e-2 if dtype == BF16 else 1e-4), (name, i)
