"""GPU: denoisers whose bodies run on the HIP operators against the same ones in plain torch, forward and
backward, with and without dropout, in-context tokens, a text.

Tolerances: the two models compute the same formulas in another order of sums, so a projection's fp32
results agree within some 1e-6; eight blocks of residual updates of size 1 pass that on about once
each: 1e-4 in relative L2. In bf16 every rounding on the way (some 20 per block, 2^-9 each, and the torch
body also rounds its angles' cosines) may fall to the other side: 6e-2."""
from __future__ import annotations

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip.e2e import SiHCDenoiser
from sihc_hip.text_denoiser import TextSiHCDenoiser

pytestmark = pytest.mark.gpu
BOUNDS = {torch.float32: 1e-4, torch.bfloat16: 6e-2}


def pair(text, dtype, **over):
    kind = TextSiHCDenoiser if text else SiHCDenoiser
    sizes = dict(hidden=96, heads=4, depth=8, stages=(8,), image=64, grid=4, patch=8, num_classes=10, **over)
    if text:
        sizes.update(kv_heads=2, vocab=60, state_dim=64, groups=8, max_tokens=24)
    models = [kind(body=b, **sizes).random_init(0.05, seed=1).cuda().to(dtype) for b in ("torch", "fused")]
    g = torch.Generator().manual_seed(2)
    inputs = [torch.randn(5, 3, 64, 64, generator=g).cuda().to(dtype), torch.rand(5, generator=g).cuda(),
              torch.randint(0, 10, (5,), generator=g).cuda()]
    if text:
        inputs += [torch.randint(1, 60, (5, 20), generator=g).cuda(),
                   torch.tensor([20, 3, 0, 1, 17], dtype=torch.int32, device="cuda")]
    return models, inputs, torch.randn(5, 3, 64, 64, generator=g).cuda()


def step(model, inputs, target, seed=0):
    torch.manual_seed(seed)  # the seed of a call's dropout is drawn from torch's generator
    out = model(*inputs)
    loss = (out.float() - target).square().mean()
    return out.detach(), torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)


@pytest.mark.parametrize("dropout", [0.0, 0.2])
@pytest.mark.parametrize("over", [{}, {"schedule": "literal"}, {"in_context_len": 3, "in_context_start": 2}], ids=str)
@pytest.mark.parametrize("text", [False, True], ids=["labels", "text"])
@pytest.mark.parametrize("dtype", BOUNDS, ids=["fp32", "bf16"])
def test_fused_bodies_match_the_torch_ones(dtype, text, over, dropout):
    announce(f"fused body {dtype} text {text} {over} dropout {dropout}")
    models, inputs, target = pair(text, dtype, dropout=dropout, **over)
    (want, wgrads), (got, grads) = (step(m, inputs, target) for m in models)
    assert rel_l2(got, want) <= BOUNDS[dtype]
    assert [g is None for g in grads] == [g is None for g in wgrads]
    flat = [torch.cat([g.double().flatten() for g in gs if g is not None]) for gs in (grads, wgrads)]
    assert rel_l2(*flat) <= BOUNDS[dtype]
    for (name, _), g, w in zip(models[0].named_parameters(), grads, wgrads):
        if g is not None and name in ("blocks.3.attn.qkv.weight", "blocks.0.mlp.w12.weight", "blocks.7.ada.1.weight",
                                      "blocks.2.attn.q_norm.weight", "cross.1.proj.weight", "t_mlp.0.weight"):
            assert rel_l2(g, w) <= 3 * BOUNDS[dtype], name


def test_dropout_is_of_training_alone_and_of_the_seed():
    models, inputs, target = pair(False, torch.float32, dropout=0.3)
    for model in models:
        first, again, other = (step(model, inputs, target, seed)[0] for seed in (1, 1, 2))
        assert torch.equal(first, again) and not torch.equal(first, other)
        model.eval()
        with torch.no_grad():
            assert torch.equal(model(*inputs), model(*inputs))
            model.dropout = 0.0
            assert torch.equal(model(*inputs), model.train()(*inputs))


def test_bodies_that_are_computed_again_have_their_masks():
    models, inputs, target = pair(False, torch.float32, dropout=0.3)
    model = models[1]
    _, want = step(model, inputs, target)
    update = model._update
    model._update = lambda *args: torch.utils.checkpoint.checkpoint(update, *args, use_reentrant=False)
    _, got = step(model, inputs, target)
    assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


def test_a_captured_sampling_step():
    models, inputs, _ = pair(True, torch.bfloat16)
    model = models[1].eval()
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(*inputs)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = model(*inputs)
        for turn in range(3):
            inputs[0].add_(0.1 * turn)
            want = model(*inputs).clone()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(kept, want)
