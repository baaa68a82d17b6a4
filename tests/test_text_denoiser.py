"""CPU: a text-conditioned denoiser keeps nothing of a call in the module: calls on several threads and
updates that are computed again in the backward see their own prompts. Routing and operators are the
plain forms, in float64, so that equal calls give equal results."""
from __future__ import annotations

import threading

import torch
from torch.utils.checkpoint import checkpoint

from oracle import sihc_oracle as O
from sihc_hip.text_denoiser import TextSiHCDenoiser
from test_gpu_text_denoiser import plain_attend, plain_lookup, plain_norm


def model_and_inputs(schedule="stage", **over):
    model = TextSiHCDenoiser(hidden=32, heads=2, vocab=40, state_dim=16, groups=4, max_tokens=8, depth=8, stages=(8,),
                             image=32, grid=2, patch=8, num_classes=4, schedule=schedule, **over)
    model = model.random_init(0.1, seed=5).double()
    model.read, model.triangular, model.write = O.read, O.triangular_torch, O.write
    model.event = lambda x, dz, beta, alpha: O.event_forward(x, dz, beta, alpha)
    model.lookup, model.attend, model.final_norm.norm = plain_lookup, plain_attend, plain_norm
    g = torch.Generator().manual_seed(6)
    x, t, y = torch.randn(2, 3, 32, 32, generator=g, dtype=torch.float64), torch.rand(2, generator=g), torch.tensor([1, 3])
    tokens = torch.randint(1, 40, (2, 2, 6), generator=g)
    lengths = torch.tensor([[6, 3], [2, 5]], dtype=torch.int32)
    return model, x, t, y, tokens, lengths


def test_calls_on_two_threads_keep_their_own_prompts():
    model, x, t, y, tokens, lengths = model_and_inputs()
    with torch.no_grad():
        want = [model(x, t, y, tokens[i], lengths[i]) for i in range(2)]
    assert float((want[0] - want[1]).abs().max()) > 1e-3  # the prompts matter
    meet, got = threading.Barrier(2, timeout=60), [None, None]

    def attend(*args):  # the two calls take turns, update by update
        meet.wait()
        return plain_attend(*args)

    def call(i):
        with torch.no_grad():
            got[i] = model(x, t, y, tokens[i], lengths[i])

    model.attend = attend
    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    for i in range(2):
        assert got[i] is not None and torch.allclose(got[i], want[i], rtol=0, atol=1e-12)


def test_updates_that_are_computed_again_see_the_prompt():
    for schedule, over in (("stage", {}), ("literal", {"in_context_len": 3, "in_context_start": 4})):
        model, x, t, y, tokens, lengths = model_and_inputs(schedule, **over)

        def grads():
            loss = model(x, t, y, tokens[0], lengths[0]).square().sum()
            return torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)

        want = grads()
        update = model._update
        model._update = lambda *args: checkpoint(update, *args, use_reentrant=False)
        for a, b in zip(grads(), want):
            assert (a is None) == (b is None) and (a is None or torch.allclose(a, b, rtol=1e-9, atol=1e-12))
        assert want[[n for n, _ in model.named_parameters()].index("tokens")].any()
