"""GPU: the text-conditioned denoiser, forward and backward, on the operators against the same model
on their plain torch forms.

Tolerances: the two models run the same torch code but for the three operators, whose fp32 results
agree within 1e-5; eight blocks of residual updates of size 1 pass that on about once each, so 1e-4
in relative L2. In bf16 every rounding on the way (some 10 per block, 2^-9 each, half of them in
common) may fall to the other side: 5e-2, and the loss of a training step within 1e-2."""
from __future__ import annotations

import pytest
import torch

from helpers import announce, rel_l2
from sihc_hip.text_denoiser import TextSiHCDenoiser

pytestmark = pytest.mark.gpu


def plain_lookup(table, ids, scale, padding):
    rows = torch.nn.functional.embedding(ids.long(), table, padding_idx=padding)
    return (rows.float() * scale).to(table.dtype)


def plain_attend(q, k, v, lengths):
    each = q.shape[2] // k.shape[2]
    qf, kf, vf = (t.float().transpose(1, 2) for t in (q, k, v))
    kf, vf = (t.repeat_interleave(each, 1).contiguous() for t in (kf, vf))
    score = (qf @ kf.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
    n = torch.arange(k.shape[1], device=q.device)
    seen = (n < lengths[:, None])[:, None, None]
    p = torch.softmax(torch.where(seen, score, -1e30), -1) * seen
    return (p @ vf).transpose(1, 2).to(q.dtype)


def plain_norm(x, w, b, groups, eps, act):
    u = torch.nn.functional.group_norm(x.float().flatten(1, -2).transpose(1, 2), groups, w.float(), b.float(), eps)
    return torch.nn.functional.silu(u).transpose(1, 2).reshape(x.shape).to(x.dtype)


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-4), (torch.bfloat16, 5e-2)], ids=["fp32", "bf16"])
@pytest.mark.parametrize("schedule", ["stage", "literal"])
def test_text_denoiser_matches_its_plain_form(dtype, bound, schedule):
    announce(f"text denoiser {dtype} {schedule}")
    model = TextSiHCDenoiser(hidden=96, heads=4, kv_heads=2, vocab=300, state_dim=64, groups=8, max_tokens=24,
                             depth=8, stages=(8,), image=64, grid=4, patch=8, num_classes=10, schedule=schedule)
    model = model.random_init(0.05, seed=1).cuda().to(dtype)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 3, 64, 64, generator=g).cuda().to(dtype)
    t, y = torch.rand(5, generator=g).cuda(), torch.randint(0, 10, (5,), generator=g).cuda()
    lengths = torch.tensor([20, 3, 0, 1, 17], dtype=torch.int32)
    tokens = torch.randint(1, 300, (5, 20), generator=g)
    tokens = torch.where(torch.arange(20) < lengths[:, None], tokens, 0).cuda()  # padded with token 0
    target = torch.randn(5, 3, 64, 64, generator=g).cuda()

    def step():
        out = model(x, t, y, tokens, lengths.cuda())
        loss = (out.float() - target).square().mean()
        names, params = zip(*[(n, p) for n, p in model.named_parameters()])
        return loss.detach(), out.detach(), dict(zip(names, torch.autograd.grad(loss, params)))

    loss, out, grads = step()
    model.lookup, model.attend, model.final_norm.norm = plain_lookup, plain_attend, plain_norm
    ploss, pout, pgrads = step()
    assert abs(float(loss) - float(ploss)) <= 1e-2 * float(ploss)
    assert rel_l2(out, pout) <= bound
    whole = [torch.cat([g.flatten().double() for g in gs.values()]) for gs in (grads, pgrads)]
    assert rel_l2(*whole) <= bound
    for name in ("tokens", "final_norm.weight", "cross.3.kv.weight", "cross.0.q.weight"):
        assert rel_l2(grads[name], pgrads[name]) <= 2 * bound, name
    assert not grads["tokens"][0].any()  # the padding token


def test_no_text_and_an_empty_prompt_are_the_label_model():
    model = TextSiHCDenoiser(hidden=32, heads=2, vocab=20, state_dim=16, groups=4, max_tokens=8, depth=8, stages=(8,),
                             image=64, grid=4, patch=8, num_classes=4).random_init(0.05, seed=3).cuda()
    with torch.no_grad():  # an attention's output without bias, so that an empty prompt adds nothing
        for c in model.cross:
            c.proj.bias.zero_()
    x, t, y = torch.randn(2, 3, 64, 64, device="cuda"), torch.rand(2, device="cuda"), torch.tensor([1, 3], device="cuda")
    with torch.no_grad():
        want = model(x, t, y)
        got = model(x, t, y, torch.ones(2, 5, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
        assert torch.equal(got, want)
        with pytest.raises(ValueError, match="at most 8 tokens"):
            model(x, t, y, torch.ones(2, 9, dtype=torch.int32, device="cuda"))
