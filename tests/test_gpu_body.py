"""GPU: the body operators against their definitions in 64 bits, at the sizes where they can go wrong."""
from __future__ import annotations

import itertools

import pytest
import torch

import body_reference as R
from helpers import announce
from sihc_hip import body

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
THETA = 10000.0


def rand(*shape, seed=0, dtype=F32, std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (mean + std * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def leaf(t):
    return None if t is None else t.detach().requires_grad_()


# ------------------------------------------------------------------------------------ linear
def linear_case(batch, tokens, inner, outer, act, gate, residual, bias, dtype, seed=1):
    wide = 2 * outer if act == "swiglu" else outer
    shape = (batch, outer) if tokens is None else (batch, tokens, outer)
    x = rand(*shape[:-1], inner, seed=seed, dtype=dtype)
    return dict(x=x, weight=rand(wide, inner, seed=seed + 1, dtype=dtype, std=inner ** -0.5),
                bias=rand(wide, seed=seed + 2, dtype=dtype, std=0.3) if bias else None, act=act,
                gate=rand(batch, 3, outer, seed=seed + 3, dtype=dtype)[:, 1] if gate else None,
                residual=rand(*shape, seed=seed + 4, dtype=dtype) if residual else None,
                grad=rand(*shape, seed=seed + 5, dtype=dtype))


def check_linear(c, what):
    want = R.linear(**c)
    leaves = {n: leaf(c[n]) for n in ("x", "weight", "bias", "gate", "residual")}
    y = body.linear_act(leaves["x"], leaves["weight"], leaves["bias"], c["act"], leaves["gate"], leaves["residual"])
    assert y.is_contiguous() and y.dtype == c["x"].dtype
    R.check(y, *want[0], f"{what} result")
    with torch.no_grad():
        again = body.linear_act(c["x"], c["weight"], c["bias"], c["act"], c["gate"], c["residual"])
    assert torch.equal(again, y)  # what the backward keeps changes nothing
    given = [n for n in leaves if leaves[n] is not None]
    grads = dict(zip(given, torch.autograd.grad(y, [leaves[n] for n in given], c["grad"])))
    for name, w in zip(leaves, want[1:]):
        if w is not None:
            R.check(grads[name], *w, f"{what} gradient of {name}")


LINEAR_SIZES = [  # batch, tokens, inner, outer
    (1, None, 1, 1), (1, 1, 8, 8), (2, 1, 64, 96), (3, 7, 5, 3), (2, 33, 72, 40), (1, 257, 130, 67), (5, 40, 203, 331),
    (2, 129, 264, 136), (16, None, 1152, 200),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
@pytest.mark.parametrize("size", LINEAR_SIZES, ids=str)
def test_linear(size, act, dtype):
    for i, (gate, residual, bias) in enumerate(((False, False, True), (True, True, True), (True, False, False))):
        announce(f"linear_act {size} {act} gate {gate} residual {residual} bias {bias} {dtype}")
        check_linear(linear_case(*size, act, gate, residual, bias, dtype, seed=10 * i), f"{size} {act} {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size,act", [((8, 256, 512, 640), "none"), ((4, 300, 2730, 520), "silu"),
                                      ((32, 64, 192, 1024), "swiglu"), ((2, 4100, 96, 80), "none"),
                                      ((1, 31, 4099, 72), "silu")], ids=str)
def test_linear_of_many_tiles(size, act, dtype):
    announce(f"linear_act {size} {act} {dtype}")
    check_linear(linear_case(*size, act, True, True, True, dtype), f"{size} {act} {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("batch,tokens", [(300, None), (1, 1), (70, 2), (33, 63), (9, 64), (5, 65), (2, 130)])
def test_gates_of_few_and_many_rows(batch, tokens, act, dtype):
    """A gate for every row, images that one partial sum holds, and larger ones."""
    announce(f"linear_act gates of {tokens} rows {act} {dtype}")
    check_linear(linear_case(batch, tokens, 48, 264, act, True, True, True, dtype), f"{batch} x {tokens} {act} {dtype}")


# Sizes for which the forward and the two gradients' products take the larger tiles, one and several parts of
# the contraction, and tiles that end inside the result.
@pytest.mark.parametrize("size,act", [((64, 256, 768, 2048), "swiglu"), ((64, 256, 1152, 1152), "none"),
                                      ((32, 256, 2730, 1024), "none"), ((64, 256, 768, 768), "silu"),
                                      ((61, 259, 2050, 700), "none"), ((16, 256, 4096, 4096), "none"),
                                      ((2, None, 1152, 6912), "none"), ((8, 250, 520, 1030), "swiglu")], ids=str)
def test_linear_of_large_tiles(size, act):
    announce(f"linear_act {size} {act}")
    check_linear(linear_case(*size, act, True, True, True, BF16), f"{size} {act}")


@pytest.mark.parametrize("size,act", [((16, 256, 1024, 1100), "swiglu"), ((3, 1500, 640, 1000), "silu")], ids=str)
def test_linear_of_large_tiles_fp32(size, act):
    announce(f"linear_act {size} {act} fp32")
    check_linear(linear_case(*size, act, True, True, True, F32), f"{size} {act} fp32")


# ------------------------------------------------------------------------- heads and rotation
GRIDS = {"1": (1,), "grid": (5, 7), "clip": (2, 3, 5), "line": (67,)}


def positions_of(grid, dtype=torch.int32, batch=None, far=0, seed=3):
    at = torch.stack(torch.meshgrid(*(torch.arange(n) for n in GRIDS[grid]), indexing="ij"), dim=-1)
    at = at.reshape(-1, len(GRIDS[grid]))
    g = torch.Generator().manual_seed(seed)
    if batch:
        at = at + torch.randint(0, 1000, (batch, 1, at.shape[-1]), generator=g)
    at = at + far
    if dtype == torch.float32:
        return (at * 0.37 - 2.0).to(dtype).cuda()
    return at.to(dtype).cuda()


HEADS = [  # grid, batch, heads, key heads, channels, axes, far, positions' type, one grid for each row
    ("1", 1, 1, 1, 2, (2,), 0, torch.int32, False),
    ("1", 3, 4, 2, 8, (8,), 2 ** 31 - 1000, torch.int32, False),
    ("line", 2, 3, 1, 16, (10,), 500000, torch.int32, True),
    ("grid", 2, 16, 16, 72, (36, 36), 0, torch.int32, False),
    ("grid", 3, 6, 3, 40, (20, 20), 0, torch.float32, True),
    ("clip", 2, 16, 4, 128, (32, 48, 48), 0, torch.float32, False),
    ("clip", 1, 5, 5, 67, (22, 20, 22), -7, torch.int32, False),
    ("grid", 2, 2, 1, 256, (128, 100), 0, torch.int32, False),
    ("line", 2, 7, 7, 1, (0,), 0, torch.int32, False),
    ("grid", 2, 9, 3, 130, (64, 66), 0, torch.int32, True),
    ("line", 40, 1, 1, 32, (32,), 0, torch.int32, False),
]


def strided(x, how):
    """The same values as a part of a projection, head-major, or packed."""
    if how == "packed":
        return x
    if how == "heads":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    b, n, h, d = x.shape
    whole = torch.full((b, n, h + 3, d + 1), float("nan"), dtype=x.dtype, device=x.device)
    whole[:, :, 1:h + 1, :d] = x
    return whole[:, :, 1:h + 1, :d]


@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (BF16, F32), (F32, F32)], ids=str)
@pytest.mark.parametrize("case", HEADS, ids=str)
def test_heads(case, dtype, weights):
    grid, batch, heads, kv_heads, dim, axes, far, kind, each = case
    positions = positions_of(grid, kind, batch if each else None, far)
    n = positions.shape[-2]
    for layout in ("packed", "part", "heads"):
        announce(f"qk_norm_rotary {case} {layout} {dtype} {weights}")
        sides = [strided(rand(batch, n, h, dim, seed=i, dtype=dtype, std=s), layout).detach().requires_grad_()
                 for i, (h, s) in enumerate(((heads, 1.0), (kv_heads, 3.0)))]
        w = [leaf(rand(dim, seed=5 + i, dtype=weights, std=0.2, mean=1.0)) for i in range(2)]
        out = body.qk_norm_rotary(*sides, *w, positions, axes, THETA, 1e-6)
        grads = [rand(*t.shape, seed=8 + i, dtype=dtype) for i, t in enumerate(out)]
        got = torch.autograd.grad(out, [*sides, *w], grads)
        for i, name in enumerate("qk"):
            want = R.heads(sides[i], w[i], positions, axes, THETA, 1e-6, grads[i])
            assert out[i].is_contiguous()
            R.check(out[i], *want[0], f"{name} of {case} {layout}")
            R.check(got[i], *want[1], f"gradient of {name}, {case} {layout}")
            R.check(got[2 + i], *want[2], f"gradient of {name}_weight, {case} {layout}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", HEADS, ids=str)
def test_rotary(case, dtype):
    grid, batch, heads, _, dim, axes, far, kind, each = case
    positions = positions_of(grid, kind, batch if each else None, far)
    for layout in ("packed", "part", "heads"):
        announce(f"axis_rotary {case} {layout} {dtype}")
        x = strided(rand(batch, positions.shape[-2], heads, dim, dtype=dtype), layout).detach().requires_grad_()
        y = body.axis_rotary(x, positions, axes, THETA)
        grad = rand(*y.shape, seed=2, dtype=dtype)
        (dx,) = torch.autograd.grad(y, x, grad)
        for name, got, want in zip(("result", "gradient"), (y, dx), R.rotary(x, positions, axes, THETA, grad)):
            R.check(got, *want, f"{name} of {case} {layout}")


# ------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (5, 7), (2, 129, 67), (4, 256, 1152)], ids=str)
@pytest.mark.parametrize("p,seed,stream", [(0.1, 7, 0), (0.0, 1, 1), (0.5, -3, 2 ** 40 + 5), (0.999, 2 ** 62 + 11, 3)])
def test_dropout(shape, p, seed, stream, dtype):
    announce(f"dropout {shape} {p} {seed} {stream} {dtype}")
    t = R.half(dtype)
    x, residual, grad = (rand(*shape, seed=i, dtype=dtype) for i in range(3))
    key = torch.tensor([seed], device="cuda")
    keep = R.mask(x.numel(), p, seed, stream).reshape(shape).cuda()
    scale = 1.0 / (1.0 - p)
    for add in (None, residual):
        lx, lr = leaf(x), leaf(add)
        y = body.dropout(lx, p, key, stream, lr)
        dropped = torch.where(keep, x.double() * scale, 0.0)
        want = dropped if add is None else dropped + add.double()
        R.check(y, want, 4 * R.F32 * (dropped.abs() + want.abs()) + t * want.abs() * 1.001, f"dropout {shape}")
        got = torch.autograd.grad(y, [lx] if add is None else [lx, lr], grad)
        want = torch.where(keep, grad.double() * scale, 0.0)
        R.check(got[0], want, (2 * R.F32 + t * 1.001) * want.abs(), f"gradient of dropout {shape}")
        assert torch.equal(got[0] == 0, ~keep | (grad == 0))
        assert add is None or torch.equal(got[1], grad)


def test_dropout_drops_what_is_not_finite():
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 64, device="cuda")
    keep = R.mask(256, 0.5, 5, 0).cuda()
    y = body.dropout(x, 0.5, torch.tensor([5], device="cuda"))
    assert torch.equal(y[~keep], torch.zeros_like(y[~keep]))
    assert torch.equal(y[keep].nan_to_num(7.0), (x[keep] * 2).nan_to_num(7.0))


def test_dropout_past_32_bits():
    count = 2 ** 32 + 1003
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.ones(count, device="cuda", dtype=BF16)
    y = body.dropout(x, 0.25, torch.tensor([9], device="cuda"), 4)
    first = 2 ** 32 - 1000
    keep = R.mask(count - first, 0.25, 9, 4, first).cuda()
    assert torch.equal(y[first:] != 0, keep)
    assert torch.equal(y[:1000] != 0, R.mask(1000, 0.25, 9, 4).cuda())
