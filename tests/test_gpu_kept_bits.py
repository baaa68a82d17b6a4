"""GPU: the 20 bits of h that linear_act keeps in bfloat16 before an activation's slope, where they are written and
where they are read.

The products of bfloat16 values are exact in fp32 and a sum of n of them, with the bias, is off by at most n + 4
half steps of fp32 of the terms' magnitudes, in any order; rounding to 20 bits adds 2^-12 of the value. The
exponential and the reciprocal in the sigmoid are good to (2 |v| + 8) 2^-24."""
from __future__ import annotations

import ctypes

import pytest
import torch

import body_reference as R
import kept_bits as K
from helpers import announce
from sihc_hip import _lib, body

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def normal(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(shape, generator=g)).to(BF16).cuda()


def workspace(rows, inner, outer, act):
    sizes = _lib.Linear(rows, inner, outer, {"silu": 1, "swiglu": 2}[act], 1, rows, 0)
    return _lib.lib().sihc_linear_act_workspace_size(ctypes.byref(sizes))


# rows, inner, outer; what the product is: small ones (a block's waves share the contraction), parts of the contraction
# that are joined, and tiles of several sizes, whole and ragged
SIZES = [(1, 8, 8, "small"), (2, 64, 13, "small"), (37, 203, 67, "small"), (16, 1152, 200, "small"),
         (512, 16384, 1024, "joined"), (130, 12000, 333, "joined"), (16384, 768, 2048, "tile"), (8192, 520, 1030, "tile"),
         (4099, 264, 1001, "tile"), (9000, 72, 40, "tile")]


@pytest.mark.parametrize("act", ["silu", "swiglu"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_what_is_written(size, act):
    rows, inner, outer, kind = size
    announce(f"linear_act keeps h of {size} {act}")
    if kind != "small":
        assert (workspace(rows, inner, outer, act) > 0) == (kind == "joined")
    parts = 2 if act == "swiglu" else 1
    x, w = normal(1, rows, inner), normal(parts * outer, inner, seed=1, std=inner ** -0.5)
    b = normal(parts * outer, seed=2)
    y, h, low = body._linear_act(x, w, b, act, normal(1, outer, seed=3), None)
    assert h.shape == (1, rows, parts * outer) and low.shape == (1, rows, parts, (outer + 7) // 8)
    got = K.unpack(h[0], low[0]).double()
    # (all columns of some rows: a whole product in 64 bits would be the test's own bottleneck)
    some = torch.unique(torch.cat([torch.arange(min(rows, 64)), torch.arange(max(rows - 300, 0), rows),
                                   torch.randint(0, rows, (400,), generator=torch.Generator().manual_seed(4))])).cuda()
    want = x[0, some].double() @ w.double().t() + b.double()
    error = (inner + 4) * R.F32 * (x[0, some].double().abs() @ w.double().abs().t() + b.double().abs())
    R.check(got[some], want, error + K.HALF * (want.abs() + error), f"h of {size} {act}")


def test_rounding_is_not_one_sided():
    """Whole numbers, whose products' sums fp32 holds exactly. The errors are at most half a step each, and their mean
    over 2^20 values lies within six standard deviations (1 / sqrt(3 n) half steps, if they are spread evenly) of none."""
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randint(-255, 256, shape, generator=g).to(BF16).cuda() for shape in ((1, 1024, 64), (1024, 64)))
    _, h, low = body._linear_act(x, w, None, "silu", None, None)
    want = x[0].double() @ w.double().t()
    got = K.unpack(h[0], low[0]).double()
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(1.0)))) * K.HALF
    errors = (got.abs() - want.abs()) / half
    assert float(errors.abs().max()) <= 1 and abs(float(errors.mean())) <= 6 / (3 * 2 ** 20) ** 0.5


MOST = (2 - 2.0 ** -7) * 2.0 ** 127  # bfloat16's largest


@pytest.mark.parametrize("first,second", [(float("inf"), 0.0), (-float("inf"), 0.0), (float("nan"), 0.0), (0.0, 0.0),
                                          (MOST, 2.0 ** 120 * 255 / 256), (-MOST, -(2.0 ** 120) * 255 / 256), (2.0 ** -126, 0.0)])
def test_values_at_the_ends_of_the_range(first, second):
    """Infinities and NaN stay what they are, and what would round past fp32's largest value stays finite."""
    w = torch.tensor([[first, second]], device="cuda").to(BF16)
    _, h, low = body._linear_act(torch.ones(1, 1, 2, device="cuda", dtype=BF16), w, None, "silu", None, None)
    got, want = K.unpack(h[0], low[0]).double()[0, 0], w.double().sum()
    assert w.double().tolist() == [[first, second]] or first != first
    if torch.isfinite(want):
        assert abs(float(got) - float(want)) <= 2 * K.HALF * abs(float(want))
    else:
        assert got.isnan() == want.isnan() and (want.isnan() or got == want)


@pytest.mark.parametrize("act", ["silu", "swiglu"])
@pytest.mark.parametrize("outer", [8, 1, 13, 67, 264, 300])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 1), (2, 9), (1, 130)])
def test_what_is_read(batch, tokens, outer, act):
    """The sums of the slopes and of the gate's terms from given bits, which no product has rounded again; with
    all sorts of bits behind the last channel."""
    announce(f"linear_act_backward reads {batch} x {tokens} x {outer} {act}")
    parts, rows = 2 if act == "swiglu" else 1, batch * tokens
    g = torch.Generator().manual_seed(rows + outer)
    values = (2 * torch.randn(rows, parts * outer, generator=g)).cuda()
    h, low = K.pack(values, parts)
    values = K.unpack(h, low).double()
    if outer % 8:
        low[:, :, -1] |= (-1 << (4 * (outer % 8)))
    x, w = normal(batch, tokens, 16), normal(parts * outer, 16, seed=1)
    gate, grad = normal(batch, outer, seed=2), normal(batch, tokens, outer, seed=3)
    _, _, db, dg = body._linear_act_backward(grad, x, w, h.reshape(batch, tokens, -1), low.reshape(batch, tokens, parts, -1),
                                             gate, act, False, False, True, True)
    a = values[:, :outer]
    sigma = torch.sigmoid(a)
    esigma = (2 * a.abs() + 8) * R.F32  # relative; 1 - sigma is off by that of sigma
    g64, gates = grad.reshape(rows, outer).double(), gate.double().repeat_interleave(tokens, 0)
    du = g64 * gates
    slope = sigma * (1 + a * (1 - sigma))
    eslope = sigma * (esigma * (1 + 2 * a.abs()) + 4 * R.F32 * (1 + a.abs()))
    u, eu = a * sigma, a.abs() * sigma * (esigma + 2 * R.F32)
    if act == "swiglu":
        c = values[:, outer:]
        dh, edh = torch.cat([du * c * slope, du * u], 1), torch.cat([(du * c).abs() * eslope, du.abs() * eu], 1)
        u, eu = u * c, eu * c.abs()
    else:
        dh, edh = du * slope, du.abs() * eslope
    edh = edh + 4 * R.F32 * dh.abs()
    t = R.half(BF16)
    want, error = dh.sum(0), edh.sum(0) + (rows + 8) * R.F32 * (dh.abs() + edh).sum(0)
    R.check(db, want, error + t * (want.abs() + error), "bias")
    terms, eterms = g64 * u, g64.abs() * eu + 4 * R.F32 * (g64 * u).abs()
    error = (eterms + (tokens + 8) * R.F32 * (terms.abs() + eterms)).reshape(batch, tokens, outer).sum(1)
    want = terms.reshape(batch, tokens, outer).sum(1)
    R.check(dg, want, error + t * (want.abs() + error), "gate")


# |v| of 20 to 80, where the exponential's rounded argument is off by the most: the sigmoid and what is made of it
@pytest.mark.parametrize("act", ["silu", "swiglu"])
def test_far_slopes_in_fp32(act):
    v = torch.cat([torch.linspace(-80, -20, 1001), torch.linspace(20, 80, 1001), torch.linspace(-20, 20, 1001)]).cuda()
    x = v.reshape(1, -1, 1).contiguous().requires_grad_()
    w = torch.ones(2 if act == "swiglu" else 1, 1, device="cuda")
    b = torch.tensor([0.0, 1.0], device="cuda") if act == "swiglu" else None
    if act == "swiglu":
        w[1] = 0.0  # the second half is 1
    y = body.linear_act(x, w, b, act)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    a = v.double()
    sigma = torch.sigmoid(a)
    error = (2 * a.abs() + 8) * R.F32
    want, slope = a * sigma, sigma * (1 + a * (1 - sigma))
    assert ((y.reshape(-1) - want).abs() <= want.abs() * (error + 2 * R.F32)).all()
    # (1 - sigma is off by what sigma is off by, and where a is large by half a step of 1)
    assert ((dx.reshape(-1) - slope).abs() <= sigma * (error * (1 + 2 * a.abs()) + 6 * R.F32 * (1 + a.abs()))).all()
