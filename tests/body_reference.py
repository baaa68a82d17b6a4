"""The body operators from their definitions in 64 bits, and how far a kernel's results may be off.

A bound is made with the result, element by element: `half(t)` is half a step of a rounding to t
relative to the value; a sum of n products in fp32 in any order is off by at most n + 4 half steps of
fp32 of the sum of their magnitudes; an error of a factor reaches the result times the other
factor. The kernels' exponential and reciprocal are good to 2^-20 (they are of 2 and 1 ulp, and the
argument's rounding moves exp(v) by |v| 2^-24, for |v| < 16).
"""
from __future__ import annotations

import numpy as np
import torch

F32 = 2.0 ** -24
FUNCTION = 2.0 ** -20


def half(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    got, want, bound = (t.detach().double().cpu() for t in (got, want, bound))
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    off = (got - want).abs()
    bad = ~(off <= bound + 1e-30)
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values are off, the first at {at}: "
                             f"{float(got[at])!r} for {float(want[at])!r}, allowed {float(bound[at]):.3g}")


def linear(x, weight, bias, act, gate, residual, grad):
    """[(result, bound), ...] of the result and the gradients of x, weight, bias, gate, residual
    (None in a missing one's place). All on one device, in the type under test."""
    t = half(x.dtype)
    dtype64 = lambda v: None if v is None else v.detach().double()  # noqa: E731
    shape = x.shape
    x, weight, bias, gate, residual, grad = map(dtype64, (x, weight, bias, gate, residual, grad))
    rows, inner = x.numel() // shape[-1], shape[-1]
    outer = weight.shape[0] // (2 if act == "swiglu" else 1)
    x2, g2 = x.reshape(rows, inner), grad.reshape(rows, outer)
    each = max(rows // max(shape[0], 1), 1)
    gates = None if gate is None else gate.repeat_interleave(each, dim=0)
    b = 0.0 if bias is None else bias
    h = x2 @ weight.t() + b
    eh = (inner + 4) * F32 * (x2.abs() @ weight.abs().t() + (0.0 if bias is None else bias.abs()))

    def activated(h, eh):
        """(u, its error, du/dh's parts, their errors) for an h that is off by eh."""
        if act == "none":
            return h, eh, [torch.ones_like(h)], [torch.zeros_like(h)]
        a = h[:, :outer]
        sigma = torch.sigmoid(a)
        silu, slope = a * sigma, sigma * (1 + a * (1 - sigma))
        ea = eh[:, :outer]
        # |silu'| <= 1.1, |silu''| <= 0.5; the functions' own errors, of values up to |a| + 1
        es, ed = 1.1 * ea + FUNCTION * silu.abs(), 0.5 * ea + 4 * FUNCTION * (1 + a.abs()) * sigma
        if act == "silu":
            return silu, es, [slope], [ed]
        c, ec = h[:, outer:], eh[:, outer:]
        return (silu * c, es * c.abs() + silu.abs() * ec + es * ec + F32 * (silu * c).abs(),
                [slope * c, silu], [ed * c.abs() + slope.abs() * ec + ed * ec, es])

    u, eu, _, _ = activated(h, eh)
    y, ey = u, eu
    if gate is not None:
        y, ey = y * gates, ey * gates.abs() + F32 * (y * gates).abs()
    if residual is not None:
        r = residual.reshape(rows, outer)
        y, ey = y + r, ey + F32 * (y + r).abs()
    out = [(y.reshape(*shape[:-1], outer), (ey + t * (y.abs() + ey)).reshape(*shape[:-1], outer))]

    # the backward: h is kept rounded, and so is its gradient, as the products' operand
    kept = act != "none" or gate is not None
    eh = eh + t * (h.abs() + eh) if kept else eh
    u, eu, slopes, eslopes = activated(h, eh)
    du = g2 if gate is None else g2 * gates
    dh = torch.cat([du * s for s in slopes], dim=1)
    edh = torch.cat([du.abs() * e for e in eslopes], dim=1) + 4 * F32 * dh.abs()
    db, edb = dh.sum(0), edh.sum(0) + (rows + 4) * F32 * (dh.abs() + edh).sum(0)
    if kept:
        edh = edh + t * (dh.abs() + edh)
    mag = dh.abs() + edh
    for value, error in ((dh @ weight, edh @ weight.abs() + (dh.shape[1] + 4) * F32 * (mag @ weight.abs())),
                         (dh.t() @ x2, edh.t() @ x2.abs() + (rows + 4) * F32 * (mag.t() @ x2.abs()))):
        out.append((value, error + t * (value.abs() + error)))
    out[1] = tuple(v.reshape(shape) for v in out[1])
    out.append((db, edb + t * (db.abs() + edb)) if bias is not None else None)
    if gate is None:
        out.append(None)
    else:
        terms, errors = g2 * u, g2.abs() * eu
        errors = errors + (each + 4) * F32 * (terms.abs() + errors)
        value, error = (v.reshape(shape[0], each, outer).sum(1) if rows else torch.zeros_like(gate)
                        for v in (terms, errors))
        out.append((value, error + t * (value.abs() + error)))
    out.append(None if residual is None else (grad, torch.zeros_like(grad)))
    return out


def turned(x, positions, axes, theta, sign=1.0):
    """The rotation, as complex products."""
    parts, start = [], 0
    for i, width in enumerate(axes):
        z = torch.view_as_complex(x[..., start:start + width].reshape(*x.shape[:-1], width // 2, 2).contiguous())
        rate = theta ** (-2.0 * torch.arange(width // 2, dtype=torch.float64, device=x.device) / max(width, 1))
        angle = sign * positions[..., i, None, None].double() * rate
        parts.append(torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)).reshape(*x.shape[:-1], width))
        start += width
    return torch.cat([*parts, x[..., start:]], dim=-1)


def pair_norm(x, axes):
    """Of every channel: the length of the pair that it turns in (its own magnitude past the axes)."""
    n = sum(axes)
    pairs = x[..., :n].reshape(*x.shape[:-1], n // 2, 2).norm(dim=-1).repeat_interleave(2, dim=-1)
    return torch.cat([pairs, x[..., n:].abs()], dim=-1)


# cos and sin are rounded to fp32, of an angle that is off by 2^-24 of a half turn, and the turned pair has
# three more roundings: 8 half steps of the pair's length
TURN = 8 * F32


def rotary(x, positions, axes, theta, grad):
    t = half(x.dtype)
    x, grad = x.detach().double(), grad.detach().double()
    out = []
    for v, sign in ((x, 1.0), (grad, -1.0)):
        y = turned(v, positions, axes, theta, sign)
        out.append((y, TURN * pair_norm(v, axes) + t * y.abs() * 1.001))
    return out


def heads(x, weight, positions, axes, theta, eps, grad):
    """[(y, bound), (dx, bound), (dweight, bound)] of one side."""
    t, tw, dim = half(x.dtype), half(weight.dtype), x.shape[-1]
    x, w, grad = x.detach().double(), weight.detach().double(), grad.detach().double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = x * r
    er = (dim / 2 + 8) * F32  # of r, relative: the sum of squares' error halves; root and division
    n = hat * w
    y = turned(n, positions, axes, theta)
    out = [(y, (TURN + er + 4 * F32) * pair_norm(n, axes) + t * y.abs() * 1.001)]
    dn = turned(grad, positions, axes, theta, -1.0)
    edn = TURN * pair_norm(grad, axes)
    dhat = dn * w
    mean = (dhat * hat).mean(-1, keepdim=True)
    mag = (dhat * hat).abs().mean(-1, keepdim=True)
    edhat = edn * w.abs() + F32 * dhat.abs()
    emean = (edhat * hat.abs()).mean(-1, keepdim=True) + (er + (dim + 8) * F32) * mag
    dx = r * (dhat - hat * mean)
    edx = r * (edhat + hat.abs() * emean) + (2 * er + 8 * F32) * r * (dhat.abs() + (hat * mean).abs())
    out.append((dx, edx + t * (dx.abs() + edx)))
    terms = dn * hat
    count = terms.numel() // dim
    eterms = edn * hat.abs() + (er + 4 * F32 + (count + 64) * F32) * terms.abs()
    dw, edw = terms.sum((0, 1, 2)), eterms.sum((0, 1, 2))
    out.append((dw, edw + tw * (dw.abs() + edw)))
    return out


def philox(counter: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """The blocks of counters [n, 4] (uint32 values in uint64) under a key, 10 rounds: [n, 4]."""
    low, shift = np.uint64(0xffffffff), np.uint64(32)
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & low, (a >> shift) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return np.stack(c, axis=1)


def mask(count: int, p: float, seed: int, stream: int, first: int = 0) -> torch.Tensor:
    """Which of the elements first .. first + count - 1 (first a multiple of 4) are kept."""
    block = np.arange(first // 4, (first + count + 3) // 4, dtype=np.uint64)
    low, shift = np.uint64(0xffffffff), np.uint64(32)
    counter = np.stack([block & low, block >> shift, np.full_like(block, stream & 0xffffffff),
                        np.full_like(block, stream >> 32)], axis=1)
    key = seed & ((1 << 64) - 1)
    words = philox(counter, (key & 0xffffffff, key >> 32)).reshape(-1)[:count]
    return torch.from_numpy(words >= np.uint64(min(round(p * 2 ** 32), 2 ** 32 - 1)))
