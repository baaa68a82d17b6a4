"""The operators of a block's body, as cases that can be timed.

Every case is one pass through a public entry point of `sihc_hip`, as a training or sampling
program calls it, or through the same operator in plain torch operations in 32 bits:

    linear   linear_act: a projection with its bias, an activation (SiLU or SwiGLU), an image's
             gate and a residual
    heads    qk_norm_rotary: the RMS norm of every query and key head and the rotation by the
             token's positions on one to three axes
    rotary   axis_rotary: the rotation alone
    dropout  dropout: a mask from a counter-based generator, with a residual

`train` cases return the output and every gradient, the others the output alone. Gradients come
from torch.autograd.grad, which returns them without accumulating. The sizes are those of this
repository's denoisers (768 channels and a SwiGLU of 2048, 1024 and one of 2730, 1152 in 16 heads
of 72, a 16 x 16 workspace) and generic ones between them.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6
_THETA = 10000.0


def _linear(batch, tokens, inner, outer, act="none", gate=False, residual=False, dtype="bf16", train=False):
    return {"kind": "linear", "batch": batch, "tokens": tokens, "inner": inner, "outer": outer, "act": act,
            "gate": gate, "residual": residual, "dtype": dtype, "train": train}


def _heads(batch, grid, heads, kv_heads, dim, axes, far=0, scaled=False, dtype="bf16", train=False):
    """grid: the workspace's extent on each axis, "16,16"; axes: the channels that each axis turns."""
    return {"kind": "heads", "batch": batch, "grid": grid, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "axes": axes, "far": far, "scaled": scaled, "dtype": dtype, "train": train}


def _rotary(batch, grid, heads, dim, axes, far=0, scaled=False, dtype="bf16", train=False):
    return {"kind": "rotary", "batch": batch, "grid": grid, "heads": heads, "dim": dim, "axes": axes, "far": far,
            "scaled": scaled, "dtype": dtype, "train": train}


def _dropout(batch, tokens, channels, p, residual=False, dtype="bf16", train=True):
    return {"kind": "dropout", "batch": batch, "tokens": tokens, "channels": channels, "p": p,
            "residual": residual, "dtype": dtype, "train": train}


def listed() -> list[dict]:
    def named(name, case):
        return {"name": name, **case}

    return [
        # the modulation of the two halves of one guided image, XL: two rows, the weights' bytes
        named("linear_modulation", _linear(2, 1, 1152, 6912)),
        # the attention's projection in a sampling step of 64 images, XL: gate and residual
        named("linear_sample", _linear(64, 256, 1152, 1152, "none", True, True)),
        # the first product of a training step's SwiGLU, B
        named("linear_swiglu_train", _linear(64, 256, 768, 2048, "swiglu", train=True)),
        # the second one, L: 2730 channels, rows that are not whole vectors
        named("linear_ragged_train", _linear(32, 256, 2730, 1024, "none", True, train=True)),
        # a small fp32 model of odd sizes
        named("linear_train_fp32", _linear(3, 147, 203, 331, "silu", True, True, "fp32", True)),
        # one guided image's queries and keys, XL: latency
        named("heads_sample", _heads(2, "16,16", 16, 16, 72, "36,36")),
        # a training step's, XL
        named("heads_train", _heads(64, "16,16", 16, 16, 72, "36,36", train=True)),
        # a training step on clips: time, height and width, shared key heads, scaled positions
        named("heads_train_video", _heads(4, "8,32,32", 16, 4, 128, "32,48,48", scaled=True, train=True)),
        # one token per sequence far along one axis: serving
        named("rotary_token", _rotary(8, "1", 16, 128, "128", far=500000)),
        # a training step on clips in fp32, part of each head turned
        named("rotary_train_fp32", _rotary(4, "8,24,24", 12, 64, "16,20,20", dtype="fp32", train=True)),
        # a training step's update, XL
        named("dropout_train", _dropout(64, 256, 1152, 0.1, True)),
        # a small fp32 model of odd sizes
        named("dropout_train_fp32", _dropout(3, 147, 67, 0.25, False, "fp32")),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("linear", "linear", "heads", "rotary", "dropout"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    train = rng.random() < 0.6
    if kind == "linear":
        inner, outer = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
        if rng.random() < 0.6:
            inner, outer = -(-inner // 8) * 8, -(-outer // 8) * 8
        act = rng.choice(("none", "none", "silu", "swiglu"))
        tokens = rng.choice((1, 64, 147, 256, 264))
        most = (1 << (33 if dtype == "fp32" else 35)) // (inner * outer * tokens * (2 if act == "swiglu" else 1)) + 1
        return _linear(_spread(rng, 1, min(64, most)), tokens, inner, outer, act, rng.random() < 0.4,
                       rng.random() < 0.4, dtype, train)
    grid, axes = rng.choice((("1", 1), ("509", 1), ("4096", 1), ("16,16", 2), ("31,17", 2), ("64,64", 2),
                             ("8,16,16", 3), ("5,24,40", 3)))
    tokens = math.prod(int(n) for n in grid.split(","))
    if kind == "dropout":
        channels = rng.choice((67, 768, 1024, 1152, 2730))
        return _dropout(_spread(rng, 1, min(64, (1 << 25) // (tokens * channels) + 1)), tokens, channels,
                        rng.choice((0.05, 0.1, 0.25, 0.5)), rng.random() < 0.5, dtype, train)
    dim = rng.choice((32, 40, 64, 72, 80, 96, 128))
    width = dim // axes // 2 * 2 - rng.choice((0, 0, 2))
    widths = ",".join([str(dim - (axes - 1) * width if rng.random() < 0.5 else width)] + [str(width)] * (axes - 1))
    kv_heads = rng.choice((1, 2, 4, 6, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    batch = _spread(rng, 1, min(64, (1 << 26) // (tokens * heads * dim) + 1))
    far, scaled = rng.choice((0, 0, 300000)), rng.random() < 0.3
    if kind == "heads":
        return _heads(batch, grid, heads, kv_heads, dim, widths, far, scaled, dtype, train)
    return _rotary(batch, grid, heads, dim, widths, far, scaled, dtype, train)


# ------------------------------------------------------------------------------------- inputs
def _positions(case, gen):
    """[tokens, axes] of one grid, or [batch, tokens, axes] where every sequence stands elsewhere."""
    extent = [int(n) for n in case["grid"].split(",")]
    at = torch.stack(torch.meshgrid(*(torch.arange(n, device="cuda") for n in extent), indexing="ij"), dim=-1)
    at = at.reshape(-1, len(extent))
    if case["far"]:
        at = at + torch.randint(0, case["far"], (case["batch"], 1, len(extent)), device="cuda", generator=gen)
    if case["scaled"]:
        return at * (0.5 + torch.rand(len(extent), device="cuda", generator=gen))
    return at.to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train, kind, batch = _DTYPES[case["dtype"]], case["train"], case["kind"], case["batch"]

    def normal(*shape, mean=0.0, std=1.0):
        return (mean + std * torch.randn(*shape, device="cuda", generator=gen)).to(dtype)

    state = {**case}
    if kind == "linear":
        inner, outer, tokens = case["inner"], case["outer"], case["tokens"]
        rows = 2 * outer if case["act"] == "swiglu" else outer
        state.update(x=normal(batch, tokens, inner), weight=normal(rows, inner, std=1.0 / math.sqrt(inner)),
                     bias=normal(rows, std=0.1), gate=None, residual=None)
        leaves, shapes = ["x", "weight", "bias"], [(batch, tokens, outer)]
        if case["gate"]:  # one of the modulation's parts
            state["gate"] = normal(batch, 6, outer, std=0.5)[:, 2]
            leaves.append("gate")
        if case["residual"]:
            state["residual"] = normal(batch, tokens, outer)
            leaves.append("residual")
    elif kind in ("heads", "rotary"):
        state["positions"] = _positions(case, gen)
        state["widths"] = tuple(int(n) for n in case["axes"].split(","))
        tokens, heads, dim = state["positions"].shape[-2], case["heads"], case["dim"]
        if kind == "heads":
            kv_heads = case["kv_heads"]
            # parts of one projection, as a block has them
            qkv = normal(batch, tokens, heads + 2 * kv_heads, dim)
            qkv *= 0.5 + torch.rand(heads + 2 * kv_heads, 1, device="cuda", generator=gen)
            state.update(q=qkv[:, :, :heads], k=qkv[:, :, heads:heads + kv_heads],
                         q_weight=normal(dim, mean=1.0, std=0.1), k_weight=normal(dim, mean=1.0, std=0.1))
            leaves = ["q", "k", "q_weight", "k_weight"]
            shapes = [(batch, tokens, heads, dim), (batch, tokens, kv_heads, dim)]
        else:
            state["x"] = normal(batch, tokens, heads, dim)
            leaves, shapes = ["x"], [(batch, tokens, heads, dim)]
    else:
        shape = (batch, case["tokens"], case["channels"])
        state.update(x=normal(*shape), rng=torch.randint(0, 1 << 62, (1,), device="cuda", generator=gen),
                     stream=int(seed) % 7, residual=normal(*shape) if case["residual"] else None)
        leaves, shapes = ["x", "residual"] if case["residual"] else ["x"], [shape]
    if train:
        state["grads"] = [normal(*s) for s in shapes]
        for name in leaves:
            state[name] = state[name].detach().requires_grad_()
    state["leaves"] = leaves
    return state


# --------------------------------------------------------------------------- the plain operators
def _plain_linear(s):
    dtype, act = s["x"].dtype, s["act"]
    x, w = s["x"].float().reshape(-1, s["inner"]), s["weight"].float()
    shape = (s["batch"], s["tokens"], s["outer"])
    h = x @ w.t() + s["bias"].float()
    sigma = None
    if act == "none":
        u = h
    else:
        a = h[:, :s["outer"]]
        sigma = 1.0 / (1.0 + torch.exp(-a))
        u = a * sigma
        if act == "swiglu":
            u = u * h[:, s["outer"]:]
    u = u.reshape(shape)
    gate = None if s["gate"] is None else s["gate"].float()[:, None]
    y = u if gate is None else u * gate
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return y.to(dtype)
    grad = s["grads"][0].float()
    du = (grad if gate is None else grad * gate).reshape(-1, s["outer"])
    if act == "none":
        dh = du
    else:
        slope = sigma * (1.0 + a * (1.0 - sigma))
        dh = du * slope if act == "silu" else torch.cat((du * h[:, s["outer"]:] * slope, du * a * sigma), dim=1)
    out = [y, (dh @ w).reshape(s["x"].shape), dh.t() @ x, dh.sum(0)]
    if gate is not None:
        out.append((grad * u).sum(1))
    if s["residual"] is not None:
        out.append(grad)
    return tuple(t.to(dtype) for t in out)


def _turns(s):
    """cos and sin of every token's angles [.., tokens, 1, pairs], and how many channels they turn."""
    angles = []
    for axis, width in enumerate(s["widths"]):
        rate = _THETA ** (-torch.arange(0, width, 2, dtype=torch.float64, device="cuda") / width)
        angles.append(s["positions"][..., axis, None].double() * rate)
    angle = torch.cat(angles, dim=-1)[..., None, :]
    return angle.cos().float(), angle.sin().float(), sum(s["widths"])


def _turn(x, cos, sin, turned):
    even, odd = x[..., 0:turned:2], x[..., 1:turned:2]
    pairs = torch.stack((even * cos - odd * sin, even * sin + odd * cos), dim=-1).flatten(-2)
    return torch.cat((pairs, x[..., turned:]), dim=-1)


def _plain_heads(s):
    cos, sin, turned = _turns(s)
    dtype = s["q"].dtype
    outs, grads = [], []
    for i, (name, weight) in enumerate((("q", "q_weight"), ("k", "k_weight"))):
        x, w = s[name].float(), s[weight].float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        hat = x * r
        outs.append(_turn(hat * w, cos, sin, turned).to(dtype))
        if s["train"]:
            dn = _turn(s["grads"][i].float(), cos, -sin, turned)
            dhat = dn * w
            dx = r * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
            grads.append((dx.to(dtype), (dn * hat).sum((0, 1, 2)).to(dtype)))
    if not s["train"]:
        return tuple(outs)
    return (*outs, grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _plain_rotary(s):
    cos, sin, turned = _turns(s)
    out = _turn(s["x"].float(), cos, sin, turned).to(s["x"].dtype)
    if not s["train"]:
        return out
    return out, _turn(s["grads"][0].float(), cos, -sin, turned).to(s["x"].dtype)


def _high_product(a: int, b):
    """The upper and the lower 32 bits of a * b for 32-bit values b held in 64."""
    low, high = b & 0xffff, b >> 16
    first, second = a * low, a * high          # < 2^48
    middle = second + (first >> 16)
    return middle >> 16, ((middle & 0xffff) << 16) | (first & 0xffff)


def _bits(count, key, stream):
    """Words 0 .. count - 1 of the generator (Philox 4x32, 10 rounds): word i is part i % 4 of the
    block of counter (i / 4, stream) under the key."""
    mask = 0xffffffff
    block = torch.arange((count + 3) // 4, dtype=torch.int64, device="cuda")
    c = [block & mask, block >> 32, torch.full_like(block, stream & mask), torch.full_like(block, stream >> 32)]
    k0, k1 = key & mask, (key >> 32) & mask
    for _ in range(10):
        h0, l0 = _high_product(0xD2511F53, c[0])
        h1, l1 = _high_product(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack(c, dim=-1).reshape(-1)[:count]


def _plain_dropout(s):
    x, p = s["x"], s["p"]
    keep = (_bits(x.numel(), s["rng"], s["stream"]) >= round(p * (1 << 32))).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return y.to(x.dtype)
    out = (y.to(x.dtype), torch.where(keep, s["grads"][0].float() * scale, 0.0).to(x.dtype))
    return out if s["residual"] is None else (*out, s["grads"][0].clone())


# ----------------------------------------------------------------------------- the entry points
_calls = None


def _package():
    global _calls
    if _calls is None:
        path = str(Path.cwd() / "residual-stream-burden_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from sihc_hip import body as _calls
    return _calls


def run(state: dict):
    s, kind = state, state["kind"]
    if not own:
        with torch.no_grad():
            return {"linear": _plain_linear, "heads": _plain_heads, "rotary": _plain_rotary,
                    "dropout": _plain_dropout}[kind](s)
    c = _package()
    if kind == "linear":
        def call():
            return c.linear_act(s["x"], s["weight"], s["bias"], s["act"], s["gate"], s["residual"])
    elif kind == "heads":
        def call():
            return c.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["widths"],
                                    _THETA, _EPS)
    elif kind == "rotary":
        def call():
            return c.axis_rotary(s["x"], s["positions"], s["widths"], _THETA)
    else:
        def call():
            return c.dropout(s["x"], s["p"], s["rng"], s["stream"], s["residual"])
    if not s["train"]:
        with torch.no_grad():
            return call()
    out = call()
    out = out if isinstance(out, tuple) else (out,)
    return (*(t.detach() for t in out), *torch.autograd.grad(out, [s[n] for n in s["leaves"]], s["grads"]))


# ------------------------------------------------------------------------------ in 64 bits
def _exact_turn(x, s):
    """Each axis' run of channels as complex numbers, multiplied by the angle's."""
    parts, start = [], 0
    for axis, width in enumerate(s["widths"]):
        pairs = torch.view_as_complex(x[..., start:start + width].reshape(*x.shape[:-1], width // 2, 2))
        step = torch.arange(width // 2, dtype=torch.float64, device="cuda")
        angle = s["positions"][..., axis, None, None].double() * torch.exp(step * (-2.0 * math.log(_THETA) / width))
        turned = pairs * torch.polar(torch.ones_like(angle), angle)
        parts.append(torch.view_as_real(turned).reshape(*x.shape[:-1], width))
        start += width
    return torch.cat([*parts, x[..., start:]], dim=-1)


def _exact_keep(s):
    """The mask by Python's and numpy's whole numbers: counters and products as unsigned 64-bit words."""
    import numpy as np

    count, key, stream = s["x"].numel(), int(s["rng"]), s["stream"]
    low = np.uint64(0xffffffff)
    block = np.arange(-(-count // 4), dtype=np.uint64)
    word = [block & low, block >> np.uint64(32), np.full_like(block, stream % (1 << 32)),
            np.full_like(block, stream >> 32)]
    for turn in range(10):
        a, b = word[0] * np.uint64(0xD2511F53), word[2] * np.uint64(0xCD9E8D57)
        first = np.uint64((key % (1 << 32) + turn * 0x9E3779B9) % (1 << 32))
        second = np.uint64((key // (1 << 32) + turn * 0xBB67AE85) % (1 << 32))
        word = [(b >> np.uint64(32)) ^ word[1] ^ first, b & low, (a >> np.uint64(32)) ^ word[3] ^ second, a & low]
    bits = np.stack(word, axis=1).reshape(-1)[:count]
    kept = bits >= np.uint64(round(s["p"] * (1 << 32)))
    return torch.from_numpy(kept).to("cuda").reshape(s["x"].shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, train = case["kind"], case["train"]
    leaf = {n: s[n].detach().double().requires_grad_(train) for n in s["leaves"]}
    with torch.set_grad_enabled(train):
        if kind == "linear":
            h = torch.nn.functional.linear(leaf["x"], leaf["weight"], leaf["bias"])
            if case["act"] == "silu":
                h = torch.nn.functional.silu(h)
            elif case["act"] == "swiglu":
                first, second = h.chunk(2, dim=-1)
                h = torch.nn.functional.silu(first) * second
            if case["gate"]:
                h = leaf["gate"].unsqueeze(1) * h
            outs = (leaf["residual"] + h if case["residual"] else h,)
        elif kind == "heads":
            outs = tuple(_exact_turn(leaf[n] / (leaf[n].pow(2).mean(-1, keepdim=True) + _EPS).sqrt() *
                                     leaf[n + "_weight"], s) for n in ("q", "k"))
        elif kind == "rotary":
            outs = (_exact_turn(leaf["x"], s),)
        else:
            y = leaf["x"] * _exact_keep(s) / (1.0 - case["p"])
            outs = (leaf["residual"] + y if case["residual"] else y,)
    if not train:
        return outs if kind == "heads" else outs[0]
    grads = torch.autograd.grad(outs, list(leaf.values()), [g.double() for g in s["grads"]])
    return (*(t.detach() for t in outs), *grads)


# ------------------------------------------------------------------------- bytes and operations
def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    train, batch = case["train"], case["batch"]
    if case["kind"] == "linear":
        rows, inner, outer = batch * case["tokens"], case["inner"], case["outer"]
        wide = 2 * outer if case["act"] == "swiglu" else outer
        moved = rows * inner + wide * inner + rows * outer * (2 if case["residual"] else 1)
        if train:  # the inputs and the gradient in again, the gradients out
            moved += 2 * (rows * inner + wide * inner) + rows * outer * (2 if case["residual"] else 1)
        return {"bytes": moved * size, "flops": (6 if train else 2) * rows * inner * wide}
    tokens = case["tokens"] if case["kind"] == "dropout" else math.prod(int(n) for n in case["grid"].split(","))
    if case["kind"] == "dropout":
        n = batch * tokens * case["channels"]
        moved = n * (3 if case["residual"] else 2) + (n * (3 if case["residual"] else 2) if train else 0)
        return {"bytes": moved * size, "flops": (6 if train else 3) * n}
    n = batch * tokens * (case["heads"] + case.get("kv_heads", 0)) * case["dim"]
    each = (5 if train else 2) if case["kind"] == "heads" else (4 if train else 2)
    return {"bytes": each * n * size, "flops": n * ((30 if train else 9) if case["kind"] == "heads" else
                                                    (6 if train else 3))}
