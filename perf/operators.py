"""The operators that condition a denoiser on an encoder's states, as cases that can be timed.

Every case is one pass through a public entry point of `sihc_hip`, as a training or sampling
program calls it, or through the same operator in plain torch operations in 32 bits:

    embed    embedding_lookup: token ids (or class labels) to scaled rows of a table; its
             gradient is the whole table's, zero where no token selects a row
    attend   cross_attention: the workspace's tokens over an encoder's states of another length,
             each image with a length of its own (0 and 1 among them)
    norm     group_norm_act: group norm and SiLU over the NHWC carrier

`train` cases return the output and every gradient, the others the output alone. Gradients come
from torch.autograd.grad, which returns them without accumulating. The sizes are those of this
repository's denoisers (768 channels in 12 heads, 1152 in 16, a 16 x 16 workspace, carriers of
32 x 32 and 64 x 64 pixels, 1000 classes and the empty one) and generic ones between them.
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


def _embed(vocab, channels, tokens, dtype="bf16", train=False, skew=1.0, padding=0.0):
    return {"kind": "embed", "vocab": vocab, "channels": channels, "tokens": tokens, "dtype": dtype,
            "train": train, "skew": skew, "padding": padding}


def _attend(batch, queries, keys, heads, kv_heads, dim, dtype="bf16", train=False, empty=0.0):
    return {"kind": "attend", "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train, "empty": empty}


def _norm(batch, edge, channels, groups, dtype="bf16", train=False):
    return {"kind": "norm", "batch": batch, "edge": edge, "channels": channels, "groups": groups,
            "dtype": dtype, "train": train}


def listed() -> list[dict]:
    def named(name, case):
        return {"name": name, **case}

    return [
        # the two prompts of one guided image, embedded before sampling: a latency-bound lookup
        named("embed_prompt", _embed(32768, 768, 154)),
        # the class labels of a training batch in fp32: 1000 classes and the empty one
        named("embed_labels_train", _embed(1001, 1152, 256, "fp32", True)),
        # the captions of a training batch: natural frequencies, half of the positions padding
        named("embed_captions_train", _embed(32768, 1152, 32768, "bf16", True, 3.0, 0.5)),
        # one query token per sequence over long encoder states, shared heads: serving
        named("attend_token", _attend(8, 1, 4096, 16, 4, 128)),
        # a sampling step of 64 guided images, XL: half of the rows have an empty prompt
        named("attend_sample", _attend(128, 256, 128, 16, 16, 72, empty=0.5)),
        # a training step's cross attention, XL
        named("attend_train", _attend(64, 256, 256, 16, 16, 72, "bf16", True, 0.1)),
        # a 64 x 64 carrier's pixels over a long document, shared heads
        named("attend_train_long", _attend(4, 4096, 2048, 16, 4, 64, "bf16", True)),
        # a small fp32 model of odd sizes
        named("attend_train_fp32", _attend(3, 147, 203, 6, 3, 40, "fp32", True, 0.2)),
        # one guided image's 32 x 32 carrier, B: a latency-bound norm
        named("norm_sample", _norm(2, 32, 768, 32)),
        # a sampling step of 64 images on a 64 x 64 carrier, XL
        named("norm_sample_large", _norm(64, 64, 1152, 32)),
        # a training step's norm, XL
        named("norm_train", _norm(64, 32, 1152, 32, "bf16", True)),
        # fp32, an odd width and a 28 x 28 carrier
        named("norm_train_fp32", _norm(5, 28, 136, 8, "fp32", True)),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("embed", "attend", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    train = rng.random() < 0.6
    if kind == "embed":
        vocab, channels = _spread(rng, 10, 60000), rng.choice((64, 67, 320, 768, 1024, 1152))
        return _embed(vocab, channels, _spread(rng, 1, 40000), dtype, train, rng.choice((1.0, 3.0)),
                      rng.choice((0.0, 0.3)))
    if kind == "attend":
        kv_heads = rng.choice((1, 2, 4, 6, 8, 12, 16))
        heads = kv_heads * rng.choice((1, 1, 1, 2, 4)) if kv_heads <= 4 else kv_heads
        dim = rng.choice((32, 40, 64, 72, 80, 96, 128))
        queries, keys = _spread(rng, 1, 4096), _spread(rng, 1, 8192)
        most = (1 << 26 if dtype == "fp32" else 1 << 28) // (heads * queries * keys) + 1
        most = min(most, (1 << 24) // (heads * dim * max(queries, keys)) + 1)
        return _attend(_spread(rng, 1, max(1, min(128, most))), queries, keys, heads, kv_heads, dim, dtype, train,
                       rng.choice((0.0, 0.3)))
    edge = _spread(rng, 1, 64)
    groups, width = rng.choice((1, 4, 8, 16, 32)), rng.choice((1, 4, 8, 17, 24, 32, 36))
    most = (1 << 27) // (edge * edge * groups * width) + 1
    return _norm(_spread(rng, 1, min(256, most)), edge, groups * width, groups, dtype, train)


# ------------------------------------------------------------------------------------- inputs
def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = _DTYPES[case["dtype"]], case["train"]

    def normal(*shape, mean=0.0, std=1.0):
        return (mean + std * torch.randn(*shape, device="cuda", generator=gen)).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    state = {**case}
    if case["kind"] == "embed":
        vocab, tokens = case["vocab"], case["tokens"]
        ids = (vocab * uniform(tokens).pow(case["skew"])).long().clamp_(max=vocab - 1)
        ids = torch.where(uniform(tokens) < case["padding"], vocab - 1, ids)
        state.update(table=normal(vocab, case["channels"], std=0.02), ids=ids.to(torch.int32),
                     scale=math.sqrt(case["channels"]), padding_idx=vocab - 1 if case["padding"] else None)
        leaves, shape = ("table",), (tokens, case["channels"])
    elif case["kind"] == "attend":
        batch, keys, dim = case["batch"], case["keys"], case["dim"]
        # keys and values are the two halves of one projection of the states
        kv = normal(batch, keys, 2, case["kv_heads"], dim)
        lengths = 1 + (keys * uniform(batch).sqrt()).to(torch.int32).clamp_(max=keys - 1)
        lengths = torch.where(uniform(batch) < case["empty"], 0, lengths).to(torch.int32)
        state.update(q=normal(batch, case["queries"], case["heads"], dim), k=kv[:, :, 0], v=kv[:, :, 1],
                     lengths=lengths, scale=1.0 / math.sqrt(dim))
        leaves, shape = ("q", "k", "v"), (batch, case["queries"], case["heads"], dim)
    else:
        batch, edge, channels = case["batch"], case["edge"], case["channels"]
        x = normal(batch, edge, edge, channels)
        x += normal(batch, 1, 1, channels, std=0.5)
        state.update(x=x, weight=normal(channels, mean=1.0, std=0.1), bias=normal(channels, std=0.1))
        leaves, shape = ("x", "weight", "bias"), (batch, edge, edge, channels)
    if train:
        state["grad"] = normal(*shape)
        for name in leaves:
            state[name] = state[name].detach().requires_grad_()
    return state


# --------------------------------------------------------------------------- the plain operators
def _plain_embed(s):
    ids = s["ids"].long()
    out = (s["table"][ids].float() * s["scale"]).to(s["table"].dtype)
    if not s["train"]:
        return out
    rows = s["grad"].float() * s["scale"]
    if s["padding_idx"] is not None:
        rows = rows * (ids != s["padding_idx"])[:, None]
    total = torch.zeros(s["table"].shape, dtype=torch.float32, device=rows.device)
    return out, total.index_add_(0, ids, rows).to(s["table"].dtype)


def _plain_attend(s):
    dtype, batch, queries, heads, dim = s["q"].dtype, *s["q"].shape
    keys, shared = s["k"].shape[1], s["k"].shape[2]
    each = heads // shared

    def by_head(t):  # [batch, queries, heads, dim] -> [batch, shared, each * queries, dim]
        t = t.float().reshape(batch, queries, shared, each, dim).permute(0, 2, 3, 1, 4)
        return t.reshape(batch, shared, each * queries, dim)

    def from_heads(t):
        t = t.reshape(batch, shared, each, queries, dim).permute(0, 3, 1, 2, 4)
        return t.reshape(batch, queries, heads, dim).to(dtype)

    q, k, v = by_head(s["q"]), s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    seen = (torch.arange(keys, device=q.device) < s["lengths"][:, None])[:, None, None, :]
    score = torch.where(seen, (q @ k.transpose(2, 3)) * s["scale"], -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    p = p / p.sum(3, keepdim=True).clamp_min(1e-30)
    out = p @ v
    if not s["train"]:
        return from_heads(out)
    grad = by_head(s["grad"])
    ds = p * (grad @ v.transpose(2, 3) - (grad * out).sum(3, keepdim=True)) * s["scale"]
    dk, dv = ds.transpose(2, 3) @ q, p.transpose(2, 3) @ grad
    return (from_heads(out), from_heads(ds @ k), dk.permute(0, 2, 1, 3).to(dtype).contiguous(),
            dv.permute(0, 2, 1, 3).to(dtype).contiguous())


def _plain_norm(s):
    x, dtype, groups = s["x"], s["x"].dtype, s["groups"]
    batch, channels = x.shape[0], x.shape[-1]
    shape = (batch, -1, groups, channels // groups)
    w, b = (s[n].float().reshape(groups, -1) for n in ("weight", "bias"))
    xf = x.float().reshape(shape)
    mean = xf.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((xf - mean).square().mean((1, 3), keepdim=True) + _EPS)
    hat = (xf - mean) * rstd
    u = hat * w + b
    gate = 1.0 / (1.0 + torch.exp(-u))
    out = (u * gate).to(dtype).reshape(x.shape)
    if not s["train"]:
        return out
    du = s["grad"].float().reshape(shape) * gate * (1.0 + u * (1.0 - gate))
    dw, db = (du * hat).sum((0, 1)), du.sum((0, 1))
    dh = du * w
    dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - hat * (dh * hat).mean((1, 3), keepdim=True))
    return out, dx.to(dtype).reshape(x.shape), dw.reshape(-1).to(dtype), db.reshape(-1).to(dtype)


# ----------------------------------------------------------------------------- the entry points
_calls = None


def _package():
    global _calls
    if _calls is None:
        path = str(Path.cwd() / "residual-stream-burden_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from sihc_hip import conditioning as _calls
    return _calls


def _own_pass(s, call, leaves):
    if not s["train"]:
        with torch.no_grad():
            return call()
    out = call()
    return (out.detach(), *torch.autograd.grad(out, [s[n] for n in leaves], s["grad"]))


def run(state: dict):
    s, kind = state, state["kind"]
    if not own:
        with torch.no_grad():
            return {"embed": _plain_embed, "attend": _plain_attend, "norm": _plain_norm}[kind](s)
    c = _package()
    if kind == "embed":
        return _own_pass(s, lambda: c.embedding_lookup(s["table"], s["ids"], s["scale"], s["padding_idx"],
                                                       validate=False), ("table",))
    if kind == "attend":
        return _own_pass(s, lambda: c.cross_attention(s["q"], s["k"], s["v"], s["lengths"], s["scale"],
                                                      validate=False), ("q", "k", "v"))
    return _own_pass(s, lambda: c.group_norm_act(s["x"], s["weight"], s["bias"], s["groups"], _EPS, "silu"),
                     ("x", "weight", "bias"))


# ------------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind, train = case["kind"], case["train"]
    if kind == "embed":
        table = s["table"].detach().double()
        rows = [table[s["ids"].long()] * s["scale"]]
        if train:
            # sums of each row's run of sorted tokens, as differences of running sums
            total = torch.zeros_like(table)
            keep = torch.ones_like(s["ids"], dtype=torch.bool) if s["padding_idx"] is None else s["ids"] != s["padding_idx"]
            order = torch.argsort(s["ids"].long(), stable=True)
            order = order[keep[order]]
            ids, count = torch.unique_consecutive(s["ids"][order].long(), return_counts=True)
            sums = torch.cat([torch.zeros(1, table.shape[1], dtype=torch.float64, device="cuda"),
                              (s["grad"].double()[order] * s["scale"]).cumsum(0)])
            end = count.cumsum(0)
            total[ids] = sums[end] - sums[end - count]
            rows.append(total)
        return rows[0] if not train else tuple(rows)
    if kind == "attend":
        batch, keys = case["batch"], case["keys"]
        each = case["heads"] // case["kv_heads"]
        outs = []
        for b in range(batch):
            n = int(s["lengths"][b])
            q, k, v = (s[t][b].detach().double().requires_grad_(train) for t in ("q", "k", "v"))
            kk, vv = (t[:n].repeat_interleave(each, dim=1).transpose(0, 1) for t in (k, v))
            p = torch.softmax(q.transpose(0, 1) @ kk.transpose(1, 2) * s["scale"], dim=-1)
            out = (p @ vv).transpose(0, 1) if n else q * 0.0
            row = [out.detach()]
            if train:
                row += (torch.autograd.grad(out, (q, k, v), s["grad"][b].double()) if n else
                        [torch.zeros_like(t) for t in (q, k, v)])
            outs.append(row)
        got = tuple(torch.stack(t) for t in zip(*outs))
        return got if train else got[0]
    outs = []
    w, b = (s[n].detach().double().requires_grad_(train) for n in ("weight", "bias"))
    total = [torch.zeros_like(w), torch.zeros_like(b)]
    for i in range(case["batch"]):
        x = s["x"][i].detach().double().requires_grad_(train)
        y = torch.nn.functional.silu(torch.nn.functional.group_norm(
            x.reshape(1, -1, case["channels"]).transpose(1, 2), case["groups"], w, b, _EPS))
        y = y.transpose(1, 2).reshape(x.shape)
        row = [y.detach()]
        if train:
            dx, dw, db = torch.autograd.grad(y, (x, w, b), s["grad"][i].double())
            row.append(dx)
            total[0] += dw
            total[1] += db
        outs.append(row)
    got = tuple(torch.stack(t) for t in zip(*outs))
    return (*got, *(t.detach() for t in total)) if train else got[0]


# ------------------------------------------------------------------------- bytes and operations
def work(case: dict) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    train = case["train"]
    if case["kind"] == "embed":
        vocab, tokens, channels = case["vocab"], case["tokens"], case["channels"]
        rows = min(vocab, tokens)  # the table's rows that can be read
        moved, flops = (rows + tokens) * channels * size + tokens * 4, tokens * channels
        if train:
            kept = tokens * (1.0 - case["padding"])
            moved, flops = moved + (kept + vocab) * channels * size, 2 * flops
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "attend":
        seen = 0.66 * case["keys"] * (1.0 - case["empty"])  # of each row, on average
        q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
        kv = 2 * case["batch"] * case["kv_heads"] * case["dim"] * seen
        whole = 2 * case["batch"] * case["kv_heads"] * case["dim"] * case["keys"]
        if not train:
            return {"bytes": (2 * q + kv) * size, "flops": 4 * q * seen}
        # forward: q, k, v in, out back; backward: those and the gradient in, three gradients back
        return {"bytes": (6 * q + 2 * kv + whole) * size, "flops": 14 * q * seen}
    n = case["batch"] * case["edge"] ** 2 * case["channels"]
    return {"bytes": (5 if train else 2) * n * size, "flops": (35 if train else 12) * n}
