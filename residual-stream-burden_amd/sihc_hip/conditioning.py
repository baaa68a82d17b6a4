"""Conditioning a denoiser on an encoder's states: embedding lookup, cross attention and group norm.

Specification (the reference conditions on class labels alone and has no such op; its class
table, norms and self attention are plain PyTorch, sihc/models/sihc/components.py:18-30,184-235):

* ``embedding_lookup(table, ids, scale, padding_idx)``: out[n] = scale * table[ids[n]]. The
  gradient of the table is dense: row r gets scale times the sum of the output gradients of the
  tokens that select it, zero where none does, and zero for row ``padding_idx``.
* ``cross_attention(q, k, v, lengths, scale)``: every query row q[b, i, h] attends the first
  ``lengths[b]`` of the keys and values k, v[b, :, h // (H / KH)]: query heads share key heads in
  groups of H / KH, and their gradients are summed. A length of zero gives zeros and no gradient,
  and nothing that k and v hold past a length has an effect, NaN included.
* ``group_norm_act(x, weight, bias, groups, eps, act)``: over a channels-last tensor [B, ..., C],
  act(weight * (x - mean) * rstd + bias) with the mean and variance of each image's groups of
  C / groups adjacent channels: at most 4,096 of them in bfloat16 where 8 divides the width, otherwise
  2,048 of an even width and 1,024 of an odd one, and C at most 2^24.

All sums and statistics are fp32, in a fixed order without atomics on values: identical inputs
give identical bits. float32 and bfloat16; the norm's weights may be float32 beside a bfloat16
input. The kernels read q, k and v through their strides (the channels of a head adjacent); other
tensors are packed. Values of ids and lengths are checked on the host (a device-to-host sync);
pass ``validate=False`` in hot loops once they are known good. The kernels clamp ids to the last
row and lengths to [0, Lk], so that no access can leave a tensor.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor
from torch.library import custom_op, register_autograd

from . import launch
from ._lib import MAX_HEAD_DIM
from ._native import native
from .sublayer_kernels import _require_packed

_TYPES = (torch.float32, torch.bfloat16)


def _require_gpu(op_name: str, first: Tensor, **others: Tensor) -> None:
    if not first.is_cuda or any(t.device != first.device for t in others.values()):
        raise ValueError(f"{op_name}: tensors must share one CUDA device")


# ------------------------------------------------------------------------- embedding lookup
def _check_embedding(table: Tensor, ids: Tensor) -> None:
    _require_packed("embedding_lookup", table=table, ids=ids)
    if table.ndim != 2 or 0 in table.shape:
        raise ValueError(f"embedding_lookup: expected a [rows, channels] table, got {tuple(table.shape)}")
    if table.dtype not in _TYPES:
        raise ValueError("embedding_lookup: table dtype must be float32 or bfloat16")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"embedding_lookup: ids must be int32 or int64, got {ids.dtype}")
    _require_gpu("embedding_lookup", table, ids=ids)


@custom_op("sihc::embedding_lookup", mutates_args=())
def _embedding_lookup(table: Tensor, ids: Tensor, scale: float, padding: int) -> Tensor:
    _check_embedding(table, ids)
    return launch.embedding(table, ids, scale)


@_embedding_lookup.register_fake
def _embedding_lookup_fake(table, ids, scale, padding):
    return table.new_empty((*ids.shape, table.shape[1]))


@custom_op("sihc::embedding_lookup_backward", mutates_args=())
def _embedding_lookup_backward(grad: Tensor, ids: Tensor, rows: int, scale: float, padding: int) -> Tensor:
    _require_packed("embedding_lookup backward", grad=grad, ids=ids)
    if grad.shape[:-1] != ids.shape or grad.dtype not in _TYPES or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("embedding_lookup backward: the output gradient must match the ids")
    _require_gpu("embedding_lookup backward", grad, ids=ids)
    return launch.embedding_backward(grad, ids, rows, scale, padding)


@_embedding_lookup_backward.register_fake
def _embedding_lookup_backward_fake(grad, ids, rows, scale, padding):
    return grad.new_empty((rows, grad.shape[-1]))


def _embedding_setup(ctx, inputs, output):
    table, ids, ctx.scale, ctx.padding = inputs
    ctx.rows = table.shape[0]
    ctx.save_for_backward(ids)


def _embedding_autograd(ctx, grad):
    (ids,) = ctx.saved_tensors
    return _embedding_lookup_backward(grad.contiguous(), ids, ctx.rows, ctx.scale, ctx.padding), None, None, None


register_autograd(_embedding_lookup, _embedding_autograd, setup_context=_embedding_setup)
native(_embedding_lookup, "embedding_lookup")


def embedding_lookup(table: Tensor, ids: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None, *,
                     validate: bool = True) -> Tensor:
    """scale * table[ids] as [*ids.shape, C]; row `padding_idx` of the table gets no gradient."""
    if validate:
        _check_embedding(table, ids)
        if padding_idx is not None and not -table.shape[0] <= padding_idx < table.shape[0]:
            raise ValueError(f"embedding_lookup: padding_idx {padding_idx} is not a row of the table")
        if ids.numel():
            low, high = int(ids.min()), int(ids.max())
            if low < 0 or high >= table.shape[0]:
                raise ValueError(f"embedding_lookup: ids must lie in [0, {table.shape[0]}), got [{low}, {high}]")
    padding = -1 if padding_idx is None else padding_idx if padding_idx >= 0 else padding_idx + table.shape[0]
    return _embedding_lookup(table, ids, scale, padding)


# ------------------------------------------------------------------------ group norm and act
def _widest_group(width: int, dtype: torch.dtype) -> int:
    """The most channels of a group of such a width: a block takes a pixel's part of one in vectors."""
    return 4096 if dtype == torch.bfloat16 and width % 8 == 0 else 2048 if width % 2 == 0 else 1024


def _check_group_width(x: Tensor, groups: int) -> None:
    if x.shape[-1] > 1 << 24:
        raise ValueError(f"group_norm_act: at most {1 << 24} channels, got {x.shape[-1]}")
    width = x.shape[-1] // max(groups, 1)
    if width > _widest_group(width, x.dtype):
        raise ValueError(f"group_norm_act: groups of {width} channels, at most {_widest_group(width, x.dtype)} of "
                         f"that width and type")


def _check_norm(x: Tensor, weight: Tensor, bias: Tensor, groups: int, act: str) -> None:
    _require_packed("group_norm_act", x=x, weight=weight, bias=bias)
    if x.ndim < 2:
        raise ValueError(f"group_norm_act: expected [batch, ..., channels], got {tuple(x.shape)}")
    channels = x.shape[-1]
    if groups < 1 or channels < 1 or channels % groups:
        raise ValueError(f"group_norm_act: {channels} channels cannot be cut into {groups} groups")
    _check_group_width(x, groups)
    if weight.shape != (channels,) or bias.shape != (channels,):
        raise ValueError("group_norm_act: weight and bias must be [channels]")
    if x.dtype not in _TYPES or weight.dtype != bias.dtype or weight.dtype not in (x.dtype, torch.float32):
        raise ValueError("group_norm_act: float32 or bfloat16, with weights of the input's type or float32")
    if act not in launch.ACTIVATIONS:
        raise ValueError(f"group_norm_act: act must be one of {sorted(launch.ACTIVATIONS)}, got {act!r}")
    _require_gpu("group_norm_act", x, weight=weight, bias=bias)


@custom_op("sihc::group_norm_act", mutates_args=())
def _group_norm_act(x: Tensor, weight: Tensor, bias: Tensor, groups: int, eps: float,
                    act: str) -> tuple[Tensor, Tensor]:
    _check_norm(x, weight, bias, groups, act)
    return launch.group_norm(x, weight, bias, groups, eps, act)


@_group_norm_act.register_fake
def _group_norm_act_fake(x, weight, bias, groups, eps, act):
    _check_group_width(x, groups)
    return torch.empty_like(x), x.new_empty((x.shape[0], groups, 2), dtype=torch.float32)


@custom_op("sihc::group_norm_act_backward", mutates_args=())
def _group_norm_act_backward(grad: Tensor, x: Tensor, weight: Tensor, bias: Tensor, stats: Tensor, groups: int,
                             act: str) -> tuple[Tensor, Tensor, Tensor]:
    _check_norm(x, weight, bias, groups, act)  # saved tensors come back through the caller's hooks
    _require_packed("group_norm_act backward", grad=grad, stats=stats)
    if grad.shape != x.shape or grad.dtype != x.dtype or stats.shape != (x.shape[0], groups, 2):
        raise ValueError("group_norm_act backward: the output gradient must match the output")
    _require_gpu("group_norm_act backward", x, grad=grad, stats=stats)
    return launch.group_norm_backward(grad, x, weight, bias, stats, groups, act)


@_group_norm_act_backward.register_fake
def _group_norm_act_backward_fake(grad, x, weight, bias, stats, groups, act):
    return torch.empty_like(x), torch.empty_like(weight), torch.empty_like(bias)


def _norm_setup(ctx, inputs, output):
    x, weight, bias, ctx.groups, _, ctx.act = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)  # zeros for the statistics' gradient would be a launch
    ctx.save_for_backward(x, weight, bias, output[1])


def _norm_autograd(ctx, grad, _):
    if grad is None:
        return (None,) * 6
    x, weight, bias, stats = ctx.saved_tensors
    return (*_group_norm_act_backward(grad.contiguous(), x, weight, bias, stats, ctx.groups, ctx.act), None, None,
            None)


register_autograd(_group_norm_act, _norm_autograd, setup_context=_norm_setup)
native(_group_norm_act, "group_norm_act")


def group_norm_act(x: Tensor, weight: Tensor, bias: Tensor, groups: int = 32, eps: float = 1e-6,
                   act: str = "silu") -> Tensor:
    """act(group norm) of a packed channels-last tensor [B, ..., C]; act is "silu" or "none"."""
    return _group_norm_act(x, weight, bias, groups, eps, act)[0]


# ----------------------------------------------------------------------------- cross attention
def _check_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor]) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape:
        raise ValueError("cross_attention: expected q [B, Lq, H, D] and k, v [B, Lk, KH, D]")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"cross_attention: q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or channels")
    if not 1 <= q.shape[3] <= MAX_HEAD_DIM:
        raise ValueError(f"cross_attention: heads of 1..{MAX_HEAD_DIM} channels, got {q.shape[3]}")
    if q.shape[2] < 1 or k.shape[2] < 1 or q.shape[2] % k.shape[2]:
        raise ValueError(f"cross_attention: {q.shape[2]} query heads cannot share {k.shape[2]} key heads")
    if any(t.dtype != q.dtype for t in (k, v)) or q.dtype not in _TYPES:
        raise ValueError("cross_attention: q, k and v must share float32 or bfloat16")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"cross_attention requires contiguous channels of {name}, got stride {t.stride()}")
    _require_gpu("cross_attention", q, k=k, v=v)
    if lengths is not None:
        _require_packed("cross_attention", lengths=lengths)
        if lengths.dtype != torch.int32 or lengths.shape != (q.shape[0],):
            raise ValueError(f"lengths must be int32 [{q.shape[0]}], got {lengths.dtype} {tuple(lengths.shape)}")
        _require_gpu("cross_attention", q, lengths=lengths)


@custom_op("sihc::cross_attention", mutates_args=())
def _cross_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], scale: float,
                     train: bool) -> tuple[Tensor, Tensor, Tensor]:
    _check_attention(q, k, v, lengths)
    return launch.cross_attention(q, k, v, lengths, scale, train)


@_cross_attention.register_fake
def _cross_attention_fake(q, k, v, lengths, scale, train):
    b, n, h, _ = q.shape
    return (q.new_empty(q.shape), q.new_empty((b, h, n, 2) if train else (0,), dtype=torch.float32),
            q.new_empty(q.shape if train and q.dtype == torch.bfloat16 else (0,)))


@custom_op("sihc::cross_attention_backward", mutates_args=())
def _cross_attention_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], out: Tensor,
                              stats: Tensor, low: Tensor, scale: float) -> tuple[Tensor, Tensor, Tensor]:
    _check_attention(q, k, v, lengths)  # saved tensors come back through the caller's hooks
    _require_packed("cross_attention backward", grad=grad, out=out, stats=stats, low=low)
    b, n, h, _ = q.shape
    like = (grad, out, low) if q.dtype == torch.bfloat16 else (grad, out)
    if any(t.shape != q.shape or t.dtype != q.dtype for t in like) or stats.shape != (b, h, n, 2):
        raise ValueError("cross_attention backward: the gradient and the saved tensors must match the output of a "
                         "call with train=True")
    _require_gpu("cross_attention backward", q, grad=grad, out=out, stats=stats, low=low)
    return launch.cross_attention_backward(grad, q, k, v, lengths, out, stats, low, scale)


@_cross_attention_backward.register_fake
def _cross_attention_backward_fake(grad, q, k, v, lengths, out, stats, low, scale):
    return tuple(t.new_empty(t.shape) for t in (q, k, v))


def _attention_setup(ctx, inputs, output):
    q, k, v, lengths, ctx.scale, _ = inputs
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(q, k, v, lengths, *output)


def _attention_autograd(ctx, grad, _, __):
    if grad is None:
        return (None,) * 6
    q, k, v, lengths, out, stats, low = ctx.saved_tensors
    return (*_cross_attention_backward(grad.contiguous(), q, k, v, lengths, out, stats, low, ctx.scale), None, None,
            None)


register_autograd(_cross_attention, _attention_autograd, setup_context=_attention_setup)
native(_cross_attention, "cross_attention")


def cross_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor] = None,
                    scale: Optional[float] = None, *, validate: bool = True) -> Tensor:
    """Attention of q [B,Lq,H,D] over k, v [B,Lk,KH,D], of which row b has the first lengths[b]
    (int32 [B]; None: all). scale defaults to 1 / sqrt(D). Returns [B,Lq,H,D], packed."""
    if validate:
        _check_attention(q, k, v, lengths)
        if lengths is not None and lengths.numel():
            low, high = int(lengths.min()), int(lengths.max())
            if low < 0 or high > k.shape[1]:
                raise ValueError(f"lengths must lie in [0, {k.shape[1]}], got [{low}, {high}]")
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _cross_attention(q, k, v, lengths, 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale, train)[0]


__all__ = ["embedding_lookup", "cross_attention", "group_norm_act"]
