"""The body of a block between its read and its write: projections, head norms with rotation, dropout.

Specification (the reference's bodies are plain PyTorch, sihc/models/sihc/components.py:18-70,184-251):

* ``linear_act(x, weight, bias, act, gate, residual)``: h = x weight^T + bias; u is h (act "none"),
  silu(h) ("silu") or silu(h_a) * h_b ("swiglu", h = [h_a, h_b], so the weight has twice the result's
  rows); the result is residual + gate * u. x is [batch, ..., inner]; the gate is one row of the
  result's channels for each index of x's first dimension (a part of a modulation), its rows any
  distance apart.
* ``qk_norm_rotary(q, k, q_weight, k_weight, positions, axes, theta, eps)``: the RMS norm of every head
  of q [B, N, H, D] and k [B, N, KH, D] with its weight [D], then the rotation, in one pass.
* ``axis_rotary(x, positions, axes, theta)``: the rotation alone, of x [B, N, H, D].
  Positions are [N, len(axes)], the same for every batch row, or [B, N, len(axes)], in int32 or
  float32. Axis i turns the adjacent pairs of the next axes[i] channels, pair j by the angle
  position * theta^(-2 j / axes[i]); channels past the axes stay. Angles are taken in 64 bits, so
  that far positions have theirs. Positions have no gradient.
* ``dropout(x, p, seed, stream, residual)``: residual + x / (1 - p) where the mask keeps an element.
  The mask is a function of the seed (an int64 tensor of one element on the GPU), the stream (which
  call it is among those of one seed) and the element's place in the packed tensor: word i % 4 of the
  Philox 4x32 block of counter (i / 4, stream) under the seed, kept if it is at least p 2^32. It is never
  stored: the backward, a recomputed forward and a replayed graph make it again from the seed's
  value at that time.

All sums and statistics are fp32, in a fixed order without atomics: identical inputs give identical
bits. float32 and bfloat16; the norm's weights may be float32 beside bfloat16 heads. In bfloat16 the
backward of a gate works on h rounded to bfloat16, that of an activation on 20 bits of it, and the
gradient of h enters the products rounded to bfloat16. q, k and x of the
rotations are read through their strides (the channels of a head adjacent); the other tensors are packed.
Derivatives are reverse-mode ones: a forward-mode tangent is refused.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
from torch import Tensor
from torch.library import custom_op, register_autograd

from . import launch
from ._lib import MAX_AXES, MAX_ROTARY_DIM
from ._native import native, refuse_tangents
from .conditioning import _TYPES, _require_gpu
from .sublayer_kernels import _require_packed

_MOST_ROWS, _MOST_CHANNELS, _MOST_TOKENS = 1 << 30, 1 << 24, (1 << 31) - 64


# ----------------------------------------------------------------------------------- linear
def _given(**tensors: Optional[Tensor]) -> dict[str, Tensor]:
    return {name: t for name, t in tensors.items() if t is not None}


def _linear_outer(weight: Tensor, act: str) -> int:
    return weight.shape[0] // 2 if act == "swiglu" else weight.shape[0]


def _linear_rows(x: Tensor) -> int:
    return math.prod(x.shape[:-1])


def _check_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, gate: Optional[Tensor],
                  residual: Optional[Tensor]) -> None:
    if act not in launch.LINEAR_ACTIVATIONS:
        raise ValueError(f"linear_act: act must be one of {sorted(launch.LINEAR_ACTIVATIONS)}, got {act!r}")
    _require_packed("linear_act", x=x, weight=weight, **_given(bias=bias, residual=residual))
    if x.ndim < 2 or weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_act: expected x [batch, ..., inner] and a weight [rows, inner], got "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    if 0 in weight.shape or max(weight.shape) > _MOST_CHANNELS or (act == "swiglu" and weight.shape[0] % 2):
        raise ValueError(f"linear_act: a weight of 1..{_MOST_CHANNELS} rows (swiglu: an even number) and channels, got "
                         f"{tuple(weight.shape)}")
    if _linear_rows(x) > _MOST_ROWS:
        raise ValueError(f"linear_act: at most {_MOST_ROWS} rows, got {_linear_rows(x)}")
    outer = _linear_outer(weight, act)
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"linear_act: expected a bias [{weight.shape[0]}], got {tuple(bias.shape)}")
    if gate is not None:
        if gate.shape != (x.shape[0], outer):
            raise ValueError(f"linear_act: expected a gate [{x.shape[0]}, {outer}], got {tuple(gate.shape)}")
        if outer > 1 and gate.stride(1) != 1:
            raise ValueError(f"linear_act requires contiguous channels of the gate, got stride {gate.stride()}")
    if residual is not None and residual.shape != (*x.shape[:-1], outer):
        raise ValueError(f"linear_act: expected a residual {(*x.shape[:-1], outer)}, got {tuple(residual.shape)}")
    others = _given(weight=weight, bias=bias, gate=gate, residual=residual)
    if x.dtype not in _TYPES or any(t.dtype != x.dtype for t in others.values()):
        raise ValueError("linear_act: all tensors must share float32 or bfloat16")
    _require_gpu("linear_act", x, **others)


# The result alone, for a call that nothing differentiates.
@custom_op("sihc::linear_act_result", mutates_args=())
def _linear_act_result(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, gate: Optional[Tensor],
                       residual: Optional[Tensor]) -> Tensor:
    _check_linear(x, weight, bias, act, gate, residual)
    return launch.linear_act(x, weight, bias, act, gate, residual, False)[0]


@_linear_act_result.register_fake
def _linear_act_result_fake(x, weight, bias, act, gate, residual):
    return x.new_empty((*x.shape[:-1], _linear_outer(weight, act)))


native(_linear_act_result, "linear_act_result", tangents=False)


# The result and what the backward needs of h (empty where it needs nothing).
@custom_op("sihc::linear_act", mutates_args=())
def _linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, gate: Optional[Tensor],
                residual: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    _check_linear(x, weight, bias, act, gate, residual)
    return launch.linear_act(x, weight, bias, act, gate, residual, True)


@_linear_act.register_fake
def _linear_act_fake(x, weight, bias, act, gate, residual):
    outer = _linear_outer(weight, act)
    kept = (*x.shape[:-1], weight.shape[0]) if act != "none" or gate is not None else (0,)
    return (x.new_empty((*x.shape[:-1], outer)), x.new_empty(kept),
            x.new_empty(launch.low_shape(x, outer, act), dtype=torch.int32))


@custom_op("sihc::linear_act_backward", mutates_args=())
def _linear_act_backward(grad: Tensor, x: Tensor, weight: Tensor, h: Tensor, low: Tensor, gate: Optional[Tensor],
                         act: str, want_x: bool, want_weight: bool, want_bias: bool,
                         want_gate: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    _check_linear(x, weight, None, act, gate, None)  # saved tensors come back through the caller's hooks
    _require_packed("linear_act backward", grad=grad, h=h, low=low)
    if grad.shape != (*x.shape[:-1], _linear_outer(weight, act)) or grad.dtype != x.dtype:
        raise ValueError("linear_act backward: the output gradient must match the output")
    if act != "none" or gate is not None:
        if h.shape != (*x.shape[:-1], weight.shape[0]) or h.dtype != x.dtype:
            raise ValueError("linear_act backward: h must be that of the forward")
    bits = launch.low_shape(x, _linear_outer(weight, act), act)
    if bits != (0,) and (low.shape != bits or low.dtype != torch.int32):
        raise ValueError("linear_act backward: low must be that of the forward")
    if want_gate and gate is None:
        raise ValueError("linear_act backward: no gate, no gradient of it")
    _require_gpu("linear_act backward", x, grad=grad, h=h, low=low)
    return launch.linear_act_backward(grad, x, weight, h, low, gate, act, want_x, want_weight, want_bias, want_gate)


@_linear_act_backward.register_fake
def _linear_act_backward_fake(grad, x, weight, h, low, gate, act, want_x, want_weight, want_bias, want_gate):
    return (x.new_empty(x.shape if want_x else (0,)), x.new_empty(weight.shape if want_weight else (0,)),
            x.new_empty(weight.shape[:1] if want_bias else (0,)),
            x.new_empty((x.shape[0], _linear_outer(weight, act)) if want_gate else (0,)))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, ctx.act, gate, residual = inputs
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, gate, output[1], output[2])


def _linear_autograd(ctx, grad, _, __):
    if grad is None:
        return (None,) * 6
    x, weight, gate, h, low = ctx.saved_tensors
    want = [ctx.needs_input_grad[i] for i in (0, 1, 2, 4)]
    if not any(want):
        return None, None, None, None, None, grad
    refuse_tangents("linear_act backward", (grad,))
    grads = _linear_act_backward(grad.contiguous(), x, weight, h, low, gate, ctx.act, *want)
    dx, dweight, dbias, dgate = (g if w else None for g, w in zip(grads, want))
    return dx, dweight, dbias, None, dgate, grad if ctx.needs_input_grad[5] else None


register_autograd(_linear_act, _linear_autograd, setup_context=_linear_setup)
native(_linear_act, "linear_act", tangents=False)


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none",
               gate: Optional[Tensor] = None, residual: Optional[Tensor] = None) -> Tensor:
    """residual + gate * act(x weight^T + bias) of x [batch, ..., inner]; act is "none", "silu" or
    "swiglu"; gate [batch, outer], residual like the result [batch, ..., outer]."""
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
            (gate is not None and gate.requires_grad) or (residual is not None and residual.requires_grad)):
        return _linear_act(x, weight, bias, act, gate, residual)[0]
    return _linear_act_result(x, weight, bias, act, gate, residual)


# --------------------------------------------------------------------- head norms and rotation
def _most_tokens(heads: int, dim: int) -> int:
    """What the forward's launch takes: fewer than 2^26 waves, each of one token if its heads fill four passes of the
    wave (8 channels a lane, a power of two of lanes a head), else of as many as do, up to 8."""
    lanes = 1 << ((dim - 1) // 8).bit_length()
    return min(_MOST_TOKENS, ((1 << 26) - 4) * max(1, min(8, 4 * (64 // lanes) // heads)))


def _check_heads(op: str, positions: Tensor, axes: Sequence[int], theta: float, **heads: Tensor) -> None:
    first = next(iter(heads.values()))
    for name, x in heads.items():
        if x.ndim != 4 or x.shape[:2] != first.shape[:2] or x.shape[3] != first.shape[3]:
            raise ValueError(f"{op}: expected [batch, tokens, heads, channels] of the same batch, tokens and channels, "
                             f"got {[tuple(t.shape) for t in heads.values()]}")
        if not 1 <= x.shape[3] <= MAX_ROTARY_DIM or not 1 <= x.shape[2] <= 1 << 20:
            raise ValueError(f"{op}: 1..{1 << 20} heads of 1..{MAX_ROTARY_DIM} channels, got {tuple(x.shape)}")
        if x.shape[3] > 1 and x.stride(3) != 1:
            raise ValueError(f"{op} requires contiguous channels of {name}, got stride {x.stride()}")
        if x.dtype not in _TYPES or x.dtype != first.dtype:
            raise ValueError(f"{op}: heads must share float32 or bfloat16")
    batch, tokens, _, dim = first.shape
    most = _most_tokens(sum(x.shape[2] for x in heads.values()), dim)
    if batch * tokens > most:
        raise ValueError(f"{op}: at most {most} tokens of these heads, got {batch * tokens}")
    if len(axes) > MAX_AXES or any(w < 0 or w % 2 for w in axes) or sum(axes) > dim:
        raise ValueError(f"{op}: up to {MAX_AXES} axes of even widths within {dim} channels, got {list(axes)}")
    if not 0.0 < theta < math.inf:
        raise ValueError(f"{op}: theta must be positive, got {theta}")
    _require_packed(op, positions=positions)
    if positions.shape not in ((tokens, len(axes)), (batch, tokens, len(axes))):
        raise ValueError(f"{op}: expected positions [{tokens}, {len(axes)}] or [{batch}, {tokens}, {len(axes)}], got "
                         f"{tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.float32):
        raise ValueError(f"{op}: positions must be int32 or float32, got {positions.dtype}")


def _check_qk(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, positions: Tensor, axes: Sequence[int],
              theta: float, eps: float) -> None:
    op = "qk_norm_rotary"
    _check_heads(op, positions, axes, theta, q=q, k=k)
    _require_packed(op, q_weight=q_weight, k_weight=k_weight)
    if q_weight.shape != q.shape[3:] or k_weight.shape != q.shape[3:]:
        raise ValueError(f"{op}: weights must be [{q.shape[3]}]")
    if q_weight.dtype != k_weight.dtype or q_weight.dtype not in (q.dtype, torch.float32):
        raise ValueError(f"{op}: weights of the heads' type or float32")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{op}: eps must not be negative, got {eps}")
    _require_gpu(op, q, k=k, q_weight=q_weight, k_weight=k_weight, positions=positions)


@custom_op("sihc::qk_norm_rotary", mutates_args=())
def _qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, positions: Tensor,
                    axes: Sequence[int], theta: float, eps: float) -> tuple[Tensor, Tensor]:
    _check_qk(q, k, q_weight, k_weight, positions, axes, theta, eps)
    return launch.qk_norm_rotary(q, k, q_weight, k_weight, positions, axes, theta, eps)


@_qk_norm_rotary.register_fake
def _qk_norm_rotary_fake(q, k, q_weight, k_weight, positions, axes, theta, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@custom_op("sihc::qk_norm_rotary_backward", mutates_args=())
def _qk_norm_rotary_backward(grad_q: Tensor, grad_k: Tensor, q: Tensor, k: Tensor, q_weight: Tensor,
                             k_weight: Tensor, positions: Tensor, axes: Sequence[int], theta: float,
                             eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    _check_qk(q, k, q_weight, k_weight, positions, axes, theta, eps)  # (saved tensors, through hooks)
    _require_packed("qk_norm_rotary backward", grad_q=grad_q, grad_k=grad_k)
    if grad_q.shape != q.shape or grad_k.shape != k.shape or any(g.dtype != q.dtype for g in (grad_q, grad_k)):
        raise ValueError("qk_norm_rotary backward: the output gradients must match the outputs")
    _require_gpu("qk_norm_rotary backward", q, grad_q=grad_q, grad_k=grad_k)
    return launch.qk_norm_rotary_backward(grad_q, grad_k, q, k, q_weight, k_weight, positions, axes, theta, eps)


@_qk_norm_rotary_backward.register_fake
def _qk_norm_rotary_backward_fake(grad_q, grad_k, q, k, q_weight, k_weight, positions, axes, theta, eps):
    return tuple(t.new_empty(t.shape) for t in (q, k, q_weight, k_weight))


def _qk_setup(ctx, inputs, output):
    *tensors, ctx.axes, ctx.theta, ctx.eps = inputs
    ctx.save_for_backward(*tensors)


def _qk_autograd(ctx, grad_q, grad_k):
    refuse_tangents("qk_norm_rotary backward", (grad_q, grad_k))
    return (*_qk_norm_rotary_backward(grad_q.contiguous(), grad_k.contiguous(), *ctx.saved_tensors, ctx.axes,
                                      ctx.theta, ctx.eps), None, None, None, None)


register_autograd(_qk_norm_rotary, _qk_autograd, setup_context=_qk_setup)
native(_qk_norm_rotary, "qk_norm_rotary", tangents=False)


def qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, positions: Tensor,
                   axes: Sequence[int], theta: float = 10000.0, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """RMS norm of every head of q [B,N,H,D] and k [B,N,KH,D], turned by positions [N,A] or [B,N,A]
    (int32 or float32), axes[i] channels by the i-th. Returns both packed."""
    return _qk_norm_rotary(q, k, q_weight, k_weight, positions, list(axes), theta, eps)


@custom_op("sihc::axis_rotary", mutates_args=())
def _axis_rotary(x: Tensor, positions: Tensor, axes: Sequence[int], theta: float, inverse: bool) -> Tensor:
    _check_heads("axis_rotary", positions, axes, theta, x=x)
    _require_gpu("axis_rotary", x, positions=positions)
    return launch.axis_rotary(x, positions, axes, theta, inverse)


@_axis_rotary.register_fake
def _axis_rotary_fake(x, positions, axes, theta, inverse):
    return x.new_empty(x.shape)


def _rotary_setup(ctx, inputs, output):
    _, positions, ctx.axes, ctx.theta, ctx.inverse = inputs
    ctx.save_for_backward(positions)


def _rotary_autograd(ctx, grad):
    (positions,) = ctx.saved_tensors
    return _axis_rotary(grad.contiguous(), positions, ctx.axes, ctx.theta, not ctx.inverse), None, None, None, None


register_autograd(_axis_rotary, _rotary_autograd, setup_context=_rotary_setup)
native(_axis_rotary, "axis_rotary", tangents=False)


def axis_rotary(x: Tensor, positions: Tensor, axes: Sequence[int], theta: float = 10000.0) -> Tensor:
    """x [B,N,H,D] turned by positions [N,A] or [B,N,A] (int32 or float32), axes[i] channels by the
    i-th. Returns it packed."""
    return _axis_rotary(x, positions, list(axes), theta, False)


# ------------------------------------------------------------------------------------ dropout
def _check_dropout(x: Tensor, p: float, seed: Tensor, stream: int, residual: Optional[Tensor]) -> None:
    _require_packed("dropout", x=x, seed=seed, **_given(residual=residual))
    if x.dtype not in _TYPES:
        raise ValueError("dropout: float32 or bfloat16")
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: p must lie in [0, 1), got {p}")
    if seed.dtype != torch.int64 or seed.numel() != 1:
        raise ValueError(f"dropout: the seed must be one int64, got {seed.dtype} {tuple(seed.shape)}")
    if not 0 <= stream < 1 << 63:
        raise ValueError(f"dropout: the stream must lie in [0, 2^63), got {stream}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("dropout: the residual must match x")
    _require_gpu("dropout", x, seed=seed, **_given(residual=residual))


@custom_op("sihc::dropout", mutates_args=())
def _dropout(x: Tensor, p: float, seed: Tensor, stream: int, residual: Optional[Tensor]) -> Tensor:
    _check_dropout(x, p, seed, stream, residual)
    return launch.dropout(x, p, seed, stream, residual)


@_dropout.register_fake
def _dropout_fake(x, p, seed, stream, residual):
    return torch.empty_like(x)


def _dropout_setup(ctx, inputs, output):
    _, ctx.p, seed, ctx.stream, _ = inputs
    ctx.save_for_backward(seed)


def _dropout_autograd(ctx, grad):
    (seed,) = ctx.saved_tensors
    dx = _dropout(grad.contiguous(), ctx.p, seed, ctx.stream, None) if ctx.needs_input_grad[0] else None
    return dx, None, None, None, grad if ctx.needs_input_grad[4] else None


register_autograd(_dropout, _dropout_autograd, setup_context=_dropout_setup)
native(_dropout, "dropout", tangents=False)


def dropout(x: Tensor, p: float, seed: Tensor, stream: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """residual + x / (1 - p) where the mask of (seed, stream) keeps an element, residual elsewhere."""
    return _dropout(x, p, seed, stream, residual)


__all__ = ["linear_act", "qk_norm_rotary", "axis_rotary", "dropout"]
