"""Tensor-level launchers over the C ABI (include/sihc_hip.h).

Each function allocates its outputs from the PyTorch caching allocator, passes raw
device pointers to libsihc_hip.so and enqueues on the current HIP stream of the
inputs' device. No host synchronisation happens here, so the launchers are safe
under HIP-graph capture. Shape/layout validation that the reference performs in
Python lives in the op modules (sublayer_kernels, event_ops, indexed); these
launchers only assert what the C ABI itself needs.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence

import torch
from torch import Tensor

from ._lib import (ACT_NONE, ACT_SILU, ACT_SWIGLU, DTYPE_BF16, DTYPE_F32, MAX_AXES, MAX_EVENTS, POSITION_F32, POSITION_I32,
                   Attention, Heads, Linear, check, lib, ptr_array)

_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}
ACTIVATIONS = {"none": ACT_NONE, "silu": ACT_SILU}
LINEAR_ACTIVATIONS = {**ACTIVATIONS, "swiglu": ACT_SWIGLU}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {dtype}: expected float32 or bfloat16") from None


def _on_tensor_device(fn):
    """Run a launcher with its first tensor argument's GPU as the current HIP device:
    the library launches on that device's current stream and sizes grids from the
    current device's properties, which must be the same device."""

    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        dev = next((a.device for a in (*args, *kwargs.values()) if isinstance(a, Tensor) and a.is_cuda), None)
        if dev is None or dev.index is None or dev.index == torch.cuda.current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(dev):
            return fn(*args, **kwargs)

    return wrapper


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device: torch.device) -> Tensor:
    # Rounded up to 16 floats; torch allocations are at least 256-byte aligned.
    return torch.empty((max(nbytes, 4) + 63) // 64 * 16, dtype=torch.float32, device=device)


def carrier_geometry(x: Tensor, slots: int) -> tuple[int, int, int, int]:
    """(batch, grid, cell, channels) of a packed NHWC carrier with `slots` per cell."""
    b, h, w, c = x.shape
    k = 2 if slots == 4 else 4
    return b, h // k, k, c


@_on_tensor_device
def read(x: Tensor, alpha: Tensor, index: Optional[Tensor] = None,
         out: Optional[Sequence[Tensor]] = None) -> list[Tensor]:
    """E base reads of carrier x [B,H,W,C] with stacked alpha [E,C,S] (into `out` if given)."""
    b, g, k, c = carrier_geometry(x, alpha.shape[2])
    events = alpha.shape[0]
    if out is None:
        out = [torch.empty((b, g * g, c), device=x.device, dtype=x.dtype) for _ in range(events)]
    out = list(out)
    check(lib().sihc_read(x.data_ptr(), alpha.data_ptr(), ptr_array(o.data_ptr() for o in out), events,
                          b, g, k, c, _ptr(index), dtype_code(x.dtype), _stream(x.device)))
    return out


@_on_tensor_device
def write(x: Tensor, updates: Sequence[Tensor], beta: Tensor, add_x: bool = True,
          index: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """(add_x ? x : 0) + sum_e beta_e * updates_e written into a new carrier."""
    b, g, k, c = carrier_geometry(x, beta.shape[2])
    if out is None:
        out = torch.empty_like(x)
    check(lib().sihc_write(x.data_ptr() if add_x else None, ptr_array(u.data_ptr() for u in updates),
                           beta.data_ptr(), out.data_ptr(), len(updates), b, g, k, c, int(add_x),
                           _ptr(index), dtype_code(x.dtype), dtype_code(beta.dtype), _stream(x.device)))
    return out


@_on_tensor_device
def weight_grad(x: Tensor, updates: Sequence[Tensor], weights: Optional[Tensor],
                index: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                slots: Optional[int] = None) -> Tensor:
    """[E,C,S] = sum over tokens of x[m,s,c] * updates_e[m,c], reduced in fp32.

    Stored in out_dtype (default: the weights' dtype); `slots` and `out_dtype` stand in
    for `weights` when there is no weight tensor at hand.
    """
    b, g, k, c = carrier_geometry(x, slots if weights is None else weights.shape[-1])
    events = len(updates)
    out = torch.empty((events, c, k * k), device=x.device, dtype=out_dtype or weights.dtype)
    L = lib()
    nbytes = L.sihc_weight_grad_workspace_size(events, b, g, k, c)
    ws = _workspace(nbytes, x.device)
    check(L.sihc_weight_grad(x.data_ptr(), ptr_array(u.data_ptr() for u in updates), out.data_ptr(), events,
                             b, g, k, c, _ptr(index), dtype_code(x.dtype), dtype_code(out.dtype),
                             ws.data_ptr(), ws.numel() * 4, _stream(x.device)))
    return out


@_on_tensor_device
def read_backward(x: Tensor, grads: Sequence[Tensor], alpha: Tensor, index: Optional[Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> tuple[Tensor, Tensor]:
    """Adjoint of `read`: (dx, dalpha [E,C,S]); dalpha in out_dtype (default alpha's dtype)."""
    b, g, k, c = carrier_geometry(x, alpha.shape[2])
    events = len(grads)
    dx = torch.empty_like(x)
    da = torch.empty((events, c, k * k), device=x.device, dtype=out_dtype or alpha.dtype)
    L = lib()
    ws = _workspace(L.sihc_weight_grad_workspace_size(events, b, g, k, c), x.device)
    check(L.sihc_read_backward(x.data_ptr(), ptr_array(t.data_ptr() for t in grads), alpha.data_ptr(), dx.data_ptr(),
                               da.data_ptr(), events, b, g, k, c, _ptr(index), dtype_code(x.dtype),
                               dtype_code(da.dtype), ws.data_ptr(), ws.numel() * 4, _stream(x.device)))
    return dx, da


@_on_tensor_device
def write_backward(grad: Tensor, updates: Sequence[Tensor], beta: Tensor, index: Optional[Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> tuple[list[Tensor], Tensor]:
    """Adjoint of `write` except the identity to x: (update gradients, dbeta [E,C,S]); dbeta in
    out_dtype (default beta's dtype)."""
    b, g, k, c = carrier_geometry(grad, beta.shape[2])
    events = len(updates)
    ddz = [torch.empty((b, g * g, c), device=grad.device, dtype=grad.dtype) for _ in range(events)]
    db = torch.empty((events, c, k * k), device=grad.device, dtype=out_dtype or beta.dtype)
    L = lib()
    ws = _workspace(L.sihc_weight_grad_workspace_size(events, b, g, k, c), grad.device)
    check(L.sihc_write_backward(grad.data_ptr(), ptr_array(u.data_ptr() for u in updates), beta.data_ptr(),
                                ptr_array(d.data_ptr() for d in ddz), db.data_ptr(), events, b, g, k, c, _ptr(index),
                                dtype_code(grad.dtype), dtype_code(db.dtype), ws.data_ptr(), ws.numel() * 4,
                                _stream(grad.device)))
    return ddz, db


@_on_tensor_device
def triangular(base: Tensor, updates: Sequence[Tensor], gamma: Tensor) -> Tensor:
    """base + sum_j gamma[j] * updates_j over a [B,N,C] workspace."""
    c = base.shape[-1]
    rows = base.numel() // c if c else 0
    out = torch.empty_like(base)
    check(lib().sihc_triangular(base.data_ptr(), ptr_array(u.data_ptr() for u in updates), gamma.data_ptr(),
                                out.data_ptr(), len(updates), rows, c, dtype_code(base.dtype),
                                dtype_code(gamma.dtype), _stream(base.device)))
    return out


@_on_tensor_device
def triangular_gamma_grad(grad: Tensor, updates: Sequence[Tensor], gamma: Optional[Tensor],
                          out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """[A,C] (out_dtype, default gamma's dtype) = sum over rows of grad * updates_j."""
    c = grad.shape[-1]
    rows = grad.numel() // c if c else 0
    active = len(updates)
    out = torch.empty((active, c), device=grad.device, dtype=out_dtype or gamma.dtype)
    L = lib()
    ws = _workspace(L.sihc_triangular_gamma_grad_workspace_size(active, rows, c), grad.device)
    check(L.sihc_triangular_gamma_grad(grad.data_ptr(), ptr_array(u.data_ptr() for u in updates),
                                       out.data_ptr(), active, rows, c, dtype_code(grad.dtype),
                                       dtype_code(out.dtype), ws.data_ptr(), ws.numel() * 4,
                                       _stream(grad.device)))
    return out


@_on_tensor_device
def triangular_backward(grad: Tensor, updates: Sequence[Tensor], gamma: Tensor,
                        out_dtype: Optional[torch.dtype] = None) -> tuple[Tensor, Tensor]:
    """One pass: ([A,B,N,C] stack of grad * gamma[j], [A,C] sum over rows of grad * updates_j).

    The update gradients share grad's dtype; the gamma gradient is out_dtype (default
    gamma's dtype), reduced in fp32.
    """
    c = grad.shape[-1]
    rows = grad.numel() // c if c else 0
    active = len(updates)
    ddz = torch.empty((active, *grad.shape), device=grad.device, dtype=grad.dtype)
    dg = torch.empty((active, c), device=grad.device, dtype=out_dtype or gamma.dtype)
    L = lib()
    ws = _workspace(L.sihc_triangular_gamma_grad_workspace_size(active, rows, c), grad.device)
    check(L.sihc_triangular_backward(grad.data_ptr(), ptr_array(u.data_ptr() for u in updates), gamma.data_ptr(),
                                     ptr_array(d.data_ptr() for d in ddz.unbind(0)), dg.data_ptr(), active, rows,
                                     c, dtype_code(grad.dtype), dtype_code(gamma.dtype), dtype_code(dg.dtype),
                                     ws.data_ptr(), ws.numel() * 4, _stream(grad.device)))
    return ddz, dg


@_on_tensor_device
def event_forward(x: Tensor, dz: Tensor, beta: Tensor, alpha_next: Optional[Tensor],
                  index: Optional[Tensor] = None) -> tuple[Tensor, Optional[Tensor]]:
    """x_out = x + beta*dz and z_out = read(x_out, alpha_next) in one pass."""
    b, g, k, c = carrier_geometry(x, beta.shape[1])
    x_out = torch.empty_like(x)
    z_out = None if alpha_next is None else torch.empty((b, g * g, c), device=x.device, dtype=x.dtype)
    check(lib().sihc_event_forward(x.data_ptr(), dz.data_ptr(), beta.data_ptr(), _ptr(alpha_next),
                                   x_out.data_ptr(), _ptr(z_out), b, g, k, c, _ptr(index),
                                   dtype_code(x.dtype), _stream(x.device)))
    return x_out, z_out


@_on_tensor_device
def event_backward(grad_x_out: Optional[Tensor], grad_z_out: Optional[Tensor], x_out: Optional[Tensor],
                   dz: Optional[Tensor], beta: Optional[Tensor], alpha_next: Optional[Tensor],
                   index: Optional[Tensor] = None, grad_x: Optional[Tensor] = None,
                   alias_grad_x: bool = False, carrier_like: Optional[Tensor] = None):
    """Adjoint of event_forward: (grad_x, grad_dz, grad_beta, grad_alpha_next).

    `beta`/`dz` None drops the write part (adjoint of a plain read). With
    `alias_grad_x` and no read part, grad_x is grad_x_out itself (not copied).
    `carrier_like` supplies the carrier shape when x_out is None.
    """
    ref = x_out if x_out is not None else (carrier_like if carrier_like is not None else grad_x_out)
    w = beta if beta is not None else alpha_next
    for t in (beta, alpha_next):
        if t is not None and t.dtype != ref.dtype:
            raise ValueError(f"event weights must share the carrier dtype {ref.dtype}, got {t.dtype}")
    b, g, k, c = carrier_geometry(ref, w.shape[1])
    alias = alias_grad_x and grad_z_out is None
    if alias:
        grad_x = grad_x_out
    elif grad_x is None:
        grad_x = torch.empty(ref.shape, device=ref.device, dtype=ref.dtype)
    grad_dz = None if beta is None else torch.empty((b, g * g, c), device=ref.device, dtype=ref.dtype)
    grad_beta = None if beta is None else torch.empty_like(beta)
    grad_alpha = None if alpha_next is None else torch.empty_like(alpha_next)
    L = lib()
    ws = _workspace(L.sihc_event_backward_workspace_size(b, g, k, c), ref.device)
    check(L.sihc_event_backward(_ptr(grad_x_out), _ptr(grad_z_out), _ptr(x_out), _ptr(dz), _ptr(beta),
                                _ptr(alpha_next), None if alias else grad_x.data_ptr(), _ptr(grad_dz),
                                _ptr(grad_beta), _ptr(grad_alpha), b, g, k, c, _ptr(index),
                                dtype_code(ref.dtype), dtype_code(w.dtype), ws.data_ptr(),
                                ws.numel() * 4, _stream(ref.device)))
    return grad_x, grad_dz, grad_beta, grad_alpha


@_on_tensor_device
def gather_cells(x: Tensor, index: Optional[Tensor], slots: int) -> Tensor:
    """[B,G*G,S,C] bit-exact copy of each token's cell (cell index[b,n] when given)."""
    b, g, k, c = carrier_geometry(x, slots)
    cells = torch.empty((b, g * g, k * k, c), device=x.device, dtype=x.dtype)
    check(lib().sihc_gather_cells(x.data_ptr(), _ptr(index), cells.data_ptr(), b, g, k, c,
                                  dtype_code(x.dtype), _stream(x.device)))
    return cells


@_on_tensor_device
def scatter_cells(cells: Tensor, index: Optional[Tensor], out: Optional[Tensor] = None) -> Tensor:
    """Inverse of gather_cells for a permutation index: new (or `out`) NHWC carrier."""
    b, n, s, c = cells.shape
    k = 2 if s == 4 else 4
    g = int(round(n ** 0.5))
    if out is None:
        out = torch.empty((b, g * k, g * k, c), device=cells.device, dtype=cells.dtype)
    check(lib().sihc_scatter_cells(cells.data_ptr(), _ptr(index), out.data_ptr(), b, g, k, c,
                                   dtype_code(cells.dtype), _stream(cells.device)))
    return out


@_on_tensor_device
def scatter_add_cells(cells: Tensor, index: Optional[Tensor], out: Optional[Tensor] = None) -> Tensor:
    """Adjoint of gather_cells for any in-range index (repeats allowed): each carrier cell
    gets the fp32 sum, in ascending token order, of the cells rows that select it, and
    zeros where none does. Equals scatter_cells bit for bit for a permutation index."""
    b, n, s, c = cells.shape
    k = 2 if s == 4 else 4
    g = int(round(n ** 0.5))
    if out is None:
        out = torch.empty((b, g * k, g * k, c), device=cells.device, dtype=cells.dtype)
    check(lib().sihc_scatter_add_cells(cells.data_ptr(), _ptr(index), out.data_ptr(), b, g, k, c,
                                       dtype_code(cells.dtype), _stream(cells.device)))
    return out


@_on_tensor_device
def copy_(dst: Tensor, src: Tensor) -> Tensor:
    """Byte copy src -> dst (same number of bytes) with the library's copy kernel."""
    nbytes = src.numel() * src.element_size()
    if dst.numel() * dst.element_size() != nbytes:
        raise ValueError("copy_ needs equally sized tensors")
    check(lib().sihc_copy(src.data_ptr(), dst.data_ptr(), nbytes, _stream(src.device)))
    return dst


def _id_bits(ids: Tensor) -> int:
    return 32 if ids.dtype == torch.int32 else 64


@_on_tensor_device
def embedding(table: Tensor, ids: Tensor, scale: float) -> Tensor:
    """scale * table[ids] as [*ids.shape, C]."""
    out = torch.empty((*ids.shape, table.shape[1]), device=table.device, dtype=table.dtype)
    check(lib().sihc_embedding(table.data_ptr(), ids.data_ptr(), out.data_ptr(), ids.numel(), *table.shape, scale,
                               _id_bits(ids), dtype_code(table.dtype), _stream(table.device)))
    return out


@_on_tensor_device
def embedding_backward(grad: Tensor, ids: Tensor, rows: int, scale: float, padding: int) -> Tensor:
    """The whole table's gradient [rows, C]: zero where no id selects a row, and for row `padding`."""
    channels = grad.shape[-1]
    out = torch.empty((rows, channels), device=grad.device, dtype=grad.dtype)
    L = lib()
    ws = _workspace(L.sihc_embedding_backward_workspace_size(ids.numel(), rows, channels), grad.device)
    check(L.sihc_embedding_backward(grad.data_ptr(), ids.data_ptr(), out.data_ptr(), ids.numel(), rows, channels,
                                    scale, padding, _id_bits(ids), dtype_code(grad.dtype), ws.data_ptr(),
                                    ws.numel() * 4, _stream(grad.device)))
    return out


def _pixels(x: Tensor) -> int:
    return x[0, ..., 0].numel() if x.shape[0] else 0


@_on_tensor_device
def group_norm(x: Tensor, weight: Tensor, bias: Tensor, groups: int, eps: float,
               act: str) -> tuple[Tensor, Tensor]:
    """(act(group norm of x [B,...,C]), [B,groups,2] means and reciprocal deviations)."""
    batch, pixels, channels = x.shape[0], _pixels(x), x.shape[-1]
    out = torch.empty_like(x)
    stats = torch.empty((batch, groups, 2), device=x.device, dtype=torch.float32)
    L, code = lib(), dtype_code(x.dtype)
    nbytes = L.sihc_group_norm_workspace_size(batch, pixels, channels, groups, code)
    ws = _workspace(nbytes, x.device) if nbytes else None
    check(L.sihc_group_norm(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), out.data_ptr(), stats.data_ptr(), batch,
                            pixels, channels, groups, eps, ACTIVATIONS[act], code, dtype_code(weight.dtype), _ptr(ws),
                            nbytes, _stream(x.device)))
    return out, stats


@_on_tensor_device
def group_norm_backward(grad: Tensor, x: Tensor, weight: Tensor, bias: Tensor, stats: Tensor, groups: int,
                        act: str) -> tuple[Tensor, Tensor, Tensor]:
    """(input gradient, weight gradient, bias gradient) of group_norm."""
    batch, pixels, channels = x.shape[0], _pixels(x), x.shape[-1]
    dx, dw, db = torch.empty_like(x), torch.empty_like(weight), torch.empty_like(bias)
    L, code = lib(), dtype_code(x.dtype)
    ws = _workspace(L.sihc_group_norm_backward_workspace_size(batch, pixels, channels, groups, code), x.device)
    check(L.sihc_group_norm_backward(grad.data_ptr(), x.data_ptr(), weight.data_ptr(), bias.data_ptr(),
                                     stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), batch, pixels,
                                     channels, groups, ACTIVATIONS[act], code, dtype_code(weight.dtype),
                                     ws.data_ptr(), ws.numel() * 4, _stream(x.device)))
    return dx, dw, db


def _attention(q: Tensor, k: Tensor, v: Tensor, scale: float) -> Attention:
    strides = [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, v)]
    return Attention(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], *strides, scale,
                     dtype_code(q.dtype))


@_on_tensor_device
def cross_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], scale: float,
                    train: bool) -> tuple[Tensor, Tensor, Tensor]:
    """(attention of q [B,Lq,H,D] over k, v [B,Lk,KH,D], and for the backward [B,H,Lq,2] softmax statistics
    and, in bf16, what the output lost in rounding; both empty unless `train`)."""
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    stats = torch.empty((q.shape[0], q.shape[2], q.shape[1], 2) if train else (0,), device=q.device,
                        dtype=torch.float32)
    low = torch.empty(q.shape if train and q.dtype == torch.bfloat16 else (0,), device=q.device, dtype=q.dtype)
    L, a = lib(), _attention(q, k, v, scale)
    nbytes = L.sihc_cross_attention_workspace_size(ctypes.byref(a))
    ws = _workspace(nbytes, q.device) if nbytes else None
    check(L.sihc_cross_attention(ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(lengths),
                                 out.data_ptr(), stats.data_ptr() or None, low.data_ptr() or None, _ptr(ws), nbytes,
                                 _stream(q.device)))
    return out, stats, low


@_on_tensor_device
def cross_attention_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], out: Tensor,
                             stats: Tensor, low: Tensor, scale: float) -> tuple[Tensor, Tensor, Tensor]:
    """(query, key, value gradients) of cross_attention, packed."""
    dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
    L, a = lib(), _attention(q, k, v, scale)
    ws = _workspace(L.sihc_cross_attention_backward_workspace_size(ctypes.byref(a)), q.device)
    check(L.sihc_cross_attention_backward(ctypes.byref(a), grad.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                          _ptr(lengths), out.data_ptr(), stats.data_ptr(), low.data_ptr() or None,
                                          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws.numel() * 4,
                                          _stream(q.device)))
    return dq, dk, dv


def _linear(x: Tensor, weight: Tensor, act: str, gate: Optional[Tensor]) -> Linear:
    rows = x.numel() // x.shape[-1]
    outer = weight.shape[0] // 2 if act == "swiglu" else weight.shape[0]
    each = max(rows, 1) if gate is None or not rows else rows // x.shape[0]
    return Linear(rows, x.shape[-1], outer, LINEAR_ACTIVATIONS[act], dtype_code(x.dtype), each,
                  0 if gate is None else gate.stride(0))


def low_shape(x: Tensor, outer: int, act: str) -> tuple[int, ...]:
    """Of the words in which linear_act keeps more bits of h than its type has: bfloat16 before an
    activation's slope; (0,) elsewhere."""
    if act == "none" or x.dtype != torch.bfloat16:
        return (0,)
    return (*x.shape[:-1], 2 if act == "swiglu" else 1, (outer + 7) // 8)


@_on_tensor_device
def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, gate: Optional[Tensor],
               residual: Optional[Tensor], train: bool) -> tuple[Tensor, Tensor, Tensor]:
    """(residual + gate * act(h) with h = x weight^T + bias, and for the backward h [..., weight rows] and 4 more
    bits of each of its values; empty where the backward needs none or `train` is not set)."""
    l = _linear(x, weight, act, gate)
    keeps = train and (act != "none" or gate is not None)
    out = torch.empty((*x.shape[:-1], l.outer), device=x.device, dtype=x.dtype)
    wide = (*x.shape[:-1], weight.shape[0])
    h = torch.empty(wide if keeps else (0,), device=x.device, dtype=x.dtype)
    low = torch.empty(low_shape(x, l.outer, act) if train else (0,), device=x.device, dtype=torch.int32)
    L = lib()
    nbytes = L.sihc_linear_act_workspace_size(ctypes.byref(l))
    ws = _workspace(nbytes, x.device) if nbytes else None
    check(L.sihc_linear_act(ctypes.byref(l), x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(gate), _ptr(residual),
                            out.data_ptr(), h.data_ptr() or None, low.data_ptr() or None, _ptr(ws), nbytes,
                            _stream(x.device)))
    return out, h, low


@_on_tensor_device
def linear_act_backward(grad: Tensor, x: Tensor, weight: Tensor, h: Tensor, low: Tensor, gate: Optional[Tensor],
                        act: str, want_x: bool, want_weight: bool, want_bias: bool,
                        want_gate: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(input, weight, bias and gate gradients) of linear_act, those that are not wanted empty."""
    l = _linear(x, weight, act, gate)

    def output(wanted, shape):
        return torch.empty(shape if wanted else (0,), device=x.device, dtype=x.dtype)

    dx, dw = output(want_x, x.shape), output(want_weight, weight.shape)
    db, dg = output(want_bias, weight.shape[:1]), output(want_gate, (x.shape[0], l.outer))
    L = lib()
    ws = _workspace(L.sihc_linear_act_backward_workspace_size(ctypes.byref(l), int(gate is not None)), x.device)
    check(L.sihc_linear_act_backward(ctypes.byref(l), grad.data_ptr(), x.data_ptr(), weight.data_ptr(),
                                     h.data_ptr() or None, low.data_ptr() or None, _ptr(gate),
                                     *(t.data_ptr() if wanted else None for t, wanted in
                                       ((dx, want_x), (dw, want_weight), (db, want_bias), (dg, want_gate))),
                                     ws.data_ptr(), ws.numel() * 4, _stream(x.device)))
    if want_gate and not l.rows:
        dg.zero_()  # a gate of no rows
    return dx, dw, db, dg


def _heads(q: Tensor, k: Optional[Tensor], weight: Optional[Tensor], positions: Tensor, axes: Sequence[int],
           theta: float, eps: float, inverse: bool) -> Heads:
    strides = [(ctypes.c_int64 * 3)(*(t.stride()[:3] if t is not None else ())) for t in (q, k)]
    code = dtype_code(q.dtype)
    return Heads(q.shape[0], q.shape[1], q.shape[2], 0 if k is None else k.shape[2], q.shape[3], len(axes),
                 (ctypes.c_int * MAX_AXES)(*axes), *strides, q.shape[1] if positions.ndim == 3 else 0, theta, eps, code,
                 code if weight is None else dtype_code(weight.dtype),
                 POSITION_F32 if positions.dtype == torch.float32 else POSITION_I32, int(inverse))


@_on_tensor_device
def qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, positions: Tensor, axes: Sequence[int],
                   theta: float, eps: float) -> tuple[Tensor, Tensor]:
    """q [B,N,H,D] and k [B,N,KH,D], normed by head and turned, packed."""
    oq, ok = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k))
    if not q.numel():
        return oq, ok
    h = _heads(q, k, q_weight, positions, axes, theta, eps, False)
    check(lib().sihc_qk_norm_rotary(ctypes.byref(h), q.data_ptr(), k.data_ptr(), q_weight.data_ptr(),
                                    k_weight.data_ptr(), positions.data_ptr(), oq.data_ptr(), ok.data_ptr(),
                                    _stream(q.device)))
    return oq, ok


@_on_tensor_device
def qk_norm_rotary_backward(grad_q: Tensor, grad_k: Tensor, q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor,
                            positions: Tensor, axes: Sequence[int], theta: float,
                            eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(q, k, q_weight, k_weight gradients) of qk_norm_rotary, packed."""
    dq, dk = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k))
    if not q.numel():
        return dq, dk, torch.zeros_like(q_weight), torch.zeros_like(k_weight)
    dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
    L, h = lib(), _heads(q, k, q_weight, positions, axes, theta, eps, False)
    ws = _workspace(L.sihc_qk_norm_rotary_backward_workspace_size(ctypes.byref(h)), q.device)
    check(L.sihc_qk_norm_rotary_backward(ctypes.byref(h), grad_q.data_ptr(), grad_k.data_ptr(), q.data_ptr(),
                                         k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                                         positions.data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(),
                                         ws.data_ptr(), ws.numel() * 4, _stream(q.device)))
    return dq, dk, dqw, dkw


@_on_tensor_device
def axis_rotary(x: Tensor, positions: Tensor, axes: Sequence[int], theta: float, inverse: bool) -> Tensor:
    """x [B,N,H,D] turned by its positions, or back, packed."""
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    h = _heads(x, None, None, positions, axes, theta, 0.0, inverse)
    check(lib().sihc_qk_norm_rotary(ctypes.byref(h), x.data_ptr(), None, None, None, positions.data_ptr(),
                                    out.data_ptr(), None, _stream(x.device)))
    return out


@_on_tensor_device
def dropout(x: Tensor, p: float, seed: Tensor, stream: int, residual: Optional[Tensor]) -> Tensor:
    """residual + x / (1 - p) where the mask of (seed, stream) keeps an element."""
    out = torch.empty_like(x)
    check(lib().sihc_dropout(x.data_ptr(), _ptr(residual), out.data_ptr(), x.numel(), p, seed.data_ptr(), stream,
                             dtype_code(x.dtype), _stream(x.device)))
    return out


__all__ = [
    "MAX_EVENTS", "ACTIVATIONS", "LINEAR_ACTIVATIONS", "linear_act", "linear_act_backward", "qk_norm_rotary",
    "qk_norm_rotary_backward", "axis_rotary", "dropout", "embedding", "embedding_backward", "group_norm", "group_norm_backward",
    "cross_attention", "cross_attention_backward", "dtype_code", "carrier_geometry", "read", "write", "weight_grad", "read_backward",
    "write_backward", "triangular",
    "triangular_gamma_grad", "triangular_backward", "event_forward", "event_backward", "gather_cells",
    "scatter_cells", "scatter_add_cells", "copy_",
]
