"""CPU: what the body operators refuse, in the C entries and in the Python ones, the shapes of their fakes, and
the generator's published answers."""
from __future__ import annotations

import ctypes
import subprocess
import sys

import numpy as np
import pytest
import torch

import body_reference as R
from sihc_hip import _lib, body
from sihc_hip.e2e import SiHCDenoiser, rope_positions, rope_tables

FAKE = 0x1000  # never dereferenced


def refused(rc, text):
    assert rc == 1 and text in _lib.lib().sihc_last_error(), _lib.lib().sihc_last_error()


def linear_sizes(**over):
    values = dict(rows=32, inner=64, outer=48, act=0, dtype=1, rows_per_gate=16, gate_stride=48)
    return ctypes.byref(_lib.Linear(*{**values, **over}.values()))


def test_linear_arguments():
    L = _lib.lib()

    def call(l, x=FAKE, y=FAKE * 9, h=None, low=None, ws=FAKE * 8, n=1 << 40):
        return L.sihc_linear_act(l, x, FAKE * 2, None, FAKE * 3, None, y, h, low, ws, n, None)

    refused(call(None), b"null sizes")
    refused(call(linear_sizes(dtype=4)), b"bad dtype")
    refused(call(linear_sizes(act=3)), b"bad activation")
    for over in (dict(rows=-1), dict(inner=0), dict(outer=0), dict(outer=(1 << 24) + 1), dict(rows=(1 << 30) + 1)):
        refused(call(linear_sizes(**over)), b"at most 2^30 rows")
    refused(call(linear_sizes(rows_per_gate=5)), b"of 5 a gate")
    refused(call(linear_sizes(), x=None), b"null pointer")
    refused(call(linear_sizes(), low=FAKE * 4, h=FAKE * 5), b"for bf16 with an activation")
    refused(call(linear_sizes(), y=FAKE), b"one of the inputs")
    assert call(linear_sizes(rows=0)) == 0
    # few rows over a long contraction: parts, whose sums need a workspace
    need = L.sihc_linear_act_workspace_size(linear_sizes(rows=512, inner=16384, outer=1024, rows_per_gate=512))
    if need:
        refused(call(linear_sizes(rows=512, inner=16384, outer=1024, rows_per_gate=512), n=need - 1), b"workspace of")

    def back(l, h=FAKE * 4, low=None, dx=FAKE * 5, dgate=FAKE * 6, gate=FAKE * 3, ws=FAKE * 8, n=1 << 40):
        return L.sihc_linear_act_backward(l, FAKE * 9, FAKE, FAKE * 2, h, low, gate, dx, FAKE * 10, FAKE * 11, dgate, ws, n, None)

    refused(back(linear_sizes(), h=None), b"null pointer")
    refused(back(linear_sizes(act=1)), b"null pointer")  # bf16 with an activation wants the other bits
    refused(back(linear_sizes(), gate=None), b"no gate")
    refused(back(linear_sizes(), dx=FAKE), b"one of the inputs")
    need = L.sihc_linear_act_backward_workspace_size(linear_sizes(), 1)
    assert need >= 32 * 48 * 2 + 2 * 48 * 4
    refused(back(linear_sizes(), n=need - 1), b"workspace of")
    assert L.sihc_linear_act_backward_workspace_size(linear_sizes(rows=-4), 1) == 0


def heads_sizes(**over):
    three, widths = (ctypes.c_int64 * 3)(64, 64, 8), (ctypes.c_int * 4)(4, 4)
    values = dict(batch=2, tokens=4, heads=4, kv_heads=2, dim=16, axes=2, widths=widths, q_stride=three, k_stride=three,
                  position_batch_stride=0, theta=1e4, eps=1e-6, dtype=1, w_dtype=1, position_dtype=0, inverse=0)
    return ctypes.byref(_lib.Heads(*{**values, **over}.values()))


def test_heads_arguments():
    L = _lib.lib()

    def call(h, k=FAKE * 2, qw=FAKE * 3, kw=FAKE * 4, positions=FAKE * 5, out=FAKE * 6):
        return L.sihc_qk_norm_rotary(h, FAKE, k, qw, kw, positions, out, FAKE * 7, None)

    refused(call(None), b"null sizes")
    refused(call(heads_sizes(dtype=3)), b"bad dtype")
    refused(call(heads_sizes(dtype=0, w_dtype=1)), b"weights of the heads' type")
    refused(call(heads_sizes(position_dtype=2)), b"positions are")
    refused(call(heads_sizes(heads=0)), b"bad sizes")
    refused(call(heads_sizes(dim=257)), b"1..256 channels")
    refused(call(heads_sizes(heads=(1 << 20) + 1)), b"too many heads")
    refused(call(heads_sizes(batch=1 << 40, tokens=1 << 20)), b"at most 2^31 - 64 tokens")
    refused(call(heads_sizes(batch=1, tokens=1 << 30, heads=64, dim=64)), b"too many tokens for a launch")
    refused(call(heads_sizes(axes=5)), b"0..4 axes")
    refused(call(heads_sizes(widths=(ctypes.c_int * 4)(3, 4))), b"turns 3 channels")
    refused(call(heads_sizes(widths=(ctypes.c_int * 4)(10, 8))), b"turn 18 channels of 16")
    refused(call(heads_sizes(theta=0.0)), b"theta")
    refused(call(heads_sizes(eps=-1.0)), b"eps")
    refused(call(heads_sizes(), k=None), b"keys go with kv_heads")
    refused(call(heads_sizes(), kw=None), b"both sides or of none")
    refused(call(heads_sizes(), positions=None), b"null pointer")
    refused(call(heads_sizes(), out=FAKE), b"one of the inputs")
    assert call(heads_sizes(batch=0)) == 0
    need = L.sihc_qk_norm_rotary_backward_workspace_size(heads_sizes())
    assert need == 2 * 16 * 4  # eight tokens of few heads: one wave, one block
    back = lambda n: L.sihc_qk_norm_rotary_backward(heads_sizes(), *[FAKE * i for i in range(1, 8)],  # noqa: E731
                                                    *[FAKE * i for i in range(8, 12)], FAKE * 12, n, None)
    refused(back(need - 1), b"workspace of")


def test_dropout_arguments():
    L = _lib.lib()
    call = lambda p=0.1, n=8, stream=0, dtype=1, key=FAKE: L.sihc_dropout(FAKE, None, FAKE, n, p, key, stream, dtype,  # noqa: E731
                                                                          None)
    refused(call(p=1.0), b"p must lie")
    refused(call(p=float("nan")), b"p must lie")
    refused(call(n=-1), b"negative")
    refused(call(stream=-1), b"negative")
    refused(call(dtype=2), b"bad dtype")
    refused(call(key=None), b"null pointer")
    assert call(n=0) == 0


# The library's answers to sizes that no tensor has, asked in a process of their own.
ASK = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from sihc_hip import _lib
L = _lib.lib()
l = lambda rows, inner, outer, each, act=0: ctypes.byref(_lib.Linear(rows, inner, outer, act, 1, each, outer))
print({})
"""


@pytest.mark.parametrize("sizes", ["1 << 62, 8, 8, 1", "1 << 30, 1 << 24, 1 << 24, 1 << 30, 2", "1 << 30, 1 << 24, 1 << 24, 1",
                                   "(1 << 63) - 1, 1, 1, 1", "1, 1 << 24, 1 << 24, 1", "1 << 30, 1, 1, 1 << 30", "4, 8, 8, 0"])
def test_the_largest_sizes_have_an_answer(sizes):
    call = f"L.sihc_linear_act_workspace_size(l({sizes})) >= 0, L.sihc_linear_act_backward_workspace_size(l({sizes}), 1) >= 0"
    done = subprocess.run([sys.executable, "-c", ASK.format(call), str(_lib.LIB_PATH.parents[1])], capture_output=True,
                          text=True, timeout=60)
    assert done.returncode == 0 and done.stdout.split() == ["True", "True"], done.stderr


# ----------------------------------------------------------------------------- the public entries
def x_(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("match,call", [
    ("act must be", lambda: body.linear_act(x_(2, 4), x_(3, 4), act="relu")),
    ("requires contiguous x", lambda: body.linear_act(x_(4, 2).t(), x_(3, 4))),
    ("requires contiguous weight", lambda: body.linear_act(x_(2, 4), x_(4, 3).t())),
    ("expected x", lambda: body.linear_act(x_(2, 4), x_(3, 5))),
    ("expected x", lambda: body.linear_act(x_(4), x_(3, 4))),
    ("an even number", lambda: body.linear_act(x_(2, 4), x_(3, 4), act="swiglu")),
    ("a weight of", lambda: body.linear_act(x_(2, 0), x_(3, 0))),
    ("a bias", lambda: body.linear_act(x_(2, 4), x_(6, 4), x_(3), "swiglu")),
    ("a gate", lambda: body.linear_act(x_(2, 5, 4), x_(6, 4), None, "swiglu", x_(2, 6))),
    ("a gate", lambda: body.linear_act(x_(2, 5, 4), x_(6, 4), None, "none", x_(10, 6))),
    ("contiguous channels of the gate", lambda: body.linear_act(x_(2, 4), x_(3, 4), None, "none", x_(3, 2).t())),
    ("a residual", lambda: body.linear_act(x_(2, 5, 4), x_(3, 4), residual=x_(10, 3))),
    ("share float32 or bfloat16", lambda: body.linear_act(x_(2, 4), x_(3, 4, dtype=torch.bfloat16))),
    ("share float32 or bfloat16", lambda: body.linear_act(*(x_(3, 4, dtype=torch.float64),) * 2)),
    ("CUDA device", lambda: body.linear_act(x_(2, 4), x_(3, 4))),
    ("expected \\[batch", lambda: body.axis_rotary(x_(2, 4, 8), x_(4, 1), (8,))),
    ("expected \\[batch", lambda: body.qk_norm_rotary(x_(2, 4, 2, 8), x_(2, 5, 2, 8), x_(8), x_(8), x_(4, 1), (8,))),
    ("1..256 channels", lambda: body.axis_rotary(x_(1, 1, 1, 260), x_(1, 1), (8,))),
    ("contiguous channels of x", lambda: body.axis_rotary(x_(2, 4, 8, 2).transpose(2, 3), x_(4, 1), (8,))),
    ("even widths", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 1), (7,))),
    ("even widths", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 2), (6, 4))),
    ("even widths", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 5), (0,) * 5)),
    ("theta", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 1), (8,), -1.0)),
    ("expected positions", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(3, 4, 1), (8,))),
    ("int32 or float32", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 1, dtype=torch.int64), (8,))),
    ("requires contiguous positions", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(2, 4).t(), (4, 4))),
    ("weights must be", lambda: body.qk_norm_rotary(*(x_(2, 4, 2, 8),) * 2, x_(8), x_(4), x_(4, 1), (8,))),
    ("weights of the heads", lambda: body.qk_norm_rotary(*(x_(2, 4, 2, 8),) * 2, *(x_(8, dtype=torch.bfloat16),) * 2, x_(4, 1),
                                                         (8,))),
    ("eps", lambda: body.qk_norm_rotary(*(x_(2, 4, 2, 8),) * 2, x_(8), x_(8), x_(4, 1), (8,), 1e4, -1.0)),
    ("CUDA device", lambda: body.qk_norm_rotary(*(x_(2, 4, 2, 8),) * 2, x_(8), x_(8), x_(4, 1), (8,))),
    ("CUDA device", lambda: body.axis_rotary(x_(2, 4, 2, 8), x_(4, 1), (8,))),
    ("p must lie", lambda: body.dropout(x_(4), 1.0, x_(1, dtype=torch.int64))),
    ("one int64", lambda: body.dropout(x_(4), 0.1, x_(2, dtype=torch.int64))),
    ("one int64", lambda: body.dropout(x_(4), 0.1, x_(1, dtype=torch.int32))),
    ("stream must lie", lambda: body.dropout(x_(4), 0.1, x_(1, dtype=torch.int64), -1)),
    ("residual must match", lambda: body.dropout(x_(4), 0.1, x_(1, dtype=torch.int64), 0, x_(5))),
    ("requires contiguous x", lambda: body.dropout(x_(4, 2).t(), 0.1, x_(1, dtype=torch.int64))),
    ("CUDA device", lambda: body.dropout(x_(4), 0.1, x_(1, dtype=torch.int64))),
])
def test_public_entries_refuse(match, call):
    with pytest.raises(ValueError, match=match):
        call()


def test_fakes_give_the_real_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        assert body.linear_act(e(2, 5, 8), e(12, 8), e(12), "swiglu", e(2, 6), e(2, 5, 6)).shape == (2, 5, 6)
        y, h, low = body._linear_act(e(2, 5, 8), e(36, 8), None, "swiglu", None, None)
        assert y.shape == (2, 5, 18) and h.shape == (2, 5, 36) and low.shape == (2, 5, 2, 3) and low.dtype == torch.int32
        y, h, low = body._linear_act(e(2, 5, 8), e(36, 8), None, "none", None, None)
        assert y.shape == (2, 5, 36) and h.shape == (0,) and low.shape == (0,)
        qkv = e(2, 5, 8, 16)
        q, k = body.qk_norm_rotary(qkv[:, :, :4], qkv[:, :, 4:6], e(16), e(16), e(5, 2, dtype=torch.int32), (8, 6))
        assert q.shape == (2, 5, 4, 16) and k.shape == (2, 5, 2, 16) and q.is_contiguous()
        assert body.axis_rotary(qkv, e(5, 1, dtype=torch.float32), (16,)).shape == qkv.shape
        assert body.dropout(e(3, 4), 0.5, e(1, dtype=torch.int64)).shape == (3, 4)


def test_the_generators_published_answers():
    """The known answers of Philox 4x32 with 10 rounds for counters and keys of zeros and of ones."""
    zeros = R.philox(np.zeros((1, 4), np.uint64), (0, 0))[0]
    assert [hex(int(v)) for v in zeros] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = R.philox(np.full((1, 4), 0xffffffff, np.uint64), (0xffffffff, 0xffffffff))[0]
    assert [hex(int(v)) for v in ones] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_the_denoisers_positions_are_its_tables():
    """The rotation by rows and columns is that of the denoiser's cosines and sines."""
    cos, sin = rope_tables(24, 5)
    x = torch.randn(1, 25, 3, 24, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    pairs = x.reshape(1, 25, 3, 12, 2)
    rotated = torch.stack((-pairs[..., 1], pairs[..., 0]), -1).reshape(x.shape)
    want = x * cos.double()[None, :, None] + rotated * sin.double()[None, :, None]
    got = R.turned(x, rope_positions(5), (12, 12), 10000.0)
    assert float((got - want).abs().max()) < 4 * 2.0 ** -24
    assert torch.equal(rope_positions(5, 3)[:3], torch.zeros(3, 2, dtype=torch.int32))


def test_the_denoisers_choices():
    with pytest.raises(ValueError, match="body must be"):
        SiHCDenoiser(hidden=32, heads=2, depth=8, stages=(8,), body="other")
    with pytest.raises(ValueError, match="at most 128 channels"):
        SiHCDenoiser(hidden=320, heads=2, depth=8, stages=(8,), body="fused")
    with pytest.raises(ValueError, match="dropout must lie"):
        SiHCDenoiser(hidden=32, heads=2, depth=8, stages=(8,), dropout=1.0)
    plain, fused = (SiHCDenoiser(hidden=32, heads=2, depth=8, stages=(8,), body=b) for b in ("torch", "fused"))
    assert list(plain.state_dict()) == list(fused.state_dict())
