"""CPU: the sizes that the body operators refuse, of tensors that take no memory."""
from __future__ import annotations

import ctypes

import pytest
import torch

from sihc_hip import _lib, body

FAKE = 0x1000  # never dereferenced
FULL = (1 << 26) - 4  # waves of a launch


def heads(tokens, count, dim):
    return torch.zeros(1, 1, 1, dim).expand(1, tokens, count, dim)


@pytest.mark.parametrize("count,dim,each", [(129, 8, 1), (128, 8, 2), (16, 64, 2), (9, 72, 1), (1, 256, 8), (3, 256, 2), (5, 256, 1),
                                            (64, 1, 4), (65, 16, 1), (64, 16, 2), (2, 136, 4)])
def test_tokens_of_a_launch(count, dim, each):
    """The limit is the C entry's: its last size passes every check but the device's, one more does not."""
    most = FULL * each
    none = torch.zeros(most, 0, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        body.axis_rotary(heads(most, count, dim), none, ())
    with pytest.raises(ValueError, match=f"at most {most} tokens"):
        body.axis_rotary(heads(most + 1, count, dim), torch.zeros(most + 1, 0, dtype=torch.int32), ())
    if count > 1:  # queries and keys share a wave
        w = torch.ones(dim)
        with pytest.raises(ValueError, match=f"at most {most} tokens"):
            body.qk_norm_rotary(heads(most + 1, count - 1, dim), heads(most + 1, 1, dim), w, w,
                                torch.zeros(most + 1, 0, dtype=torch.int32), ())
    L = _lib.lib()
    sizes = _lib.Heads(1, most + 1, count, 0, dim, 0, (ctypes.c_int * 4)(), (ctypes.c_int64 * 3)(0, 0, dim),
                       (ctypes.c_int64 * 3)(), 0, 1e4, 0.0, 1, 1, 0, 0)
    assert L.sihc_qk_norm_rotary(ctypes.byref(sizes), FAKE, None, None, None, None, FAKE * 2, None, None) == 1
    assert b"too many tokens for a launch" in L.sihc_last_error()
