"""CPU: what the conditioning operators refuse by size, in the C entries and in the Python ones alike."""
from __future__ import annotations

import subprocess
import sys

import pytest
import torch

from sihc_hip import _lib, conditioning

FAKE = 0x1000  # never dereferenced


def refused(rc, text):
    assert rc == 1 and text in _lib.lib().sihc_last_error()


# channels of one group: the widest, and the next of the same divisors
@pytest.mark.parametrize("dtype,code,most,more", [(torch.bfloat16, 1, 4096, 4104), (torch.bfloat16, 1, 2044, 2052),
                                                  (torch.bfloat16, 1, 2046, 2050), (torch.bfloat16, 1, 1023, 1025),
                                                  (torch.float32, 0, 2048, 2052), (torch.float32, 0, 2046, 2050),
                                                  (torch.float32, 0, 1023, 1025), (torch.float32, 0, 1023, 4097)])
@pytest.mark.parametrize("groups", [1, 3])
def test_the_widest_groups(dtype, code, most, more, groups):
    from torch._subclasses.fake_tensor import FakeTensorMode
    L = _lib.lib()
    assert conditioning._widest_group(most, dtype) >= most and conditioning._widest_group(more, dtype) < more
    for width, taken in ((most, True), (more, False)):
        need = L.sihc_group_norm_backward_workspace_size(2, 4, groups * width, groups, code)
        assert (need > 0) == taken
        with FakeTensorMode():
            x, w = torch.empty(2, 4, groups * width, dtype=dtype, device="cuda"), torch.empty(groups * width, device="cuda")
            if taken:
                assert conditioning.group_norm_act(x, w, w, groups).shape == x.shape
            else:
                with pytest.raises(ValueError, match=f"groups of {width} channels"):
                    conditioning.group_norm_act(x, w, w, groups)
        if not taken:
            refused(L.sihc_group_norm(FAKE, FAKE, FAKE, FAKE, None, 2, 4, groups * width, groups, 1e-6, 1, code, code, None,
                                      0, None), b"too wide")
            with pytest.raises(ValueError, match=f"groups of {width} channels"):  # (CPU tensors: sizes are looked at first)
                conditioning._check_norm(torch.zeros(2, 1, groups * width, dtype=dtype), torch.zeros(groups * width),
                                         torch.zeros(groups * width), groups, "silu")


def test_the_most_channels_of_a_norm():
    """A width whose two sums a channel pass int32 was taken."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    L = _lib.lib()
    most = 1 << 24
    assert L.sihc_group_norm_backward_workspace_size(1, 1, most, most // 8, 1) == 2 * most * 4 + 2 * most * 4 + most // 8 * 8
    for channels in (2 * most, 1 << 30):
        refused(L.sihc_group_norm(FAKE, FAKE, FAKE, FAKE, None, 1, 1, channels, channels // 8, 1e-6, 1, 1, 1, FAKE, 1 << 40,
                                  None), b"bad sizes")
        with FakeTensorMode():
            x, w = torch.empty(1, channels, dtype=torch.bfloat16, device="cuda"), torch.empty(channels, device="cuda")
            with pytest.raises(ValueError, match="at most 16777216 channels"):
                conditioning.group_norm_act(x, w, w, channels // 8)


# The library's answers to sizes that no tensor has, asked in a process of their own: such a call has ended
# in an arithmetic fault and in a loop without end.
ASK = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from sihc_hip import _lib
three = (ctypes.c_int64 * 3)(1, 1, 1)
L, a = _lib.lib(), lambda batch, kv: ctypes.byref(_lib.Attention(batch, 4, 6, 2 * kv, kv, 16, three, three, three, 1.0, 1))
print({})
"""


def answer(call):
    done = subprocess.run([sys.executable, "-c", ASK.format(call), str(_lib.LIB_PATH.parents[1])], capture_output=True,
                          text=True, timeout=60)
    assert done.returncode == 0, (done.returncode, done.stderr)
    return done.stdout.split()


def test_batches_past_64_bits_of_attention_blocks():
    for batch, heads in ((1 << 62, 4), (1 << 61, 8), ((1 << 63) - 1, 2)):
        assert answer(f"L.sihc_cross_attention_workspace_size(a({batch}, {heads})), "
                      f"L.sihc_cross_attention_backward_workspace_size(a({batch}, {heads})), b'too large' in L.sihc_last_error()"
                      ) == ["0", "0", "True"]


def test_workspaces_of_tables_that_no_memory_holds():
    calls = [f"L.sihc_embedding_backward_workspace_size({tokens}, {rows}, {channels})"
             for tokens, rows, channels in ((4096, (1 << 62) + 1, 64), (4096, (1 << 63) - 1, 64), (1 << 62, 100, 64),
                                            (4096, 100, 1 << 30), (-1, 100, 64), (4096, 0, 64))]
    assert answer(", ".join(calls)) == ["0"] * len(calls)
