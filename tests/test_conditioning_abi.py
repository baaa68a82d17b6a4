"""CPU: the C entries of the conditioning operators reject bad arguments before any launch, and their
fake implementations give the shapes and types of the real ones."""
from __future__ import annotations

import ctypes

import pytest
import torch

from sihc_hip import _lib, conditioning

FAKE = 0x1000  # never dereferenced


def refused(rc, text):
    assert rc == 1 and text in _lib.lib().sihc_last_error()


def test_embedding_arguments():
    L = _lib.lib()
    refused(L.sihc_embedding(FAKE, FAKE, FAKE, 4, 9, 8, 1.0, 16, 1, None), b"16 bits")
    refused(L.sihc_embedding(FAKE, FAKE, FAKE, 4, 9, 8, 1.0, 32, 5, None), b"bad dtype")
    refused(L.sihc_embedding(FAKE, FAKE, FAKE, 4, 0, 8, 1.0, 32, 1, None), b"bad sizes")
    refused(L.sihc_embedding(FAKE, None, FAKE, 4, 9, 8, 1.0, 32, 1, None), b"null pointer")
    assert L.sihc_embedding(None, None, None, 0, 9, 8, 1.0, 32, 1, None) == 0
    assert L.sihc_embedding_backward_workspace_size(1024, 1000, 64) == 0
    need = L.sihc_embedding_backward_workspace_size(4096, 1000, 64)
    assert need >= 2 * 4096 * 8 + 128 * 2 * 64 * 4
    refused(L.sihc_embedding_backward(FAKE, FAKE, 2 * FAKE, 4096, 1000, 64, 1.0, -1, 64, 1, FAKE, need - 1, None),
            b"workspace of")
    refused(L.sihc_embedding_backward(FAKE, FAKE, FAKE, 4096, 1000, 64, 1.0, -1, 64, 1, FAKE, need, None),
            b"one of the inputs")


def test_group_norm_arguments():
    L = _lib.lib()
    call = lambda c, g, act, dt, wt: L.sihc_group_norm(FAKE, FAKE, FAKE, FAKE, None, 2, 16, c, g, 1e-6, act, dt,  # noqa: E731
                                                        wt, None, 0, None)
    refused(call(10, 3, 1, 1, 1), b"are not 3 groups")
    refused(call(8, 2, 7, 1, 1), b"bad activation")
    refused(call(8, 2, 1, 4, 1), b"bad dtype")
    refused(call(8, 2, 1, 0, 1), b"weights must be fp32 or share")
    refused(call(1025, 1, 1, 1, 1), b"too wide")
    need = L.sihc_group_norm_backward_workspace_size(2, 16, 8, 2, 1)
    assert need == 2 * 2 * 8 * 4
    refused(L.sihc_group_norm_backward(FAKE, FAKE * 2, FAKE * 3, FAKE * 4, FAKE * 5, FAKE * 6, FAKE * 7, FAKE * 8, 2, 16, 8,
                                       2, 1, 1, 1, FAKE, need - 4, None), b"workspace of")
    refused(L.sihc_group_norm_backward(FAKE, FAKE * 2, FAKE * 3, FAKE * 4, FAKE * 5, FAKE, FAKE * 7, FAKE * 8, 2, 16, 8, 2,
                                       1, 1, 1, FAKE, need, None), b"one of the inputs")
    # a slice of 128 x 128 pixels does not fit a block: its chunks' statistics need a workspace
    assert L.sihc_group_norm_workspace_size(1, 128 * 128, 36, 1, 1) > 0
    assert L.sihc_group_norm_workspace_size(1, 32 * 32, 36, 1, 1) == 0


def test_cross_attention_arguments():
    L = _lib.lib()

    def sizes(**over):
        three = (ctypes.c_int64 * 3)(1, 1, 1)
        values = dict(batch=2, queries=4, keys=6, heads=4, kv_heads=2, dim=16, q_stride=three, k_stride=three,
                      v_stride=three, scale=1.0, dtype=1)
        return ctypes.byref(_lib.Attention(*{**values, **over}.values()))

    call = lambda a, q=FAKE: L.sihc_cross_attention(a, q, FAKE, FAKE, None, FAKE, None, None, None, 0, None)  # noqa: E731
    refused(call(sizes(heads=3)), b"do not share")
    refused(call(sizes(dim=129)), b"at most 128")
    refused(call(sizes(dtype=3)), b"bad dtype")
    refused(call(sizes(queries=-1)), b"bad sizes")
    refused(call(sizes(batch=1 << 40)), b"too large")
    refused(call(sizes(), None), b"null pointer")
    refused(call(None), b"null sizes")
    assert call(sizes(batch=0)) == 0
    back = lambda a, dq, n: L.sihc_cross_attention_backward(a, FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE,  # noqa: E731
                                                            dq, FAKE * 2, FAKE * 3, FAKE, n, None)
    need = L.sihc_cross_attention_backward_workspace_size(sizes())
    assert need >= 2 * 4 * 4 * 4
    refused(back(sizes(), FAKE * 4, need - 1), b"workspace of")
    refused(back(sizes(), FAKE, need), b"one of the inputs")


def test_fakes_give_the_real_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        table, ids = torch.empty(9, 8, device="cuda"), torch.empty(2, 3, dtype=torch.int64, device="cuda")
        assert conditioning.embedding_lookup(table, ids, validate=False).shape == (2, 3, 8)
        x, w = torch.empty(2, 4, 4, 8, device="cuda"), torch.empty(8, device="cuda")
        assert conditioning.group_norm_act(x, w, w, 2).shape == x.shape
        q, k = torch.empty(2, 5, 4, 16, device="cuda"), torch.empty(2, 7, 2, 16, device="cuda")
        assert conditioning.cross_attention(q, k, k, None, validate=False).shape == q.shape


@pytest.mark.parametrize("call", [
    lambda: conditioning.embedding_lookup(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)),
    lambda: conditioning.group_norm_act(torch.zeros(1, 2, 2, 4), torch.ones(4), torch.zeros(4), 2),
    lambda: conditioning.cross_attention(*[torch.zeros(1, 2, 1, 4)] * 3),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA device"):
        call()
