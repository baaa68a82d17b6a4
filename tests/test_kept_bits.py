"""CPU: the oracle of the kept bits of h, and that it tells a misplaced word or nibble from a right one."""
from __future__ import annotations

import pytest
import torch

import kept_bits as K


@pytest.mark.parametrize("outer,parts", [(8, 1), (13, 2), (1, 2), (40, 1)])
def test_what_is_packed_is_what_is_read(outer, parts):
    values = torch.randn(6, parts * outer, generator=torch.Generator().manual_seed(outer)) * 3
    h, low = K.pack(values, parts)
    assert h.shape == values.shape and low.shape == (6, parts, (outer + 7) // 8)
    back = K.unpack(h, low)
    assert ((back - values).abs() <= 2 * K.HALF * values.abs()).all()
    again = K.pack(back, parts)
    assert torch.equal(again[0].view(torch.int16), h.view(torch.int16)) and torch.equal(again[1], low)


def test_misplaced_bits_leave_the_bound():
    outer = 16
    values = torch.randn(64, 2 * outer, generator=torch.Generator().manual_seed(0))
    h, low = K.pack(values, 2)
    reverse = sum(((low.to(torch.int64) >> (4 * i)) & 15) << (4 * (7 - i)) for i in range(8))
    wrong = {"nibbles in reverse": (reverse - ((reverse >> 31) << 32)).to(torch.int32), "another row": low.roll(1, 0),
             "the other half": low.flip(1), "another word": low.flip(2), "zeros": torch.zeros_like(low),
             "a constant": torch.full_like(low, 0x77777777)}
    for what, words in wrong.items():
        off = (K.unpack(h, words).double() - values.double()).abs()
        assert (off > 2 * K.HALF * values.abs()).any(), what
