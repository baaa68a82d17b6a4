"""CPU: a product in parts is refused without the whole of its workspace."""
from __future__ import annotations

import ctypes

from sihc_hip import _lib

FAKE = 0x1000  # never dereferenced


def test_a_small_workspace_is_refused():
    """Of products of few rows over long contractions at least one is in parts, whatever the plans' costs."""
    L, seen = _lib.lib(), 0
    for rows, inner, outer in ((512, 16384, 1024), (256, 32768, 512), (1024, 65536, 256), (128, 65536, 2048)):
        for dtype in (0, 1):
            sizes = ctypes.byref(_lib.Linear(rows, inner, outer, 0, dtype, rows, 0))
            need = L.sihc_linear_act_workspace_size(sizes)
            if not need:
                continue
            seen += 1
            for pointer, bytes_ in ((FAKE, need - 1), (None, need), (FAKE, 0)):
                rc = L.sihc_linear_act(sizes, FAKE * 2, FAKE * 3, None, None, None, FAKE * 4, None, None, pointer, bytes_, None)
                assert rc == 1 and b"workspace of" in L.sihc_last_error()
    assert seen >= 4
