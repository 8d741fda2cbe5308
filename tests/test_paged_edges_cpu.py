"""Host side of the paged serving step at its edges (no GPU)."""

from __future__ import annotations

from fade_b200 import _lib


def test_wait_polls_are_bounded():
    lib = _lib.load()
    try:
        assert lib.fade_set_wait_polls((1 << 22) + 1) == _lib.FADE_ERR_INVALID_ARG
        assert lib.fade_set_wait_polls(0) == lib.fade_set_wait_polls(1 << 22) == _lib.FADE_OK
    finally:
        assert lib.fade_set_wait_polls(-1) == _lib.FADE_OK
