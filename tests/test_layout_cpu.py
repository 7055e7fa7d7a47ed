"""The binding checks that the library was built with its layout (CPU)."""
import ctypes as C

import pytest

from kascade_b200 import _native as nat


def test_size_of_the_layout():
    assert nat.load().kb200_kv_layout_bytes() == C.sizeof(nat.KvLayout) == nat._LAYOUT.size

    class Old:                                                       # a library without the call
        pass

    class Other:
        kb200_kv_layout_bytes = staticmethod(type("F", (), {"__call__": lambda self: 104})())

    for lib in (Old(), Other()):
        with pytest.raises(nat.KascadeNativeError, match="other sources"):
            nat._check_layout(lib)
