"""The packed argument layouts are the structs they stand for."""
import ctypes as C
import struct

import pytest

from cutlass_b200 import lib as L

_SIZE = {C.c_int32: "i", C.c_int64: "q", C.c_void_p: "P"}


@pytest.mark.parametrize("cls,layout", [(L.Int8Args, L.INT8_LAYOUT), (L.ActArgs, L.ACT_LAYOUT), (L.RouteArgs, L.ROUTE_LAYOUT)])
def test_layout_equals_the_struct(cls, layout):
    s = struct.Struct("@" + layout)
    assert s.size == C.sizeof(cls)
    values = list(range(1, len(cls._fields_) + 1))
    a = cls.from_buffer_copy(s.pack(*values))
    assert [getattr(a, name) for name, _ in cls._fields_] == values
