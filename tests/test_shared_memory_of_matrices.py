"""Which matrices share memory: what decides whether a result may be written while its input is still read."""
import itertools

import torch

from cutlass_b200.int8 import _share_memory


def test_against_the_bytes():
    buf = torch.zeros(400, dtype=torch.int16)

    def view(at, rows, cols, pitch, wide):
        base = buf.view(torch.int32) if wide else buf
        return base[at:at + (rows - 1) * pitch + cols].as_strided((rows, cols), (pitch, 1))

    def bytes_of(t):
        size = t.element_size()
        return {t.data_ptr() + size * (r * t.stride(0) + c) + i for r in range(t.shape[0]) for c in range(t.shape[1]) for i in range(size)}
    views = [view(at, rows, cols, pitch, wide) for at, rows, cols, pitch, wide in itertools.product((0, 5, 8, 20, 60), (1, 4), (3, 10), (10, 20), (False, True))
             if cols <= pitch]
    for a, b in itertools.product(views, views):
        common = bool(bytes_of(a) & bytes_of(b))
        said = _share_memory(a, b)
        assert said or not common
        one_buffer = a.stride(0) * a.element_size() == b.stride(0) * b.element_size() and a.shape[0] > 1 and b.shape[0] > 1
        far = a.data_ptr() + 4 * 20 * a.element_size() <= b.data_ptr()
        if one_buffer and not common and a.shape == b.shape and a.data_ptr() // (a.stride(0) * a.element_size()) == b.data_ptr() // (a.stride(0) * a.element_size()):
            assert not said
        if far and not common:
            assert not said
