"""How much of what O's rounding drops a training call keeps (CPU: sizes only)."""
import torch

from lv_xattn_b200 import _lib, ops


def rows(sq, skv, start=-1, lengths=None, dtype=torch.bfloat16):
    return ops.window_low_rows(torch.empty(2, 4, sq, 128, dtype=dtype), torch.empty(2, 2, skv, 128, dtype=dtype), start, lengths)


def test_no_more_rows_than_are_early():
    """Against the positions one by one; with lengths, whatever they are."""
    for sq in (1, 2, 16, 255, 256, 257, 1000):
        for skv in (0, 1, 16, 200, 256, 300, 1000, 1300):
            early = sum(0 <= skv - sq + i < _lib.LOW_ROWS for i in range(sq))
            assert rows(sq, skv) == early
            lengths = torch.full((2,), skv)
            assert early <= rows(sq, skv, -1, lengths) <= min(sq, _lib.LOW_ROWS)
        for start in (0, 1, 100, 255, 256, 5000):
            early = sum(start + i < _lib.LOW_ROWS for i in range(sq))
            assert rows(sq, 1300, start) == early and rows(sq, 1300, start, torch.zeros(2)) == early


def test_short_texts_keep_no_more_than_their_output():
    assert rows(16, 16) == 16 and rows(16, 16, 0) == 16 and rows(1, 1) == 1
    assert rows(1000, 9192) == 0 and rows(1, 8192) == 0      # a chunk and a token behind a long cache
    assert rows(16, 16, dtype=torch.float32) == 0 and rows(4096, 4096) == _lib.LOW_ROWS


def test_abi_refusals():
    import ctypes
    lib = _lib.load()
    f, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    for n, rc in ((0, 0), (1, 0), (256, 0), (257, -2), (-1, -2)):
        assert lib.lvx_window_workspace(ctypes.byref(_lib.LvxShape(1, 4, 2, 16, 16, 128, 0, 0)), ctypes.byref(_lib.LvxWindow(8, 0, -1, n)),
                                        ctypes.byref(f), ctypes.byref(b)) == rc
