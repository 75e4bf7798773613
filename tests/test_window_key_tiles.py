"""The list of key tiles that the windowed kernels walk, as the library makes it, against the keys that their queries see."""
import ctypes
import itertools

import pytest

from lv_xattn_b200 import _lib

FAR = 1 << 28


def walked(window, sinks, valid, p0, p1, shift):
    tiles, count = (ctypes.c_int * 4096)(), ctypes.c_int(-1)
    rc = _lib.load().lvx_selftest_key_tiles(ctypes.byref(_lib.LvxWindow(window or 0, sinks, -1, 0)), valid, p0, p1, shift, tiles, 4096,
                                            ctypes.byref(count))
    assert rc == 0 and 0 <= count.value <= 4096
    return list(tiles[:count.value])


def seen(window, sinks, valid, p0, p1, shift):
    """From the definition: query p sees the keys j < valid, j <= p, of which j > p - window or j < sinks."""
    out = set()
    for p in range(p0, p1 + 1):
        last = min(p, valid - 1)
        for first, end in ((0 if window is None else max(0, p - window + 1), last), (0, min(sinks - 1, last))):
            if first <= end:
                out.update(range(first >> shift, (end >> shift) + 1))
    return out


@pytest.mark.parametrize("shift", [6, 7])
@pytest.mark.parametrize("window", [None, 1, 60, 64, 129, 400])
def test_every_seen_tile_once_and_no_other(shift, window):
    for sinks, valid, p0, n in itertools.product((0, 1, 64, 65, 200, 1000), (0, 1, 63, 64, 65, 128, 300, 700),
                                                 (-300, -3, 0, 63, 64, 130, 700, 1200), (1, 5, 33, 128)):
        got = walked(window, sinks, valid, p0, p0 + n - 1, shift)
        assert got == sorted(set(got)), (sinks, valid, p0, n)
        assert set(got) == seen(window, sinks, valid, p0, p0 + n - 1, shift), (sinks, valid, p0, n)


@pytest.mark.parametrize("shift", [6, 7])
def test_far_positions(shift):
    """The largest lengths and positions that a call may have: no product of them leaves 32 bits."""
    t = 1 << shift
    last = FAR - 1
    assert walked(100, 0, last, last - 1, last - 1, shift) == sorted({(last - 100) // t, (last - 1) // t})
    assert walked(1, 3, last, FAR - 2, FAR - 2, shift) == [0, (FAR - 2) // t]
    assert walked(FAR + 5, 0, 300, 2 * FAR - 2, 2 * FAR - 1, shift) == []      # the window ends before the last valid key
    assert walked(None, FAR, 300, 2 * FAR - 2, 2 * FAR - 1, shift) == list(range((299 >> shift) + 1))
    assert walked(None, 0, 5, -FAR + 1, -FAR + 20, shift) == []


def test_refusals():
    lib, n = _lib.load(), ctypes.c_int(0)
    win, tiles = ctypes.byref(_lib.LvxWindow(8, 0, -1, 0)), (ctypes.c_int * 4)()
    assert lib.lvx_selftest_key_tiles(win, 300, 0, 299, 6, tiles, 2, ctypes.byref(n)) == 0 and n.value == 5 and list(tiles) == [0, 1, 0, 0]
    assert lib.lvx_selftest_key_tiles(None, 3, 0, 2, 6, tiles, 4, ctypes.byref(n)) == -1
    assert lib.lvx_selftest_key_tiles(win, 3, 0, 2, 6, None, 4, ctypes.byref(n)) == -1
    for args in ((-1, 0, 2, 6), (3, 2, 1, 6), (3, 0, 2, -1), (3, 0, 2, 21), (FAR, 0, 2, 6)):
        assert lib.lvx_selftest_key_tiles(win, *args, tiles, 4, ctypes.byref(n)) == -2
