"""How a decode step's key tiles are dealt to warps, and found again by the joining kernel, against whole-number arithmetic without
a limit: calls of more than 2^32 tiles are within the documented sizes (4096 entries that name one row of 2^21 keys, 8 kv heads)."""
import ctypes as C
import random

import pytest

from runtherder_b200 import _lib


def line(tiles, warps, tile):
    w, first = C.c_longlong(), C.c_longlong()
    assert _lib.lib.rh_selfcheck_decode_line(tiles, warps, tile, C.byref(w), C.byref(first)) == 0
    return w.value, first.value


def check(tiles, warps, tile):
    w, first = line(tiles, warps, tile)
    # the last warp whose share starts at or in front of the tile
    assert first == tiles * w // warps
    assert first <= tile < tiles * (w + 1) // warps, (tiles, warps, tile, w)


@pytest.mark.parametrize("tiles", [1 << 32, (1 << 32) + 8, (1 << 32) - 1, (1 << 33) + 3, 4097 * (1 << 20), 1 << 41])
def test_more_tiles_than_32_bits_count(tiles):
    for warps in (1, 7, 2368, 2367):
        for tile in (0, 1, (1 << 17), tiles // 4096, tiles // 4096 + 1, (1 << 32) // warps, tiles // 2, tiles - 1):
            check(tiles, warps, min(tile, tiles - 1))


def test_any_line():
    rng = random.Random(1)
    for _ in range(3000):
        tiles = int(2.0 ** rng.uniform(0, 41))
        check(tiles, rng.randint(1, min(tiles, 4000)), rng.randrange(tiles))
    for tiles in range(1, 60):
        for warps in range(1, tiles + 1):
            for tile in range(tiles):
                check(tiles, warps, tile)


def test_refusals():
    f, w = _lib.lib.rh_selfcheck_decode_line, C.c_longlong()
    for bad in ((0, 1, 0), (5, 0, 0), (5, 1, 5), (5, 1, -1), ((1 << 42) + 1, 1, 0), (5, (1 << 16) + 1, 0)):
        assert f(*bad, C.byref(w), C.byref(w)) == 1
    assert f(5, 1, 0, None, C.byref(w)) == 1
