"""Which workgroup works on which tile of a windowed call: every tile of every head once."""

import ctypes

import pytest

from bitnet_tt import _native as N


@pytest.fixture(scope="module")
def L():
    return N.lib()


def at(L, tiles, splits, Hkv, x):
    out = (ctypes.c_int64 * 3)()
    return L.btl_attention_window_tile(tiles, splits, Hkv, x, out), tuple(out)


@pytest.mark.parametrize("least", [0, 320, 640, 1280])
@pytest.mark.parametrize("Hkv", [1, 2, 3, 5, 8, 40])
@pytest.mark.parametrize("more", [0, 1, 2, 3, 7, 9, 30])
def test_every_tile_once(L, least, Hkv, more):
    n = -(-least // Hkv) + more + (least == 0)  # of a head
    neighbours = 8 if n * Hkv >= 1280 else 4 if n * Hkv >= 640 else 2 if n * Hkv >= 320 else 1  # on 256 CUs
    groups, (each, _, _) = at(L, n * Hkv, 1, Hkv, 0)
    assert each == neighbours
    seen = set()
    for x in range(groups):
        same, (_, head, tile) = at(L, n * Hkv, 1, Hkv, x)
        assert same == groups and 0 <= head and head < Hkv and tile >= 0 and (head, tile) not in seen
        seen.add((head, tile))
    # those behind the last are found to be none
    assert {(h, t) for h in range(Hkv) for t in range(n)} <= seen
    assert at(L, n * Hkv, 1, Hkv, groups)[0] == 0
    # neighbours: the same remainder by 8, one after the other
    where = {at(L, n * Hkv, 1, Hkv, x)[1][1:]: x for x in range(groups)}
    for h in range(Hkv):
        for t in range(n):
            if t % each:
                assert where[h, t] == where[h, t - 1] + 8


def test_splits_have_no_neighbours(L):
    assert at(L, 5000, 2, 5, 7)[1][0] == 1 and at(L, 5000, 1, 5, 7)[1][0] == 8


@pytest.mark.parametrize("bad", [(0, 1, 1, 0), (10, 1, 3, 0), (10, 0, 5, 0), (10, 1, 0, 0), (10, 1, 5, -1), (10, 1, 5, 1 << 40)])
def test_of_what_no_call_takes(L, bad):
    assert at(L, *bad)[0] == 0
