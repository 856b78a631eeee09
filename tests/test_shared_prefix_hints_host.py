"""The plan of attention behind a shared prefix where the caller gives no hint of its length."""

import pytest

from test_shared_prefix_host import plan

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa


def test_a_prefix_of_no_known_length_leaves_contexts_split():
    """4 users of 1024 shared and 16000 own positions: where max_shared is not given, their own positions are split too."""
    L = N.lib()
    table, longest = 2048 * 16, 1024 + 16000
    known = plan(L, 4, 20, 5, 128, 4, 1, longest, 1024)
    assert known[4] > 4
    for max_kv in (longest, table):
        shared = pa._shared_positions(None, 16, max_kv)
        assert shared == max_kv
        open_ = plan(L, 4, 20, 5, 128, 4, 1, max_kv, shared)
        assert open_[4] > 4 and open_[5] <= max_kv // 4
    # nor are a long prefix's splits those of the table
    assert plan(L, 32, 20, 5, 128, 32, 1, 8692, pa._shared_positions(None, 64, 8692))[2] <= 512


@pytest.mark.parametrize("pages_,page_size,max_kv,want", [
    (None, 16, 500, 500), (10, 16, 500, 160), (10, 64, 500, 500), (0, 16, 500, 0), (2 ** 40, 128, 2 ** 20, 2 ** 20)])
def test_the_hint_in_positions(pages_, page_size, max_kv, want):
    assert pa._shared_positions(pages_, page_size, max_kv) == want
