"""Attention of a batch that shares its first pages without a GPU: argument checks and the plan."""

import ctypes

import pytest

from bitnet_tt import _native as N


@pytest.fixture(scope="module")
def L():
    return N.lib()


FAKE = 1 << 20  # never followed: every call here is refused before a launch
NULL, SHAPE, ALIGN, WORKSPACE, ARG = 1, 2, 3, 4, 5


def pages(**kw):
    d = dict(k=FAKE, v=FAKE, k_exp=None, v_exp=None, num_pages=8, num_kv_heads=2, page_size=16, head_dim=64)
    d.update(kw)
    return N.Pages(*d.values())


def shared(L, **kw):
    a = dict(q=FAKE, ldq=256, T=4, H=4, pages=pages(), table=FAKE, max_pages=2, cu=FAKE, kv=FAKE, shared=FAKE, B=2, scale=0.125,
             max_q=4, max_kv=32, max_shared=16, out=FAKE, ldo=256, scratch=FAKE, nbytes=1 << 30, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_shared_prefix_attention(*a.values())


@pytest.mark.parametrize("want,kw", [
    (NULL, dict(pages=None)), (NULL, dict(table=None)), (NULL, dict(kv=None)), (NULL, dict(err=None)), (NULL, dict(shared=None)),
    (NULL, dict(q=None)), (NULL, dict(cu=None)), (NULL, dict(out=None)),
    (SHAPE, dict(H=5)), (SHAPE, dict(max_q=0)), (SHAPE, dict(max_kv=0)), (SHAPE, dict(max_pages=0)), (SHAPE, dict(max_shared=-1)),
    (SHAPE, dict(B=0)), (SHAPE, dict(T=-1)), (SHAPE, dict(pages=pages(head_dim=96))), (SHAPE, dict(ldo=128)),
    (SHAPE, dict(max_pages=1 << 24, pages=pages(page_size=1 << 20))), (ARG, dict(scale=0.0)), (ALIGN, dict(out=FAKE + 2)),
    (ALIGN, dict(shared=FAKE + 2)), (ALIGN, dict(scratch=FAKE + 4)), (WORKSPACE, dict(scratch=None)),
    (WORKSPACE, dict(nbytes=64)),
])
def test_refuses(L, want, kw):
    assert shared(L, **kw) == want
    assert b"btl_shared_prefix_attention" in L.btl_last_error()


def test_no_rows_is_no_launch(L):
    assert shared(L, T=0) == 0


def plan(L, *sizes):
    out = (ctypes.c_int64 * 6)()
    assert L.btl_shared_prefix_attention_plan(*sizes, out) == 1
    return tuple(out)


@pytest.mark.parametrize("T,B,max_q", [(1, 1, 1), (32, 32, 1), (67, 1, 67), (2047, 4, 700), (3, 1, 2 ** 62), (64, 64, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_plan_of_any_hint(L, T, B, max_q, D):
    """Positions are 32-bit numbers: the end of the last split of a sequence's own positions stays below 2^31 behind
    any prefix that a table has room for; the scratch has a partial of every split of both parts."""
    for max_kv in (1, 1024, 40067, 2 ** 30, 2 ** 31, 2 ** 62, 2 ** 63 - 1):
        for max_shared in (0, 16, 1000, 65536, 2 ** 30, 2 ** 31, 2 ** 63 - 1):
            sizes = (T, 20, 5, D, B, max_q, max_kv, max_shared)
            few, n, chunk, own_few, own_n, own_chunk = plan(L, *sizes)
            assert 1 <= n <= 256 and 64 <= chunk and n * chunk < 2 ** 31
            assert 1 <= own_n <= 256 and 256 <= own_chunk and 2 ** 30 + own_n * own_chunk < 2 ** 31
            assert n * chunk >= min(max_shared, 2 ** 30 - 1)
            assert own_few == (min(max_q, T) * 4 <= 16) and few == (T * 4 <= 16 and own_few)
            assert L.btl_shared_prefix_attention_scratch_bytes(*sizes) == (n + own_n) * T * 20 * (D + 2) * 4


@pytest.mark.parametrize("sizes", [
    (0, 20, 5, 128, 1, 1, 4096, 16), (1, 20, 3, 128, 1, 1, 4096, 16), (1, 20, 5, 96, 1, 1, 4096, 16), (1, 20, 5, 128, 0, 1, 4096, 16),
    (1, 20, 5, 128, 1, 0, 4096, 16), (1, 20, 5, 128, 1, 1, 0, 16), (1, 20, 5, 128, 1, 1, 4096, -1), (1 << 62, 20, 5, 128, 1, 1, 1, 1),
])
def test_scratch_of_what_no_call_takes(L, sizes):
    assert L.btl_shared_prefix_attention_scratch_bytes(*sizes) == 0
    assert L.btl_shared_prefix_attention_plan(*sizes, (ctypes.c_int64 * 6)()) == 0
