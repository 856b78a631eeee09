"""Attention within a window without a GPU: argument checks of the C entry points and of the
Python layer, and the plan of a window."""

import ctypes

import pytest
import torch

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa


@pytest.fixture(scope="module")
def L():
    return N.lib()


FAKE = 1 << 20  # never followed: every call here is refused before a launch
NULL, SHAPE, ALIGN, WORKSPACE, ARG = 1, 2, 3, 4, 5


def pages(**kw):
    d = dict(k=FAKE, v=FAKE, k_exp=None, v_exp=None, num_pages=8, num_kv_heads=2, page_size=16, head_dim=64)
    d.update(kw)
    return N.Pages(*d.values())


def prompt(L, **kw):
    a = dict(q=FAKE, ldq=256, k=FAKE, ldk=128, v=FAKE, ldv=128, T=4, H=4, Hkv=2, D=64, cu=FAKE, B=2, scale=0.125, max_q=4,
             window=2, sinks=1, out=FAKE, ldo=256, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_prompt_attention_window(*a.values())


def paged(L, **kw):
    a = dict(q=FAKE, ldq=256, T=4, H=4, pages=pages(), table=FAKE, max_pages=2, cu=FAKE, kv=FAKE, B=2, scale=0.125,
             max_q=4, max_kv=32, window=2, sinks=1, out=FAKE, ldo=256, scratch=None, nbytes=0, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_paged_attention_window(*a.values())


@pytest.mark.parametrize("want,kw", [
    (ARG, dict(window=0)), (ARG, dict(window=-3)), (ARG, dict(sinks=-1)), (ARG, dict(scale=0.0)), (SHAPE, dict(D=80)),
    (SHAPE, dict(H=5)), (SHAPE, dict(ldk=64)), (ALIGN, dict(q=FAKE + 8)), (NULL, dict(k=None)), (NULL, dict(out=None)),
    (SHAPE, dict(max_q=-1)), (SHAPE, dict(B=0)),
])
def test_prompts_refuse(L, want, kw):
    assert prompt(L, **kw) == want
    assert b"btl_prompt_attention_window" in L.btl_last_error()


@pytest.mark.parametrize("want,kw", [
    (ARG, dict(window=0)), (ARG, dict(sinks=-2 ** 60)), (NULL, dict(pages=None)), (NULL, dict(table=None)), (NULL, dict(kv=None)),
    (SHAPE, dict(max_q=0)), (SHAPE, dict(max_kv=0)), (SHAPE, dict(max_pages=0)), (ALIGN, dict(out=FAKE + 2)),
    (WORKSPACE, dict(max_pages=512, max_kv=8192, window=5000)),
    (WORKSPACE, dict(max_pages=512, max_kv=8192, window=5000, scratch=FAKE, nbytes=64)),
    (SHAPE, dict(B=70000, T=70000, max_q=1)),
])
def test_paged_refuses(L, want, kw):
    assert paged(L, **kw) == want
    assert b"btl_paged_attention_window" in L.btl_last_error()


def test_no_rows_is_no_launch(L):
    assert prompt(L, T=0) == 0 and paged(L, T=0) == 0


def plan(L, *sizes):
    out = (ctypes.c_int64 * 3)()
    assert L.btl_paged_attention_window_plan(*sizes, out) == 1
    return tuple(out)


@pytest.mark.parametrize("T,B,max_q", [(1, 1, 1), (32, 32, 1), (67, 1, 67), (2047, 4, 700), (3, 1, 2 ** 62)])
@pytest.mark.parametrize("D", [64, 128])
def test_plan_of_any_window(L, T, B, max_q, D):
    """A split's positions are 32-bit numbers, whatever the hints and the window; the scratch is that of the plan."""
    for max_kv in (1, 1024, 40067, 2 ** 31, 2 ** 62):
        for window in (1, 100, 1024, 9000, 2 ** 31, 2 ** 63 - 1):
            for sinks in (0, 4, 700, 2 ** 31, 2 ** 63 - 1):
                sizes = (T, 20, 5, D, B, max_q, max_kv, window, sinks)
                few, splits, chunk = plan(L, *sizes)
                assert 1 <= splits <= 256 and 128 <= chunk <= 2 ** 30 and chunk % 64 == 0 and splits * chunk < 2 ** 31
                assert splits * chunk >= min(max_kv, window, 2 ** 30 - 1)
                assert L.btl_paged_attention_window_scratch_bytes(*sizes) == (
                    splits * T * 20 * (D + 2) * 4 if splits > 1 else 0)
                assert few == (min(max_q, T) * 4 <= 16)


def test_a_long_context_is_split_by_its_window(L):
    far = plan(L, 1, 20, 5, 128, 1, 1, 131072, 4096, 4)
    near = plan(L, 1, 20, 5, 128, 1, 1, 4096 + 300, 4096, 4)
    assert far == near and far[1] > 1


@pytest.mark.parametrize("sizes", [
    (1, 20, 5, 128, 1, 1, 4096, 0, 0), (1, 20, 5, 128, 1, 1, 4096, -1, 0), (1, 20, 5, 128, 1, 1, 4096, 10, -1),
    (1, 20, 5, 96, 1, 1, 4096, 10, 0), (0, 20, 5, 128, 1, 1, 4096, 10, 0), (1, 20, 5, 128, 1, 1, 0, 10, 0),
])
def test_scratch_of_what_no_call_takes(L, sizes):
    assert L.btl_paged_attention_window_scratch_bytes(*sizes) == 0
    assert L.btl_paged_attention_window_plan(*sizes, (ctypes.c_int64 * 3)()) == 0


def test_python_refuses():
    x = torch.zeros((4, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm GPU"):
        pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], torch.zeros(2, dtype=torch.int32), window=4)
    assert pa.check_window(None, 0) == (None, 0) and pa.check_window(7, 2) == (7, 2)
    assert pa.check_window(2 ** 63, 2 ** 70) == (2 ** 30, 2 ** 30)
    for bad in ((None, 3), (0, 0), (-1, 0), (5, -1)):
        with pytest.raises(ValueError):
            pa.check_window(*bad)
    for bad in ((4.5, 0), (4, 1.0), ("4", 0)):  # no whole numbers
        with pytest.raises(TypeError):
            pa.check_window(*bad)
