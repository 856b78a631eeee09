"""Attention within a window in the forms that large batches take, on shapes that are asserted to take them:
single tokens over 8-bit pages with 4 waves a workgroup, and the splits of a call without a window."""

import ctypes

import pytest
import torch

from paged_helpers import check_close, dev
from window_helpers import WindowBatch

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def plan(wb, max_q, max_kv):
    out = (ctypes.c_int64 * 3)()
    sizes = (sum(wb.new), wb.H, wb.Hkv, wb.D, len(wb.new), max_q, max_kv, wb.window, wb.sinks)
    assert N.lib().btl_paged_attention_window_plan(*sizes, out) == 1
    return tuple(out)


def run(wb, max_q, max_kv):
    out = torch.full((sum(wb.new), wb.H, wb.D), 7.0, dtype=torch.bfloat16, device=dev())
    got = pa.paged_attention(wb.q_dev, wb.cache, wb.table, wb.cu, wb.len, max_q=max_q, max_kv=max_kv, out=out,
                             window=wb.window, sinks=wb.sinks)
    pa.check("cuda:0")
    check_close(got, *wb.reference())


def ragged(B, most):
    """Lengths up to ``most``, with an empty slot, one of one position and one of a page's end."""
    n = [1 + (most * (17 * i % B)) // B for i in range(B)]
    n[0], n[B // 3], n[B // 2], n[B - 1] = most, 0, 1, 64
    return n


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("H,Hkv,D", [(20, 5, 128), (5, 5, 64), (10, 5, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 70), (300, 4)])
def test_more_contexts_than_compute_units(kv, page, H, Hkv, D, window, sinks):
    """Over 8-bit pages the kernel of 4 waves: a workgroup alone on its context."""
    total = ragged(60, 500)
    wb = WindowBatch([1] * 60, total, H, Hkv, D, page, kv, window, sinks)
    few, splits, _ = plan(wb, 1, 500)
    assert few == 1 and splits == 1 and 60 * Hkv > cus()
    run(wb, 1, 500)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("H,Hkv,D", [(16, 8, 64), (8, 8, 128)])
@pytest.mark.parametrize("page,window,sinks", [(16, 2700, 4), (64, 2600, 300), (80, 3000, 0)])
def test_long_windows_of_many_contexts(kv, H, Hkv, D, page, window, sinks):
    """More than half as many contexts as compute units: the splits of a call without a window."""
    total = [3300, 2900, 2750, 64, 1, 0] + [20 + 31 * i for i in range(14)]
    wb = WindowBatch([1] * 20, total, H, Hkv, D, page, kv, window, sinks)
    few, splits, _ = plan(wb, 1, 3300)
    assert few == 1 and splits == 4 and cus() < 2 * 20 * Hkv <= 2 * cus()
    run(wb, 1, 3300)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_more_rows_than_the_hint_in_many_contexts(kv):
    """The kernel of few rows in several passes: 3 to 9 rows of 4 heads each."""
    new = [3 + i % 7 for i in range(60)]
    total = [max(n, m) if m else 0 for n, m in zip(new, ragged(60, 400))]
    wb = WindowBatch(new, total, 20, 5, 64, 32, kv, 90, 5)
    few, splits, _ = plan(wb, 1, 400)
    assert few == 1 and splits == 1
    run(wb, 1, 400)
