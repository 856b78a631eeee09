"""Attention within a window with sinks on the GPU against 64 bits: packed prompts, and
chunks and single tokens over pages."""

import math

import pytest
import torch

from paged_helpers import check_close, cu_of, dev, ints, normal
from window_helpers import WindowBatch, attend_window64

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


# ---- prompts --------------------------------------------------------------


def prompt_case(lens, H, Hkv, D, window, sinks, seed=1, spare=0, change=None, **kw):
    T = sum(lens) + spare
    x = normal((T, H + 2 * Hkv, D), seed, 1.4).to(torch.bfloat16)
    if change is not None:
        change(x[:, H:H + Hkv], x[:, H + Hkv:])
    d = x.to(dev())
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=dev())
    got = pa.prompt_attention(d[:, :H], d[:, H:H + Hkv], d[:, H + Hkv:], cu_of(lens), out=out, window=window,
                              sinks=sinks, **kw)
    at = 0
    for n in lens:
        y = x[at:at + n].double()
        want, tol = attend_window64(y[:, :H], y[:, H:H + Hkv].transpose(0, 1), y[:, H + Hkv:].transpose(0, 1), window,
                                    sinks, kw.get("scale"))
        check_close(got[at:at + n], want, tol)
        at += n
    assert bool((got[at:] == 7.0).all())


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (63, 0), (64, 4), (65, 64), (130, 70), (200, 1), (7, 400)])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (3, 3, 128), (8, 1, 64)])
def test_prompts(H, Hkv, D, window, sinks):
    prompt_case([1, 70, 0, 129, 311], H, Hkv, D, window, sinks, spare=3)


@pytest.mark.parametrize("window,sinks", [(1, 2), (100, 4), (256, 0)])
def test_prompts_of_the_large_heads(window, sinks):
    prompt_case([200, 33, 402], 20, 5, 128, window, sinks)


@pytest.mark.parametrize("window,sinks", [(600, 4), (700, 200), (1000, 0)])
def test_long_prompts_have_whole_steps(window, sinks):
    """Rows of one head: 128 tokens a tile, a window of many steps that every row of the tile sees, of either parity."""
    prompt_case([1411], 1, 1, 64, window, sinks, seed=3)
    prompt_case([1347], 2, 1, 128, window, sinks, seed=4)


@pytest.mark.parametrize("window", [300, 301, 5000])
def test_a_window_as_long_as_the_batch_is_none(window):
    x = normal((300, 8, 64), 3).to(torch.bfloat16).to(dev())
    args = (x[:, :4], x[:, 4:6], x[:, 6:], cu_of([120, 180]))
    assert torch.equal(pa.prompt_attention(*args, window=window, sinks=3), pa.prompt_attention(*args))


def test_a_window_of_the_longest_sequence():
    """Shorter than the batch, no shorter than any sequence: the windowed kernel, every position seen."""
    prompt_case([90, 150], 4, 2, 64, 150, 2)


def test_values_that_are_not_finite():
    """They reach the rows that see them, and no other; neither do keys."""

    def change(k, v):
        v[20, 0, 3] = math.inf
        v[21, 1, 5] = math.nan
        v[2, 0, 7] = -math.inf  # in the sinks
        k[100, 0, 0] = math.nan
        v[150, 1, 60] = -math.inf

    prompt_case([260], 4, 2, 64, 70, 4, change=change)
    prompt_case([260], 4, 2, 64, 33, 0, change=change)
    prompt_case([260], 2, 2, 128, 129, 64, change=change)


# ---- over pages ---------------------------------------------------------


def paged_case(wb, max_q=None, max_kv=None, scale=None):
    out = torch.full((sum(wb.new), wb.H, wb.D), 7.0, dtype=torch.bfloat16, device=dev())
    got = pa.paged_attention(wb.q_dev, wb.cache, wb.table, wb.cu, wb.len, scale=scale, max_q=max_q, max_kv=max_kv, out=out,
                             window=wb.window, sinks=wb.sinks)
    pa.check("cuda:0")
    check_close(got, *wb.reference(scale))
    return got


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (20, 4), (64, 0), (100, 70), (250, 33), (33, 500)])
def test_single_tokens(kv, page, window, sinks):
    total = [1, 2, 17, 64, 65, 300, 511, 0, 800]
    wb = WindowBatch([1] * len(total), total, 4, 2, 64, page, kv, window, sinks)
    paged_case(wb, max_q=1)
    paged_case(wb)  # the tiles' kernel


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 64, 80])
@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 4), (129, 66), (400, 0)])
@pytest.mark.parametrize("H,Hkv,D", [(20, 5, 128), (3, 3, 64)])
def test_chunks(kv, page, window, sinks, H, Hkv, D):
    wb = WindowBatch([70, 1, 0, 33, 5], [470, 300, 12, 33, 2], H, Hkv, D, page, kv, window, sinks)
    paged_case(wb, max_q=70)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("new,H,Hkv,D", [([1], 20, 5, 128), ([1, 1], 4, 2, 64), ([40], 4, 2, 64), ([3, 2], 8, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(1500, 4), (2600, 300)])
def test_windows_that_are_split(kv, new, H, Hkv, D, window, sinks):
    """Few rows and a long window: several workgroups a context, tiles of unlike length."""
    total = [5000, 777][: len(new)]
    wb = WindowBatch(new, total, H, Hkv, D, 64, kv, window, sinks)
    paged_case(wb, max_q=max(new))
    paged_case(wb, max_q=max(new), max_kv=1024)  # hints below what is there
    wb = WindowBatch(new, total, H, Hkv, D, 16, kv, window, sinks)
    paged_case(wb, max_q=max(new), max_kv=5000)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 64, 80])
@pytest.mark.parametrize("new,total", [([40, 1, 30, 2, 0], [4000, 1, 90, 0, 60]), ([1, 1, 1, 1], [4000, 1, 0, 700])])
@pytest.mark.parametrize("window,sinks", [(1500, 4), (700, 500), (2000, 0)])
def test_windows_that_are_split_beside_short_contexts(kv, page, new, total, window, sinks):
    """Splits that end inside the sinks, in the gap and in the windows; contexts that one workgroup has alone, and none."""
    wb = WindowBatch(new, total, 4, 2, 64, page, kv, window, sinks)
    paged_case(wb, max_q=max(new), max_kv=max(total))
    sizes = (sum(new), 4, 2, 64, len(new), max(new), max(total), window, sinks)
    assert N.lib().btl_paged_attention_window_scratch_bytes(*sizes) > 0  # they are split


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("new", [[1, 1], [40, 9]])
def test_splits_with_values_that_are_not_finite(kv, new):
    """Seen by some of the rows of a split only, in sinks, at the windows' beginnings and at their ends."""
    total, window, sinks = [3000, 1700], 1400, 70
    wb = WindowBatch(new, total, 4, 2, 64, 16, kv, window, sinks, release=False)
    first = total[0] - window  # the last row's first position
    for position in (3, first - 20, first + 1, 2400, 2999):
        page, row = int(wb.full_table[0][position // 16]), position % 16
        if kv == "fp8":
            wb.cache.value_pages.view(torch.uint8)[page, 1, row, position % 64] = 0x7F
            wb.v64[page, 1, row, position % 64] = math.nan
        else:
            wb.cache.value_pages[page, 1, row, position % 64] = math.inf
            wb.v64[page, 1, row, position % 64] = math.inf
    paged_case(wb, max_q=max(new))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_more_rows_than_the_hint(kv):
    """The kernel of few rows in several passes, each with its own window."""
    wb = WindowBatch([30, 9], [900, 400], 4, 2, 64, 16, kv, 100, 20)
    paged_case(wb, max_q=1, max_kv=100)
    wb = WindowBatch([30, 9], [2900, 400], 4, 2, 64, 32, kv, 1400, 20)
    paged_case(wb, max_q=1)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("max_q", [1, 40])
def test_a_window_as_long_as_the_table_is_none(kv, max_q):
    wb = WindowBatch([1, 1], [200, 90], 4, 2, 64, 16, kv, 10 ** 12, 3)
    args = (wb.q_dev, wb.cache, wb.table, wb.cu, wb.len)
    a = pa.paged_attention(*args, max_q=max_q, window=10 ** 12, sinks=10 ** 12)
    assert torch.equal(a, pa.paged_attention(*args, max_q=max_q))


@pytest.mark.parametrize("max_q", [1, 40])
def test_a_page_that_is_seen_and_is_none(max_q):
    """The pages of the window and of the sinks are looked up: an entry outside the pool is an error."""
    for position, window, sinks in ((799, 100, 0), (701, 100, 0), (3, 100, 4)):
        wb = WindowBatch([1], [800], 4, 2, 64, 16, "bf16", window, sinks)
        wb.table[0, position // 16] = 2 ** 30
        pa.paged_attention(wb.q_dev, wb.cache, wb.table, wb.cu, wb.len, max_q=max_q, window=window, sinks=sinks)
        with pytest.raises(RuntimeError, match="paged workspace"):
            pa.check("cuda:0")


@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pages_with_values_that_are_not_finite(kv, max_q):
    """In the pages of the window and of the sinks, before the one and behind the others."""
    wb = WindowBatch([2], [400], 4, 2, 64, 64, kv, 100, 4, std=1.0)
    for pool, pool64 in ((wb.cache.key_pages, wb.k64), (wb.cache.value_pages, wb.v64)):
        for position in (10, 290, 298):  # rows see 299 .. 399 and 0 .. 3
            page, row = int(wb.full_table[0, position // 64]), position % 64
            if kv == "fp8":
                pool.view(torch.uint8)[page, :, row] = 0x7F
            else:
                pool[page, :, row] = math.inf
            pool64[page, :, row] = math.nan
    paged_case(wb, max_q=max_q)


def test_captured_and_on_another_stream():
    """Lengths that move on between replays: the window moves with them."""
    wb = WindowBatch([1, 1], [3000, 40], 4, 2, 64, 64, "bf16", 700, 4, release=False, extra_pages=2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    lens = wb.len.clone()

    def call():
        return pa.paged_attention(wb.q_dev, wb.cache, wb.table, wb.cu, lens, max_q=1, max_kv=3000, window=700, sinks=4)

    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    for total in ([3000, 40], [2999, 39], [900, 1], [2, 0]):
        lens.copy_(ints(total))
        out.fill_(9.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        eager = call()
        assert torch.equal(out, eager)
        wb.total = total
        check_close(out, *wb.reference())


def test_scales_and_strided_rows():
    x = torch.full((37, 10, 64), 7.0, dtype=torch.bfloat16, device=dev())
    wb = WindowBatch([30, 7], [230, 7], 4, 2, 64, 32, "bf16", 50, 5)
    q = torch.zeros((37, 12, 64), dtype=torch.bfloat16, device=dev())[:, 3:7]
    q.copy_(wb.q_dev)
    pa.paged_attention(q, wb.cache, wb.table, wb.cu, wb.len, scale=0.3, out=x[:, 2:6], window=50, sinks=5)
    check_close(x[:, 2:6], *wb.reference(0.3))
    assert bool((x[:, :2] == 7.0).all()) and bool((x[:, 6:] == 7.0).all())
    prompt_case([150], 4, 2, 64, 40, 3, scale=0.4)
