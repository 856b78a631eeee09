"""Attention of a batch that shares its first pages on the GPU against 64 bits."""

import math

import pytest
import torch

from paged_helpers import check_close, dev, ints, normal
from window_helpers import SharedBatch

from bitnet_tt import paged_attention as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


def expect_error():
    with pytest.raises(RuntimeError, match="paged workspace"):
        pa.check("cuda:0")


def call(sb, **kw):
    return pa.shared_prefix_attention(sb.q_dev, sb.cache, sb.table, sb.cu, sb.len, sb.pages, **kw)


def case(sb, scale=None, **kw):
    out = torch.full((sum(sb.new), sb.H, sb.D), 7.0, dtype=torch.bfloat16, device=dev())
    got = call(sb, scale=scale, out=out, **kw)
    pa.check("cuda:0")
    check_close(got, *sb.reference(scale))
    return got


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page,shared", [(16, 1), (16, 9), (48, 5), (64, 4), (256, 1)])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (20, 5, 128), (3, 3, 128)])
def test_single_tokens(kv, page, shared, H, Hkv, D):
    """Few rows in all, a tile of rows, and more than one; lengths that end anywhere in a page."""
    for own in ([1], [5, 1, 100], [1 + (37 * i) % 150 for i in range(35)]):
        sb = SharedBatch([1] * len(own), own, shared, H, Hkv, D, page, kv)
        case(sb, max_q=1)
    case(sb)  # the tiles' kernel for the sequences too


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 64, 80])
@pytest.mark.parametrize("new,own", [([3, 1, 0, 5], [40, 1, 12, 5]), ([70, 129, 1], [170, 129, 300])])
@pytest.mark.parametrize("H,Hkv,D", [(20, 5, 128), (8, 1, 64)])
def test_drafts_and_chunks(kv, page, new, own, H, Hkv, D):
    sb = SharedBatch(new, own, 3, H, Hkv, D, page, kv)
    case(sb, max_q=max(new))
    case(sb, max_q=1)  # a hint below what is there


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("new", [[1], [1, 1, 1], [1] * 12, [9, 4]])
def test_long_prefixes_and_contexts_are_split(kv, new):
    own = [1500 + 331 * i if i < 2 else 20 + i for i in range(len(new))]
    sb = SharedBatch(new, own, 40, 4, 2, 64, 64, kv)
    case(sb, max_q=max(new), max_kv=max(sb.total), max_shared=40)
    case(sb, max_q=max(new), max_kv=2700, max_shared=3)  # hints below what is there
    case(sb)
    sb = SharedBatch(new, own, 70, 20, 5, 128, 16, kv)
    case(sb, max_q=max(new))


def test_nothing_is_shared():
    sb = SharedBatch([1, 3], [40, 17], 0, 4, 2, 64, 16, "bf16")
    case(sb, max_q=3)
    sb = SharedBatch([1, 3], [40, 17], 0, 4, 2, 64, 16, "bf16")
    case(sb, max_q=1, max_shared=0)


@pytest.mark.parametrize("max_q", [1, None])
def test_empty_slots(max_q):
    """Slots of a captured batch that hold no user: rows with a negative position give zeros, whatever is shared."""
    sb = SharedBatch([1, 1, 1, 2], [7, 0, 30, 0], 6, 4, 2, 64, 16, "bf16")
    got = case(sb, max_q=max_q)
    assert bool((got[1] == 0).all()) and bool((got[3:] == 0).all())


@pytest.mark.parametrize("max_q", [1, None])
def test_the_first_slot_is_empty(max_q):
    """Its table still names the shared pages; its user is gone."""
    sb = SharedBatch([2, 1, 1], [0, 9, 40], 6, 4, 2, 64, 16, "fp8")
    got = case(sb, max_q=max_q)
    assert bool((got[:2] == 0).all())


def test_rows_of_no_sequence_stay():
    sb = SharedBatch([2, 5], [7, 30], 6, 4, 2, 64, 16, "bf16")
    q = torch.zeros((12, 4, 64), dtype=torch.bfloat16, device=dev())
    q[3:10] = sb.q_dev
    out = torch.full_like(q, 7.0)
    cu = sb.cu + 3
    for max_q in (1, 5):
        pa.shared_prefix_attention(q, sb.cache, sb.table, cu, sb.len, sb.pages, max_q=max_q, out=out)
        check_close(out[3:10], *sb.reference())
        assert bool((out[:3] == 7.0).all()) and bool((out[10:] == 7.0).all())


def test_groups_as_slices():
    """A call for each group of users, on parts of the batch's arrays."""
    a = SharedBatch([1, 1], [7, 30], 3, 4, 2, 64, 16, "bf16", seed=1)
    cu = ints([0, 1, 2, 3, 4])
    q = torch.cat((a.q_dev, a.q_dev))
    out = torch.full_like(q, 7.0)
    for g in (0, 1):
        pa.shared_prefix_attention(q, a.cache, a.table, cu[2 * g:2 * g + 3], a.len, a.pages, max_q=1, out=out)
    want, tol = a.reference()
    check_close(out[:2], want, tol)
    check_close(out[2:], want, tol)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("max_q", [1, None])
def test_values_that_are_not_finite(kv, max_q):
    """One in the prefix reaches every row, one in a sequence's own pages the rows that see it."""
    sb = SharedBatch([1, 2, 2], [20, 31, 2], 5, 4, 2, 64, 16, kv)
    for b, position in ((0, 33), (1, 5 * 16 + 30)):
        page, row = int(sb.full_tables[b][position // 16]), position % 16
        for pool, pool64 in ((sb.cache.value_pages, sb.v64),):
            if kv == "fp8":
                pool.view(torch.uint8)[page, 1, row, 7] = 0x7F
                pool64[page, 1, row, 7] = math.nan
            else:
                pool[page, 1, row, 7] = math.inf
                pool64[page, 1, row, 7] = math.inf
    case(sb, max_q=max_q)


@pytest.mark.parametrize("max_q", [1, None])
@pytest.mark.parametrize("change", ["pages", "many", "before", "outside"])
def test_batches_that_are_not_well_formed(max_q, change):
    sb = SharedBatch([1, 1], [7, 30], 4, 4, 2, 64, 16, "bf16")
    if change == "pages":
        sb.pages.fill_(-1)
    elif change == "many":
        sb.pages.fill_(sb.table.shape[1] + 1)
    elif change == "before":
        sb.len[1] = 4 * 16  # its row's position is the last shared one
    else:
        sb.table[0, 2] = 10 ** 6
    call(sb, max_q=max_q)
    expect_error()


def test_captured_and_two_at_once():
    """Lengths and the number of shared pages move on between replays, on two streams with a scratch each."""
    runs = []
    for seed in (1, 2):
        sb = SharedBatch([1] * 5, [300, 20, 5, 77, 64], 9, 4, 2, 64, 64, "bf16", seed=seed)  # no length below is longer
        for b in range(1, 5):  # whole tables: any number of the pages may be shared
            sb.table[b, :9] = sb.table[0, :9]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call(sb, max_q=1)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = call(sb, max_q=1)
        runs.append((sb, stream, graph, out))
    for shared, own in ((9, [300, 20, 1, 77, 64]), (3, [299, 19, 1, 70, 60]), (0, [5, 5, 5, 5, 5]), (9, [1, 1, 1, 1, 1])):
        for sb, _, _, out in runs:
            sb.pages.fill_(shared)
            sb.total = [9 * 64 + n for n in own]
            sb.len.copy_(ints(sb.total))
            out.fill_(9.0)
        torch.cuda.synchronize()
        for _, stream, graph, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for sb, _, _, out in runs:
            assert torch.equal(out, call(sb, max_q=1))
            check_close(out, *sb.reference())


def test_strided_rows_and_scales():
    sb = SharedBatch([3, 7], [30, 7], 2, 4, 2, 64, 32, "bf16")
    q = torch.zeros((10, 12, 64), dtype=torch.bfloat16, device=dev())[:, 3:7]
    q.copy_(sb.q_dev)
    x = torch.full((10, 10, 64), 7.0, dtype=torch.bfloat16, device=dev())
    pa.shared_prefix_attention(q, sb.cache, sb.table, sb.cu, sb.len, sb.pages, scale=0.3, out=x[:, 2:6])
    check_close(x[:, 2:6], *sb.reference(0.3))
    assert bool((x[:, :2] == 7.0).all()) and bool((x[:, 6:] == 7.0).all())
    assert pa.shared_prefix_attention(q[:0], sb.cache, sb.table, sb.cu, sb.len, sb.pages).shape == (0, 4, 64)


def test_the_same_as_attention_over_the_pages():
    """Within the two calls' bounds: a different order of the same sums."""
    sb = SharedBatch([1] * 3, [30, 7, 100], 6, 20, 5, 128, 64, "bf16")
    sb.table[:, :6] = sb.table[0, :6]
    a = call(sb, max_q=1).double()
    b = pa.paged_attention(sb.q_dev, sb.cache, sb.table, sb.cu, sb.len, max_q=1).double()
    _, tol = sb.reference()
    assert bool(((a - b).abs().cpu() <= 2 * tol).all())


def test_host_arrays_are_refused():
    sb = SharedBatch([1], [7], 1, 4, 2, 64, 16, "bf16")
    with pytest.raises(ValueError, match="shared_pages"):
        pa.shared_prefix_attention(sb.q_dev, sb.cache, sb.table, sb.cu, sb.len, sb.pages.cpu())
    with pytest.raises(ValueError, match="shared_pages"):
        pa.shared_prefix_attention(sb.q_dev, sb.cache, sb.table, sb.cu, sb.len, ints([1, 1]))
    with pytest.raises(ValueError, match="max_shared"):
        call(sb, max_shared=-1)
    x = normal((1, 3, 64), 1).to(torch.bfloat16).to(dev())
    with pytest.raises(ValueError, match="query heads"):
        pa.shared_prefix_attention(x, sb.cache, sb.table, sb.cu, sb.len, sb.pages)
