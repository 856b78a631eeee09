"""Prompts and the paged cache on the GPU where a call is allowed and rare:
shared pages, pools past 32-bit offsets, captured calls at once, entries of
cu_q that no row reads, rows in wide buffers."""

import math

import pytest
import torch

from paged_helpers import BF16_HALF, PagedBatch, attend64, check_close, cu_of, dev, ints, normal, quantise, values_of

from bitnet_tt import paged_attention as pa
from bitnet_tt.utils.rope import rope_tables

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


def expect_error():
    with pytest.raises(RuntimeError, match="paged workspace"):
        pa.check("cuda:0")


@pytest.mark.parametrize("B", [3, 65, 130])
@pytest.mark.parametrize("bad", [[1, 0], [2, 1], [1, -1]])
def test_a_last_sequence_that_ends_before_it_begins(B, bad):
    """One row, many empty sequences, and a last entry that is wrong: no row is in it."""
    cu = ints([0] + [bad[0]] * (B - 1) + [bad[1]])
    x = normal((1, 8, 64), 1).to(torch.bfloat16).to(dev())
    pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu)
    expect_error()
    cache = pa.PagedKVCache.allocate(2, 2, 64, dev(), page_size=16)
    table, lens = torch.zeros((B, 1), dtype=torch.int32, device=dev()), ints([1] + [0] * (B - 1))
    for max_q in (1, 40):
        pa.paged_attention(x[:, :4].contiguous(), cache, table, cu, lens, max_q=max_q)
        expect_error()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("max_q", [1, 40])
def test_sequences_that_share_pages(kv, max_q):
    """The same pages in every row of the table, lengths that end in different places of them."""
    pb = PagedBatch([1], [100], 4, 2, 64, 16, kv, seed=4)
    lens = [100, 1, 64, 17, 100]
    q = normal((len(lens), 4, 64), 8, 1.5).to(torch.bfloat16)
    table = pb.table.expand(len(lens), -1).contiguous()
    out = pa.paged_attention(q.to(dev()), pb.cache, table, cu_of([1] * len(lens)), ints(lens), max_q=max_q)
    k, v = pb.rows(pb.k64, 0), pb.rows(pb.v64, 0)
    for b, n in enumerate(lens):
        want, tol = attend64(q[b:b + 1].double(), k[:, :n], v[:, :n])
        check_close(out[b:b + 1], want, tol)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pools_past_32_bit_offsets(kv):
    """Pages whose rows lie more than 2^32 bytes (2^31 elements, where a row has two bytes) into the pool."""
    H, Hkv, D, page = 4, 2, 128, 64
    each = Hkv * page * D * (2 if kv == "bf16" else 1)
    P = 2 ** 32 // each + 40
    cache = pa.PagedKVCache.allocate(P, Hkv, D, dev(), page_size=page, dtype=kv)
    near, far = 3, P - 2  # the last one's rows begin behind 2^32 bytes
    assert far * each > 2 ** 32
    ids = [far, near, far + 1]
    table = torch.tensor([ids], dtype=torch.int32, device=dev())
    n = 2 * page + 9
    qkv = normal((n, (H + 2 * Hkv) * D), 5).to(torch.bfloat16)
    cos, sin = (torch.from_numpy(t) for t in rope_tables(D, n, 1e4))
    pa.rope_write(qkv.to(dev()), cos.to(dev()), sin.to(dev()), cu_of([n]), None, H, Hkv, cache=cache, page_table=table)
    k = torch.empty((1, Hkv, n, D), dtype=torch.bfloat16, device=dev())
    v = torch.empty_like(k)
    pa.read_pages(cache, table, ints([n]), k, v)
    want_v = qkv.view(n, H + 2 * Hkv, D)[:, H + Hkv:].float()
    if kv == "fp8":
        want_v = values_of(*quantise(want_v)).float()
    assert torch.equal(v[0].cpu().float().transpose(0, 1), want_v)
    for pool in (cache.key_pages, cache.value_pages):  # nothing landed where a wrapped offset would be
        raw = pool.view(torch.uint8)
        assert not bool(raw[:near].any()) and not bool(raw[near + 1: near + 40].any())
    k64, v64 = k[0].double().cpu(), v[0].double().cpu()
    for new, max_q in ((1, 1), (40, 40)):
        q = normal((new, H, D), 7, 1.5).to(torch.bfloat16)
        want, tol = attend64(q.double(), k64, v64)
        out = pa.paged_attention(q.to(dev()), cache, table, cu_of([new]), ints([n]), max_q=max_q)
        check_close(out, want, tol)


def test_two_graphs_with_split_contexts_at_once():
    """Each captured call has its own partials: replays on two streams, with eager work between."""
    pbs = [PagedBatch([1], [5000], 4, 2, 64, 64, "bf16", seed=s) for s in (1, 2)]
    runs = []
    for pb in pbs:
        args = (pb.q_dev, pb.cache, pb.table, pb.cu, pb.len)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            want = pa.paged_attention(*args, max_q=1)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = pa.paged_attention(*args, max_q=1)
        runs.append((stream, graph, out, want, args))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, _, out, _, _ in runs:
            out.fill_(9.0)
        torch.cuda.synchronize()
        for stream, graph, _, _, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [pa.paged_attention(*args, max_q=1) for _, _, _, _, args in runs]
        torch.cuda.synchronize()
        for (_, _, out, want, _), e in zip(runs, eager):
            assert torch.equal(out, want) and torch.equal(e, want)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_in_wide_buffers(D):
    """Row strides of a million elements: a tile's rows span more than 2^27 bytes."""
    n, H, Hkv, ld = 70, 2, 1, 1 << 20
    x = normal((n, H + 2 * Hkv, D), 3, 1.2).to(torch.bfloat16)
    wide = torch.full((n, ld), math.nan, dtype=torch.bfloat16, device=dev())
    wide[:, : (H + 2 * Hkv) * D] = x.view(n, -1).to(dev())
    w = wide[:, : (H + 2 * Hkv) * D].unflatten(1, (H + 2 * Hkv, D))
    out = wide[:, -H * D:].unflatten(1, (H, D))
    pa.prompt_attention(w[:, :H], w[:, H:H + Hkv], w[:, H + Hkv:], cu_of([n]), out=out)
    want, tol = attend64(x[:, :H].double(), x[:, H:H + Hkv].double().transpose(0, 1),
                         x[:, H + Hkv:].double().transpose(0, 1))
    check_close(out, want, tol)
    assert bool(wide[:, (H + 2 * Hkv) * D: ld - H * D].isnan().all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_read_of_lengths_around_a_workgroups_rows(D, kv):
    total = [0, 1, 15, 16, 17, 31, 32, 33, 47, 48]
    pb = PagedBatch([0] * len(total), total, 2, 1, D, 16, kv)
    k = torch.full((len(total), 1, 48, D), 3.0, dtype=torch.bfloat16, device=dev())
    v = k.clone()
    pa.read_pages(pb.cache, pb.table, pb.len, k, v)
    for got, pool in ((k, pb.k64), (v, pb.v64)):
        got = got.cpu()
        for b, n in enumerate(total):
            assert torch.equal(got[b, :, :n].double(), pb.rows(pool, b))
            assert bool((got[b, :, n:] == 3.0).all())


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_many_users_of_unlike_lengths(kv):
    """Contexts that are split beside ones that are not, empty ones and padding."""
    total = [0, 1, 2600] + [(i * 389) % 2600 for i in range(67)]
    new = [1] * len(total)
    pb = PagedBatch(new, total, 4, 2, 64, 32, kv, seed=6)
    assert pa._scratch_bytes(0, 70, 4, 2, 64, 70, 1, 2600) == 4 * 70 * 4 * 66 * 4  # four splits
    want, tol = pb.reference()
    args = (pb.q_dev, pb.cache, pb.table, pb.cu, pb.len)
    out = pa.paged_attention(*args, max_q=1, max_kv=2600)
    check_close(out, want, tol)
    assert bool((out[0] == 0).all())
    assert torch.equal(out, pa.paged_attention(*args, max_q=1, max_kv=2600))


def test_few_rows_over_bf16_pages_use_16_bits_of_p():
    """Half a step of the output's bf16 is nearly all of the bound that is left."""
    pb = PagedBatch([1, 1], [300, 77], 4, 2, 128, 16, "bf16", seed=2)
    out = pa.paged_attention(pb.q_dev, pb.cache, pb.table, pb.cu, pb.len, max_q=1)
    for b in range(2):
        want, tol = attend64(pb.q[b:b + 1].double(), pb.rows(pb.k64, b), pb.rows(pb.v64, b), p_half=BF16_HALF ** 2)
        check_close(out[b:b + 1], want, tol)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("total,max_kv", [(300, None), (5000, 5000)])
def test_values_not_finite_early_in_a_context(bad, D, total, max_kv):
    """A value that every row sees, in the first round, in a later one and in another split:
    infinite where the weights are positive, whichever kernel max_q chooses."""
    H, Hkv = 4, 2
    pb = PagedBatch([1], [total], H, Hkv, D, 32, "bf16", seed=5)
    if max_kv:
        assert pa._scratch_bytes(0, 1, H, Hkv, D, 1, 1, max_kv) > 0
    for dim, where in ((1, 3), (2, 130), (7, total // 2), (D - 1, total - 40)):
        pid, row = int(pb.table_host[0, where // 32]), where % 32
        pb.cache.value_pages[pid, :, row, dim] = bad
        pb.v64[pid, :, row, dim] = bad
    want, tol = pb.reference()
    assert int((~torch.isfinite(want)).sum()) == 4 * H
    for max_q in (1, 40):
        check_close(pa.paged_attention(pb.q_dev, pb.cache, pb.table, pb.cu, pb.len, max_q=max_q, max_kv=max_kv), want, tol)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("max_kv", [2 ** 31 + 7, 3 * 2 ** 31, 2 ** 40, 2 ** 63 - 1])
@pytest.mark.parametrize("new,max_q", [([1, 1], 1), ([40, 3], 40), ([1, 1], 2 ** 62)])
def test_hints_of_the_c_entry_behind_the_table(kv, max_kv, new, max_q):
    """The C entry point with hints far behind the page table's room, in its own scratch: rounding only."""
    from bitnet_tt import _native as N

    H, Hkv, D = 4, 2, 64
    pb = PagedBatch(new, [700, 41], H, Hkv, D, 16, kv, seed=3)
    T, B, L = sum(new), len(new), N.lib()
    nbytes = L.btl_paged_attention_scratch_bytes(T, H, Hkv, D, B, max_q, max_kv)
    scratch = torch.empty(max(16, nbytes), dtype=torch.uint8, device=dev())
    word = torch.zeros(1, dtype=torch.int32, device=dev())
    out = torch.empty_like(pb.q_dev)
    rc = L.btl_paged_attention(pb.q_dev.data_ptr(), H * D, T, H, pb.cache._pages, pb.table.data_ptr(), pb.table.shape[1],
                               pb.cu.data_ptr(), pb.len.data_ptr(), B, D ** -0.5, max_q, max_kv, out.data_ptr(), H * D,
                               scratch.data_ptr(), nbytes, word.data_ptr(), N.raw_stream(0))
    assert rc == 0
    want, tol = pb.reference()
    check_close(out, want, tol)
    assert int(word) == 0


@pytest.mark.parametrize("power", [21, 29])
def test_large_scores_that_are_equal(power):
    """scale q.k of 2^power at every position: weights are equal whatever 32 bits make of the offset, so the
    output is the value that all positions have."""
    H, Hkv, D, n = 4, 2, 64, 40
    side = 2.0 ** ((power + 3 - 6) // 2)  # D side^2 / 8
    assert side * side * D / 8 == 2.0 ** power
    q = torch.full((n, H, D), side, dtype=torch.bfloat16, device=dev())
    k = torch.full((n, Hkv, D), side, dtype=torch.bfloat16, device=dev())
    v = torch.full((n, Hkv, D), 3.0, dtype=torch.bfloat16, device=dev())
    assert torch.equal(pa.prompt_attention(q, k, v, cu_of([n])), torch.full_like(q, 3.0))
    cache = pa.PagedKVCache.allocate(3, Hkv, D, dev(), page_size=16)
    cache.key_pages.fill_(side)
    cache.value_pages.fill_(3.0)
    table = torch.arange(3, dtype=torch.int32, device=dev())[None]
    for max_q in (1, 40):
        out = pa.paged_attention(q, cache, table, cu_of([n]), ints([n]), max_q=max_q)
        assert torch.equal(out, torch.full_like(q, 3.0))
