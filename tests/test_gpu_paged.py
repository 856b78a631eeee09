"""The paged key-value cache on the GPU against 64 bits: rotation and page
writes, page reads, attention over the pages."""

import math

import pytest
import torch

from paged_helpers import (BF16_HALF, E4M3_HALF, F32_HALF, PagedBatch, attend64, check_close, cu_of, dev, ints, normal,
                           quantise, values_of)

from bitnet_tt import paged_attention as pa
from bitnet_tt.utils.rope import rope_tables

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


# ---- write ------------------------------------------------------------


def plain_rotation(x, cos, sin, R, adjacent):
    if adjacent:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2:R]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., R:]), -1)


def write_case(new, total, H, Hkv, D, R, adjacent, page, kv, seed=1, pad_rows=0, k_out=False, in_place=False):
    T = sum(new) + pad_rows
    S = max(max(total), 1) + 5
    qkv = normal((T, (H + 2 * Hkv) * D), seed, 1.3).to(torch.bfloat16)
    cos, sin = (torch.from_numpy(t) for t in rope_tables(R, S, 10000.0))
    pb = PagedBatch(new, total, H, Hkv, D, page, kv, seed=seed)
    q_seq = [b for b, n in enumerate(new) for _ in range(n)]
    pos = [total[b] - new[b] + i for b in range(len(new)) for i in range(new[b])]
    d_qkv = qkv.to(dev())
    kout = torch.full((T, Hkv, D), 7.0, dtype=torch.bfloat16, device=dev()) if k_out else None
    q_out = torch.full((T, H, D), 5.0, dtype=torch.bfloat16, device=dev())
    if in_place:
        x = d_qkv.view(T, H + 2 * Hkv, D)
        q_out, kout = x[:, :H], x[:, H:H + Hkv]
    before = [t.clone() for t in (pb.cache.key_pages.view(torch.uint8), pb.cache.value_pages.view(torch.uint8))]
    q = pa.rope_write(d_qkv, cos.to(dev()), sin.to(dev()), pb.cu, pb.len, H, Hkv, cache=pb.cache, page_table=pb.table,
                      rope_adjacent=adjacent, q_out=q_out, k_out=kout)
    torch.cuda.synchronize()
    x = qkv.float().view(T, H + 2 * Hkv, D)
    n = len(pos)
    at = torch.tensor(pos).clamp(min=0)
    y = plain_rotation(x[:n, : H + Hkv], cos[at][:, None], sin[at][:, None], R, adjacent)
    y64 = plain_rotation(x[:n, : H + Hkv].double(), cos[at][:, None].double(), sin[at][:, None].double(), R, adjacent)
    dead = torch.tensor([p < 0 for p in pos], dtype=torch.bool)
    y[dead] = 0
    y64[dead] = 0
    # 64 bits: two products and a sum in 32 bits, then one rounding
    mag = plain_rotation(x[:n, : H + Hkv].double().abs(), cos[at][:, None].double().abs(), -sin[at][:, None].double().abs(),
                         R, adjacent).abs() + y64.abs()
    got_q = q[:n].float().cpu()
    assert float(((got_q.double() - y64[:, :H]).abs() - BF16_HALF * y64[:, :H].abs() - 4 * F32_HALF * mag[:, :H]).max()) <= 0
    assert torch.equal(got_q, y[:, :H].to(torch.bfloat16).float())
    if k_out or in_place:
        assert torch.equal(kout[:n].float().cpu(), y[:, H:].to(torch.bfloat16).float())
    if pad_rows and not in_place:
        assert bool((q[n:] == 5.0).all())
        if k_out:
            assert bool((kout[n:] == 7.0).all())
    # pages: the written rows, and every other byte as it was
    want = [t.cpu() for t in before]
    exps = [None if e is None else e.cpu() for e in (pb.cache.key_exp, pb.cache.value_exp)]
    rows = [y[:, H:], x[:n, H + Hkv:]]
    pools = [pb.cache.key_pages, pb.cache.value_pages]
    for w, r, e in zip(want, rows, exps):
        if kv == "bf16":
            raw = r.to(torch.bfloat16).view(torch.uint8).view(n, Hkv, -1)
        else:
            codes, byte = quantise(r)
            raw = codes.view(torch.uint8)
            off = (values_of(codes, byte) - r.double()).abs()
            assert float((off - E4M3_HALF * r.double().abs() - torch.exp2(byte.double() - 137)[..., None]).max()) <= 0
        for i, (b, p) in enumerate(zip(q_seq, pos)):
            if p < 0:
                continue
            page_id = int(pb.table_host[b, p // page])
            w[page_id, :, p % page] = raw[i]
            if kv != "bf16":
                assert torch.equal(e[page_id, :, p % page], byte[i])
    for w, pool in zip(want, pools):
        assert torch.equal(pool.view(torch.uint8).cpu(), w)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("H,Hkv,D,R,adjacent", [(20, 5, 128, 128, False), (4, 2, 64, 64, True), (3, 3, 128, 32, True),
                                                (8, 1, 64, 16, False), (4, 2, 128, 96, False)])
@pytest.mark.parametrize("new,total", [([1], [1]), ([1, 1, 1], [5, 64, 129]), ([7, 0, 33], [7, 12, 50]),
                                       ([3, 2], [1, 2])])
def test_write(kv, H, Hkv, D, R, adjacent, new, total):
    write_case(new, total, H, Hkv, D, R, adjacent, 16, kv)


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_write_many_tokens(page, kv):
    """Eight tokens a workgroup (over 1024 rows), more than 64 sequences, rows behind the last."""
    new = [(37 * i) % 29 + (i % 5 == 0) for i in range(90)]
    total = [n + (53 * i) % 301 for i, n in enumerate(new)]
    assert sum(new) > 1024
    write_case(new, total, 4, 2, 64, 64, False, page, kv, pad_rows=5, k_out=True)


def test_write_in_place():
    write_case([5, 9], [5, 40], 4, 2, 64, 64, False, 32, "bf16", in_place=True)
    write_case([5, 9], [5, 40], 20, 5, 128, 64, True, 32, "fp8", in_place=True)


def test_write_without_pages_is_a_prompt():
    T, H, Hkv, D = 70, 4, 2, 64
    qkv = normal((T, (H + 2 * Hkv) * D), 3).to(torch.bfloat16)
    cos, sin = (torch.from_numpy(t) for t in rope_tables(D, 64, 10000.0))
    k = torch.empty((T, Hkv, D), dtype=torch.bfloat16, device=dev())
    q = pa.rope_write(qkv.to(dev()), cos.to(dev()), sin.to(dev()), cu_of([50, 20]), None, H, Hkv, k_out=k)
    at = torch.tensor(list(range(50)) + list(range(20)))
    y = plain_rotation(qkv.float().view(T, -1, D)[:, : H + Hkv], cos[at][:, None], sin[at][:, None], D, False)
    assert torch.equal(torch.cat((q, k), 1).float().cpu(), y.to(torch.bfloat16).float())


def test_write_extreme_rows():
    """Zeros, subnormals, the largest values, and values that are not finite."""
    H, Hkv, D, page = 1, 1, 64, 16
    x = torch.zeros(8, 3, D)
    x[1, 2] = 1e-38
    x[2, 2] = 3.3e38
    x[3, 2, 5] = math.inf
    x[4, 2, 63] = math.nan
    x[5, 2] = torch.linspace(-448, 448, D)
    x[6, 2, 0] = 2.0 ** -133
    x[7, 2] = normal((D,), 5) * 1e-20
    x = x.to(torch.bfloat16)
    pb = PagedBatch([8], [8], H, Hkv, D, page, "fp8")
    cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(D, 8, 10000.0))
    pa.rope_write(x.view(8, -1).to(dev()), cos, sin, pb.cu, pb.len, H, Hkv, cache=pb.cache, page_table=pb.table)
    pid = int(pb.table_host[0, 0])
    codes, byte = quantise(x[:, 2].float())
    assert torch.equal(pb.cache.value_exp[pid, 0, :8].cpu(), byte)
    assert torch.equal(pb.cache.value_pages[pid, 0, :8].cpu().view(torch.uint8), codes.view(torch.uint8))
    k = torch.zeros((1, 1, 8, D), dtype=torch.bfloat16, device=dev())
    v = torch.zeros_like(k)
    pa.read_pages(pb.cache, pb.table, pb.len, k, v)
    want = values_of(codes, byte).to(torch.bfloat16)
    assert torch.isnan(want[3:5]).all()
    assert torch.equal(torch.isnan(v[0, 0].cpu()), torch.isnan(want))
    assert torch.equal(v[0, 0].cpu().nan_to_num(0.0), want.nan_to_num(0.0))


# ---- read ---------------------------------------------------------------


def test_read_every_code():
    """All codes under exponents across the range."""
    P, D, page = 4, 128, 64
    codes = torch.arange(P * page * D, dtype=torch.int64).remainder(256).to(torch.uint8).view(P, 1, page, D)
    exps = (torch.arange(P * page) * 254 // (P * page - 1) + 0).clamp(min=1).to(torch.uint8).view(P, 1, page)
    exps = exps.clamp(max=127 + 119)
    cache = pa.PagedKVCache(codes.view(torch.float8_e4m3fn).to(dev()), codes.flip(0).contiguous().view(torch.float8_e4m3fn).to(dev()),
                            exps.to(dev()), exps.to(dev()))
    n = P * page
    k = torch.zeros((1, 1, n, D), dtype=torch.bfloat16, device=dev())
    v = torch.zeros_like(k)
    pa.read_pages(cache, torch.arange(P, dtype=torch.int32, device=dev()).view(1, P), ints([n]), k, v)
    for got, c in ((k, codes), (v, codes.flip(0))):
        want = values_of(c.view(torch.float8_e4m3fn), exps).view(n, D).to(torch.bfloat16)
        got = got[0, 0].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,total", [(16, [1, 0, 17]), (48, [100, 47, 48]), (256, [300])])
def test_read(kv, D, page, total):
    pb = PagedBatch([0] * len(total), total, 2, 2, D, page, kv)
    S = max(total) + 9
    k = torch.full((len(total), 2, S, D), 3.0, dtype=torch.bfloat16, device=dev())
    v = k.clone()
    pa.read_pages(pb.cache, pb.table, pb.len, k, v)
    for got, pool in ((k, pb.k64), (v, pb.v64)):
        got = got.cpu()
        for b, n in enumerate(total):
            assert torch.equal(got[b, :, :n].double(), pb.rows(pool, b))
            assert bool((got[b, :, n:] == 3.0).all())


# ---- attention ------------------------------------------------------------

HEADS = [(20, 5, 128), (4, 2, 64), (7, 1, 128), (3, 3, 64), (16, 1, 64)]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("total", [[1], [5, 16, 17, 32, 33], [255, 256, 257, 0, 700], [1000]])
def test_single_tokens(kv, H, Hkv, D, total):
    new = [1 if n else 0 for n in total]
    pb = PagedBatch(new, total, H, Hkv, D, 16, kv)
    want, tol = pb.reference()
    out = pa.paged_attention(pb.q_dev, pb.cache, pb.table, pb.cu, pb.len, max_q=1, max_kv=max(total))
    check_close(out, want, tol)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("new,total", [([2], [2]), ([3, 0, 2], [40, 9, 2]), ([33], [33]), ([65, 1, 20], [130, 64, 300]),
                                       ([5, 70], [3, 70])])
def test_chunks(kv, H, Hkv, D, new, total):
    pb = PagedBatch(new, total, H, Hkv, D, 48, kv)
    want, tol = pb.reference()
    out = pa.paged_attention(pb.q_dev, pb.cache, pb.table, pb.cu, pb.len)
    check_close(out, want, tol)
    if any(n > t for n, t in zip(new, total)):
        assert bool((want[:2] == 0).all())


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,total,max_q", [([1], [5000], 1), ([1, 1], [3001, 40], 1), ([40], [4100], 40),
                                             ([3, 1], [2600, 2049], 3)])
def test_split_contexts(kv, D, new, total, max_q):
    """Few rows over long contexts: partials of several workgroups, empty ones too."""
    pb = PagedBatch(new, total, 4, 2, D, 64, kv)
    assert pa._scratch_bytes(0, sum(new), 4, 2, D, len(new), max_q, max(total)) > 0
    want, tol = pb.reference()
    args = (pb.q_dev, pb.cache, pb.table, pb.cu, pb.len)
    first = pa.paged_attention(*args, max_q=max_q, max_kv=max(total))
    check_close(first, want, tol)
    assert torch.equal(first, pa.paged_attention(*args, max_q=max_q, max_kv=max(total)))  # a fixed order
    # hints that are wrong, or not given: other kernels, the same values
    for mq, mkv in ((None, None), (1, 600), (sum(new), 1), (1, 10 ** 9)):
        check_close(pa.paged_attention(*args, max_q=mq, max_kv=mkv), want, tol)


def test_contiguous_cache_as_pages():
    from bitnet_tt.layers.attention import DecodeAttention

    H, Hkv, D, S, B = 8, 2, 128, 160, 3
    att = DecodeAttention(H, Hkv, D, S, dev())
    kv = att.new_cache(B)
    kv.key_cache.copy_(normal(kv.key_cache.shape, 1))
    kv.value_cache.copy_(normal(kv.value_cache.shape, 2))
    pos = ints([0, 77, 159])
    qkv = normal((B, (H + 2 * Hkv) * D), 3).to(torch.bfloat16).to(dev())
    k0, v0 = kv.key_cache.clone(), kv.value_cache.clone()
    want = att(qkv, kv, pos)
    k1, v1 = kv.key_cache.clone(), kv.value_cache.clone()
    kv.key_cache.copy_(k0)
    kv.value_cache.copy_(v0)
    cache = pa.PagedKVCache.of_cache(kv)
    table = torch.arange(B, dtype=torch.int32, device=dev())[:, None]
    q = pa.rope_write(qkv, att.rope_cos, att.rope_sin, cu_of([1] * B), pos + 1, H, Hkv, cache=cache, page_table=table)
    out = pa.paged_attention(q, cache, table, cu_of([1] * B), pos + 1, max_q=1)
    assert torch.equal(kv.key_cache, k1) and torch.equal(kv.value_cache, v1)
    o64 = [attend64(q[b:b + 1].double().cpu(), k1[b, :, : int(pos[b]) + 1].double().cpu(),
                    v1[b, :, : int(pos[b]) + 1].double().cpu()) for b in range(B)]
    check_close(out, torch.cat([o for o, _ in o64]), torch.cat([t for _, t in o64]))
    check_close(want.view(B, H, D), torch.cat([o for o, _ in o64]), torch.cat([t for _, t in o64]))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,max_q", [(3, 3), (40, 40)])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_values_not_finite_reach_only_rows_that_see_them(bad, new, max_q, kv):
    """The last chunk's values: a row does not feel a later position's."""
    H, Hkv, D, total = 4, 2, 64, 90
    pb = PagedBatch([new], [total], H, Hkv, D, 16, kv)
    where = total - 2
    pid, row = int(pb.table_host[0, where // 16]), where % 16
    if kv == "bf16":
        pb.cache.value_pages[pid, :, row, 7] = bad
        pb.v64[pid, :, row, 7] = bad
    else:  # a row that holds such a value reads as NaN whole
        pb.cache.value_pages.view(torch.uint8)[pid, :, row] = 0x7F
        pb.v64[pid, :, row] = math.nan
        pb.cache.key_pages.view(torch.uint8)[pid, :, row, 3] = 0x7F  # and a masked score is no score
        pb.k64[pid, :, row, 3] = math.nan
    want, tol = pb.reference()
    out = pa.paged_attention(pb.q_dev, pb.cache, pb.table, pb.cu, pb.len, max_q=max_q)
    assert torch.isfinite(want[: new - 2]).all() and not torch.isfinite(want[new - 2:]).all()
    check_close(out, want, tol)


def test_rows_behind_the_last_sequence_and_strided_rows():
    pb = PagedBatch([3, 2], [20, 30], 4, 2, 64, 16, "bf16")
    want, tol = pb.reference()
    wide = torch.full((8, 8, 64), math.nan, dtype=torch.bfloat16, device=dev())
    wide[:5, :4] = pb.q_dev
    out = torch.full((8, 6, 64), 2.0, dtype=torch.bfloat16, device=dev())
    for mq in (None, 3):
        pa.paged_attention(wide[:, :4], pb.cache, pb.table, pb.cu, pb.len, max_q=mq, out=out[:, :4])
        check_close(out[:5, :4], want, tol)
        assert bool((out[5:] == 2.0).all()) and bool((out[:, 4:] == 2.0).all())


def test_padded_batch():
    """Entries of kv_len 0 with a row each, as a captured batch pads: zeros, nothing written."""
    H, Hkv, D = 4, 2, 64
    pb = PagedBatch([1, 1, 1], [9, 0, 0], H, Hkv, D, 16, "bf16")
    before = pb.cache.key_pages.view(torch.int16).clone()
    cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(D, 16, 1e4))
    qkv = normal((3, (H + 2 * Hkv) * D), 2).to(torch.bfloat16).to(dev())
    q = pa.rope_write(qkv, cos, sin, pb.cu, pb.len, H, Hkv, cache=pb.cache, page_table=pb.table)
    out = pa.paged_attention(q, pb.cache, pb.table, pb.cu, pb.len, max_q=1)
    assert bool((q[1:] == 0).all()) and bool((out[1:] == 0).all()) and bool((out[0] != 0).any())
    changed = (pb.cache.key_pages.view(torch.int16) != before).any(-1).nonzero().cpu().tolist()
    assert changed == [[int(pb.table_host[0, 0]), h, 8] for h in range(Hkv)]


def test_graph_replays_and_advances():
    """Write and attend, captured: lengths, pages and rows advance between replays."""
    H, Hkv, D, B = 4, 2, 64, 2
    cache = pa.PagedKVCache.allocate(8, Hkv, D, dev(), page_size=32)
    table = torch.tensor([[5, 0, 7], [2, 3, 6]], dtype=torch.int32, device=dev())
    cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(D, 96, 1e4))
    cu, kv_len = cu_of([1] * B), ints([30, 60])
    qkv = normal((B, (H + 2 * Hkv) * D), 1).to(torch.bfloat16).to(dev())
    for pool, seed in ((cache.key_pages, 3), (cache.value_pages, 4)):
        pool.copy_(normal(pool.shape, seed))

    def step(c):
        q = pa.rope_write(qkv, cos, sin, cu, kv_len, H, Hkv, cache=c, page_table=table)
        return pa.paged_attention(q, c, table, cu, kv_len, max_q=1)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(cache)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(cache)
    torch.cuda.synchronize()
    for i in range(4):
        kv_len += 1
        qkv.copy_(normal(qkv.shape, 10 + i))
        twin = pa.PagedKVCache(cache.key_pages.clone(), cache.value_pages.clone())
        want = step(twin)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(cache.key_pages, twin.key_pages) and torch.equal(cache.value_pages, twin.value_pages)


def test_two_streams_read_one_cache():
    """Calls with split contexts at once: nothing is shared."""
    pb = PagedBatch([1], [6000], 4, 2, 64, 64, "bf16")
    args = (pb.q_dev, pb.cache, pb.table, pb.cu, pb.len)
    want = pa.paged_attention(*args, max_q=1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(pa.paged_attention(*args, max_q=1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- batches that are not well formed -------------------------------------


def expect_error():
    with pytest.raises(RuntimeError, match="paged workspace"):
        pa.check("cuda:0")


@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pages_outside_the_pool(max_q, kv):
    """A page that the pool does not have sets the error word and is not followed; other
    sequences are right."""
    pb = PagedBatch([1, 1], [40, 40], 4, 2, 64, 16, kv)
    want, tol = pb.reference()
    for wrong in (-1, pb.cache.num_pages, 2 ** 31 - 1, -2 ** 31):
        table = pb.table.clone()
        table[0, 1] = wrong
        out = pa.paged_attention(pb.q_dev, pb.cache, table, pb.cu, pb.len, max_q=max_q)
        expect_error()
        check_close(out[1:], want[1:], tol[1:])
        before = pb.cache.key_pages.view(torch.uint8).clone()
        cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(64, 64, 1e4))
        x = normal((2, 8 * 64), 2).to(torch.bfloat16).to(dev())
        pa.rope_write(x, cos, sin, pb.cu, ints([20, 0]), 4, 2, cache=pb.cache, page_table=table)
        expect_error()
        assert torch.equal(pb.cache.key_pages.view(torch.uint8), before)
        k = torch.zeros((2, 2, 40, 64), dtype=torch.bfloat16, device=dev())
        pa.read_pages(pb.cache, table, pb.len, k, torch.zeros_like(k))
        expect_error()
        assert torch.equal(k[1].double().cpu(), pb.rows(pb.k64, 1)) and bool((k[0, :, 16:32] == 0).all())


@pytest.mark.parametrize("cu,lens", [([0, 5, 2], [40, 40]), ([0, 1, 900], [40, 40]), ([-3, 1, 2], [40, 40]),
                                     ([0, 1, 2], [40, 2 ** 30]), ([0, 1, 2], [-5, 40])])
def test_batches_not_well_formed(cu, lens):
    pb = PagedBatch([1, 1], [40, 40], 4, 2, 64, 16, "bf16")
    cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(64, 64, 1e4))
    x = normal((2, 8 * 64), 2).to(torch.bfloat16).to(dev())
    for mq in (1, 40):
        pa.paged_attention(pb.q_dev, pb.cache, pb.table, ints(cu), ints(lens), max_q=mq)
        expect_error()
    pa.rope_write(x, cos, sin, ints(cu), ints(lens), 4, 2, cache=pb.cache, page_table=pb.table)
    expect_error()


def test_position_behind_the_angle_tables():
    pb = PagedBatch([2], [40], 4, 2, 64, 16, "bf16")
    cos, sin = (torch.from_numpy(t).to(dev()) for t in rope_tables(64, 39, 1e4))
    x = normal((2, 8 * 64), 2).to(torch.bfloat16).to(dev())
    q = pa.rope_write(x, cos, sin, pb.cu, pb.len, 4, 2, cache=pb.cache, page_table=pb.table)
    expect_error()
    assert bool((q[0] != 0).any()) and bool((q[1] == 0).all())
