"""Prompts, chunks and single tokens through the layers of a model over a paged
cache: the operators together, as a program uses them."""

import numpy as np
import pytest
import torch

from paged_helpers import attend64, check_close, cu_of, dev, ints, normal

from bitnet_tt import paged_attention as pa
from bitnet_tt.config import BitNetMiniConfig
from bitnet_tt.decode import BitLinearDecodeStep
from bitnet_tt.layers.attention import DecodeAttention, PagedAttention
from bitnet_tt.ternary_matmul import ternary_matmul
from bitnet_tt.utils.rope import long_rope_tables, rope_tables, scaled_frequencies


def rotate64(x, cos, sin, adjacent):
    """x [n, heads, D] in 64 bits, whole heads."""
    c, s = cos[:, None].double(), sin[:, None].double()
    if adjacent:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("adjacent", [False, True])
def test_prompt_then_chunk_then_tokens(dtype, adjacent):
    """Two users: a prompt each, a chunk of one beside a token of the other, tokens.
    Every attention output against 64 bits over what the pages hold."""
    H, Hkv, D, page = 4, 2, 64, 16
    att = PagedAttention(H, Hkv, D, 128, dev(), use_fused_rope=adjacent)
    cache = att.new_cache(20, page, dtype)
    table = torch.arange(20, dtype=torch.int32).view(2, 10).flip(1).contiguous()
    length = [0, 0]
    for i, new in enumerate(([37, 20], [9, 1], [1, 1], [1, 1], [0, 1])):
        length = [a + b for a, b in zip(length, new)]
        qkv = normal((sum(new), (H + 2 * Hkv) * D), 50 + i).to(torch.bfloat16)
        out = att(qkv.to(dev()), cache, table.to(dev()), cu_of(new), ints(length), max_q=max(new))
        att.check()
        k = torch.zeros((2, Hkv, 160, D), dtype=torch.bfloat16, device=dev())
        v = torch.zeros_like(k)
        pa.read_pages(cache, table.to(dev()), ints(length), k, v)
        # the rotated queries as the write gives them (its own tests hold them to 64 bits)
        q = pa.rope_write(qkv.to(dev()), att.rope_cos, att.rope_sin, cu_of(new), ints(length), H, Hkv,
                          rope_adjacent=adjacent).double().cpu()
        at, x = 0, qkv.double().view(-1, H + 2 * Hkv, D)
        for b in range(2):
            n, m = new[b], length[b]
            pos = torch.arange(m - n, m)
            turned = rotate64(x[at:at + n, :H], att.rope_cos.cpu()[pos], att.rope_sin.cpu()[pos], adjacent)
            assert n == 0 or float((q[at:at + n] - turned).abs().max()) <= 2.0 ** -7 * float(turned.abs().max())
            want, tol = attend64(q[at:at + n], k[b, :, :m].double().cpu(), v[b, :, :m].double().cpu())
            check_close(out[at:at + n].view(n, H, D), want, tol)
            at += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_prompt_of_packed_rows_and_its_pages(dtype):
    """prompt() attends to the rows themselves and caches them; the cached chunk call over
    the same pages is the same up to what 8 bits cost."""
    H, Hkv, D = 8, 2, 128
    att = PagedAttention(H, Hkv, D, 128, dev())
    lens = [33, 70]
    qkv = normal((sum(lens), (H + 2 * Hkv) * D), 9).to(torch.bfloat16).to(dev())
    cu, table = cu_of(lens), torch.arange(8, dtype=torch.int32, device=dev()).view(2, 4)
    cache = att.new_cache(8, 32, dtype)
    o = att.prompt(qkv, cu, cache, table)
    again = att.prompt(qkv, cu)
    assert torch.equal(o, again)
    fresh = att.new_cache(8, 32, dtype)
    paged = att(qkv, fresh, table, cu, ints(lens))
    att.check()
    assert torch.equal(fresh.key_pages.view(torch.uint8), cache.key_pages.view(torch.uint8))
    assert torch.equal(fresh.value_pages.view(torch.uint8), cache.value_pages.view(torch.uint8))
    if dtype == "bf16":
        assert torch.equal(o, paged)  # the same kernel arithmetic on the same values


@pytest.mark.gpu
def test_forward_rows_is_the_layers_chain():
    """Each layer of forward_rows: the BitLinears are the calls of the rest of the package on
    the same rows (bits), the attention is PagedAttention's."""
    cfg = BitNetMiniConfig()
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=2, num_layers=2)
    step.alloc_paged(16, 256, page_size=32)
    new, total = [50, 7], [50, 7]
    table = torch.arange(16, dtype=torch.int32, device=dev()).view(2, 8)
    hidden = normal((57, cfg.hidden_size), 4).to(torch.bfloat16).to(dev())
    h = hidden.clone()
    got = step.forward_rows(hidden, table, cu_of(new), ints(total))
    step.check()
    assert got is hidden
    att = PagedAttention(cfg.num_attention_heads, cfg.num_kv_heads, cfg.head_dim, 256, dev(), rope_theta=cfg.rope_theta)
    for w in step.layers:
        qkv = ternary_matmul(h, w.qkv, norm_weight=w.input_layernorm, norm_epsilon=step.eps)
        a = att(qkv, att.new_cache(16, 32), table, cu_of(new), ints(total))
        h = ternary_matmul(a, w.o_proj, norm_weight=w.attn_sub_norm, norm_epsilon=step.eps, residual=h)
        f = ternary_matmul(h, w.gate_up, norm_weight=w.post_attention_layernorm, norm_epsilon=step.eps,
                           epilogue="relu2_mul")
        h = ternary_matmul(f, w.down, norm_weight=w.ffn_sub_norm, norm_epsilon=step.eps, residual=h)
    assert torch.equal(got, h)


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [0, 2])
def test_rows_of_no_sequence_meet_no_stale_memory(lead):
    """A batch padded before and behind its rows, in memory that held other values: the padding's rows are what zeros for
    their attention make of them, the others the unpadded call's; eager and replayed."""
    cfg = BitNetMiniConfig()
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=2, num_layers=2)
    step.alloc_paged(16, 256, page_size=32)
    table = torch.arange(16, dtype=torch.int32, device=dev()).view(2, 8)
    hidden = normal((40, cfg.hidden_size), 4).to(torch.bfloat16).to(dev())
    cu, total = cu_of([20, 7]), ints([20, 7])
    real = slice(lead, lead + 27)
    alone = step.forward_rows(hidden[real].clone(), table, cu, total)
    pad = torch.cat((hidden[:lead], hidden[lead + 27:]))
    want = torch.empty_like(hidden)
    want[real] = alone
    h = pad.clone()
    for w in step.layers:
        a = torch.zeros((len(pad), cfg.num_attention_heads * cfg.head_dim), dtype=torch.bfloat16, device=dev())
        h = ternary_matmul(a, w.o_proj, norm_weight=w.attn_sub_norm, norm_epsilon=step.eps, residual=h)
        f = ternary_matmul(h, w.gate_up, norm_weight=w.post_attention_layernorm, norm_epsilon=step.eps,
                           epilogue="relu2_mul")
        h = ternary_matmul(f, w.down, norm_weight=w.ffn_sub_norm, norm_epsilon=step.eps, residual=h)
    want[:lead], want[lead + 27:] = h[:lead], h[lead:]
    padded = cu + lead

    def stale():
        return [torch.full((40, n), 3.0, dtype=torch.bfloat16, device=dev())
                for n in (cfg.qkv_dim, cfg.hidden_size, cfg.intermediate_size) for _ in range(20)]

    got = hidden.clone()
    stale()  # (freed at once)
    assert torch.equal(step.forward_rows(got, table, padded, total), want)
    stream, rows = torch.cuda.Stream(), hidden.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step.forward_rows(rows, table, padded, total)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.forward_rows(rows, table, padded, total)
    for _ in range(3):
        rows.copy_(hidden)
        stale()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, want)
    step.check()


@pytest.mark.gpu
def test_pages_to_the_contiguous_step():
    """A prompt over pages, then decode steps on the contiguous caches: the attention of the
    first step sees what the pages held."""
    from bitnet_tt.config import BitNetConfig

    cfg = BitNetConfig(hidden_size=512, num_layers=2, num_attention_heads=4, num_key_value_heads=1,
                       intermediate_size=1024, vocab_size=1000, max_position_embeddings=256)
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=5, batch=3)
    step.alloc_buffers().alloc_attention(max_seq_len=128, pos=0)
    step.alloc_paged(12, 128, page_size=32)
    lens = [40, 1, 90]
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(3, 4).to(dev())
    step.forward_rows(normal((sum(lens), 512), 6).to(torch.bfloat16).to(dev()), table, cu_of(lens), ints(lens), max_kv=90)
    step.load_contiguous(table, ints(lens))
    for i in range(2):
        k, v = step.kv[i].key_cache, step.kv[i].value_cache
        for b, n in enumerate(lens):
            ids = table[b, : -(-n // 32)].long()
            assert torch.equal(k[b, 0, :n], step.pages[i].key_pages[ids, 0].flatten(0, 1)[:n])
            assert torch.equal(v[b, 0, :n], step.pages[i].value_pages[ids, 0].flatten(0, 1)[:n])
    # one more token each, both ways
    step.pos.copy_(ints(lens))
    step.reset_hidden()
    rows = step.hidden.clone()
    step.step_full()
    step.forward_rows(rows, table, cu_of([1, 1, 1]), ints([n + 1 for n in lens]), max_q=1)
    step.check()
    a, b = step.hidden.double(), rows.double()
    # two attention kernels that round differently, then int8 codes: normwise
    assert float((a - b).norm() / a.norm()) < 0.05
    with pytest.raises(RuntimeError, match="alloc_paged"):
        BitLinearDecodeStep(cfg, dev()).forward_rows(rows, table, cu_of([1]), ints([1]))


@pytest.mark.gpu
def test_the_step_goes_on_where_the_prompts_end():
    """alloc_attention's own positions (the last) and random caches, prompts, load_contiguous,
    and a step: it attends to the prompts and its own token, not to what else the caches hold."""
    from bitnet_tt.config import BitNetConfig

    cfg = BitNetConfig(hidden_size=512, num_layers=2, num_attention_heads=4, num_key_value_heads=1,
                       intermediate_size=1024, vocab_size=1000, max_position_embeddings=256)
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=5, batch=3)
    step.alloc_buffers().alloc_attention(max_seq_len=128).alloc_paged(12, 128, page_size=32)
    lens = [40, 1, 90]
    table = torch.arange(12, dtype=torch.int32, device=dev()).view(3, 4)
    step.forward_rows(normal((sum(lens), 512), 6).to(torch.bfloat16).to(dev()), table, cu_of(lens), ints(lens), max_q=90)
    step.load_contiguous(table, ints(lens))
    assert step.pos.tolist() == lens
    step.reset_hidden()
    rows = step.hidden.clone()
    step.step_full()
    step.forward_rows(rows, table, cu_of([1, 1, 1]), ints([n + 1 for n in lens]), max_q=1)
    step.check()
    a, b = step.hidden.double(), rows.double()
    # two attention kernels that round differently, then int8 codes: normwise
    assert float((a - b).norm() / a.norm()) < 0.05


@pytest.mark.gpu
def test_captured_hand_over_to_the_one_launch_step():
    """load_contiguous and the one-launch step in a graph: what the pages hold, positions and far angles follow at
    every replay, and the step is the eager calls' bit for bit."""
    from bitnet_tt.config import BitNetConfig

    cfg = BitNetConfig(hidden_size=512, num_layers=2, num_attention_heads=4, num_key_value_heads=1,
                       intermediate_size=1024, vocab_size=1000, max_position_embeddings=256)
    S = 4160
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=5, batch=2)
    step.alloc_buffers().alloc_attention(max_seq_len=S).alloc_paged(2 * S // 64, S, page_size=64)
    assert not torch.equal(step.attention.rope_cos[4096:], step.paged.rope_cos[4096:])
    table = torch.arange(2 * S // 64, dtype=torch.int32, device=dev()).view(2, -1)
    for pages, seed in zip(step.pages, (1, 2)):
        pages.key_pages.copy_(normal(pages.shape, seed))
        pages.value_pages.copy_(normal(pages.shape, seed + 2))
    kv_len = ints([100, 4130])

    def go():
        step.reset_hidden()
        step.load_contiguous(table, kv_len)
        step.step_persistent_full()

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        go()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            go()
    for lens in ([100, 4130], [0, 4159], [4100, 1], [64, 65]):
        kv_len.copy_(ints(lens))
        for kv in step.kv:
            kv.key_cache.fill_(3.0)
            kv.value_cache.fill_(3.0)
        step.pos.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, caches = step.hidden.clone(), [kv.key_cache.clone() for kv in step.kv]
        assert step.pos.tolist() == lens
        assert torch.equal(step.attention.rope_sin[4096:], step.paged.rope_sin[4096:])
        for kv, pages in zip(step.kv, step.pages):
            for b, n in enumerate(lens):
                rows = pages.key_pages[table[b].long(), 0].flatten(0, 1)
                assert torch.equal(kv.key_cache[b, 0, :n], rows[:n])
                assert bool((kv.key_cache[b, 0, n + 1:] == 3.0).all())  # row n is the step's own
        step.reset_hidden()
        step.load_contiguous(table, kv_len)
        step.step_full()
        assert torch.equal(got, step.hidden)
        assert all(torch.equal(a, kv.key_cache) for a, kv in zip(caches, step.kv))
    step.check()


def stepping(paged=(), attention=()):
    """A model of no layers on the host with both kinds of attention."""
    cfg = BitNetMiniConfig(num_attention_heads=2)
    step = BitLinearDecodeStep(cfg, torch.device("cpu"), batch=2)
    step.alloc_attention(**{"max_seq_len": 64, **dict(attention)})
    step.paged = PagedAttention(cfg.num_attention_heads, cfg.num_kv_heads, cfg.head_dim,
                                **{"max_seq_len": 64, "device": "cpu", "rope_theta": cfg.rope_theta, **dict(paged)})
    step.pages = []
    return step


@pytest.mark.parametrize("hidden,match", [
    (torch.zeros((3, 256)), "bf16"), (torch.zeros((3, 256), dtype=torch.int8), "bf16"),
    (torch.zeros((3, 256), dtype=torch.float16), "bf16"), (torch.zeros((3, 128), dtype=torch.bfloat16), "bf16"),
    (torch.zeros((1, 3, 256), dtype=torch.bfloat16), "bf16"), (torch.zeros(256, dtype=torch.bfloat16), "bf16"),
    (torch.zeros((3, 256), dtype=torch.bfloat16), "ROCm GPU"), (torch.zeros((3, 1, 256), dtype=torch.bfloat16), "ROCm GPU"),
    (torch.zeros((3, 2, 256), dtype=torch.bfloat16), "bf16"),
])
def test_rows_that_forward_rows_refuses(hidden, match):
    """Before anything reads them: rows of fewer bytes than bf16's would be read behind their end."""
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match=match):
        stepping().forward_rows(hidden, i32[None], i32, i32[:1])


@pytest.mark.parametrize("paged,attention", [
    ({"use_fused_rope": True}, {}), ({}, {"use_fused_rope": True}), ({"rope_theta": 10000.0}, {}), ({"rotary_dim": 64}, {}),
    ({"rope_scaling": {"type": "linear", "factor": 2.0}}, {}),
    ({"rope_scaling": {"rope_type": "yarn", "factor": 4.0}, "use_fused_rope": True}, {"use_fused_rope": True}),
])
def test_keys_that_the_steps_queries_do_not_match(paged, attention):
    step = stepping(paged, attention)
    with pytest.raises(ValueError, match="rotated by"):
        step.load_contiguous(torch.zeros((2, 1), dtype=torch.int32), torch.tensor([5, 7], dtype=torch.int32))
    assert step.pos.tolist() == [63, 63]


@pytest.mark.parametrize("paged,attention", [
    ({}, {}), ({"use_fused_rope": True}, {"use_fused_rope": True}), ({"max_seq_len": 32}, {}),
    ({"rope_scaling": {"rope_type": "default"}}, {}),
])
def test_keys_that_match_and_the_next_positions(paged, attention):
    step = stepping(paged, attention)
    step.load_contiguous(torch.zeros((2, 1), dtype=torch.int32), torch.tensor([5, 7], dtype=torch.int32))
    assert step.pos.tolist() == [5, 7]


# ---- angle tables (host) --------------------------------------------------


def test_long_tables_without_scaling_are_the_plain_angles():
    cos, sin = long_rope_tables(64, 300, 10000.0)
    c, s = rope_tables(64, 300, 10000.0)
    # float32 angles of up to 300: off by 300 x 2^-24 and the frequency's own half step
    assert float((cos - torch.from_numpy(c)).abs().max()) < 300 * 2.0 ** -23 + 2.0 ** -23
    assert float((sin - torch.from_numpy(s)).abs().max()) < 300 * 2.0 ** -23 + 2.0 ** -23
    far, _ = long_rope_tables(16, 100001, 10000.0)
    want = np.cos(100000.0 * 10000.0 ** (-np.arange(0, 16, 2) / 16.0))
    assert np.abs(far[100000].double().numpy() - want).max() <= 2.0 ** -24


@pytest.mark.parametrize("theta,dim,rotary", [(500000.0, 128, None), (10000.0, 64, 32)])
def test_the_layers_own_angles_at_far_positions(theta, dim, rotary):
    """Float32 angles are off by up to 0.006 at position 100000; the layer's tables are rounded once. The first
    4096 rows are DecodeAttention's."""
    n, R = 100001, rotary or dim
    for kw in ({}, {"rope_scaling": {"type": "default"}}):
        att = PagedAttention(4, 2, dim, n, "cpu", rope_theta=theta, rotary_dim=rotary, **kw)
        assert att.rope_cos.shape == att.rope_sin.shape == (n, R // 2) and att.rope_cos.dtype is torch.float32
        c, s = rope_tables(R, 5000, theta)
        assert np.array_equal(att.rope_cos[:4096], c[:4096]) and np.array_equal(att.rope_sin[:4096], s[:4096])
        freq = theta ** (-np.arange(0, R, 2) / R)
        for p in (4096, 4097, 65536, 100000):
            # a 64-bit angle of up to 1e5: off by 1e5 x 2^-52
            for got, f in ((att.rope_cos, np.cos), (att.rope_sin, np.sin)):
                assert np.abs(got[p].double().numpy() - f(p * freq)).max() <= 2.0 ** -24 / 2 + 1e-10
    for n in (1, 4095, 4096):
        c, s = rope_tables(R, n, theta)
        att = PagedAttention(4, 2, dim, n, "cpu", rope_theta=theta, rotary_dim=rotary)
        assert np.array_equal(att.rope_cos, c) and np.array_equal(att.rope_sin, s)


@pytest.mark.parametrize("paged,contiguous", [(5000, 5000), (6000, 5000), (5000, 6000), (4096, 5000), (4100, 64)])
def test_the_step_takes_the_far_angles_of_the_cached_keys(paged, contiguous):
    step = stepping({"max_seq_len": paged}, {"max_seq_len": contiguous})
    before = step.attention.rope_cos.clone(), step.attention.rope_sin.clone()
    where = step.attention.rope_cos.data_ptr()
    step.load_contiguous(torch.zeros((2, 1), dtype=torch.int32), torch.tensor([5, 7], dtype=torch.int32))
    n = min(paged, contiguous)
    for got, own, old in ((step.attention.rope_cos, step.paged.rope_cos, before[0]),
                          (step.attention.rope_sin, step.paged.rope_sin, before[1])):
        assert got.shape[0] == contiguous and torch.equal(got[:n], own[:n]) and torch.equal(got[n:], old[n:])
    assert step.attention.rope_cos.data_ptr() == where  # captured steps read them


def test_linear_and_llama3_frequencies():
    plain, one = scaled_frequencies(128, 500000.0)
    f, a = scaled_frequencies(128, 500000.0, {"type": "linear", "factor": 4})
    assert one == a == 1.0 and np.allclose(f * 4, plain, rtol=1e-15)
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    f, a = scaled_frequencies(128, 500000.0, cfg)
    for x, y in zip(plain, f):  # dim by dim
        wave = 2 * np.pi / x
        if wave < 8192 / 4:
            want = x
        elif wave > 8192:
            want = x / 8
        else:
            t = (8192 / wave - 1.0) / 3.0
            want = (1 - t) * x / 8 + t * x
        assert abs(y - want) <= 1e-14 * want
    assert a == 1.0 and f[0] == plain[0] and abs(f[-1] * 8 / plain[-1] - 1) < 1e-14


def test_yarn_frequencies():
    cfg = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    plain, _ = scaled_frequencies(64, 10000.0)
    f, a = scaled_frequencies(64, 10000.0, cfg)
    assert abs(a - (0.1 * np.log(16.0) + 1.0)) < 1e-15
    turns = 4096 * plain / (2 * np.pi)
    assert np.allclose(f[turns > 40], plain[turns > 40], rtol=1e-15)
    assert np.allclose(f[turns < 0.5] * 16, plain[turns < 0.5], rtol=1e-15)
    assert (np.diff(f) < 0).all() and (f <= plain).all() and (f >= plain / 16 * (1 - 1e-15)).all()
    assert scaled_frequencies(64, 10000.0, {**cfg, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("bad", [{"type": "dynamic", "factor": 2.0}, {"type": "linear", "factor": 0.5}])
def test_scalings_refused(bad):
    with pytest.raises(ValueError):
        scaled_frequencies(64, 10000.0, bad)


def test_layer_refuses():
    for kw in (dict(head_dim=96), dict(num_kv_heads=3), dict(rotary_dim=24), dict(rotary_dim=128)):
        a = dict(num_heads=4, num_kv_heads=2, head_dim=64, max_seq_len=32, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError):
            PagedAttention(**a)
