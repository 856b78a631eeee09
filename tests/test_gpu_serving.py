"""Windows, shared prefixes and the 8-bit head together, as a serving program uses them: the layers of a model
over pages that are given away and used again, users behind one prompt, the greedy token of every row."""

import pytest
import torch

from paged_helpers import check_close, cu_of, dev, ints, normal
from window_helpers import attend_window64, seen

from bitnet_tt import paged_attention as pa
from bitnet_tt.config import BitNetMiniConfig
from bitnet_tt.decode import BitLinearDecodeStep
from bitnet_tt.int8_matmul import int8_matmul, quantize_rows
from bitnet_tt.layers.attention import PagedAttention
from bitnet_tt.lm_head import LMHead
from bitnet_tt.ternary_matmul import ternary_matmul

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(40, 3), (17, 0), (64, 20)])
def test_a_layer_with_a_window(dtype, window, sinks):
    """Two users: prompts, chunks and tokens against 64 bits over what the pages hold; prompt() too."""
    H, Hkv, D, page = 4, 2, 64, 16
    att = PagedAttention(H, Hkv, D, 256, dev(), window=window, sinks=sinks)
    cache = att.new_cache(32, page, dtype)
    table = torch.arange(32, dtype=torch.int32).view(2, 16).flip(1).contiguous().to(dev())
    length = [0, 0]
    for i, new in enumerate(([90, 20], [70, 1], [1, 1], [1, 64], [0, 1])):
        length = [a + b for a, b in zip(length, new)]
        qkv = normal((sum(new), (H + 2 * Hkv) * D), 50 + i).to(torch.bfloat16).to(dev())
        out = att(qkv, cache, table, cu_of(new), ints(length), max_q=max(new))
        att.check()
        k = torch.zeros((2, Hkv, 256, D), dtype=torch.bfloat16, device=dev())
        v = torch.zeros_like(k)
        pa.read_pages(cache, table, ints(length), k, v)
        q = pa.rope_write(qkv, att.rope_cos, att.rope_sin, cu_of(new), ints(length), H, Hkv).double().cpu()
        at = 0
        for b in range(2):
            n, m = new[b], length[b]
            want, tol = attend_window64(q[at:at + n], k[b, :, :m].double().cpu(), v[b, :, :m].double().cpu(), window, sinks)
            check_close(out[at:at + n].view(n, H, D), want, tol)
            at += n
        if i == 0:  # whole prompts; what 8 bits cost is not in prompt()
            o = att.prompt(qkv, cu_of(new))
            x = qkv.double().cpu().view(-1, H + 2 * Hkv, D)
            kr = torch.empty((sum(new), Hkv, D), dtype=torch.bfloat16, device=dev())
            pa.rope_write(qkv, att.rope_cos, att.rope_sin, cu_of(new), None, H, Hkv, k_out=kr)
            want, tol = attend_window64(q[:90], kr[:90].double().cpu().transpose(0, 1), x[:90, H + Hkv:].transpose(0, 1),
                                        window, sinks)
            check_close(o[:90].view(90, H, D), want, tol)


def test_pages_behind_the_window_are_used_again():
    """A user whose pages go back to a small pool as the window leaves them, against one that keeps all: the same bits."""
    cfg = BitNetMiniConfig()
    window, sinks, page = 40, 5, 16
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=1, num_layers=2)
    new = [30] + [1] * 40 + [25] + [1] * 10
    rows = [normal((n, cfg.hidden_size), 7 + i).to(torch.bfloat16).to(dev()) for i, n in enumerate(new)]

    def run(keep):
        step.alloc_paged(16 if keep else 7, 256, page_size=page, window=window, sinks=sinks)
        free, table, total, out = list(range(16 if keep else 7)), {}, 0, []
        for x in rows:
            total += x.shape[0]
            used = {j // page for p in range(total - x.shape[0], total) for j in seen(p, window, sinks)}
            if not keep:
                for i in [i for i in table if i not in used]:
                    free.append(table.pop(i))
            for i in sorted(used):
                if i not in table:
                    table[i] = free.pop(0)
            t = torch.full((1, 16), -1, dtype=torch.int32)
            for i, p in table.items():
                t[0, i] = p
            out.append(step.forward_rows(x.clone(), t.to(dev()), cu_of([x.shape[0]]), ints([total])))
        step.check()
        return out

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_users_behind_one_prompt(dtype):
    """A prompt cached once; users that go on from it, tokens and drafts, through the layers and the 8-bit head: each
    layer is the chain of the package's calls (bits), the attention that over each user's own whole table within both
    calls' bounds."""
    cfg = BitNetMiniConfig()
    H, Hkv, D, page = cfg.num_attention_heads, cfg.num_kv_heads, cfg.head_dim, 16
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=4, num_layers=2)
    step.alloc_paged(64, 256, page_size=page, dtype=dtype)
    prompt = normal((5 * page, cfg.hidden_size), 1).to(torch.bfloat16).to(dev())
    shared = torch.arange(5, dtype=torch.int32)
    table = torch.full((4, 16), -9, dtype=torch.int32)
    for b in range(4):
        table[b, 5:] = torch.arange(5 + 11 * b, 16 + 11 * b)
    whole = table.clone()
    whole[:, :5] = shared
    table[0, :5] = shared
    table, whole = table.to(dev()), whole.to(dev())
    step.forward_rows(prompt.clone(), whole[:1], cu_of([80]), ints([80]))
    head = LMHead(cfg.hidden_size, cfg.vocab_size, dev(), weight_dtype="int8")
    head.load_final_weights(torch.ones(cfg.hidden_size), normal((cfg.vocab_size, cfg.hidden_size), 2, 0.05))
    total = [80] * 4
    count = ints([5])
    for i, new in enumerate(([9, 1, 30, 2], [1, 1, 1, 1], [4, 4, 4, 4])):
        total = [a + b for a, b in zip(total, new)]
        x = normal((sum(new), cfg.hidden_size), 20 + i).to(torch.bfloat16).to(dev())
        pools = [[t.clone() for t in p._tensors if t is not None] for p in step.pages]
        h = x.clone()
        got = step.forward_rows(x, table, cu_of(new), ints(total), max_q=max(new), shared_pages=count, max_shared=5)
        step.check()
        for w, p in zip(step.layers, pools):
            cache = pa.PagedKVCache(*p)
            qkv = ternary_matmul(h, w.qkv, norm_weight=w.input_layernorm, norm_epsilon=step.eps)
            a = step.paged(qkv, cache, table, cu_of(new), ints(total), max_q=max(new), shared_pages=count, max_shared=5)
            b = step.paged(qkv, cache, whole, cu_of(new), ints(total), max_q=max(new))
            q = pa.rope_write(qkv, step.paged.rope_cos, step.paged.rope_sin, cu_of(new), ints(total), H, Hkv).double().cpu()
            k = torch.zeros((4, Hkv, 256, D), dtype=torch.bfloat16, device=dev())
            v = torch.zeros_like(k)
            pa.read_pages(cache, whole, ints(total), k, v)
            at = 0
            for u, n in enumerate(new):
                want, tol = attend_window64(q[at:at + n], k[u, :, :total[u]].double().cpu(), v[u, :, :total[u]].double().cpu())
                check_close(a[at:at + n].view(n, H, D), want, tol)
                check_close(b[at:at + n].view(n, H, D), want, tol)
                at += n
            h = ternary_matmul(a, w.o_proj, norm_weight=w.attn_sub_norm, norm_epsilon=step.eps, residual=h)
            f = ternary_matmul(h, w.gate_up, norm_weight=w.post_attention_layernorm, norm_epsilon=step.eps,
                               epilogue="relu2_mul")
            h = ternary_matmul(f, w.down, norm_weight=w.ffn_sub_norm, norm_epsilon=step.eps, residual=h)
        assert torch.equal(got, h)
        logits, tokens = head(got)
        codes, scales = quantize_rows(h, head.norm_weight, head.eps)
        assert torch.equal(logits, int8_matmul(codes, scales, head.weight, out_dtype=torch.float32))
        assert torch.equal(tokens.long(), logits.argmax(-1))


def test_a_step_of_all_in_a_graph():
    """Tokens of users behind one prompt and their greedy tokens, captured; lengths move on between replays."""
    cfg = BitNetMiniConfig()
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=3, num_layers=2)
    step.alloc_paged(40, 256, page_size=16)
    head = LMHead(cfg.hidden_size, cfg.vocab_size, dev(), weight_dtype="int8")
    head.load_final_weights(torch.ones(cfg.hidden_size), normal((cfg.vocab_size, cfg.hidden_size), 2, 0.05))
    table = torch.zeros((3, 13), dtype=torch.int32)
    table[:, 3:] = torch.arange(3, 33).view(3, 10)
    table[:, :3] = torch.arange(3)
    table = table.to(dev())
    step.forward_rows(normal((48, cfg.hidden_size), 1).to(torch.bfloat16).to(dev()), table[:1], cu_of([48]), ints([48]))
    x = torch.zeros((3, cfg.hidden_size), dtype=torch.bfloat16, device=dev())
    cu, lens, count = cu_of([1, 1, 1]), ints([49, 49, 49]), ints([3])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def call(h):
        step.forward_rows(h, table, cu, lens, max_q=1, shared_pages=count, max_shared=3)
        return head(h)

    with torch.cuda.stream(stream):
        call(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            logits, tokens = call(x)
    torch.cuda.synchronize()
    for i in range(4):
        rows = normal((3, cfg.hidden_size), 30 + i).to(torch.bfloat16).to(dev())
        lens.copy_(ints([49 + i, 49 + i, 49 + i]))
        before = [[t.clone() for t in p._tensors if t is not None] for p in step.pages]
        want = call(rows.clone())
        for p, b in zip(step.pages, before):
            for t, o in zip([t for t in p._tensors if t is not None], b):
                t.copy_(o)
        x.copy_(rows)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want[0]) and torch.equal(tokens, want[1])
    step.check()


def test_what_does_not_go_together():
    cfg = BitNetMiniConfig()
    step = BitLinearDecodeStep.random_init(cfg, dev(), seed=3, batch=1, num_layers=1)
    step.alloc_paged(8, 64, page_size=16, window=20)
    x = normal((1, cfg.hidden_size), 1).to(torch.bfloat16).to(dev())
    table = torch.arange(4, dtype=torch.int32, device=dev()).view(1, 4)
    with pytest.raises(ValueError, match="window"):
        step.forward_rows(x, table, cu_of([1]), ints([17]), shared_pages=ints([1]))
    with pytest.raises(ValueError, match="window"):
        PagedAttention(4, 2, 64, 64, dev(), window=0)
    with pytest.raises(ValueError, match="sinks"):
        PagedAttention(4, 2, 64, 64, dev(), sinks=3)
    step.kv = []  # (load_contiguous refuses before it reads any)
    with pytest.raises(ValueError, match="window"):
        step.load_contiguous(table, ints([17]))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pages_far_into_a_pool(kv):
    """Offsets that pass 32 bits: the same pages at the end of a large pool give the same bits."""
    page, Hkv, D, H = 64, 2, 128, 4
    each = Hkv * page * D * (2 if kv == "bf16" else 1)
    P = 2 ** 32 // each + 40
    n = 30  # pages of two users of one prefix
    small = pa.PagedKVCache.allocate(n, Hkv, D, dev(), page, kv)
    big = pa.PagedKVCache.allocate(P, Hkv, D, dev(), page, kv)
    for a, b in ((small.key_pages, big.key_pages), (small.value_pages, big.value_pages)):
        x = normal((n, Hkv, page, D), a.element_size() + (b is big.value_pages))
        a.copy_(x.to(a.dtype).to(dev()))
        b.view(torch.uint8)[P - n:] = a.view(torch.uint8)
    if kv == "fp8":
        for a, b in ((small.key_exp, big.key_exp), (small.value_exp, big.value_exp)):
            a.fill_(127)
            b[P - n:] = a
    table = torch.arange(n, dtype=torch.int32).view(2, -1)
    table[1, :4] = table[0, :4]
    len_, one = ints([900, 700]), ints([4])
    for rows in (1, 40):
        q = normal((2 * rows, H, D), 5).to(torch.bfloat16).to(dev())
        cu = ints([0, rows, 2 * rows])
        for call in (lambda c, t: pa.paged_attention(q, c, t, cu, len_, max_q=rows, window=500, sinks=70),
                     lambda c, t: pa.shared_prefix_attention(q, c, t, cu, len_, one, max_q=rows)):
            want = call(small, table.to(dev()))
            assert bool(torch.isfinite(want).all()) and float(want.abs().max()) > 0
            assert torch.equal(call(big, (table + (P - n)).to(dev())), want)
    pa.check("cuda:0")


def test_products_of_more_than_2_to_the_31_outputs():
    """Offsets of outputs that pass 32 bits: the last rows are those of a call of their own."""
    M, K, V = 17000, 32, 128256
    head = LMHead(K, V, dev(), weight_dtype="int8")
    head.load_final_weights(1 + 0.1 * normal((K,), 1), normal((V, K), 2))
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    logits, tokens = head(x)
    few, last = head(x[-40:])
    assert torch.equal(logits[-40:], few) and torch.equal(tokens[-40:], last)
    assert torch.equal(logits[:40], head(x[:40])[0])
