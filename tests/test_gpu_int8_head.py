"""The 8-bit LM head on the GPU: logits exactly the product of the quantised rows and weights, tokens the
first index of each row's largest logit."""

import math

import numpy as np
import pytest
import torch

from paged_helpers import dev, gen, normal

from bitnet_tt.int8_matmul import int8_matmul, quantize_rows
from bitnet_tt.lm_head import LMHead

pytestmark = pytest.mark.gpu


def head_of(K, V, seed=1, w=None):
    head = LMHead(K, V, dev(), eps=1e-5, weight_dtype="int8")
    g = 1 + 0.1 * normal((K,), seed)
    head.load_final_weights(g, normal((V, K), seed + 1, 0.05) if w is None else w)
    return head


def codes_of(weight):
    """The codes of the device layout, in 64 bits: blocks of 16 columns x 64 k, a lane's 16 bytes of column lane % 16."""
    n, k = weight.out_features, weight.in_features
    w = weight.data.view(torch.int8).view(-(-n // 16), -(-k // 64), 4, 16, 16).permute(0, 3, 1, 2, 4)
    return w.reshape(-(-n // 16) * 16, -1)[:n, :k].double()


def first_max(logits):
    """The first index of each row's largest number; -1: none is one."""
    x = logits.double().cpu().numpy()
    out = []
    for row in x:
        ok = ~np.isnan(row)
        out.append(int(np.flatnonzero(ok & (row == row[ok].max()))[0]) if ok.any() else -1)
    return out


@pytest.mark.parametrize("M", [1, 3, 16, 17, 32, 50, 64, 65, 130, 1100])
@pytest.mark.parametrize("K,V", [(32, 1), (64, 37), (256, 1000), (2560, 5003)])
def test_logits_and_tokens(M, K, V):
    head = head_of(K, V)
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    normed = torch.empty_like(x)
    logits, tokens = head(x, normed_out=normed)
    q, s = quantize_rows(x, head.norm_weight, 1e-5)
    assert torch.equal(logits, int8_matmul(q, s, head.weight, out_dtype=torch.float32))
    assert tokens.tolist() == first_max(logits)
    q2, s2 = quantize_rows(normed)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    none, again = head(x, return_logits=False)
    assert none is None and torch.equal(again, tokens)


@pytest.mark.parametrize("M", [2, 16, 17, 40, 64])
@pytest.mark.parametrize("K,V", [(64, 33001), (576, 33001), (2592, 3001), (2592, 33001)])
def test_tokens_of_few_rows_by_either_way(M, K, V):
    """With and without logits, pairs of column blocks, rows that stay in registers and rows that do not."""
    head = head_of(K, V)
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    logits, tokens = head(x)
    q, s = quantize_rows(x, head.norm_weight, 1e-5)
    acc = (q.double() @ codes_of(head.weight).t()).float()  # whole numbers below 2^53
    assert torch.equal(logits, acc * s[:, None] * head.weight.scale)
    assert tokens.tolist() == first_max(logits)
    assert torch.equal(head(x, return_logits=False)[1], tokens)


@pytest.mark.parametrize("M", [1023, 1024, 1025, 1090, 2047, 2112])
def test_many_rows_without_logits(M):
    """Passes over the rows that share a buffer, the last one short."""
    head = head_of(32, 9000)
    x = normal((M, 32), 3).to(torch.bfloat16).to(dev())
    normed = torch.zeros_like(x)
    _, tokens = head(x, return_logits=False, normed_out=normed)
    all_normed = torch.zeros_like(x)
    logits, want = head(x, normed_out=all_normed)
    assert torch.equal(tokens, want) and torch.equal(normed, all_normed)
    assert tokens.tolist() == first_max(logits)


@pytest.mark.parametrize("M", [2, 100])
def test_near_the_float_head(M):
    """Against the weights in 64 bits: half a step of either operand's scale, summed over K."""
    K, V = 512, 3000
    w = normal((V, K), 5, 0.05)
    head = head_of(K, V, w=w)
    x = normal((M, K), 6).to(torch.bfloat16).to(dev())
    normed = torch.empty_like(x)
    logits, _ = head(x, normed_out=normed)
    y, wd = normed.double().cpu(), w.double()
    half_x, half_w = y.abs().amax(1) / 254, wd.abs().amax(1) / 254
    bound = (half_x[:, None] * wd.abs().sum(1) + half_w * y.abs().sum(1)[:, None] + K * half_x[:, None] * half_w) * 1.001
    assert bool(((logits.double().cpu() - y @ wd.t()).abs() <= bound).all())


@pytest.mark.parametrize("M", [2, 33, 70])
def test_ties_take_the_first_index(M):
    K, V = 256, 9000
    w = normal((V, K), 7, 0.01)
    x = normal((M, K), 8)
    w[5] = w[700] = w[8999] = x[0].sign() * 0.5
    x[1] = 0.0
    head = head_of(K, V, w=w)
    logits, tokens = head(x.to(torch.bfloat16).to(dev()))
    assert logits[0, 5] == logits[0, 700] == logits[0, 8999]
    assert int(tokens[0]) == 5 and int(tokens[1]) == 0
    assert tokens.tolist() == first_max(logits)


@pytest.mark.parametrize("M", [2, 70])
def test_columns_that_are_not_numbers(M):
    """A weight row with a NaN gives NaN logits, which are never a token; a row of x that is all NaN has none."""
    K, V = 64, 300
    w = normal((V, K), 9)
    w[0, 3] = math.nan
    w[77, 0] = math.inf
    head = head_of(K, V, w=w)
    x = normal((M, K), 10)
    logits, tokens = head(x.to(torch.bfloat16).to(dev()))
    assert bool(torch.isnan(logits[:, 0]).all()) and bool(torch.isnan(logits[:, 77]).all())
    assert tokens.tolist() == first_max(logits)
    head.weight.scale.fill_(math.nan)
    _, tokens = head(x.to(torch.bfloat16).to(dev()))
    assert tokens.tolist() == [-1] * M
    head.weight.scale.fill_(-math.inf)
    logits, tokens = head(x.to(torch.bfloat16).to(dev()))
    assert tokens.tolist() == first_max(logits)


def test_two_graphs_at_once():
    """Captured on one stream, replayed on two: each call has its own scratch.  Eager calls between."""
    K, V = 512, 5000
    head = head_of(K, V)
    runs = []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for M in (32, 31, 200, 199):
            x = normal((M, K), 20 + M).to(torch.bfloat16).to(dev())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = head(x)
            runs.append((x, g, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    want = [head(x) for x, _, _, _ in runs]
    for _ in range(4):
        for _, _, (logits, tokens), _ in runs:
            logits.fill_(-7)
            tokens.fill_(-7)
        torch.cuda.synchronize()
        for _, g, _, s in runs:
            with torch.cuda.stream(s):
                g.replay()
        again = head(runs[0][0])
        torch.cuda.synchronize()
        assert torch.equal(again[1], want[0][1])
        for (_, _, (logits, tokens), _), (l, t) in zip(runs, want):
            assert torch.equal(logits, l) and torch.equal(tokens, t)


def test_full_vocabulary():
    """The 2B model's head."""
    K, V = 2560, 128256
    w = torch.randn((V, K), generator=torch.Generator(device=dev()).manual_seed(1), device=dev(), dtype=torch.bfloat16) * 0.02
    head = LMHead(K, V, dev(), weight_dtype="int8")
    head.load_final_weights(torch.ones(K), w)
    assert head.weight_bytes() == V * (K + 4)
    for M in (1, 32, 96):
        x = normal((M, K), M).to(torch.bfloat16).to(dev())
        logits, tokens = head(x)
        assert tokens.tolist() == first_max(logits)
        cols = torch.randint(0, V, (300,), generator=gen(5)).to(dev())
        q, s = quantize_rows(x, head.norm_weight, 1e-5)
        codes = torch.round(w[cols].float() / head.weight.scale[cols][:, None]).double()
        acc = q.double() @ codes.t()
        assert torch.equal(logits[:, cols], acc.float() * s[:, None] * head.weight.scale[cols])


def test_refusals():
    with pytest.raises(ValueError, match="weight_dtype"):
        LMHead(64, 10, dev(), weight_dtype="fp8")
    with pytest.raises(ValueError, match="multiples of 32"):
        LMHead(48, 10, dev(), weight_dtype="int8")
    head = LMHead(64, 10, dev(), weight_dtype="int8")
    x = normal((4, 64), 3).to(torch.bfloat16).to(dev())
    with pytest.raises(RuntimeError, match="load_final_weights"):
        head(x)
    head.load_final_weights(torch.ones(64), normal((10, 64), 1))
    with pytest.raises(ValueError, match="hidden"):
        head(x.float())
    with pytest.raises(ValueError, match="logits_out"):
        head(x, logits_out=torch.empty((4, 9), device=dev()))
    with pytest.raises(ValueError, match="tokens_out"):
        head(x, tokens_out=torch.empty(4, dtype=torch.int64, device=dev()))
