"""The 8-bit head's tokens without logits in passes of any length on the GPU."""

import pytest
import torch

from paged_helpers import dev, normal
from test_gpu_int8_head import first_max, head_of

from bitnet_tt import lm_head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [65, 128, 200, 333])
@pytest.mark.parametrize("rows", [1, 64, 65, 100])
@pytest.mark.parametrize("K,V", [(64, 3001), (2592, 700)])
def test_passes(monkeypatch, M, rows, K, V):
    """Of 64 rows, which need no logits, and of more; the last one short."""
    head = head_of(K, V)
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    logits, want = head(x)
    assert want.tolist() == first_max(logits)
    monkeypatch.setattr(lm_head, "_BUFFER", 4 * V * rows)
    assert lm_head._pass_rows(M, V) == min(M, max(64, rows))
    normed = torch.zeros_like(x)
    none, tokens = head(x, return_logits=False, normed_out=normed)
    assert none is None and torch.equal(tokens, want)
    again = torch.zeros_like(x)
    head(x, normed_out=again)
    assert torch.equal(normed, again)


def test_a_pass_keeps_its_bound():
    """2^20 columns: 1024 rows of logits would be 4 GiB."""
    K, V, M = 32, 1 << 20, 1024
    head = lm_head.LMHead(K, V, dev(), weight_dtype="int8")
    w = torch.randn((V, K), generator=torch.Generator(device=dev()).manual_seed(1), device=dev())
    head.load_final_weights(torch.ones(K), w)
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    _, tokens = head(x, return_logits=False)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < (1 << 29) + (1 << 22)
    some = [0, 127, 128, 500, 1023]
    assert tokens[some].tolist() == head(x[some].contiguous())[1].tolist()
