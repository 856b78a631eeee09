"""Every form of the kernels of 8-bit products on the GPU, each on shapes that are asserted to take it: sums
exactly, scales as 32 bits round them."""

import pytest
import torch

from int8_helpers import CASES, plan
from paged_helpers import dev, normal
from test_gpu_int8_head import codes_of, first_max, head_of

from bitnet_tt import _native as N
from bitnet_tt.int8_matmul import Int8Weight, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu


def codes(shape, seed):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, device=dev(), dtype=torch.int8)


@pytest.mark.parametrize("tile,shape,halves", CASES)
def test_tiles(tile, shape, halves):
    M, K, Nf = shape
    assert plan(N.lib(), M, K, Nf) == (0, *tile, halves)
    a, w = codes((M, K), 1), codes((Nf, K), 2)
    sa = (normal((M,), 3).abs() * 0.02 + 1e-3).to(dev())
    sw = (normal((Nf,), 4) * 0.01).to(dev())
    acc = a.double() @ w.double().t()  # whole numbers below 2^53
    want = acc.float() * sa[:, None] * sw
    del acc
    weight = Int8Weight.from_codes(w, sw)
    for dtype in (torch.float32, torch.bfloat16):
        into = torch.full((M, Nf + 5), 3.0, dtype=dtype, device=dev())  # rows of any alignment
        int8_matmul(a, sa, weight, out=into[:, 2:2 + Nf])
        assert torch.equal(into[:, 2:2 + Nf], want.to(dtype))
        assert bool((into[:, :2] == 3.0).all()) and bool((into[:, 2 + Nf:] == 3.0).all())
        ld = (Nf + 15) // 8 * 8
        into = torch.full((M, ld), 3.0, dtype=dtype, device=dev())  # of 16 bytes
        int8_matmul(a, sa, weight, out=into[:, :Nf])
        assert torch.equal(into[:, :Nf], want.to(dtype)) and bool((into[:, Nf:] == 3.0).all())


@pytest.mark.parametrize("M", [1, 20, 33, 50, 64])
@pytest.mark.parametrize("K", [544, 1600, 2560])
def test_tokens_of_pairs_of_column_blocks(M, K):
    """The head's stream with rows in registers, up to four blocks of them, two column blocks at a time."""
    V = 33001
    head = head_of(K, V)
    x = normal((M, K), 3).to(torch.bfloat16).to(dev())
    logits, tokens = head(x)
    q, s = quantize_rows(x, head.norm_weight, 1e-5)
    acc = (q.double() @ codes_of(head.weight).t()).float()
    assert torch.equal(logits, acc * s[:, None] * head.weight.scale)
    assert tokens.tolist() == first_max(logits)
    assert torch.equal(head(x, return_logits=False)[1], tokens)
