"""Products of 8-bit integers on the GPU: the sums exactly, the scales as 32 bits round them."""

import math

import pytest
import torch

from paged_helpers import dev, gen, normal

from bitnet_tt import _native as N
from bitnet_tt.int8_matmul import Int8Weight, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu


def codes(shape, seed):
    return torch.randint(-128, 128, shape, generator=gen(seed), dtype=torch.int8)


def case(M, K, Nf, seed=1, fill=None):
    a, w = codes((M, K), seed), codes((Nf, K), seed + 1)
    if fill is not None:
        a.fill_(fill[0])
        w.fill_(fill[1])
    sa = normal((M,), seed + 2).abs() * 0.02 + 1e-3
    sw = normal((Nf,), seed + 3) * 0.01
    return a, sa, w, sw


def want(a, sa, w, sw):
    """The sum in 64 bits (whole numbers below 2^53); then the roundings of 32 bits, in their order."""
    acc = (a.to(dev()).double() @ w.to(dev()).double().t()).cpu()
    return acc.float() * sa[:, None] * sw, acc * sa[:, None].double() * sw.double()


def check(a, sa, w, sw, **kw):
    y32, y64 = want(a, sa, w, sw)
    weight = Int8Weight.from_codes(w.to(dev()), sw.to(dev()))
    for dtype in (torch.float32, torch.bfloat16):
        got = int8_matmul(a.to(dev()), sa.to(dev()), weight, out_dtype=dtype).cpu()
        assert torch.equal(got, y32.to(dtype))
    # three roundings to 32 bits: the sum, and each scale
    assert bool(((y32.double() - y64).abs() <= 3.01 * 2.0 ** -24 * y64.abs()).all())


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 64])
@pytest.mark.parametrize("K,Nf", [(16, 1), (32, 15), (48, 16), (64, 17), (80, 33), (1040, 100), (2560, 129), (4112, 48)])
def test_few_rows(M, K, Nf):
    check(*case(M, K, Nf))


@pytest.mark.parametrize("M", [1, 16, 32, 50])
@pytest.mark.parametrize("K,Nf", [(64, 9000), (576, 20011), (2560, 8209)])
def test_few_rows_of_many_columns(M, K, Nf):
    """Several groups of columns a workgroup, the last of them short."""
    check(*case(M, K, Nf, seed=5))


@pytest.mark.parametrize("M", [1, 16, 32])
@pytest.mark.parametrize("K", [64, 592, 1600])
def test_few_rows_of_pairs_of_column_blocks(M, K):
    check(*case(M, K, 33001, seed=6))


@pytest.mark.parametrize("M", [1, 16, 17, 40])
@pytest.mark.parametrize("Nf", [4096, 4100])
def test_few_rows_that_do_not_stay_in_registers(M, Nf):
    check(*case(M, 2576, Nf, seed=7))


@pytest.mark.parametrize("M", [65, 100, 128, 129, 255, 256, 257, 400, 513])
@pytest.mark.parametrize("K,Nf", [(16, 3), (64, 64), (144, 255), (192, 257), (640, 130), (2560, 300)])
def test_many_rows(M, K, Nf):
    check(*case(M, K, Nf, seed=2))


@pytest.mark.parametrize("M,K,Nf", [(1000, 2560, 1000), (300, 6912, 520), (2000, 320, 3000), (96, 2560, 20000)])
def test_many_rows_of_many_columns(M, K, Nf):
    check(*case(M, K, Nf, seed=3))


@pytest.mark.parametrize("M", [1, 32, 300])
@pytest.mark.parametrize("fill", [(-128, -128), (127, 127), (-128, 127), (0, 5)])
def test_the_largest_sums(M, fill):
    """K = 16384: sums up to 2^28, rounded once on their way to 32-bit floats."""
    check(*case(M, 16384, 40, fill=fill))


@pytest.mark.parametrize("M", [5, 40, 200])
def test_strided_rows(M):
    K, Nf = 208, 77
    a, sa, w, sw = case(M, K, Nf)
    wide = torch.full((M, K + 64), 99, dtype=torch.int8, device=dev())
    wide[:, 32:32 + K] = a.to(dev())
    w_wide = torch.full((Nf, K + 16), 99, dtype=torch.int8, device=dev())
    w_wide[:, :K] = w.to(dev())
    weight = Int8Weight.from_codes(w_wide[:, :K], sw.to(dev()))
    y, _ = want(a, sa, w, sw)
    for dtype in (torch.float32, torch.bfloat16):
        into = torch.full((M, Nf + 6), 3.0, dtype=dtype, device=dev())  # rows of any alignment
        int8_matmul(wide[:, 32:32 + K], sa.to(dev()), weight, out=into[:, 3:3 + Nf])
        assert torch.equal(into[:, 3:3 + Nf].cpu(), y.to(dtype))
        assert bool((into[:, :3] == 3.0).all()) and bool((into[:, 3 + Nf:] == 3.0).all())
    odd = torch.empty(Nf * K + 8, dtype=torch.int8, device=dev())[8:].view(Nf, K)  # not 16-byte aligned: copied first
    odd.copy_(w.to(dev()))
    assert torch.equal(Int8Weight.from_codes(odd, sw.to(dev())).data, weight.data)


def test_any_shape_of_rows():
    a, sa, w, sw = case(12, 64, 40)
    weight = Int8Weight.from_codes(w.to(dev()), sw.to(dev()))
    y = int8_matmul(a.to(dev()), sa.to(dev()), weight)
    z = int8_matmul(a.to(dev()).view(3, 2, 2, 64), sa.to(dev()).view(3, 2, 2), weight)
    assert z.shape == (3, 2, 2, 40) and torch.equal(z.view(12, 40), y)
    one = int8_matmul(a[0].to(dev()), sa[0].to(dev()), weight)
    assert one.shape == (40,) and torch.equal(one, y[0])
    none = int8_matmul(a[:0].to(dev()), sa[:0].to(dev()), weight)
    assert none.shape == (0, 40)


def test_scales_that_are_not_finite():
    a, sa, w, sw = case(20, 64, 40)
    sa[3], sw[7], sw[9] = math.inf, math.nan, 0.0
    y32, _ = want(a, sa, w, sw)
    weight = Int8Weight.from_codes(w.to(dev()), sw.to(dev()))
    got = int8_matmul(a.to(dev()), sa.to(dev()), weight, out_dtype=torch.float32).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(y32))
    assert torch.equal(got.nan_to_num(), y32.nan_to_num())


def unlaid(weight):
    """Codes [N, K] of a device layout."""
    n, k = weight.out_features, weight.in_features
    x = weight.data.view(torch.int8).cpu().view(-(-n // 16), -(-k // 64), 4, 16, 16)  # block, block, k / 16, column, k % 16
    full = x.permute(0, 3, 1, 2, 4).reshape(-(-n // 16) * 16, -(-k // 64) * 64)
    assert not bool(full[n:].any()) and not bool(full[:, k:].any())
    return full[:n, :k]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Nf,K", [(1, 16), (17, 80), (130, 2560), (16, 64)])
def test_quantised_weights(dtype, Nf, K):
    w = normal((Nf, K), 4, 0.02).to(dtype)
    w[0, 3] = 0.0
    got = Int8Weight.quantize(w.to(dev()))
    scale = w.float().abs().amax(1) / 127.0
    assert torch.equal(got.scale.cpu(), scale)
    q = unlaid(got)
    assert torch.equal(q, torch.round(w.float() / scale[:, None]).to(torch.int8))
    # half a step of the scale, and the quotient's own rounding of up to 127 steps
    off = (q.double() * scale.double()[:, None] - w.double()).abs()
    assert bool((off <= scale.double()[:, None] * (0.5 + 127 * 2.0 ** -23)).all())


def test_rows_of_weights_that_are_extreme():
    w = torch.zeros(6, 32)
    w[1] = 3e38
    w[2, 5] = 1e-40
    w[3, 5] = math.inf
    w[4, 7] = math.nan
    w[5] = torch.linspace(-1e-30, 1e-30, 32)
    got = Int8Weight.quantize(w.to(dev()))
    s, q = got.scale.cpu(), unlaid(got)
    assert s[0] == 1 and not bool(q[0].any())
    assert bool((q[1] == 127).all()) and float(s[1]) == float(torch.tensor(3e38) / 127)
    assert s[2] == 1 and not bool(q[2].any())
    assert bool(torch.isnan(s[3:5]).all()) and not bool(q[3:5].any())
    assert int(q[5, 0]) == -127 and int(q[5, -1]) == 127


@pytest.mark.parametrize("norm", [False, True])
def test_quantised_rows(norm):
    """The codes and scales of the ternary layers."""
    x = normal((5, 7, 96), 4).to(torch.bfloat16).to(dev())
    g = (1 + 0.1 * normal((96,), 5)).to(torch.bfloat16).to(dev()) if norm else None
    q, s = quantize_rows(x, g, 1e-5 if norm else None)
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    y = x.reshape(-1, 96)
    if norm:
        out = torch.empty_like(y)
        N.check(N.lib().btl_rmsnorm(y.data_ptr(), 35, 96, 96, g.data_ptr(), 1e-5, out.data_ptr(), N.raw_stream(0)), "norm")
        y = out
    y, big = y.float().cpu(), y.float().abs().amax(1).clamp(min=1e-5).cpu()
    assert torch.equal(s.view(-1).cpu(), big / 127)
    inverse = torch.full_like(big, 127.0) / big  # a quotient (of a number and a tensor torch takes a reciprocal's product)
    assert torch.equal(q.view(-1, 96).cpu(), torch.clamp(torch.round(y * inverse[:, None]), -128, 127).to(torch.int8))
    none, _ = quantize_rows(x[:0])
    assert none.shape == (0, 7, 96)


def test_captured_and_on_another_stream():
    a, sa, w, sw = case(48, 576, 500)
    weight = Int8Weight.from_codes(w.to(dev()), sw.to(dev()))
    da, dsa = a.to(dev()), sa.to(dev())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = int8_matmul(da, dsa, weight, out_dtype=torch.float32)
    for seed in (8, 9, 10):
        a = codes((48, 576), seed)
        da.copy_(a)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, int8_matmul(da, dsa, weight, out_dtype=torch.float32))
        assert torch.equal(out.cpu(), want(a, sa, w, sw)[0])
