"""Causal attention of packed prompts on the GPU against 64 bits."""

import math

import pytest
import torch

from paged_helpers import attend64, check_close, cu_of, dev, ints, normal

from bitnet_tt import paged_attention as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


def reference(q, k, v, lens, scale=None):
    o, tol, at = [], [], 0
    for n in lens:
        a, t = attend64(q[at:at + n].double(), k[at:at + n].double().transpose(0, 1), v[at:at + n].double().transpose(0, 1),
                        scale)
        o.append(a)
        tol.append(t)
        at += n
    return torch.cat(o), torch.cat(tol)


def packed(lens, H, Hkv, D, seed=0, extra=0):
    T = sum(lens) + extra
    x = normal((T, H + 2 * Hkv, D), seed, 1.2)
    x[sum(lens):] = math.nan  # rows of no sequence
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("H,Hkv,D", [(20, 5, 128), (4, 2, 64), (7, 1, 128), (2, 2, 64), (64, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [2], [31, 33], [64], [65], [0, 5, 0, 63, 1], [128, 1, 130], [200]])
def test_prompt(H, Hkv, D, lens):
    x = packed(lens, H, Hkv, D, extra=3)
    want, tol = reference(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], lens)
    d = x.to(dev())
    out = torch.full((x.shape[0], H, D), 4.0, dtype=torch.bfloat16, device=dev())
    got = pa.prompt_attention(d[:, :H], d[:, H:H + Hkv], d[:, H + Hkv:], cu_of(lens), out=out)
    assert got is out
    check_close(out[: sum(lens)], want, tol)
    assert bool((out[sum(lens):] == 4.0).all())


@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences(D):
    lens = [(31 * i) % 23 for i in range(150)]
    x = packed(lens, 4, 2, D, seed=3)
    want, tol = reference(x[:, :4], x[:, 4:6], x[:, 6:], lens)
    d = x.to(dev())
    check_close(pa.prompt_attention(d[:, :4], d[:, 4:6], d[:, 6:], cu_of(lens)), want, tol)


def test_long_prompt_rows():
    """Rows of a prompt of many steps, against 64 bits where they are cheap to have."""
    n, H, Hkv, D = 2500, 4, 2, 128
    x = packed([n], H, Hkv, D, seed=5)
    d = x.to(dev())
    out = pa.prompt_attention(d[:, :H], d[:, H:H + Hkv], d[:, H + Hkv:], cu_of([n]))
    for i in (0, 63, 64, 1000, 2047, 2048, 2499):
        want, tol = attend64(x[i:i + 1, :H].double(), x[: i + 1, H:H + Hkv].double().transpose(0, 1),
                             x[: i + 1, H + Hkv:].double().transpose(0, 1))
        check_close(out[i:i + 1], want, tol)


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
def test_scales_and_growing_scores(scale):
    """Maxima that grow from step to step (the running maximum is raised often) and
    that never do."""
    n, D = 300, 64
    q = normal((n, 1, D), 1).abs()
    k = normal((n, 1, D), 2).abs() * torch.linspace(0.01, 2.0, n)[:, None, None]
    v = normal((n, 1, D), 3)
    for order in (slice(None), torch.arange(n - 1, -1, -1)):
        x = [t.to(torch.bfloat16) for t in (q, k[order], v)]
        want, tol = reference(*x, [n], scale)
        check_close(pa.prompt_attention(*[t.to(dev()) for t in x], cu_of([n]), scale=scale), want, tol)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_values_not_finite_reach_only_rows_that_see_them(bad, D):
    lens = [70, 100, 40]
    x = packed(lens, 4, 2, D, seed=7)
    x[70 + 37, 6 + 1, 9] = bad  # a value
    x[70 + 90, 4, 3] = math.nan  # a key
    want, tol = reference(x[:, :4], x[:, 4:6], x[:, 6:], lens)
    d = x.to(dev())
    out = pa.prompt_attention(d[:, :4], d[:, 4:6], d[:, 6:], cu_of(lens))
    assert torch.isfinite(want[: 70 + 37]).all() and torch.isfinite(want[170:]).all()
    check_close(out, want, tol)


def test_a_row_of_infinite_scores_spoils_only_itself():
    x = packed([50], 2, 2, 64)
    x[20, 0] = math.nan
    want, tol = reference(x[:, :2], x[:, 2:4], x[:, 4:], [50])
    d = x.to(dev())
    check_close(pa.prompt_attention(d[:, :2], d[:, 2:4], d[:, 4:], cu_of([50])), want, tol)


def test_graph_replays():
    lens = [100, 29]
    x = packed(lens, 4, 2, 64).to(dev())
    cu = cu_of(lens)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu)
    torch.cuda.synchronize()
    for i, lens in enumerate(([100, 29], [1, 128], [129, 0], [60, 9])):
        x.copy_(packed([129], 4, 2, 64, seed=i))
        cu.copy_(cu_of(lens))
        out.fill_(1.0)
        want = torch.ones_like(out)
        pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu, out=want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("cu", [[0, 60, 20], [0, 10, 500], [-1, 10, 50]])
def test_sequences_not_well_formed(cu):
    x = packed([50], 4, 2, 64).to(dev())
    pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], ints(cu))
    with pytest.raises(RuntimeError, match="paged workspace"):
        pa.check("cuda:0")


@pytest.mark.parametrize("cu", [[0, 40, 60], [0, 49, 99], [0, 50, 2 ** 31 - 1], [-2 ** 31, 10, 50], [0, 20, 51]])
def test_offsets_behind_the_rows(cu):
    """The sequences as clamped, the error word set; the rows behind k and v, here another
    tensor's, are not read."""
    x = packed([50], 4, 2, 64, extra=60)  # NaN from row 50 on
    d = x.to(dev())
    out = pa.prompt_attention(d[:50, :4], d[:50, 4:6], d[:50, 6:], ints(cu))
    with pytest.raises(RuntimeError, match="paged workspace"):
        pa.check("cuda:0")
    at = [min(max(c, 0), 50) for c in cu]
    lens = [b - a for a, b in zip(at, at[1:])]
    want, tol = reference(x[:50, :4], x[:50, 4:6], x[:50, 6:], lens)
    check_close(out, want, tol)
