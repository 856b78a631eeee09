"""Windowed calls of so many tiles that neighbours run on one XCD, 2, 4 or 8 of them, on shapes that are asserted
to do so: packed prompts, and chunks over pages."""

import ctypes

import pytest
import torch

from paged_helpers import BF16_HALF, F32_HALF, check_close, cu_of, dev, normal
from window_helpers import WindowBatch

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    pa.check("cuda:0")


def neighbours(new, H, Hkv):
    """The tiles of the call (of 128 rows; a sequence may have one that is not full), and how many are neighbours."""
    T, B = sum(new), len(new)
    tiles = (T * (H // Hkv) // 128 + min(B, T)) * Hkv
    out = (ctypes.c_int64 * 3)()
    assert N.lib().btl_attention_window_tile(tiles, 1, Hkv, 0, out) > 0
    return tiles, out[0]


def attend(q, k, v, window, sinks):
    """As window_helpers.attend_window64, with all rows at once on the GPU, and a wider bound: q [n, H, D], k and v [Hkv, m, D] in
    64 bits.  The output is off by sum w d (v - o) / ..., |d| <= half a step of bf16 and what 32 bits make of scores and
    sums; |v - o| <= |v| + |o|."""
    n, H, D = q.shape
    Hkv, m = k.shape[:2]
    G = H // Hkv
    p, j = torch.arange(m - n, m, device=q.device)[:, None], torch.arange(m, device=q.device)[None]
    see = (j <= p) & ((j > p - window) | (j < sinks))
    x = q.transpose(0, 1).reshape(Hkv, G * n, D)
    s = torch.matmul(x, k.transpose(1, 2).contiguous()).view(Hkv, G, n, m) / D ** 0.5
    big = torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()).amax(-1).view(Hkv, G, n, 1) / D ** 0.5
    w = torch.softmax(s.masked_fill(~see, -torch.inf), -1).view(Hkv, G * n, m)
    o = torch.matmul(w, v).view(Hkv, G, n, D)
    spread = torch.matmul(w, v.abs()).view(Hkv, G, n, D) + o.abs()
    slack = 2 * (D + 4) * F32_HALF * big + (m + 16) * F32_HALF
    tol = (BF16_HALF + 2 * slack) * (1 + 2 * BF16_HALF) * spread + (BF16_HALF + 2 * slack) * o.abs() + 1e-30
    return [y.reshape(H, n, D).transpose(0, 1).cpu() for y in (o, tol)]


# sequences, heads: 2, 4 and 8 neighbours, for 1, 2 and 5 key-value heads; the tiles of a head are no multiple of them
SHAPES = [
    (2, [400, 1, 0, 245], 64, 1), (2, [333, 320], 64, 2), (2, [100, 425, 3], 80, 5),
    (4, [700, 1, 0, 591], 64, 1), (4, [640, 655], 64, 2), (4, [500, 532, 13], 80, 5),
    (8, [900, 1, 0, 800, 871], 64, 1), (8, [655, 640, 1279], 64, 2), (8, [700, 20, 1340], 80, 5), (8, [7] * 40, 40, 40),
]


@pytest.mark.parametrize("each,lens,H,Hkv", SHAPES)
@pytest.mark.parametrize("window,sinks", [(100, 4), (300, 0)])
def test_prompts(each, lens, H, Hkv, window, sinks):
    D = 64
    tiles, got_each = neighbours(lens, H, Hkv)
    assert got_each == each and tiles // Hkv % each
    assert window < sum(lens) or len(lens) == 40  # (of the 40 short ones a window of 300 is none)
    x = normal((sum(lens), H + 2 * Hkv, D), 1, 1.4).to(torch.bfloat16).to(dev())
    out = torch.full((sum(lens), H, D), 7.0, dtype=torch.bfloat16, device=dev())
    pa.prompt_attention(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], cu_of(lens), out=out, window=window, sinks=sinks)
    at = 0
    for n in lens:
        if n:
            y = x[at:at + n].double()
            k, v = (t.transpose(0, 1).contiguous() for t in (y[:, H:H + Hkv], y[:, H + Hkv:]))
            check_close(out[at:at + n], *attend(y[:, :H], k, v, window, sinks))
        at += n


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("each,new,H,Hkv", SHAPES[:9])
def test_chunks_over_pages(kv, each, new, H, Hkv):
    D, window, sinks = 64, 150, 20
    tiles, got_each = neighbours(new, H, Hkv)
    assert got_each == each and tiles // Hkv % each
    total = [n + 91 * i for i, n in enumerate(new)]
    wb = WindowBatch(new, total, H, Hkv, D, 48, kv, window, sinks)
    plan = (ctypes.c_int64 * 3)()
    assert N.lib().btl_paged_attention_window_plan(sum(new), H, Hkv, D, len(new), max(new), max(total), window, sinks, plan) == 1
    assert tuple(plan)[:2] == (0, 1)  # tiles, no splits
    out = torch.full((sum(new), H, D), 7.0, dtype=torch.bfloat16, device=dev())
    pa.paged_attention(wb.q_dev, wb.cache, wb.table, wb.cu, wb.len, max_q=max(new), max_kv=max(total), out=out, window=window,
                       sinks=sinks)
    at = 0
    for b, n in enumerate(new):
        if n:
            k, v = (wb.rows(pool, b).to(dev()).contiguous() for pool in (wb.k64, wb.v64))
            check_close(out[at:at + n], *attend(wb.q_dev[at:at + n].double(), k, v, window, sinks))
        at += n
