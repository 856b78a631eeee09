"""Batches over pages and references in 64 bits for the tests of prompts and
of the paged cache."""

import math

import numpy as np
import torch

BF16_HALF = torch.finfo(torch.bfloat16).eps / 2  # 2^-8
F32_HALF = torch.finfo(torch.float32).eps / 2  # 2^-24
E4M3_HALF = torch.finfo(torch.float8_e4m3fn).eps / 2  # 2^-4


def dev():
    return torch.device("cuda:0")


def cu_of(lens, device=None):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=device or dev())


def ints(values, device=None):
    return torch.tensor(values, dtype=torch.int32, device=device or dev())


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(shape, seed, std=1.0):
    return torch.randn(shape, generator=gen(seed), dtype=torch.float32) * std


def quantise(x):
    """(codes as float8, exponent bytes) of rows [..., D] fp32, the plain form."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    bad = ~torch.isfinite(x).all(-1)
    raw = codes.view(torch.uint8).clone()
    raw[bad] = 0x7F
    e = torch.where(bad, torch.zeros_like(e), e)
    return raw.view(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def values_of(codes, exps):
    """What codes with exponent bytes stand for, in 64 bits."""
    return codes.float().double() * torch.exp2(exps.double() - 127)[..., None]


class PagedBatch:
    """Sequences of ``past + new`` positions with random keys and values in
    scattered pages (spare pages, and every row that holds no position, are
    NaN), and what the pages hold in 64 bits: k, v lists of [Hkv, len, D]."""

    def __init__(self, new, total, H, Hkv, D, page, kv, seed=0, spare=3, extra_pages=0, std=1.0):
        from bitnet_tt.paged_attention import PagedKVCache

        self.new, self.total, self.H, self.Hkv, self.D = list(new), list(total), H, Hkv, D
        self.page, self.kv = page, kv
        B = len(new)
        T = sum(new)
        need = [-(-n // page) for n in total]
        P = sum(need) + spare
        order = torch.randperm(P, generator=gen(seed + 1)).tolist()
        width = max(1, max(need)) + extra_pages
        table = torch.full((B, width), -7, dtype=torch.int32)  # entries that no position needs are no pages
        k = torch.full((P, Hkv, page, D), math.nan)
        v = torch.full((P, Hkv, page, D), math.nan)
        at = 0
        for b in range(B):
            for i in range(need[b]):
                table[b, i] = order[at]
                rows = min(page, total[b] - i * page)
                k[order[at], :, :rows] = normal((Hkv, rows, D), seed * 1000 + 17 * at + 3, std)
                v[order[at], :, :rows] = normal((Hkv, rows, D), seed * 1000 + 17 * at + 5)
                at += 1
        self.table_host = table
        if kv == "bf16":
            kq, vq = k.to(torch.bfloat16), v.to(torch.bfloat16)
            self.k64, self.v64 = kq.double(), vq.double()
            self.cache = PagedKVCache(kq.to(dev()), vq.to(dev()))
        else:
            kq, ke = quantise(k)
            vq, ve = quantise(v)
            self.k64, self.v64 = values_of(kq, ke), values_of(vq, ve)
            self.cache = PagedKVCache(kq.to(dev()), vq.to(dev()), ke.to(dev()), ve.to(dev()))
        self.table = table.to(dev())
        self.cu, self.len = cu_of(new), ints(total)
        self.q = normal((T, H, D), seed + 9, 1.5).to(torch.bfloat16)
        self.q_dev = self.q.to(dev())

    def rows(self, pool64, b):
        """[Hkv, total_b, D]"""
        n = self.total[b]
        ids = self.table_host[b, : -(-n // self.page)].long()
        return pool64[ids].transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :n]

    def reference(self, scale=None):
        o, tol = [], []
        at = 0
        for b, n in enumerate(self.new):
            x, t = attend64(self.q[at:at + n].double(), self.rows(self.k64, b), self.rows(self.v64, b), scale)
            o.append(x)
            tol.append(t)
            at += n
        return torch.cat(o), torch.cat(tol)


def attend64(q, k, v, scale=None, p_half=BF16_HALF):
    """q [n, H, D], k and v [Hkv, m, D] in 64 bits: rows at positions m - n ..
    m - 1 (negative: zeros).  Returns the output and how far a kernel may be from it.

    A kernel's weights are p_j (1 + d_j), the same in the product and in the sum that
    it is divided by, so with o = sum p v / sum p its output is off by
    sum p_j d_j (v_j - o) / sum p_j (1 + d_j).  |d_j| is p_half, half a step of bf16 (the
    operands of the second product; of two bf16 values that make up p the square of that), and
    what 32 bits make of scores, exponentials and sums; the denominator is within twice p_half
    of sum p.  The result is rounded to bf16 once more."""
    n, H, D = q.shape
    Hkv, m = k.shape[0], k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((n, H, D), dtype=torch.float64)
    tol = torch.zeros((n, H, D), dtype=torch.float64)
    for i in range(n):
        p = m - n + i
        if p < 0:
            continue
        for h in range(H):
            kh, vh = k[h // (H // Hkv), : p + 1], v[h // (H // Hkv), : p + 1]
            s = (kh @ q[i, h]) * scale
            w = torch.softmax(s, 0)
            out[i, h] = w @ vh
            big = float((kh.abs() @ q[i, h].abs()).max()) * scale
            # a score is D products and sums, then a scaling, and 2^x to about a step: each relative
            # 2^-24 of at most `big` (x 2: against the maximum's own error); L a sum of p + 1 terms
            slack = 2 * (D + 4) * F32_HALF * big + (p + 16) * F32_HALF
            spread = w @ (vh - out[i, h]).abs() if torch.isfinite(out[i, h]).all() else w @ vh.abs() + out[i, h].abs()
            tol[i, h] = (p_half + 2 * slack) * (1 + 2 * p_half) * spread + (BF16_HALF + 2 * slack) * out[i, h].abs()
    return out, tol + 1e-30


def check_close(got, want, tol):
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{int((off > 0).sum())} of {off.numel()} beyond, by {float(off.max()):.3g}"
