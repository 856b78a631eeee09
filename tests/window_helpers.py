"""References in 64 bits of attention within a window and of shared prefixes."""

import math

import torch

from paged_helpers import BF16_HALF, F32_HALF, PagedBatch


def seen(p, window=None, sinks=0):
    """Positions that the row at position p sees."""
    if p < 0:
        return []
    if window is None:
        return list(range(p + 1))
    lo = max(0, p - window + 1)
    return list(range(min(sinks, lo))) + list(range(lo, p + 1))


def attend_window64(q, k, v, window=None, sinks=0, scale=None, p_half=BF16_HALF):
    """As paged_helpers.attend64, with its bound, over the positions that a row sees: q [n, H, D],
    k and v [Hkv, m, D] in 64 bits, rows at positions m - n .. m - 1."""
    n, H, D = q.shape
    Hkv, m = k.shape[0], k.shape[1]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((n, H, D), dtype=torch.float64)
    tol = torch.zeros((n, H, D), dtype=torch.float64)
    for i in range(n):
        at = seen(m - n + i, window, sinks)
        if not at:
            continue
        ki, vi, qi = k[:, at], v[:, at], q[i].view(Hkv, G, D)
        w = torch.softmax(torch.matmul(qi, ki.transpose(1, 2)) * scale, -1)  # [Hkv, G, len]
        o = torch.matmul(w, vi)
        big = (torch.matmul(qi.abs(), ki.abs().transpose(1, 2)).amax(-1) * scale)[..., None]
        slack = 2 * (D + 4) * F32_HALF * big + (len(at) + 16) * F32_HALF
        if bool(torch.isfinite(o).all()):
            spread = torch.stack([torch.matmul(w[:, g, None], (vi - o[:, g, None]).abs())[:, 0] for g in range(G)], 1)
        else:
            spread = torch.matmul(w, vi.abs()) + o.abs()
        t = (p_half + 2 * slack) * (1 + 2 * p_half) * spread + (BF16_HALF + 2 * slack) * o.abs()
        out[i], tol[i] = o.reshape(H, D), t.reshape(H, D)
    return out, tol + 1e-30


class WindowBatch(PagedBatch):
    """A PagedBatch whose pages that no row sees are released: their table entries are no pages."""

    def __init__(self, new, total, H, Hkv, D, page, kv, window, sinks, release=True, **kw):
        super().__init__(new, total, H, Hkv, D, page, kv, **kw)
        self.window, self.sinks = window, sinks
        self.full_table = self.table_host.clone()
        if release:
            for b, (n, m) in enumerate(zip(new, total)):
                used = {j // page for i in range(max(0, m - n), m) for j in seen(i, window, sinks)}
                for i in range(self.table_host.shape[1]):
                    if i not in used:
                        self.table_host[b, i] = (-1, 2 ** 31 - 1, -2 ** 31)[i % 3]
            self.table = self.table_host.to(self.table.device)

    def rows(self, pool64, b):
        n = self.total[b]
        ids = self.full_table[b, : -(-n // self.page)].long()
        return pool64[ids].transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :n]

    def reference(self, scale=None):
        o, tol, at = [], [], 0
        for b, n in enumerate(self.new):
            x, t = attend_window64(self.q[at:at + n].double(), self.rows(self.k64, b), self.rows(self.v64, b),
                                   self.window, self.sinks, scale)
            o.append(x)
            tol.append(t)
            at += n
        return torch.cat(o), torch.cat(tol)


class SharedBatch(PagedBatch):
    """Sequences that begin with the same ``shared`` pages, then ``own`` positions each (the new ones among
    them); what the tables of all but the first sequence have for the shared pages is no page."""

    def __init__(self, new, own, shared, H, Hkv, D, page, kv, **kw):
        super().__init__([0] + list(new), [shared * page] + list(own), H, Hkv, D, page, kv, **kw)
        self.shared = shared
        both = self.table_host
        width = max(shared + max(-(-n // page) for n in own), 1)
        table = torch.full((len(new), width), -7, dtype=torch.int32)
        self.full_tables = []
        for b in range(len(new)):
            table[b, shared:] = both[b + 1, : width - shared]
            self.full_tables.append(torch.cat((both[0, :shared], both[b + 1])))
        table[0, :shared] = both[0, :shared]
        self.table_host = table
        self.new = list(new)
        self.total = [shared * page + n if n else 0 for n in own]  # an empty slot has no prefix either
        device = self.table.device
        self.table = table.to(device)
        self.cu, self.len = self.cu[1:], torch.tensor(self.total, dtype=torch.int32, device=device)
        self.pages = torch.tensor([shared], dtype=torch.int32, device=device)

    def rows(self, pool64, b):
        n = self.total[b]
        ids = self.full_tables[b][: -(-n // self.page)].long()
        return pool64[ids].transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :n]

    def reference(self, scale=None):
        o, tol, at = [], [], 0
        for b, n in enumerate(self.new):
            x, t = attend_window64(self.q[at:at + n].double(), self.rows(self.k64, b), self.rows(self.v64, b), scale=scale)
            o.append(x)
            tol.append(t)
            at += n
        return torch.cat(o), torch.cat(tol)
