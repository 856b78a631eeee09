"""What a decode step reads beside the ternary weights, as measurable cases:
cached positions of which a row sees a window only, cached positions that a batch
shares, and an 8-bit head.

A case is a dict of plain values; ``prepare`` makes what a serving program holds
before the call (a batch's projections, page pools and page tables, laid-out
weights), ``run`` is one pass through an operator: its plain form, or the package's
entry point where ``own`` is set.  ``exact`` is the same result in 64 bits.  Heads are
those of the BitNet b1.58 2B model (20 query and 5 key-value heads of 128, hidden
2560, feed-forward 6912, vocabulary 128256) and of the small test model (4 and 2 of 64).

Operators:
  win_prompt  causal attention within packed sequences over the last ``window``
              positions and the first ``sinks`` ones
  win_paged   the same of the newest tokens of each sequence over its pages
  prefix      attention of the newest tokens of a batch whose first positions are
              in the same pages
  int8        a matrix product of 8-bit integers, a scale for each row and each column
"""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitnet-tt_amd")

BIG = {"heads": 20, "kv_heads": 5, "dim": 128}  # the 2B model
MINI = {"heads": 4, "kv_heads": 2, "dim": 64}  # the small model of the tests


def listed():
    return [
        # short prompts of several users in one batch, a short window
        {"name": "win_prompt_short", "op": "win_prompt", **MINI, "seqs": 9, "tokens": 1003, "window": 64, "sinks": 4},
        # documents of different lengths, packed
        {"name": "win_prompt_16k", "op": "win_prompt", **BIG, "seqs": 4, "tokens": 16001, "window": 1024, "sinks": 4},
        # one decode step's attention of 32 users, ragged contexts, 8-bit cache
        {"name": "win_decode_b32_fp8", "op": "win_paged", **BIG, "kv": "fp8", "page": 64, "seqs": 32, "tokens": 32,
         "past": 8000, "window": 1024, "sinks": 4},
        # one user far into a long conversation: latency of a single stream
        {"name": "win_decode_b1_far", "op": "win_paged", **BIG, "kv": "bf16", "page": 16, "seqs": 1, "tokens": 1,
         "past": 131000, "window": 4096, "sinks": 20},
        # chunked prompts of four users over what is cached already, no sinks
        {"name": "win_chunk_b4", "op": "win_paged", **BIG, "kv": "bf16", "page": 64, "seqs": 4, "tokens": 2047,
         "past": 8000, "window": 2000, "sinks": 0},
        # three users of the small model behind a short system prompt: the smallest call
        {"name": "prefix_decode_b3", "op": "prefix", **MINI, "kv": "bf16", "page": 16, "seqs": 3, "tokens": 3,
         "shared": 480, "past": 37},
        # 32 users of one system prompt with documents
        {"name": "prefix_decode_b32", "op": "prefix", **BIG, "kv": "bf16", "page": 64, "seqs": 32, "tokens": 32,
         "shared": 8192, "past": 500},
        # many answers over one long document, 8-bit cache
        {"name": "prefix_decode_b64_fp8", "op": "prefix", **BIG, "kv": "fp8", "page": 128, "seqs": 64, "tokens": 64,
         "shared": 65536, "past": 2000},
        # drafts of a few tokens checked for 16 users at once
        {"name": "prefix_draft_b16", "op": "prefix", **BIG, "kv": "bf16", "page": 32, "seqs": 16, "tokens": 81,
         "shared": 16000, "past": 1000},
        # the head of a decode step of 32 users
        {"name": "int8_head_b32", "op": "int8", "rows": 32, "inner": 2560, "cols": 128256, "out": "fp32"},
        # a projection of a short prompt
        {"name": "int8_proj_511", "op": "int8", "rows": 511, "inner": 2560, "cols": 3840, "out": "bf16"},
        # the feed-forward's two projections of a long one
        {"name": "int8_ffn_4096", "op": "int8", "rows": 4096, "inner": 2560, "cols": 13824, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["win_prompt", "win_paged", "win_paged", "prefix", "prefix", "int8", "int8"])
    if op == "int8":
        c = {"op": op, "rows": 1 if rng.random() < 0.15 else _log(rng, 2, 4096), "inner": 16 * _log(rng, 4, 432),
             "out": rng.choice(["bf16", "fp32"])}
        # no more work than the largest listed case
        most = min(128256, 4096 * 2560 * 13824 // (c["rows"] * c["inner"]), 2560 * 128256 // c["inner"],
                   2 ** 26 // c["rows"])
        return {**c, "cols": _log(rng, 64, most)}
    c = {"op": op, **(BIG if rng.random() < 0.7 else MINI)}
    if op != "win_prompt":
        c["kv"] = rng.choice(["bf16", "fp8"])
        c["page"] = rng.choice([16, 32, 48, 64, 128, 256])
    if op != "prefix":
        c["window"] = _log(rng, 1, 8000)
        c["sinks"] = rng.choice([0, 1, 4, 4, 16, 64, 100, 300])
    if op == "win_prompt":
        c["seqs"] = _log(rng, 1, 32)
        c["tokens"] = max(c["seqs"], _log(rng, 1, 12000))
    elif op == "win_paged":
        if rng.random() < 0.6:
            c["seqs"] = _log(rng, 1, 64)
            c["tokens"] = c["seqs"]
            c["past"] = _log(rng, 1, 120000 // c["seqs"])
        else:
            c["seqs"] = _log(rng, 1, 8)
            c["tokens"] = c["seqs"] + _log(rng, 1, 2000)
            c["past"] = _log(rng, 1, 60000 // c["seqs"])
    else:
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = c["seqs"] * (1 if rng.random() < 0.6 else _log(rng, 2, 16))
        c["shared"] = c["page"] * max(1, _log(rng, 16, min(65536, 64 * 65536 // c["tokens"])) // c["page"])
        c["past"] = _log(rng, 1, 2000)
    return c


def _counts(total, n):
    """n ragged counts of at least one with this sum."""
    if n == 1 or total == n:
        return [1] * n if total == n else [total]
    r = random.Random(total * 131 + n)
    w = [r.uniform(0.2, 1.8) for _ in range(n)]
    c = [1 + int((total - n) * x / sum(w)) for x in w]
    c[0] += total - sum(c)
    return c


def _pasts(past, n):
    """n ragged context lengths, the first of them ``past``."""
    r = random.Random(past * 137 + n)
    return [past] + [r.randint(past // 4, past) for _ in range(n - 1)]


def _sizes(case):
    """(new tokens, total positions) of each sequence."""
    new = _counts(case["tokens"], case["seqs"])
    past = _pasts(case["past"], case["seqs"]) if "past" in case else [0] * case["seqs"]
    return new, [case.get("shared", 0) + a + b for a, b in zip(new, past)]


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _cu(counts, dev):
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    return _ints(cu, dev)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 7919 + 13)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    if case["op"] == "int8":
        M, K, N = case["rows"], case["inner"], case["cols"]
        # rows quantised by their largest value: codes of a normal distribution, every scale its own
        a = (normal(M, K) * 35).round_().clamp_(-127, 127).to(torch.int8)
        w = torch.empty((N, K), dtype=torch.int8, device=dev)
        for lo in range(0, N, 16384):
            w[lo:lo + 16384] = (normal(min(16384, N - lo), K) * 35).round_().clamp_(-127, 127).to(torch.int8)
        s = {"case": case, "a": a, "a_scale": 0.01 + 0.02 * normal(M).abs(), "w": w,
             "w_scale": 0.0005 + 0.0002 * normal(N).abs()}
        if own:
            _package()
            from bitnet_tt.int8_matmul import Int8Weight

            s["weight"] = Int8Weight.from_codes(w, s["w_scale"])
        return s
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    new, total = _sizes(case)
    T, B = sum(new), case["seqs"]
    s = {"case": case, "cu_q": _cu(new, dev), "kv_len": _ints(total, dev), "max_q": max(new), "max_kv": max(total),
         "scale": 1.0 / math.sqrt(D)}
    if case["op"] == "win_prompt":
        # channels of different size, as a projection's outputs are
        s["qkv"] = (normal(T, (H + 2 * Hkv) * D) * (0.3 + normal((H + 2 * Hkv) * D).abs())).to(torch.bfloat16)
        return s
    s["q"] = (2.0 * normal(T, H, D)).to(torch.bfloat16)
    ps, shared = case["page"], case.get("shared", 0) // case["page"]
    pages = [-(-n // ps) - shared for n in total]
    P = shared + sum(pages)
    order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros((B, shared + max(pages)), dtype=torch.int32, device=dev)
    table[:, :shared] = order[:shared]
    at = shared
    for b, n in enumerate(pages):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    s["page_table"] = table
    s["k_exp"] = s["v_exp"] = None
    if case["op"] == "prefix":
        s["shared_pages"] = _ints([shared], dev)
        s["max_shared"] = shared
    if case["kv"] == "bf16":
        s["k_pages"] = normal(P, Hkv, ps, D).to(torch.bfloat16)
        s["v_pages"] = normal(P, Hkv, ps, D).to(torch.bfloat16)
    else:
        s["k_pages"] = (100 * normal(P, Hkv, ps, D)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s["v_pages"] = (100 * normal(P, Hkv, ps, D)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s["k_exp"] = torch.randint(119, 122, (P, Hkv, ps), generator=gen, device=dev, dtype=torch.uint8)
        s["v_exp"] = torch.randint(119, 122, (P, Hkv, ps), generator=gen, device=dev, dtype=torch.uint8)
    return s


# ---- plain forms --------------------------------------------------------


def _rows(s):
    """Sequence and place in it of every packed token."""
    cu = s["cu_q"].long()
    t = torch.arange(s["case"]["tokens"], device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return seq, t - cu[seq]


def _values(s, pages, exps, page, row):
    """What rows of pages stand for, in 32 bits: page and row are index tensors alike."""
    if exps is None:
        return pages[page, :, row].float()
    x = pages.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float()
    return torch.ldexp(x, exps[page, :, row].int()[..., None] - 127)


def _from_pages(s, pages, exps, first=0):
    """[B, Hkv, max_kv - first, D] in 32 bits: positions from ``first``, zero behind each sequence."""
    ps = s["case"]["page"]
    rows = torch.arange(first, s["max_kv"], device=s["kv_len"].device)
    x = _values(s, pages, exps, s["page_table"].long()[:, rows // ps], (rows % ps).expand(s["case"]["seqs"], -1))
    inside = rows < s["kv_len"][:, None]
    return torch.where(inside[..., None, None], x, 0.0).transpose(1, 2)


def _softmax(sc, see):
    """Scores to weights, in place; rows that see nothing get zeros."""
    sc.masked_fill_(~see, -math.inf)
    sc.sub_(sc.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    return sc.div_(sc.sum(-1, keepdim=True).clamp_(min=1e-30))


def _attend(q, k, v, see, scale):
    """q [B, H, n, D], k and v [B, Hkv, m, D] in 32 bits, see [B, n, m]."""
    B, H, n, D = q.shape
    Hkv, m = k.shape[1], k.shape[2]
    sc = torch.matmul(q.reshape(B, Hkv, H // Hkv * n, D) * scale, k.transpose(2, 3)).view(B, Hkv, H // Hkv, n, m)
    return torch.matmul(_softmax(sc, see[:, None, None]).view(B, Hkv, H // Hkv * n, m), v).view(B, H, n, D)


def _padded(s, x):
    """Packed rows [T, heads, D] as [B, heads, max_q, D] in 32 bits."""
    seq, i = _rows(s)
    y = torch.zeros((s["case"]["seqs"], s["max_q"], *x.shape[1:]), dtype=torch.float32, device=x.device)
    y[seq, i] = x.float()
    return y.transpose(1, 2)


def _packed(s, y):
    seq, i = _rows(s)
    return y.transpose(1, 2)[seq, i].to(torch.bfloat16)


def _split(s):
    c = s["case"]
    x = s["qkv"].view(-1, c["heads"] + 2 * c["kv_heads"], c["dim"])
    return x[:, : c["heads"]], x[:, c["heads"]:-c["kv_heads"]], x[:, -c["kv_heads"]:]


def _positions(s):
    """Position of each sequence's rows, [B, max_q]."""
    first = s["kv_len"] - (s["cu_q"][1:] - s["cu_q"][:-1])
    return first[:, None] + torch.arange(s["max_q"], device=first.device)


def _in_window(s, m):
    """[B, max_q, m]: the positions that a row sees."""
    p, j = _positions(s)[..., None], torch.arange(m, device=s["kv_len"].device)
    return (j <= p) & ((j > p - s["case"]["window"]) | (j < s["case"]["sinks"]))


def _win_prompt(s):
    q, k, v = _split(s)
    return _packed(s, _attend(_padded(s, q), _padded(s, k), _padded(s, v), _in_window(s, s["max_q"]), s["scale"]))


def _win_paged(s):
    return _packed(s, _attend(_padded(s, s["q"]), _from_pages(s, s["k_pages"], s["k_exp"]),
                              _from_pages(s, s["v_pages"], s["v_exp"]), _in_window(s, s["max_kv"]), s["scale"]))


def _prefix(s):
    """The shared positions as one matrix for every row, the others sequence by sequence."""
    c = s["case"]
    H, Hkv, D, ps, n, B = c["heads"], c["kv_heads"], c["dim"], c["page"], s["max_q"], c["seqs"]
    shared = c["shared"]
    rows = torch.arange(shared, device=s["q"].device)
    page = s["page_table"].long()[0, rows // ps]
    kp, vp = (_values(s, s[x + "_pages"], s[x + "_exp"], page, rows % ps).transpose(0, 1) for x in "kv")
    ko, vo = (_from_pages(s, s[x + "_pages"], s[x + "_exp"], shared) for x in "kv")
    q = (_padded(s, s["q"]) * s["scale"]).reshape(B, Hkv, H // Hkv * n, D)
    sp = torch.matmul(q.transpose(0, 1).reshape(Hkv, -1, D), kp.transpose(1, 2))
    sp = sp.view(Hkv, B, -1, shared).transpose(0, 1)
    so = torch.matmul(q, ko.transpose(2, 3))
    p = _positions(s)
    see = torch.arange(s["max_kv"], device=p.device) <= p[..., None]
    sc = torch.cat((sp, so), -1).view(B, Hkv, H // Hkv, n, -1)
    w = _softmax(sc, see[:, None, None]).view(B, Hkv, H // Hkv * n, -1)
    o = torch.matmul(w[..., shared:], vo)
    o += torch.matmul(w[..., :shared].transpose(0, 1).reshape(Hkv, -1, shared), vp).view(Hkv, B, -1, D).transpose(0, 1)
    return _packed(s, o.view(B, H, n, D))


def _int8(s):
    """Sums of 1024 products are whole numbers below 2^24: exact in 32 bits, in any order."""
    a, w = s["a"], s["w"]
    acc = torch.zeros((a.shape[0], w.shape[0]), dtype=torch.int32, device=a.device)
    for lo in range(0, a.shape[1], 1024):
        acc += torch.matmul(a[:, lo:lo + 1024].float(), w[:, lo:lo + 1024].float().t()).int()
    y = acc.float() * s["a_scale"][:, None] * s["w_scale"]
    return y if s["case"]["out"] == "fp32" else y.to(torch.bfloat16)


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)


def _own(s):
    """The calls of the package."""
    _package()
    c = s["case"]
    if c["op"] == "int8":
        from bitnet_tt.int8_matmul import int8_matmul

        out = torch.float32 if c["out"] == "fp32" else torch.bfloat16
        return int8_matmul(s["a"], s["a_scale"], s["weight"], out_dtype=out)
    from bitnet_tt import paged_attention as pa

    if c["op"] == "win_prompt":
        q, k, v = _split(s)
        return pa.prompt_attention(q, k, v, s["cu_q"], scale=s["scale"], max_q=s["max_q"], window=c["window"],
                                   sinks=c["sinks"])
    cache = pa.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
    if c["op"] == "win_paged":
        return pa.paged_attention(s["q"], cache, s["page_table"], s["cu_q"], s["kv_len"], scale=s["scale"],
                                  max_q=s["max_q"], max_kv=s["max_kv"], window=c["window"], sinks=c["sinks"])
    return pa.shared_prefix_attention(s["q"], cache, s["page_table"], s["cu_q"], s["kv_len"], s["shared_pages"],
                                      scale=s["scale"], max_q=s["max_q"], max_kv=s["max_kv"],
                                      max_shared=s["max_shared"])


def run(state):
    if own:
        return _own(state)
    return {"win_prompt": _win_prompt, "win_paged": _win_paged, "prefix": _prefix,
            "int8": _int8}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "int8":
        M, K, N = case["rows"], case["inner"], case["cols"]
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * (4 if case["out"] == "fp32" else 2),
                "flops": 2 * M * N * K}
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    new, total = _sizes(case)
    T = sum(new)
    row = 2 * D if case.get("kv") != "fp8" else D + 1  # bytes of a key or value row in a page
    if case["op"] == "prefix":
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, total))
        rows = case["shared"] + sum(m - case["shared"] for m in total)
    else:
        W, S = case["window"], case["sinks"]
        pairs = sum(min(p + 1, W) + max(0, min(S, p + 1 - W)) for n, m in zip(new, total) for p in range(m - n, m))
        # positions that any row of a sequence sees
        rows = sum(min(m, n + W - 1) + max(0, min(S, m - (n + W - 1))) for n, m in zip(new, total))
    if case["op"] == "win_prompt":
        return {"bytes": T * (2 * H + 2 * Hkv) * D * 2, "flops": 4 * H * D * pairs}
    return {"bytes": T * 2 * H * D * 2 + rows * Hkv * 2 * row, "flops": 4 * H * D * pairs}


# ---- in 64 bits, sequence by sequence ----------------------------------


def _exact_rows(s, b, n, pages, exps):
    """Positions 0..n-1 of sequence b: [Hkv, n, D]."""
    ps = s["case"]["page"]
    ids = s["page_table"][b, : -(-n // ps)].long()
    x = pages[ids].double() if exps is None else pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
    if exps is not None:
        x = x * torch.exp2(exps[ids].double() - 127)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_attend(q, k, v, scale, window, sinks):
    """q [n, H, D], k and v [Hkv, m, D]: the last n of m positions ask, each the last ``window``
    positions up to its own and the first ``sinks`` of those."""
    n, H, D = q.shape
    Hkv, m = k.shape[0], k.shape[1]
    o = torch.empty((n, H, D), dtype=torch.float64, device=q.device)
    j = torch.arange(m, device=q.device)[None]
    for lo in range(0, n, 2048):
        at = torch.arange(m - n, m, device=q.device)[lo:lo + 2048, None]
        away = at - j  # how far back a position lies
        hidden = (away < 0) | ((away >= window) & (j >= sinks))
        for h in range(H):
            w = (q[lo:lo + 2048, h].double() @ k[h // (H // Hkv)].T) * scale
            w = torch.softmax(w.masked_fill_(hidden, -math.inf), -1)
            o[lo:lo + 2048, h] = w @ v[h // (H // Hkv)]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int8":
        y = torch.empty((case["rows"], case["cols"]), dtype=torch.float64, device=s["a"].device)
        a = s["a"].double()
        for lo in range(0, case["cols"], 16384):
            w = s["w"][lo:lo + 16384].double()
            y[:, lo:lo + 16384] = a @ w.t()  # whole numbers below 2^53
        return y * s["a_scale"].double()[:, None] * s["w_scale"].double()
    new, total = _sizes(case)
    H, Hkv = case["heads"], case["kv_heads"]
    window, sinks = case.get("window", max(total)), case.get("sinks", 0)
    at = [sum(new[:b]) for b in range(len(new))]
    if case["op"] == "win_prompt":
        x = s["qkv"].double().view(-1, H + 2 * Hkv, case["dim"])
        o = [_exact_attend(x[a:a + n, :H], x[a:a + n, H:H + Hkv].transpose(0, 1),
                           x[a:a + n, H + Hkv:].transpose(0, 1), s["scale"], window, sinks) for a, n in zip(at, new)]
        return torch.cat(o)
    o = [_exact_attend(s["q"][a:a + n], _exact_rows(s, b, m, s["k_pages"], s["k_exp"]),
                       _exact_rows(s, b, m, s["v_pages"], s["v_exp"]), s["scale"], window, sinks)
         for b, (a, n, m) in enumerate(zip(at, new, total))]
    return torch.cat(o)
