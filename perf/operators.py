"""The operators of prompts and of the paged key-value cache, as measurable cases.

A case is a dict of plain values; ``prepare`` makes what a serving program
holds before the call (a batch's projections, page pools and page tables, the
rotation tables), ``run`` is one pass through an operator: its plain form, or
the package's entry point where ``own`` is set.  ``exact`` is the same result in
64 bits.  Heads are those of the BitNet b1.58 2B model (20 query and 5
key-value heads of 128) and of the small test model (4 and 2 of 64).

Operators:
  write   the fused QKV rows of a batch: q rotated, k rotated and v put into
          their pages, in bf16 or in 8 bits with a power of two per row
  read    pages of a batch into a contiguous bf16 cache
  prompt  causal attention within packed sequences
  paged   attention of the newest tokens of each sequence over its pages
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
THETA = 500000.0


def listed():
    return [
        # every decode step of 32 users: one row each, the smallest call
        {"name": "write_decode_b32", "op": "write", **BIG, "rot": 128, "adjacent": False, "kv": "bf16", "page": 64,
         "seqs": 32, "tokens": 32, "past": 4000},
        # prompts of eleven users arriving together, into an 8-bit cache of small pages
        {"name": "write_prompts_fp8", "op": "write", **BIG, "rot": 128, "adjacent": False, "kv": "fp8", "page": 16,
         "seqs": 11, "tokens": 8191, "past": 0},
        # part of the head rotated, adjacent pairs, far positions
        {"name": "write_part_far", "op": "write", **MINI, "rot": 32, "adjacent": True, "kv": "bf16", "page": 32,
         "seqs": 3, "tokens": 777, "past": 120000},
        # an 8-bit cache of 32 users handed to the contiguous decode step
        {"name": "read_fp8_b32", "op": "read", **BIG, "kv": "fp8", "page": 64, "seqs": 32, "past": 4096},
        # a few users of the small model, odd lengths
        {"name": "read_bf16_b3", "op": "read", **MINI, "kv": "bf16", "page": 16, "seqs": 3, "past": 509},
        # short prompts of several users in one batch
        {"name": "prompt_short_packed", "op": "prompt", **MINI, "seqs": 9, "tokens": 1003},
        # one user's prompt of the model's whole context
        {"name": "prompt_4096", "op": "prompt", **BIG, "seqs": 1, "tokens": 4096},
        # documents of different lengths, packed
        {"name": "prompt_packed_16k", "op": "prompt", **BIG, "seqs": 4, "tokens": 16001},
        # one decode step's attention of 32 users, ragged contexts, 8-bit cache
        {"name": "paged_decode_b32_fp8", "op": "paged", **BIG, "kv": "fp8", "page": 64, "seqs": 32, "tokens": 32,
         "past": 4000},
        # one user far into a long context: latency of a single stream
        {"name": "paged_decode_b1_long", "op": "paged", **BIG, "kv": "bf16", "page": 64, "seqs": 1, "tokens": 1,
         "past": 131000},
        # chunked prompts of four users over what is cached already
        {"name": "paged_chunk_b4", "op": "paged", **BIG, "kv": "bf16", "page": 64, "seqs": 4, "tokens": 2047,
         "past": 8000},
        # a short chunk over a long 8-bit context: few rows, a long axis
        {"name": "paged_chunk_long_fp8", "op": "paged", **BIG, "kv": "fp8", "page": 32, "seqs": 1, "tokens": 67,
         "past": 40000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "prompt", "paged", "prompt", "paged"])
    c = {"op": op, **(BIG if rng.random() < 0.75 else MINI)}
    if op != "prompt":
        c["kv"] = rng.choice(["bf16", "fp8"])
        c["page"] = rng.choice([16, 32, 64, 128, 256])
    if op == "write":
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 16])
        c["adjacent"] = rng.random() < 0.5
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = c["seqs"] if rng.random() < 0.4 else max(c["seqs"], _log(rng, 1, 8000))
        c["past"] = _log(rng, 1, 100000 // c["seqs"])
    elif op == "read":
        c["seqs"] = _log(rng, 1, 32)
        c["past"] = _log(rng, 1, 4096)
    elif op == "prompt":
        c["seqs"] = _log(rng, 1, 32)
        c["tokens"] = max(c["seqs"], _log(rng, 1, 12000))
    elif rng.random() < 0.5:
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = c["seqs"]
        c["past"] = _log(rng, 1, 120000 // c["seqs"])
    else:
        c["seqs"] = _log(rng, 1, 8)
        c["tokens"] = c["seqs"] + _log(rng, 1, 2000)
        c["past"] = _log(rng, 1, 60000 // c["seqs"])
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
    if case["op"] == "read":
        new = [0] * case["seqs"]
    else:
        new = _counts(case["tokens"], case["seqs"])
    past = _pasts(case["past"], case["seqs"]) if "past" in case else [0] * case["seqs"]
    return new, [a + b for a, b in zip(new, past)]


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
    gen.manual_seed(int(seed) * 7919 + 11)
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    new, total = _sizes(case)
    T, B = sum(new), case["seqs"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    s = {"case": case, "cu_q": _cu(new, dev), "kv_len": _ints(total, dev), "max_q": max(new), "max_kv": max(total),
         "scale": 1.0 / math.sqrt(D)}
    if case["op"] in ("write", "prompt"):
        # channels of different size, as a projection's outputs are
        s["qkv"] = (normal(T, (H + 2 * Hkv) * D) * (0.3 + normal((H + 2 * Hkv) * D).abs())).to(torch.bfloat16)
    if case["op"] == "paged":
        s["q"] = (2.0 * normal(T, H, D)).to(torch.bfloat16)
    if case["op"] != "prompt":
        ps = case["page"]
        pages = [-(-n // ps) for n in total]
        P = sum(pages)
        order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
        table = torch.zeros((B, max(pages)), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(pages):
            table[b, :n] = order[at:at + n]
            at += n
        s["page_table"] = table
        s["k_exp"] = s["v_exp"] = None
        if case["kv"] == "bf16":
            s["k_pages"] = normal(P, Hkv, ps, D).to(torch.bfloat16)
            s["v_pages"] = normal(P, Hkv, ps, D).to(torch.bfloat16)
        else:
            s["k_pages"] = (100 * normal(P, Hkv, ps, D)).clamp(-448, 448).to(torch.float8_e4m3fn)
            s["v_pages"] = (100 * normal(P, Hkv, ps, D)).clamp(-448, 448).to(torch.float8_e4m3fn)
            s["k_exp"] = torch.randint(119, 122, (P, Hkv, ps), generator=gen, device=dev, dtype=torch.uint8)
            s["v_exp"] = torch.randint(119, 122, (P, Hkv, ps), generator=gen, device=dev, dtype=torch.uint8)
    if case["op"] == "write":
        i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev)
        angle = torch.arange(max(total), dtype=torch.float64, device=dev)[:, None] * THETA ** (-i / case["rot"])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if case["op"] == "read":
        s["k"] = torch.zeros((B, Hkv, max(total), D), dtype=torch.bfloat16, device=dev)
        s["v"] = torch.zeros((B, Hkv, max(total), D), dtype=torch.bfloat16, device=dev)
    return s


# ---- plain forms --------------------------------------------------------


def _rows(s):
    """Sequence, place in it and position of every packed token."""
    cu = s["cu_q"].long()
    T = s["case"]["tokens"]
    t = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[seq]
    return seq, i, s["kv_len"].long()[seq] - (cu[seq + 1] - cu[seq]) + i


def _rotate(x, c, sn, R, adjacent):
    """x [T, heads, D] in 32 bits, c and sn [T, 1, R/2]."""
    if adjacent:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2:R]
        y = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
    return torch.cat((y, x[..., R:]), dim=-1)


def _quantise(x):
    """(codes, exponent bytes) of rows x [..., D] in 32 bits."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp_(min=-126)
    e = torch.where(m == 0, -126, e)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _write(s):
    c = s["case"]
    H, Hkv, D, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    seq, _, pos = _rows(s)
    x = s["qkv"].float().view(-1, H + 2 * Hkv, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = _rotate(x[:, : H + Hkv], cos, sin, c["rot"], c["adjacent"])
    k, v = qk[:, H:], x[:, H + Hkv:]
    page, row = s["page_table"].long()[seq, pos // ps], pos % ps
    if c["kv"] == "bf16":
        s["k_pages"][page, :, row] = k.to(torch.bfloat16)
        s["v_pages"][page, :, row] = v.to(torch.bfloat16)
    else:
        kc, ke = _quantise(k)
        vc, ve = _quantise(v)
        s["k_pages"].view(torch.uint8)[page, :, row] = kc.view(torch.uint8)
        s["v_pages"].view(torch.uint8)[page, :, row] = vc.view(torch.uint8)
        s["k_exp"][page, :, row] = ke
        s["v_exp"][page, :, row] = ve
    return [qk[:, :H].to(torch.bfloat16), s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"]]


def _from_pages(s, pages, exps):
    """[B, Hkv, max_kv, D] in 32 bits, zero behind each sequence."""
    ps, n = s["case"]["page"], s["max_kv"]
    table = s["page_table"].long()
    rows = torch.arange(n, device=table.device)
    page = table[:, rows // ps]
    if exps is None:
        x = pages[page, :, rows % ps].float()
    else:
        x = pages.view(torch.uint8)[page, :, rows % ps].view(torch.float8_e4m3fn).float()
        x = torch.ldexp(x, exps[page, :, rows % ps].int()[..., None] - 127)
    inside = rows < s["kv_len"][:, None]
    return torch.where(inside[..., None, None], x, 0.0).transpose(1, 2)


def _read(s):
    inside = (torch.arange(s["max_kv"], device=s["kv_len"].device) < s["kv_len"][:, None])[:, None, :, None]
    s["k"].copy_(torch.where(inside, _from_pages(s, s["k_pages"], s["k_exp"]).to(torch.bfloat16), s["k"]))
    s["v"].copy_(torch.where(inside, _from_pages(s, s["v_pages"], s["v_exp"]).to(torch.bfloat16), s["v"]))
    return [s["k"], s["v"]]


def _attend(q, k, v, first, scale):
    """q [B, H, n, D], k and v [B, Hkv, m, D] in 32 bits; row i sees positions
    up to first[b] + i."""
    B, H, n, D = q.shape
    Hkv, m = k.shape[1], k.shape[2]
    see = torch.arange(m, device=q.device) <= first[:, None, None] + torch.arange(n, device=q.device)[:, None]
    sc = torch.matmul(q.reshape(B, Hkv, H // Hkv * n, D) * scale, k.transpose(2, 3)).view(B, Hkv, H // Hkv, n, m)
    sc.masked_fill_(~see[:, None, None], -math.inf)
    sc.sub_(sc.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = sc.sum(-1)
    o = torch.matmul(sc.view(B, Hkv, H // Hkv * n, m), v).view(B, H, n, D)
    total = total.view(B, H, n, 1)
    return torch.where(total > 0, o / total, 0.0)


def _padded(s, x):
    """Packed rows [T, heads, D] as [B, heads, max_q, D] in 32 bits."""
    seq, i, _ = _rows(s)
    y = torch.zeros((s["case"]["seqs"], s["max_q"], *x.shape[1:]), dtype=torch.float32, device=x.device)
    y[seq, i] = x.float()
    return y.transpose(1, 2)


def _packed(s, y):
    seq, i, _ = _rows(s)
    return y.transpose(1, 2)[seq, i].to(torch.bfloat16)


def _split(s):
    c = s["case"]
    x = s["qkv"].view(-1, c["heads"] + 2 * c["kv_heads"], c["dim"])
    return x[:, : c["heads"]], x[:, c["heads"]:-c["kv_heads"]], x[:, -c["kv_heads"]:]


def _prompt(s):
    q, k, v = _split(s)
    first = torch.zeros_like(s["kv_len"])
    return _packed(s, _attend(_padded(s, q), _padded(s, k), _padded(s, v), first, s["scale"]))


def _paged(s):
    first = s["kv_len"] - (s["cu_q"][1:] - s["cu_q"][:-1])
    o = _attend(_padded(s, s["q"]), _from_pages(s, s["k_pages"], s["k_exp"]),
                _from_pages(s, s["v_pages"], s["v_exp"]), first, s["scale"])
    return _packed(s, o)


def _own(s):
    """The calls of the package."""
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from bitnet_tt import paged_attention as pa

    c = s["case"]
    if c["op"] == "prompt":
        q, k, v = _split(s)
        return pa.prompt_attention(q, k, v, s["cu_q"], scale=s["scale"], max_q=s["max_q"])
    cache = pa.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
    if c["op"] == "write":
        q = pa.rope_write(s["qkv"], s["cos"], s["sin"], s["cu_q"], s["kv_len"], c["heads"], c["kv_heads"], cache=cache,
                          page_table=s["page_table"], rope_adjacent=c["adjacent"])
        return [q, s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"]]
    if c["op"] == "read":
        pa.read_pages(cache, s["page_table"], s["kv_len"], s["k"], s["v"])
        return [s["k"], s["v"]]
    return pa.paged_attention(s["q"], cache, s["page_table"], s["cu_q"], s["kv_len"], scale=s["scale"],
                              max_q=s["max_q"], max_kv=s["max_kv"])


def run(state):
    if own:
        return _own(state)
    return {"write": _write, "read": _read, "prompt": _prompt, "paged": _paged}[state["case"]["op"]](state)


def work(case):
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    new, total = _sizes(case)
    T = sum(new)
    row = 2 * D if case.get("kv") != "fp8" else D + 1  # bytes of a key or value row in a page
    if case["op"] == "write":
        tables = T * 4 * case["rot"]
        return {"bytes": T * (H + 2 * Hkv) * D * 2 + tables + T * H * D * 2 + T * 2 * Hkv * row,
                "flops": T * (H + Hkv) * 3 * case["rot"]}
    if case["op"] == "read":
        return {"bytes": sum(total) * Hkv * 2 * (row + 2 * D), "flops": 0}
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, total))
    if case["op"] == "prompt":
        return {"bytes": T * (2 * H + 2 * Hkv) * D * 2, "flops": 4 * H * D * pairs}
    return {"bytes": T * 2 * H * D * 2 + sum(total) * Hkv * 2 * row, "flops": 4 * H * D * pairs}


# ---- in 64 bits, sequence by sequence ----------------------------------


def _e4m3(x):
    """x rounded to three fraction bits, ties to even, no exponent below -6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _row_exponent(x):
    """The least e >= -126 with max|x| <= 448 * 2^e, per row."""
    big = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140)
    e = torch.ceil(torch.log2(big / 448))
    e = torch.where(big <= 448 * torch.exp2(e - 1), e - 1, e)
    return torch.where(big > 448 * torch.exp2(e), e + 1, e).clamp(min=-126)


def _exact_rows(s, b, n, pages, exps):
    """Positions 0..n-1 of sequence b: [Hkv, n, D]."""
    ps = s["case"]["page"]
    ids = s["page_table"][b, : -(-n // ps)].long()
    x = pages[ids].double() if exps is None else pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
    if exps is not None:
        x = x * torch.exp2(exps[ids].double() - 127)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_attend(q, k, v, scale):
    """q [n, H, D], k and v [Hkv, m, D]: the last n of m positions ask."""
    n, H, D = q.shape
    Hkv, m = k.shape[0], k.shape[1]
    o = torch.empty((n, H, D), dtype=torch.float64, device=q.device)
    at = torch.arange(m - n, m, device=q.device)
    for lo in range(0, n, 4096):
        for h in range(H):
            w = (q[lo:lo + 4096, h].double() @ k[h // (H // Hkv)].T) * scale
            w[torch.arange(m, device=q.device)[None] > at[lo:lo + 4096, None]] = -math.inf
            w = torch.softmax(w, -1)
            o[lo:lo + 4096, h] = w @ v[h // (H // Hkv)]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    new, total = _sizes(case)
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "read":
        out = []
        for pages, exps, into in ((s["k_pages"], s["k_exp"], s["k"]), (s["v_pages"], s["v_exp"], s["v"])):
            y = into.double()
            for b, n in enumerate(total):
                y[b, :, :n] = _exact_rows(s, b, n, pages, exps)
            out.append(y)
        return out
    at = [sum(new[:b]) for b in range(len(new))]
    if case["op"] == "prompt":
        x = s["qkv"].double().view(-1, H + 2 * Hkv, D)
        o = [_exact_attend(x[a:a + n, :H], x[a:a + n, H:H + Hkv].transpose(0, 1),
                           x[a:a + n, H + Hkv:].transpose(0, 1), s["scale"]) for a, n in zip(at, new)]
        return torch.cat(o)
    if case["op"] == "paged":
        o = [_exact_attend(s["q"][a:a + n], _exact_rows(s, b, m, s["k_pages"], s["k_exp"]),
                           _exact_rows(s, b, m, s["v_pages"], s["v_exp"]), s["scale"])
             for b, (a, n, m) in enumerate(zip(at, new, total))]
        return torch.cat(o)
    # write: pairs as complex numbers times the tables' unit numbers
    x = s["qkv"].double().view(-1, H + 2 * Hkv, D).clone()
    R, ps = case["rot"], case["page"]
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, total)]).to(x.device)
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    one, two = (slice(0, R, 2), slice(1, R, 2)) if case["adjacent"] else (slice(0, R // 2), slice(R // 2, R))
    z = torch.complex(x[:, : H + Hkv, one], x[:, : H + Hkv, two]) * turn
    x[:, : H + Hkv, one], x[:, : H + Hkv, two] = z.real, z.imag
    k, v = s["k_pages"].double(), s["v_pages"].double()
    for pages, rows in ((k, x[:, H:H + Hkv]), (v, x[:, H + Hkv:])):
        if case["kv"] == "fp8":
            rows = _e4m3(rows * torch.exp2(-_row_exponent(rows)))
        for b, (a, n, m) in enumerate(zip(at, new, total)):
            p = torch.arange(m - n, m, device=x.device)
            pages[s["page_table"][b].long()[p // ps], :, p % ps] = rows[a:a + n]
    return [x[:, :H], k, v, None, None]
