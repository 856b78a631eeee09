"""Prompts and the paged key-value cache: rotation with page writes, page reads,
attention within packed prompts and over the pages, on gfx950 (include/btl.h,
"prompts and the paged key-value cache").

The reference's prompt path is src/bitnet_tt/layers/attention.py:1348-1507,
its caches :115-458.  A *batch* here is T packed rows: sequence b's rows are
``cu_q[b] .. cu_q[b + 1] - 1``, its newest tokens, at positions
``kv_len[b] - n_b .. kv_len[b] - 1``.  Position p is row ``p % page_size`` of
page ``page_table[b][p // page_size]``.  cu_q [B + 1], kv_len [B] and
page_table [B, max_pages] are int32 device tensors, so a captured graph can
advance them; what they hold is checked on the device: a batch that is not
well formed sets the error word that ``bitnet_tt.ternary_matmul.check()``
and the other ``check()`` methods read, and its outputs are invalid.  Rows with a
negative position (kv_len below the number of rows: padding) give zeros and
write nothing; rows outside [cu_q[0], cu_q[B]) are left as they were.

Calls are ordered on the current stream of their tensors' device.  Calls that
write one cache, and calls that read what another writes, must be ordered by the caller;
calls that only read it may overlap (each has its own scratch).
"""

from __future__ import annotations

import functools
import math

import torch

from . import _native as N

_BF16 = torch.bfloat16
_ERROR_BYTES = 256


class PagedKVCache:
    """One layer's page pools: ``key_pages`` and ``value_pages`` [num_pages,
    kv_heads, page_size, head_dim] bf16, or float8_e4m3fn with one exponent byte
    per row in ``key_exp`` and ``value_exp`` [num_pages, kv_heads, page_size]
    uint8 (a value is code x 2^(byte - 127)).  page_size is a multiple of 16;
    head_dim 64 or 128.  The contiguous caches of DecodeAttention are pages
    of max_seq_len rows: :meth:`of_cache`."""

    def __init__(self, key_pages, value_pages, key_exp=None, value_exp=None) -> None:
        fp8 = key_exp is not None
        if key_pages.dim() != 4 or key_pages.shape != value_pages.shape:
            raise ValueError("key_pages and value_pages must be [num_pages, kv_heads, page_size, head_dim], alike")
        if (value_exp is not None) != fp8:
            raise ValueError("key_exp and value_exp come together")
        dtype = torch.float8_e4m3fn if fp8 else _BF16
        if key_pages.dtype != dtype or value_pages.dtype != dtype:
            raise ValueError(f"pages must be {dtype} {'with' if fp8 else 'without'} exponent bytes")
        P, H, S, D = key_pages.shape
        if S < 16 or S % 16:
            raise ValueError(f"page_size {S} is not a multiple of 16")
        if D not in (64, 128):
            raise ValueError(f"head_dim {D}: 64 and 128 are supported")
        N.require_cuda(key_pages, "key_pages")
        N.require_cuda(value_pages, "value_pages")
        if fp8:
            for t, name in ((key_exp, "key_exp"), (value_exp, "value_exp")):
                N.require_cuda(t, name)
                if t.dtype != torch.uint8 or t.shape != (P, H, S):
                    raise ValueError(f"{name} must be uint8 [num_pages, kv_heads, page_size]")
        for t in (value_pages, key_exp, value_exp):
            if t is not None and t.device != key_pages.device:
                raise ValueError("the pools are on different devices")
        self.key_pages, self.value_pages = key_pages, value_pages
        self.key_exp, self.value_exp = key_exp, value_exp

    @classmethod
    def allocate(cls, num_pages: int, num_kv_heads: int, head_dim: int, device, page_size: int = 64,
                 dtype: str = "bf16") -> "PagedKVCache":
        """Zero-filled pools; dtype "bf16" or "fp8"."""
        if dtype not in ("bf16", "fp8"):
            raise ValueError(f"cache dtype {dtype!r}: 'bf16' or 'fp8'")
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        if dtype == "bf16":
            return cls(torch.zeros(shape, dtype=_BF16, device=device), torch.zeros(shape, dtype=_BF16, device=device))
        pages = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        return cls(*pages, *[torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)])

    @classmethod
    def of_cache(cls, kv_cache) -> "PagedKVCache":
        """A contiguous cache (layers.attention.KVCache) as pages: page b is
        sequence b's, so its page table is arange(batch)[:, None]."""
        return cls(kv_cache.key_cache, kv_cache.value_cache)

    @property
    def num_pages(self) -> int:
        return self.key_pages.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.key_pages.shape[1]

    @property
    def page_size(self) -> int:
        return self.key_pages.shape[2]

    @property
    def head_dim(self) -> int:
        return self.key_pages.shape[3]

    @property
    def device(self):
        return self.key_pages.device

    def _struct(self) -> N.Pages:
        P, H, S, D = self.key_pages.shape
        fp8 = self.key_exp is not None
        return N.Pages(self.key_pages.data_ptr(), self.value_pages.data_ptr(),
                       self.key_exp.data_ptr() if fp8 else None, self.value_exp.data_ptr() if fp8 else None, P, H, S, D)


def _on(t, device, name):
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call's tensors on {device}")


def _int32(t, device, shape, name):
    if t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)}")
    _on(t, device, name)


def _batch(cu_q, kv_len, page_table, device):
    """(B, max_pages) after checks of the host-visible side."""
    B = cu_q.shape[0] - 1 if cu_q.dim() == 1 else -1
    if B < 1:
        raise ValueError("cu_q must be int32 [B + 1] of at least one sequence")
    _int32(cu_q, device, (B + 1,), "cu_q")
    if kv_len is not None:
        _int32(kv_len, device, (B,), "kv_len")
    if page_table is None:
        return B, 0
    if page_table.dim() != 2 or page_table.shape[1] < 1:
        raise ValueError("page_table must be int32 [B, max_pages]")
    _int32(page_table, device, (B, page_table.shape[1]), "page_table")
    return B, page_table.shape[1]


def _rows(t, heads, dim, name, device=None):
    """Row stride of a packed bf16 tensor [T, heads, dim] whose rows are dense."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a ROCm GPU device; this path runs only through the gfx950 kernels")
    if t.dtype != _BF16 or t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise ValueError(f"{name} must be bf16 [T, {heads}, {dim}]")
    if device is not None:
        _on(t, device, name)
    st = t.stride()
    if st[2] != 1 or (st[1] != dim and heads > 1):
        raise ValueError(f"{name}: the heads of a row must be dense")
    ld = st[0] if t.shape[0] > 1 else max(st[0], heads * dim)
    if ld < heads * dim or ld % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows must be 16-byte aligned and not overlap")
    return ld


def _error_word(device, stream):
    if not N.has_workspace(device, _ERROR_BYTES, "paged") and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("run one eager call on this stream before capturing it in a graph")
    return N.workspace_ptr(device.index, _ERROR_BYTES, "paged", 0, stream)[0]


def _on_device(fn):
    """Runs fn with its first argument's device current: a launch belongs there."""

    @functools.wraps(fn)
    def call(first, *args, **kwargs):
        index = first.device.index
        if not torch.cuda.is_available() or index is None or index == torch.cuda.current_device():
            return fn(first, *args, **kwargs)
        with torch.cuda.device(index):
            return fn(first, *args, **kwargs)

    return call


@_on_device
def rope_write(qkv, rope_cos, rope_sin, cu_q, kv_len, num_heads: int, num_kv_heads: int, cache: PagedKVCache | None = None,
               page_table=None, rope_adjacent: bool = False, q_out=None, k_out=None):
    """Rotates the q and k heads of fused QKV rows and writes k and v to their pages.

    qkv: bf16 [T, (H + 2 Hkv) D].  rope_cos / rope_sin: fp32 [S, R / 2], the
    angles of the first R dims of a head (pairs (i, i + R/2), or (2i, 2i+1) with
    ``rope_adjacent``); see utils.rope.rope_tables.  kv_len None: whole prompts,
    positions from 0.  Without ``cache`` nothing but q (and k_out) is written.  An 8-bit
    row keeps the least exponent e with max|x| <= 448 * 2^e and is rounded once,
    from the fp32 rotation; a row with a value that is not finite reads back as NaN.  Returns q [T, H, D] (``q_out``, which may
    be the q part of qkv itself, as ``k_out`` [T, Hkv, D] may be its k part)."""
    H, Hkv = int(num_heads), int(num_kv_heads)
    N.require_cuda(qkv, "qkv")
    if qkv.dtype != _BF16 or qkv.dim() != 2 or H < 1 or Hkv < 1 or qkv.shape[1] % (H + 2 * Hkv):
        raise ValueError(f"qkv must be bf16 [T, ({H} + 2 * {Hkv}) * head_dim]")
    T, D = qkv.shape[0], qkv.shape[1] // (H + 2 * Hkv)
    dev = qkv.device
    for t, name in ((rope_cos, "rope_cos"), (rope_sin, "rope_sin")):
        if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.shape != rope_cos.shape:
            raise ValueError(f"{name} must be contiguous fp32 [positions, rotated dims / 2]")
        _on(t, dev, name)
    B, max_pages = _batch(cu_q, kv_len, page_table if cache is not None else None, dev)
    if cache is not None:
        if page_table is None:
            raise ValueError("a cache needs a page table")
        if cache.num_kv_heads != Hkv or cache.head_dim != D:
            raise ValueError(f"cache of {cache.num_kv_heads} heads of {cache.head_dim}, rows of {Hkv} of {D}")
        _on(cache.key_pages, dev, "cache")
    if q_out is None:
        q_out = torch.empty((T, H, D), dtype=_BF16, device=dev)
    elif q_out.shape[0] != T:
        raise ValueError(f"q_out must have {T} rows")
    ldq = _rows(q_out, H, D, "q_out", dev)
    ldk = 0
    if k_out is not None:
        if k_out.shape[0] != T:
            raise ValueError(f"k_out must have {T} rows")
        ldk = _rows(k_out, Hkv, D, "k_out", dev)
    stream = N.raw_stream(dev.index)
    rc = N.lib().btl_rope_write(
        qkv.data_ptr(), T, (H + 2 * Hkv) * D, H, Hkv, D, rope_cos.data_ptr(), rope_sin.data_ptr(),
        2 * rope_cos.shape[1], rope_cos.shape[0], int(bool(rope_adjacent)), cu_q.data_ptr(),
        None if kv_len is None else kv_len.data_ptr(), B, q_out.data_ptr(), ldq,
        None if k_out is None else k_out.data_ptr(), ldk, None if cache is None else cache._struct(),
        None if cache is None else page_table.data_ptr(), max_pages, _error_word(dev, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_rope_write")
    return q_out


@_on_device
def read_pages(cache: PagedKVCache, page_table, kv_len, key_cache, value_cache) -> None:
    """Copies rows [0, kv_len[b]) of every sequence from its pages into the
    contiguous bf16 caches [B, Hkv, S, D] (those of layers.attention.KVCache, which
    the decode steps read); the rows behind stay as they were."""
    dev = cache.device
    if page_table.dim() != 2 or page_table.shape[0] < 1 or page_table.shape[1] < 1:
        raise ValueError("page_table must be int32 [B, max_pages]")
    B, max_pages = page_table.shape
    _int32(page_table, dev, (B, max_pages), "page_table")
    _int32(kv_len, dev, (B,), "kv_len")
    for t, name in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        N.require_cuda(t, name)
        _on(t, dev, name)
        if (t.dtype != _BF16 or t.dim() != 4 or t.shape[:2] != (B, cache.num_kv_heads) or t.shape[3] != cache.head_dim
                or t.shape != key_cache.shape):
            raise ValueError(f"{name} must be bf16 [{B}, {cache.num_kv_heads}, positions, {cache.head_dim}]")
    stream = N.raw_stream(dev.index)
    rc = N.lib().btl_read_pages(cache._struct(), page_table.data_ptr(), B, max_pages, kv_len.data_ptr(),
                                key_cache.shape[2], key_cache.data_ptr(), value_cache.data_ptr(),
                                _error_word(dev, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_read_pages")


def _scale(scale, D):
    return 1.0 / math.sqrt(D) if scale is None else float(scale)


@_on_device
def prompt_attention(q, k, v, cu_seqlens, scale: float | None = None, max_q: int | None = None, out=None):
    """Causal attention within packed sequences: row i attends to the rows up to
    itself of its own sequence, query head h to key-value head h // (H / Hkv).

    q bf16 [T, H, D], k and v [T, Hkv, D] (parts of a QKV row will do: rows may
    be strided); cu_seqlens int32 [B + 1]; scale defaults to 1/sqrt(D); max_q, where known, is the longest
    sequence (a hint).  Returns bf16 [T, H, D] (``out``, which must not overlap the inputs)."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or k.shape[0] != q.shape[0] or v.shape != k.shape:
        raise ValueError("q must be [T, H, D], k and v [T, Hkv, D]")
    T, H, D = q.shape
    Hkv = k.shape[1]
    if Hkv < 1 or H % Hkv:
        raise ValueError(f"{H} query heads over {Hkv} key-value heads")
    ldq = _rows(q, H, D, "q")
    dev = q.device
    ldk, ldv = _rows(k, Hkv, D, "k", dev), _rows(v, Hkv, D, "v", dev)
    B, _ = _batch(cu_seqlens, None, None, dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=_BF16, device=dev)
    elif out.shape[0] != T:
        raise ValueError(f"out must have {T} rows")
    ldo = _rows(out, H, D, "out", dev)
    stream = N.raw_stream(dev.index)
    rc = N.lib().btl_prompt_attention(
        q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, T, H, Hkv, D, cu_seqlens.data_ptr(), B,
        _scale(scale, D), T if max_q is None else int(max_q), out.data_ptr(), ldo, _error_word(dev, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_prompt_attention")
    return out


@_on_device
def paged_attention(q, cache: PagedKVCache, page_table, cu_q, kv_len, scale: float | None = None,
                    max_q: int | None = None, max_kv: int | None = None, out=None):
    """Attention of each sequence's newest tokens over its pages: the row at
    position p attends to positions [0, p], which have been written before.

    q bf16 [T, H, D], rotated.  max_q and max_kv, where known, are the most new
    tokens and the longest kv_len of any sequence: they choose the kernel and how a long
    context is split over workgroups, and a wrong one costs time only.  Single-token
    steps should pass max_q=1.  Returns bf16 [T, H, D] (``out``, not overlapping q)."""
    if q.dim() != 3:
        raise ValueError("q must be [T, H, D]")
    T, H, D = q.shape
    ldq = _rows(q, H, cache.head_dim, "q", cache.device)
    if H % cache.num_kv_heads:
        raise ValueError(f"{H} query heads over {cache.num_kv_heads} key-value heads")
    dev = q.device
    if page_table is None or kv_len is None:
        raise ValueError("paged attention needs a page table and kv_len")
    B, max_pages = _batch(cu_q, kv_len, page_table, dev)
    cap = max_pages * cache.page_size
    mq = T if max_q is None else min(int(max_q), T)
    mkv = cap if max_kv is None else min(int(max_kv), cap)
    if out is None:
        out = torch.empty((T, H, D), dtype=_BF16, device=dev)
    elif out.shape[0] != T:
        raise ValueError(f"out must have {T} rows")
    ldo = _rows(out, H, D, "out", dev)
    if T == 0:
        return out
    if mq < 1 or mkv < 1:
        raise ValueError(f"max_q {max_q} and max_kv {max_kv} must be at least 1")
    stream = N.raw_stream(dev.index)
    nbytes = _scratch_bytes(dev.index, T, H, cache.num_kv_heads, D, B, mq, mkv)
    # the call's own, from the stream-ordered allocator: calls that overlap share nothing
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    rc = N.lib().btl_paged_attention(
        q.data_ptr(), ldq, T, H, cache._struct(), page_table.data_ptr(), max_pages, cu_q.data_ptr(), kv_len.data_ptr(),
        B, _scale(scale, D), mq, mkv, out.data_ptr(), ldo, None if scratch is None else scratch.data_ptr(), nbytes,
        _error_word(dev, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_paged_attention")
    return out


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, T: int, H: int, Hkv: int, D: int, B: int, max_q: int, max_kv: int) -> int:
    return int(N.lib().btl_paged_attention_scratch_bytes(T, H, Hkv, D, B, max_q, max_kv))


def check(device=None) -> None:
    """Raise RuntimeError if a call since the last check met a batch that is not
    well formed (or any other launch on the device set its error word);
    synchronises the device."""
    N.check_errors(device)
