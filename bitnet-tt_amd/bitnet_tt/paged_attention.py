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

Sequences may share pages that they only read; two rows of one call that are
written must not be the same row of the same page, nor may outputs overlap pages.

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
_ERROR_KIND = "paged"


class PagedKVCache:
    """One layer's page pools: ``key_pages`` and ``value_pages`` [num_pages,
    kv_heads, page_size, head_dim] bf16, or float8_e4m3fn with one exponent byte
    per row in ``key_exp`` and ``value_exp`` [num_pages, kv_heads, page_size]
    uint8 (a value is code x 2^(byte - 127), bytes 1 .. 247).  page_size is a multiple of 16;
    head_dim 64 or 128.  The pools are written in place, never replaced.  The
    contiguous caches of DecodeAttention are pages of max_seq_len rows: :meth:`of_cache`."""

    __slots__ = ("_tensors", "_pages", "shape", "index")

    def __init__(self, key_pages, value_pages, key_exp=None, value_exp=None) -> None:
        shape = key_pages.shape
        if len(shape) != 4 or value_pages.shape != shape:
            raise ValueError("key_pages and value_pages must be [num_pages, kv_heads, page_size, head_dim], alike")
        P, H, S, D = shape
        fp8 = key_exp is not None
        if (value_exp is not None) != fp8:
            raise ValueError("key_exp and value_exp come together")
        dtype = torch.float8_e4m3fn if fp8 else _BF16
        if key_pages.dtype is not dtype or value_pages.dtype is not dtype:
            raise ValueError(f"pages must be {dtype} {'with' if fp8 else 'without'} exponent bytes")
        if S < 16 or S % 16:
            raise ValueError(f"page_size {S} is not a multiple of 16")
        if D != 128 and D != 64:
            raise ValueError(f"head_dim {D}: 64 and 128 are supported")
        N.require_cuda(key_pages, "key_pages")
        N.require_cuda(value_pages, "value_pages")
        index = key_pages.get_device()
        if fp8:
            for t, name in ((key_exp, "key_exp"), (value_exp, "value_exp")):
                N.require_cuda(t, name)
                if t.dtype is not torch.uint8 or t.shape != shape[:3]:
                    raise ValueError(f"{name} must be uint8 [num_pages, kv_heads, page_size]")
                if t.get_device() != index:
                    raise ValueError("the pools are on different devices")
        if value_pages.get_device() != index:
            raise ValueError("the pools are on different devices")
        self._tensors = (key_pages, value_pages, key_exp, value_exp)
        self._pages = N.Pages(key_pages.data_ptr(), value_pages.data_ptr(), key_exp.data_ptr() if fp8 else None,
                              value_exp.data_ptr() if fp8 else None, P, H, S, D)
        self.shape = shape
        self.index = index

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

    key_pages = property(lambda self: self._tensors[0])
    value_pages = property(lambda self: self._tensors[1])
    key_exp = property(lambda self: self._tensors[2])
    value_exp = property(lambda self: self._tensors[3])
    num_pages = property(lambda self: self.shape[0])
    num_kv_heads = property(lambda self: self.shape[1])
    page_size = property(lambda self: self.shape[2])
    head_dim = property(lambda self: self.shape[3])
    device = property(lambda self: self._tensors[0].device)


def _int32(t, index, shape, name):
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call's tensors on cuda:{index}")


def _sequences(cu_q, index):
    """B, of cu_q [B + 1]."""
    shape = cu_q.shape
    if len(shape) != 1 or shape[0] < 2:
        raise ValueError("cu_q must be int32 [B + 1] of at least one sequence")
    _int32(cu_q, index, shape, "cu_q")
    return shape[0] - 1


def _table(page_table, index, B):
    """max_pages, of page_table [B, max_pages]."""
    shape = page_table.shape
    if len(shape) != 2 or shape[0] != B or shape[1] < 1:
        raise ValueError(f"page_table must be int32 [{B}, max_pages]")
    _int32(page_table, index, shape, "page_table")
    return shape[1]


def _rows(t, T, heads, dim, name, index):
    """Row stride of a packed bf16 tensor [T, heads, dim] whose rows are dense."""
    shape = t.shape
    if t.dtype is not _BF16 or len(shape) != 3 or shape[0] != T or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{name} must be bf16 [{T}, {heads}, {dim}]")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call's tensors on cuda:{index}")
    ld, sh, sd = t.stride()
    if sd != 1 or (sh != dim and heads > 1):
        raise ValueError(f"{name}: the heads of a row must be dense")
    if T <= 1:  # its stride says nothing
        ld = heads * dim
    if ld < heads * dim or ld % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows must be 16-byte aligned and not overlap")
    return ld


def _gpu(t, name):
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a tensor on a ROCm GPU device; this path runs only through the gfx950 kernels")
    return index


def _error_word(index, stream):
    """Address of the stream's error word."""
    hit = N._fast.get((_ERROR_KIND, index, stream, 0, 0))
    if hit is None:
        device = torch.device("cuda", index)
        if not N.has_workspace(device, _ERROR_BYTES, _ERROR_KIND) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("run one eager call on this stream before capturing it in a graph")
        hit = N.workspace_ptr(index, _ERROR_BYTES, _ERROR_KIND, 0, stream)
    return hit[0]


def rope_write(qkv, rope_cos, rope_sin, cu_q, kv_len, num_heads: int, num_kv_heads: int, cache: PagedKVCache | None = None,
               page_table=None, rope_adjacent: bool = False, q_out=None, k_out=None):
    """Rotates the q and k heads of fused QKV rows and writes k and v to their pages.

    qkv: bf16 [T, (H + 2 Hkv) D].  rope_cos / rope_sin: fp32 [S, R / 2], the
    angles of the first R dims of a head (pairs (i, i + R/2), or (2i, 2i+1) with
    ``rope_adjacent``); see utils.rope.rope_tables.  kv_len None: whole prompts,
    positions from 0.  Without ``cache`` nothing but q (and k_out) is written.  An
    8-bit row keeps the least exponent e with max|x| <= 448 * 2^e and is rounded
    once, from the fp32 rotation; a row with a value that is not finite reads
    back as NaN.  Returns q [T, H, D] (``q_out``, which may be the q part of qkv
    itself, as ``k_out`` [T, Hkv, D] may be its k part)."""
    index = _gpu(qkv, "qkv")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return rope_write(qkv, rope_cos, rope_sin, cu_q, kv_len, num_heads, num_kv_heads, cache, page_table,
                              rope_adjacent, q_out, k_out)
    H, Hkv = int(num_heads), int(num_kv_heads)
    shape, heads = qkv.shape, H + 2 * Hkv
    if qkv.dtype is not _BF16 or len(shape) != 2 or H < 1 or Hkv < 1 or shape[1] % heads or not qkv.is_contiguous():
        raise ValueError(f"qkv must be contiguous bf16 [T, ({H} + 2 * {Hkv}) * head_dim]")
    T, D = shape[0], shape[1] // heads
    angles = rope_cos.shape
    if (len(angles) != 2 or rope_sin.shape != angles or rope_cos.dtype is not torch.float32
            or rope_sin.dtype is not torch.float32 or not rope_cos.is_contiguous() or not rope_sin.is_contiguous()):
        raise ValueError("rope_cos and rope_sin must be contiguous fp32 [positions, rotated dims / 2], alike")
    if rope_cos.get_device() != index or rope_sin.get_device() != index:
        raise ValueError(f"rope_cos is on {rope_cos.device}, rope_sin on {rope_sin.device}, qkv on {qkv.device}")
    B = _sequences(cu_q, index)
    if kv_len is not None:
        _int32(kv_len, index, (B,), "kv_len")
    pages = table = None
    max_pages = 0
    if cache is not None:
        if page_table is None:
            raise ValueError("a cache needs a page table")
        if cache.shape[1] != Hkv or cache.shape[3] != D:
            raise ValueError(f"cache of {cache.shape[1]} heads of {cache.shape[3]}, rows of {Hkv} of {D}")
        if cache.index != index:
            raise ValueError(f"cache is on cuda:{cache.index}, qkv on {qkv.device}")
        max_pages = _table(page_table, index, B)
        pages, table = cache._pages, page_table.data_ptr()
    if q_out is None:
        q_out = qkv.new_empty(T, H, D)
        ldq = H * D
    else:
        ldq = _rows(q_out, T, H, D, "q_out", index)
    ldk = 0 if k_out is None else _rows(k_out, T, Hkv, D, "k_out", index)
    stream = N.raw_stream(index)
    rc = N.lib().btl_rope_write(
        qkv.data_ptr(), T, heads * D, H, Hkv, D, rope_cos.data_ptr(), rope_sin.data_ptr(), 2 * angles[1], angles[0],
        1 if rope_adjacent else 0, cu_q.data_ptr(), None if kv_len is None else kv_len.data_ptr(), B, q_out.data_ptr(),
        ldq, None if k_out is None else k_out.data_ptr(), ldk, pages, table, max_pages, _error_word(index, stream),
        stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_rope_write")
    return q_out


def read_pages(cache: PagedKVCache, page_table, kv_len, key_cache, value_cache) -> None:
    """Copies rows [0, kv_len[b]) of every sequence from its pages into the
    contiguous bf16 caches [B, Hkv, S, D] (those of layers.attention.KVCache, which
    the decode steps read); the rows behind stay as they were."""
    index = cache.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return read_pages(cache, page_table, kv_len, key_cache, value_cache)
    B = page_table.shape[0]
    if B < 1:
        raise ValueError("page_table must be int32 [B, max_pages] of at least one sequence")
    max_pages = _table(page_table, index, B)
    _int32(kv_len, index, (B,), "kv_len")
    shape, (_, Hkv, _, D) = key_cache.shape, cache.shape
    for t, name in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        if (t.dtype is not _BF16 or len(shape) != 4 or t.shape != shape or shape[0] != B or shape[1] != Hkv
                or shape[3] != D or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous bf16 [{B}, {Hkv}, positions, {D}]")
        if t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the pages on cuda:{index}")
    stream = N.raw_stream(index)
    rc = N.lib().btl_read_pages(cache._pages, page_table.data_ptr(), B, max_pages, kv_len.data_ptr(), shape[2],
                                key_cache.data_ptr(), value_cache.data_ptr(), _error_word(index, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_read_pages")


def prompt_attention(q, k, v, cu_seqlens, scale: float | None = None, max_q: int | None = None, out=None):
    """Causal attention within packed sequences: row i attends to the rows up to
    itself of its own sequence, query head h to key-value head h // (H / Hkv).

    q bf16 [T, H, D], k and v [T, Hkv, D] (parts of a QKV row will do: rows may
    be strided); cu_seqlens int32 [B + 1]; scale, positive, defaults to 1/sqrt(D); max_q,
    where known, is the longest sequence (a hint that the present kernel has no use for).  Returns bf16 [T, H, D]
    (``out``, which must not overlap the inputs)."""
    index = _gpu(q, "q")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return prompt_attention(q, k, v, cu_seqlens, scale, max_q, out)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q must be [T, H, D], k and v [T, Hkv, D]")
    T, H, D = q.shape
    Hkv = k.shape[1]
    if Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads over {Hkv} key-value heads")
    ldq = _rows(q, T, H, D, "q", index)
    ldk, ldv = _rows(k, T, Hkv, D, "k", index), _rows(v, T, Hkv, D, "v", index)
    B = _sequences(cu_seqlens, index)
    if out is None:
        out = q.new_empty(T, H, D)
        ldo = H * D
    else:
        ldo = _rows(out, T, H, D, "out", index)
    stream = N.raw_stream(index)
    rc = N.lib().btl_prompt_attention(
        q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, T, H, Hkv, D, cu_seqlens.data_ptr(), B,
        1.0 / math.sqrt(D) if scale is None else scale, T if max_q is None else max_q, out.data_ptr(), ldo,
        _error_word(index, stream), stream)
    if rc != N.BTL_OK:
        N.check(rc, "btl_prompt_attention")
    return out


def paged_attention(q, cache: PagedKVCache, page_table, cu_q, kv_len, scale: float | None = None,
                    max_q: int | None = None, max_kv: int | None = None, out=None):
    """Attention of each sequence's newest tokens over its pages: the row at
    position p attends to positions [0, p], which have been written before.

    q bf16 [T, H, D], rotated.  max_q and max_kv, where known, are the most new
    tokens and the longest kv_len of any sequence: they choose the kernel and how
    a long context is split over workgroups, and a wrong one costs time only.
    Single-token steps should pass max_q=1.  Returns bf16 [T, H, D] (``out``,
    which must not overlap q)."""
    index = cache.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return paged_attention(q, cache, page_table, cu_q, kv_len, scale, max_q, max_kv, out)
    if q.dim() != 3:
        raise ValueError("q must be [T, H, D]")
    T, H, D = q.shape
    _, Hkv, page_size, dim = cache.shape
    ldq = _rows(q, T, H, dim, "q", index)
    if H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads over {Hkv} key-value heads")
    B = _sequences(cu_q, index)
    _int32(kv_len, index, (B,), "kv_len")
    max_pages = _table(page_table, index, B)
    most = max_pages * page_size
    max_q = T if max_q is None or max_q > T else max_q
    max_kv = most if max_kv is None or max_kv > most else max_kv
    if out is None:
        out = q.new_empty(T, H, D)
        ldo = H * D
    else:
        ldo = _rows(out, T, H, D, "out", index)
    if T == 0:
        return out
    if max_q < 1 or max_kv < 1:
        raise ValueError(f"max_q {max_q} and max_kv {max_kv} must be at least 1")
    stream = N.raw_stream(index)
    nbytes = _scratch_bytes(index, T, H, Hkv, D, B, max_q, max_kv)
    # the call's own, from the stream-ordered allocator: calls that overlap share nothing
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    rc = N.lib().btl_paged_attention(
        q.data_ptr(), ldq, T, H, cache._pages, page_table.data_ptr(), max_pages, cu_q.data_ptr(), kv_len.data_ptr(), B,
        1.0 / math.sqrt(D) if scale is None else scale, max_q, max_kv, out.data_ptr(), ldo,
        None if scratch is None else scratch.data_ptr(), nbytes, _error_word(index, stream), stream)
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
