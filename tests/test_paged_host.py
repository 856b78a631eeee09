"""Prompts and the paged cache without a GPU: argument checks of the C entry points
and of the Python layer, and the functions that place a position."""

import ctypes
import random

import pytest
import torch

from bitnet_tt import _native as N
from bitnet_tt import paged_attention as pa


@pytest.fixture(scope="module")
def L():
    return N.lib()


FAKE = 1 << 20  # never followed: every call here is refused before a launch


def pages(**kw):
    d = dict(k=FAKE, v=FAKE, k_exp=None, v_exp=None, num_pages=8, num_kv_heads=2, page_size=16, head_dim=64)
    d.update(kw)
    return N.Pages(*d.values())


def rope(L, **kw):
    a = dict(qkv=FAKE, T=4, ldx=512, H=4, Hkv=2, D=64, cos=FAKE, sin=FAKE, R=64, S=32, adj=0, cu=FAKE, kv=FAKE, B=2, q=FAKE,
             ldq=256, k=None, ldk=0, pages=pages(), table=FAKE, max_pages=2, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_rope_write(*a.values())


def read(L, **kw):
    a = dict(pages=pages(), table=FAKE, B=2, max_pages=2, kv=FAKE, S=32, k=FAKE, v=FAKE, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_read_pages(*a.values())


def prompt(L, **kw):
    a = dict(q=FAKE, ldq=256, k=FAKE, ldk=128, v=FAKE, ldv=128, T=4, H=4, Hkv=2, D=64, cu=FAKE, B=2, scale=0.125, max_q=4,
             out=FAKE, ldo=256, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_prompt_attention(*a.values())


def paged(L, **kw):
    a = dict(q=FAKE, ldq=256, T=4, H=4, pages=pages(), table=FAKE, max_pages=2, cu=FAKE, kv=FAKE, B=2, scale=0.125,
             max_q=4, max_kv=32, out=FAKE, ldo=256, scratch=None, nbytes=0, err=FAKE, stream=None)
    a.update(kw)
    return L.btl_paged_attention(*a.values())


NULL, SHAPE, ALIGN, WORKSPACE, ARG = 1, 2, 3, 4, 5


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(D=96)), (SHAPE, dict(D=256)), (SHAPE, dict(H=0)), (SHAPE, dict(H=5)), (SHAPE, dict(Hkv=0)),
    (SHAPE, dict(R=8)), (SHAPE, dict(R=72)), (SHAPE, dict(R=128)), (SHAPE, dict(S=0)), (SHAPE, dict(B=0)),
    (SHAPE, dict(T=-1)), (SHAPE, dict(T=1 << 25)), (SHAPE, dict(ldx=504)), (SHAPE, dict(ldq=248)),
    (ALIGN, dict(qkv=FAKE + 2)), (ALIGN, dict(ldx=516)), (ALIGN, dict(cos=FAKE + 4)), (ALIGN, dict(ldq=260)),
    (NULL, dict(qkv=None)), (NULL, dict(cu=None)), (NULL, dict(q=None)), (NULL, dict(err=None)), (NULL, dict(sin=None)),
    (NULL, dict(table=None)), (NULL, dict(pages=pages(k=None))), (NULL, dict(pages=pages(k_exp=FAKE))),
    (SHAPE, dict(pages=pages(page_size=24))), (SHAPE, dict(pages=pages(page_size=8))),
    (SHAPE, dict(pages=pages(num_pages=0))), (SHAPE, dict(pages=pages(num_kv_heads=3))),
    (SHAPE, dict(pages=pages(head_dim=128))), (ALIGN, dict(pages=pages(v=FAKE + 8))),
    (SHAPE, dict(k=FAKE, ldk=64)), (ALIGN, dict(k=FAKE + 2, ldk=128)), (SHAPE, dict(max_pages=-1)),
])
def test_rope_write_refuses(L, want, kw):
    assert rope(L, **kw) == want
    assert b"btl_rope_write" in L.btl_last_error()


@pytest.mark.parametrize("want,kw", [
    (NULL, dict(pages=None)), (NULL, dict(table=None)), (NULL, dict(kv=None)), (NULL, dict(k=None)), (NULL, dict(err=None)),
    (SHAPE, dict(B=0)), (SHAPE, dict(B=70000)), (SHAPE, dict(S=0)), (SHAPE, dict(max_pages=0)),
    (SHAPE, dict(S=2 ** 31 - 1)), (ALIGN, dict(v=FAKE + 2)), (SHAPE, dict(pages=pages(head_dim=80))),
])
def test_read_pages_refuses(L, want, kw):
    assert read(L, **kw) == want


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(D=80)), (SHAPE, dict(H=5)), (SHAPE, dict(H=130, Hkv=2, ldq=130 * 64, ldo=130 * 64)), (SHAPE, dict(B=0)),
    (SHAPE, dict(ldk=64)), (SHAPE, dict(ldo=128)), (SHAPE, dict(max_q=-1)), (ALIGN, dict(ldv=132)), (ALIGN, dict(q=FAKE + 8)),
    (ARG, dict(scale=0.0)), (ARG, dict(scale=-1.0)), (ARG, dict(scale=float("nan"))), (ARG, dict(scale=float("inf"))),
    (NULL, dict(k=None)), (NULL, dict(out=None)), (NULL, dict(cu=None)), (NULL, dict(err=None)),
    (SHAPE, dict(T=1 << 24, H=128, Hkv=2, ldq=8192, ldo=8192)),
])
def test_prompt_attention_refuses(L, want, kw):
    assert prompt(L, **kw) == want


@pytest.mark.parametrize("want,kw", [
    (NULL, dict(pages=None)), (NULL, dict(table=None)), (NULL, dict(kv=None)), (NULL, dict(err=None)),
    (SHAPE, dict(H=5)), (SHAPE, dict(max_q=0)), (SHAPE, dict(max_kv=0)), (SHAPE, dict(max_pages=0)),
    (SHAPE, dict(max_pages=1 << 24, pages=pages(page_size=1 << 20))), (ARG, dict(scale=0.0)), (ALIGN, dict(out=FAKE + 2)),
    (WORKSPACE, dict(max_pages=512, max_kv=8192)), (WORKSPACE, dict(max_pages=512, max_kv=8192, scratch=FAKE, nbytes=64)),
    (SHAPE, dict(B=70000, T=70000, max_q=1)),
])
def test_paged_attention_refuses(L, want, kw):
    assert paged(L, **kw) == want


def test_no_rows_is_no_launch(L):
    assert rope(L, T=0) == 0 and prompt(L, T=0) == 0 and paged(L, T=0) == 0


def test_scratch_bytes(L):
    f = L.btl_paged_attention_scratch_bytes
    assert f(32, 20, 5, 128, 32, 1, 512) == 0  # a context that is not worth a split
    n = f(1, 20, 5, 128, 1, 1, 131072)
    assert n > 0 and n % (20 * 130 * 4) == 0
    assert f(0, 20, 5, 128, 1, 1, 4096) == 0 and f(1, 20, 3, 128, 1, 1, 4096) == 0
    assert f(32, 20, 5, 128, 32, 1, 4096) > f(300, 20, 5, 128, 300, 1, 4096) == 0  # 160 workgroups, 1500


def plan(L, *sizes):
    out = (ctypes.c_int64 * 3)()
    assert L.btl_paged_attention_plan(*sizes, out) == 1
    return tuple(out)


@pytest.mark.parametrize("T,B,max_q", [(1, 1, 1), (32, 32, 1), (67, 1, 67), (2047, 4, 700), (3, 1, 2 ** 62)])
@pytest.mark.parametrize("D", [64, 128])
def test_plan_of_any_hint(L, T, B, max_q, D):
    """The kernels' positions are 32-bit numbers: the end of the last split stays below 2^31, however far
    behind the page table's room the hint is, and the scratch is that of the splits that run."""
    for max_kv in (1, 255, 1024, 40067, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 7, 3 * 2 ** 31, 2 ** 33 + 2 ** 31,
                   2 ** 40, 2 ** 62, 2 ** 63 - 1):
        sizes = (T, 20, 5, D, B, max_q, max_kv)
        few, splits, chunk = plan(L, *sizes)
        assert 1 <= splits <= 256 and 256 <= chunk <= 2 ** 30 and splits * chunk < 2 ** 31
        assert splits * chunk >= min(max_kv, 2 ** 30 - 1)
        assert L.btl_paged_attention_scratch_bytes(*sizes) == (splits * T * 20 * (D + 2) * 4 if splits > 1 else 0)
        if max_kv >= 2 ** 30:
            assert (few, splits, chunk) == plan(L, T, 20, 5, D, B, max_q, 2 ** 30 - 1)
    assert plan(L, T, 20, 5, D, B, max_q, 4096)[0] == (min(max_q, T) * 4 <= 16)


@pytest.mark.parametrize("sizes", [
    (1 << 10, 16, 16, 64, 1 << 60, 1, 4096), (1, 1 << 62, 1 << 62, 128, 4, 1, 1 << 17), (1 << 62, 20, 5, 128, 32, 1, 1 << 17),
    (1 << 24, 128, 2, 64, 4, 1, 1 << 17), (1, 130, 2, 64, 1, 1, 1 << 17), (1, 20, 5, 96, 1, 1, 1 << 17),
    (1, 20, 5, 128, (1 << 20) + 1, 1, 1 << 17), (1, 20, 5, 128, 1, -1, 1 << 17), (1, 20, 5, 128, 1, 1, -2 ** 63),
])
def test_scratch_of_sizes_that_no_call_takes(L, sizes):
    assert L.btl_paged_attention_scratch_bytes(*sizes) == 0
    assert L.btl_paged_attention_plan(*sizes, (ctypes.c_int64 * 3)()) == 0


def test_page_of_a_position(L):
    """The division by multiplication, and pages outside the pool."""
    r = random.Random(1)
    sizes = [16, 32, 48, 80, 1008, 4096, 65520, 1 << 20] + [16 * r.randint(1, 1 << 16) for _ in range(200)]
    for ps in sizes:
        for p in [0, 1, ps - 1, ps, ps + 1, 2 ** 31 - 1, 2 ** 31 - 2] + [r.randint(0, 2 ** 31 - 1) for _ in range(20)]:
            assert L.btl_page_row(7, 9, 5, 3, ps, p) == (7 * 5 + 3) * ps + p % ps
            k = p // ps * ps  # the last and first positions of a page
            if k:
                assert L.btl_page_row(0, 1, 1, 0, ps, k) == 0 and L.btl_page_row(0, 1, 1, 0, ps, k - 1) == ps - 1
    for page in (-1, 9, 2 ** 31 - 1, -2 ** 31):
        assert L.btl_page_row(page, 9, 5, 3, 64, 70) == -1
    # far pages: more than 2^32 rows
    assert L.btl_page_row(2 ** 31 - 2, 2 ** 31 - 1, 8, 7, 256, 255) == ((2 ** 31 - 2) * 8 + 7) * 256 + 255


def test_run_of_positions(L):
    """What attention places its rows with: as btl_page_row, whatever the pool's size."""
    out = (ctypes.c_int64 * 2)()

    def f(*a):
        return L.btl_page_run(*a, out), tuple(out)

    r = random.Random(3)
    for _ in range(3000):
        ps = 16 * r.choice([1, 2, 3, 4, 16, 63, 4096, 65536, r.randint(1, 65536)])
        heads = r.choice([1, 2, 5, 8, 128, 1024])
        P = r.choice([1, 9, 1 << 20, 2 ** 31 - 1])
        page = r.choice([0, P - 1, r.randrange(P)])
        hk, at = r.randrange(heads), 16 * r.randrange(2 ** 26)
        most = r.choice([16, 32, 64])
        end = min(2 ** 31 - 1, max(0, at + r.randint(-40, 80)))
        left = max(0, min(most, end - at))
        assert f(page, P, heads, hk, ps, at, end, most) == (0, ((page * heads + hk) * ps + at % ps, left))
        assert L.btl_page_row(page, P, heads, hk, ps, at) == out[0]
        for outside in (-1, P, 2 ** 31 - 1, -2 ** 31):
            if outside != page and not 0 <= outside < P:
                bad, (row, n) = f(outside, P, heads, hk, ps, at, end, most)
                assert (bad, n) == (left > 0, 0) and 0 <= row < heads * ps
    assert L.btl_page_run(0, 1, 1, 1, 16, 0, 1, 16, out) == -1 and L.btl_page_run(0, 1, 1, 0, 8, 0, 1, 16, out) == -1


def test_clamped_sequences(L):
    out = (ctypes.c_int64 * 3)()

    def f(lo, hi, n, T=100, cap=64):
        ok = L.btl_clamp_seq(lo, hi, n, T, cap, out)
        return ok, tuple(out)

    assert f(0, 10, 20) == (1, (0, 10, 20))
    assert f(10, 10, 0) == (1, (10, 0, 0))
    assert f(10, 4, 20) == (0, (10, 0, 20))
    assert f(90, 200, 20) == (0, (90, 10, 20))
    assert f(-5, 10, 20) == (0, (0, 10, 20))
    assert f(500, 600, 20) == (0, (100, 0, 20))
    assert f(0, 10, 65) == (0, (0, 10, 0))
    assert f(0, 10, -1) == (0, (0, 10, 0))


def test_rows_without_lengths_stay_in_their_buffer(L):
    """Prompts have no lengths: a sequence's positions are its rows as clamped, whatever the offsets say,
    so that no key or value row from T on is read."""
    out = (ctypes.c_int64 * 3)()

    def f(lo, hi, T):
        return L.btl_clamp_seq(lo, hi, 0, T, -1, out), tuple(out)

    assert f(0, 40, 50) == (1, (0, 40, 40)) and f(50, 50, 50) == (1, (50, 0, 0))
    assert f(40, 60, 50) == (0, (40, 10, 10))
    assert f(-2 ** 31, 2 ** 31 - 1, 50) == (0, (0, 50, 50))
    r = random.Random(4)
    some = [0, 1, -1, 2 ** 31 - 1, -2 ** 31]
    for _ in range(5000):
        T = r.choice([0, 1, 50, 1 << 24])
        lo, hi = (r.choice(some + [T, T + 1, r.randint(-60, 120), r.randint(0, T)]) for _ in range(2))
        ok, (row0, n, length) = f(lo, hi, T)
        assert 0 <= row0 <= row0 + n <= T and length == n
        assert ok == (0 <= lo <= hi <= T)


def test_row_exponent(L):
    f = L.btl_row_exponent
    assert f(448.0) == 0 and f(1.75) == -8 and f(1.7500001) == -7 and f(0.0) == -126 and f(1e-40) == -126
    r = random.Random(2)
    for _ in range(2000):
        a = ctypes.c_float(r.uniform(0.5, 1) * 2.0 ** r.randint(-110, 126)).value
        e = f(a)
        assert a <= 448 * 2.0 ** e and (a > 448 * 2.0 ** (e - 1))


# ---- Python layer -----------------------------------------------------------


def test_host_tensors_are_refused():
    bf = torch.zeros((4, 8 * 64), dtype=torch.bfloat16)
    i32 = torch.zeros(3, dtype=torch.int32)
    f32 = torch.zeros((8, 32))
    with pytest.raises(ValueError, match="ROCm GPU"):
        pa.rope_write(bf, f32, f32, i32, i32[:2], 4, 2)
    x = bf.view(4, 8, 64)
    with pytest.raises(ValueError, match="ROCm GPU"):
        pa.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], i32)
    with pytest.raises(ValueError, match="ROCm GPU"):
        pa.PagedKVCache(torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16))


def test_cache_arguments():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)  # noqa: E731
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(ValueError, match="alike"):
        pa.PagedKVCache(z(2, 2, 16, 64), z(2, 2, 32, 64))
    with pytest.raises(ValueError, match="together"):
        pa.PagedKVCache(z(2, 2, 16, 64), z(2, 2, 16, 64), u8(2, 2, 16))
    with pytest.raises(ValueError, match="pages must be"):
        pa.PagedKVCache(z(2, 2, 16, 64), z(2, 2, 16, 64), u8(2, 2, 16), u8(2, 2, 16))
    with pytest.raises(ValueError, match="multiple of 16"):
        pa.PagedKVCache(z(2, 2, 24, 64), z(2, 2, 24, 64))
    with pytest.raises(ValueError, match="head_dim"):
        pa.PagedKVCache(z(2, 2, 16, 80), z(2, 2, 16, 80))
    with pytest.raises(ValueError, match="cache dtype"):
        pa.PagedKVCache.allocate(2, 2, 64, "cpu", dtype="int4")
