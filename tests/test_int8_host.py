"""Products of 8-bit integers without a GPU: sizes and argument checks."""

import pytest
import torch

from bitnet_tt import _native as N
from bitnet_tt.int8_matmul import Int8Weight, int8_matmul, quantize_rows
from bitnet_tt.lm_head import LMHead


@pytest.fixture(scope="module")
def L():
    return N.lib()


FAKE = 1 << 20  # never followed: every call here is refused before a launch
NULL, SHAPE, ALIGN, WORKSPACE, ARG = 1, 2, 3, 4, 5


def matmul(L, **kw):
    a = dict(a=FAKE, lda=64, sa=FAKE, M=4, K=64, N=10, w=FAKE, sw=FAKE, out=FAKE, ldo=10, f32=1, stream=None)
    a.update(kw)
    return L.btl_int8_matmul(*a.values())


def head(L, **kw):
    a = dict(x=FAKE, M=4, K=64, N=10, gamma=FAKE, eps=1e-5, w=FAKE, sw=FAKE, normed=None, out=FAKE, tokens=FAKE, scratch=FAKE,
             nbytes=1 << 40, stream=None)
    a.update(kw)
    return L.btl_int8_head(*a.values())


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(K=0)), (SHAPE, dict(K=24)), (SHAPE, dict(K=16400, lda=16400)), (SHAPE, dict(N=0)), (SHAPE, dict(N=(1 << 24) + 1)),
    (SHAPE, dict(M=-1)), (SHAPE, dict(M=(1 << 24) + 1)), (SHAPE, dict(lda=48)), (SHAPE, dict(lda=(1 << 22) + 16)),
    (SHAPE, dict(ldo=9)), (ALIGN, dict(lda=72)), (ALIGN, dict(a=FAKE + 8)), (ALIGN, dict(w=FAKE + 8)), (ALIGN, dict(out=FAKE + 2)),
    (ALIGN, dict(sa=FAKE + 1)), (ALIGN, dict(sw=FAKE + 2)), (NULL, dict(a=None)), (NULL, dict(sa=None)), (NULL, dict(w=None)),
    (NULL, dict(sw=None)), (SHAPE, dict(M=1 << 24, N=1 << 24, ldo=1 << 24)),
    (NULL, dict(out=None)), (ALIGN, dict(out=FAKE + 1, f32=0)),
])
def test_matmul_refuses(L, want, kw):
    assert matmul(L, **kw) == want
    assert b"btl_int8_matmul" in L.btl_last_error()


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(M=65536)), (SHAPE, dict(M=-1)), (SHAPE, dict(K=0)), (SHAPE, dict(K=48)), (SHAPE, dict(K=16416)), (SHAPE, dict(N=0)),
    (SHAPE, dict(N=(1 << 24) + 1)), (NULL, dict(x=None)), (NULL, dict(gamma=None)), (NULL, dict(w=None)), (NULL, dict(sw=None)),
    (NULL, dict(tokens=None)), (NULL, dict(scratch=None)), (NULL, dict(out=None, M=65)), (ALIGN, dict(x=FAKE + 8)),
    (ALIGN, dict(gamma=FAKE + 2)), (ALIGN, dict(normed=FAKE + 8)), (ALIGN, dict(scratch=FAKE + 64)), (ALIGN, dict(tokens=FAKE + 2)),
    (ALIGN, dict(w=FAKE + 8)), (ALIGN, dict(sw=FAKE + 2)), (ALIGN, dict(out=FAKE + 2)), (WORKSPACE, dict(nbytes=1024)),
])
def test_head_refuses(L, want, kw):
    assert head(L, **kw) == want
    assert b"btl_int8_head" in L.btl_last_error()


def test_no_rows_is_no_launch(L):
    assert matmul(L, M=0, a=None, out=None) == 0 and head(L, M=0, x=None) == 0


def test_sizes(L):
    f = L.btl_int8_weight_bytes
    assert f(128256, 2560) == 128256 * 2560 and f(1, 16) == 1024 and f(17, 80) == 2 * 2 * 1024
    assert f(10, 8) == 0 and f(10, 16400) == 0 and f(0, 64) == 0 and f(-5, 64) == 0 and f((1 << 24) + 1, 64) == 0
    g = L.btl_int8_head_scratch_bytes
    for bad in ((0, 64, 10), (65536, 64, 10), (4, 48, 10), (4, 16416, 10), (4, 64, 0), (-1, 64, 10), (4, 64, (1 << 24) + 1)):
        assert g(*bad) == 0
    for M in (1, 64, 65, 1000, 65535):  # the cleared words, codes twice, scales
        assert g(M, 2560, 128256) >= 1024 + M * 2560 + L.btl_act_bytes(M, 2560) + 4 * M


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(K=8)), (SHAPE, dict(N=0)), (SHAPE, dict(ldw=32)), (ALIGN, dict(ldw=72)), (ALIGN, dict(w=FAKE + 4)), (NULL, dict(w=None)),
    (NULL, dict(out=None)),
])
def test_layout_refuses(L, want, kw):
    a = dict(w=FAKE, ldw=64, N=10, K=64, out=FAKE, stream=None)
    a.update(kw)
    assert L.btl_int8_weight_layout(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(K=8)), (SHAPE, dict(ldw=32)), (ALIGN, dict(w=FAKE + 2)), (NULL, dict(scale=None)), (ALIGN, dict(out=FAKE + 4)),
    (ALIGN, dict(w=FAKE + 1, bf16=1)),
])
def test_quantise_refuses(L, want, kw):
    a = dict(w=FAKE, bf16=0, ldw=64, N=10, K=64, out=FAKE, scale=FAKE, stream=None)
    a.update(kw)
    assert L.btl_int8_weight_quantise(*a.values()) == want


def test_python_refuses():
    codes, scale = torch.zeros((4, 64), dtype=torch.int8), torch.ones(4)
    with pytest.raises(ValueError, match="ROCm GPU"):
        Int8Weight.from_codes(codes, scale)
    with pytest.raises(ValueError, match="int8"):
        Int8Weight.from_codes(codes.float(), scale)
    with pytest.raises(ValueError, match="scale"):
        Int8Weight.from_codes(codes, torch.ones(5))
    with pytest.raises(ValueError, match="ROCm GPU"):
        Int8Weight.quantize(codes.float())
    with pytest.raises(ValueError, match="float"):
        Int8Weight.quantize(codes)
    with pytest.raises(ValueError, match="ROCm GPU"):
        int8_matmul(codes, scale, None)
    with pytest.raises(ValueError, match="ROCm GPU"):
        quantize_rows(codes.to(torch.bfloat16))
    with pytest.raises(ValueError, match="in_features"):
        Int8Weight._empty((4, 24), "cpu")
    with pytest.raises(ValueError, match="weight_dtype"):
        LMHead(64, 10, "cpu", weight_dtype="bfp8")
