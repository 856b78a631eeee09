"""Products of 8-bit integers with a scale for each row (token) and each column
(channel), on gfx950 (include/btl.h, "products of 8-bit integers"):

    out[m, n] = (sum_k a[m, k] w[n, k]) a_scale[m] w_scale[n]

The sum is exact.  For layers that are not ternary: the LM head (lm_head.LMHead,
``weight_dtype="int8"``) streams half the bytes of its bf16 form.  Rows are quantised as
the ternary layers quantise theirs (:func:`quantize_rows`).  The reference's
8-bit weights (``bfp8``) are a Tensix block format.

Calls are ordered on the current stream of their tensors' device and use no workspace.
"""

from __future__ import annotations

from . import _native as N


class Int8Weight:
    """An [out_features, in_features] weight of 8-bit integers in the device layout
    with its scales, fp32 [out_features].  in_features: a multiple of 16 up to 16384."""

    __slots__ = ("data", "scale", "out_features", "in_features")

    def __init__(self, data, scale, out_features: int, in_features: int) -> None:
        self.data, self.scale, self.out_features, self.in_features = data, scale, out_features, in_features

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel() + 4 * self.out_features

    @classmethod
    def _empty(cls, shape, device):
        import torch

        n, k = shape
        nbytes = int(N.lib().btl_int8_weight_bytes(n, k))
        if nbytes <= 0:
            raise ValueError(f"weight ({n}, {k}): in_features must be a multiple of 16 up to {N.MAX_K}")
        return cls(torch.empty(nbytes, dtype=torch.uint8, device=device),
                   torch.empty(n, dtype=torch.float32, device=device), n, k)

    @classmethod
    def from_codes(cls, codes, scale) -> "Int8Weight":
        """codes int8 [out, in] (rows may be strided) and scale fp32 [out], on the device; both are copied."""
        import torch

        if codes.dtype is not torch.int8 or codes.dim() != 2:
            raise ValueError("codes must be int8 [out_features, in_features]")
        if scale.dtype is not torch.float32 or tuple(scale.shape) != (codes.shape[0],):
            raise ValueError(f"scale must be fp32 [{codes.shape[0]}]")
        index = _gpu(codes, "codes")
        if scale.get_device() != index:
            raise ValueError(f"codes are on {codes.device}, scale on {scale.device}")
        with torch.cuda.device(index):
            n, k = codes.shape
            w = cls._empty((n, k), codes.device)
            if codes.stride(1) != 1 or codes.stride(0) < k or codes.stride(0) % 16 or codes.data_ptr() % 16:
                codes = codes.contiguous()
                if codes.data_ptr() % 16:
                    codes = codes.clone()
            w.scale.copy_(scale)
            N.check(N.lib().btl_int8_weight_layout(codes.data_ptr(), codes.stride(0) if n > 1 else k, n, k,
                                                   w.data.data_ptr(), N.raw_stream(index)), "btl_int8_weight_layout")
        return w

    @classmethod
    def quantize(cls, weight) -> "Int8Weight":
        """A float weight [out, in] on the device: scale max|w| / 127 of each row, codes
        round(w / scale).  A row with a value that is not finite has a NaN scale."""
        import torch

        if weight.dim() != 2 or not weight.is_floating_point():
            raise ValueError("weight must be a float tensor [out_features, in_features]")
        index = _gpu(weight, "weight")
        with torch.cuda.device(index):
            if weight.dtype not in (torch.float32, torch.bfloat16):
                weight = weight.to(torch.float32)
            weight = weight.contiguous()
            n, k = weight.shape
            w = cls._empty((n, k), weight.device)
            N.check(N.lib().btl_int8_weight_quantise(weight.data_ptr(), int(weight.dtype is torch.bfloat16), k, n, k,
                                                     w.data.data_ptr(), w.scale.data_ptr(), N.raw_stream(index)),
                    "btl_int8_weight_quantise")
        return w


def _gpu(t, name):
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a tensor on a ROCm GPU device; this path runs only through the gfx950 kernels")
    return index


def int8_matmul(a, a_scale, weight: Int8Weight, out_dtype=None, out=None):
    """a int8 [..., in_features] and a_scale fp32 [...] -> bf16 (or ``out_dtype`` fp32)
    [..., out_features].  The rows of a two-dimensional ``a`` (and of ``out``, [M, out_features],
    which must not overlap the inputs) may be strided; a's rows must be 16-byte aligned."""
    import torch

    index = _gpu(a, "a")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return int8_matmul(a, a_scale, weight, out_dtype, out)
    shape, K, Nf = a.shape, weight.in_features, weight.out_features
    if a.dtype is not torch.int8 or len(shape) < 1 or shape[-1] != K:
        raise ValueError(f"a must be int8 [..., {K}]")
    if a_scale.dtype is not torch.float32 or a_scale.shape != shape[:-1] or not a_scale.is_contiguous():
        raise ValueError(f"a_scale must be contiguous fp32 {list(shape[:-1])}")
    if weight.data.get_device() != index or a_scale.get_device() != index:
        raise ValueError(f"a is on {a.device}, a_scale on {a_scale.device}, the weight on {weight.device}")
    M = a_scale.numel()
    lda = K
    if len(shape) == 2 and M > 1:
        lda = a.stride(0)
        if (a.stride(1) != 1 and K > 1) or lda < K:
            raise ValueError("a: the values of a row must be dense and rows must not overlap")
    elif not a.is_contiguous():
        raise ValueError("a must be contiguous, or two-dimensional with dense rows")
    if lda % 16 or a.data_ptr() % 16:
        raise ValueError("a: rows must be 16-byte aligned")
    if out is None:
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        out = a.new_empty((*shape[:-1], Nf), dtype=out_dtype)
        ldo = Nf
    else:
        if out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        if out.shape != (*shape[:-1], Nf):
            raise ValueError(f"out must be {[*shape[:-1], Nf]}")
        if out.get_device() != index:
            raise ValueError(f"out is on {out.device}, a on {a.device}")
        ldo = Nf
        if len(shape) == 2 and M > 1:
            ldo = out.stride(0)
            if (out.stride(1) != 1 and Nf > 1) or ldo < Nf:
                raise ValueError("out: the values of a row must be dense and rows must not overlap")
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous, or two-dimensional with dense rows")
    if out.dtype is not torch.bfloat16 and out.dtype is not torch.float32:
        raise ValueError("the output is bfloat16 or float32")
    rc = N.lib().btl_int8_matmul(a.data_ptr(), lda, a_scale.data_ptr(), M, K, Nf, weight.data.data_ptr(),
                                 weight.scale.data_ptr(), out.data_ptr(), ldo, 1 if out.dtype is torch.float32 else 0,
                                 N.raw_stream(index))
    if rc != N.BTL_OK:
        N.check(rc, "btl_int8_matmul")
    return out


def quantize_rows(x, norm_weight=None, norm_epsilon: float | None = None):
    """Rows of bf16 [..., K] as the ternary layers quantise them: (codes int8 [..., K],
    scales fp32 [...], the largest magnitude / 127), behind an RMSNorm where
    ``norm_weight`` bf16 [K] and ``norm_epsilon`` are given.  K a multiple of 32."""
    import torch

    index = _gpu(x, "x")
    N.require_cuda(x, "x")
    if x.dtype is not torch.bfloat16 or x.dim() < 1:
        raise ValueError("x must be bf16 [..., K]")
    K = x.shape[-1]
    gamma, eps = None, 0.0
    if norm_weight is not None:
        if norm_epsilon is None:
            raise ValueError("norm_weight needs norm_epsilon")
        N.require_cuda(norm_weight, "norm_weight")
        if norm_weight.dtype is not torch.bfloat16 or norm_weight.numel() != K or norm_weight.get_device() != index:
            raise ValueError("norm_weight must be bf16 with K elements, on the device of x")
        gamma, eps = norm_weight.data_ptr(), float(norm_epsilon)
    with torch.cuda.device(index):
        codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        M = x.numel() // K if K else 0
        if M == 0:
            return codes, torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        L = N.lib()
        blocked = torch.empty(int(L.btl_act_bytes(M, K)), dtype=torch.int8, device=x.device)
        scale = torch.empty((M + 31) // 32 * 32, dtype=torch.float32, device=x.device)
        N.check(L.btl_quant_absmax(x.data_ptr(), M, K, K, gamma, eps, blocked.data_ptr(), scale.data_ptr(), None, None,
                                   codes.data_ptr(), None, N.raw_stream(index)), "btl_quant_absmax")
    return codes, scale[:M].view(x.shape[:-1])
