"""Final RMSNorm + LM head + greedy argmax of a decode step on gfx950.

The reference loads the head as the pre-transposed (hidden, vocab) matrix
(src/bitnet_tt/model/bitnet.py:139-215), runs ``norm`` then the head matmul on
the decode rows (src/bitnet_tt/inference/generator_batch32.py:768-811) and
takes ``ttnn.argmax`` over the vocabulary (:1170-1174).  Here the head stays
bf16 (the checkpoint's dtype; the reference's bfp8 is a Tensix block format)
in an MFMA operand layout made once at load time, and one launch streams it
for up to 32 rows, writing fp32 logits (optional) and the token ids.

``weight_dtype="int8"`` keeps 8-bit integers with a scale for each vocabulary row
instead, half the bytes: the normed rows are quantised as the ternary layers quantise
theirs, and up to 65535 rows are taken in a call (a prompt's, to score it).
"""

from __future__ import annotations

import functools
import math

import numpy as np

from . import _native as N


_ROWS = 1024  # of a pass without logits over many rows, at most
_BUFFER = 1 << 29  # bytes of such a pass's logits, for at least _FEW rows
_FEW = 64  # rows that need no logits
_MAX_ROWS = 65535


def _pass_rows(m: int, v: int) -> int:
    """Rows of a pass of the 8-bit head without logits."""
    return min(m, max(_FEW, min(_ROWS, _BUFFER // (4 * v))))


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, m: int, k: int, v: int) -> int:
    """Of an 8-bit head's call on device ``index``."""
    return int(N.lib().btl_int8_head_scratch_bytes(m, k, v))


class LMHead:
    """``norm`` + head + argmax; API pieces of bitnet.py:139-215.  ``weight_dtype``: "bf16", or
    "int8" (hidden_size a multiple of 32)."""

    def __init__(self, hidden_size: int, vocab_size: int, device=None, eps: float = 1e-5,
                 weight_dtype: str = "bf16") -> None:
        import torch

        if weight_dtype not in ("bf16", "int8"):
            raise ValueError(f"weight_dtype {weight_dtype!r}: 'bf16' or 'int8'")
        if weight_dtype == "int8" and (hidden_size % 32 or hidden_size > N.MAX_K):
            raise ValueError(f"hidden size {hidden_size}: the 8-bit head takes multiples of 32 up to {N.MAX_K}")
        self.weight_dtype = weight_dtype
        self.hidden_size = hidden_size
        self.vocab_size = vocab_size
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.eps = eps
        self.norm_weight = None
        self.weight = None  # device layout (uint8 bytes; int8: an Int8Weight)

    def load_final_weights(self, norm_weight, lm_head_weight) -> None:
        """Final norm gain [hidden] and head [vocab, hidden] (numpy or tensor,
        any float dtype; stored as bf16, or quantised from bf16 or fp32)."""
        import torch

        H, V = self.hidden_size, self.vocab_size
        g = torch.as_tensor(np.asarray(norm_weight, dtype=np.float32)) if not isinstance(norm_weight, torch.Tensor) \
            else norm_weight
        g = g.reshape(-1).to(device=self.device, dtype=torch.bfloat16).contiguous()
        if g.numel() != H:
            raise ValueError(f"norm weight has {g.numel()} elements, expected {H}")
        w = lm_head_weight if isinstance(lm_head_weight, torch.Tensor) else torch.from_numpy(
            np.ascontiguousarray(np.asarray(lm_head_weight, dtype=np.float32)))
        if tuple(w.shape) != (V, H):
            raise ValueError(f"head weight is {tuple(w.shape)}, expected ({V}, {H})")
        if self.weight_dtype == "int8":
            from .int8_matmul import Int8Weight

            self.weight = Int8Weight.quantize(w.to(self.device))
            self.norm_weight = g
            return
        w = w.to(device=self.device, dtype=torch.bfloat16).contiguous()
        L = N.lib()
        nbytes = int(L.btl_lm_head_weight_bytes(V, H))
        if nbytes <= 0:
            raise ValueError(f"unsupported head shape vocab={V} hidden={H}")
        dev = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        N.check(L.btl_lm_head_repack(N.ptr(w), V, H, N.ptr(dev), N.stream_of(self.device)), "btl_lm_head_repack")
        self.norm_weight = g
        self.weight = dev

    def __call__(self, hidden, return_logits: bool = True, normed_out=None, logits_out=None, tokens_out=None):
        """bf16 hidden [M, hidden] (M <= 32; int8: up to 65535) -> (fp32 logits [M, vocab] or None,
        int32 token ids [M]).  The ``*_out`` tensors, when given, are written
        in place.  The bf16 head then allocates nothing: it can be captured in a graph
        after one eager call on the same stream.  The 8-bit head needs no eager call; each of its calls
        allocates a scratch (about 2 M hidden bytes), and without logits for more than 64 rows
        those of a pass of up to 1024 rows, at most 512 MiB or 64 rows of them.  A captured graph keeps both."""
        import torch

        if self.weight is None:
            raise RuntimeError("Weights not loaded. Call load_final_weights() first.")
        N.require_cuda(hidden, "hidden")
        H, V = self.hidden_size, self.vocab_size
        if hidden.dtype != torch.bfloat16 or hidden.shape[-1] != H:
            raise ValueError("hidden must be bf16 [..., hidden_size]")
        M = hidden.numel() // H
        if self.weight_dtype == "int8":
            return self._int8(hidden.reshape(M, H), return_logits, normed_out, logits_out, tokens_out)
        if M > 32:
            raise ValueError(f"{M} rows: the head launch takes up to 32")
        x = hidden.reshape(M, H)
        xn = normed_out if normed_out is not None else torch.empty((M, H), dtype=torch.bfloat16, device=hidden.device)
        logits = logits_out if logits_out is not None else (
            torch.empty((M, V), dtype=torch.float32, device=hidden.device) if return_logits else None)
        tokens = tokens_out if tokens_out is not None else torch.empty(M, dtype=torch.int32, device=hidden.device)
        L = N.lib()
        index = hidden.device.index
        stream = N.raw_stream(index)
        nbytes = int(L.btl_lm_head_workspace_bytes())
        if torch.cuda.is_current_stream_capturing() and not N.has_workspace(hidden.device, nbytes, "lm_head"):
            # a workspace made inside a capture would be re-zeroed by every replay
            raise RuntimeError("run one eager head call on this stream before capturing it in a graph")
        ws, ws_bytes, _ = N.workspace_ptr(index, nbytes, "lm_head", None, stream)
        N.check(L.btl_rmsnorm(x.data_ptr(), M, H, H, N.ptr(self.norm_weight), float(self.eps), xn.data_ptr(), stream),
                "btl_rmsnorm")
        N.check(L.btl_lm_head(xn.data_ptr(), M, H, V, self.weight.data_ptr(), N.ptr(logits), tokens.data_ptr(), ws,
                              ws_bytes, stream), "btl_lm_head")
        return logits, tokens

    def _int8(self, x, return_logits, normed_out, logits_out, tokens_out):
        """The 8-bit head on x [M, hidden]."""
        import torch

        M, H = x.shape
        V, dev = self.vocab_size, x.device
        if M > _MAX_ROWS:
            raise ValueError(f"{M} rows: a call takes up to {_MAX_ROWS}")
        for t, shape, dtype, name in ((normed_out, (M, H), torch.bfloat16, "normed_out"),
                                      (logits_out, (M, V), torch.float32, "logits_out"),
                                      (tokens_out, (M,), torch.int32, "tokens_out")):
            if t is not None and (t.dtype is not dtype or t.numel() != math.prod(shape) or not t.is_contiguous()
                                  or t.device != dev):
                raise ValueError(f"{name} must be contiguous {dtype} {list(shape)} on {dev}")
        if self.weight.device != dev:
            raise ValueError(f"hidden is on {dev}, the head on {self.weight.device}")
        with torch.cuda.device(dev):
            logits = logits_out if logits_out is not None else (
                torch.empty((M, V), dtype=torch.float32, device=dev) if return_logits else None)
            tokens = tokens_out if tokens_out is not None else torch.empty(M, dtype=torch.int32, device=dev)
            if M == 0:
                return logits, tokens
            L, stream = N.lib(), N.raw_stream(dev.index)
            # without logits up to _FEW rows need none; more go in passes that share a buffer
            rows = M if logits is not None else _pass_rows(M, V)
            part = logits
            if logits is None and rows > _FEW:
                part = torch.empty((rows, V), dtype=torch.float32, device=dev)
            nbytes = max(_scratch_bytes(dev.index, rows, H, V), _scratch_bytes(dev.index, M % rows or rows, H, V))
            # the call's own: calls that overlap share nothing
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            w = self.weight
            for lo in range(0, M, rows):
                n = min(rows, M - lo)
                at = None if normed_out is None else normed_out.data_ptr() + 2 * lo * H
                N.check(L.btl_int8_head(x.data_ptr() + 2 * lo * H, n, H, V, self.norm_weight.data_ptr(), float(self.eps),
                                        w.data.data_ptr(), w.scale.data_ptr(), at, N.ptr(part), tokens.data_ptr() + 4 * lo,
                                        scratch.data_ptr(), nbytes, stream), "btl_int8_head")
        return logits, tokens

    def weight_bytes(self) -> int:
        """Compulsory HBM bytes of one head call's weights (vocab x hidden, bf16, or int8 and the scales)."""
        if self.weight_dtype == "int8":
            return self.vocab_size * (self.hidden_size + 4)
        return 2 * self.vocab_size * self.hidden_size
