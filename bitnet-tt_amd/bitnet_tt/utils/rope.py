"""Rotary position tables (API of bitnet-tt's ``src/bitnet_tt/utils/rope.py``).

Frequencies are computed in float32 exactly as the reference does
(utils/rope.py:7-23): ``freq_i = 1 / theta ** (2i / dim)``, angle = position x
freq_i, cos/sin in float32.
"""

from __future__ import annotations

import numpy as np


def precompute_freqs_cis(dim: int, max_seq_len: int, theta: float = 10000.0):
    """(cos, sin), each [1, 1, max_seq_len, dim] float32 in the interleaved
    format [f0, f0, f1, f1, ...] of adjacent-pair RoPE (utils/rope.py:7-23)."""
    freqs = 1.0 / (theta ** (np.arange(0, dim, 2, dtype=np.float32) / dim))
    positions = np.arange(max_seq_len, dtype=np.float32)
    emb = np.repeat(np.outer(positions, freqs), 2, axis=-1)
    cos = np.cos(emb).astype(np.float32).reshape(1, 1, max_seq_len, dim)
    sin = np.sin(emb).astype(np.float32).reshape(1, 1, max_seq_len, dim)
    return cos, sin


def rope_tables(dim: int, max_seq_len: int, theta: float = 10000.0):
    """(cos, sin), each [max_seq_len, dim/2] float32: one value per position and
    frequency (the same numbers as precompute_freqs_cis, not repeated); the
    decode-attention kernel reads these."""
    cos, sin = precompute_freqs_cis(dim, max_seq_len, theta)
    return np.ascontiguousarray(cos[0, 0, :, 0::2]), np.ascontiguousarray(sin[0, 0, :, 0::2])


def scaled_frequencies(dim: int, theta: float = 10000.0, scaling: dict | None = None, max_position: int = 4096):
    """(float64 frequencies [dim/2], factor of cos and sin) for contexts longer
    than the model was trained on.  ``scaling`` as in a model's config
    ("rope_type" or "type"):

    - None, "default": theta^(-2i/dim).
    - "linear" (factor): every frequency / factor.
    - "llama3" (factor, low_freq_factor, high_freq_factor,
      original_max_position_embeddings): wavelengths below original / high keep
      their frequency, those above original / low get it / factor, and between
      the two the mix goes linearly with original / wavelength.
    - "yarn" (factor, beta_fast 32, beta_slow 1, attention_factor,
      original_max_position_embeddings): a ramp between the dims that turn
      beta_fast and beta_slow times within the original context; cos and sin
      times attention_factor (0.1 ln(factor) + 1).

    original_max_position_embeddings defaults to ``max_position``."""
    i = np.arange(0, dim, 2, dtype=np.float64)
    freq = float(theta) ** (-i / dim)
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return freq, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"rope scaling {kind!r}: default, linear, llama3 and yarn are supported")
    factor = float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError(f"rope scaling factor {factor} must be at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    original = float(scaling.get("original_max_position_embeddings", max_position))
    if kind == "llama3":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        turns = original * freq / (2.0 * np.pi)  # original / wavelength
        mix = np.clip((turns - low) / (high - low), 0.0, 1.0)
        return freq * (mix + (1.0 - mix) / factor), 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

    def dim_of(turns):  # the dim pair that turns this often within the original context
        return dim * np.log(original / (turns * 2.0 * np.pi)) / (2.0 * np.log(float(theta)))

    first, last = max(np.floor(dim_of(fast)), 0.0), min(np.ceil(dim_of(slow)), dim - 1.0)
    ramp = np.clip((np.arange(dim // 2) - first) / max(last - first, 0.001), 0.0, 1.0)
    attention = scaling.get("attention_factor")
    return freq * (1.0 - ramp) + freq / factor * ramp, 0.1 * np.log(factor) + 1.0 if attention is None else float(attention)


def is_scaled(scaling: dict | None) -> bool:
    """Whether a model config's ``scaling`` changes the plain frequencies."""
    return scaling is not None and scaling.get("rope_type", scaling.get("type", "default")) != "default"


def long_rope_tables(dim: int, max_seq_len: int, theta: float = 10000.0, scaling: dict | None = None,
                     max_position: int = 4096, device="cpu", first: int = 0):
    """(cos, sin) torch tensors [max_seq_len - first, dim/2] fp32 of scaled_frequencies
    at positions first, first + 1 .., angles in float64; rope_tables keeps the
    reference's float32 angles."""
    import torch

    freq, factor = scaled_frequencies(dim, theta, scaling, max_position)
    pos = torch.arange(first, max_seq_len, dtype=torch.float64, device=device)
    angle = pos[:, None] * torch.from_numpy(freq).to(device)
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


# Positions whose float32 angles are as good as any: what they cost cos and sin (theta 5e5 and 1e4, up to
# 2.4e-4 before position 4096, 0.004 at 65536, 0.008 at 131072) is a sixteenth of half a step of bf16 near one.
FLOAT32_POSITIONS = 4096


def paged_rope_tables(dim: int, max_seq_len: int, theta: float = 10000.0, scaling: dict | None = None,
                      max_position: int = 4096, device="cpu"):
    """(cos, sin) torch tensors [max_seq_len, dim/2] fp32 of a paged layer: without scaling the
    rows of rope_tables before FLOAT32_POSITIONS, so that its keys are those of DecodeAttention
    bit for bit, and angles in float64 behind them; with scaling long_rope_tables."""
    import torch

    if is_scaled(scaling):
        return long_rope_tables(dim, max_seq_len, theta, scaling, max_position, device)
    near = [torch.from_numpy(t).to(device) for t in rope_tables(dim, min(max_seq_len, FLOAT32_POSITIONS), theta)]
    if max_seq_len <= FLOAT32_POSITIONS:
        return tuple(near)
    far = long_rope_tables(dim, max_seq_len, theta, device=device, first=FLOAT32_POSITIONS)
    return tuple(torch.cat(t) for t in zip(near, far))
