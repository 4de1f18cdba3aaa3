"""Rotary positions of q and k in one kernel (`csrc/rotary.cu`), and the frequencies that it takes."""

from __future__ import annotations

import math
from typing import Any

import torch

from saelens_b200.ops._build import load

__all__ = ["rotary", "rotary_frequencies"]

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: dict[str, Any] | None = None,
                       n_positions: int | None = None, device: Any = None) -> tuple[torch.Tensor, float]:
    """Angle per position of each of the dim / 2 pairs (fp64 [dim / 2]) and the factor on cos and sin.

    Pair i turns by base^(-2i / dim) a position.  `scaling` stretches the context, as checkpoints name
    it ("rope_type" or "type"): "linear" divides every frequency by `factor`; "dynamic" raises the
    base with the length, from `original_max_position_embeddings` on (`n_positions` is the length in
    use); "llama3" divides those that turn fewer than `low_freq_factor` times in the original context
    by `factor`, keeps those above `high_freq_factor` and blends between; "yarn" (Peng et al. 2023)
    blends over pairs between `beta_slow` and `beta_fast` turns (whole pairs, unless `truncate` is
    false) and puts `attention_factor` (0.1 ln(factor) + 1 unless given, or the ratio of 0.1 m
    ln(factor) + 1 for m = `mscale` and `mscale_all_dim`) on cos and sin; "default" or None keeps them."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if not base > 0:
        raise ValueError(f"rotary_frequencies: base must be positive, got {base}")
    s = dict(scaling or {})
    kind = s.get("rope_type", s.get("type", "default")) or "default"
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if kind == "default":
        return (float(base) ** (-i / dim)).to(device), 1.0
    if kind not in ("linear", "dynamic", "llama3", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {kind!r}")
    if "factor" not in s or not float(s["factor"]) >= 1.0:
        raise ValueError(f"rotary_frequencies: {kind} scaling needs a factor of 1 or more, got {s.get('factor')}")
    factor = float(s["factor"])
    freq = float(base) ** (-i / dim)
    if kind == "linear":
        return (freq / factor).to(device), 1.0
    if "original_max_position_embeddings" not in s:
        raise ValueError(f"rotary_frequencies: {kind} scaling needs original_max_position_embeddings")
    before = float(s["original_max_position_embeddings"])
    if kind == "dynamic":
        length = max(float(n_positions or 0), before)
        if dim > 2:
            base = base * (factor * length / before - (factor - 1.0)) ** (dim / (dim - 2.0))
        return (float(base) ** (-i / dim)).to(device), 1.0
    if kind == "llama3":
        low, high = float(s.get("low_freq_factor", 1.0)), float(s.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("rotary_frequencies: high_freq_factor must be above low_freq_factor")
        keep = ((before * freq / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return (freq * (keep + (1 - keep) / factor)).to(device), 1.0

    def pair_of(turns: float) -> float:  # the pair that turns so often in the original context
        return dim * math.log(before / (turns * 2 * math.pi)) / (2 * math.log(base))

    first, last = pair_of(float(s.get("beta_fast") or 32.0)), pair_of(float(s.get("beta_slow") or 1.0))
    if s.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    lo, hi = max(first, 0), min(last, dim - 1)
    ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)

    def stretch(m: float) -> float:
        return 0.1 * m * math.log(factor) + 1.0

    attention = s.get("attention_factor")
    if attention is None:
        both = s.get("mscale") and s.get("mscale_all_dim")
        attention = stretch(float(s["mscale"])) / stretch(float(s["mscale_all_dim"])) if both else stretch(1.0)
    attention = float(attention)
    return (freq * (1 - ramp) + freq / factor * ramp).to(device), attention


def rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    freq: torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    offset: int = 0,
    interleaved: bool = False,
    factor: float = 1.0,
    inplace: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """q [B, S, H, d] and k [B, S, KV, d] (or None) with the first 2 * len(freq) channels of each head
    turned by position * freq, in 64 bits, and scaled by `factor`; further channels pass through.

    Channels (i, rot/2 + i) form a pair, or (2i, 2i + 1) with `interleaved`.  bf16, fp16 or fp32, any
    strides with contiguous channels (views of a fused projection); freq fp64 [rot / 2] on q's device
    (`rotary_frequencies`).  `positions` int64 or int32, [B, S] or what broadcasts to it, any value;
    without it token s is at offset + s.  Returns new tensors, or with `inplace` q and k themselves
    (not under autograd).  Differentiable in q and k, any number of times; tangents (forward mode) are
    refused."""
    if q.is_cuda:  # checked where it is launched
        out = load().rotary(q, k, freq, positions, offset, interleaved, factor, inplace)
        return out if k is not None else out[0]
    if q.dim() != 4 or q.dtype not in _FLOATS:
        raise ValueError(f"rotary: q must be bf16, fp16 or fp32 [B, S, H, d], got {q.dtype} {tuple(q.shape)}")
    B, S, _, d = q.shape
    if k is not None and (k.dim() != 4 or k.dtype != q.dtype or k.device != q.device or k.shape[:2] != q.shape[:2] or k.shape[3] != d):
        raise ValueError(f"rotary: k {k.dtype} {tuple(k.shape)} does not match q {q.dtype} {tuple(q.shape)}")
    if freq.dim() != 1 or freq.dtype != torch.float64 or freq.requires_grad or not 2 <= 2 * freq.shape[0] <= d:
        raise ValueError(f"rotary: freq must be constant fp64 [rot / 2] with rot from 2 to {d}, got {freq.dtype} {tuple(freq.shape)}")
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32) or positions.dim() > 2:
            raise ValueError(f"rotary: positions must be int64 or int32 [B, S], got {positions.dtype} {tuple(positions.shape)}")
        if offset:
            raise ValueError("rotary: either positions or an offset")
        if any(n not in (1, want) for n, want in zip(reversed(positions.shape), (S, B))):
            raise ValueError(f"rotary: positions {tuple(positions.shape)} do not broadcast to {(B, S)}")
    raise ValueError("rotary: all tensors must be on one CUDA device")
