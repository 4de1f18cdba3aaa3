"""The residual update between two norms of a decoder block in one kernel (`csrc/block_norm.cu`)."""

from __future__ import annotations

import torch

from saelens_b200.ops._build import load

__all__ = ["residual_norm"]

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _check_gate(gate: torch.Tensor, shape: torch.Size) -> None:
    lead, own = shape[:-1], gate.shape[:-1]
    if gate.dim() < 1 or gate.shape[-1] != shape[-1] or len(own) > len(lead):
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} does not match x {tuple(shape)}")
    own = (1,) * (len(lead) - len(own)) + tuple(own)
    last = max((i for i, n in enumerate(own) if n != 1), default=-1)
    if own[: last + 1] != tuple(lead[: last + 1]):
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} must be one row for all of x {tuple(shape)} or one "
                         "for each entry of its leading dimensions")


def residual_norm(
    x: torch.Tensor,
    branch: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    kind: str = "rms",
    eps: float = 1e-5,
    one_plus: bool = False,
    post_weight: torch.Tensor | None = None,
    post_bias: torch.Tensor | None = None,
    post_eps: float | None = None,
    gate: torch.Tensor | None = None,
    scale: float = 1.0,
    round_branch: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The end of one sub-block and the start of the next:

        stream = x + scale * gate * post_norm(branch),    normed = norm(stream)

    x, branch [..., D] and every vector of one type (bf16, fp16 or fp32).  `kind` "rms": t *
    rsqrt(mean(t^2) + eps) * w; "layer": (t - mean) * rsqrt(var + eps) * w + b.  `one_plus` weighs with
    1 + w.  Without `post_weight` the branch is taken as it is (`post_eps` defaults to `eps`).  `gate`
    [D], or one row of D for each entry of x's leading dimensions with ones behind (for x [B, S, D]:
    [B, 1, D] a sequence's, [B, S, D] a token's).  The stream is rounded to its type once and the norm
    reads it as stored; `round_branch` also rounds the post-norm's output and the gated and scaled
    branch, as a program does that stores them.  Sums are 32-bit and deterministic.

    Differentiable in all tensors, once and backward (tangents are refused).  D up to 16384 for rows of 16-byte vectors (D a multiple of
    8, rows starting on 16 bytes), 8192 otherwise; with gradients the wanted column sums (one for
    each vector and a gate that rows share) of D fp32 have to fit 224 KB together."""
    if kind not in ("rms", "layer"):
        raise ValueError(f"residual_norm: kind must be 'rms' or 'layer', got {kind!r}")
    layer = kind == "layer"
    if x.is_cuda:  # checked where it is launched
        return load().residual_norm(x, branch, weight, bias, layer, eps, one_plus, post_weight, post_bias,
                                    eps if post_eps is None else post_eps, gate, scale, round_branch)
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1:
        raise ValueError(f"residual_norm: x must be bf16, fp16 or fp32 [..., D], got {x.dtype} {tuple(x.shape)}")
    if branch.shape != x.shape:
        raise ValueError(f"residual_norm: branch {tuple(branch.shape)} must have x's shape {tuple(x.shape)}")
    D = x.shape[-1]
    if not layer and (bias is not None or post_bias is not None):
        raise ValueError("residual_norm: RMS norms have no bias")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: post_bias without post_weight")
    for name, t in (("branch", branch), ("weight", weight), ("bias", bias), ("post_weight", post_weight),
                    ("post_bias", post_bias), ("gate", gate)):
        if t is None:
            continue
        if t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"residual_norm: {name} must be {x.dtype} on {x.device}, got {t.dtype} on {t.device}")
        if name not in ("branch", "gate") and t.shape != (D,):
            raise ValueError(f"residual_norm: {name} must be [{D}], got {tuple(t.shape)}")
    if gate is not None:
        _check_gate(gate, x.shape)
    raise ValueError("residual_norm: x must be on a CUDA device")
