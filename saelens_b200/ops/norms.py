"""The residual update between two norms of a decoder block in one kernel (`csrc/block_norm.cu`)."""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

__all__ = ["residual_norm"]

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _gate_rows(gate: torch.Tensor, shape: torch.Size) -> tuple[torch.Tensor, int, int]:
    """gate as contiguous [gate rows, D], how many consecutive rows share one, and its mode (1 one for
    all rows, 2 one for several, 3 one each)."""
    lead, own = shape[:-1], gate.shape[:-1]
    if gate.dim() < 1 or gate.shape[-1] != shape[-1] or len(own) > len(lead):
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} does not match x {tuple(shape)}")
    own = (1,) * (len(lead) - len(own)) + tuple(own)
    last = max((i for i, n in enumerate(own) if n != 1), default=-1)
    if own[: last + 1] != tuple(lead[: last + 1]):
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} must be one row for all of x {tuple(shape)} or one "
                         "for each entry of its leading dimensions")
    div = math.prod(lead[last + 1 :])
    gate = gate.reshape(-1, shape[-1]).contiguous()
    if last < 0:
        return gate, max(div, 1), 1
    return gate, max(div, 1), 3 if div == 1 else 2


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, w, b, post_w, post_b, gate, div, mode, eps, post_eps, scale, layer, one_plus, round_branch):
        from saelens_b200.ops import native

        stream, normed = torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty_like(x, memory_format=torch.contiguous_format)
        stats = torch.empty(4, x.shape[0], dtype=torch.float32, device=x.device)
        native().residual_norm_fwd(x, branch, w, b, post_w, post_b, gate, div, eps, post_eps, scale, layer, one_plus,
                                   round_branch, stream, normed, stats)
        # the branch is read again only where its own values enter a gradient
        ctx.save_for_backward(stream, branch if post_w is not None or gate is not None else stream, w, post_w, post_b, gate, stats)
        ctx.args = (div, mode, scale, layer, one_plus)
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, d_stream, d_normed):
        from saelens_b200.ops import native

        stream, branch, w, post_w, post_b, gate, stats = ctx.saved_tensors
        div, mode, scale, layer, one_plus = ctx.args
        need = ctx.needs_input_grad
        none = (None,) * 8
        if d_stream is None and d_normed is None:
            return (None,) * 7 + none

        def rows(t):
            return t if t is None or t.stride(1) == 1 else t.contiguous()

        dx = torch.empty_like(stream)
        alike = post_w is None and gate is None and scale == 1.0
        d_branch = torch.empty_like(stream) if need[1] and not alike else None

        def like(t, wanted):
            return torch.empty_like(t) if wanted and t is not None else None

        dw, db = like(w, need[2]), like(w, need[3])
        dpw, dpb, dg = like(post_w, need[4]), like(post_b, need[5]), like(gate, need[6])
        native().residual_norm_bwd(rows(d_stream), rows(d_normed), stream, branch, w, post_w, post_b, gate, div, mode,
                                   scale, layer, one_plus, stats, dx, d_branch, dw, db, dpw, dpb, dg)
        return (dx, dx if alike else d_branch, dw, db, dpw, dpb, dg) + none


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

    Differentiable in all tensors (once).  D up to 16384 for rows of 16-byte vectors (D a multiple of
    8, rows starting on 16 bytes), 8192 otherwise; with gradients the wanted column sums (one for
    each vector and a gate that rows share) of D fp32 have to fit 224 KB together."""
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1:
        raise ValueError(f"residual_norm: x must be bf16, fp16 or fp32 [..., D], got {x.dtype} {tuple(x.shape)}")
    if branch.shape != x.shape:
        raise ValueError(f"residual_norm: branch {tuple(branch.shape)} must have x's shape {tuple(x.shape)}")
    if kind not in ("rms", "layer"):
        raise ValueError(f"residual_norm: kind must be 'rms' or 'layer', got {kind!r}")
    D = x.shape[-1]
    layer = kind == "layer"
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
    g, div, mode = (None, 1, 0) if gate is None else _gate_rows(gate, x.shape)
    if not x.is_cuda:
        raise ValueError("residual_norm: x must be on a CUDA device")

    def rows(t):
        t = t.reshape(-1, D)
        return t if t.stride(1) == 1 or D == 1 else t.contiguous()

    def vector(t):
        return t if t is None else t.contiguous()

    from saelens_b200.ops import native

    x2, b2 = rows(x), rows(branch)
    weight, bias, post_weight, post_bias = vector(weight), vector(bias), vector(post_weight), vector(post_bias)
    post_eps = eps if post_eps is None else post_eps
    learned = [t for t in (weight, bias, post_weight, post_bias, g) if t is not None and t.requires_grad]
    if torch.is_grad_enabled() and (x.requires_grad or branch.requires_grad or learned):
        sums = len(learned) - (1 if mode == 3 and g is not None and g.requires_grad else 0)
        if not native().residual_norm_bwd_fits(D, sums):
            raise ValueError(f"residual_norm: {sums} column sums of width {D} do not fit the backward pass")
        stream, normed = _ResidualNorm.apply(x2, b2, weight, bias, post_weight, post_bias, g, div, mode, float(eps),
                                             float(post_eps), float(scale), layer, bool(one_plus), bool(round_branch))
    else:
        stream, normed = torch.empty(x2.shape, dtype=x.dtype, device=x.device), torch.empty(x2.shape, dtype=x.dtype, device=x.device)
        native().residual_norm_fwd(x2, b2, weight, bias, post_weight, post_bias, g, div, float(eps), float(post_eps),
                                   float(scale), layer, bool(one_plus), bool(round_branch), stream, normed, None)
    return stream.view(x.shape), normed.view(x.shape)
