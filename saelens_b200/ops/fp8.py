"""Projections with frozen 8-bit weights (`csrc/fp8.cu`).

A weight is held in e4m3 with one fp32 scale per 128 x 128 block; the rows that it multiplies are
quantised on the way in, one scale per row and 128 columns.  Role of the 8-bit weight option of the
reference's producer engine (the engine arguments of sae_lens/vllm_model.py:548-625).
"""

from __future__ import annotations

import torch

from saelens_b200.ops._build import load
from saelens_b200.ops.status import StatusWord

__all__ = ["quantize_fp8", "gemm_fp8", "linear_fp8"]

BLOCK = 128
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def quantize_fp8(x: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values and fp32 scales of x [rows, columns] (bf16, fp16 or fp32 on CUDA).

    `block_rows=1`: a scale for each row's 128 columns, scales [rows, ceil(columns / 128)] (what
    `gemm_fp8` takes for its rows).  `block_rows=128`: one for each 128 x 128 block, scales
    [ceil(rows / 128), ceil(columns / 128)] (what it takes for its weight).  x ~ values * scale, with
    scale = max|x| / 448 of the block and values = e4m3(448 x / max|x|), ties to even; a block of
    zeros has the least normal scale, one that holds an infinity or a NaN gives NaN in the product.
    The values' rows start on 16 bytes, so they are a view of wider storage where the number of
    columns is no multiple of 16."""
    if x.dim() != 2 or x.shape[1] < 1 or x.dtype not in _FLOATS:
        raise ValueError(f"quantize_fp8: bf16, fp16 or fp32 [rows, columns], got {x.dtype} {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"quantize_fp8: block_rows must be 1 or {BLOCK}, got {block_rows}")
    if not x.is_cuda:
        raise ValueError("quantize_fp8: x must be on a CUDA device")
    x = x.detach()
    return load().quantize_fp8(x if x.stride(1) == 1 else x.contiguous(), block_rows)


def _check_weight(name: str, width: int, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None,
                  device: torch.device) -> None:
    if weight.dim() != 2 or weight.dtype != torch.float8_e4m3fn or weight.shape[0] < 1 or weight.shape[1] != width:
        raise ValueError(f"{name}: the weight must be float8_e4m3fn [features, {width}], got {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape
    if scale.dtype != torch.float32 or scale.shape != (_blocks(n), _blocks(k)):
        raise ValueError(f"{name}: the weight's scales must be fp32 {(_blocks(n), _blocks(k))}, got {scale.dtype} {tuple(scale.shape)}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"{name}: bias must be contiguous fp32 [{n}], got {bias.dtype} {tuple(bias.shape)}")
    if weight.stride(1) != 1 and k > 1 or (n > 1 and weight.stride(0) % 16) or weight.data_ptr() % 16:
        raise ValueError(f"{name}: rows of the weight must be contiguous and start on 16 bytes (quantize_fp8 lays them out so)")
    if device.type != "cuda" or weight.device != device or scale.device != device or (bias is not None and bias.device != device):
        raise ValueError(f"{name}: all tensors must be on one CUDA device")


def gemm_fp8(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    b: torch.Tensor,
    b_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
    status: StatusWord | None = None,
) -> torch.Tensor:
    """`(a * a_scale) @ (b * b_scale).T + bias` of e4m3 operands on the tcgen05 tensor cores, fp32 sums.

    a [M, K] with scales [M, ceil(K / 128)] as `quantize_fp8` returns them (stride 1 between rows);
    b [N, K] with scales [ceil(N / 128), ceil(K / 128)]; rows 16-byte aligned; bias fp32 [N].  Any M
    (0 included), N and K.  Returns [M, N] of `out_dtype` (bf16, fp16 or fp32), contiguous unless `out`
    is given."""
    if a.dim() != 2 or a.dtype != torch.float8_e4m3fn:
        raise ValueError(f"gemm_fp8: a must be float8_e4m3fn [rows, width], got {a.dtype} {tuple(a.shape)}")
    M, K = a.shape
    if a_scale.dtype != torch.float32 or a_scale.shape != (M, _blocks(K)):
        raise ValueError(f"gemm_fp8: a's scales must be fp32 {(M, _blocks(K))}, got {a_scale.dtype} {tuple(a_scale.shape)}")
    if (M > 1 and a_scale.stride(0) != 1) or (a.stride(1) != 1 and K > 1) or (M > 1 and a.stride(0) % 16) or a.data_ptr() % 16:
        raise ValueError("gemm_fp8: a and its scales must be laid out as quantize_fp8 does")
    _check_weight("gemm_fp8", K, b, b_scale, bias, a.device)
    if out is None:
        if out_dtype not in _FLOATS:
            raise ValueError(f"gemm_fp8: out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
        out = torch.empty(M, b.shape[0], dtype=out_dtype, device=a.device)
    elif out.requires_grad and torch.is_grad_enabled():
        raise ValueError("gemm_fp8: out must not require a gradient, the product has none")
    elif not out.is_inference():
        torch.autograd.graph.increment_version(out)  # autograd notices where it had saved the old values
    st = status or StatusWord(a.device)
    load().gemm_fp8(a, a_scale, b, b_scale, bias, out, st.tensor)
    if status is None:
        st.check("gemm_fp8")
    return out


def linear_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    status: StatusWord | None = None,
) -> torch.Tensor:
    """`x @ (weight * scale).T + bias` with x quantised to e4m3 on the way in (a scale per row and 128
    columns), in x's type.

    x [..., K] bf16, fp16 or fp32; weight float8_e4m3fn [N, K] and scale [ceil(N / 128), ceil(K / 128)]
    from `quantize_fp8(w, 128)`; bias fp32 [N].  The weight, its scales and the bias are frozen; the
    gradient of x is the product with the weight's other side, its incoming gradient quantised the
    same way (the quantisation of x counts as the identity); tangents (forward mode) are refused.  Without `status` every call reads its
    own status word, which waits for the device; a program passes one word and checks it when it
    waits anyway (and has to under CUDA graph capture)."""
    if x.is_cuda and status is not None:  # checked where it is launched
        return load().linear_fp8(x, weight, scale, bias, status.tensor, False)
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1:
        raise ValueError(f"linear_fp8: x must be bf16, fp16 or fp32 [..., width], got {x.dtype} {tuple(x.shape)}")
    _check_weight("linear_fp8", x.shape[-1], weight, scale, bias, x.device)
    st = StatusWord(x.device)
    y = load().linear_fp8(x, weight, scale, bias, st.tensor, True)
    st.check("linear_fp8")
    return y
