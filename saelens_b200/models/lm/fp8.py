"""Projections of a producer LM with frozen 8-bit weights (e4m3, a scale per 128 x 128 block).

`HookedLM.quantize_weights("fp8")`, or `weight_quantization="fp8"` when the model is made, replaces
the q/k/v, output and MLP projections; embeddings, norms and the unembedding keep their type.  The
weights take half the memory and traffic of bf16 ones, and the products run on `ops.linear_fp8` on
CUDA (rows quantised on the way in); elsewhere the same arithmetic runs in PyTorch.  q, k and v, and
gate and up, are one weight each, so that one product computes them.  Role of the 8-bit weight
option of the reference's producer engine (engine arguments, sae_lens/vllm_model.py:548-625).
"""

from __future__ import annotations

from typing import Any

import torch
from torch import nn

BLOCK = 128
_MAX = 448.0  # the largest e4m3 value
_LEAST = _MAX * torch.finfo(torch.float32).tiny  # least maximum of a block, so that a scale is a normal number


def _native(x: torch.Tensor) -> bool:
    from saelens_b200.models.lm import transformer

    if not x.is_cuda or transformer.FORCE_TORCH:
        return False
    from saelens_b200 import ops

    return ops.available()


def quantize_torch(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """`ops.quantize_fp8` in PyTorch: e4m3 values [rows, columns] and fp32 scales."""
    m, k = x.shape
    mb, kb = -(-m // block_rows), -(-k // BLOCK)
    t = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k, 0, mb * block_rows - m)).view(mb, block_rows, kb, BLOCK)
    most = t.abs().amax(dim=(1, 3), keepdim=True).clamp_min(_LEAST)
    q = (t * (_MAX / 1024.0) / most * 1024.0).to(torch.float8_e4m3fn).view(mb * block_rows, kb * BLOCK)[:m, :k]
    return q, (most / torch.full_like(most, _MAX))[:, 0, :, 0]


def _dequantized(q: torch.Tensor, scale: torch.Tensor, block_rows: int) -> torch.Tensor:
    m, k = q.shape
    return q.float() * scale.repeat_interleave(block_rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


class _TorchLinear(torch.autograd.Function):
    """`ops.linear_fp8` in PyTorch: fp32 products of quantised rows, the gradient's rows quantised too."""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
        ctx.save_for_backward(weight, scale)
        y = _dequantized(*quantize_torch(x.reshape(-1, x.shape[-1]), 1), 1) @ _dequantized(weight, scale, BLOCK).T
        return (y if bias is None else y + bias).to(x.dtype).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dy: torch.Tensor) -> tuple[torch.Tensor, None, None, None]:
        weight, scale = ctx.saved_tensors
        dx = _dequantized(*quantize_torch(dy.reshape(-1, dy.shape[-1]), 1), 1) @ _dequantized(weight, scale, BLOCK)
        return dx.to(dy.dtype).view(*dy.shape[:-1], weight.shape[1]), None, None, None


_CHECKED: dict[Any, int] = {}  # the backward pass that reads the status word at its end, for each word


def _check_after_backward(status: Any) -> None:
    """Read the status word once, when the backward pass under way has ended: a product of it that gave up
    waiting raises there, not in the next forward pass.  (A capture reads nothing.)"""
    task = torch._C._current_graph_task_id()
    if _CHECKED.get(id(status)) == task:
        return
    _CHECKED[id(status)] = task

    def check() -> None:
        if not (status.tensor.is_cuda and torch.cuda.is_current_stream_capturing()):
            status.check("producer LM backward")

    torch.autograd.Variable._execution_engine.queue_callback(check)


class Fp8Linear(nn.Module):
    """y = x W^T + b with W in e4m3, made from the weights (and biases) of one or several projections."""

    def __init__(self, layers: list[nn.Module]):
        super().__init__()
        with torch.no_grad():
            w = torch.cat([m.weight.detach() for m in layers]) if len(layers) > 1 else layers[0].weight.detach()
            self.d_out, self.d_in = w.shape
            if _native(w):
                from saelens_b200 import ops

                q, scale = ops.quantize_fp8(w, BLOCK)
            else:
                q, scale = quantize_torch(w, BLOCK)
            # rows start on 16 bytes; columns behind d_in hold nothing
            data = torch.zeros(self.d_out, -(-self.d_in // 16) * 16, dtype=torch.float8_e4m3fn, device=w.device)
            data[:, : self.d_in] = q
            self.register_buffer("data", data)
            self.register_buffer("scale", scale)
            biases = [m.bias for m in layers]
            bias = None
            if any(b is not None for b in biases):
                bias = torch.cat([m.bias.detach().float() if m.bias is not None else
                                  torch.zeros(m.weight.shape[0], device=w.device) for m in layers])
            self.register_buffer("bias", bias)

    @property
    def weight(self) -> torch.Tensor:
        return self.data[:, : self.d_in]

    def _apply(self, fn: Any, recurse: bool = True) -> Fp8Linear:
        # a change of type (model.to(dtype), model.half()) moves the buffers and keeps their types
        for name, buf in self._buffers.items():
            if buf is not None:
                self._buffers[name] = buf.to(fn(torch.empty(0, dtype=torch.float32, device=buf.device)).device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if _native(x):
            from saelens_b200 import ops
            from saelens_b200.models.lm.transformer import _status_for

            status = _status_for(x)
            y = ops.linear_fp8(x, self.weight, self.scale, self.bias, status=status)
            if y.requires_grad:
                y.register_hook(lambda _: _check_after_backward(status))
            return y
        return _TorchLinear.apply(x, self.weight, self.scale, self.bias)


class Fp8Part(nn.Module):
    """One projection of an `Fp8Linear` that several share."""

    def __init__(self, whole: Fp8Linear, start: int, stop: int):
        super().__init__()
        self._whole = (whole,)  # not a submodule: the buffers are registered once
        self.start, self.stop = start, stop

    @property
    def weight(self) -> torch.Tensor:
        return self._whole[0].weight[self.start : self.stop]

    @property
    def bias(self) -> torch.Tensor | None:
        b = self._whole[0].bias
        return None if b is None else b[self.start : self.stop]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self._whole[0](x)[..., self.start : self.stop]


def _shared(layers: list[nn.Module]) -> tuple[Fp8Linear, list[Fp8Part]]:
    whole, parts, at = Fp8Linear(layers), [], 0
    for m in layers:
        parts.append(Fp8Part(whole, at, at + m.weight.shape[0]))
        at += m.weight.shape[0]
    return whole, parts


@torch.no_grad()
def quantize_lm_fp8(model: Any) -> Any:
    """Replace the projections of `model` (a HookedLM in bf16, fp16 or fp32) in place; returns the model."""
    for blk in model.blocks:
        at, mlp = blk.attn, blk.mlp
        if at.qkv_fp8 is not None:
            raise ValueError("the model's weights are quantised already")
        at.qkv_fp8, (at.q, at.k, at.v) = _shared([at.q, at.k, at.v])
        at.o = Fp8Linear([at.o])
        if mlp.gated:
            mlp.gate_up_fp8, (mlp.gate, mlp.up) = _shared([mlp.gate, mlp.up])
        else:
            mlp.up = Fp8Linear([mlp.up])
        mlp.down = Fp8Linear([mlp.down])
    return model


__all__ = ["Fp8Linear", "quantize_lm_fp8", "quantize_torch"]
