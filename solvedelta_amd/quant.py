"""8-bit integer linear layers for serving on MI355X.

A weight is quantised once, a scale per output channel; activations are
quantised on the way, a scale per token (``sd_quantize_int8`` /
``sd_linear_int8``, include/solvedelta_mixer.h).  Inference only.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import nn

from . import _lib
from .ffn import _row_stride, _rows
from .operator import _call, _has_tangent, _ptr


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 [..., K], scale FP32 [...]): rows of x in 8 bits, x ~ q * scale.

    scale = max |x| / 127 over the row, q = rint(x / scale); a zero row has scale
    0 and q 0, a row that holds an infinity or a NaN the scale NaN.  x is bf16 or
    FP32 on a ROCm device; the results are detached from it."""
    if not x.is_cuda:
        raise TypeError("quantize_int8 runs on a ROCm device only")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("quantize_int8 takes a bf16 or FP32 tensor")
    if x.dim() < 1 or not x.shape[-1]:
        raise ValueError("quantize_int8 takes rows [...,K] with K >= 1")
    x = x.detach()
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if not x.numel():
        return q, scale
    x2 = _rows(x)
    rc = _call(_lib.load().sd_quantize_int8, x.device, x2.shape[0], x2.shape[1],
               int(x.dtype == torch.float32), x2.data_ptr(), _row_stride(x2), q.data_ptr(),
               x2.shape[1], scale.data_ptr())
    _lib.check(rc, "sd_quantize_int8")
    return q, scale


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x W^T + bias with x's rows and the weight in 8 bits.

    x bf16 [..., K]; weight int8 [O, K] and weight_scale FP32 [O], as
    ``quantize_int8`` gives them; bias bf16 [O].  Returns bf16 [..., O].  Integer
    sums are exact; a token that holds an infinity or a NaN comes out NaN.  There
    is no backward: it raises where a gradient would be asked for."""
    for t in (x, weight, weight_scale, bias):
        if t is None:
            continue
        if not t.is_cuda:
            raise TypeError("int8_linear runs on a ROCm device only")
        if t.device != x.device:
            raise ValueError("int8_linear arguments must share a device")
    if (x.dtype != torch.bfloat16 or weight.dtype != torch.int8
            or weight_scale.dtype != torch.float32
            or (bias is not None and bias.dtype != torch.bfloat16)):
        raise TypeError("int8_linear takes x bf16, weight int8, weight_scale FP32, bias bf16")
    if x.dim() < 1 or weight.dim() != 2 or not weight.numel() or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    O, K = weight.shape
    if weight_scale.shape != (O,) or (bias is not None and bias.shape != (O,)):
        raise ValueError("weight_scale and bias must have shape [O]")
    if torch.is_grad_enabled() and (x.requires_grad or weight_scale.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        raise RuntimeError("int8_linear has no backward: call it under torch.no_grad()")
    if _has_tangent(x, weight_scale, bias):
        raise RuntimeError("int8_linear has no forward-mode derivative")
    dev = x.device
    y = torch.empty((*x.shape[:-1], O), dtype=torch.bfloat16, device=dev)
    if not x.numel():
        return y
    lib = _lib.load()
    x2, w = _rows(x), _rows(weight)
    N, w_st = x2.shape[0], max(w.stride(0), K)
    weight_scale = weight_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    nws = lib.sd_linear_int8_workspace_bytes(N, K, O, w.data_ptr(), w_st)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    rc = _call(lib.sd_linear_int8, dev, N, K, O, x2.data_ptr(), max(x2.stride(0), K), w.data_ptr(),
               w_st, weight_scale.data_ptr(), _ptr(bias), y.data_ptr(), _ptr(ws), nws)
    _lib.check(rc, "sd_linear_int8")
    return y


class Int8Linear(nn.Module):
    """A Linear whose weight is held in 8 bits, for inference.

    Its buffers follow the module from device to device but keep their types: a cast of
    the model would round the scales, and the product takes no others."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, *,
                 device=None) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("weight", torch.zeros(out_features, in_features, dtype=torch.int8,
                                                   device=device))
        self.register_buffer("weight_scale", torch.zeros(out_features, dtype=torch.float32,
                                                         device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.bfloat16,
                                                 device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        """``linear`` (bf16 or FP32, on a ROCm device) in 8 bits."""
        q = cls(linear.in_features, linear.out_features, linear.bias is not None,
                device=linear.weight.device)
        q.weight, q.weight_scale = quantize_int8(linear.weight)
        if linear.bias is not None:
            q.bias = linear.bias.detach().to(torch.bfloat16)
        return q

    def _apply(self, fn, recurse=True):
        # casts change floating tensors alone: they see the bits
        bits = {torch.float32: torch.int32, torch.bfloat16: torch.int16}
        return super()._apply(lambda t: fn(t.view(bits[t.dtype])).view(t.dtype) if t.dtype in bits
                              else fn(t), recurse)

    def forward(self, x):
        return int8_linear(x.to(torch.bfloat16), self.weight, self.weight_scale, self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}")


def quantize_linears(module: nn.Module, names: Sequence[str] = ("gate_up_proj", "down_proj",
                                                                "lm_head")) -> nn.Module:
    """Every ``nn.Linear`` in ``module`` with one of these attribute names becomes an
    ``Int8Linear``, in place; returns the module.  The defaults are the causal LM's
    MLP projections and its head; ``in_proj`` is the mixer's."""
    names = (names,) if isinstance(names, str) else tuple(names)
    found = [(parent, name, child) for parent in module.modules()
             for name, child in parent.named_children()
             if name in names and type(child) is nn.Linear]
    if not found:
        raise ValueError(f"no nn.Linear named {', '.join(names)} in the module")
    for parent, name, child in found:
        setattr(parent, name, Int8Linear.from_linear(child))
    return module


__all__ = ["Int8Linear", "int8_linear", "quantize_int8", "quantize_linears"]
