"""Gated feed-forward block of the causal LM on MI355X, forward and backward.

``gated_ffn(x, gate_up_weight, down_weight)`` is the reference's SwiGLU MLP
(causallsso/modeling_solvedelta.py:31-100) behind its two projections:

    y = (silu(x Wg^T) * (x Wu^T)) Wd^T,    gate_up_weight = [Wg; Wu]

bf16 activations and weights, FP32 sums; the HIP kernels (``sd_ffn_*``,
include/solvedelta_mixer.h) run on the current stream with no host sync.
"""
from __future__ import annotations

import torch

from . import _lib
from .operator import _call, _has_tangent, _ptr


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows [N, width] with unit column stride and rows that do not
    overlap; a view where its strides allow."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    width = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        t = t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _ffn_args(x2, gate_up, down) -> _lib.SdFfn:
    N, D = x2.shape
    O, I = down.shape
    return _lib.SdFfn(N, D, I, O, x2.data_ptr(), max(x2.stride(0), D), gate_up.data_ptr(),
                      max(gate_up.stride(0), D), down.data_ptr(), max(down.stride(0), I))


def _ffn_fwd(x2, gate_up, down, keep: bool):
    """(y [N, O], what the backward reads or None)."""
    lib = _lib.load()
    dev = x2.device
    f = _ffn_args(x2, gate_up, down)
    y = torch.empty((f.N, f.O), dtype=torch.bfloat16, device=dev)
    nws = lib.sd_ffn_fwd_workspace_bytes(f)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    saved = torch.empty(lib.sd_ffn_saved_bytes(f), dtype=torch.uint8, device=dev) if keep else None
    rc = _call(lib.sd_ffn_fwd, dev, f, y.data_ptr(), _ptr(saved), ws.data_ptr(), nws)
    _lib.check(rc, "sd_ffn_fwd")
    return y, saved


class _GatedFFNFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up_weight, down_weight):
        x2, gate_up, down = _rows(x), _rows(gate_up_weight), _rows(down_weight)
        y, saved = _ffn_fwd(x2, gate_up, down, True)
        ctx.save_for_backward(x2, gate_up, down, saved)
        ctx.shape = x.shape
        return y if x.dim() == 2 else y.view(*x.shape[:-1], down.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _lib.load()
        x2, gate_up, down, saved = ctx.saved_tensors
        dy2 = _rows(dy)
        dev = dy.device
        dx, dgu, dd = (torch.empty(t.shape, dtype=torch.bfloat16, device=dev) if need else None
                       for t, need in zip((x2, gate_up, down), ctx.needs_input_grad))
        f = _ffn_args(x2, gate_up, down)
        nws = lib.sd_ffn_bwd_workspace_bytes(f, dy2.data_ptr(), _row_stride(dy2))
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _call(lib.sd_ffn_bwd, dev, f, saved.data_ptr(), dy2.data_ptr(), _row_stride(dy2),
                   _ptr(dx), _ptr(dgu), _ptr(dd), ws.data_ptr(), nws)
        _lib.check(rc, "sd_ffn_bwd")
        return None if dx is None else dx.view(ctx.shape), dgu, dd


def gated_ffn(x: torch.Tensor, gate_up_weight: torch.Tensor,
              down_weight: torch.Tensor) -> torch.Tensor:
    """The gated feed-forward block on bf16 tensors of one ROCm device.

    x [..., D]; gate_up_weight [2 I, D], the gate's rows first; down_weight
    [O, I].  Returns [..., O].  Rows may be strided; gradients flow to all
    three arguments (once: no double backward, and no forward mode).  What the backward reads is
    kept in 16 bits, 6 I bytes a token and a little more.
    """
    for t in (x, gate_up_weight, down_weight):
        if not t.is_cuda:
            raise TypeError("gated_ffn runs on a ROCm device only")
        if t.dtype != torch.bfloat16:
            raise TypeError("gated_ffn takes bf16 tensors")
        if t.device != x.device:
            raise ValueError("gated_ffn arguments must share a device")
    if x.dim() < 1 or gate_up_weight.dim() != 2 or down_weight.dim() != 2:
        raise ValueError("gated_ffn takes x [...,D], gate_up_weight [2I,D], down_weight [O,I]")
    O, I = down_weight.shape
    if gate_up_weight.shape != (2 * I, x.shape[-1]) or not I or not O or not x.shape[-1]:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, gate_up_weight "
                         f"{tuple(gate_up_weight.shape)}, down_weight {tuple(down_weight.shape)}")
    if _has_tangent(x, gate_up_weight, down_weight):
        raise RuntimeError("gated_ffn has no forward-mode derivative")
    grad = torch.is_grad_enabled() and (x.requires_grad or gate_up_weight.requires_grad
                                        or down_weight.requires_grad)
    if not x.numel():   # no tokens: an empty result with zero gradients
        out = x.new_zeros(*x.shape[:-1], O)
        return out + 0 * (x.sum() + gate_up_weight.sum() + down_weight.sum()) if grad else out
    if grad:
        return _GatedFFNFn.apply(x, gate_up_weight, down_weight)
    y, _ = _ffn_fwd(_rows(x), _rows(gate_up_weight), _rows(down_weight), False)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], O)


__all__ = ["gated_ffn"]
