"""Drawing tokens on MI355X: temperature, top-k, top-p and min-p from given
uniform random numbers, in one HIP kernel (``sd_sample_tokens``,
include/solvedelta_mixer.h) with no sort and no host sync.
"""
from __future__ import annotations

import functools
import math
from typing import Union

import torch

from . import _lib
from .operator import _call

Setting = Union[int, float, torch.Tensor]


# name, type, least, most of each setting, in the C entry's order
_SETTINGS = (("temperature", torch.float32, 0.0, 3e38), ("top_k", torch.int64, -math.inf, math.inf),
             ("top_p", torch.float32, 0.0, math.inf), ("min_p", torch.float32, -math.inf, 1.0))


def _number(v, name: str, dtype, lo: float, hi: float) -> float:
    if isinstance(v, bool) or not isinstance(v, int if dtype == torch.int64 else (int, float)):
        raise TypeError(f"{name} must be a number or a tensor")
    if not lo <= v <= hi:
        raise ValueError(f"{name} must lie in [{lo}, {hi}], got {v}")
    return float(v)


def _rows_of(v: torch.Tensor, name: str, like: torch.Tensor, dtype) -> torch.Tensor:
    if v.device != like.device:
        raise ValueError(f"{name} must be on the logits' device")
    if v.shape != like.shape[:-1]:
        raise ValueError(f"{name} must be a number or have one entry per row of logits")
    if dtype == torch.int64 and (v.is_floating_point() or v.is_complex()):
        raise TypeError(f"{name} must be an integer tensor")
    return v.to(dtype).contiguous()


@functools.lru_cache(maxsize=256, typed=True)
def _numbers(*values):
    """The C entry's settings for numbers alone: most calls' are the same each time."""
    return (_lib.SdSampleSetting * 4)(*((_number(v, *s), None) for v, s in zip(values, _SETTINGS)))


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor, temperature: Setting = 1.0,
                  top_k: Setting = 0, top_p: Setting = 1.0, min_p: Setting = 0.0) -> torch.Tensor:
    """One token per row of ``logits`` [..., V] (bf16 or FP32), int64 [...].

    ``noise`` holds uniform numbers in [0, 1), FP32, of the same shape
    (``torch.rand``); the same noise always gives the same tokens.  Each setting
    is a number, or a tensor with one entry per row.

    With L a row's largest logit and z = (logit - L) / temperature, tokens rank by
    (logit descending, index ascending).  Kept are the first ``top_k``; of these
    the ones whose predecessors hold less than ``top_p`` of the mass of exp(z) over
    the top_k; of these the ones with z >= log(min_p), at least the first.  The
    token is the kept one with the largest z - log(-log(noise)): a draw from the
    softmax over the kept tokens.  temperature 0 takes the first token;
    top_k <= 0, top_p >= 1 and min_p <= 0 switch a filter off.  Logits of -infinity
    or NaN are never drawn; a row that holds nothing else gives -1.
    Masses are FP32 exponentials, summed to 2^-28 of the largest.

    Entries of setting tensors are not checked (that would wait for the GPU): a
    temperature that is not positive reads as 0.
    """
    if not logits.is_cuda or not noise.is_cuda:
        raise TypeError("sample_tokens runs on a ROCm device only")
    if logits.dtype not in (torch.bfloat16, torch.float32) or noise.dtype != torch.float32:
        raise TypeError("sample_tokens takes bf16 or FP32 logits and FP32 noise")
    if logits.device != noise.device:
        raise ValueError("logits and noise must share a device")
    if logits.dim() < 1 or not logits.shape[-1] or logits.shape != noise.shape:
        raise ValueError("logits and noise must have the same shape [...,V]")
    lead = logits.shape[:-1]
    V = logits.shape[-1]
    rows = lead[0] if len(lead) == 1 else math.prod(lead)
    values = (temperature, top_k, top_p, min_p)
    keep = None     # tensors of settings, alive until the launch
    if any(map(torch.is_tensor, values)):
        keep = [_rows_of(v, s[0], logits, s[1]) if torch.is_tensor(v) else None
                for v, s in zip(values, _SETTINGS)]
        settings = (_lib.SdSampleSetting * 4)(
            *((0.0, t.data_ptr()) if t is not None else (_number(v, *s), None)
              for v, t, s in zip(values, keep, _SETTINGS)))
    else:
        settings = _numbers(*values)
    token = torch.empty(lead, dtype=torch.int64, device=logits.device)
    if not rows:
        return token
    l2, n2 = (t if t.dim() == 2 else t.detach().reshape(rows, V) for t in (logits, noise))
    l2, n2 = (t if V == 1 or t.stride(1) == 1 else t.contiguous() for t in (l2, n2))
    rc = _call(_lib.load().sd_sample_tokens, logits.device, rows, V,
               int(logits.dtype == torch.float32), l2.data_ptr(), l2.stride(0), n2.data_ptr(),
               n2.stride(0), settings, token.data_ptr())
    _lib.check(rc, "sd_sample_tokens")
    return token


__all__ = ["sample_tokens"]
