"""Derivatives that the causal LM's operators do not have are refused, not dropped."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _z(*s, dtype=BF16):
    return torch.zeros(*s, dtype=dtype, device="cuda")


def test_int8_linear_has_no_gradient_for_its_scales():
    from solvedelta_amd import int8_linear
    x, w, ws, bias = _z(2, 8), _z(4, 8, dtype=torch.int8), _z(4, dtype=torch.float32), _z(4)
    for i, t in enumerate((x, ws, bias)):
        args = [a.clone().requires_grad_(j == i) for j, a in enumerate((x, ws, bias))]
        with pytest.raises(RuntimeError):
            int8_linear(args[0], w, args[1], args[2])
        with torch.no_grad():
            assert not int8_linear(args[0], w, args[1], args[2]).requires_grad
