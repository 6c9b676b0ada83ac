"""The 8-bit product's sums stay within 32 bits for every weight it takes, -128 among them."""
import ctypes

import pytest
import torch

WIDEST = (2 ** 31 - 1) // (127 * 128)   # 132104


def test_rows_whose_sums_could_pass_32_bits_are_refused():
    """On the host, before any launch (the workspace is too small in any case)."""
    from solvedelta_amd import _lib
    lib = _lib.load()
    p = [ctypes.c_void_p(4096 * (i + 1)) for i in range(5)]
    call = lambda K: lib.sd_linear_int8(4, K, 32, p[0], K, p[1], K, p[2], None, p[3], p[4], 0, None)
    assert call(WIDEST) == _lib.SD_ERR_WORKSPACE
    assert call(WIDEST + 1) == _lib.SD_ERR_SHAPE
    assert lib.sd_linear_int8_workspace_bytes(4, WIDEST + 1, 32, p[1], WIDEST + 1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 70])
def test_the_largest_sums(N):
    """127 * -128 over the widest row: 1024 short of -2^31, exact up to the output's rounding."""
    from solvedelta_amd import int8_linear
    x = torch.ones(N, WIDEST, dtype=torch.bfloat16, device="cuda")
    w = torch.full((16, WIDEST), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    y = int8_linear(x, w, torch.full((16,), 2.0 ** -20, device="cuda")).double()
    want = torch.full((16,), -128.0 * WIDEST * 2.0 ** -20, dtype=torch.float64, device="cuda")
    want[1::2] = 127.0 * WIDEST * 2.0 ** -20
    # rounding to bf16, the scale 1/127 and two FP32 products
    assert torch.all((y - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want.abs())
