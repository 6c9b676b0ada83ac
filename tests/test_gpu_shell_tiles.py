"""Every tile form of the causal LM's products, with whole tiles and with shared ones, at ragged
sizes, against the definitions in 64 bits.

That the shapes below reach every form is asserted on the host, so that another choice of tiles
does not take one out of the tests unseen.  Beside the bounds of the operators' other tests,
each whole 32 x 32 block of a result keeps twice the bound on the norm: a block's 1024 errors
average out to within a few percent, and rows and columns differ in size."""
import ctypes

import pytest
import torch

from test_gpu_ffn import E, check_grads, check_y, grads, make
from test_gpu_int8 import check, rows

# N, D, I, O
FFN = [(91, 69, 69, 67), (258, 122, 4229, 331), (1551, 1298, 867, 1405), (4110, 95, 2007, 207),
       (3783, 603, 350, 3459), (239, 861, 5217, 1996), (4163, 2759, 103, 151), (67, 2526, 69, 2946),
       (1852, 1508, 5495, 73), (3347, 142, 93, 3647), (100, 3805, 1314, 169), (4945, 3429, 1597, 113),
       (2906, 130, 5804, 1465), (1426, 403, 4822, 3559), (5889, 740, 1363, 2749)]
# N, K, O
INT8 = [(69, 69, 66), (74, 3980, 71), (145, 65, 11513), (69, 2671, 8914), (3331, 386, 2420),
        (70, 5545, 8670), (1219, 5627, 840), (5064, 2754, 3283)]


def _form(M, N, k_bytes):
    from solvedelta_amd import _lib
    plan = (ctypes.c_int * 3)()
    assert _lib.load().sd_product_plan(M, N, k_bytes, plan) == 0
    return plan[0], plan[2] > 0


def _products(N, D, I, O):
    row = lambda n: (n + 7) // 8 * 16
    return {"gate_up": _form(N, 2 * I, row(D)), "down": _form(N, O, row(I)), "da": _form(N, I, row(O)),
            "dx": _form(N, D, row(2 * I)), "dgate_up": _form(2 * I, D, 2 * N), "ddown": _form(O, I, 2 * N)}


FORMS = {(tile, shared) for tile in range(4) for shared in (False, True)}


def test_the_shapes_reach_every_form():
    reached = {}
    for shape in FFN:
        for name, form in _products(*shape).items():
            reached.setdefault(name, set()).add(form)
    reached["int8"] = {_form(N, O, K) for N, K, O in INT8}
    for name, forms in reached.items():
        assert forms == FORMS, (name, FORMS - forms)


def test_plans_of_no_product():
    from solvedelta_amd import _lib
    lib, plan = _lib.load(), (ctypes.c_int * 3)()
    for bad in ((0, 1, 1), (1, -1, 1), (1, 1, 0), (1 << 31, 1, 1)):
        assert lib.sd_product_plan(*bad, plan) == _lib.SD_ERR_SHAPE


def _blocks(got, ref, bound):
    m, n = ref.shape[0] // 32, ref.shape[1] // 32
    norm = lambda t: t[:32 * m, :32 * n].reshape(m, 32, n, 32).square().sum((1, 3)).sqrt()
    assert torch.all(norm(got.double() - ref) <= bound * norm(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,I,O", FFN)
def test_gated_ffn(N, D, I, O):
    from solvedelta_amd import gated_ffn
    print(f"case tiles N{N} D{D} I{I} O{O} {_products(N, D, I, O)}", flush=True)
    x, gate_up, down, dy = make(N, D, I, O, seed=N)
    leaves = [t.requires_grad_() for t in (x, gate_up, down)]
    y = gated_ffn(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    x, gate_up, down = (t.detach() for t in leaves)
    for a in (y.detach(), *got):
        assert torch.isfinite(a).all()
    check_y(y.detach(), x, gate_up, down)
    ref = grads(x, gate_up, down, dy)
    check_grads(got, ref)
    for a, b in zip(got, ref):
        _blocks(a, b, 2 * (2 * E + 2.0 ** -10))
    # without a gradient to keep for, the same bits
    with torch.no_grad():
        assert torch.equal(gated_ffn(x, gate_up, down), y.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,O", INT8)
@pytest.mark.parametrize("with_bias", [False, True])
def test_int8_linear(N, K, O, with_bias):
    from solvedelta_amd import int8_linear, quantize_int8
    print(f"case tiles int8 N{N} K{K} O{O} {_form(N, O, K)}", flush=True)
    x = rows(N, K, seed=N)
    w, ws = quantize_int8(rows(O, K, seed=O, dtype=torch.float32))
    bias = rows(1, O, seed=3)[0] if with_bias else None
    check(int8_linear(x, w, ws, bias), x, w, ws, bias)
