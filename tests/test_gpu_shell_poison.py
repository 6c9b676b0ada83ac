"""Uninitialised-memory check of the causal LM's operators: every buffer they take from
torch.empty (outputs, gradients, what the backward keeps, workspaces) is filled with NaN bytes
first.  A kernel that reads what nothing wrote, even to multiply it by 0, then changes the
result: all results must be finite and agree bitwise with the same call on ordinary buffers."""
import pytest
import torch

from test_gpu_poison import _PoisonTorch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _poisoned(module, call):
    saved = module.torch
    module.torch = _PoisonTorch()
    try:
        return call()
    finally:
        module.torch = saved


def _same(names, clean, dirty):
    for name, a, b in zip(names, clean, dirty):
        assert torch.isfinite(a).all() and torch.isfinite(b).all(), name
        assert torch.equal(a, b), name


# Inner widths whose two halves end inside 16 bytes, some at the last columns of a 32-column
# block (29 to 31 of 32); outer widths off 8 as well.
@pytest.mark.parametrize("N,D,I,O", [
    (N, 64, I, 64) for N in (1, 65, 300) for I in (29, 30, 31, 61, 62, 63, 95, 2749)
] + [(1, 1, 1, 1), (3, 33, 31, 7), (65, 33, 30, 17), (300, 250, 61, 41), (2100, 130, 285, 66),
     (777, 1024, 2750, 1024)])
def test_gated_ffn(N, D, I, O):
    from solvedelta_amd import ffn
    print(f"case ffn poison N{N} D{D} I{I} O{O}", flush=True)
    g = torch.Generator().manual_seed(I)
    n = lambda *s: torch.randn(*s, generator=g)
    x, gate_up, down, dy = (t.to(torch.bfloat16).to(DEV) for t in (
        n(N, D), n(2 * I, D) * D ** -0.5, n(O, I) * I ** -0.5, n(N, O)))
    leaves = [t.requires_grad_() for t in (x, gate_up, down)]

    def both():
        y = ffn.gated_ffn(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    _same(("y", "dx", "dgate_up", "ddown"), both(), _poisoned(ffn, both))
    with torch.no_grad():
        one = lambda: (ffn.gated_ffn(*leaves),)
        _same(("y without a gradient",), one(), _poisoned(ffn, one))


@pytest.mark.parametrize("N,K,O", [(1, 1, 1), (1, 1000, 333), (2, 17, 40), (5, 300, 4100), (40, 77, 130),
                                   (64, 333, 5000), (65, 144, 96), (300, 1001, 130), (700, 2000, 1001),
                                   (3, 9001, 50)])
def test_int8_linear_and_quantised_rows(N, K, O):
    from solvedelta_amd import quant
    print(f"case int8 poison N{N} K{K} O{O}", flush=True)
    g = torch.Generator().manual_seed(K)
    x = torch.randn(N, K, generator=g).to(torch.bfloat16).to(DEV)
    w = torch.randint(-127, 128, (O, K), generator=g, dtype=torch.int8).to(DEV)
    ws, bias = torch.rand(O, generator=g).to(DEV), torch.randn(O, generator=g).to(torch.bfloat16).to(DEV)
    call = lambda: (quant.int8_linear(x, w, ws), quant.int8_linear(x, w, ws, bias))
    _same(("y", "y with a bias"), call(), _poisoned(quant, call))
    for t in (x, x.float()):
        rows = lambda: quant.quantize_int8(t)
        _same(("q", "scale"), rows(), _poisoned(quant, rows))


@pytest.mark.parametrize("B,V", [(1, 1), (3, 63), (2, 5000), (300, 4099)])
def test_sample_tokens(B, V):
    from solvedelta_amd import sampling
    g = torch.Generator().manual_seed(V)
    logits, noise = (2.5 * torch.randn(B, V, generator=g)).to(DEV), torch.rand(B, V, generator=g).to(DEV)
    for kw in ({}, dict(temperature=0.0), dict(top_k=40), dict(top_p=0.9), dict(top_k=400, top_p=0.5),
               dict(min_p=0.05)):
        call = lambda: (sampling.sample_tokens(logits, noise, **kw),)
        _same((str(kw),), call(), _poisoned(sampling, call))
