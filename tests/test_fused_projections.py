"""The fused MLP runs as one operator only where its projections are plain bias-free Linears
that nothing watches or changes; else they run on their own (here on the CPU, where the fused
operator would raise)."""
import pytest
import torch
from torch import nn
import torch.nn.functional as F

NAMES = ("gate_up_proj", "down_proj")


def _mlp():
    from solvedelta_amd.lm import SolveDeltaMLP
    torch.manual_seed(0)
    return SolveDeltaMLP(16, 2, fused=True)


def _apart(mlp, x):
    gate, up = mlp.gate_up_proj(x).chunk(2, -1)
    return mlp.down_proj(F.silu(gate) * up)


def test_plain_projections_run_as_one():
    with pytest.raises(TypeError):
        _mlp()(torch.randn(2, 16))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook",
                                      "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_see_the_projection(name, register):
    mlp, seen = _mlp(), []
    handle = getattr(getattr(mlp, name), register)(lambda *a: seen.append(1) and None)
    x = torch.randn(2, 16, requires_grad=True)
    mlp(x).sum().backward()
    assert seen
    handle.remove()
    with pytest.raises(TypeError):
        mlp(x)


def test_hooks_of_all_modules_see_the_projections():
    mlp, seen = _mlp(), []
    handle = nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m) and None)
    try:
        mlp(torch.randn(2, 16))
    finally:
        handle.remove()
    assert mlp.gate_up_proj in seen and mlp.down_proj in seen


@pytest.mark.parametrize("name", NAMES)
def test_a_bias_counts(name):
    mlp, old = _mlp(), getattr(_mlp(), name)
    setattr(mlp, name, nn.Linear(old.in_features, old.out_features))
    x = torch.randn(2, 16)
    assert torch.equal(mlp(x), _apart(mlp, x))


@pytest.mark.parametrize("name", NAMES)
def test_a_forward_of_its_own_counts(name):
    mlp = _mlp()
    proj = getattr(mlp, name)
    plain = proj.forward
    proj.forward = lambda t: 2 * plain(t)
    x = torch.randn(2, 16)
    y = mlp(x)
    assert torch.equal(y, _apart(mlp, x))
    del proj.forward
    assert not torch.equal(y, _apart(mlp, x))
