"""An Int8Linear keeps the types its product takes wherever its model is moved or cast."""
import pytest
import torch
from torch import nn


def _filled(device="cpu"):
    from solvedelta_amd import Int8Linear
    q = Int8Linear(6, 3, bias=True, device=device)
    g = torch.Generator().manual_seed(0)
    q.weight.copy_(torch.randint(-127, 128, (3, 6), generator=g))
    q.weight_scale.copy_(torch.rand(3, generator=g))
    q.bias.copy_(torch.randn(3, generator=g))
    return q


CASTS = [lambda m: m.to(torch.bfloat16), lambda m: m.to(torch.float16), lambda m: m.float(),
         lambda m: m.double(), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to("cpu"),
         lambda m: m.to(torch.device("cpu"), torch.float64)]


@pytest.mark.parametrize("cast", CASTS)
def test_casts_of_a_model_leave_it(cast):
    q = _filled()
    want = {k: v.clone() for k, v in q.state_dict().items()}
    model = cast(nn.Sequential(nn.Linear(6, 6), q))
    assert model[1] is q
    got = q.state_dict()
    assert list(got) == list(want)
    for k, v in want.items():
        assert got[k].dtype == v.dtype and torch.equal(got[k], v), k


def test_the_meta_device_and_back():
    q = _filled().to("meta")
    assert {v.device.type for v in q.state_dict().values()} == {"meta"}
    q = q.to_empty(device="cpu")
    assert (q.weight.dtype, q.weight_scale.dtype, q.bias.dtype) == (torch.int8, torch.float32, torch.bfloat16)
    q.load_state_dict(_filled().state_dict())
    assert torch.equal(q.weight_scale, _filled().weight_scale)


@pytest.mark.gpu
def test_it_runs_after_a_cast():
    q = _filled().to("cuda")
    x = torch.randn(4, 6, generator=torch.Generator().manual_seed(1)).cuda()
    want = q(x)
    for cast in CASTS[:6]:
        assert torch.equal(cast(q)(x), want)
