"""``generate``'s tokens are ``sample_tokens``' for the last position's logits, under every
setting, with the generator's random numbers one step after another."""
import pytest
import torch

from test_gpu_generate import _ids, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("kw", [{}, dict(temperature=0.0), dict(temperature=0.8, top_k=20, top_p=0.9),
                                dict(temperature=1.4, top_p=0.6), dict(min_p=0.2), dict(top_k=3)])
def test_every_token_is_the_draw(fused, kw):
    from solvedelta_amd import sample_tokens
    from solvedelta_amd.cache import RecurrentCache
    model = _model(seed=6, fused=fused).to(torch.bfloat16).eval()
    ids, new = _ids(8, 17), 12
    out = model.generate(ids, new, generator=torch.Generator("cuda").manual_seed(7), **kw)
    assert out.shape == (8, 17 + new) and torch.equal(out[:, :17], ids)
    g, cache, step = torch.Generator("cuda").manual_seed(7), RecurrentCache(), ids
    with torch.no_grad():
        for i in range(new):
            h, cache = model.model(step, past_key_values=cache, use_cache=True)
            last = model.lm_head(h[:, -1])
            noise = torch.rand(last.shape, dtype=torch.float32, device="cuda", generator=g)
            step = sample_tokens(last, noise, **kw)[:, None]
            assert torch.equal(out[:, 17 + i], step[:, 0]), i


def test_the_settings_matter_here():
    """Each filter changes some of the tokens that the test above compares."""
    model = _model(seed=6).to(torch.bfloat16).eval()
    draw = lambda **kw: model.generate(_ids(8, 17), 12, generator=torch.Generator("cuda").manual_seed(7), **kw)
    free = draw()
    for kw in (dict(temperature=1.4), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2)):
        assert not torch.equal(draw(**kw), free), kw
