"""Where the sampler's cuts fall, exactly, against a full sort in 64 bits: logits on the edge
of two bins of the histogram."""
import math

import pytest
import torch

from test_gpu_sampling import check

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _edges(n):
    """FP32 logits at which 64 (12 - l log2 e), the bin below a largest logit of 0, has another
    whole part with one rounding than with two."""
    g = torch.Generator().manual_seed(0)
    l = -8 * torch.rand(1 << 22, generator=g)
    c = torch.tensor(1.44269504)
    two = ((12 - l * c) * 64).int()
    one = ((12 - l.double() * c.double()).float() * 64).int()
    found = l[two != one]
    assert len(found) >= n
    return found[:n].tolist()


@pytest.mark.parametrize("run", [60, 2500])
@pytest.mark.parametrize("rows", [48, 300])
def test_equal_logits_on_a_bins_edge(run, rows):
    """The cut of top-p and of top-k lies in the middle of a run of equal tokens: it is found
    where the tokens were counted."""
    g = torch.Generator().manual_seed(run)
    for level in _edges(6):
        logits = torch.full((rows, run + 300), level - 6.0)
        logits[:, 0] = 0.0
        logits[:, 1:run + 1] = level
        logits, noise = logits.to(DEV), torch.rand(rows, run + 300, generator=g).to(DEV)
        mass = math.exp(level)
        total = 1 + (run + 299 * math.exp(-6.0)) * mass
        check(logits, noise, top_p=(1 + (run // 2 + 0.5) * mass) / total)
        if run > 600:
            check(logits, noise, top_k=run // 2)
            check(logits, noise, top_k=run // 2, top_p=0.5)
