"""Where the sampler's cuts fall, exactly, against a full sort in 64 bits: logits on the edge
of two bins of the histogram, and a heavy token over very many light ones."""
import math

import pytest
import torch

from test_gpu_sampling import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOW, HIGH = 2.0 ** -25, 1 - 2.0 ** -24   # the ends that random numbers are read between


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


@pytest.mark.parametrize("V", [5000, 131072, 1 << 20])
@pytest.mark.parametrize("first", [True, False])
def test_half_of_a_light_tail_is_kept(V, first):
    """One token with nearly all of the mass over V - 1 light ones, of which top-p keeps half:
    a light token's mass is not rounded to a share of the largest's.  Two thousandths of the
    tail before and behind the cut (FP32's rounding of a mass moves it by 1e-6 of itself)."""
    g = torch.Generator().manual_seed(V)
    units = 4.5 * 2.0 ** -30     # half way between two multiples of 2^-30
    z = torch.tensor(math.log(units)).item()
    n, mass = V - 1, math.exp(z)
    head = 0 if first else V - 1
    places = [int(n * f) for f in (0.1, 0.4, 0.45, 0.48, 0.498, 0.502, 0.52, 0.55, 0.6, 0.9)]
    logits = torch.full((len(places), V), z)
    logits[:, head] = 0.0
    # the head is as slow as can be, one light token as fast: it is drawn if it is kept
    noise = torch.full((len(places), V), 0.5)
    noise[:, head] = LOW
    for i, j in enumerate(places):
        noise[i, j + (1 if first else 0)] = HIGH
    p = (1 + 0.5 * n * mass) / (1 + n * mass)
    check(logits.to(DEV), noise.to(DEV), top_p=p)
    check(logits.to(DEV), noise.to(DEV), top_p=p, top_k=V - 1)


@pytest.mark.parametrize("V", [32000, 131072, 1 << 22])
def test_a_tail_too_light_to_be_drawn_moves_the_cut(V):
    """A head, 20 tokens far below it, and a flat tail whose tokens hold less than 2^-31 each but
    together as much as the 20: ten of these are kept, whatever the tail's tokens round to."""
    z_mid, z_tail = -12.0, math.log(0.45 * 2.0 ** -30)
    tail = (V - 21) * math.exp(z_tail)
    if tail < 20 * math.exp(z_mid):
        z_mid = math.log(tail / 20)
    z_mid, z_tail = (torch.tensor(z).item() for z in (z_mid, z_tail))
    mid, tail = math.exp(z_mid), (V - 21) * math.exp(z_tail)
    rows = (0, 5, 8, 9, 10, 19)
    logits = torch.full((len(rows), V), z_tail)
    logits[:, 7] = 0.0
    logits[:, 100:120] = z_mid
    noise = torch.full((len(rows), V), 0.5)
    for i, j in enumerate(rows):
        noise[i, 100 + j] = HIGH
    p = (1 + 9.5 * mid) / (1 + 20 * mid + tail)
    check(logits.to(DEV), noise.to(DEV), top_p=p)
