"""What a bound that grows with the number of tokens cannot see: each bfloat16
term of a gradient, and each segment of a long sum.  All on whole numbers
whose sums float32 holds exactly in any order, so results must be equal."""

import pytest
import torch

pytestmark = pytest.mark.gpu

# Odd whole numbers: their lowest bit is in the last term that the type has
# (three bfloat16 terms of 8 bits from 17 bits on, two of float16's 11).
BITS = {torch.float32: 20, torch.float16: 11, torch.bfloat16: 8}
PER_COLUMN = 8  # summands of an output: below 2^(20 + 3), so every partial sum is exact


@pytest.mark.parametrize("shape", [(1, 96, 64), (333, 160, 130), (4100, 513, 77), (20000, 96, 64), (1500, 2600, 2050),
                                   (2500, 256 * 2, 256 * 37)], ids=str)
@pytest.mark.parametrize("dt", list(BITS), ids=str)
@pytest.mark.parametrize("layout", ["io", "oi"])
def test_every_term_of_every_token_counts(shape, dt, layout):
    import rollfast_b200 as rf

    rows, k, n = shape
    gen = torch.Generator("cuda").manual_seed(rows)
    x = torch.zeros(rows, k, device="cuda")
    at = torch.randint(rows, (PER_COLUMN, k), generator=gen, device="cuda")
    x.scatter_(0, at, torch.randint(2, at.shape, generator=gen, device="cuda") * 2.0 - 1.0)
    x[:, ::32] = 127.0  # each block's step is 1; these columns' own sums are left out below
    g = torch.randint(-2 ** (BITS[dt] - 1), 2 ** (BITS[dt] - 1), (rows, n), generator=gen, device="cuda") * 2 + 1
    g = g.float().to(dt)
    saved = rf.save_activation(x)
    assert torch.equal(rf.load_activation(saved, dtype=torch.float32), x)
    want = x.double().t() @ g.double()
    got = rf.weight_gradient(saved, g, layout=layout)
    got = got if layout == "io" else got.t()
    keep = torch.arange(k, device="cuda") % 32 != 0
    assert want[keep].abs().max() < 2 ** 24 and torch.equal(got[keep].double(), want[keep])


@pytest.mark.parametrize("dt", list(BITS), ids=str)
@pytest.mark.parametrize("shape", [(512, 9472), (96, 64), (768, 2304)], ids=str)
@pytest.mark.parametrize("layout", ["io", "oi"])
def test_small_summands_survive_a_large_one(shape, dt, layout):
    """The first token adds 2^30 (float16: 2^21 by 2^9), tokens 2048 and
    later 1 each: in one accumulator their units are below the large sum's
    last place and are lost; apart from it they add up to whole 128s, which
    float32 holds beside 2^30."""
    import rollfast_b200 as rf

    (k, n), rows = shape, 6144
    x = torch.zeros(rows, k, device="cuda")
    g = torch.zeros(rows, n, device="cuda")
    step = 2.0 ** 15 if dt == torch.float16 else 1.0
    x[0], g[0] = 64.0 * step, 2.0 ** 24 / step
    x[2048:], g[2048:] = 64.0, 2.0 ** -6
    saved = rf.save_activation(x)
    assert torch.equal(rf.load_activation(saved, dtype=torch.float32), x)
    got = rf.weight_gradient(saved, g.to(dt), layout=layout)
    assert (got == 2.0 ** 30 + (rows - 2048)).all()
