"""Small weights and small random numbers where few tokens are kept: sums are decided as in float64, in which a weight of
2^-60 beside one of 1 is nothing, and beside a random number of 2^-60 is much.

The wanted tokens are float64's by test_sampling.plain_row.  Small weights come first by index, so its running sums are
right to 2^-53 or so of themselves there; the rows are made so that no border of these lies within 2^-30 of the target,
except at the ties, which are exact in float64: 1 and 1, of weights that round away beside them."""
import math

import pytest
import torch

from qlinear.kernels.sampling import sample_tokens
from test_sampling import TYPES, agree, on_gpu

COUNTS = [40, 128, 129, 700, 1024]         # one CTA compares up to 128 tokens, sorts up to 1024


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", COUNTS)
def test_tokens_of_no_weight_are_not_drawn_at_ties(dtype, n):
    """Two largest and others e^-500 of them: u = 1/2 is between the two, 1 - 2^-24 behind them."""
    x = torch.full((4, n), -500.0)
    x[0, [0, n - 1]] = 0.0                               # the others between the two
    x[1, [n // 2, n // 2 + 1]] = 0.0                     # around them
    x[2, [0, 1]] = 0.0
    x[3, [n - 2, n - 1]] = 0.0
    x = x.to(dtype).cuda()
    wide = torch.full((4, 5000), -math.inf, dtype=dtype, device="cuda")
    wide[:, 17:17 + n] = x
    for u in (0.25, 0.5, 0.75, 1.0 - 2.0 ** -24):
        uniform = torch.full((4,), u, device="cuda")
        for logits in (x, wide):
            for f in (dict(), dict(top_k=n), dict(top_k=30), dict(top_p=0.5), dict(top_p=0.75), dict(top_k=n, top_p=0.5),
                      dict(top_k=n, top_p=0.9), dict(min_p=1e-30)):
                ids = agree(logits, uniform, **f)
                picked = logits.gather(1, ids[:, None])
                assert bool((picked == 0).all()), (u, f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", COUNTS)
def test_small_random_numbers(dtype, n):
    """Tokens of 2^-60 to 2^-20 of the largest, which comes last; random numbers among their sums."""
    g = torch.Generator().manual_seed(n)
    for low, high in ((-60, -50), (-52, -45), (-40, -20), (-140, -100)):
        x = (low + (high - low) * torch.rand(6, n, generator=g)) * math.log(2.0)
        x[:, n - 1] = 0.0
        logits = x.to(dtype)
        # targets in the middle of a token's share
        w = logits.double().exp()
        sums = w.cumsum(1)
        at = torch.randint(0, n - 1, (6,), generator=g)
        rows = torch.arange(6)
        middle = (sums[rows, at] - 0.5 * w[rows, at]) / sums[:, -1]
        u = middle.float()
        near = (sums - u.double()[:, None] * sums[:, -1:]).abs() / (u.double()[:, None] * sums[:, -1:])
        # fp32's rounding of u has not moved it to a border.  (Two rows of six at least: over 40 octaves a token is mostly
        # a small part of the sum up to it, less than 2^-21 with a chance of about one in two.)
        fine = near.amin(1) > 2.0 ** -22
        assert int(fine.sum()) >= 2
        logits, u = logits[fine].cuda(), u[fine].cuda()
        for f in (dict(top_k=n), dict(top_p=1.0 - 1e-9), dict(min_p=1e-44), dict(top_k=n, top_p=1.0 - 1e-9)):
            want = agree(logits, u, **f)
            if "top_p" not in f:
                assert torch.equal(want.cpu(), at[fine])


@on_gpu
@pytest.mark.parametrize("n", COUNTS)
def test_the_ends(n):
    """0 draws the first token that has a weight at all; 1 and above the last such."""
    x = torch.full((2, n), -600.0)
    x[:, n // 2] = 0.0
    x[1, :3] = x[1, -2:] = -800.0                        # none: below e^-700
    logits = x.cuda()
    for f in (dict(top_k=n), dict(min_p=1e-44), dict(top_k=n, top_p=0.999)):
        for u in (0.0, 2.0 ** -149, 1.0):
            agree(logits, torch.full((2,), u, device="cuda"), **f)


@on_gpu
@pytest.mark.parametrize("n", [40, 128, 129, 700, 1000])
def test_small_random_numbers_under_top_k(n):
    """The same where top-k leaves tokens out, which lie among the others by index."""
    g = torch.Generator().manual_seed(100 + n)
    for low, high in ((-60, -55), (-45, -40), (-30, -25)):
        x = (low + (high - low) * torch.rand(6, n + 20, generator=g)) * math.log(2.0)
        x[:, -1] = 0.0
        out = torch.randint(0, n, (6, 20), generator=g)
        x.scatter_(1, out, -200.0)
        w = x.double().exp()
        sums = w.cumsum(1)
        at = torch.randint(n // 2, n, (6,), generator=g)
        rows = torch.arange(6)
        u = ((sums[rows, at] - 0.5 * w[rows, at]) / sums[:, -1]).float()
        # every token left out is e^-200, beneath all sums here; shares are 2^-15 of the sum and more
        for f in (dict(top_k=n + 20 - len(set(out[0].tolist()))), dict(top_k=n, min_p=1e-40)):
            agree(x.cuda(), u.cuda(), **f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 6, 40, 128, 130, 700, 1024])
def test_exact_halves(dtype, n):
    """The second half's tokens weigh what the first half's do: 1/2 of the sum is not exceeded by the first half, whatever
    the weights are and however they are rounded; the next token is drawn."""
    g = torch.Generator().manual_seed(n)
    half = 3.0 * torch.randn(200, n // 2, generator=g)
    other = half.gather(1, torch.rand(half.shape, generator=g).argsort(1))
    x = torch.cat([half, other], 1).to(dtype).cuda()
    uniform = torch.full((200,), 0.5, device="cuda")
    more = torch.cat([x, torch.full_like(x[:, :1], -60000.0)], 1)
    for logits, f in ((more, dict(top_k=n)), (x, dict(min_p=1e-12)), (more[:, :n], dict(top_p=1.0 - 2.0 ** -53))):
        if logits.shape[1] > 1024:
            continue
        assert bool((sample_tokens(logits, uniform, **f) == n // 2).all()), f
