"""Running sums over whole rows: small weights before the largest, and a random number among them.  What lies before a
token is added up, never had by taking a part away from what lies up to it: where the largest weight is of that part, all
that is smaller than 2^-53 of it would be gone.

Small weights come first by index, so float64's running sums (test_sampling.plain_row) are right to 2^-53 or so of
themselves; targets lie in the middle of a token's share, and rows whose fp32 random number has moved from there are left
out."""
import math

import pytest
import torch

from test_sampling import TYPES, agree, on_gpu


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1024, 5003, 70001])
def test_small_random_numbers_over_the_row(dtype, vocab):
    """The target is 1, 3, 50 or 2000 tokens before the largest: in the same run, warp or CTA as that, or in another."""
    g = torch.Generator().manual_seed(vocab)
    for low, high in ((-60, -50), (-45, -35), (-140, -120)):
        for back in (1, 3, 50, 2000):
            if back >= vocab // 2:
                continue
            most = torch.randint(vocab // 2, vocab, (8,), generator=g)
            x = (low + (high - low) * torch.rand(8, vocab, generator=g)) * math.log(2.0)
            rows = torch.arange(8)
            x[rows, most] = 0.0
            x[torch.arange(vocab) > most[:, None]] = -math.inf
            logits = x.to(dtype)
            w = logits.double().exp()
            sums, at = w.cumsum(1), most - back
            u = ((sums[rows, at] - 0.5 * w[rows, at]) / sums[:, -1]).float()
            target = u.double() * sums[:, -1]
            fine = ((sums - target[:, None]).abs().amin(1) > 2.0 ** -24 * target) & (u > 0)
            if int(fine.sum()) == 0:
                continue
            want = agree(logits[fine].cuda(), u[fine].cuda())
            assert torch.equal(want.cpu(), at[fine])
