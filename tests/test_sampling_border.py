"""top-p's border among thousands of tokens where the histogram that narrows it down is at its least precise: logits so far
from 0, for their temperature, that fp32's steps are a good part of an octave of the weight.  Tokens are the float64
definition's, as in test_sampling.py; whatever the histogram leaves, the border is asked of exact sums."""
import math

import pytest
import torch

from test_sampling import agree, on_gpu

# top * log2(e) / T: fp32 weights are used below 2^20, and a histogram's sums are right to 2^-23 of it and some
SHARES = [2.0 ** 8, -2.0 ** 12, 2.0 ** 16, -2.0 ** 18, 2.0 ** 19, -1.04e6, 1.04e6]


@on_gpu
@pytest.mark.parametrize("octaves", [0.5, 6.0, 40.0])
@pytest.mark.parametrize("share", SHARES)
def test_far_from_zero(share, octaves):
    """Logits over so many octaves of the weight, evenly, and heaped at either end."""
    g = torch.Generator().manual_seed(int(abs(share)) + int(octaves))
    for vocab in (2500, 50021):
        even = torch.rand(4, vocab, generator=g, dtype=torch.float64)
        even[1], even[2] = even[1] ** 4, 1.0 - even[2] ** 4
        even[3] = torch.where(torch.rand(vocab, generator=g) < 0.9, 0.3 + 0.01 * even[3], even[3])
        # T = 1: x log2(e) is the share at the top and `octaves` less at the bottom; then other units of the logits
        x = (share - octaves * (1.0 - even)) / math.log2(math.e)
        uniform = torch.rand(4, generator=g).cuda()
        for heat in (1.0, 2.0 ** -10):
            logits = (x * heat).float().cuda()
            for f in (dict(top_p=0.05), dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.9999), dict(top_k=2000, top_p=0.8)):
                agree(logits, uniform, temperature=heat, **f)
