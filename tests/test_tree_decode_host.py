"""examples/tree_decode.py without a GPU."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_tokens_that_do_not_fit_are_refused():
    """Behind the last page their rows would be skipped and their attention cut short, and other tokens come out."""
    import tree_decode
    d = tree_decode.PagedDecoder.__new__(tree_decode.PagedDecoder)
    d.max_positions, d.length = 512, 510
    with pytest.raises(ValueError, match="do not fit"):
        d.forward(torch.zeros(3, dtype=torch.int64))
