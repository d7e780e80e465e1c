"""Which kernel tree_attention takes, told by its bits: the two families and the
tile sizes add in different orders."""
import sys

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.tree_attention import tree_attention

from test_tree_attention import Problem

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def forced(p, monkeypatch, flag, **more):
    with monkeypatch.context() as m:
        m.setattr(sys.modules[tree_attention.__module__], "call_flags", lambda: _lib.QL_FLAG_PDL | flag)
        return p.run(**more)[0]


def test_single_tokens_are_streamed_whatever_is_known_of_them(monkeypatch):
    """64 requests of one token, with cu_q alone: the kernel and the bits of the call without cu_q, not those of the
    tensor-core kernel, which 64 requests of 64 tokens would take."""
    p = Problem([1] * 64, [3000 - 20 * i for i in range(64)], 32, 8, 128, 8, 64, torch.float16, seed=41)
    plain = p.run(cu_q=None)[0]
    other = forced(p, monkeypatch, _lib.QL_FLAG_FORCE_GEMM)
    assert not torch.equal(plain, other)                     # so that bits do tell
    for more in ({}, dict(max_q=1), dict(max_q=64), dict(max_q=1 << 40, max_kv=1 << 60)):
        assert torch.equal(p.run(**more)[0], plain)
    p.check(p.run())


@pytest.mark.parametrize("trees,tensor", [(1, False), (40, True)])
def test_a_mixed_batch_goes_by_its_mean(trees, tensor, monkeypatch):
    p = Problem([32] * trees + [1] * (48 - trees), [1500] * 48, 28, 4, 128, 8, 16, torch.float16, "tree", seed=42)
    got, sides = p.run(max_q=32), [forced(p, monkeypatch, f, max_q=32) for f in (_lib.QL_FLAG_FORCE_GEMV, _lib.QL_FLAG_FORCE_GEMM)]
    assert not torch.equal(*sides)
    assert torch.equal(got[0], sides[tensor])
    p.check(got)


def test_ragged_trees_go_by_the_largest_above_the_mean(monkeypatch):
    """16 requests of up to 600 positions and 9 tokens, 57 rows on the average and 72 at most: the tensor-core kernel."""
    p = Problem([9 - i % 5 for i in range(16)], [600 - 14 * i for i in range(16)], 32, 4, 128, 8, 16, torch.float16, "tree",
                seed=43)
    got, sides = p.run(max_q=9), [forced(p, monkeypatch, f, max_q=9) for f in (_lib.QL_FLAG_FORCE_GEMV, _lib.QL_FLAG_FORCE_GEMM)]
    assert not torch.equal(*sides) and torch.equal(got[0], sides[1])
    p.check(got)
