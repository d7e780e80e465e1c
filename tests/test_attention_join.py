"""Items in many parts, whose last group has one part and in whose last CTA
the next item begins: the same bits on every call while another stream holds
part of the SMs, and a scratch head that each call leaves zero."""
import sys

import pytest
import torch

from qlinear import _lib
from qlinear.kernels import _launch
from qlinear.kernels.tree_attention import tree_attention

from test_tree_attention import Problem

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]

# requests, positions, new tokens, query and key/value heads, and the kernel that is forced: with 148 SMs the first two
# have items of 17 parts one after another (see test_work_split.py), the others many parts of other counts
CASES = [(9, 8192, 1, 8, 2, "streaming"), (9, 9000, 64, 4, 1, "tensor cores"), (4, 60185, 1, 16, 4, "streaming"),
         (3, 33000, 70, 8, 2, "tensor cores"), (5, 20011, 3, 12, 2, "streaming")]


def head(stream):
    buf = _launch._scratches[(torch.cuda.current_device(), stream.cuda_stream)]
    return buf[:_launch._SCRATCH_HEADER]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,kv,q_len,q_heads,kv_heads,family", CASES)
def test_parts_meet_while_sms_are_held(batch, kv, q_len, q_heads, kv_heads, family, dtype, monkeypatch):
    force = _lib.QL_FLAG_FORCE_GEMM if family == "tensor cores" else _lib.QL_FLAG_FORCE_GEMV
    monkeypatch.setattr(sys.modules[tree_attention.__module__], "call_flags", lambda: _lib.QL_FLAG_PDL | force)
    p = Problem([q_len] * batch, [kv] * batch, q_heads, kv_heads, 128, 8, 64, dtype, seed=kv)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda", dtype=torch.float16)
    c = torch.empty_like(a)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = p.run()
        assert int(head(stream).count_nonzero()) == 0
        got, heads = [], []
        for i in range(24):
            if i % 4 == 0:                              # products that start at another point of each call
                with torch.cuda.stream(other):
                    for _ in range(1 + i // 4):
                        torch.mm(a, a, out=c)
            got.append(p.run())
            heads.append(head(stream).count_nonzero())
    torch.cuda.synchronize()
    assert [int(h) for h in heads] == [0] * len(heads)
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    p.check(want)
