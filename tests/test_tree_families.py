"""The tests of tree attention once more, with each kernel family forced: the
dispatch takes the tensor-core kernel for many rows and much work only, and
both have to be right at every size."""
import sys

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv
from qlinear.kernels.tree_attention import tree_attention

from attn_helpers import heads
from test_tree_attention import *  # noqa: F401,F403  (collected here again)

pytestmark = pytest.mark.gpu
for _name in ("test_masks", "test_host_checks_without_gpu", "test_refusals", "test_pool_past_32_bit_offsets"):
    globals().pop(_name)               # no family to choose there, or 4 GB a run


@pytest.fixture(autouse=True, params=["tensor cores", "streaming"])
def family(request, monkeypatch):
    force = _lib.QL_FLAG_FORCE_GEMM if request.param == "tensor cores" else _lib.QL_FLAG_FORCE_GEMV
    monkeypatch.setattr(sys.modules[tree_attention.__module__], "call_flags", lambda: _lib.QL_FLAG_PDL | force)
    return request.param


@pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")
def test_pool_past_32_bit_offsets_of_128():
    """Codes of more than 2^32 bytes at the head_dim that both families take: the same as from a small pool."""
    pages, page, hk, d, n = 33000, 256, 4, 128, 300
    ts = [torch.empty(pages, hk, page, w, dtype=t, device="cuda")
          for w, t in ((d, torch.int8), (1, torch.bfloat16)) * 2]
    cache = QuantizedKVCache(*ts)
    assert cache.k_codes.numel() > 1 << 32
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    k, v = heads(n, hk, d, torch.float16, 17), heads(n, hk, d, torch.float16, 18)
    i = torch.arange(n, device="cuda")
    append_kv(cache, k, v, table[0, i // page].long() * page + i % page)
    small = QuantizedKVCache.empty(3, page, hk, d, 8)
    append_kv(small, k, v, i)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    for q_len in (1, 40, 150):
        q = heads(q_len, 8, d, torch.float16, 19)
        assert torch.equal(tree_attention(q, cache, table, lens), tree_attention(q, small, near, lens))
