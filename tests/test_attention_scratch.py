"""Scratch of tree attention: a buffer that a larger call outgrows stays for
the graphs that captured it; one that is too small is refused."""
import sys
import weakref

import pytest
import torch

from qlinear import _lib
from qlinear.kernels import _launch
from qlinear.kernels.kv_cache import QuantizedKVCache
from qlinear.kernels.tree_attention import tree_attention

from attn_helpers import heads, random_cache

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def test_outgrown_scratch_stays_for_captured_graphs():
    stream = torch.cuda.Stream()
    lens = torch.tensor([1500], dtype=torch.int32, device="cuda")
    table = torch.arange(94, dtype=torch.int32, device="cuda")[None]
    sizes = [_lib.load().ql_tree_attention_workspace_size(d) for d in (64, 128)]
    assert sizes[0] < sizes[1]
    small, large = (QuantizedKVCache(*random_cache(94, 16, 2, d, 8, 1)) for d in (64, 128))
    q = heads(3, 4, 64, torch.float16, 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = tree_attention(q, small, table, lens)
        held = weakref.ref(_launch._scratches[(torch.cuda.current_device(), stream.cuda_stream)])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = tree_attention(q, small, table, lens)
        tree_attention(heads(3, 4, 128, torch.float16, 3), large, table, lens)
        assert held() is not None
        graph.replay()
    stream.synchronize()
    assert torch.equal(out, want)


def test_small_scratch_is_refused(monkeypatch):
    module = sys.modules[tree_attention.__module__]
    monkeypatch.setattr(module, "scratch", lambda device, stream, n: torch.zeros(8192, dtype=torch.uint8, device=device))
    with pytest.raises(_lib.QLinearError):
        tree_attention(heads(1, 4, 64, torch.float16, 4), QuantizedKVCache(*random_cache(2, 16, 2, 64, 8, 5)),
                       torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"),
                       torch.tensor([20], dtype=torch.int32, device="cuda"))


def test_graphs_have_scratch_of_their_own():
    """A graph captured on a stream that has scratch, another captured after it there, and eager calls on that stream,
    all at once: their scratch is apart, and each gives the bits that it gives alone."""
    stream, aside = torch.cuda.Stream(), torch.cuda.Stream()
    cache = QuantizedKVCache(*random_cache(626, 64, 2, 128, 8, 6))
    lens = torch.tensor([40000], dtype=torch.int32, device="cuda")
    table = torch.arange(626, dtype=torch.int32, device="cuda")[None]
    qs = [heads(3, 4, 128, torch.float16, s) for s in (7, 8, 9)]
    key = (torch.cuda.current_device(), stream.cuda_stream)
    torch.cuda.synchronize()
    graphs, outs, buffers = [], [], []
    with torch.cuda.stream(stream):
        want = [tree_attention(q, cache, table, lens) for q in qs]
        buffers.append(_launch._scratches[key].data_ptr())
        for q in qs[1:]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                outs.append([tree_attention(q, cache, table, lens) for _ in range(3)])
                buffers.append(_launch._graph_scratches[key][1].data_ptr())
    torch.cuda.synchronize()
    assert len(set(buffers)) == 3
    for _ in range(20):
        with torch.cuda.stream(aside):
            graphs[0].replay()
        graphs[1].replay()
        with torch.cuda.stream(stream):
            got = [tree_attention(qs[0], cache, table, lens) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[0]) for g in got)
    for out, w in zip(outs, want[1:]):
        assert all(torch.equal(o, w) for o in out)
