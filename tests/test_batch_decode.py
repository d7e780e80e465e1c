"""examples/batch_decode.py: it runs, a captured step draws the tokens that an eager one draws, and all pages come back."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


@pytest.mark.parametrize("bits", [8, 4])
def test_batch_decode(bits):
    pytest.importorskip("transformers")
    from batch_decode import BatchDecoder, serve
    from tree_decode import build_model
    model = build_model(layers=2)
    g = torch.Generator().manual_seed(2)
    vocab = model.config.vocab_size
    prompt = torch.randint(0, vocab, (70,), generator=g).cuda()
    asked = [torch.randint(0, vocab, (3 + 5 * i % 17,), generator=g).cuda() for i in range(7)]
    lengths = [4 + 3 * i % 20 for i in range(7)]
    runs = []
    for graph in (False, True):
        # pages for two of the three at their longest: some requests wait for pages, one begins again
        decoder = BatchDecoder(model, prompt, 3, num_pages=5 + 6, pages_each=3, bits=bits, graph=graph, temperature=0.9,
                               top_k=30, top_p=0.9)
        out, steps = serve(decoder, asked, lengths, seed=5)
        assert [len(o) for o in out] == lengths and all(0 <= t < vocab for o in out for t in o)
        assert int(decoder.pages.free_count) == 6 and decoder.pages.lens.tolist() == [0] * 3
        assert sorted(decoder.pages.free_pages[:6].tolist() + decoder.prefix.page_table[0].tolist()) == list(range(11))
        runs.append((out, steps))
    assert runs[0] == runs[1]
