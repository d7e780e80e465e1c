"""The parts together, as examples/tree_decode.py runs them: a quantised model
over the quantised paged cache, against the same model's own attention over
unquantised keys and values, and trees against token-by-token decoding."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


@pytest.fixture(scope="module")
def model():
    import tree_decode
    return tree_decode.build_model(layers=2)


@pytest.mark.parametrize("bits,bound", [(8, 0.9995), (4, 0.97)])
def test_paged_forward_matches_the_models_own(model, bits, bound):
    """Logits of a prompt and of the tokens after it.  8-bit rows are within
    0.4 % of their elements' largest, 4-bit ones within 7 %; in two random-init
    layers that leaves a cosine well above the bounds."""
    import tree_decode
    ids = torch.randint(0, 8192, (45,), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        want = model(ids[None]).logits[0].float()
    d = tree_decode.PagedDecoder(model, bits=bits)
    got = [d.forward(ids[:37])]
    d.accept(range(37))
    for i in range(37, 45):
        got.append(d.forward(ids[i:i + 1]))
        d.accept([0])
    got = torch.cat(got).float()
    cos = torch.nn.functional.cosine_similarity(got, want, dim=-1)
    assert cos.min().item() > bound, cos.min().item()


@pytest.mark.parametrize("bits", [8, 4])
def test_trees_give_the_tokens_of_plain_decoding(model, bits):
    import tree_decode
    from qlinear import _lib
    prompt = torch.randint(0, 8192, (21,), generator=torch.Generator().manual_seed(3)).cuda()
    plain = tree_decode.PagedDecoder(model, bits=bits)
    want = tree_decode.decode_plain(plain, prompt, 24)
    tree = tree_decode.PagedDecoder(model, bits=bits)
    got, passes = tree_decode.decode_tree(tree, prompt, 24, want)
    assert got[:24] == want
    assert passes < 16
    # and the cache holds the same accepted rows, but for what rounding did to their inputs
    n = min(plain.length, tree.length)
    for a, b in zip(plain.cached(1), tree.cached(1)):
        rel = (a[:n].float() - b[:n].float()).norm() / a[:n].float().norm()
        assert rel.item() < (0.02 if bits == 8 else 0.1), rel.item()
    assert _lib.device_error() == 0
