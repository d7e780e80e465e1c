"""examples/batch_decode.py without a GPU: how requests are served by a decoder that only counts, and what becomes of a row
that had nothing to draw."""
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


class Counter:
    """A decoder of `batch` places and `room` tokens, whose requests' tokens count up from their prompt's length."""

    def __init__(self, batch: int, room: int):
        self.batch, self.room = batch, room
        self.tokens = torch.zeros(batch + 1, dtype=torch.int64)
        self.held, self.left = [0] * batch, 200

    def start(self, place, ids, uniform):
        self.left -= 1
        assert self.left > 0, "serve goes on without end"
        if sum(self.held) + len(ids) > self.room:
            return False
        self.held[place], self.tokens[place] = len(ids), len(ids)
        return True

    def end(self, place):
        self.held[place] = 0

    def step(self, uniform):
        self.left -= 1
        assert self.left > 0, "serve goes on without end"
        served = torch.zeros(self.batch, dtype=torch.bool)
        for place in range(self.batch):
            if self.held[place] and sum(self.held) < self.room:
                self.held[place] += 1
                self.tokens[place] += 1
                served[place] = True
        return self.tokens[:self.batch], served


def prompts(*lengths):
    return [torch.zeros(n, dtype=torch.int64) for n in lengths]


def test_requests_wait_for_one_another():
    from batch_decode import serve
    out, _ = serve(Counter(2, 12), prompts(3, 2, 4), [5, 9, 4])
    assert out == [list(range(3, 8)), list(range(2, 11)), list(range(4, 8))]


def test_a_request_that_never_fits_is_refused():
    """Behind others that do, or at once: nothing runs whose end could make room."""
    from batch_decode import serve
    with pytest.raises(ValueError, match="too small"):
        serve(Counter(2, 10), prompts(3, 11), [2, 2])
    with pytest.raises(ValueError, match="too small"):
        serve(Counter(1, 10), prompts(11), [2])


def test_as_many_tokens_as_asked_for():
    """The first comes with the prompt: a request for one token has no step, one for none does not begin."""
    from batch_decode import serve
    out, steps = serve(Counter(2, 40), prompts(3, 5, 6, 7), [1, 0, 2, 1])
    assert out == [[3], [], [6, 7], [7]]
    out, _ = serve(Counter(1, 5), prompts(5, 4, 5), [1, 1, 1])          # no room for a step
    assert out == [[5], [4], [5]]


def test_a_prompt_that_does_not_fit_the_pool(monkeypatch):
    """Its plan has no tokens, and all requests would be answered without it."""
    import batch_decode
    refused = SimpleNamespace(refused=torch.tensor([1], dtype=torch.int32))
    monkeypatch.setattr(batch_decode, "plan_step", lambda *args, **kwargs: refused)
    monkeypatch.setattr(batch_decode.BatchDecoder, "_fill", lambda *args: pytest.fail("goes on without its prompt"))
    monkeypatch.setattr(batch_decode.BatchDecoder, "_ints", staticmethod(lambda v: torch.tensor(v, dtype=torch.int32)))
    monkeypatch.setattr(batch_decode.QuantizedKVCache, "empty", lambda *args, **kwargs: None)
    monkeypatch.setattr(batch_decode.RotaryTable, "from_config", lambda *args, **kwargs: None)
    empty, zeros = batch_decode.PageTables.empty, torch.zeros
    monkeypatch.setattr(batch_decode.PageTables, "empty", lambda *args: empty(*args, device="cpu"))
    monkeypatch.setattr(torch, "zeros", lambda *args, device="cpu", **kwargs: zeros(*args, **kwargs))
    config = SimpleNamespace(hidden_size=128, num_attention_heads=2, num_key_value_heads=1)
    model = SimpleNamespace(config=config, model=SimpleNamespace(layers=[]))
    with pytest.raises(ValueError, match="prompt"):
        batch_decode.BatchDecoder(model, torch.arange(70), 2, num_pages=4, pages_each=2)


def test_a_row_with_nothing_to_draw():
    """sample_tokens gives -1 for it (all of its logits NaN): no index of the embedding, where it would end the process on
    a GPU, and no token for the user either."""
    from batch_decode import BatchDecoder, serve
    d = BatchDecoder.__new__(BatchDecoder)
    inner = SimpleNamespace(embed_tokens=torch.nn.Embedding(5, 4), layers=[], norm=lambda h: h)
    d.model, d.caches = SimpleNamespace(model=inner, lm_head=lambda h: h), []
    plan = SimpleNamespace(positions=torch.zeros(3, dtype=torch.int32))
    got = d._layers(torch.tensor([1, -1, 4]), plan, None, 0)
    assert torch.equal(got, inner.embed_tokens.weight[[1, 0, 4]])

    class Nothing(Counter):
        def step(self, uniform):
            tokens, served = super().step(uniform)
            tokens[0] = -1
            return tokens, served

    with pytest.raises(ValueError, match="nothing to draw"):
        serve(Nothing(2, 40), prompts(3, 5), [4, 4])

    class AtOnce(Counter):
        def start(self, place, ids, uniform):
            started = super().start(place, ids, uniform)
            self.tokens[place] = -1
            return started

    with pytest.raises(ValueError, match="nothing to draw"):
        serve(AtOnce(2, 40), prompts(3, 5), [4, 4])
