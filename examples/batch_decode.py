"""Serving a batch of requests behind one system prompt with a quantised model:
page tables, slots and positions of each step from the requests' lengths,
attention that reads the shared prompt once for all of them, and tokens drawn
with temperature, top-k, top-p and min-p.  Every step is one replay of a captured
graph; requests end and others take their places between replays.

    python examples/batch_decode.py [--bits 8|4] [--batch 8] [--requests 20] [--layers 4]

A random-init model (Qwen2.5-1.5B's layer shapes) is quantised in place.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
for _p in (ROOT / "llm-inference-optimizer_b200", ROOT / "examples"):
    if str(_p) not in sys.path:
        sys.path.insert(0, str(_p))

from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv              # noqa: E402
from qlinear.kernels.paging import PageTables, plan_step                      # noqa: E402
from qlinear.kernels.rotary import RotaryTable                                # noqa: E402
from qlinear.kernels.sampling import sample_tokens                            # noqa: E402
from qlinear.kernels.shared_attention import shared_prefix_attention          # noqa: E402
from qlinear.kernels.tree_attention import tree_attention                     # noqa: E402
from tree_decode import build_model                                           # noqa: E402


class BatchDecoder:
    """Decodes up to `batch` requests at a time behind one prompt, a token each
    a step, with one quantised cache per layer whose pages they share."""

    def __init__(self, model, prompt: torch.Tensor, batch: int, num_pages: int, pages_each: int, bits: int = 8,
                 page_size: int = 16, graph: bool = True, **sampling):
        cfg = model.config
        self.model, self.batch, self.sampling = model, batch, sampling
        self.head_dim = cfg.hidden_size // cfg.num_attention_heads
        self.caches = [QuantizedKVCache.empty(num_pages, page_size, cfg.num_key_value_heads, self.head_dim, bits)
                       for _ in model.model.layers]
        self.rotary = RotaryTable.from_config(cfg, prompt.shape[0] + pages_each * page_size)
        self.pages = PageTables.empty(batch, pages_each, num_pages, page_size)
        # the prompt's pages come from the same stack
        room = -(-prompt.shape[0] // page_size)
        self.prefix = PageTables(torch.zeros(1, room, dtype=torch.int32, device="cuda"),
                                 torch.zeros(1, dtype=torch.int32, device="cuda"), self.pages.free_pages,
                                 self.pages.free_count, page_size)
        self.prompt_len = prompt.shape[0]
        plan = plan_step(self.prefix, self._ints([self.prompt_len]), self.prompt_len)
        if int(plan.refused):
            raise ValueError(f"a prompt of {self.prompt_len} tokens needs {room} pages, the pool has {num_pages}")
        self._fill(prompt, plan, self.prefix, None)
        # a step's buffers, which the graph reads and writes
        self.new = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.keep = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.uniform = torch.zeros(batch, device="cuda")
        self.tokens = torch.zeros(batch + 1, dtype=torch.int64, device="cuda")   # each request's last; one for no request
        self.plan = self.pages.step_buffers(batch)
        self.places = torch.arange(batch, device="cuda", dtype=torch.int32)
        self.graph = None
        if graph:
            self._step()                             # nothing is asked for: buffers and workspaces come to be
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._step()

    @staticmethod
    def _ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    @torch.no_grad()
    def _layers(self, ids, plan, attend, offset):
        """Logits of tokens ids at the plan's slots and positions, these counted from `offset`."""
        inner = self.model.model
        positions = plan.positions + offset
        h = inner.embed_tokens(ids.clamp(min=0))              # -1: a row that had nothing to draw
        for layer, cache in zip(inner.layers, self.caches):
            attn = layer.self_attn
            q, k, v = (t.unflatten(-1, (-1, self.head_dim)) for t in attn.qkv_proj(layer.input_layernorm(h)))
            q = append_kv(cache, k, v, plan.slots, q=q, positions=positions, rotary=self.rotary)
            h = h + attn.o_proj(attend(q, cache).flatten(1))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        return self.model.lm_head(inner.norm(h))

    def _fill(self, ids, plan, tables, prefix):
        """Caches a prompt's tokens; the last one's logits."""
        def attend(q, cache):
            if prefix is None:
                return tree_attention(q, cache, tables.page_table, plan.kv_lens, cu_q=plan.cu_q)
            return shared_prefix_attention(q, cache, prefix.page_table, prefix.lens, tables.page_table, plan.kv_lens,
                                           cu_q=plan.cu_q)
        return self._layers(ids, plan, attend, 0 if prefix is None else self.prompt_len)[-1:]

    def _step(self):
        plan = plan_step(self.pages, self.new, self.batch, keep=self.keep, out=self.plan)
        # rows are the served requests' in order; the others, behind them, belong to none
        owner = torch.searchsorted(plan.cu_q[1:], self.places, right=True).clamp(max=self.batch - 1)
        owner = torch.where(self.places < plan.cu_q[-1], owner, self.batch)

        def attend(q, cache):
            return shared_prefix_attention(q, cache, self.prefix.page_table, self.prefix.lens, self.pages.page_table,
                                           plan.kv_lens, cu_q=plan.cu_q, max_q=1, out=torch.zeros_like(q))
        logits = self._layers(self.tokens[owner], plan, attend, self.prompt_len)
        ids = sample_tokens(logits, self.uniform, **self.sampling)
        self.tokens.scatter_(0, owner, ids)
        self.keep.copy_(self.pages.lens)

    def start(self, place: int, ids: torch.Tensor, uniform: torch.Tensor) -> bool:
        """Begins a request at a free place: caches its tokens and draws its first by uniform (1,).  False if the pool has
        no pages for it."""
        new = self._ints([ids.shape[0] if b == place else 0 for b in range(self.batch)])
        plan = plan_step(self.pages, new, ids.shape[0], keep=self.keep)
        if int(plan.refused):
            return False
        logits = self._fill(ids, plan, self.pages, self.prefix)
        self.tokens[place] = sample_tokens(logits, uniform, **self.sampling)[0]
        self.keep.copy_(self.pages.lens)
        self.new[place] = 1
        return True

    def end(self, place: int) -> None:
        """Ends a request; the next step gives its pages back."""
        self.new[place] = 0
        self.keep[place] = 0

    def step(self, uniform: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """A token for each request that runs, by uniform (batch,): each place's last token, and whether the place was
        served (one that needs a page when none is free is not)."""
        self.uniform.copy_(uniform)
        if self.graph is None:
            self._step()
        else:
            self.graph.replay()
        return self.tokens[:self.batch], self.plan.cu_q[1:] > self.plan.cu_q[:-1]


def serve(decoder: BatchDecoder, prompts, lengths, seed: int = 0):
    """Runs all prompts, each for its number of tokens; returns their tokens and the number of steps.  Where the running
    requests wait for one another's pages, the last one begins again later."""
    device = decoder.tokens.device
    g = torch.Generator(device=device).manual_seed(seed)
    waiting, at, out = [r for r, n in enumerate(lengths) if n > 0], [None] * decoder.batch, [[] for _ in prompts]
    steps, short = 0, False

    def take(r: int, token: int) -> None:
        if token < 0:
            raise ValueError(f"request {r} has nothing to draw from after {len(out[r])} tokens: are its logits NaN?")
        out[r].append(token)
    while waiting or any(r is not None for r in at):
        refused = False
        for place, running in enumerate(at):
            if running is None and waiting and not short:
                draw = torch.rand(1, generator=g, device=device)
                if decoder.start(place, prompts[waiting[0]], draw):
                    at[place] = waiting.pop(0)
                    take(at[place], int(decoder.tokens[place]))
                    if lengths[at[place]] == 1:
                        decoder.end(place)
                        at[place] = None
                else:
                    refused = True
        if refused and all(r is None for r in at):
            raise ValueError(f"the pool is too small for request {waiting[0]}'s prompt alone")
        tokens, served = (t.tolist() for t in decoder.step(torch.rand(decoder.batch, generator=g, device=device)))
        steps += 1
        running = [place for place, r in enumerate(at) if r is not None]
        short = not all(served[place] for place in running)
        for place in running:
            r = at[place]
            if served[place]:
                take(r, tokens[place])
            if len(out[r]) >= lengths[r]:
                decoder.end(place)
                at[place] = None
        if running and not any(served[place] for place in running):
            if len(running) == 1:
                raise ValueError("the pool is too small for a request alone")
            place = max(running, key=lambda place: at[place])
            decoder.end(place)
            waiting.insert(0, at[place])
            out[at[place]], at[place] = [], None
    decoder.step(torch.zeros(decoder.batch, device=device))          # the last ones' pages
    return out, steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--bits", type=int, default=8, choices=(8, 4), help="bits of a cached element")
    ap.add_argument("--batch", type=int, default=8, help="requests at a time")
    ap.add_argument("--requests", type=int, default=20)
    ap.add_argument("--layers", type=int, default=4)
    args = ap.parse_args()
    model = build_model(args.layers)
    vocab = model.config.vocab_size
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, vocab, (200,), generator=g).cuda()
    asked = [torch.randint(0, vocab, (5 + 7 * i % 30,), generator=g).cuda() for i in range(args.requests)]
    lengths = [12 + 5 * i % 40 for i in range(args.requests)]
    decoder = BatchDecoder(model, prompt, args.batch, num_pages=13 + 6 * args.batch, pages_each=6, bits=args.bits,
                           temperature=0.8, top_k=50, top_p=0.95)
    torch.cuda.synchronize()
    t = time.perf_counter()
    out, steps = serve(decoder, asked, lengths)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    print(f"{args.requests} requests, {sum(map(len, out))} tokens in {steps} steps, {1e3 * t:.1f} ms; "
          f"{int(decoder.pages.free_count)} of {decoder.pages.num_pages} pages free")


if __name__ == "__main__":
    main()
