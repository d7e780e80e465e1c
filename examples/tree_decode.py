"""Speculative decoding of a quantised Qwen2-style model over a quantised paged
cache: the weight-only quantised projections with rotary positions, the cache
and tree attention between them.

    python examples/tree_decode.py [--bits 8|4] [--new 48] [--layers 4]

A random-init model (Qwen2.5-1.5B's layer shapes) is quantised in place and
decoded twice from the same prompt: token by token, and with trees of drafted
tokens that one pass verifies.  Both give the same tokens; the second needs
fewer passes.  The drafts stand in for a draft model: the continuation with
some tokens replaced, plus side branches.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / "llm-inference-optimizer_b200") not in sys.path:
    sys.path.insert(0, str(ROOT / "llm-inference-optimizer_b200"))

from qlinear.kernels.fused_mlp import fuse_mlp_gate_up                      # noqa: E402
from qlinear.kernels.fused_qkv import fuse_attention_qkv                    # noqa: E402
from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv, read_kv   # noqa: E402
from qlinear.kernels.rotary import RotaryTable                              # noqa: E402
from qlinear.kernels.tree_attention import tree_attention, tree_mask_from_parents  # noqa: E402
from qlinear.quantization.int4 import quantize_model_int4                   # noqa: E402


class PagedDecoder:
    """Runs a quantised decoder model over one quantised cache per layer, for
    one request whose pages are the pool's in order."""

    def __init__(self, model, bits: int = 8, page_size: int = 16, max_positions: int = 512):
        cfg = model.config
        self.model = model
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim = cfg.hidden_size // self.heads
        pages = -(-max_positions // page_size)
        self.caches = [QuantizedKVCache.empty(pages, page_size, self.kv_heads, self.head_dim, bits)
                       for _ in model.model.layers]
        self.rotary = RotaryTable.from_config(cfg, pages * page_size)
        self.page_table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        self.max_positions = pages * page_size
        self.length = 0                              # positions that hold accepted tokens

    @torch.no_grad()
    def forward(self, ids: torch.Tensor, depth: torch.Tensor = None, mask: torch.Tensor = None) -> torch.Tensor:
        """Logits of new tokens ids (n,), written behind the accepted ones.
        `depth` is each token's distance from the first (its place in the
        sequence), `mask` which of the new tokens each sees; by default a chain."""
        n = ids.shape[0]
        if self.length + n > self.max_positions:
            raise ValueError(f"{n} tokens behind {self.length} do not fit {self.max_positions} positions")
        slots = torch.arange(self.length, self.length + n, device="cuda")
        positions = slots if depth is None else self.length + depth
        kv_lens = torch.tensor([self.length + n], dtype=torch.int32, device="cuda")
        inner = self.model.model
        h = inner.embed_tokens(ids)
        for layer, cache in zip(inner.layers, self.caches):
            attn = layer.self_attn
            q, k, v = (t.unflatten(-1, (-1, self.head_dim)) for t in attn.qkv_proj(layer.input_layernorm(h)))
            q = append_kv(cache, k, v, slots, q=q, positions=positions, rotary=self.rotary)
            o = tree_attention(q, cache, self.page_table, kv_lens, mask=mask)
            h = h + attn.o_proj(o.flatten(1))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        return self.model.lm_head(inner.norm(h))

    def accept(self, path) -> None:
        """Keeps the new tokens on `path` (indexes, in order) and closes their
        rows up behind the accepted ones."""
        src = self.length + torch.tensor(path, device="cuda")
        dst = self.length + torch.arange(len(path), device="cuda")
        if not torch.equal(src, dst):
            for cache in self.caches:
                cache.move(src, dst)
        self.length += len(path)

    def cached(self, layer: int):
        """The accepted tokens' keys and values of a layer, as 16-bit values."""
        return read_kv(self.caches[layer], torch.arange(self.length, device="cuda"))


def build_model(layers: int = 4, vocab: int = 8192):
    from transformers import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=vocab, hidden_size=1536, intermediate_size=8960, num_hidden_layers=layers,
                      num_attention_heads=12, num_key_value_heads=2, max_position_embeddings=512,
                      tie_word_embeddings=False)
    torch.manual_seed(0)
    model = Qwen2ForCausalLM(cfg)
    with torch.no_grad():
        for p in model.parameters():
            p.normal_(0.0, 0.02)
        for m in model.modules():                    # norms at their usual scale
            if hasattr(m, "variance_epsilon"):
                m.weight.fill_(1.0)
    model = model.half().cuda().eval()
    quantize_model_int4(model)
    fuse_attention_qkv(model)
    fuse_mlp_gate_up(model)
    return model


def decode_plain(decoder: PagedDecoder, prompt: torch.Tensor, new: int) -> list[int]:
    """Greedy decoding, one token a pass."""
    logits = decoder.forward(prompt)
    decoder.accept(range(prompt.shape[0]))
    out = [int(logits[-1].argmax())]
    while len(out) < new:
        logits = decoder.forward(torch.tensor(out[-1:], device="cuda"))
        decoder.accept([0])
        out.append(int(logits[-1].argmax()))
    return out


def draft_tree(guess: list[int], seed: int, vocab: int):
    """A tree of drafted tokens below the last accepted one: the guess as the
    main branch, some of its tokens replaced, and a random side branch of two
    at each of its first tokens.  Returns tokens, parents and depths; entry 0
    is the accepted token itself (to be filled in)."""
    g = torch.Generator().manual_seed(seed)

    def token():
        return int(torch.randint(0, vocab, (1,), generator=g))

    tokens, parents, depth = [0], [-1], [0]
    last = 0
    for i, t in enumerate(guess):
        if i < 3:
            tokens += [token(), token()]
            parents += [last, len(tokens) - 2]
            depth += [depth[last] + 1, depth[last] + 2]
        wrong = float(torch.rand(1, generator=g)) < 0.2
        tokens.append(token() if wrong else t)
        parents.append(last)
        depth.append(depth[last] + 1)
        last = len(tokens) - 1
    return tokens, parents, depth


def decode_tree(decoder: PagedDecoder, prompt: torch.Tensor, new: int, guesses: list[int], span: int = 6):
    """Greedy decoding with drafted trees: each pass verifies a tree and
    accepts the longest path on which every token is the model's own choice.
    Returns the tokens and the number of passes."""
    vocab = decoder.model.config.vocab_size
    logits = decoder.forward(prompt)
    decoder.accept(range(prompt.shape[0]))
    out, passes = [int(logits[-1].argmax())], 1
    while len(out) < new:
        tokens, parents, depth = draft_tree(guesses[len(out):len(out) + span], len(out), vocab)
        tokens[0] = out[-1]
        logits = decoder.forward(torch.tensor(tokens, device="cuda"), torch.tensor(depth, device="cuda"),
                                 tree_mask_from_parents(parents).cuda())
        passes += 1
        choice = logits.argmax(-1).tolist()
        path, at = [0], 0
        while True:
            out.append(choice[at])
            following = [i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == choice[at]]
            if not following or len(out) >= new:
                break
            at = following[0]
            path.append(at)
        decoder.accept(path)
    return out, passes


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--bits", type=int, default=8, choices=(8, 4), help="bits of a cached element")
    ap.add_argument("--new", type=int, default=48, help="tokens to decode")
    ap.add_argument("--layers", type=int, default=4)
    args = ap.parse_args()
    model = build_model(args.layers)
    prompt = torch.randint(0, model.config.vocab_size, (37,), generator=torch.Generator().manual_seed(1)).cuda()
    runs = {}
    for name in ("plain", "tree"):
        decoder = PagedDecoder(model, bits=args.bits, max_positions=prompt.shape[0] + args.new + 64)   # and a tree
        torch.cuda.synchronize()
        t = time.perf_counter()
        if name == "plain":
            runs[name], passes = decode_plain(decoder, prompt, args.new), args.new
        else:
            runs[name], passes = decode_tree(decoder, prompt, args.new, runs["plain"])
        torch.cuda.synchronize()
        print(f"{name}: {len(runs[name])} tokens in {passes} passes, {1e3 * (time.perf_counter() - t):.1f} ms")
    k, _ = decoder.cached(0)
    print(f"cache: {decoder.length} positions, {sum(c.num_bytes() for c in decoder.caches) >> 10} KB in all, "
          f"layer 0 keys back as {tuple(k.shape)} {k.dtype}")
    print("the same tokens" if runs["plain"] == runs["tree"] else "DIFFERENT tokens")


if __name__ == "__main__":
    main()
