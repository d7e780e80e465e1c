"""The attention-side operators between the fused q/k/v projection and o_proj, as they are measured.

Four operators, on the head layouts of the decoder models this package serves:

  rotary   rotary positions applied to query and key heads (columns of the fused q/k/v output)
  cache    quantising keys and values into a paged 8- or 4-bit cache as they are written, with the
           rotation of q and k in the same call, then reading the written rows back
  read     reading cached rows back as 16-bit values
  attend   attention of one token, or of a tree of drafted tokens, per request over the paged cache

A cached row is one token of one key/value head: integer codes (two to a byte at 4 bits, the even
element in the low nibble, offset by 8) times a bfloat16 scale for each group of elements (the whole
head at 8 bits, 64 elements at 4 bits).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
GROUP4 = 64


# ------------------------------------------------------------------ the cases
def _rotary(name, tokens, heads, head_dim, rotary_dim, layout, dtype, scaling, where, inverse=False):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "head_dim": head_dim,
            "rotary_dim": rotary_dim, "layout": layout, "dtype": dtype, "scaling": scaling, "where": where,
            "inverse": inverse}


def _cache(name, tokens, q_heads, kv_heads, head_dim, rotary_dim, layout, dtype, bits, page, where, skipped=0):
    return {"name": name, "op": "cache", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "layout": layout, "dtype": dtype, "bits": bits,
            "page": page, "where": where, "skipped": skipped, "scaling": "none"}


def _read(name, batch, context, kv_heads, head_dim, dtype, bits, page):
    return {"name": name, "op": "read", "batch": batch, "context": context, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "bits": bits, "page": page}


def _attend(name, batch, context, tree, q_heads, kv_heads, head_dim, dtype, bits, page, mask, lse=False):
    return {"name": name, "op": "attend", "batch": batch, "context": context, "tree": tree, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "bits": bits, "page": page, "mask": mask,
            "lse": lse}


def listed():
    return [
        # one decode step of one request, the 1.5B layer's 12 + 2 heads: latency only
        _rotary("rotary: one token", 1, 14, 128, 128, "half", "f16", "none", "decode"),
        # a ragged chunk, pairs side by side, a part of each small head turned, turned back (the gradient's direction)
        _rotary("rotary: part of a head, back", 1777, 20, 64, 32, "interleaved", "bf16", "linear", "prompt", True),
        # a long prompt of the 7B layer (28 + 4 heads) with frequencies stretched for long contexts
        _rotary("rotary: 16k prompt, long", 16384, 32, 128, 128, "half", "bf16", "llama3", "prompt"),
        # one decode step of 64 requests: every token goes to a page of its own
        _cache("cache: 64 requests, 8 bits", 64, 12, 2, 128, 128, "half", "f16", 8, 16, "decode"),
        # a chunk of prompts packed together, padding rows among them, four bits
        _cache("cache: 2501 tokens, 4 bits", 2501, 28, 4, 128, 128, "half", "f16", 4, 32, "prompt", 61),
        # a whole prompt of the wide layer (32 + 8 heads)
        _cache("cache: 8k prompt, 8 bits", 8192, 32, 8, 128, 128, "half", "bf16", 8, 64, "prompt"),
        # a cached prefix of one request, read for a dense prefill
        _read("read: prefix of 1000, 8 bits", 1, 1000, 2, 128, "f16", 8, 16),
        # 32 requests' caches, four bits
        _read("read: 32 requests, 4 bits", 32, 4001, 8, 128, "bf16", 4, 64),
        # the first tokens of a chat: one request, one token, a short cache; latency only
        _attend("attend: one token, short", 1, 97, 1, 12, 2, 128, "f16", 8, 16, "causal"),
        # a decode step of a full batch with ragged lengths
        _attend("attend: 64 requests, 8k", 64, 8192, 1, 32, 8, 128, "bf16", 8, 64, "causal"),
        # one token over a long document, four bits
        _attend("attend: 130k context, 4 bits", 1, 130001, 1, 28, 4, 128, "f16", 4, 32, "causal"),
        # trees of up to 64 drafted tokens for 16 requests: the verification step of speculative decoding
        _attend("attend: trees of 64", 16, 8197, 64, 28, 4, 128, "f16", 8, 16, "tree", True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "read", "attend", "attend"])
    q_heads, kv_heads, head_dim = rng.choice([(12, 2, 128), (28, 4, 128), (32, 8, 128), (16, 16, 64), (20, 4, 64),
                                              (8, 1, 128), (16, 4, 256), (5, 5, 64)])
    dtype = rng.choice(["f16", "bf16"])
    bits = rng.choice([8, 8, 4])
    page = rng.choice([16, 32, 64, 128])
    rotary_dim = head_dim if rng.random() < 0.6 else rng.choice([head_dim // 2, head_dim // 4])
    layout = rng.choice(["half", "interleaved"])
    if op == "rotary":
        most = min(16384, 16384 * 32 * 128 // ((q_heads + kv_heads) * head_dim))
        c = _rotary("", _spread(rng, 1, most), q_heads + kv_heads, head_dim, rotary_dim, layout, dtype,
                    rng.choice(["none", "linear", "llama3", "yarn"]), rng.choice(["decode", "prompt"]),
                    rng.random() < 0.3)
    elif op == "cache":
        most = min(8192, 8192 * 48 * 128 // ((q_heads + 2 * kv_heads) * head_dim))
        tokens = _spread(rng, 1, most)
        c = _cache("", tokens, q_heads, kv_heads, head_dim, rotary_dim, layout, dtype, bits, page,
                   rng.choice(["decode", "prompt"]) if tokens <= 512 else "prompt", tokens // 40)
    elif op == "read":
        batch = _spread(rng, 1, 48)
        most = 32 * 4001 * 8 * 128 // (batch * kv_heads * head_dim)
        c = _read("", batch, _spread(rng, 1, min(most, 60000)), kv_heads, head_dim, dtype, bits, page)
    else:
        tree = 1 if rng.random() < 0.5 else _spread(rng, 2, 64)
        batch = _spread(rng, 1, 64)
        # no more rows read than the fullest listed batch, no more products than the listed trees
        rows = 64 * 8192 * 8 * 128 // (2 * batch * kv_heads * head_dim)
        work = 16 * 8197 * 64 * 28 * 128 // (2 * batch * tree * q_heads * head_dim)
        most = max(tree, min(rows, 100000 if tree == 1 else work))
        c = _attend("", batch, max(tree, _spread(rng, 1, most)), tree, q_heads, kv_heads, head_dim, dtype, bits,
                    page, "causal" if tree == 1 or rng.random() < 0.25 else "tree", rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------- lengths, by the case alone
def _kv_lens(case):
    """Requests' lengths, from the full context down to three eighths of it."""
    n, b = case["context"], case["batch"]
    least = case.get("tree", 1)
    return [max(least, n - (5 * n * i) // (8 * b) - (i % 3)) for i in range(b)]


def _tree_lens(case):
    """Drafted tokens of each request: the full tree for the first, fewer for others."""
    t, b = case["tree"], case["batch"]
    return [max(1, t - (t * ((5 * i) % b)) // (2 * b)) for i in range(b)]


def _frequencies(case):
    """Radians per position of each pair, float64 on the CPU, and the factor on cos and sin."""
    r, base, max_pos = case["rotary_dim"], 1.0e6, 32768
    i = torch.arange(r // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":          # positions squeezed by 4
        return f / 4.0, 1.0
    if case["scaling"] == "llama3":          # long wavelengths stretched by 8, a smooth step between
        wave, old = 2 * math.pi / f, 8192.0
        smooth = ((old / wave - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return (1 - smooth) * f / 8.0 + smooth * f, 1.0
    if case["scaling"] == "yarn":            # by turns made over the trained length, and sharper scores
        factor, old = 4.0, max_pos / 4.0
        dim_of = lambda turns: r * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), r - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


MAX_POSITIONS = 32768


def _table(case):
    """cos and sin of every position, float32 [positions, rotary_dim / 2, 2]: the plan a program keeps."""
    f, factor = _frequencies(case)
    a = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * f.cuda()
    return (torch.stack([a.cos(), a.sin()], dim=-1) * factor).float()


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _heads(g, tokens, heads, head_dim, dtype):
    """Projected heads: normal values, a few channels several times larger than the others, as keys have them."""
    x = torch.randn(tokens, heads, head_dim, generator=g, device="cuda")
    gain = torch.exp(0.5 * torch.randn(heads, head_dim, generator=g, device="cuda"))
    return (x * gain).to(dtype)


def _positions(case, g):
    t = case["tokens"]
    if case["where"] == "decode":
        return torch.randint(0, MAX_POSITIONS, (t,), generator=g, device="cuda")
    return torch.arange(t, device="cuda") + int(torch.randint(0, MAX_POSITIONS - t + 1, (1,), generator=g,
                                                              device="cuda"))


def _groups(case):
    """Scales of a cached row."""
    return 1 if case["bits"] == 8 else max(1, case["head_dim"] // GROUP4)


def _pool(case, pages, g, std):
    """Codes and scales of a pool whose rows hold quantised normal values."""
    h, p, d, n = case["kv_heads"], case["page"], case["head_dim"], _groups(case)
    codes = torch.empty(pages, h, p, d if case["bits"] == 8 else d // 2,
                        dtype=torch.int8 if case["bits"] == 8 else torch.uint8, device="cuda")
    scales = torch.empty(pages, h, p, n, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 26) // (h * p * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = std * torch.randn(b - a, h, p, d, generator=g, device="cuda")
        codes[a:b], scales[a:b] = _quantise(x, case["bits"])
    return codes, scales


def _paged(case, lens, g):
    """A pool with some room to spare and a page table whose pages lie in no order."""
    page, width = case["page"], -(-max(lens) // case["page"])
    counts = [-(-n // page) for n in lens]
    order = torch.randperm(sum(counts) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(counts) + 3


def _inputs(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        # query and key heads are the first columns of the fused projection's output, values behind them
        qkv = _heads(g, case["tokens"], case["heads"] + 2, case["head_dim"], dtype)
        return {"x": qkv[:, :case["heads"]], "positions": _positions(case, g), "table": _table(case)}
    if case["op"] == "cache":
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        qkv = _heads(g, t, hq + 2 * hk, case["head_dim"], dtype)
        page = case["page"]
        pages = -(-t // page) + 4 if case["where"] == "prompt" else t + 4
        order = torch.randperm(pages, generator=g, device="cuda")
        if case["where"] == "prompt":
            i = torch.arange(t, device="cuda")
            slots = order[i // page] * page + i % page
        else:
            slots = order[:t] * page + torch.randint(0, page, (t,), generator=g, device="cuda")
        if case["skipped"]:
            slots[torch.randperm(t, generator=g, device="cuda")[:case["skipped"]]] = -1
        s = {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "v": qkv[:, hq + hk:], "slots": slots,
             "positions": _positions(case, g), "table": _table(case)}
        s["k_codes"], s["k_scales"] = _pool(case, pages, g, 1.0)
        s["v_codes"], s["v_scales"] = _pool(case, pages, g, 1.0)
        return s
    lens = _kv_lens(case)
    table, pages = _paged(case, lens, g)
    s = {"page_table": table, "kv_lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    s["k_codes"], s["k_scales"] = _pool(case, pages, g, 1.0)
    s["v_codes"], s["v_scales"] = _pool(case, pages, g, 0.7)
    if case["op"] == "read":
        page = case["page"]
        rows = [torch.arange(n, device="cuda") for n in lens]
        s["slots"] = torch.cat([table[b, r // page].long() * page + r % page for b, r in enumerate(rows)])
        return s
    trees = _tree_lens(case)
    total = sum(trees)
    # sharper than unit scores, as trained heads are
    s["q"] = (1.5 * torch.randn(total, case["q_heads"], case["head_dim"], generator=g, device="cuda")).to(dtype)
    s["cu_q"] = torch.tensor([sum(trees[:i]) for i in range(len(trees) + 1)], dtype=torch.int32, device="cuda")
    s["mask"] = None
    if case["mask"] == "tree":
        # each drafted token has a parent among the earlier ones and sees its ancestors and itself
        t, b = case["tree"], case["batch"]
        sees = torch.zeros(b, t, t, dtype=torch.bool, device="cuda")
        parents = (torch.rand(b, t, generator=g, device="cuda") * torch.arange(t, device="cuda")).long()
        every = torch.arange(b, device="cuda")
        sees[:, 0, 0] = True
        for i in range(1, t):
            sees[:, i] = sees[every, parents[:, i]]
            sees[:, i, i] = True
        words = -(-t // 64)
        bits = torch.zeros(b, t, words * 64, dtype=torch.int64, device="cuda")
        bits[:, :, :t] = sees
        packed = (bits.reshape(b, t, words, 64) << torch.arange(64, device="cuda")).sum(-1)
        s["mask"] = torch.cat([packed[i, :n] for i, n in enumerate(trees)])
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        # what a serving program keeps from step to step: the handles of the table of angles and of the cache
        ops = _package()
        if "table" in state:
            state["rotary"] = ops["rotary"].RotaryTable(state["table"], layout=case["layout"])
        if "k_codes" in state:
            state["cache"] = ops["kv_cache"].QuantizedKVCache(
                *(state[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")))
    return state


# ------------------------------------------------------------------ plain forms
def _rotate(x, positions, table, case, sign=1.0):
    r = case["rotary_dim"]
    c, s = table[positions, :, 0].unsqueeze(1), sign * table[positions, :, 1].unsqueeze(1)
    x = x.float()
    y = x.clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def _quantise(x, bits):
    """Codes and scales of rows x[..., head_dim] in float32."""
    top, d = (127.0, x.shape[-1]) if bits == 8 else (7.0, min(GROUP4, x.shape[-1]))
    x = x.unflatten(-1, (-1, d))
    scales = (x.abs().amax(-1) * (1.0 / top)).to(torch.bfloat16)
    s = scales.float().unsqueeze(-1)
    q = torch.where(s > 0, torch.round(x / s), 0.0).clamp(-top, top).flatten(-2)
    if bits == 8:
        return q.to(torch.int8), scales
    q = (q + 8).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), scales


def _values(codes, scales, bits):
    """What codes and scales stand for, in float32."""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    q = codes.float() - (8.0 if bits == 4 else 0.0)
    return (q.unflatten(-1, (scales.shape[-1], -1)) * scales.float().unsqueeze(-1)).flatten(-2)


def _rows(codes, scales, slots, case):
    """The cached rows at the given slots, [tokens, heads, head_dim] float32; zeros where a slot is -1."""
    page, at = slots.clamp(min=0) // case["page"], slots.clamp(min=0) % case["page"]
    rows = _values(codes[page, :, at], scales[page, :, at], case["bits"])
    return torch.where((slots >= 0)[:, None, None], rows, 0.0)


def _attend_plain(s):
    case = s["case"]
    q, table, lens, cu = s["q"], s["page_table"].long(), s["kv_lens"].long(), s["cu_q"].long()
    b, t, hk, d = table.shape[0], case["tree"], case["kv_heads"], case["head_dim"]
    g, n = case["q_heads"] // hk, table.shape[1] * case["page"]
    k = _values(s["k_codes"][table], s["k_scales"][table], case["bits"]).transpose(1, 2).reshape(b, hk, n, d)
    v = _values(s["v_codes"][table], s["v_scales"][table], case["bits"]).transpose(1, 2).reshape(b, hk, n, d)
    count = cu[1:] - cu[:-1]
    row = torch.arange(t, device="cuda")
    at = torch.minimum(cu[:-1, None] + row, cu[1:, None] - 1)            # padded rows repeat the last one
    qs = q[at].float().reshape(b, t, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * t, d)
    key = torch.arange(n, device="cuda")
    draft = key[None] - (lens - count)[:, None]                          # [b, n]: which drafted token a key is
    if s["mask"] is None:
        sees = draft[:, None] <= row[:, None]
    else:
        bits = s["mask"][at]                                             # [b, t, words]
        bits = ((bits.unsqueeze(-1) >> torch.arange(64, device="cuda")) & 1).flatten(2).bool()
        sees = bits.gather(2, draft.clamp(0, bits.shape[2] - 1)[:, None].expand(b, t, n)) | (draft < 0)[:, None]
    sees = (sees & (key[None] < lens[:, None])[:, None])[:, None, None]  # [b, 1, 1, t, n]
    scores = (qs @ k.transpose(2, 3)).div_(math.sqrt(d)).unflatten(2, (g, t)).masked_fill_(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (g, t)) / total
    real = row[None] < count[:, None]
    out = out.permute(0, 3, 1, 2, 4).reshape(b, t, hk * g, d)[real].to(q.dtype)
    if not case["lse"]:
        return [out]
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, t, hk * g)[real]
    return [out, lse]


def _run_plain(s):
    case = s["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        return [_rotate(s["x"], s["positions"], s["table"], case, -1.0 if case["inverse"] else 1.0).to(dtype)]
    if case["op"] == "cache":
        q = _rotate(s["q"], s["positions"], s["table"], case).to(dtype)
        kept = torch.nonzero(s["slots"] >= 0).squeeze(1)
        slots = s["slots"][kept]
        page, at = slots // case["page"], slots % case["page"]
        k = _rotate(s["k"], s["positions"], s["table"], case)[kept]
        s["k_codes"][page, :, at], s["k_scales"][page, :, at] = _quantise(k, case["bits"])
        s["v_codes"][page, :, at], s["v_scales"][page, :, at] = _quantise(s["v"].float()[kept], case["bits"])
    if case["op"] == "attend":
        return _attend_plain(s)
    rows = [_rows(s[n + "_codes"], s[n + "_scales"], s["slots"], case).to(dtype) for n in "kv"]
    return [q] + rows if case["op"] == "cache" else rows


# ------------------------------------------------------------- this package's
_modules = {}


def _package():
    """The package's modules, from the folder that it is imported from everywhere."""
    if not _modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "llm-inference-optimizer_b200"))
        from qlinear.kernels import kv_cache, rotary, tree_attention
        _modules.update(rotary=rotary, kv_cache=kv_cache, tree_attention=tree_attention)
    return _modules


def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    dtype = DTYPES[case["dtype"]]
    if op == "rotary":
        return [_modules["rotary"].apply_rotary(s["x"], s["positions"], s["rotary"], inverse=case["inverse"])]
    if op == "attend":
        # every request has up to `tree` tokens; without a mask each sees what came before it
        got = _modules["tree_attention"].tree_attention(
            s["q"], s["cache"], s["page_table"], s["kv_lens"], cu_q=None if case["tree"] == 1 else s["cu_q"],
            max_q=case["tree"], mask=s["mask"], return_lse=case["lse"])
        return list(got) if case["lse"] else [got]
    cache = _modules["kv_cache"]
    q = []
    if op == "cache":
        q = [cache.append_kv(s["cache"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"],
                             rotary=s["rotary"])]
    return q + list(cache.read_kv(s["cache"], s["slots"], dtype=dtype))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------- the definitions, 64 bits
def _exact_rotated(x, positions, case, back=False):
    f, factor = _frequencies(case)
    angle = positions.double()[:, None, None] * f.cuda()
    if back:
        angle = -angle
    turn = torch.polar(torch.full_like(angle, factor), angle)            # factor * exp(i * angle)
    x, r = x.double(), case["rotary_dim"]
    pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" \
        else x[..., :r].unflatten(-1, (r // 2, 2))
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = pairs.transpose(-1, -2) if case["layout"] == "half" else pairs
    return torch.cat([turned.flatten(-2), x[..., r:]], dim=-1)


def _exact_stored(x, case):
    """What rows x stand for once they are cached."""
    top = 127.0 if case["bits"] == 8 else 7.0
    parts = []
    for group in x.split(x.shape[-1] if case["bits"] == 8 else GROUP4, dim=-1):
        step = (group.abs().max(-1, keepdim=True).values / top).to(torch.bfloat16).double()
        parts.append(torch.where(step > 0, (group / step).round().clamp(-top, top) * step, torch.zeros_like(group)))
    return torch.cat(parts, dim=-1)


def _exact_rows(codes, scales, case):
    if case["bits"] == 8:
        return codes.double() * scales.double()
    q = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device="cuda")
    q[..., 0::2], q[..., 1::2] = (codes & 15).double() - 8, (codes >> 4).double() - 8
    return q * scales.double().repeat_interleave(q.shape[-1] // scales.shape[-1], dim=-1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        return [_exact_rotated(s["x"], s["positions"], case, case["inverse"])]
    if case["op"] == "cache":
        kept = (s["slots"] >= 0)[:, None, None]
        k = _exact_stored(_exact_rotated(s["k"], s["positions"], case), case)
        v = _exact_stored(s["v"].double(), case)
        return [_exact_rotated(s["q"], s["positions"], case), torch.where(kept, k, 0.0), torch.where(kept, v, 0.0)]
    lens = _kv_lens(case)
    whole = []
    outs, lses, first = [], [], 0
    trees = _tree_lens(case) if case["op"] == "attend" else [0] * len(lens)
    for b, n in enumerate(lens):
        pages = s["page_table"][b, : -(-n // case["page"])].long()
        k, v = (_exact_rows(s[x + "_codes"][pages], s[x + "_scales"][pages], case).transpose(1, 2).flatten(0, 1)[:n]
                for x in "kv")                                           # [n, heads, head_dim]
        if case["op"] == "read":
            whole.append((k, v))
            continue
        t, hk = trees[b], case["kv_heads"]
        q = s["q"][first:first + t].double().unflatten(1, (hk, -1))      # [t, heads, group, head_dim]
        scores = torch.einsum("thgd,nhd->hgtn", q, k) / math.sqrt(case["head_dim"])
        sees = torch.ones(t, n, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            sees[:, n - t:] = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
        else:
            for j in range(t):
                sees[:, n - t + j] = (s["mask"][first:first + t, j // 64] >> (j % 64)) & 1 == 1
        scores = scores.masked_fill(~sees, -math.inf)
        outs.append(torch.einsum("hgtn,nhd->thgd", torch.softmax(scores, -1), v).flatten(1, 2))
        lses.append(torch.logsumexp(scores, -1).permute(2, 0, 1).flatten(1))
        first += t
    if case["op"] == "read":
        return [torch.cat([w[i] for w in whole]) for i in (0, 1)]
    return [torch.cat(outs), torch.cat(lses)] if case["lse"] else [torch.cat(outs)]


# --------------------------------------------------- what a pass cannot do without
def work(case):
    d = case["head_dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"]
        turned = n * case["rotary_dim"]
        return {"bytes": 4.0 * n * d + case["tokens"] * (8.0 + 4.0 * case["rotary_dim"]), "flops": 3.0 * turned}
    cached = 2.0 * (d * case["bits"] // 8 + 2 * _groups(case))           # one token's key and value of one head
    if case["op"] == "cache":
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        kept = t - case["skipped"]
        rotated = t * (2.0 * 2 * hq * d + 8 + 8 + 4.0 * case["rotary_dim"])
        written = kept * hk * (2.0 * 2 * d + cached)
        read = kept * hk * cached + t * hk * 2.0 * 2 * d + 8.0 * t
        return {"bytes": rotated + written + read,
                "flops": 3.0 * t * (hq + hk) * case["rotary_dim"] + kept * hk * 2.0 * 4 * d}
    lens = _kv_lens(case)
    rows = float(sum(lens)) * case["kv_heads"]
    if case["op"] == "read":
        return {"bytes": rows * (cached + 2.0 * 2 * d) + 8.0 * sum(lens), "flops": rows * 2 * d}
    trees = _tree_lens(case)
    hq = case["q_heads"]
    queries = 2.0 * 2 * sum(trees) * hq * d + (4.0 * sum(trees) * hq if case["lse"] else 0.0)
    tables = 4.0 * sum(-(-n // case["page"]) for n in lens) + 8.0 * len(lens)
    products = sum(t * (n - t) + t * (t + 1) / 2 for t, n in zip(trees, lens))
    return {"bytes": rows * cached + queries + tables, "flops": 4.0 * d * hq * products}
