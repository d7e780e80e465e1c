"""The operators of a serving step around the layers, as they are measured.

Three operators, on the head layouts and vocabularies of the decoder models this package serves:

  plan    a step's page tables, slots and positions from request lengths: every request is cut to the tokens that
          it keeps, its spare pages go back to the stack of free pages, and it grows by its new tokens
  sample  drawing a token from each row of logits, with temperature, top-k, top-p and min-p, by given random numbers
  shared  attention of one token, or of a tree of drafted tokens, per request over the quantised paged cache, where
          groups of requests share a long prefix that is read once for all of them

A cached row is one token of one key/value head: integer codes (two to a byte at 4 bits, the even
element in the low nibble, offset by 8) times a bfloat16 scale for each group of elements (the whole
head at 8 bits, 64 elements at 4 bits).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GROUP4 = 64


# ------------------------------------------------------------------ the cases
def _plan(name, batch, context, new, page, kind):
    return {"name": name, "op": "plan", "batch": batch, "context": context, "new": new, "page": page, "kind": kind}


def _sample(name, rows, vocab, dtype, filters, hidden=False):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters,
            "hidden": hidden}


def _shared(name, batch, groups, prefix, context, tree, q_heads, kv_heads, head_dim, dtype, bits, page, mask, lse=False):
    return {"name": name, "op": "shared", "batch": batch, "groups": groups, "prefix": prefix, "context": context,
            "tree": tree, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "bits": bits,
            "page": page, "mask": mask, "lse": lse}


def listed():
    return [
        # one decode step of one request: latency only
        _plan("plan: one request", 1, 97, 1, 16, "decode"),
        # speculative decoding of a batch: what was refused is cut off, the next trees are planned
        _plan("plan: 64 trees", 64, 8197, 64, 16, "tree"),
        # a large batch's decode step, a chunk of a prompt for some of its requests
        _plan("plan: 1000 requests", 1000, 3001, 40, 32, "mixed"),
        # packed prompts: all pages are new
        _plan("plan: prompts, 131k tokens", 23, 0, 11001, 64, "prompt"),
        # one chat's next token, the usual settings; latency only
        _sample("sample: one row, top-k top-p", 1, 151936, "f16", "k50 p95"),
        # a batch of constrained requests with a small vocabulary: some tokens hidden, each row its own settings
        _sample("sample: 37 rows, all filters", 37, 32003, "f32", "rows", True),
        # a batch's step, the smallest probabilities cut off
        _sample("sample: 64 rows, top-p min-p", 64, 128256, "bf16", "p90 m05"),
        # samples of a full batch from the whole distribution
        _sample("sample: 256 rows, whole", 256, 151936, "f16", "none"),
        # a few answers to one question: a short shared prompt; latency only
        _shared("shared: 4 answers, short", 4, 1, 500, 60, 1, 12, 2, 128, "f16", 8, 16, "causal"),
        # a full batch behind one system prompt
        _shared("shared: 64 behind 8k", 64, 1, 8192, 512, 1, 32, 8, 128, "bf16", 8, 64, "causal"),
        # three system prompts, four bits, trees of drafted tokens
        _shared("shared: 3 prompts, trees", 48, 3, 12001, 701, 8, 28, 4, 128, "f16", 4, 32, "tree", True),
        # many questions about one long document
        _shared("shared: 16 behind 100k", 16, 1, 100003, 300, 1, 28, 4, 128, "bf16", 8, 16, "causal"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "sample", "sample", "shared", "shared"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        kind = rng.choice(["decode", "tree", "mixed", "prompt"])
        batch = _spread(rng, 1, 2000 if kind != "prompt" else 100)
        new = {"decode": 1, "tree": _spread(rng, 2, 64), "mixed": _spread(rng, 2, 100),
               "prompt": _spread(rng, 1, min(60000, 200000 // batch))}[kind]
        c = _plan("", batch, 0 if kind == "prompt" else _spread(rng, 64, min(16000, 8000000 // batch)), new, page, kind)
    elif op == "sample":
        vocab = rng.choice([151936, 128256, 8192, _spread(rng, 50, 160000)])
        dtype = rng.choice(["f16", "bf16", "f32"])
        rows = _spread(rng, 1, min(512, 256 * 151936 // vocab // (2 if dtype == "f32" else 1)))
        c = _sample("", rows, vocab, dtype, rng.choice(["k50 p95", "rows", "p90 m05", "none", "k8", "p99"]), rng.random() < 0.3)
    else:
        q_heads, kv_heads, head_dim = rng.choice([(12, 2, 128), (28, 4, 128), (32, 8, 128), (16, 16, 64), (20, 4, 64),
                                                  (8, 1, 128), (16, 4, 256), (5, 5, 64)])
        tree = 1 if rng.random() < 0.6 else _spread(rng, 2, 16)
        groups = 1 if rng.random() < 0.6 else _spread(rng, 2, 8)
        batch = _spread(rng, max(2, groups), 64)
        # no more products than the listed trees, no more rows than the long document and the full batch
        rows = 48 * 8 * 12001 * 28 * 128 // (batch * tree * q_heads * head_dim)
        most = min(100000, rows, 100003 * 4 * 128 // (groups * kv_heads * head_dim))
        mine = min(2000, 64 * 8 * 512 * 128 * 2 // (batch * kv_heads * head_dim))
        c = _shared("", batch, groups, _spread(rng, 1, max(2, most)), max(tree, _spread(rng, tree, max(tree + 1, mine))), tree,
                    q_heads, kv_heads, head_dim, rng.choice(["f16", "bf16"]), rng.choice([8, 8, 4]), page,
                    "causal" if tree == 1 or rng.random() < 0.25 else "tree", rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------- lengths, by the case alone
def _kv_lens(case):
    """Requests' lengths, from the full context down to three eighths of it."""
    n, b = case["context"], case["batch"]
    least = case.get("tree", 0)
    return [max(least, n - (5 * n * i) // (8 * b) - (i % 3)) for i in range(b)]


def _tree_lens(case):
    """Drafted tokens of each request: the full tree for the first, fewer for others."""
    t, b = case["tree"], case["batch"]
    return [max(1, t - (t * ((5 * i) % b)) // (2 * b)) for i in range(b)]


def _groups_of(case):
    """First request of each group, and the end: later groups are larger."""
    b, g = case["batch"], case["groups"]
    return [(b * i * (i + g)) // (2 * g * g) for i in range(g + 1)]


def _prefix_lens(case):
    """The groups' prefixes, the first the longest."""
    n, g = case["prefix"], case["groups"]
    return [max(1, n - (n * i) // (2 * g)) for i in range(g)]


def _news(case):
    """Each request's cached tokens before the step, those that it keeps, and its new ones."""
    b, n, kind = case["batch"], case["new"], case["kind"]
    have = _kv_lens(case)
    if kind == "prompt":                     # new requests, of a half to the whole of the longest
        return [0] * b, [0] * b, [max(1, n - (n * i) // (2 * b)) for i in range(b)]
    if kind == "tree":                       # a few drafted tokens are kept, the next tree is as large or smaller
        keep = [max(0, h - (7 * i) % n) for i, h in enumerate(have)]
        return have, keep, [max(1, n - (3 * i) % n) for i in range(b)]
    if kind == "mixed":                      # a token each, a chunk of a prompt for one in eight, nothing for some; some end
        keep = [0 if i % 50 == 49 else h for i, h in enumerate(have)]
        return have, keep, [n if i % 8 == 3 else 0 if i % 10 == 9 else 1 for i in range(b)]
    return have, [max(0, h - 1) for h in have], [n] * b


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _groups4(case):
    """Scales of a cached row."""
    return 1 if case["bits"] == 8 else max(1, case["head_dim"] // GROUP4)


def _pool(case, pages, g, std):
    """Codes and scales of a pool whose rows hold quantised normal values."""
    h, p, d, n = case["kv_heads"], case["page"], case["head_dim"], _groups4(case)
    top = 127.0 if case["bits"] == 8 else 7.0
    codes = torch.empty(pages, h, p, d if case["bits"] == 8 else d // 2,
                        dtype=torch.int8 if case["bits"] == 8 else torch.uint8, device="cuda")
    scales = torch.empty(pages, h, p, n, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 26) // (h * p * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = (std * torch.randn(b - a, h, p, d, generator=g, device="cuda")).unflatten(-1, (n, -1))
        scales[a:b] = (x.abs().amax(-1) * (1.0 / top)).to(torch.bfloat16)
        q = torch.round(x / scales[a:b].float().unsqueeze(-1)).clamp(-top, top).flatten(-2)
        if case["bits"] == 4:
            q = (q + 8).to(torch.uint8)
            q = q[..., 0::2] | (q[..., 1::2] << 4)
        codes[a:b] = q.to(codes.dtype)
    return codes, scales


def _tables(lens, page, g, spare):
    """Page tables of several sets of lengths in one pool, whose pages lie in no order, and the pages that are left."""
    counts = [[-(-n // page) for n in some] for some in lens]
    total = sum(map(sum, counts))
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)
    tables, at = [], 0
    for some in counts:
        table = torch.zeros(len(some), max(1, max(some)), dtype=torch.int32, device="cuda")
        for i, n in enumerate(some):
            table[i, :n] = order[at:at + n]
            at += n
        tables.append(table)
    return tables, order[at:]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _plan_inputs(case, g):
    page = case["page"]
    have, keep, new = _news(case)
    # the requests' pages before the step, room for what they may grow by, and a pool with some pages to spare
    want = [max(h, k + n) for h, k, n in zip(have, keep, new)]
    more = sum(-(-w // page) for w in want) + 5
    held = sum(-(-h // page) for h in have)
    (table,), free = _tables([have], page, g, more - held)
    width = -(-(max(want) + case["new"]) // page) + 2
    whole = torch.zeros(len(have), width, dtype=torch.int32, device="cuda")
    whole[:, :table.shape[1]] = table
    stack = torch.zeros(more, dtype=torch.int32, device="cuda")
    stack[:free.shape[0]] = free
    return {"page_table": whole, "lens": _ints(have), "free": stack, "count": _ints([free.shape[0]]), "keep": _ints(keep),
            "new": _ints(new), "max_tokens": sum(new) + (-sum(new)) % 8}


def _sample_inputs(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # spread logits, a few tokens well above the others
    x = 2.2 * torch.randn(rows, vocab, generator=g, device="cuda")
    lift = 12.0 * torch.rand(rows, 24, generator=g, device="cuda") ** 2
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 24), generator=g, device="cuda"), lift)
    if case["hidden"]:
        x[torch.rand(rows, vocab, generator=g, device="cuda") < 0.6] = -math.inf
    s = {"logits": x.to(DTYPES[case["dtype"]]), "uniform": torch.rand(rows, generator=g, device="cuda")}
    f = case["filters"]
    s |= {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if f == "rows":                          # each request its own settings, one in nine greedy, some filters off
        i = torch.arange(rows, device="cuda")
        s["temperature"] = torch.where(i % 9 == 4, 0.0, 0.5 + torch.rand(rows, generator=g, device="cuda"))
        s["top_k"] = torch.where(i % 4 == 1, 0, torch.randint(1, 200, (rows,), generator=g, device="cuda")).to(torch.int32)
        s["top_p"] = torch.where(i % 5 == 2, 1.0, 0.5 + 0.5 * torch.rand(rows, generator=g, device="cuda"))
        s["min_p"] = torch.where(i % 3 == 0, 0.0, 0.1 * torch.rand(rows, generator=g, device="cuda"))
    elif f == "k50 p95":
        s |= {"temperature": 0.7, "top_k": 50, "top_p": 0.95}
    elif f == "k8":
        s |= {"top_k": 8}
    elif f == "p90 m05":
        s |= {"temperature": 1.1, "top_p": 0.9, "min_p": 0.05}
    elif f == "p99":
        s |= {"temperature": 1.2, "top_p": 0.99}
    return s


def _shared_inputs(case, g):
    page, lens, prefix = case["page"], _kv_lens(case), _prefix_lens(case)
    (first, table), left = _tables([prefix, lens], page, g, 3)
    pages = sum(-(-n // page) for n in lens + prefix) + left.shape[0]
    s = {"prefix_table": first, "prefix_lens": _ints(prefix), "cu_group": _ints(_groups_of(case)), "page_table": table,
         "kv_lens": _ints(lens)}
    s["k_codes"], s["k_scales"] = _pool(case, pages, g, 1.0)
    s["v_codes"], s["v_scales"] = _pool(case, pages, g, 0.7)
    trees = _tree_lens(case)
    total = sum(trees)
    # sharper than unit scores, as trained heads are
    s["q"] = (1.5 * torch.randn(total, case["q_heads"], case["head_dim"], generator=g,
                                device="cuda")).to(DTYPES[case["dtype"]])
    s["cu_q"] = _ints([sum(trees[:i]) for i in range(len(trees) + 1)])
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
        packed = (sees.long() << torch.arange(t, device="cuda")).sum(-1)
        s["mask"] = torch.cat([packed[i, :n] for i, n in enumerate(trees)]).unsqueeze(1)
    return s


def _inputs(case, seed):
    g = _generator(seed)
    return {"plan": _plan_inputs, "sample": _sample_inputs, "shared": _shared_inputs}[case["op"]](case, g)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        # what a serving program keeps from step to step: the handles of its page tables and of the cache
        ops = _package()
        if case["op"] == "plan":
            state["pages"] = ops["paging"].PageTables(state["page_table"], state["lens"], state["free"], state["count"],
                                                      case["page"])
        if case["op"] == "shared":
            state["cache"] = ops["kv_cache"].QuantizedKVCache(
                *(state[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")))
    return state


# ------------------------------------------------------------------ plain forms
def _plan_plain(s):
    page, most = s["case"]["page"], s["max_tokens"]
    table, stack = s["page_table"], s["free"]
    width = table.shape[1]
    pages_of = lambda n: torch.div(n + (page - 1), page, rounding_mode="floor")  # noqa: E731
    lens = s["lens"].long()
    keep = torch.minimum(s["keep"].long(), lens)
    new = s["new"].long()
    held, kept, need = pages_of(lens), pages_of(keep), pages_of(keep + new)
    fits = need <= width
    new, grow, freed = torch.where(fits, new, 0), torch.where(fits, need - kept, 0), held - kept
    count, back = s["count"].long(), freed.sum()
    served = fits & (new.cumsum(0) <= most) & ((grow == 0) | (grow.cumsum(0) <= count + back))
    refused = ((s["new"] > 0) & ~served).sum().reshape(1).to(torch.int32)
    new, grow = torch.where(served, new, 0), torch.where(served, grow, 0)
    # the pages that are cut off, on the stack so that the first of them is the first to be taken again
    k = torch.arange(width, device="cuda")
    spare = torch.zeros(1, dtype=torch.int32, device="cuda")
    at = (freed.cumsum(0) - freed)[:, None] + k - kept[:, None]
    going = (k >= kept[:, None]) & (k < held[:, None])
    to = torch.where(going, count + back - 1 - at, stack.shape[0])
    stack.copy_(torch.cat([stack, spare]).scatter_(0, to.flatten(), table.flatten())[:-1])
    # the pages that are taken
    at = (grow.cumsum(0) - grow)[:, None] + k - kept[:, None]
    coming = (k >= kept[:, None]) & (k < (kept + grow)[:, None])
    taken = stack[(count + back - 1 - at).clamp(0, stack.shape[0] - 1)]
    table.copy_(torch.where(coming, taken, table))
    s["count"].copy_((count + back - grow.sum()).to(torch.int32))
    s["lens"].copy_((keep + new).to(torch.int32))
    ends = new.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(most, device="cuda")
    b = torch.searchsorted(ends, t, right=True).clamp(max=lens.shape[0] - 1)
    live = t < ends[-1]
    position = torch.where(live, keep[b] + t - cu[b], 0)
    slot = table[b, (position // page).clamp(max=width - 1)].long() * page + position % page
    return [cu.to(torch.int32), torch.where(live, slot, -1), position.to(torch.int32), refused, table, s["lens"], stack,
            s["count"]]


def _setting(v, rows, dtype):
    return (v.to(dtype) if torch.is_tensor(v) else torch.full((rows,), v, dtype=dtype, device="cuda")).unsqueeze(1)


def _sample_plain(s):
    # in 64 bits: which token is drawn is decided between sums that may differ by little
    rows, vocab = s["logits"].shape
    heat, top_p, min_p = (_setting(s[n], rows, torch.float64) for n in ("temperature", "top_p", "min_p"))
    top_k = _setting(s["top_k"], rows, torch.int64)
    x = s["logits"].double()
    x = torch.where(x != x, -math.inf, x)
    x, order = x.sort(dim=1, descending=True, stable=True)           # equal logits: the lowest index first
    most, rank = x[:, :1], torch.arange(vocab, device="cuda")
    a = (x - most) / torch.where(heat > 0, heat, 1.0)
    w = torch.where(x == most, 1.0, torch.where(a < -700.0, 0.0, a.exp()))
    w = torch.where(x > -math.inf, w, 0.0)
    w = torch.where((top_k <= 0) | (rank < top_k), w, 0.0)
    sums = w.cumsum(1)
    before = torch.cat([sums.new_zeros(rows, 1), sums[:, :-1]], dim=1)
    kept = (top_p >= 1.0) | (before < top_p * sums[:, -1:])
    kept &= w >= min_p.clamp(max=1.0)
    kept &= heat > 0
    kept[:, 0] = True
    w = torch.where(kept, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    sums = w.cumsum(1)
    total = sums[:, -1:]
    last = (rank * (w > 0)).amax(1, keepdim=True)
    drawn = torch.minimum((sums <= s["uniform"].double().unsqueeze(1) * total).sum(1, keepdim=True), last)
    chance = (w.gather(1, drawn) / total).log()
    some = total > 0
    return [torch.where(some, drawn, -1).squeeze(1), torch.where(some, chance, -math.inf).squeeze(1).float()]


def _values(codes, scales, bits):
    """What codes and scales stand for, in float32."""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    q = codes.float() - (8.0 if bits == 4 else 0.0)
    return (q.unflatten(-1, (scales.shape[-1], -1)) * scales.float().unsqueeze(-1)).flatten(-2)


def _softmax_over(q, s, table, sees, case):
    """Maximum, sum and sum of values of rows q [n, heads, rows, head_dim] over the pages of a table, where
    sees [n, rows or 1, keys]."""
    n, keys, hk, d = table.shape[0], table.shape[1] * case["page"], case["kv_heads"], case["head_dim"]
    k = _values(s["k_codes"][table], s["k_scales"][table], case["bits"]).transpose(1, 2).reshape(n, hk, keys, d)
    scores = (q @ k.transpose(2, 3)).div_(math.sqrt(d)).masked_fill_(~sees.unsqueeze(1), -math.inf)
    del k
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.clamp(min=-1e30)).exp_()
    v = _values(s["v_codes"][table], s["v_scales"][table], case["bits"]).transpose(1, 2).reshape(n, hk, keys, d)
    return top, p.sum(-1, keepdim=True), p @ v


def _shared_plain(s):
    case = s["case"]
    q, cu, lens, of = s["q"], s["cu_q"].long(), s["kv_lens"].long(), s["cu_group"].long()
    b, t, hk, d, total = lens.shape[0], case["tree"], case["kv_heads"], case["head_dim"], q.shape[0]
    g = case["q_heads"] // hk
    # rows by group (padded), over the groups' prefixes
    most = max(1, min(total, t * max(y - x for x, y in zip(_groups_of(case)[:-1], _groups_of(case)[1:]))))
    first = cu[of]
    at = (first[:-1, None] + torch.arange(most, device="cuda")).clamp(max=total - 1)     # [groups, rows]
    rows = q[at].float().unflatten(2, (hk, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)      # [groups, heads, rows g, d]
    keys = torch.arange(s["prefix_table"].shape[1] * case["page"], device="cuda")
    sees = (keys < s["prefix_lens"][:, None])[:, None]
    parts = _softmax_over(rows, s, s["prefix_table"].long(), sees, case)
    row = torch.arange(total, device="cuda")
    mine = torch.searchsorted(first[1:], row, right=True)
    early = [x.unflatten(2, (most, g))[mine, :, row - first[mine]] for x in parts]       # [rows, heads, g, 1 or d]
    # rows by request (padded), over what the requests have of their own
    count, i = cu[1:] - cu[:-1], torch.arange(t, device="cuda")
    at = torch.minimum(cu[:-1, None] + i, cu[1:, None] - 1)
    rows = q[at].float().unflatten(2, (hk, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    keys = torch.arange(s["page_table"].shape[1] * case["page"], device="cuda")
    draft = keys - (lens - count)[:, None]                                               # which drafted token a key is
    if s["mask"] is None:
        sees = draft[:, None] <= i[:, None]
    else:
        bits = ((s["mask"][at] >> torch.arange(64, device="cuda")) & 1).bool()           # [b, t, 64]
        sees = bits.gather(2, draft.clamp(0, 63)[:, None].expand(b, t, keys.shape[0])) | (draft < 0)[:, None]
    sees = (sees & (keys < lens[:, None])[:, None]).repeat_interleave(g, dim=1)
    parts = _softmax_over(rows, s, s["page_table"].long(), sees, case)
    mine = torch.searchsorted(cu[1:], row, right=True)
    late = [x.unflatten(2, (t, g))[mine, :, row - cu[mine]] for x in parts]
    top = torch.maximum(early[0], late[0])
    x, y = (early[0] - top).exp(), (late[0] - top).exp()
    sums = x * early[1] + y * late[1]
    out = ((x * early[2] + y * late[2]) / sums).flatten(1, 2).to(q.dtype)
    return [out, (top + sums.log()).flatten(1)] if case["lse"] else [out]


def _run_plain(s):
    return {"plan": _plan_plain, "sample": _sample_plain, "shared": _shared_plain}[s["case"]["op"]](s)


# ------------------------------------------------------------- this package's
_modules = {}


def _package():
    """The package's modules, from the folder that it is imported from everywhere."""
    if not _modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "llm-inference-optimizer_b200"))
        from qlinear.kernels import kv_cache, paging, sampling, shared_attention
        _modules.update(kv_cache=kv_cache, paging=paging, sampling=sampling, shared_attention=shared_attention)
    return _modules


def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "plan":
        p = _modules["paging"].plan_step(s["pages"], s["new"], s["max_tokens"], keep=s["keep"])
        return [p.cu_q, p.slots, p.positions, p.refused, s["page_table"], s["lens"], s["free"], s["count"]]
    if op == "sample":
        return list(_modules["sampling"].sample_tokens(
            s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
            return_logprobs=True))
    # every request has up to `tree` tokens; without a mask each sees what came before it
    got = _modules["shared_attention"].shared_prefix_attention(
        s["q"], s["cache"], s["prefix_table"], s["prefix_lens"], s["page_table"], s["kv_lens"],
        cu_group=None if case["groups"] == 1 else s["cu_group"], cu_q=None if case["tree"] == 1 else s["cu_q"],
        max_q=case["tree"], mask=s["mask"], return_lse=case["lse"])
    return list(got) if case["lse"] else [got]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------- the definitions, 64 bits
def _exact_sample(case, s):
    # a row at a time, by the definition: tokens in order of their chances, filters, then the draw by index
    found = []
    for r in range(case["rows"]):
        value = lambda n: float(s[n][r]) if torch.is_tensor(s[n]) else float(s[n])  # noqa: E731
        x = s["logits"][r].double()
        index = torch.nonzero(x > -math.inf).squeeze(1)
        if index.numel() == 0:
            found.append(-math.inf)
            continue
        x = x[index]
        order = torch.argsort(-x, stable=True)
        index, x = index[order], x[order]
        if value("temperature") <= 0:
            found.append(0.0)
            continue
        if value("top_k") > 0:
            index, x = index[:int(value("top_k"))], x[:int(value("top_k"))]
        p = torch.softmax((x - x[0]) / value("temperature"), 0)
        low = p >= value("min_p") * p[0]
        if value("top_p") < 1:
            low &= p.cumsum(0) - p < value("top_p")
        low[0] = True
        index, p = index[low], p[low] / p[low].sum()
        index, order = index.sort()
        p = p[order]
        i = int(torch.searchsorted(p.cumsum(0), s["uniform"][r].double(), right=True))
        found.append(float(p[min(i, p.shape[0] - 1)].log()))
    return [None, torch.tensor(found, dtype=torch.float64, device="cuda")]


def _exact_rows(codes, scales, case):
    if case["bits"] == 8:
        return codes.double() * scales.double()
    q = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device="cuda")
    q[..., 0::2], q[..., 1::2] = (codes & 15).double() - 8, (codes >> 4).double() - 8
    return q * scales.double().repeat_interleave(q.shape[-1] // scales.shape[-1], dim=-1)


def _exact_shared(case, s):
    def rows(table, n):
        pages = table[:-(-n // case["page"])].long()
        return [_exact_rows(s[x + "_codes"][pages], s[x + "_scales"][pages], case).transpose(1, 2).flatten(0, 1)[:n]
                for x in "kv"]                                           # [n, heads, head_dim]
    trees, lens, groups = _tree_lens(case), _kv_lens(case), _groups_of(case)
    outs, lses, first = [], [], 0
    for a, n in enumerate(_prefix_lens(case)):
        early = rows(s["prefix_table"][a], n)
        for b in range(groups[a], groups[a + 1]):
            t, late = trees[b], rows(s["page_table"][b], lens[b])
            k, v = (torch.cat(x) for x in zip(early, late))
            q = s["q"][first:first + t].double().unflatten(1, (case["kv_heads"], -1))
            scores = torch.einsum("thgd,nhd->hgtn", q, k) / math.sqrt(case["head_dim"])
            hide = torch.zeros(t, k.shape[0], dtype=torch.bool, device="cuda")
            if s["mask"] is None:
                hide[:, -t:] = torch.ones(t, t, dtype=torch.bool, device="cuda").triu(1)
            else:
                hide[:, -t:] = ((s["mask"][first:first + t] >> torch.arange(t, device="cuda")) & 1) == 0
            scores = scores.masked_fill(hide, -math.inf)
            outs.append(torch.einsum("hgtn,nhd->thgd", torch.softmax(scores, -1), v).flatten(1, 2))
            lses.append(torch.logsumexp(scores, -1).permute(2, 0, 1).flatten(1))
            first += t
    return [torch.cat(outs), torch.cat(lses)] if case["lse"] else [torch.cat(outs)]


def exact(case, seed):
    if case["op"] == "plan":                 # whole numbers alone
        return None
    s = _inputs(case, seed)
    return _exact_sample(case, s) if case["op"] == "sample" else _exact_shared(case, s)


# --------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "plan":
        have, keep, new = _news(case)
        page = case["page"]
        up = lambda n: -(-n // page)  # noqa: E731
        freed = sum(up(h) - up(k) for h, k in zip(have, keep))
        taken = sum(up(k + n) - up(k) for k, n in zip(keep, new))
        # lengths, what is kept and new are read, lengths and ends written; a page that moves is read and written;
        # a token's slot and position are written
        return {"bytes": 20.0 * len(have) + 8.0 * (freed + taken) + 12.0 * sum(new), "flops": 0.0}
    if case["op"] == "sample":
        n = float(case["rows"]) * case["vocab"]
        return {"bytes": n * (4.0 if case["dtype"] == "f32" else 2.0) + 16.0 * case["rows"], "flops": 4.0 * n}
    d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    lens, prefix, trees, groups = _kv_lens(case), _prefix_lens(case), _tree_lens(case), _groups_of(case)
    cached = 2.0 * (d * case["bits"] // 8 + 2 * _groups4(case))          # one token's key and value of one head
    read = float(sum(lens) + sum(n for i, n in enumerate(prefix) if groups[i + 1] > groups[i])) * hk * cached
    queries = 2.0 * 2 * sum(trees) * hq * d + (4.0 * sum(trees) * hq if case["lse"] else 0.0)
    tables = 4.0 * sum(-(-n // case["page"]) for n in lens + prefix) + 8.0 * len(lens)
    products = sum(t * (n - t) + t * (t + 1) / 2 for t, n in zip(trees, lens))
    products += sum(n * sum(trees[groups[i]:groups[i + 1]]) for i, n in enumerate(prefix))
    return {"bytes": read + queries + tables, "flops": 4.0 * d * hq * products}
