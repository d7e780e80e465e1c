"""Attention of new tokens over the quantised paged cache (ql_tree_attention)
against float64 from the same codes: one token, chains and trees; ragged
requests, rows that see nothing, pages that end inside tiles, poisoned rows
that no one sees; refusals; streams, graphs, large pools."""
import math

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv
from qlinear.kernels.tree_attention import pack_tree_mask, tree_attention, tree_mask_from_parents

from attn_helpers import attend, attention_bounds, heads, random_cache, values, visible

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


# ----------------------------------------------------------------------- CPU
def test_masks():
    m = tree_mask_from_parents([-1, 0, 0, 2, 1])
    assert m.tolist() == [[0b1], [0b11], [0b101], [0b1101], [0b10011]]
    see = torch.zeros(2, 70, 70, dtype=torch.bool)
    see[1, 3, 69] = see[1, 3, 63] = see[0, 2, 0] = True
    w = pack_tree_mask(see)
    assert w.shape == (2, 70, 2) and w[1, 3].tolist() == [-(1 << 63), 1 << 5] and w[0, 2].tolist() == [1, 0]
    assert int((w != 0).sum()) == 3
    with pytest.raises(AssertionError):
        tree_mask_from_parents([0])


def test_host_checks_without_gpu():
    lib = _lib.load()

    def call(**change):
        f = dict(kc=1024, ks=1024, vc=1024, vs=1024, num_pages=4, page_size=16, kv_heads=2, head_dim=64, bits=8,
                 kps=2048, vps=2048, ksps=32, vsps=32,
                 q=64, out=64, lse=0, page_table=64, kv_lens=64, cu_q=0, mask=0, batch=2, total_q=2, q_heads=4,
                 qt=256, qh=64, table_width=2, table_stride=2, mask_words=0, max_q=1, max_kv=32,
                 dtype=_lib.QL_DTYPE_F16, scale=0.1, ws=1024, ws_bytes=1 << 30, flags=0)
        f.update(change)
        return lib.ql_tree_attention(_lib.TREE_ATTENTION_ARGS.pack(*f.values()), None)

    assert call(total_q=0, q=0) == _lib.QL_OK
    assert call(batch=0) == _lib.QL_OK
    assert call(q_heads=0) == _lib.QL_OK
    assert call(q=0) == _lib.QL_ERR_NULL_POINTER
    assert call(out=0) == _lib.QL_ERR_NULL_POINTER
    assert call(kv_lens=0) == _lib.QL_ERR_NULL_POINTER
    assert call(page_table=0) == _lib.QL_ERR_NULL_POINTER
    assert call(kc=0) == _lib.QL_ERR_NULL_POINTER
    assert call(ws=0) == _lib.QL_ERR_NULL_POINTER
    assert call(ws=1032) == _lib.QL_ERR_UNSUPPORTED
    assert call(total_q=3) == _lib.QL_ERR_BAD_SHAPE                 # uneven without cu_q
    assert call(q_heads=5) == _lib.QL_ERR_BAD_SHAPE
    assert call(batch=-1) == _lib.QL_ERR_BAD_SHAPE
    assert call(table_stride=1) == _lib.QL_ERR_BAD_STRIDE
    assert call(qt=-1) == _lib.QL_ERR_BAD_STRIDE
    assert call(bits=16) == _lib.QL_ERR_UNSUPPORTED
    assert call(dtype=_lib.QL_DTYPE_F32) == _lib.QL_ERR_UNSUPPORTED
    assert call(out=72) == _lib.QL_ERR_UNSUPPORTED
    assert call(mask=68, mask_words=1) == _lib.QL_ERR_UNSUPPORTED
    assert lib.ql_tree_attention(None, None) == _lib.QL_ERR_NULL_POINTER


# ----------------------------------------------------------------------- GPU
class Problem:
    """Requests with the given new tokens and cached lengths over one pool.
    Rows of the pool that no request may see are poisoned: their scales are
    NaN (keys) and infinite (values)."""

    def __init__(self, q_lens, kv_lens, q_heads, kv_heads, head_dim, bits, page, dtype, mask="causal", seed=0,
                 words=None, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.lens, self.dtype, self.bits = q_lens, kv_lens, dtype, bits
        counts = [-(-n // page) for n in kv_lens]
        pages = sum(counts) + spare
        ts = random_cache(pages, page, kv_heads, head_dim, bits, seed + 1)
        width = max(max(counts), 1) + 1
        order = torch.randperm(pages, generator=g).int()
        table = torch.full((len(q_lens), width), 1 << 30, dtype=torch.int32)    # never looked at
        used = torch.zeros(pages, page, dtype=torch.bool)
        at = 0
        for b, (c, n) in enumerate(zip(counts, kv_lens)):
            table[b, :c] = order[at:at + c]
            for i in range(c):
                used[order[at + i], :min(page, n - i * page)] = True
            at += c
        hidden = ~used.cuda()[:, None, :, None].expand_as(ts[1])
        ts[1].masked_fill_(hidden, math.nan)
        ts[3].masked_fill_(hidden, math.inf)
        self.cache = QuantizedKVCache(*ts)
        self.table, self.kv = table.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda()
        total = sum(q_lens)
        self.q = heads(total, q_heads, head_dim, dtype, seed + 2, std=1.5)
        self.cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32).cuda()
        self.mask = None
        if mask != "causal":
            words = words or max(1, -(-max(q_lens) // 64))
            rows = []
            for n in q_lens:
                see = torch.rand(n, words * 64, generator=g) < 0.4
                if mask == "tree":
                    see = torch.zeros(n, words * 64, dtype=torch.bool)
                    for i in range(n):
                        if i:
                            see[i] |= see[int(torch.randint(0, i, (1,), generator=g))]
                        see[i, i] = True
                rows.append((see.unflatten(1, (words, 64)).long() << torch.arange(64)).sum(-1))
            self.mask = torch.cat(rows).cuda() if rows else None

    def run(self, **more):
        args = dict(cu_q=self.cu, mask=self.mask, return_lse=True)
        args.update(more)
        return tree_attention(self.q, self.cache, self.table, self.kv, **args)

    def check(self, got, scale=None, rows=None):
        c = self.cache
        scale = 1 / math.sqrt(c.head_dim) if scale is None else scale
        out, lse = got
        assert out.dtype == self.dtype and out.shape == self.q.shape and lse.dtype == torch.float32
        at = 0
        for b, (t, n) in enumerate(zip(self.q_lens, self.lens)):
            pages = self.table[b, :-(-n // c.page_size)].long()
            k, v = (values(x[pages], s[pages], self.bits).transpose(1, 2).flatten(0, 1)[:n]
                    for x, s in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
            see = visible(t, n, None if self.mask is None else self.mask[at:at + t])
            want = attend(self.q[at:at + t], k, v, see, scale)
            tol, tol_lse = attention_bounds(*want, self.dtype)
            off = (out[at:at + t].double() - want[0]).abs()
            assert bool((off <= tol).all()), \
                f"request {b}: off by {off.max():.3e}, {(off / tol).max():.2f} of the bound"
            low = want[1] == -math.inf
            assert torch.equal(lse[at:at + t] == -math.inf, low) and bool((out[at:at + t][low] == 0).all())
            off = (lse[at:at + t].double() - want[1]).abs()[~low]
            assert bool((off <= tol_lse[~low]).all()), f"request {b}: lse off by {off.max():.3e}"
            at += t
        assert _lib.device_error() == 0


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_heads,kv_heads,head_dim,page", [
    (12, 2, 128, 16), (28, 4, 128, 32), (8, 8, 64, 16), (8, 1, 64, 64), (6, 2, 256, 16), (40, 2, 128, 16),
    (33, 1, 64, 128)])
def test_one_token(q_heads, kv_heads, head_dim, page, bits, dtype):
    """Plain decoding: lengths of one, around tiles and pages, and longer."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 1025]
    p = Problem([1] * len(lens), lens, q_heads, kv_heads, head_dim, bits, page, dtype, seed=q_heads)
    p.check(p.run())
    p.check(p.run(cu_q=None, max_q=1, max_kv=max(lens)))


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("mask", ["causal", "tree", "random"])
@pytest.mark.parametrize("q_heads,kv_heads,head_dim,page", [
    (12, 2, 128, 16), (28, 4, 128, 64), (5, 5, 64, 16), (8, 1, 256, 32)])
def test_chains_and_trees(q_heads, kv_heads, head_dim, page, mask, bits, dtype):
    q_lens = [1, 2, 3, 8, 16, 17, 33, 64, 5]
    lens = [1, 40, 3, 300, 16, 81, 1000, 64, 777]
    p = Problem(q_lens, lens, q_heads, kv_heads, head_dim, bits, page, dtype, mask, seed=3 * q_heads)
    p.check(p.run(max_q=64, max_kv=1000))
    p.check(p.run())


@on_gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_len", [65, 100, 128, 130, 257])
def test_trees_past_a_mask_word(q_len, bits):
    for mask in ("tree", "random", "causal"):
        p = Problem([q_len, 1, q_len - 3], [q_len + 200, 30, q_len - 3], 12, 2, 128, bits, 16, torch.float16, mask,
                    seed=q_len)
        p.check(p.run())


@on_gpu
def test_rows_that_see_nothing():
    """No context and an empty mask row; more new tokens than cached
    positions; a cached length of zero; requests without rows."""
    p = Problem([3, 2, 0, 4, 1], [3, 60, 50, 4, 90], 12, 2, 128, 8, 16, torch.float16, "random", seed=5)
    p.mask[0] = 0                      # request 0 has no context: its first row sees nothing
    p.mask[1] = 1 << 2                 # and its second only its last
    p.mask[3] = 0                      # request 1 has context: an empty row sees that
    p.mask[5:9] = 0
    p.check(p.run())
    p = Problem([5, 1, 1, 70], [2, 0, 33, 0], 12, 2, 64, 4, 16, torch.bfloat16, "causal", seed=6)
    p.check(p.run())
    p = Problem([0, 0], [10, 0], 12, 2, 64, 4, 16, torch.float16, "causal", seed=7)
    out, lse = p.run()
    assert out.shape == (0, 12, 64) and lse.shape == (0, 12)


@on_gpu
@pytest.mark.parametrize("q_len", [3, 70])
def test_bits_past_the_mask_words_are_clear(q_len):
    p = Problem([q_len], [q_len + 20], 4, 2, 64, 8, 16, torch.float16, "random", seed=8, words=1)
    p.check(p.run())


@on_gpu
@pytest.mark.parametrize("kv,batch", [(20011, 1), (5003, 3), (131, 200), (33000, 2)])
@pytest.mark.parametrize("bits", [8, 4])
def test_long_and_many(kv, batch, bits):
    """Work split over the keys of few requests, and many ragged requests."""
    lens = [max(1, kv - 37 * i * (kv // 150 + 1) % kv) for i in range(batch)]
    p = Problem([1] * batch, lens, 28, 4, 128, bits, 16, torch.float16, seed=9)
    p.check(p.run(cu_q=None))
    p = Problem([1 + (7 * i) % 13 for i in range(min(batch, 8))], [n + 13 for n in lens[:8]], 12, 2, 128, bits, 16,
                torch.bfloat16, "tree", seed=10)
    p.check(p.run())


@on_gpu
def test_large_scores_and_scales():
    """Scores far apart (weights that underflow), a large and a negative
    scale, values whose quantisation scales span many orders."""
    for dtype, q_len in ((torch.float16, 1), (torch.bfloat16, 20)):
        p = Problem([q_len, q_len], [500, 90], 12, 2, 128, 8, 16, dtype, seed=11)
        for scale in (4.0, -0.5, 0.0):
            p.check(p.run(scale=scale), scale=scale)
        factors = torch.logspace(-12, 12, p.cache.v_scales.numel(), device="cuda").reshape(p.cache.v_scales.shape)
        p.cache.v_scales.mul_(factors.bfloat16())
        if dtype == torch.bfloat16:
            p.check(p.run())


@on_gpu
def test_large_and_small_queries():
    """bf16 queries near the ends of the type's range, with keys that bring
    the scores back to ordinary size."""
    for shift in (100.0, -100.0):
        p = Problem([1, 40], [200, 300], 12, 2, 128, 8, 16, torch.bfloat16, seed=12)
        p.q.mul_(2.0 ** shift)
        p.cache.k_scales.mul_(2.0 ** -shift)
        p.check(p.run())


@on_gpu
@pytest.mark.parametrize("q_len", [1, 9, 40])
def test_not_finite_rows_reach_only_those_that_see_them(q_len):
    """A NaN or infinity among a drafted token's key or value makes the rows
    that see it NaN and leaves the others' bits alone."""
    p = Problem([q_len, q_len], [q_len + 77, q_len + 50], 12, 2, 128, 8, 16, torch.float16, "tree", seed=13)
    clean, _ = p.run()
    d = q_len - 1                       # the last token: only itself sees it (a leaf)
    j = 77 + d
    page, at = p.table[0, j // 16].item(), j % 16
    for scales, value in ((p.cache.v_scales, math.nan), (p.cache.k_scales, math.nan), (p.cache.v_scales, math.inf)):
        kept = scales[page, :, at].clone()
        codes = p.cache.v_codes[page, :, at].clone()
        p.cache.v_codes[page, :, at] = 0 if value == math.inf else codes
        scales[page, :, at] = value
        out, _ = p.run()
        assert bool(out[d].isnan().all())
        others = torch.ones(2 * q_len, dtype=torch.bool)
        others[d] = False
        assert torch.equal(out[others], clean[others])
        scales[page, :, at] = kept
        p.cache.v_codes[page, :, at] = codes
    p.q[0, 3, 5] = math.nan
    out, _ = p.run()
    assert bool(out[0, 3].isnan().all()) and int(out.isnan().any(-1).sum()) == 1


@on_gpu
def test_strides_views_and_out():
    p = Problem([1, 7, 2], [33, 70, 2], 12, 2, 128, 8, 16, torch.float16, seed=14)
    want = p.run()
    fused = torch.zeros(10, 16, 128, dtype=torch.float16, device="cuda")
    fused[:, :12] = p.q
    q, p.q = p.q, fused[:, :12]
    got = p.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(10 * 12 * 129 + 1, dtype=torch.float16, device="cuda").as_strided((10, 12, 128), (12 * 129, 129, 1), 1)
    p.q = odd.copy_(q)                                  # rows that do not start on 16 bytes
    out = torch.empty_like(q)
    got = p.run(out=out)
    assert got[0] is out and torch.equal(out, want[0])
    p.q, p.table = q, torch.cat([p.table, p.table], 1)[:, :p.table.shape[1]]
    assert torch.equal(p.run(return_lse=False), want[0])


@on_gpu
def test_page_tables_of_any_strides():
    """One row of pages for all requests, as a view without a stride; rows that overlap; columns of a wider table."""
    p = Problem([1] * 3, [70, 70, 70], 4, 2, 64, 8, 16, torch.float16, seed=22)
    row = p.table[1]
    want = None
    flat = torch.cat([row, row, row])
    for table in (row.repeat(3, 1), row.expand(3, -1), row[None].expand(3, -1), flat.as_strided((3, 5), (0, 1)),
                  torch.stack([row, row], 1)[:, 0].expand(3, -1), flat.reshape(3, -1).t().contiguous().t()):
        p.table = table
        got = p.run(cu_q=None)[0]
        p.check((got, p.run()[1]))
        want = got if want is None else want
        assert torch.equal(got, want)
    p.table = torch.arange(8, dtype=torch.int32, device="cuda").as_strided((3, 5), (1, 1))     # requests a page apart
    p.cache.k_scales.nan_to_num_(nan=0.01)
    p.cache.v_scales.nan_to_num_(posinf=0.01)
    p.check(p.run())


@on_gpu
def test_pages_outside_the_pool_are_recorded_and_hidden():
    p = Problem([1, 1], [40, 64], 4, 2, 64, 8, 16, torch.float16, seed=15)
    good = p.table.clone()
    _lib.clear_device_error()
    p.table[1, 3] = p.cache.num_pages
    out, _ = p.run()
    assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
    _lib.clear_device_error()
    p.table[1, 3] = -1
    again, _ = p.run()
    assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
    _lib.clear_device_error()
    assert torch.equal(out, again)
    # as if the request ended before that page (its one row sees all that is left)
    p.table = good
    p.kv[1] = 48
    p.lens[1] = 48
    p.check(p.run())
    off = (p.run()[0][1].double() - out[1].double()).abs().max().item()
    assert off <= 2.0 ** -10 * out[1].abs().max().item()


@on_gpu
def test_lengths_past_the_table_are_clamped():
    p = Problem([1], [64], 4, 2, 64, 8, 16, torch.float16, seed=16)
    p.table = p.table[:, :4].contiguous()
    want = p.run()[0]
    p.kv[0] = 1 << 30
    assert torch.equal(p.run()[0], want)


@on_gpu
def test_pool_past_32_bit_offsets():
    pages, page, hk, d = 17300, 256, 4, 256
    ts = [torch.empty(pages, hk, page, n, dtype=t, device="cuda")
          for n, t in ((d, torch.int8), (1, torch.bfloat16)) * 2]
    cache = QuantizedKVCache(*ts)
    assert cache.k_codes.numel() > 1 << 32
    n = 300
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    k, v = heads(n, hk, d, torch.float16, 17), heads(n, hk, d, torch.float16, 18)
    i = torch.arange(n, device="cuda")
    append_kv(cache, k, v, table[0, i // page].long() * page + i % page)
    small = QuantizedKVCache.empty(3, page, hk, d, 8)
    append_kv(small, k, v, i)
    for q_len in (1, 20):
        q = heads(q_len, 8, d, torch.float16, 19)
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
        assert torch.equal(tree_attention(q, cache, table, lens), tree_attention(q, small, near, lens))


@on_gpu
def test_repeatable_bits_on_streams_and_in_a_graph():
    """The same bits on every call, on two streams at once, and from a graph
    whose lengths change between replays."""
    p = Problem([3, 9, 1], [4000, 900, 70], 28, 4, 128, 8, 16, torch.float16, "tree", seed=20)
    want = p.run()
    for _ in range(5):
        got = p.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(p.run())
    torch.cuda.synchronize()
    for o in outs[0] + outs[1]:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    s = streams[0]
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out, lse = p.run()
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    assert torch.equal(out, want[0])
    p.lens = [1500, 500, 33]
    p.kv.copy_(torch.tensor(p.lens, dtype=torch.int32))
    for _ in range(3):
        graph.replay()
        p.check((out, lse))


@on_gpu
def test_refusals():
    p = Problem([1, 1], [5, 9], 4, 2, 64, 8, 16, torch.float16, seed=21)
    q, c, t, kv = p.q, p.cache, p.table, p.kv
    for args, more in (((q[..., :32], c, t, kv), {}), ((q[:, :3], c, t, kv), {}), ((q.cpu(), c, t, kv), {}),
                       ((q, c, t[:1], kv), {}), ((q, c, t.cpu(), kv), {}), ((q[:1], c, t, kv), {}),
                       ((q, c, t, kv), dict(cu_q=p.cu[:2])), ((q, c, t, kv), dict(out=q.bfloat16())),
                       ((q, c, t, kv), dict(mask=torch.zeros(1, 1, dtype=torch.int64, device="cuda"))),
                       ((q, c, t, kv), dict(mask=torch.zeros(2, 0, dtype=torch.int64, device="cuda")))):
        with pytest.raises(AssertionError):
            tree_attention(*args, **more)
    for args, more in (((q.float(), c, t, kv), {}), ((q, c, t.long(), kv), {}), ((q, c, t, kv.long()), {}),
                       ((q, c, t, kv), dict(cu_q=p.cu.long())),
                       ((q, c, t, kv), dict(mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")))):
        with pytest.raises(TypeError):
            tree_attention(*args, **more)
