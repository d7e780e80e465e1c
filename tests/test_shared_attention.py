"""Attention behind shared prefixes (ql_shared_attention) against float64 from the same codes, with the kernels as chosen
and with each family forced for both passes: groups of one request and of many, empty ones, requests of none; prefixes from
nothing on; ragged own lengths, masks, rows that see nothing; refusals; streams and graphs.

The bound is tree_attention's: the outputs of the two passes are joined in fp32, which adds a few 2^-24 of them, as the
exponentials and sums that it allows 2^-20 for."""
import math
import sys

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.kv_cache import QuantizedKVCache
from qlinear.kernels.shared_attention import shared_prefix_attention
from qlinear.kernels.tree_attention import tree_attention

from attn_helpers import attend, attention_bounds, heads, random_cache, values, visible

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


@pytest.fixture(params=["as chosen", "tensor cores", "streaming"])
def family(request, monkeypatch):
    flag = {"as chosen": 0, "tensor cores": _lib.QL_FLAG_FORCE_GEMM, "streaming": _lib.QL_FLAG_FORCE_GEMV}[request.param]
    monkeypatch.setattr(sys.modules[shared_prefix_attention.__module__], "call_flags", lambda: _lib.QL_FLAG_PDL | flag)
    return request.param


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Problem:
    """Groups of requests (cu_group, over q_lens and kv_lens) behind prefixes.  Rows of the pool that nothing may see are
    poisoned: their scales are NaN (keys) and infinite (values)."""

    def __init__(self, prefixes, cu_group, q_lens, kv_lens, q_heads, kv_heads, head_dim, bits, page, dtype, mask="causal",
                 seed=0):
        g = torch.Generator().manual_seed(seed)
        self.prefixes, self.groups, self.q_lens, self.lens = prefixes, cu_group, q_lens, kv_lens
        self.dtype, self.bits = dtype, bits
        counts = [-(-n // page) for n in prefixes + kv_lens]
        pages = sum(counts) + 2
        ts = random_cache(pages, page, kv_heads, head_dim, bits, seed + 1)
        order = torch.randperm(pages, generator=g).int()
        used = torch.zeros(pages, page, dtype=torch.bool)
        rows, at = [], 0
        for c, n in zip(counts, prefixes + kv_lens):
            rows.append(order[at:at + c])
            for i in range(c):
                used[order[at + i], :min(page, n - i * page)] = True
            at += c
        hidden = ~used.cuda()[:, None, :, None].expand_as(ts[1])
        ts[1].masked_fill_(hidden, math.nan)
        ts[3].masked_fill_(hidden, math.inf)
        self.cache = QuantizedKVCache(*ts)

        def table(some):
            t = torch.full((len(some), max(map(len, some), default=0) + 1), 1 << 30, dtype=torch.int32)    # never looked at
            for i, r in enumerate(some):
                t[i, :len(r)] = r
            return t.cuda()
        self.first, self.table = table(rows[:len(prefixes)]), table(rows[len(prefixes):])
        self.q = heads(sum(q_lens), q_heads, head_dim, dtype, seed + 2, std=1.5)
        self.cu = ints([sum(q_lens[:i]) for i in range(len(q_lens) + 1)])
        self.mask = None
        if mask != "causal":
            words, made = max(1, -(-max(q_lens) // 64)), []
            for n in q_lens:
                see = torch.rand(n, words * 64, generator=g) < 0.4
                if mask == "tree":
                    see = torch.zeros(n, words * 64, dtype=torch.bool)
                    for i in range(n):
                        if i:
                            see[i] |= see[int(torch.randint(0, i, (1,), generator=g))]
                        see[i, i] = True
                made.append((see.unflatten(1, (words, 64)).long() << torch.arange(64)).sum(-1))
            self.mask = torch.cat(made).cuda()

    def args(self):
        return self.q, self.cache, self.first, ints(self.prefixes), self.table, ints(self.lens)

    def run(self, **more):
        args = dict(cu_group=ints(self.groups), cu_q=self.cu, mask=self.mask, return_lse=True)
        args.update(more)
        return shared_prefix_attention(*self.args(), **args)

    def rows(self, table, n):
        pages, c = table[:-(-n // self.cache.page_size)].long(), self.cache
        return [values(x[pages], s[pages], self.bits).transpose(1, 2).flatten(0, 1)[:n]
                for x, s in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales))]

    def check(self, got, scale=None):
        scale = 1 / math.sqrt(self.cache.head_dim) if scale is None else scale
        out, lse = got
        assert out.dtype == self.dtype and out.shape == self.q.shape and lse.dtype == torch.float32
        at = 0
        for b, (t, n) in enumerate(zip(self.q_lens, self.lens)):
            k, v = self.rows(self.table[b], n)
            see = visible(t, n, None if self.mask is None else self.mask[at:at + t])
            for g, m in enumerate(self.prefixes):
                if self.groups[g] <= b < self.groups[g + 1]:
                    early = self.rows(self.first[g], m)
                    k, v = torch.cat([early[0], k]), torch.cat([early[1], v])
                    see = torch.cat([torch.ones(t, m, dtype=torch.bool, device="cuda"), see], 1)
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


# ----------------------------------------------------------------------- CPU
def test_host_checks_without_gpu():
    lib = _lib.load()

    def call(**change):
        f = dict(kc=1024, ks=1024, vc=1024, vs=1024, num_pages=4, page_size=16, kv_heads=2, head_dim=64, bits=8,
                 kps=2048, vps=2048, ksps=32, vsps=32,
                 q=64, out=64, lse=0, page_table=64, kv_lens=64, cu_q=0, mask=0, batch=2, total_q=2, q_heads=4,
                 qt=256, qh=64, table_width=2, table_stride=2, mask_words=0, max_q=1, max_kv=32,
                 dtype=_lib.QL_DTYPE_F16, scale=0.1, ws=1024, ws_bytes=1 << 30, flags=0,
                 prefix_table=64, prefix_lens=64, cu_group=64, parts=64, groups=2, prefix_width=3, prefix_stride=3,
                 max_prefix=48, parts_bytes=1 << 20)
        f.update(change)
        return lib.ql_shared_attention(_lib.SHARED_ATTENTION_ARGS.pack(*f.values()), None)

    assert call(total_q=0, q=0) == call(batch=0) == call(q_heads=0) == _lib.QL_OK
    assert lib.ql_shared_attention(None, None) == _lib.QL_ERR_NULL_POINTER
    assert call(q_heads=5) == call(total_q=3) == call(batch=-1) == _lib.QL_ERR_BAD_SHAPE
    assert call(q=0) == call(out=0) == _lib.QL_ERR_NULL_POINTER
    assert call(groups=-1) == call(groups=65536) == call(prefix_width=-1) == _lib.QL_ERR_BAD_SHAPE
    assert call(cu_group=0) == _lib.QL_ERR_BAD_SHAPE                # two groups
    for name in ("prefix_table", "prefix_lens", "parts"):
        assert call(**{name: 0}) == _lib.QL_ERR_NULL_POINTER, name
    assert call(prefix_stride=2) == _lib.QL_ERR_BAD_STRIDE
    for name in ("prefix_table", "prefix_lens", "cu_group"):
        assert call(**{name: 66}) == _lib.QL_ERR_UNSUPPORTED, name
    assert call(parts=72) == _lib.QL_ERR_UNSUPPORTED
    assert call(parts_bytes=100) == _lib.QL_ERR_WORKSPACE
    assert lib.ql_shared_attention_parts_size(3, 4, 64) == 96 + 12 * 256
    assert lib.ql_shared_attention_parts_size(3, 5, 64) == 128 + 15 * 256       # the outputs begin on 16 bytes
    assert lib.ql_shared_attention_parts_size(-1, 4, 64) == 0


# ----------------------------------------------------------------------- GPU
@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_heads,kv_heads,head_dim,page", [(12, 2, 128, 16), (28, 4, 128, 32), (5, 5, 64, 16), (8, 1, 64, 64),
                                                            (6, 2, 256, 16)])
def test_one_token(q_heads, kv_heads, head_dim, page, bits, dtype, family):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700]
    for prefix in (1, 127, 128, 1000):
        p = Problem([prefix], [0, 12], [1] * 12, lens, q_heads, kv_heads, head_dim, bits, page, dtype, seed=q_heads + prefix)
        p.check(p.run())
        p.check(p.run(cu_q=None, cu_group=None, max_kv=700, max_prefix=prefix))


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("mask", ["causal", "tree", "random"])
def test_groups_and_trees(mask, bits, dtype, family):
    q_lens, lens = [1, 2, 3, 8, 16, 17, 33, 64, 5, 1, 70], [1, 40, 3, 300, 16, 81, 1000, 64, 777, 9, 80]
    p = Problem([900, 31, 2500], [0, 4, 9, 11], q_lens, lens, 12, 2, 128, bits, 16, dtype, mask, seed=3)
    p.check(p.run(max_q=70))
    p.check(p.run())


@on_gpu
def test_empty_prefixes_groups_and_requests_outside(family):
    """A prefix of no positions; groups of no request; requests before the first group and behind the last; a request
    without rows; one group given by its bounds."""
    q_lens, lens = [2, 1, 0, 3, 1, 4, 1], [9, 40, 7, 3, 1, 20, 300]
    for prefixes, groups in (([0, 300], [0, 3, 7]), ([50, 60, 70, 80], [0, 0, 4, 4, 7]), ([200], [2, 4]), ([200, 90], [1, 3, 6]),
                             ([100, 100], [7, 7, 7]), ([64], [0, 0]), ([0], [0, 7])):
        p = Problem(prefixes, groups, q_lens, lens, 12, 2, 128, 8, 16, torch.float16, "tree", seed=len(groups))
        p.check(p.run())
    p = Problem([90, 200], [1, 2, 4], [3] * 5, [30, 9, 3, 50, 77], 8, 2, 64, 4, 16, torch.bfloat16, seed=4)
    p.check(p.run(cu_q=None))
    p.prefixes, p.groups, p.first = [], [0], p.first[:0]
    p.check(p.run())


@on_gpu
def test_prefix_tables_without_pages(family):
    """Lengths are clamped to the table: there is no prefix."""
    p = Problem([90], [0, 3], [2, 1, 4], [30, 9, 50], 8, 2, 64, 8, 16, torch.float16, seed=16)
    p.first = p.first[:, :0]
    got = p.run(cu_group=None)
    p.prefixes = [0]
    p.check(got)


@on_gpu
def test_many_groups(family):
    """More groups than a warp's lanes; some of them empty, lengths from 0 to several units."""
    n = 75
    groups = [0]
    for i in range(n):
        groups.append(groups[-1] + (i * 7) % 3)
    batch = groups[-1] + 2
    p = Problem([(i * 97) % 700 for i in range(n)], groups, [1 + b % 3 for b in range(batch)], [3 + (b * 31) % 90 for b in range(batch)],
                8, 2, 64, 8, 16, torch.float16, seed=17)
    p.check(p.run())


@on_gpu
def test_rows_that_see_nothing_of_their_own(family):
    """Own lengths of zero and masks without a bit: the prefix alone; with a prefix of nothing: zeros."""
    for prefix in (400, 0):
        p = Problem([prefix], [0, 4], [3, 2, 1, 4], [3, 0, 0, 4], 12, 2, 128, 8, 16, torch.float16, "random", seed=5)
        p.mask[0], p.mask[6:9] = 0, 0
        p.check(p.run())
    p = Problem([0], [0, 2], [70, 1], [0, 0], 12, 2, 64, 4, 16, torch.bfloat16, seed=6)
    p.check(p.run())


@on_gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_long_prefixes(bits, family):
    for prefix, batch, tree in ((33001, 2, 1), (20011, 40, 1), (9001, 16, 9)):
        p = Problem([prefix], [0, batch], [tree] * batch, [tree + (37 * i) % 300 for i in range(batch)], 28, 4, 128, bits, 16,
                    torch.float16, "tree", seed=7)
        p.check(p.run(max_q=tree))


@on_gpu
def test_far_scores(family):
    """What one pass finds outweighs the other's, or hardly counts; negative and zero scales."""
    p = Problem([500], [0, 3], [1, 2, 9], [40, 90, 9], 12, 2, 128, 8, 16, torch.float16, seed=8)
    for scale in (4.0, -0.5, 0.0):
        p.check(p.run(scale=scale), scale=scale)
    pages = p.first[0, :32].long()
    for factor in (2.0 ** 6, 2.0 ** -12):                   # the prefix's scores against the requests' own
        p.cache.k_scales[pages] = p.cache.k_scales[pages] * factor
        p.check(p.run())


@on_gpu
def test_it_is_attention_over_both(family):
    """Prefix and own positions as one cache of each request, in tree_attention: the same to two roundings of the output and
    those of the weights."""
    page, batch = 16, 6
    p = Problem([320], [0, batch], [5] * batch, [5 + 31 * i for i in range(batch)], 12, 2, 128, 8, page, torch.float16, "tree",
                seed=9)
    table = torch.cat([p.first[:, :20].expand(batch, -1), p.table], 1)
    whole, lse = tree_attention(p.q, p.cache, table, ints([320 + n for n in p.lens]), cu_q=p.cu, mask=p.mask, return_lse=True)
    out, both = p.run()
    # each: weights to 2^-11 of sums up to the largest value, and half a step of the output
    most = float((p.cache.v_codes.double().abs().amax() * p.cache.v_scales[p.cache.v_scales.isfinite()].double().amax()))
    assert float((out.double() - whole.double()).abs().max()) <= 2 * (2.0 ** -11 + 2.0 ** -11) * most
    assert float((lse - both).abs().max()) <= 2.0 ** -18 * float(lse.abs().max() + 1)


@on_gpu
def test_not_finite_values(family):
    """A NaN in the prefix reaches all of its group, one among a request's own keys that request alone."""
    p = Problem([100, 60], [0, 2, 4], [1] * 4, [20, 33, 8, 50], 12, 2, 128, 8, 16, torch.float16, seed=10)
    clean, _ = p.run()
    page = int(p.first[0, 3])
    kept = p.cache.v_scales[page, :, 5].clone()
    p.cache.v_scales[page, :, 5] = math.nan
    out, _ = p.run()
    assert bool(out[:2].isnan().all()) and torch.equal(out[2:], clean[2:])
    p.cache.v_scales[page, :, 5] = kept
    p.cache.k_scales[int(p.table[3, 1]), :, 4] = math.nan
    out, _ = p.run()
    assert bool(out[3].isnan().all()) and torch.equal(out[:3], clean[:3])


@on_gpu
def test_strides_out_and_tables(family):
    p = Problem([150], [0, 3], [1, 7, 2], [33, 70, 2], 12, 2, 128, 8, 16, torch.float16, seed=11)
    want = p.run()
    q = p.q
    fused = torch.zeros(10, 16, 128, dtype=torch.float16, device="cuda")
    fused[:, :12] = q
    p.q = fused[:, :12]
    out = torch.empty_like(q)
    got = p.run(out=out)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    p.q = torch.empty(10 * 12 * 129 + 1, dtype=torch.float16, device="cuda").as_strided((10, 12, 128), (12 * 129, 129, 1), 1).copy_(q)
    p.first, p.table = torch.cat([p.first, p.first], 1)[:, :p.first.shape[1]], p.table.t().contiguous().t()
    got = p.run(return_lse=False)
    assert torch.equal(got, want[0])


@on_gpu
def test_rows_behind_the_last_request_are_left(family):
    p = Problem([150], [0, 2], [3, 2], [33, 70], 12, 2, 128, 8, 16, torch.float16, seed=12)
    want = p.run()[0]
    p.q = torch.cat([p.q, p.q])
    out = torch.full_like(p.q, 7.0)
    for more in (dict(), dict(cu_group=None)):
        p.run(out=out, **more)
        assert torch.equal(out[:5], want) and bool((out[5:] == 7).all())


@on_gpu
def test_pages_outside_the_pool_are_recorded_and_hidden(family):
    p = Problem([64, 48], [0, 2, 3], [1] * 3, [40, 30, 20], 4, 2, 64, 8, 16, torch.float16, seed=13)
    _lib.clear_device_error()
    for bad in (p.cache.num_pages, -1):
        p.first[0, 3] = bad
        out = p.run()
        assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
        _lib.clear_device_error()
        p.prefixes[0] = 48                                  # as if the prefix ended there
        p.check(out)
        p.prefixes[0] = 64


@on_gpu
def test_streams_and_graphs(family):
    p = Problem([3000, 700], [0, 2, 5], [3, 9, 1, 1, 20], [400, 90, 70, 1, 33], 28, 4, 128, 8, 16, torch.float16, "tree", seed=14)
    want = p.run()
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
    lens, prefixes, groups = ints(p.lens), ints(p.prefixes), ints(p.groups)
    s = streams[0]
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = shared_prefix_attention(p.q, p.cache, p.first, prefixes, p.table, lens, cu_group=groups, cu_q=p.cu, mask=p.mask,
                                          return_lse=True)
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    assert torch.equal(got[0], want[0])
    p.lens, p.prefixes, p.groups = [200, 70, 33, 1, 20], [1500, 64], [0, 4, 5]
    for to, v in ((lens, p.lens), (prefixes, p.prefixes), (groups, p.groups)):
        to.copy_(ints(v))
    p.first[1, :4] = p.first[1, :4].clone()
    for _ in range(3):
        graph.replay()
        p.check(got)


@on_gpu
def test_refusals():
    p = Problem([30, 20], [0, 1, 2], [1, 1], [5, 9], 4, 2, 64, 8, 16, torch.float16, seed=15)
    q, c, first, prefix, t, kv = p.args()
    cu = ints(p.groups)
    run = shared_prefix_attention
    for args, more in (((q[..., :32], c, first, prefix, t, kv), {}), ((q[:, :3], c, first, prefix, t, kv), {}),
                       ((q.cpu(), c, first, prefix, t, kv), {}), ((q, c, first[:1], prefix, t, kv), {}),
                       ((q, c, first, prefix, t[:1], kv), {}), ((q, c, first.cpu(), prefix, t, kv), {}),
                       ((q, c, first, prefix, t, kv), dict(cu_group=None)), ((q, c, first, prefix, t, kv), dict(cu_group=cu[:2])),
                       ((q[:1], c, first, prefix, t, kv), {}), ((q, c, first, prefix, t, kv), dict(cu_q=cu[:2])),
                       ((q, c, first, prefix, t, kv), dict(out=q.bfloat16())),
                       ((q, c, first, prefix, t, kv), dict(mask=torch.zeros(2, 0, dtype=torch.int64, device="cuda")))):
        with pytest.raises(AssertionError):
            run(*args, **(dict(cu_group=cu) | more))
    for args, more in (((q.float(), c, first, prefix, t, kv), {}), ((q, c, first.long(), prefix, t, kv), {}),
                       ((q, c, first, prefix.long(), t, kv), {}), ((q, c, first, prefix, t, kv.long()), {}),
                       ((q, c, first, prefix, t, kv), dict(cu_group=cu.long())), ((q, c, first, prefix, t, kv), dict(cu_q=cu.long())),
                       ((q, c, first, prefix, t, kv), dict(mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")))):
        with pytest.raises(TypeError):
            run(*args, **(dict(cu_group=cu) | more))


def test_parts_size_is_the_librarys():
    from qlinear.kernels.shared_attention import parts_size
    for total_q, q_heads, head_dim in ((0, 4, 64), (1, 1, 64), (3, 5, 128), (77, 28, 256), (100000, 64, 128)):
        assert parts_size(total_q, q_heads, head_dim) == _lib.load().ql_shared_attention_parts_size(total_q, q_heads, head_dim)
