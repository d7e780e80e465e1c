"""The quantised paged cache: append (with the rotation of q and k) must give
the codes and scales of the elementwise fp32 form bit for bit, read must give
their values rounded once; refusals; a pool past 2^32 bytes."""
import math

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv, read_kv
from qlinear.kernels.rotary import RotaryTable, apply_rotary

from attn_helpers import heads, pack, quantise, rotate_by, values

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


# ----------------------------------------------------------------------- CPU
def test_pool_forms_and_refusals():
    c = QuantizedKVCache.empty(3, 16, 2, 128, bits=8, device="cpu")
    assert (c.bits, c.head_dim, c.groups, c.num_bytes()) == (8, 128, 1, 3 * 2 * 16 * 2 * 130)
    c = QuantizedKVCache.empty(3, 32, 2, 128, bits=4, device="cpu")
    assert (c.bits, c.head_dim, c.groups, c.num_bytes()) == (4, 128, 2, 3 * 2 * 32 * 2 * 68)
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(3, 24, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(3, 8, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(3, 16, 2, 96, device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(3, 16, 2, 128, bits=6, device="cpu")
    k, s = c.k_codes, c.k_scales
    with pytest.raises(TypeError):
        QuantizedKVCache(k.float(), s, k, s)
    with pytest.raises(TypeError):
        QuantizedKVCache(k, s.float(), k, s)
    with pytest.raises(AssertionError):
        QuantizedKVCache(k, s[..., :1], k, s[..., :1])
    with pytest.raises(AssertionError):
        QuantizedKVCache(k, s, k[:1], s[:1])
    with pytest.raises(AssertionError):
        QuantizedKVCache(k[:, :, ::2], s[:, :, ::2], k[:, :, ::2], s[:, :, ::2])


def test_tensors_are_not_exchanged():
    """Calls pass on addresses taken once: a cache or table whose tensor was replaced would reach freed memory."""
    c = QuantizedKVCache.empty(3, 16, 2, 128, bits=8, device="cpu")
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    t = RotaryTable.build(64, 8, 1.0e4, device="cpu")
    with pytest.raises(AttributeError):
        t.table = t.table.clone()
    assert c.fields[0] == c.k_codes.data_ptr() and t.ptr == t.table.data_ptr()


def cache_fields(**change):
    f = dict(kc=1024, ks=1024, vc=1024, vs=1024, num_pages=4, page_size=16, kv_heads=2, head_dim=64, bits=8,
             kps=2048, vps=2048, ksps=32, vsps=32)
    f.update({n: change.pop(n) for n in list(change) if n in f})
    return list(f.values()), change


def test_host_checks_without_gpu():
    lib = _lib.load()

    def append(**change):
        c, change = cache_fields(**change)
        f = dict(k=64, v=64, q=0, q_out=0, slots=64, table=0, positions=0, tokens=2, q_heads=0, kt=128, kh=64, vt=128,
                 vh=64, qt=0, qh=0, ot=0, oh=0, dtype=_lib.QL_DTYPE_F16, slot_bytes=8, rotary_dim=0, max_positions=0,
                 layout=0, position_bytes=8, flags=0)
        f.update(change)
        return lib.ql_kv_append(_lib.KV_APPEND_ARGS.pack(*c, *f.values()), None)

    def read(**change):
        c, change = cache_fields(**change)
        f = dict(slots=64, k=64, v=64, tokens=2, dtype=_lib.QL_DTYPE_BF16, slot_bytes=4, flags=0)
        f.update(change)
        return lib.ql_kv_read(_lib.KV_READ_ARGS.pack(*c, *f.values()), None)

    for call in (append, read):
        assert call(tokens=0, slots=0) == _lib.QL_OK
        assert call(tokens=-1) == _lib.QL_ERR_BAD_SHAPE
        assert call(slots=0) == _lib.QL_ERR_NULL_POINTER
        assert call(k=0) == _lib.QL_ERR_NULL_POINTER
        assert call(kc=0) == _lib.QL_ERR_NULL_POINTER
        assert call(vs=0) == _lib.QL_ERR_NULL_POINTER
        assert call(bits=2) == _lib.QL_ERR_UNSUPPORTED
        assert call(head_dim=96) == _lib.QL_ERR_UNSUPPORTED
        assert call(page_size=24) == _lib.QL_ERR_UNSUPPORTED
        assert call(page_size=8) == _lib.QL_ERR_UNSUPPORTED
        assert call(num_pages=0) == _lib.QL_ERR_BAD_SHAPE
        assert call(kps=2032) == _lib.QL_ERR_BAD_STRIDE
        assert call(ksps=16) == _lib.QL_ERR_BAD_STRIDE
        assert call(kps=2056) == _lib.QL_ERR_UNSUPPORTED
        assert call(kc=1032) == _lib.QL_ERR_UNSUPPORTED
        assert call(slot_bytes=2) == _lib.QL_ERR_UNSUPPORTED
        assert call(dtype=_lib.QL_DTYPE_F32) == _lib.QL_ERR_UNSUPPORTED
        assert call(slots=66) == _lib.QL_ERR_UNSUPPORTED
    assert append(kt=-1) == _lib.QL_ERR_BAD_STRIDE
    assert append(rotary_dim=64) == _lib.QL_ERR_BAD_SHAPE          # no positions in the table
    assert append(rotary_dim=64, max_positions=4) == _lib.QL_ERR_NULL_POINTER
    assert append(rotary_dim=72, max_positions=4, table=64, positions=64) == _lib.QL_ERR_BAD_SHAPE
    assert append(q_heads=2) == _lib.QL_ERR_NULL_POINTER
    assert read(k=72) == _lib.QL_ERR_UNSUPPORTED                     # 16-byte rows
    assert lib.ql_kv_append(None, None) == _lib.QL_ERR_NULL_POINTER
    assert lib.ql_kv_read(None, None) == _lib.QL_ERR_NULL_POINTER


def test_queries_without_a_rotation_are_refused():
    """q_heads > 0 with rotary_dim 0 has neither angles nor positions: refused before any launch."""
    c, _ = cache_fields()
    args = dict(k=64, v=64, q=64, q_out=64, slots=64, table=0, positions=0, tokens=2, q_heads=2, kt=128, kh=64, vt=128,
                vh=64, qt=128, qh=64, ot=128, oh=64, dtype=_lib.QL_DTYPE_F16, slot_bytes=8, rotary_dim=0,
                max_positions=0, layout=0, position_bytes=8, flags=0)
    assert _lib.load().ql_kv_append(_lib.KV_APPEND_ARGS.pack(*c, *args.values()), None) == _lib.QL_ERR_BAD_SHAPE


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_move_skips_slots_outside_the_pool(device, dtype):
    """Negative slots and slots past the pool, at either end of a pair, move nothing; the other pairs of the call move."""
    cache = QuantizedKVCache.empty(3, 16, 2, 64, 8, device=device)
    ts = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    for n, t in enumerate(ts):
        t.copy_((torch.arange(48)[:, None, None] + torch.arange(2)[:, None] * 48 + n).expand(48, 2, t.shape[-1])
                .reshape(3, 16, 2, -1).transpose(1, 2).to(t.dtype))
    before = [t.clone() for t in ts]

    def rows(t):
        return t.transpose(1, 2).flatten(0, 1)

    def move(pairs):
        cache.move(*(torch.tensor([p[i] for p in pairs], dtype=dtype, device=device) for i in (0, 1)))

    for pairs in ([(-1, 3)], [(3, -1), (-1, -1)], [(5, 48)], [(48, 5), (1000, 2000)], []):
        if device == "cuda":
            _lib.clear_device_error()
        move(pairs)
        assert all(torch.equal(t, b) for t, b in zip(ts, before)), pairs
        if device == "cuda":
            past = any(s >= 48 for p in pairs for s in p)
            assert _lib.device_error() == (_lib.QL_DEVICE_ERROR_BAD_INDEX if past else 0), pairs
            _lib.clear_device_error()
    move([(-1, 4), (20, 17), (7, 0), (18, 48), (17, 16), (9, -5)])
    for t, b in zip(ts, before):
        want = rows(b).clone()
        want[17], want[0], want[16] = rows(b)[20], rows(b)[7], rows(b)[17]
        assert torch.equal(rows(t), want)
    if device == "cuda":
        _lib.clear_device_error()
    with pytest.raises(AssertionError):
        cache.move(torch.arange(2, device=device), torch.arange(3, device=device))
    with pytest.raises(TypeError):
        cache.move(torch.zeros(2, device=device), torch.zeros(2, device=device))


# ----------------------------------------------------------------------- GPU
def stored(cache, slots):
    page, at = slots // cache.page_size, slots % cache.page_size
    return [t[page, :, at] for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]


def scatter(cache, tokens, seed):
    """Distinct slots in no order."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(cache.num_pages * cache.page_size, generator=g)[:tokens].cuda()


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,head_dim,rotary_dim,layout,page", [
    (1, 12, 2, 128, 128, "half", 16), (37, 28, 4, 128, 128, "half", 32), (5, 3, 3, 64, 32, "interleaved", 16),
    (130, 8, 1, 256, 64, "half", 64), (3, 20, 4, 64, 64, "interleaved", 128), (64, 0, 5, 64, 0, "half", 16),
    (9, 0, 8, 256, 256, "interleaved", 16), (2, 40, 40, 128, 96, "half", 16)])
def test_append_and_read(tokens, q_heads, kv_heads, head_dim, rotary_dim, layout, page, bits, dtype):
    qkv = heads(tokens, q_heads + 2 * kv_heads, head_dim, dtype, tokens)
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:]
    cache = QuantizedKVCache.empty(-(-tokens // page) + 3, page, kv_heads, head_dim, bits)
    slots = scatter(cache, tokens, 1)
    rot = positions = None
    turned = k.float()
    if rotary_dim:
        rot = RotaryTable.build(rotary_dim, 700, 1.0e4, layout)
        positions = torch.randint(0, 700, (tokens,), generator=torch.Generator().manual_seed(2)).cuda()
        cos, sin = (rot.table[positions][:, None, :, i] for i in (0, 1))
        turned = rotate_by(k.float(), cos, sin, layout)
    got_q = append_kv(cache, k, v, slots, q=q if q_heads else None, positions=positions, rotary=rot)
    if q_heads:
        assert torch.equal(got_q, apply_rotary(q, positions, rot))
    else:
        assert got_q is None
    (kq, ks), (vq, vs) = quantise(turned, bits), quantise(v.float(), bits)
    want = [pack(kq, bits), ks, pack(vq, bits), vs]
    for w, s, what in zip(want, stored(cache, slots), ("k codes", "k scales", "v codes", "v scales")):
        assert torch.equal(s, w), what
    # each value is within half a step of its input: the codes' rounding, or at the top the scale's
    step = ks.double().repeat_interleave(head_dim // cache.groups, -1)
    assert bool(((values(want[0], ks, bits) - turned.double()).abs() <= step * (0.5 + 2.0 ** -7)).all())
    # read back in either type, in another order, with repeats and skipped rows; int32 slots too
    order = torch.randint(0, tokens, (2 * tokens + 1,), generator=torch.Generator().manual_seed(3)).cuda()
    at = slots[order]
    at[::5] = -1
    for out_dtype, s in ((torch.float16, at), (torch.bfloat16, at.int())):
        rk, rv = read_kv(cache, s, dtype=out_dtype)
        for r, c, sc in ((rk, want[0], ks), (rv, want[2], vs)):
            w = values(c, sc, bits)[order]
            w[::5] = 0
            assert torch.equal(r, w.float().to(out_dtype))      # code * scale is exact in fp32


@on_gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_of_zeros_tiny_huge_and_not_finite(bits):
    """Zeros; values whose scale is a bf16 subnormal or underflows; the
    largest; an infinity or NaN, which takes its own group alone."""
    x = torch.randn(8, 1, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 1e-40
    x[3] = 3.3e38
    x[3, 0, ::2] = -1.0
    x[4, 0, 5] = math.inf
    x[5, 0, 70] = math.nan
    x[6, 0, 100] = -math.inf
    x[7, 0, :64] = 0
    cache = QuantizedKVCache.empty(2, 16, 1, 128, bits)
    slots = torch.arange(8).cuda()
    append_kv(cache, x, x, slots)
    codes, scales = quantise(x.float(), bits)
    kc, ks, vc, vs = stored(cache, slots)
    assert torch.equal(kc, pack(codes, bits)) and torch.equal(vc, kc)
    assert torch.equal(ks.nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0)) and torch.equal(ks.isnan(), scales.isnan())
    k, _ = read_kv(cache, slots, torch.bfloat16)
    assert bool((k[0] == 0).all())
    assert torch.isfinite(k[[0, 1, 2, 3, 7]]).all()
    span = 64 if bits == 4 else 128
    for row, at in ((4, 5), (5, 70), (6, 100)):
        lo = at // span * span
        assert bool(k[row, 0, lo:lo + span].isnan().all())
        if bits == 4:
            other = 64 - lo
            assert bool(torch.isfinite(k[row, 0, other:other + 64]).all())


@on_gpu
def test_strides_alignment_in_place_and_skipped():
    cache, ref = (QuantizedKVCache.empty(4, 16, 2, 64, 4) for _ in range(2))
    rot = RotaryTable.build(64, 50, 1.0e4)
    pos = torch.arange(20, 29).cuda()
    qkv = heads(9, 8, 64, torch.float16, 4)
    slots = scatter(cache, 9, 5)
    want = append_kv(ref, *(qkv[:, a:b].contiguous() for a, b in ((4, 6), (6, 8))), slots, q=qkv[:, :4].contiguous(),
                     positions=pos, rotary=rot)
    # rows that do not start on 16 bytes, and q turned in place
    odd = torch.empty(9 * (8 * 64 + 1) + 3, dtype=torch.float16, device="cuda")
    odd = odd.as_strided((9, 8, 64), (8 * 64 + 1, 64, 1), 3).copy_(qkv)
    q = odd[:, :4]
    got = append_kv(cache, odd[:, 4:6], odd[:, 6:], slots.int(), q=q, positions=pos.int(), rotary=rot, q_out=q)
    assert torch.equal(got, want) and torch.equal(odd[:, :4], want) and torch.equal(odd[:, 4:], qkv[:, 4:])
    for a, b in zip(stored(cache, slots), stored(ref, slots)):
        assert torch.equal(a, b)
    # a skipped token writes nothing, but its q turns; other rows of the pool stay
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    none = torch.full((9,), -1, device="cuda")
    got = append_kv(cache, qkv[:, 6:], qkv[:, 4:6], none, q=qkv[:, :4], positions=pos, rotary=rot)
    assert torch.equal(got, want)
    for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before):
        assert torch.equal(a, b)


@on_gpu
def test_slots_past_the_pool_are_recorded_and_skipped():
    cache = QuantizedKVCache.empty(2, 16, 1, 64, 8)
    x = heads(3, 1, 64, torch.float16, 6)
    _lib.clear_device_error()
    append_kv(cache, x, x, torch.tensor([5, 32, 6]).cuda())
    assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
    _lib.clear_device_error()
    assert int((cache.k_scales != 0).sum()) == 2
    k, v = read_kv(cache, torch.tensor([5, 1 << 40, 6]).cuda())
    assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
    _lib.clear_device_error()
    assert bool((k[1] == 0).all()) and bool((v[1] == 0).all()) and bool((k[0] != 0).any())


@on_gpu
def test_pages_of_a_pool_for_all_layers():
    """A layer's slice of a [pages, layers, ...] pool: pages are strided."""
    layers = [QuantizedKVCache.empty(5, 16, 2, 64, 8) for _ in range(2)]
    both = [torch.stack([getattr(c, n) for c in layers], 1).contiguous()
            for n in ("k_codes", "k_scales", "v_codes", "v_scales")]
    second = QuantizedKVCache(*(t[:, 1] for t in both))
    x, y = heads(30, 2, 64, torch.float16, 7), heads(30, 2, 64, torch.float16, 8)
    slots = scatter(second, 30, 9)
    append_kv(second, x, y, slots)
    append_kv(layers[1], x, y, slots)
    for t, n in zip(both, ("k_codes", "k_scales", "v_codes", "v_scales")):
        assert torch.equal(t[:, 1], getattr(layers[1], n)) and int((t[:, 0] != 0).sum()) == 0
    assert all(torch.equal(a, b) for a, b in zip(read_kv(second, slots), read_kv(layers[1], slots)))


@on_gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_move_closes_up_accepted_rows(bits):
    cache = QuantizedKVCache.empty(3, 16, 2, 64, bits)
    x, y = heads(20, 2, 64, torch.float16, 10), heads(20, 2, 64, torch.float16, 11)
    slots = torch.arange(10, 30).cuda()
    append_kv(cache, x, y, slots)
    before = read_kv(cache, slots)
    cache.move(slots[[2, 5, 6, 13]], slots[[1, 2, 3, 4]])       # overlapping: all read first
    after = read_kv(cache, slots)
    for a, b in zip(after, before):
        assert torch.equal(a[[1, 2, 3, 4]], b[[2, 5, 6, 13]])
        assert torch.equal(a[5:], b[5:]) and torch.equal(a[0], b[0])


@on_gpu
def test_pool_past_32_bit_offsets():
    """Codes of 4.5 GB a side: slots in the last page."""
    pages, page, hk, d = 17300, 256, 4, 256
    cache = QuantizedKVCache(*(torch.empty(pages, hk, page, n, dtype=t, device="cuda")
                               for n, t in ((d, torch.int8), (1, torch.bfloat16)) * 2))
    assert cache.k_codes.numel() > 1 << 32
    x, y = heads(5, hk, d, torch.float16, 12), heads(5, hk, d, torch.float16, 13)
    last = pages * page
    slots = torch.tensor([last - 1, last - 300, 0, last - 257, 7]).cuda()
    append_kv(cache, x, y, slots)
    k, v = read_kv(cache, slots)
    for got, src in ((k, x), (v, y)):
        codes, scales = quantise(src.float(), 8)
        assert torch.equal(got, values(pack(codes, 8), scales, 8).float().half())


@on_gpu
def test_empty_and_refusals():
    cache = QuantizedKVCache.empty(2, 16, 2, 64, 8)
    rot = RotaryTable.build(64, 8, 1.0e4)
    x = heads(3, 2, 64, torch.float16, 14)
    q = heads(3, 4, 64, torch.float16, 15)
    slots, pos = torch.arange(3).cuda(), torch.arange(3).cuda()
    assert append_kv(cache, x[:0], x[:0], slots[:0]) is None
    assert read_kv(cache, slots[:0])[0].shape == (0, 2, 64)
    for bad in (dict(k=x[:, :1]), dict(k=x[..., :32]), dict(v=x.bfloat16()), dict(v=x[:2]), dict(slots=slots[:2]),
                dict(slots=slots.cpu()), dict(rotary=rot), dict(positions=pos), dict(q=q),
                dict(q=q.bfloat16(), rotary=rot, positions=pos), dict(q_out=q),
                dict(rotary=RotaryTable.build(128, 8, 1.0e4), positions=pos)):
        with pytest.raises(AssertionError):
            append_kv(**{**dict(cache=cache, k=x, v=x, slots=slots), **bad})
    with pytest.raises(TypeError):
        append_kv(cache, x.float(), x.float(), slots)
    with pytest.raises(TypeError):
        append_kv(cache, x, x, slots.float())
    with pytest.raises(TypeError):
        read_kv(cache, slots, dtype=torch.float32)
    with pytest.raises(AssertionError):
        read_kv(cache, slots.cpu())


@on_gpu
def test_on_another_stream_and_in_a_graph():
    cache = QuantizedKVCache.empty(4, 16, 2, 128, 8)
    rot = RotaryTable.build(128, 64, 1.0e4)
    qkv = heads(6, 16, 128, torch.float16, 16)
    slots, pos = torch.arange(6).cuda(), torch.arange(6).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        def step():
            q = append_kv(cache, qkv[:, 12:14], qkv[:, 14:], slots, q=qkv[:, :12], positions=pos, rotary=rot)
            return q, *read_kv(cache, slots)
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs = step()
    torch.cuda.current_stream().wait_stream(s)
    slots += 9
    pos += 20
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))
    assert torch.equal(outs[0], apply_rotary(qkv[:, :12], pos, rot))
