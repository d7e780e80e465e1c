"""Rotary positions: the table's frequencies (CPU) and ql_rotary (GPU)
against float64, for both pair layouts, parts of heads, strides, alignment,
both directions, and its refusals."""
import math

import numpy as np
import pytest
import torch

from qlinear import _lib
from qlinear.kernels.rotary import RotaryTable, apply_rotary, rotary_frequencies

from attn_helpers import HALF_ULP, TINY, heads, rotate

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


# ----------------------------------------------------------------------- CPU
def test_default_and_linear_frequencies():
    f, factor = rotary_frequencies(64, 5.0e5)
    want = np.array([5.0e5 ** (-2.0 * i / 64) for i in range(32)])
    assert factor == 1.0 and np.allclose(f.numpy(), want, rtol=1e-14)
    g, factor = rotary_frequencies(64, 5.0e5, {"rope_type": "linear", "factor": 4.0})
    assert factor == 1.0 and np.allclose(g.numpy(), want / 4, rtol=1e-14)


def test_llama3_frequencies_keep_stretch_and_blend():
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 8192}
    f, _ = rotary_frequencies(128, 5.0e5, s)
    for i in range(64):
        plain = 5.0e5 ** (-2.0 * i / 128)
        wavelength = 2 * math.pi / plain
        if wavelength < 8192 / 4.0:
            want = plain
        elif wavelength > 8192 / 1.0:
            want = plain / 8
        else:
            smooth = (8192 / wavelength - 1.0) / 3.0
            want = (1 - smooth) * plain / 8 + smooth * plain
        assert f[i].item() == pytest.approx(want, rel=1e-12)


def test_yarn_frequencies_and_factor():
    s = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    f, factor = rotary_frequencies(128, 1.0e6, s)
    plain, _ = rotary_frequencies(128, 1.0e6)
    assert factor == pytest.approx(0.1 * math.log(4.0) + 1.0)
    turns = 32768 * plain / (2 * math.pi)
    assert torch.allclose(f[turns > 40], plain[turns > 40], rtol=1e-12)
    assert torch.allclose(f[turns < 0.7], plain[turns < 0.7] / 4, rtol=1e-12)
    ratio = f / plain
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all()) and ratio.min() >= 0.25 - 1e-12
    _, given = rotary_frequencies(128, 1.0e6, {**s, "attention_factor": 0.5})
    assert given == 0.5


@pytest.mark.parametrize("base,old", [(1.0e4, 4096), (1.5e5, 4096), (1.0e6, 32768)])
def test_yarn_ramp_between_fractional_pairs(base, old):
    """truncate false: the ramp runs from the very pair that turns beta_fast times to the one that turns beta_slow times."""
    s = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": old, "beta_fast": 32.0, "beta_slow": 1.0,
         "truncate": False}
    f, _ = rotary_frequencies(64, base, s)
    whole, _ = rotary_frequencies(64, base, {**s, "truncate": True})
    default, _ = rotary_frequencies(64, base, {n: v for n, v in s.items() if n != "truncate"})
    assert torch.equal(whole, default) and not torch.allclose(f, whole, rtol=1e-6)
    lo, hi = (64 * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    for got, a, b in ((f, lo, hi), (whole, math.floor(lo), math.ceil(hi))):
        for i in range(32):
            stretched = min(max((i - a) / (b - a), 0.0), 1.0)
            plain = base ** (-2.0 * i / 64)
            assert got[i].item() == pytest.approx(plain * (1 - stretched) + plain / 32.0 * stretched, rel=1e-12)


def test_yarn_factor_of_two_mscales():
    s = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    m = lambda x: 0.1 * x * math.log(40.0) + 1.0                                  # noqa: E731
    assert rotary_frequencies(64, 1.0e4, {**s, "mscale": 0.707, "mscale_all_dim": 0.707})[1] == pytest.approx(1.0)
    assert rotary_frequencies(64, 1.0e4, {**s, "mscale": 1.0, "mscale_all_dim": 0.5})[1] == pytest.approx(m(1.0) / m(0.5))
    assert rotary_frequencies(64, 1.0e4, {**s, "mscale": 1.0})[1] == pytest.approx(m(1.0))
    assert rotary_frequencies(64, 1.0e4, {**s, "mscale": 0.5, "mscale_all_dim": 1.0, "attention_factor": 1.25})[1] == 1.25
    for lone in ({"mscale": 0.5}, {"mscale_all_dim": 1.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, 1.0e4, {**s, **lone})


@pytest.mark.parametrize("kind", ["yarn", "dynamic"])
def test_older_configurations_name_the_scaling_type(kind):
    """`type` in the place of `rope_type`, beside rope_theta: the same table, the original length the model's own."""
    class Config:
        hidden_size, num_attention_heads, max_position_embeddings, rope_theta = 1024, 16, 512, 5.0e5

    tables = []
    for key in ("type", "rope_type"):
        Config.rope_scaling = {key: kind, "factor": 2.0, "original_max_position_embeddings": None}
        tables.append(RotaryTable.from_config(Config, max_positions=1024, device="cpu").table)
    assert torch.equal(*tables)
    f, factor = rotary_frequencies(64, 5.0e5, {"rope_type": kind, "factor": 2.0,
                                               "original_max_position_embeddings": 512}, 1024)
    assert tables[0][1000, 3, 0].item() == pytest.approx(factor * math.cos(1000 * f[3].item()), abs=2.0 ** -23)


def test_keys_that_are_not_known_are_refused():
    with pytest.raises(ValueError, match="stretch"):
        rotary_frequencies(64, 1.0e4, {"rope_type": "linear", "factor": 2.0, "stretch": 3.0})

    class Config:                                        # parameters by kind of layer
        hidden_size, num_attention_heads, max_position_embeddings = 1024, 16, 512
        rope_parameters = {"full_attention": {"rope_type": "default", "rope_theta": 1.0e6},
                           "sliding_attention": {"rope_type": "default", "rope_theta": 1.0e4}}
    with pytest.raises(ValueError, match="full_attention"):
        RotaryTable.from_config(Config, device="cpu")


def test_dynamic_base_grows_only_past_the_original_length():
    s = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    plain, _ = rotary_frequencies(64, 1.0e4)
    assert torch.equal(rotary_frequencies(64, 1.0e4, s, 4096)[0], plain)
    grown, _ = rotary_frequencies(64, 1.0e4, s, 16384)
    base = 1.0e4 * (2.0 * 4 - 1.0) ** (64 / 62)
    assert grown[5].item() == pytest.approx(base ** (-10 / 64), rel=1e-12)


def test_table_refusals_and_config():
    with pytest.raises(ValueError):
        rotary_frequencies(64, 1.0e4, {"rope_type": "other"})
    with pytest.raises(ValueError):
        rotary_frequencies(64, 1.0e4, {"rope_type": "linear"})
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(4, 8, 2), layout="sideways")
    with pytest.raises(TypeError):
        RotaryTable(torch.zeros(4, 8, 2, dtype=torch.float64))
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(4, 6, 2))              # 12 elements: not a multiple of 8
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(0, 8, 2))

    class Config:
        hidden_size, num_attention_heads, max_position_embeddings = 1536, 12, 512
        rope_parameters = {"rope_type": "default", "rope_theta": 1.0e6}
    t = RotaryTable.from_config(Config, device="cpu")
    assert t.table.shape == (512, 64, 2)
    want = math.cos(300 * 1.0e6 ** (-2.0 * 7 / 128))
    assert t.table[300, 7, 0].item() == pytest.approx(want, abs=2.0 ** -24)


def test_host_checks_without_gpu():
    lib = _lib.load()

    def args(**change):
        f = dict(x=64, out=64, table=64, positions=64, tokens=2, heads=3, head_dim=64, rotary_dim=64, max_positions=8,
                 xt=192, xh=64, ot=192, oh=64, dtype=_lib.QL_DTYPE_F16, layout=0, position_bytes=8, inverse=0, flags=0)
        f.update(change)
        return lib.ql_rotary(_lib.ROTARY_ARGS.pack(*f.values()), None)

    assert args(tokens=0, x=0) == _lib.QL_OK
    assert args(heads=0) == _lib.QL_OK
    assert args(x=0) == _lib.QL_ERR_NULL_POINTER
    assert args(table=0) == _lib.QL_ERR_NULL_POINTER
    assert args(tokens=-1) == _lib.QL_ERR_BAD_SHAPE
    assert args(head_dim=60) == _lib.QL_ERR_BAD_SHAPE
    assert args(rotary_dim=72) == _lib.QL_ERR_BAD_SHAPE
    assert args(rotary_dim=12) == _lib.QL_ERR_BAD_SHAPE
    assert args(max_positions=0) == _lib.QL_ERR_BAD_SHAPE
    assert args(xh=-1) == _lib.QL_ERR_BAD_STRIDE
    assert args(dtype=_lib.QL_DTYPE_F32) == _lib.QL_ERR_UNSUPPORTED
    assert args(layout=2) == _lib.QL_ERR_UNSUPPORTED
    assert args(position_bytes=2) == _lib.QL_ERR_UNSUPPORTED
    assert args(table=72) == _lib.QL_ERR_UNSUPPORTED
    assert args(x=65) == _lib.QL_ERR_UNSUPPORTED
    assert lib.ql_rotary(None, None) == _lib.QL_ERR_NULL_POINTER


# ----------------------------------------------------------------------- GPU
def check(y, x, angles, layout, dtype, factor=1.0):
    """One rounding to the output's type; before it the table's two roundings,
    two products and a sum in fp32, 2^-24 each of |x1| + |x2| at most."""
    want = rotate(x.double(), angles, layout, factor)
    r = 2 * angles.shape[-1]
    size = x.double().abs()
    pair = size[..., :r].unflatten(-1, (2, r // 2)).sum(-2).repeat(1, 1, 2) if layout == "half" \
        else size[..., :r].unflatten(-1, (r // 2, 2)).sum(-1).repeat_interleave(2, -1)
    tol = HALF_ULP[dtype] * want.abs() + TINY[dtype]
    tol[..., :r] += 4 * 2.0 ** -24 * abs(factor) * pair
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(y.double() - want).abs().max():.3e}"
    assert torch.equal(y[..., r:], x[..., r:])


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,n,head_dim,rotary_dim", [
    (1, 14, 128, 128), (5, 3, 64, 64), (33, 2, 64, 16), (7, 5, 96, 48), (2, 33, 256, 64), (3, 1, 8, 8),
    (129, 4, 80, 40)])
def test_matches_definition(tokens, n, head_dim, rotary_dim, layout, dtype):
    x = heads(tokens, n, head_dim, dtype, tokens + n)
    positions = torch.randint(0, 5000, (tokens,), generator=torch.Generator().manual_seed(3)).cuda()
    rot = RotaryTable.build(rotary_dim, 5000, 1.0e4, layout)
    f, _ = rotary_frequencies(rotary_dim, 1.0e4)
    angles = positions.double()[:, None] * f.cuda()
    check(apply_rotary(x, positions, rot), x, angles, layout, dtype)
    check(apply_rotary(x, positions.int(), rot, inverse=True), x, -angles, layout, dtype)


@on_gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_alignment_and_in_place(layout):
    """Column slices of a fused projection, a transposed view, rows that do
    not start on 16 bytes, and out = x, all with the bits of the plain call."""
    rot = RotaryTable.build(64, 300, 1.0e4, layout)
    positions = torch.arange(40, 57).cuda()
    qkv = heads(17, 9, 128, torch.float16, 0)
    x = qkv[:, 2:6]
    want = apply_rotary(x.contiguous(), positions, rot)
    assert torch.equal(apply_rotary(x, positions, rot), want)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(apply_rotary(turned, positions, rot), want)
    odd = torch.empty(17 * 4 * 128 + 17 * 3 + 1, dtype=torch.float16, device="cuda")
    odd = odd.as_strided((17, 4, 128), (4 * 128 + 3, 128, 1), 1).copy_(x)
    assert torch.equal(apply_rotary(odd, positions, rot), want)
    out = torch.empty_like(odd)
    out = odd.clone(memory_format=torch.preserve_format)
    assert torch.equal(apply_rotary(odd, positions, rot, out=out), want)
    wide = torch.empty(17, 4, 256, dtype=torch.float16, device="cuda")[..., ::2].copy_(x)
    assert torch.equal(apply_rotary(wide, positions, rot), want)
    strided_positions = torch.stack([positions, positions], 1)[:, 0]
    assert torch.equal(apply_rotary(x, strided_positions, rot), want)
    kept = qkv.clone()
    apply_rotary(x, positions, rot, out=x)
    assert torch.equal(qkv[:, 2:6], want)
    assert torch.equal(qkv[:, :2], kept[:, :2]) and torch.equal(qkv[:, 6:], kept[:, 6:])


@on_gpu
def test_scaled_table_and_factor():
    s = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}
    rot = RotaryTable.build(128, 4096, 1.0e6, "half", s)
    f, factor = rotary_frequencies(128, 1.0e6, s)
    x = heads(9, 2, 128, torch.bfloat16, 1)
    positions = torch.tensor([0, 1, 2, 1023, 1024, 4095, 77, 4095, 0]).cuda()
    check(apply_rotary(x, positions, rot), x, positions.double()[:, None] * f.cuda(), "half", torch.bfloat16, factor)


@on_gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_gradient(layout):
    """The gradient of sum(w * rotate(x)) with respect to x is rotate back
    (w): against central differences of the float64 definition."""
    rot = RotaryTable.build(16, 64, 1.0e4, layout)
    positions = torch.tensor([3, 60]).cuda()
    angles = positions.double()[:, None] * rotary_frequencies(16, 1.0e4)[0].cuda()
    x, w = heads(2, 1, 24, torch.float16, 2), heads(2, 1, 24, torch.float16, 3)
    got = apply_rotary(w, positions, rot, inverse=True).double()
    h = 2.0 ** -10
    for i in range(24):
        step = torch.zeros(24, dtype=torch.float64, device="cuda")
        step[i] = h
        up, down = (rotate(x.double() + sign * step, angles, layout) for sign in (1, -1))
        slope = ((up - down) * w.double()).sum(-1) / (2 * h)
        # linear, so differences are exact to float64; the kernel rounds once (and in fp32 before)
        assert bool(((got[..., i] - slope).abs() <= 2.0 ** -11 * slope.abs() + 2.0 ** -20 * 16).all())


@on_gpu
def test_there_and_back():
    """The inverse undoes the call without a factor; with one (yarn) there and back is its square times x."""
    x = heads(9, 3, 64, torch.float16, 9)
    positions = torch.arange(100, 109).cuda()
    for scaling in (None, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}):
        rot = RotaryTable.build(64, 256, 1.0e4, "half", scaling)
        factor = rotary_frequencies(64, 1.0e4, scaling)[1]
        assert (factor > 1.1) == (scaling is not None)
        back = apply_rotary(apply_rotary(x, positions, rot), positions, rot, inverse=True).double()
        pair = factor * x.double().abs().unflatten(-1, (2, 32)).sum(-2).repeat(1, 1, 2)
        # rounded to fp16 there (2^-11 of |x1| + |x2|, which both of the pair take back) and back again
        assert bool(((back - factor ** 2 * x.double()).abs() <= 3 * 2.0 ** -11 * factor * pair + 2.0 ** -22).all())


@on_gpu
def test_infinities_and_nan_stay_in_their_pairs():
    rot = RotaryTable.build(64, 8, 1.0e4)
    x = heads(1, 2, 64, torch.float16, 5)
    x[0, 0, 3], x[0, 1, 40] = math.inf, math.nan
    y = apply_rotary(x, torch.tensor([5]).cuda(), rot)
    bad = ~torch.isfinite(y)
    assert set(bad[0, 0].nonzero().flatten().tolist()) == {3, 35}
    assert set(bad[0, 1].nonzero().flatten().tolist()) == {8, 40}


@on_gpu
def test_positions_outside_the_table_are_recorded():
    rot = RotaryTable.build(64, 8, 1.0e4)
    x = heads(3, 1, 64, torch.float16, 6)
    _lib.clear_device_error()
    y = apply_rotary(x, torch.tensor([-1, 8, 3]).cuda(), rot)
    assert _lib.device_error() == _lib.QL_DEVICE_ERROR_BAD_INDEX
    _lib.clear_device_error()
    assert torch.equal(y, apply_rotary(x, torch.tensor([0, 7, 3]).cuda(), rot))
    assert _lib.device_error() == 0


@on_gpu
def test_empty_and_refusals():
    rot = RotaryTable.build(64, 8, 1.0e4)
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    x = heads(2, 3, 64, torch.float16, 7)
    assert apply_rotary(x[:0], pos[:0], rot).shape == (0, 3, 64)
    assert apply_rotary(x[:, :0], pos, rot).shape == (2, 0, 64)
    with pytest.raises(TypeError):
        apply_rotary(x.float(), pos, rot)
    with pytest.raises(TypeError):
        apply_rotary(x, pos.float(), rot)
    with pytest.raises(AssertionError):
        apply_rotary(x, pos[:1], rot)
    with pytest.raises(AssertionError):
        apply_rotary(x, pos.cpu(), rot)
    with pytest.raises(AssertionError):
        apply_rotary(x[..., :32], pos, rot)
    with pytest.raises(AssertionError):
        apply_rotary(x, pos, rot, out=torch.empty(2, 3, 64, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(AssertionError):
        apply_rotary(x.cpu(), pos, rot)


@on_gpu
def test_on_another_stream_and_in_a_graph():
    rot = RotaryTable.build(128, 64, 1.0e4)
    x = heads(6, 14, 128, torch.float16, 8)
    pos = torch.arange(6).cuda()
    want = apply_rotary(x, pos, rot)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(apply_rotary(x, pos, rot), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = apply_rotary(x, pos, rot)
    torch.cuda.current_stream().wait_stream(s)
    pos += 3
    graph.replay()
    assert torch.equal(out, apply_rotary(x, pos, rot))
