"""Attention at the ends of the range: scores very far apart, value scales of
very different sizes, queries with a few large elements; each kernel forced."""
import sys

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.tree_attention import tree_attention

from attn_helpers import HALF_ULP, values
from test_tree_attention import Problem

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


@pytest.fixture(autouse=True, params=["tensor cores", "streaming"])
def family(request, monkeypatch):
    force = _lib.QL_FLAG_FORCE_GEMM if request.param == "tensor cores" else _lib.QL_FLAG_FORCE_GEMV
    monkeypatch.setattr(sys.modules[tree_attention.__module__], "call_flags", lambda: _lib.QL_FLAG_PDL | force)
    return request.param


def cached(p, b):
    """Keys and values of request b in float64, [positions, heads, head_dim]."""
    c, n = p.cache, p.lens[b]
    pages = p.table[b, :-(-n // c.page_size)].long()
    return [values(x[pages], s[pages], p.bits).transpose(1, 2).flatten(0, 1)[:n]
            for x, s in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales))]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("scale", [1.0e5, -3.0e7])
def test_scores_that_pass_one_another_by_millions(scale, bits, dtype):
    """The softmax picks one position: its value, rounded once.  A score is off by 2^-20 of the sum of its products'
    sizes at most (attention_bounds), so a winner that leads by 8 times that and 20 more is the kernel's too, and what
    the others weigh, e^-20 each of 1500, is under 2^-18 of the value scales' largest."""
    p = Problem([5, 40], [700, 1500], 12, 2, 128, bits, 16, dtype, seed=31)
    out, _ = p.run(scale=scale)
    assert bool(torch.isfinite(out).all())
    at = checked = 0
    for b, (t, n) in enumerate(zip(p.q_lens, p.lens)):
        k, v = cached(p, b)
        q = p.q[at:at + t].double().unflatten(1, (2, 6))
        s = torch.einsum("thgd,nhd->thgn", q, k) * scale
        size = torch.einsum("thgd,nhd->thgn", q.abs(), k.abs()).amax(-1) * abs(scale)
        see = torch.arange(n, device="cuda")[None] <= torch.arange(n - t, n, device="cuda")[:, None]
        two, who = s.masked_fill(~see[:, None, None], -torch.inf).topk(2, dim=-1)
        sure = two[..., 0] - two[..., 1] > 8 * 2.0 ** -20 * size + 20
        want = v[who[..., 0], torch.arange(2, device="cuda")[None, :, None]]
        tol = HALF_ULP[dtype] * want.abs() + 2.0 ** -18 * v.abs().max() + 2.0 ** -11 * want.abs()
        off = (out[at:at + t].double().unflatten(1, (2, 6)) - want).abs()
        assert bool((off <= tol).all(-1)[sure].all())
        checked += int(sure.sum())
        at += t
    assert checked > 0.9 * sum(p.q_lens) * 12


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("low,high", [(-70, 100), (-20, 110), (-100, 10)])
def test_value_scales_from_one_end_to_the_other(low, high, q_len, bits):
    """bf16 values near the least and then near the greatest: all positions count in the softmax's sum."""
    p = Problem([q_len], [900], 4, 2, 128, bits, 16, torch.bfloat16, seed=32)
    c = p.cache
    for j in range(900):
        c.v_scales[p.table[0, j // 16].long(), :, j % 16] *= 2.0 ** (low if j < 500 else high)
    p.check(p.run())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("kind,large,down", [("spread", 8, 20), ("first", 8, 20), ("late", 8, 20), ("late", 13, 24),
                                             ("unseen", 8, 20)])
def test_fp16_values_far_below_the_largest(kind, large, down, q_len, bits):
    """Value scales from 2^-20 to 1 of the largest, at random; and one position that takes nearly all of every row's
    weight and holds values 2^-20 or 2^-24 as large as the others': the first one, a late one, and beside large values that
    most rows do not see (the new tokens' own)."""
    n = 900
    p = Problem([q_len], [n], 4, 2, 128, bits, 16, torch.float16, seed=33)
    c = p.cache
    g = torch.Generator().manual_seed(34)

    def row(t, j):
        return t[p.table[0, j // 16].long(), :, j % 16]

    if kind == "spread":
        for j in range(n):
            row(c.v_scales, j).mul_(2.0 ** (large - down * float(torch.rand((), generator=g))))
        p.check(p.run())
        return
    for j in range(n):
        row(c.v_scales, j).mul_(2.0 ** large)
    at = {"first": 3, "late": 777, "unseen": 3}[kind]
    # q and the key at `at` have one sign, so that its score leads by far: about 70 beside 1.5 a standard deviation
    p.q.abs_()
    row(c.k_codes, at).fill_(100 if bits == 8 else 0xEE)
    row(c.k_scales, at).fill_(0.05 if bits == 8 else 0.8)
    row(c.v_scales, at).mul_(2.0 ** -down)
    if kind == "unseen":
        for j in range(n - q_len, n):
            row(c.v_scales, j).mul_(64.0)
        for j in range(n - q_len):
            if j != at:
                row(c.v_scales, j).mul_(2.0 ** -down)
    out, lse = p.run()
    p.check((out, lse))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("up", [12, 20])
def test_bf16_queries_with_a_few_large_elements(up, q_len, bits):
    """Two elements of every query 2^up times the others', where keys are zero: the others' bits decide.  (Elements keep
    theirs down to 2^-32 of the largest, and the others are normal variates, some of them 2^-10 of their deviation.)"""
    p = Problem([q_len], [700], 4, 2, 128, bits, 16, torch.bfloat16, seed=35)
    for at in (3, 70):
        p.q[..., at] *= 2.0 ** up
        if bits == 8:
            p.cache.k_codes[..., at] = 0
        else:
            byte, other = p.cache.k_codes[..., at // 2], 0x0F if at % 2 else 0xF0
            byte.copy_((byte & other) | (0x88 & ~other & 0xFF))
    p.check(p.run())
