"""Plain forms of the attention-side operators, for the tests: the quantiser
elementwise in fp32 (whose codes the kernels must reproduce bit for bit) and
everything else in float64 from the definitions."""
from __future__ import annotations

import math

import torch

# unit roundoff: half of the spacing above 1 (2^-11 for fp16's 11 significant bits, 2^-8 for bf16's 8)
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def heads(tokens, n, head_dim, dtype, seed, device="cuda", std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = std * torch.randn(tokens, n, head_dim, generator=g) * torch.exp(0.5 * torch.randn(n, head_dim, generator=g))
    return x.to(dtype).to(device)


def rotate(x, angles, layout, factor=1.0):
    """x (tokens, heads, head_dim) turned by angles (tokens, pairs), in x's
    dtype, every product and sum rounded on its own."""
    cos, sin = (angles.cos() * factor)[:, None], (angles.sin() * factor)[:, None]
    return rotate_by(x, cos, sin, layout)


def rotate_by(x, cos, sin, layout):
    r = 2 * cos.shape[-1]
    y = x.clone()
    if layout == "half":
        one, two = slice(0, r // 2), slice(r // 2, r)
    else:
        one, two = slice(0, r, 2), slice(1, r, 2)
    y[..., one] = x[..., one] * cos - x[..., two] * sin
    y[..., two] = x[..., two] * cos + x[..., one] * sin
    return y


def quantise(x, bits):
    """fp32 rows (..., head_dim) -> integer codes (..., head_dim) and bf16 scales (..., groups)."""
    top, span = (127.0, x.shape[-1]) if bits == 8 else (7.0, 64)
    g = x.unflatten(-1, (-1, span))
    scales = (g.abs().amax(-1) * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)).to(torch.bfloat16)
    s = scales.float().unsqueeze(-1)
    fine = (s > 0) & (s < math.inf)
    q = torch.where(fine, torch.round(g / s), torch.zeros_like(g)).clamp(-top, top)
    return q.flatten(-2).to(torch.int32), scales


def pack(codes, bits):
    if bits == 8:
        return codes.to(torch.int8)
    u = (codes + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def values(codes, scales, bits):
    """float64 values of stored codes (..., row bytes) and scales."""
    if bits == 8:
        q = codes.double()
    else:
        q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).double() - 8
    return (q.unflatten(-1, (scales.shape[-1], -1)) * scales.double().unsqueeze(-1)).flatten(-2)


def random_cache(num_pages, page_size, kv_heads, head_dim, bits, seed, std_v=0.7):
    """A pool of quantised normal rows, as the cache's constructor takes it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ts = []
    for std in (1.0, std_v):
        x = std * torch.randn(num_pages, kv_heads, page_size, head_dim, generator=g, device="cuda")
        codes, scales = quantise(x, bits)
        ts += [pack(codes, bits), scales]
    return ts


def visible(q_len, kv_len, mask_rows, device="cuda"):
    """(q_len, kv_len) truth values; mask_rows (q_len, words) int64 or None."""
    j = torch.arange(kv_len, device=device)
    d = j - (kv_len - q_len)
    if mask_rows is None:
        return d[None] <= torch.arange(q_len, device=device)[:, None]
    words = mask_rows.shape[1]
    bit = (mask_rows[:, (d.clamp(0, 64 * words - 1) // 64)] >> (d.clamp(min=0) % 64)) & 1
    return (d < 0)[None] | ((bit == 1) & (d < 64 * words)[None])


def attend(q, k, v, sees, scale):
    """One request in float64: q (t, hq, d), k and v (n, hk, d), sees (t, n).
    Returns out (t, hq, d), lse (t, hq), and for the error bound the sums of
    p |v| like out and the largest scale * sum |q k| like lse."""
    t, hq, d = q.shape
    n, hk = k.shape[:2]
    if n == 0:
        zero = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
        low = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
        return zero, low, zero, torch.zeros_like(low)
    qg = q.double().unflatten(1, (hk, hq // hk))
    s = torch.einsum("thgd,nhd->thgn", qg, k) * scale
    size = torch.einsum("thgd,nhd->thgn", qg.abs(), k.abs()) * abs(scale)
    s = s.masked_fill(~sees[:, None, None], -math.inf)
    size = size.masked_fill(~sees[:, None, None], 0.0)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse.unsqueeze(-1) > -math.inf, torch.exp(s - lse.unsqueeze(-1)), torch.zeros_like(s))
    p = torch.where(sees[:, None, None], p, torch.zeros_like(p))
    vv = torch.where(sees.any(0)[:, None, None], v, torch.zeros_like(v))
    out = torch.einsum("thgn,nhd->thgd", p, vv).flatten(1, 2)
    mass = torch.einsum("thgn,nhd->thgd", p, vv.abs()).flatten(1, 2)
    return out, lse.flatten(1, 2), mass, size.amax(-1).flatten(1, 2)


def attention_bounds(out, lse, mass, size, dtype):
    """How far a kernel may be from float64.  The output is rounded once to
    its type.  Before that: the weights p * scale_v are rounded to fp16 for the
    matrix product (2^-11 each at most, so 2^-11 of the sum of p |v|), and a
    score, a sum of head_dim fp32 products, is off by about sqrt(256) * 2^-24 =
    2^-20 of the sum of its products' sizes, which doubles in p (numerator and
    denominator) and enters lse once; exponentials and sums in fp32 add a few
    2^-24, taken as 2^-20."""
    tol = HALF_ULP[dtype] * out.abs() + TINY[dtype] + \
        (2.0 ** -11 + 2.0 ** -19 * size.unsqueeze(-1) + 2.0 ** -20) * mass
    tol_lse = 2.0 ** -20 * (size + 1.0 + lse.abs().nan_to_num(posinf=0.0))
    return tol, tol_lse
