"""Drawing tokens (ql_sample_tokens) against the definition in float64, row by row: every filter alone and together,
ties, hidden and infinite logits, all types, vocabularies from one token on, strides; refusals.

The draw is decided between sums that are right to 2^-45 or so of themselves (or far enough apart), so a row is decided
otherwise than in float64 with a chance of some 2^-28 over a large vocabulary: none here.  Log-probabilities are rounded to
fp32 (2^-24); the sum that they are taken of may be one of fp32 weights, 2^-19.5 off at most, which enters the log as it is."""
import math

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.sampling import sample_tokens

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def plain_row(x, u, heat, top_k, top_p, min_p):
    """Token and log-probability of one row, x float64 on the CPU."""
    x = torch.where(x.isnan(), torch.tensor(-math.inf, dtype=torch.float64), x)
    seen = torch.nonzero(x > -math.inf).squeeze(1)
    if len(seen) == 0:
        return -1, -math.inf
    order = seen[torch.argsort(-x[seen], stable=True)]
    most = x[order[0]]
    if not heat > 0:
        return int(order[0]), 0.0
    if most == math.inf:
        order, w = order[x[order] == most], torch.ones(int((x == most).sum()), dtype=torch.float64)
    else:
        a = (x[order] - most) / heat
        w = torch.where(a < -700, torch.zeros_like(a), a.exp())
    if 0 < top_k < len(order):
        order, w = order[:top_k], w[:top_k]
    kept = torch.ones(len(order), dtype=torch.bool)
    if top_p < 1:
        kept &= w.cumsum(0) - w < top_p * w.sum()
    if min_p > 0:
        kept &= w >= min_p
    kept[0] = True
    by_index, place = order[kept].sort()
    w = w[kept][place]
    sums = w.cumsum(0)
    u = min(max(0.0 if math.isnan(u) else u, 0.0), 1.0)
    i = int((sums <= u * sums[-1]).sum())
    i = min(i, int(torch.nonzero(w > 0).max()))
    return int(by_index[i]), float((w[i] / sums[-1]).log())


def setting(v, r):
    return float(v[r]) if isinstance(v, torch.Tensor) else 0 if v is None else v


def agree(logits, uniform, **settings):
    ids, logprobs = sample_tokens(logits, uniform, return_logprobs=True, **settings)
    x, u = logits.double().cpu(), uniform.double().cpu()
    s = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0} | {k: v for k, v in settings.items() if v is not None}
    s = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    want = [plain_row(x[r], float(u[r]), setting(s["temperature"], r), int(setting(s["top_k"], r)), setting(s["top_p"], r),
                      setting(s["min_p"], r)) for r in range(len(x))]
    assert ids.tolist() == [i for i, _ in want]
    chance = torch.tensor([c for _, c in want], dtype=torch.float64)
    got = logprobs.double().cpu()
    assert torch.equal(got == -math.inf, chance == -math.inf)
    fine = chance > -math.inf
    assert ((got - chance)[fine].abs() <= 2.0 ** -24 * chance[fine].abs() + 2.0 ** -19.5).all()
    assert torch.equal(ids, sample_tokens(logits, uniform, **settings))
    return ids


def rows_of(rows, vocab, dtype, seed, std=2.5, lift=9.0):
    g = torch.Generator().manual_seed(seed)
    x = std * torch.randn(rows, vocab, generator=g)
    n = min(vocab, 12)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, n), generator=g), lift * torch.rand(rows, n, generator=g))
    return x.to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


TYPES = [torch.float16, torch.bfloat16, torch.float32]
FILTERS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=3, top_p=0.6), dict(top_p=0.9), dict(top_p=0.0),
           dict(min_p=0.02), dict(min_p=1.0), dict(temperature=0.6, top_k=40, top_p=0.95, min_p=0.01),
           dict(temperature=1.7, top_p=0.99), dict(temperature=0), dict(top_k=10 ** 9), dict(temperature=1e-3, top_p=0.5)]


# ----------------------------------------------------------------------- CPU
def test_host_checks_without_gpu():
    lib = _lib.load()

    def call(**change):
        f = dict(logits=64, uniform=64, temperature=0, top_k=0, top_p=0, min_p=0, ids=64, logprobs=0, rows=2, vocab=100,
                 stride=100, dtype=_lib.QL_DTYPE_F16, k=0, t=1.0, p=1.0, m=0.0, flags=0)
        f.update(change)
        return lib.ql_sample_tokens(_lib.SAMPLE_TOKENS_ARGS.pack(*f.values()), None)

    assert call(rows=0, logits=0) == _lib.QL_OK
    for name in ("logits", "uniform", "ids"):
        assert call(**{name: 0}) == _lib.QL_ERR_NULL_POINTER, name
    for change in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 21) + 1), dict(rows=1 << 28)):
        assert call(**change) == _lib.QL_ERR_BAD_SHAPE, change
    assert call(stride=99) == _lib.QL_ERR_BAD_STRIDE
    for change in (dict(dtype=5), dict(logits=65), dict(uniform=66), dict(temperature=66), dict(top_k=66), dict(top_p=66),
                   dict(min_p=66), dict(ids=68), dict(logprobs=66)):
        assert call(**change) == _lib.QL_ERR_UNSUPPORTED, change
    assert lib.ql_sample_tokens(None, None) == _lib.QL_ERR_NULL_POINTER


def test_refusals_on_cpu():
    with pytest.raises(AssertionError, match="CUDA"):
        sample_tokens(torch.zeros(2, 5), torch.zeros(2))


def test_the_plain_row():
    x = torch.tensor([0.0, 2.0, 1.0, 2.0, -math.inf, math.nan], dtype=torch.float64)
    assert plain_row(x, 0.0, 0.0, 0, 1.0, 0.0) == (1, 0.0)
    assert plain_row(x, 0.999, 1.0, 1, 1.0, 0.0) == (1, 0.0)
    assert plain_row(x, 0.5, 1.0, 2, 1.0, 0.0) == (3, math.log(0.5))
    assert plain_row(x, 0.0, 1.0, 0, 1.0, 0.0)[0] == 0


# ----------------------------------------------------------------------- GPU
@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", range(len(FILTERS)))
def test_filters(dtype, filters):
    for vocab in (1, 2, 7, 1000, 4097, 32003):
        logits, uniform = rows_of(9, vocab, dtype, 100 * filters + vocab)
        agree(logits, uniform, **FILTERS[filters])


@on_gpu
@pytest.mark.parametrize("dtype,rows,vocab", [(torch.float16, 3, 151936), (torch.bfloat16, 70, 128256), (torch.float32, 4, 151936),
                                              (torch.float16, 2, 200003), (torch.float32, 2, 262144)])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=50, top_p=0.9), dict(temperature=1.5, top_p=0.95), dict(top_k=30000, top_p=0.8)])
def test_large_vocabularies(dtype, rows, vocab, filters):
    logits, uniform = rows_of(rows, vocab, dtype, rows + vocab)
    agree(logits, uniform, **filters)


@on_gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_vocabularies_past_the_registers(dtype):
    logits, uniform = rows_of(2, 1 << 20, dtype, 5)
    agree(logits, uniform, top_p=0.7)
    agree(logits, uniform, top_k=1000, min_p=0.001)
    logits, uniform = rows_of(1, 1 << 21, dtype, 6)
    agree(logits, uniform)


MANY = {
    "spread": lambda g, n: 2.2 * torch.randn(n, generator=g),
    "even": lambda g, n: torch.rand(n, generator=g),                                  # thousands within a small step
    "steps": lambda g, n: torch.randint(0, 6, (n,), generator=g).float(),             # thousands of each value
    "two heaps": lambda g, n: torch.where(torch.rand(n, generator=g) < 0.1, 5.0, -9.0) + 0.3 * torch.randn(n, generator=g),
    "long": lambda g, n: 40.0 * torch.rand(n, generator=g) - 1000.0,                  # all of 58 octaves alike
    "one above": lambda g, n: torch.cat([torch.tensor([60000.0]), 59990.0 + 0.0 * torch.randn(n - 1, generator=g)]),
}


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", MANY)
def test_many_tokens_kept(dtype, kind):
    """top-p's border among thousands of tokens: near its ends, behind top-k, of a large vocabulary and of a part of it."""
    g = torch.Generator().manual_seed(71)
    for vocab in (2500, 50021) + ((151936,) if kind == "spread" else ()):
        x = torch.stack([MANY[kind](g, vocab) for _ in range(3)])
        x[1, torch.rand(vocab, generator=g) < 0.5] = -math.inf
        x, u = x.to(dtype).cuda(), torch.rand(3, generator=g).cuda()
        for f in (dict(top_p=0.3), dict(top_p=0.9, temperature=1.3), dict(top_p=0.99, temperature=0.6), dict(top_p=0.99999),
                  dict(top_p=0.9, top_k=2000), dict(top_p=0.97, min_p=1e-3), dict(top_p=1e-6)):
            agree(x, u, **f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_settings_of_each_row(dtype):
    rows = 40
    logits, uniform = rows_of(rows, 5003, dtype, 7)
    g = torch.Generator().manual_seed(8)
    heat = torch.where(torch.arange(rows) % 7 == 3, 0.0, 0.3 + 1.5 * torch.rand(rows, generator=g)).cuda()
    heat[5], heat[6] = -1.0, math.nan                      # greedy, as 0
    top_k = torch.randint(-2, 300, (rows,), generator=g, dtype=torch.int32).cuda()
    top_p = (1.2 * torch.rand(rows, generator=g)).cuda()
    min_p = (0.2 * torch.rand(rows, generator=g) - 0.05).cuda()
    top_p[2], min_p[3], top_k[4] = math.nan, math.nan, 2 ** 31 - 1
    want = agree(logits, uniform, temperature=heat, top_k=top_k, top_p=torch.where(top_p.isnan(), 1.0, top_p),
                 min_p=torch.where(min_p.isnan(), 0.0, min_p))
    assert torch.equal(want, sample_tokens(logits, uniform, temperature=heat, top_k=top_k, top_p=top_p, min_p=min_p))
    twice = lambda t: torch.stack([t, t], 1)[:, 0]         # noqa: E731 - strided settings
    assert torch.equal(want, sample_tokens(logits, twice(uniform), temperature=twice(heat), top_k=twice(top_k),
                                           top_p=twice(top_p), min_p=twice(min_p)))


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_ties(dtype):
    """Rows of few values, and of one: what is kept ends among equal tokens, whose lowest indices count."""
    g = torch.Generator().manual_seed(9)
    x = torch.randint(-3, 3, (24, 9001), generator=g).float()
    x[0] = 1.5
    x[1] = 0.0
    x[1, ::2] = -0.0
    logits, uniform = x.to(dtype).cuda(), torch.rand(24, generator=g).cuda()
    for f in (dict(), dict(top_k=1), dict(top_k=700), dict(top_k=5000), dict(top_p=0.3), dict(top_k=2000, top_p=0.5),
              dict(top_k=3000, top_p=0.9), dict(min_p=0.3), dict(temperature=0), dict(temperature=100.0, top_p=0.7)):
        agree(logits, uniform, **f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_hidden_and_infinite(dtype):
    logits, uniform = rows_of(12, 3001, dtype, 10)
    logits[0] = -math.inf                                  # nothing to draw
    logits[1] = math.nan
    logits[2, 1:] = -math.inf                              # one token
    logits[3, ::3] = math.nan
    logits[4, 100:2900] = -math.inf
    logits[5, 7] = math.inf                                # only the infinite ones
    logits[6, [5, 2000, 2999]] = math.inf
    logits[7] = torch.finfo(dtype).min                     # the type's lowest value is a value
    logits[8, 17] = torch.finfo(dtype).max
    logits[9, :3000] = torch.finfo(dtype).min
    logits[10, ::2] = -math.inf
    for f in FILTERS + [dict(top_k=2), dict(top_k=2, top_p=0.4)]:
        agree(logits, uniform, **f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_temperatures_at_the_ends(dtype):
    """So cold that only the largest have a weight, so hot that all have nearly the same; fp32's smallest and infinity."""
    logits, uniform = rows_of(10, 4099, dtype, 15)
    logits[3, [7, 4000]] = 30.0                            # two largest
    for heat in (1e-45, 1e-38, 1e-30, 1e-12, 1e-4, 50.0, 1e6, 1e30, 3e38):
        heats = torch.full((10,), heat, device="cuda")
        for f in (dict(), dict(top_p=0.5), dict(top_k=20, top_p=0.9), dict(min_p=0.5)):
            agree(logits, uniform, temperature=heats, **f)
    hot = torch.full((10,), math.inf, device="cuda")       # all alike
    assert torch.equal(sample_tokens(logits, uniform, temperature=hot), (uniform.double() * 4099).long())


@on_gpu
def test_temperatures_of_64_bits():
    """Numbers, not tensors: down to those whose inverse is no number, and up to the largest."""
    logits, uniform = rows_of(6, 4099, torch.float32, 16)
    logits[3, [7, 4000]] = 30.0
    for heat in (5e-324, 1e-310, 1e-308, 1e-250, 1e-199, 1e-100):
        for f in (dict(), dict(top_p=0.5), dict(top_k=20, top_p=0.9), dict(min_p=0.5)):
            ids, logprobs = sample_tokens(logits, uniform, heat, return_logprobs=True, **f)
            want = sample_tokens(logits, uniform, 0.0)
            if f.get("top_p") != 0.5 and uniform[3] >= 0.5:          # the second of two
                want[3] = 4000
            assert torch.equal(ids, want)
            chance = torch.zeros(6, device="cuda")
            if f.get("top_p") != 0.5:
                chance[3] = -math.log(2.0)
            assert torch.allclose(logprobs, chance, rtol=2.0 ** -19, atol=0)
    for heat in (1e300, 1.7e308):                                    # all alike
        assert torch.equal(sample_tokens(logits, uniform, heat), (uniform.double() * 4099).long())


@on_gpu
def test_random_numbers_at_the_ends():
    logits, _ = rows_of(6, 5000, torch.float16, 11)
    logits[:, 0] = -math.inf
    uniform = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -149, 1.0, -0.5, math.nan], device="cuda")
    for f in (dict(), dict(top_k=20), dict(top_p=0.5)):
        agree(logits, uniform, **f)


@on_gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    wide, uniform = rows_of(5, 3100, dtype, 12)
    want = sample_tokens(wide[:, 1:3002].contiguous(), uniform, top_p=0.9)
    assert torch.equal(sample_tokens(wide[:, 1:3002], uniform, top_p=0.9), want)                  # odd start
    assert torch.equal(sample_tokens(wide[:, 1:3002].t().contiguous().t(), uniform, top_p=0.9), want)   # columns first
    assert torch.equal(sample_tokens(wide[:1, 1:3002].expand(5, 3001), uniform, top_p=0.9)[:1], want[:1])
    out = torch.full((5,), -7, device="cuda")
    assert sample_tokens(wide[:, 1:3002], uniform, top_p=0.9, out=out) is out and torch.equal(out, want)
    assert sample_tokens(wide[:0], uniform[:0]).shape == (0,)


@on_gpu
def test_what_is_drawn_follows_the_weights():
    """Evenly spaced random numbers: each token is drawn as often as its chance says, to within one."""
    n, vocab = 4096, 11
    x = torch.linspace(0, 3, vocab).half().cuda()
    uniform = (torch.arange(n, device="cuda") + 0.5) / n
    ids = sample_tokens(x.expand(n, vocab).contiguous(), uniform, temperature=0.8)
    p = torch.softmax(x.double() / 0.8, 0)
    assert ((torch.bincount(ids, minlength=vocab) - n * p).abs() <= 1).all()


@on_gpu
def test_streams_and_graphs():
    logits, uniform = rows_of(8, 151936, torch.float16, 13)
    more, others = rows_of(8, 151936, torch.float16, 14)
    want = sample_tokens(logits, uniform, top_k=50, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [sample_tokens(logits, uniform, top_k=50, top_p=0.9) for _ in range(4)]
    beside = [sample_tokens(more, others, top_p=0.9) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got) and all(torch.equal(b, beside[0]) for b in beside)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(logits, uniform, top_k=50, top_p=0.9)
    logits.copy_(more)
    uniform.copy_(others)
    graph.replay()
    assert torch.equal(out, sample_tokens(more, others, top_k=50, top_p=0.9))


@on_gpu
def test_refusals():
    x, u = torch.zeros(3, 8, device="cuda"), torch.zeros(3, device="cuda")
    with pytest.raises(TypeError, match="logits"):
        sample_tokens(x.double(), u)
    with pytest.raises(TypeError, match="uniform"):
        sample_tokens(x, u.double())
    with pytest.raises(AssertionError, match="uniform"):
        sample_tokens(x, u[:2])
    with pytest.raises(AssertionError, match="logits"):
        sample_tokens(x[0], u)
    with pytest.raises(AssertionError, match="vocab"):
        sample_tokens(x[:, :0], u)
    with pytest.raises(TypeError, match="top_k"):
        sample_tokens(x, u, top_k=torch.ones(3, device="cuda"))
    with pytest.raises(AssertionError, match="top_p"):
        sample_tokens(x, u, top_p=torch.ones(2, device="cuda"))
    with pytest.raises(AssertionError, match="min_p"):
        sample_tokens(x, u, min_p=torch.ones(3))
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_p=-0.1), dict(min_p=1.5),
                dict(top_p=math.nan)):
        with pytest.raises(ValueError):
            sample_tokens(x, u, **bad)
    with pytest.raises(TypeError, match="whole number"):
        sample_tokens(x, u, top_k=2.0)
    with pytest.raises(AssertionError, match="out"):
        sample_tokens(x, u, out=torch.zeros(3, dtype=torch.int32, device="cuda"))
