"""Page tables and slots from request lengths (ql_plan_step) against an allocator written out request by request:
growth, cuts, exhausted pools, full rows and full steps; that pages are neither lost nor held twice; refusals."""
import random

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.paging import PageTables, StepPlan, plan_step

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


class Plain:
    """The same rules with lists: `free` is a stack whose end is its top."""

    def __init__(self, batch, width, num_pages, page):
        self.width, self.page = width, page
        self.held, self.lens, self.free = [[] for _ in range(batch)], [0] * batch, list(range(num_pages - 1, -1, -1))

    def step(self, new, max_tokens, keep=None):
        page, up = self.page, lambda n: -(-n // self.page)
        new = [max(n, 0) for n in new]
        keep = list(self.lens) if keep is None else [min(max(k, 0), n) for k, n in zip(keep, self.lens)]
        back = []
        for b, k in enumerate(keep):
            back += self.held[b][up(k):]
            self.held[b] = self.held[b][:up(k)]
        self.free += reversed(back)
        cu, slots, positions, refused, tokens, pages, available = [0], [], [], 0, 0, 0, len(self.free)
        for b, (k, n) in enumerate(zip(keep, new)):
            fits, grow = up(k + n) <= self.width, up(k + n) - up(k)
            tokens += n if fits else 0
            pages += grow if fits else 0
            if fits and tokens <= max_tokens and (grow == 0 or pages <= available):
                self.held[b] += [self.free.pop() for _ in range(grow)]
            else:
                refused += n > 0
                n = 0
            self.lens[b] = k + n
            positions += range(k, k + n)
            slots += [self.held[b][t // page] * page + t % page for t in range(k, k + n)]
            cu.append(len(slots))
        return cu, slots, positions, refused


def agree(pages, plan, plain, want, max_tokens):
    cu, slots, positions, refused = want
    pad = max_tokens - len(slots)
    assert plan.cu_q.tolist() == cu and int(plan.refused) == refused
    assert plan.slots.tolist() == slots + [-1] * pad and plan.positions.tolist() == positions + [0] * pad
    assert pages.lens.tolist() == plain.lens and plan.kv_lens is pages.lens
    n = int(pages.free_count)
    assert pages.free_pages[:n].tolist() == plain.free
    table = pages.page_table.cpu()
    for b, held in enumerate(plain.held):
        assert table[b, :len(held)].tolist() == held
    every = [x for h in plain.held for x in h] + plain.free
    assert sorted(every) == list(range(pages.num_pages))


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------------- CPU
def test_host_checks_without_gpu():
    lib = _lib.load()

    def call(**change):
        f = dict(table=64, lens=64, free=64, count=64, keep=0, fresh=64, cu=64, slots=64, positions=64, refused=64,
                 batch=2, width=4, stride=4, pages=8, page=16, max_tokens=8, flags=0)
        f.update(change)
        return lib.ql_plan_step(_lib.PLAN_STEP_ARGS.pack(*f.values()), None)

    for name in ("table", "lens", "free", "count", "fresh", "cu", "slots", "positions", "refused"):
        assert call(**{name: 0}) == _lib.QL_ERR_NULL_POINTER, name
    for name in ("table", "lens", "free", "count", "keep", "fresh", "cu", "refused"):
        assert call(**{name: 66}) == _lib.QL_ERR_UNSUPPORTED, name
    assert call(slots=72) == call(positions=72) == _lib.QL_ERR_UNSUPPORTED
    assert call(page=24) == call(page=0) == call(page=131072) == _lib.QL_ERR_UNSUPPORTED
    assert call(stride=3) == _lib.QL_ERR_BAD_STRIDE
    for change in (dict(batch=-1), dict(batch=8193), dict(width=-1, stride=4), dict(pages=-1), dict(pages=1 << 31),
                   dict(max_tokens=-1), dict(max_tokens=1 << 31), dict(batch=8192, width=1 << 18, stride=1 << 18)):
        assert call(**change) == _lib.QL_ERR_BAD_SHAPE, change
    assert lib.ql_plan_step(None, None) == _lib.QL_ERR_NULL_POINTER


def test_refusals_on_cpu():
    tables = PageTables.empty(3, 4, 8, 16, device="cpu")
    assert tables.free_pages.tolist() == list(range(7, -1, -1)) and int(tables.free_count) == 8
    with pytest.raises(AssertionError, match="cpu"):
        plan_step(tables, torch.zeros(3, dtype=torch.int32), 8)
    ts = (tables.page_table, tables.lens, tables.free_pages, tables.free_count)
    with pytest.raises(ValueError, match="power of two"):
        PageTables(*ts, 24)
    with pytest.raises(TypeError, match="lens"):
        PageTables(ts[0], ts[1].long(), *ts[2:], 16)
    with pytest.raises(AssertionError):
        PageTables(ts[0], ts[1][:2], *ts[2:], 16)
    with pytest.raises(AssertionError, match="apart"):
        PageTables(ts[0][:1].expand(3, 4), *ts[1:], 16)
    with pytest.raises(AssertionError, match="free_count"):
        PageTables(*ts[:3], ts[1], 16)
    with pytest.raises(ValueError, match="8192"):
        PageTables.empty(8193, 1, 1, 16, device="cpu")


# ----------------------------------------------------------------------- GPU
@on_gpu
@pytest.mark.parametrize("batch,width,num_pages,page,max_tokens,seed", [
    (1, 8, 8, 16, 64, 0),
    (3, 5, 9, 4, 17, 1),                 # a pool and a step that are often too small
    (64, 12, 300, 16, 512, 2),
    (33, 40, 2000, 1, 900, 3),           # a page a token
    (1025, 6, 3000, 32, 6000, 4),        # more requests than threads, several CTAs
    (2500, 3, 4000, 8, 9001, 5),
    (7, 300, 2400, 64, 70000, 6),        # prompts
])
def test_steps_follow_the_plain_allocator(batch, width, num_pages, page, max_tokens, seed):
    rng = random.Random(seed)
    pages, plain = PageTables.empty(batch, width, num_pages, page), Plain(batch, width, num_pages, page)
    buffers = pages.step_buffers(max_tokens)
    most = 2 * max_tokens // batch + 2
    for i in range(12):
        new = [rng.choice([0, 1, 1, rng.randint(-2, most), rng.randint(0, width * page + 2)]) for _ in range(batch)]
        keep = None if i % 4 == 0 else [rng.choice([n, n, 0, rng.randint(-1, n + 3)]) for n in plain.lens]
        plan = plan_step(pages, ints(new), max_tokens, keep=None if keep is None else ints(keep),
                         out=buffers if i % 2 else None)
        agree(pages, plan, plain, plain.step(new, max_tokens, keep), max_tokens)


@on_gpu
def test_cut_and_grown_again_a_request_has_its_own_pages():
    pages = PageTables.empty(4, 16, 64, 16)
    plan_step(pages, ints([100, 17, 256, 0]), 400)
    before = [t.clone() for t in (pages.page_table, pages.lens, pages.free_pages, pages.free_count)]
    plan_step(pages, ints([92, 17, 255, 0]), 400, keep=ints([8, 0, 1, 0]))
    for b, (t, n) in enumerate(zip(before[0].tolist(), [7, 2, 16, 0])):
        assert pages.page_table[b, :n].tolist() == t[:n]
    assert torch.equal(pages.lens, before[1]) and torch.equal(pages.free_count, before[3])
    n = int(before[3])
    assert torch.equal(pages.free_pages[:n], before[2][:n])


@on_gpu
def test_keep_may_be_the_lengths_themselves():
    for batch, most in ((5, 64), (1500, 9000)):
        pages, plain = PageTables.empty(batch, 8, 8 * batch, 16), Plain(batch, 8, 8 * batch, 16)
        for i in range(3):
            new = [(3 * b + i) % 9 for b in range(batch)]
            agree(pages, plan_step(pages, ints(new), most, keep=pages.lens), plain, plain.step(new, most), most)


@on_gpu
def test_empty_calls():
    pages = PageTables.empty(0, 4, 8, 16)
    plan = plan_step(pages, ints([]), 5)
    assert plan.cu_q.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and int(plan.refused) == 0
    pages = PageTables.empty(2, 4, 8, 16)
    plan = plan_step(pages, ints([1, 0]), 0)
    assert plan.cu_q.tolist() == [0, 0, 0] and int(plan.refused) == 1 and pages.lens.tolist() == [0, 0]
    pages = PageTables.empty(2, 0, 0, 16)
    plan = plan_step(pages, ints([3, 0]), 4)
    assert plan.cu_q.tolist() == [0, 0, 0] and int(plan.refused) == 1


@on_gpu
def test_state_that_cannot_be_is_not_followed():
    """Lengths past the table, a count past the stack: clamped; pages outside come back as they are."""
    whole = torch.full((40,), 7, dtype=torch.int32, device="cuda")
    table, free = whole[8:16].view(2, 4), whole[24:32]
    free.copy_(torch.arange(8, dtype=torch.int32))
    table.copy_(ints([[0, 1, 2, 3], [-5, 1 << 30, 6, 7]]))
    pages = PageTables(table, ints([1 << 30, -9]), free, ints([1 << 30]), 16)
    plan_step(pages, ints([1 << 30, 40]), 64, keep=ints([17, 9]))
    torch.cuda.synchronize()
    assert whole[:8].eq(7).all() and whole[16:24].eq(7).all() and whole[32:].eq(7).all()
    assert pages.lens.tolist() == [17, 40] and int(pages.free_count) <= 8


@on_gpu
def test_strided_tables_and_another_stream():
    store = torch.full((6, 20), -3, dtype=torch.int32, device="cuda")
    pages = PageTables.empty(6, 8, 32, 16)
    view = PageTables(store[:, 5:13], pages.lens, pages.free_pages, pages.free_count, 16)
    new = ints([[5, 0], [40, 0], [0, 0], [16, 0], [17, 0], [1, 0]])[:, 0]          # a strided argument
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan = plan_step(view, new, 96)
    side.synchronize()
    plain = Plain(6, 8, 32, 16)
    agree(view, plan, plain, plain.step(new.tolist(), 96), 96)
    assert store[:, :5].eq(-3).all() and store[:, 13:].eq(-3).all()


@on_gpu
def test_a_graph_goes_on_from_step_to_step():
    pages, plain = PageTables.empty(5, 12, 40, 16), Plain(5, 12, 40, 16)
    new, keep = ints([0] * 5), ints([0] * 5)
    out = pages.step_buffers(64)
    plan_step(pages, new, 64, keep=keep, out=out)
    plain.step([0] * 5, 64, [0] * 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan_step(pages, new, 64, keep=keep, out=out)
    rng = random.Random(9)
    for _ in range(30):
        n, k = [rng.randint(0, 15) for _ in range(5)], [max(0, x - rng.randint(0, 9)) for x in plain.lens]
        new.copy_(ints(n))
        keep.copy_(ints(k))
        graph.replay()
        agree(pages, out, plain, plain.step(n, 64, k), 64)


@on_gpu
def test_refusals_of_step_arguments():
    pages = PageTables.empty(2, 4, 8, 16)
    new = ints([1, 1])
    out = pages.step_buffers(8)
    with pytest.raises(TypeError, match="new_tokens"):
        plan_step(pages, new.long(), 8)
    with pytest.raises(TypeError, match="keep"):
        plan_step(pages, new, 8, keep=new.float())
    with pytest.raises(AssertionError, match="new_tokens"):
        plan_step(pages, ints([1]), 8)
    with pytest.raises(AssertionError, match="keep"):
        plan_step(pages, new, 8, keep=ints([1, 1, 1]))
    with pytest.raises(AssertionError, match="cpu"):
        plan_step(pages, new.cpu(), 8)
    with pytest.raises(ValueError, match="max_tokens"):
        plan_step(pages, new, -1)
    with pytest.raises(AssertionError, match="does not fit"):
        plan_step(pages, new, 9, out=out)
    with pytest.raises(TypeError, match="int64"):
        plan_step(pages, new, 8, out=StepPlan(*out[:1], out.positions, *out[2:]))
    with pytest.raises(AssertionError, match="does not fit"):
        plan_step(pages, new, 8, out=out._replace(kv_lens=ints([0, 0])))
    assert pages.lens.tolist() == [0, 0]
