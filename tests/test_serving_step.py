"""A serving step's operators one after another, captured once and replayed with other lengths, tokens and numbers: the step's
plan, the cache's append with the rotation, attention behind a shared prefix, drawing tokens.  Each replay is checked against
a written-out allocator, float64 attention over what the cache then holds, and the plain draw."""
import math
import random

import pytest
import torch

from qlinear import _lib
from qlinear.kernels.kv_cache import QuantizedKVCache, append_kv, read_kv
from qlinear.kernels.paging import PageTables, plan_step
from qlinear.kernels.rotary import RotaryTable
from qlinear.kernels.sampling import sample_tokens
from qlinear.kernels.shared_attention import shared_prefix_attention

from attn_helpers import attend, attention_bounds, heads, quantise, rotate_by, values, visible
from test_paging import Plain, ints
from test_sampling import plain_row

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="requires a CUDA GPU")]


@pytest.mark.parametrize("bits", [8, 4])
def test_a_captured_step_goes_on(bits):
    batch, hq, hk, d, page, room, vocab, start = 5, 8, 2, 64, 16, 48, 3001, 70
    pages, plain = PageTables.empty(batch, 9, 60, page), Plain(batch, 9, 60, page)
    cache = QuantizedKVCache.empty(60, page, hk, d, bits)
    rotary = RotaryTable.build(d, 512, 1e4)
    # the prefix: pages from the same stack
    prefix = PageTables(torch.zeros(1, 5, dtype=torch.int32, device="cuda"), ints([0]), pages.free_pages, pages.free_count, page)
    first = plan_step(prefix, ints([start]), start)
    k0, v0 = heads(start, hk, d, torch.float16, 1), heads(start, hk, d, torch.float16, 2)
    append_kv(cache, k0, v0, first.slots, positions=first.positions, rotary=rotary)
    taken = [plain.free.pop() for _ in range(5)]
    assert prefix.page_table.tolist() == [taken]
    lost = set(taken)
    # static inputs and outputs of a step
    new, keep, uniform = ints([0] * batch), ints([0] * batch), torch.zeros(room, device="cuda")
    qkv = torch.zeros(room, hq + 2 * hk, d, dtype=torch.float16, device="cuda")
    head = torch.randn(hq * d, vocab, generator=torch.Generator().manual_seed(3)).half().cuda()
    plan = pages.step_buffers(room)
    out = torch.zeros(room, hq, d, dtype=torch.float16, device="cuda")

    def step():
        plan_step(pages, new, room, keep=keep, out=plan)
        q = append_kv(cache, qkv[:, hq:hq + hk], qkv[:, hq + hk:], plan.slots, q=qkv[:, :hq], positions=plan.positions + start,
                      rotary=rotary)
        _, lse = shared_prefix_attention(q, cache, prefix.page_table, prefix.lens, pages.page_table, plan.kv_lens, cu_q=plan.cu_q,
                                         max_q=12, out=out, return_lse=True)
        logits = out.flatten(1) @ head
        return q, lse, logits, *sample_tokens(logits, uniform, temperature=0.9, top_k=40, top_p=0.9, min_p=0.01,
                                              return_logprobs=True)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, lse, logits, ids, logprobs = step()
    rng = random.Random(4)
    for i in range(12):
        asked = [rng.choice([0, 1, 1, 1, 7, 12]) for _ in range(batch)]
        kept = [rng.choice([n, n, n, max(0, n - 5), 0]) for n in plain.lens]
        new.copy_(ints(asked))
        keep.copy_(ints(kept))
        qkv.copy_(heads(room, hq + 2 * hk, d, torch.float16, 100 + i))
        uniform.copy_(torch.rand(room, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        cu, slots, positions, refused = want = plain.step(asked, room, kept)
        assert lost.isdisjoint(plain.free) and lost.isdisjoint(x for h in plain.held for x in h)
        n = int(pages.free_count)
        assert pages.free_pages[:n].tolist() == plain.free and plan.cu_q.tolist() == cu and int(plan.refused) == refused
        assert plan.slots[:len(slots)].tolist() == slots and plan.positions[:len(slots)].tolist() == positions
        assert pages.lens.tolist() == plain.lens
        rows = len(slots)
        if rows == 0:
            continue
        # what was written: the new rows' codes, as the quantiser gives them for the rotated keys
        at = torch.tensor(positions, device="cuda") + start
        cos, sin = (rotary.table[at][..., j][:, None] for j in (0, 1))
        turned = rotate_by(qkv[:rows, hq:hq + hk].float(), cos, sin, "half")
        codes, scales = quantise(turned, bits)
        s = torch.tensor(slots, device="cuda")
        stored = cache.k_codes[s // page, :, s % page]
        if bits == 8:
            assert torch.equal(stored.int(), codes)
        assert torch.equal(cache.k_scales[s // page, :, s % page], scales)
        assert torch.equal(q[:rows], rotate_by(qkv[:rows, :hq].float(), cos, sin, "half").half())

        def cached(table, count):
            p = table[:-(-count // page)].long()
            return [values(x[p], z[p], bits).transpose(1, 2).flatten(0, 1)[:count]
                    for x, z in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))]
        early = cached(prefix.page_table[0], start)
        for b in range(batch):
            t = cu[b + 1] - cu[b]
            if t == 0:
                continue
            late = cached(pages.page_table[b], plain.lens[b])
            see = torch.cat([torch.ones(t, start, dtype=torch.bool, device="cuda"), visible(t, plain.lens[b], None)], 1)
            right = attend(q[cu[b]:cu[b + 1]], torch.cat([early[0], late[0]]), torch.cat([early[1], late[1]]), see, 1 / math.sqrt(d))
            tol, tol_lse = attention_bounds(*right, torch.float16)
            assert bool(((out[cu[b]:cu[b + 1]].double() - right[0]).abs() <= tol).all())
            assert bool(((lse[cu[b]:cu[b + 1]].double() - right[1]).abs() <= tol_lse).all())
        x, u = logits[:rows].double().cpu(), uniform.double().cpu()
        for r in range(rows):
            token, chance = plain_row(x[r], float(u[r]), 0.9, 40, 0.9, 0.01)
            assert int(ids[r]) == token and abs(float(logprobs[r]) - chance) <= 2.0 ** -24 * abs(chance) + 2.0 ** -19.5
        k, v = read_kv(cache, plan.slots[:rows])
        assert k.shape == v.shape == (rows, hk, d) and bool(k.isfinite().all())
    assert _lib.device_error() == 0
