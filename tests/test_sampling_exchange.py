"""What a cluster's CTAs send one another while they draw (csrc/qsample.cuh).

A meeting's values go to one half of a box, the next meeting's to the other: a CTA that is ahead writes those while one
that is behind still reads these.  Counts and sums share the halves, so no byte of one half may belong to the other,
whichever of the two a meeting sends.  The layout is asked of the compiler, without a GPU."""
import subprocess
from pathlib import Path

import pytest
import torch

from qlinear import _build
from qlinear.kernels.sampling import sample_tokens
from test_sampling import agree, on_gpu, rows_of

CSRC = Path(__file__).resolve().parents[1] / "llm-inference-optimizer_b200" / "csrc"

# the bytes of half t, of sums and of counts, whether the halves are members' or the box's
SOURCE = r"""
#include <cstdio>
#include "qsample.cuh"
using ql::smp::Shared;
template <class S> auto sums(S* s, int t, int) -> decltype(&s->box.f64[t]) { return &s->box.f64[t]; }
template <class S> auto sums(S* s, int t, long) -> decltype(&s->box[t].f64) { return &s->box[t].f64; }
template <class S> auto counts(S* s, int t, int) -> decltype(&s->box.u32[t]) { return &s->box.u32[t]; }
template <class S> auto counts(S* s, int t, long) -> decltype(&s->box[t].u32) { return &s->box[t].u32; }
alignas(16) static char room[sizeof(Shared)];
template <class P> void print(int t, P* p) {
  const long begin = reinterpret_cast<char*>(p) - room;
  printf("%d %ld %ld\n", t, begin, begin + (long)sizeof(*p));
}
int main() {
  Shared* s = reinterpret_cast<Shared*>(room);
  for (int t = 0; t < 2; ++t) {
    print(t, sums(s, t, 0));
    print(t, counts(s, t, 0));
  }
}
"""


def test_halves_of_the_box_lie_apart(tmp_path):
    (tmp_path / "box.cu").write_text(SOURCE)
    subprocess.run([_build.nvcc_path(), *_build.ARCH_FLAGS, "-std=c++17", f"-I{CSRC}", "-o", str(tmp_path / "box"),
                    str(tmp_path / "box.cu")], check=True, capture_output=True)
    lines = subprocess.run([str(tmp_path / "box")], check=True, capture_output=True, text=True).stdout.split("\n")
    ranges = [tuple(map(int, line.split())) for line in lines if line]
    assert len(ranges) == 4
    for t, begin, end in ranges:
        for other, b, e in ranges:
            assert t == other or end <= b or e <= begin, f"bytes {begin}..{end} of half {t}, {b}..{e} of half {other}"


@on_gpu
@pytest.mark.parametrize("rows", [1, 2, 4])
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 20001), (torch.float32, 151936), (torch.float16, 151936),
                                         (torch.bfloat16, 40000)])
def test_counts_and_sums_in_turn(dtype, vocab, rows):
    """A row of 16 CTAs whose border is searched for: meetings about counts, then about sums, again and again."""
    logits, uniform = rows_of(rows, vocab, dtype, rows + vocab)
    for f in (dict(top_k=513), dict(top_k=513, top_p=0.9), dict(top_k=15000), dict(top_k=15000, top_p=0.97),
              dict(top_p=0.99999, temperature=2.0)):
        want = agree(logits, uniform, **f)
        for _ in range(20):
            assert torch.equal(want, sample_tokens(logits, uniform, **f)), f
