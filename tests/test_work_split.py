"""How the attention kernels divide their work and join an item's parts
(csrc/qwork.h), compiled for the host: every unit has one CTA, and no two
items meet at one counter, whatever the lengths are."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llm-inference-optimizer_b200" / "csrc"

# One launch: items of `units` units (a multiple of the least), walked as the kernels walk them.  Returns 0, or what is
# wrong: 1 a unit in no or two CTAs, 2 two (item, group)s at one counter, 3 arrivals that do not add up, 4 a counter
# outside the scratch's head.
SOURCE = r"""
#include <algorithm>
#include <map>
#include <utility>
#include "qwork.h"
using namespace ql::att;
extern "C" int units(int kv_len, int min_units) { return units_of(kv_len, min_units); }
extern "C" int most_keys() { return kMostKeys; }
extern "C" int check(const int* units, int items, int min_units, int grid, int* most_parts, int* lone) {
  long long total = 0;
  for (int i = 0; i < items; ++i) total += units[i];
  Work w = {total, (int)std::min<long long>(grid, total / min_units)};
  std::map<int, std::pair<std::pair<int, int>, std::pair<int, int>>> words;   // word -> (item, group), (arrivals, due)
  std::map<std::pair<int, int>, int> seen;                                    // (item, group) -> CTAs
  int wrong = 0;
  auto arrive = [&](int word, int item, int group, int due) {
    if (word < 0 || 4 * word >= kHeaderBytes) wrong = wrong ? wrong : 4;
    auto it = words.find(word);
    if (it == words.end()) {
      words[word] = {{item, group}, {1, due}};
      return;
    }
    if (it->second.first != std::make_pair(item, group)) wrong = wrong ? wrong : 2;
    it->second.second.first++;
  };
  long long next = 0, base = 0;
  int item = 0;
  for (int c = 0; c < w.ctas; ++c) {
    long long u = w.first_unit(c);
    const long long end = w.first_unit(c + 1);
    if (u != next || end <= u) wrong = wrong ? wrong : 1;
    while (u < end) {
      while (u >= base + units[item]) base += units[item++];
      const int begin = (int)(u - base), stop = (int)std::min<long long>(units[item], begin + (end - u));
      if (begin != 0 || stop != units[item]) {
        const Join j = join_of(w, base, units[item], c);
        *most_parts = std::max(*most_parts, j.parts);
        if (j.parts % kJoin == 1 && j.groups > 1) ++*lone;
        if (j.grouped()) arrive(j.group_counter(), item, 1 + j.group, j.group_parts);
        if (++seen[{item, j.group}] == j.group_parts || j.groups == 1) arrive(j.item_counter(), item, 0, j.item_arrivals());
      }
      u += stop - begin;
    }
    next = end;
  }
  if (next != total) wrong = wrong ? wrong : 1;
  for (auto& x : words)
    if (x.second.second.first != x.second.second.second) wrong = wrong ? wrong : 3;
  return wrong;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    d = tmp_path_factory.mktemp("work")
    (d / "work.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "work.so"),
                    str(d / "work.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "work.so"))

    def run(units, least, grid):
        parts, lone = ctypes.c_int(0), ctypes.c_int(0)
        wrong = lib.check((ctypes.c_int * len(units))(*units), len(units), least, grid, ctypes.byref(parts),
                          ctypes.byref(lone))
        return wrong, parts.value, lone.value
    run.lib = lib
    return run


@pytest.mark.parametrize("least", [2, 4])
def test_units_up_to_the_most_positions(check, least):
    """As in whole numbers without an end, and the last unit's end is an int: a table of 2^15 pages of 65536 and a length
    to match would pass it."""
    most = check.lib.most_keys()
    for n in (0, 1, 127, 128, 129, 128 * least, 128 * least + 1, 1 << 30, most - 513, most - 1, most):
        units = check.lib.units(n, least)
        assert units == items([n], 1, least)[0] and 128 * units <= (1 << 31) - 1, n
    assert (1 << 31) - 1 - most < 512


def items(lens, heads, least):
    """Units of each item: requests of `lens` positions, a tile of rows each."""
    out = []
    for n in lens:
        units = -(-n // 128)
        out += [max(-(-units // least), 1) * least] * heads
    return out


def test_items_of_seventeen_parts_in_a_row(check):
    """9 requests of 8192 over 2 heads on 296 CTAs, one token: items of 17 parts, the next beginning in the last CTA of
    the one before; and the same for the kernel of 148 CTAs and 512 keys a part at least."""
    wrong, parts, lone = check(items([8192] * 9, 2, 2), 2, 296)
    assert parts >= 17 and lone > 0 and wrong == 0
    wrong, parts, lone = check(items([9000] * 9, 1, 4), 4, 148)
    assert parts >= 17 and lone > 0 and wrong == 0


@pytest.mark.parametrize("least,grid", [(2, 296), (2, 148), (4, 148), (4, 1024)])
def test_every_counter_has_one_user(check, least, grid):
    rng = random.Random(grid + least)
    many = 0
    for _ in range(1500):
        batch, heads = rng.choice([1, 2, 3, 4, 5, 8, 9, 16, 33, 64]), rng.choice([1, 2, 3, 4, 5, 8])
        top = rng.choice([300, 5000, 20000, 100000])
        lens = [top] * batch if rng.random() < 0.3 else [rng.randint(0, top) for _ in range(batch)]
        wrong, _, lone = check(items(lens, heads, least), least, grid)
        assert wrong == 0, (wrong, lens, heads)
        many += lone
    assert many > 100                       # the shapes do reach groups of one part
