// qwork.h — how the attention kernels divide their work over CTAs, and which
// counters the parts of an item meet at.  Plain C++: the kernels use it on the
// device, and it can be compiled and checked on the host.
#pragma once

#ifdef __CUDACC__
#define QL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define QL_HOST_DEVICE inline
#endif

namespace ql {
namespace att {

// Work is counted in units of 128 keys of one item: one request, one
// key/value head, one tile of ROWS rows (row r of a request is new token
// r / group under query head r % group of the key/value head).  Items
// lie one behind another, each rounded up to a multiple of kMinUnits, and
// the CTAs take equal runs of units, whatever the requests' lengths are: a
// CTA may end one item, do some whole and begin another.  Lengths are read
// on the device, so a captured launch serves other lengths later.
constexpr int kUnitKeys = 128;
constexpr int kJoin = 16;                  // parts of an item that are joined at once
constexpr int kMaxCtas = 1024;
constexpr int kHeaderBytes = 2 * 4 * kMaxCtas;   // counters of items and of groups of parts

// The most positions of a request: the end of its last unit, at 512 keys a
// part, is still an int.
constexpr int kMostKeys = 0x7FFFFFFF - 511;

// Units of an item over kv_len positions (0 .. kMostKeys): at least one part's, a multiple of it.
QL_HOST_DEVICE int units_of(int kv_len, int min_units) {
  const int n = (kv_len + kUnitKeys - 1) / kUnitKeys, parts = (n + min_units - 1) / min_units;
  return (parts > 1 ? parts : 1) * min_units;
}

struct Work {
  long long total;     // units of the launch
  int ctas;            // CTAs that take part
  QL_HOST_DEVICE long long first_unit(int cta) const { return quotient(total * cta, ctas); }
  QL_HOST_DEVICE int cta_of(long long u) const { return (int)quotient((u + 1) * ctas - 1, total); }
  // of non-negative numbers, by the short division where it does (nearly always)
  static QL_HOST_DEVICE long long quotient(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
  }
};

// How an item in several parts, one a CTA, is joined, as its CTA `cta` sees
// it.  The item's last CTA to arrive joins the parts; many parts are joined in
// groups of kJoin first, each by its last CTA, so that no CTA reads more than
// a few dozen: with 74 parts a single one took longer than the keys had.
//
// Every counter has one user.  An item in parts begins in a CTA of its own, so
// its word, c_first, is its own.  Group g counts kJoin g further on in a second
// array, up to the item's last CTA.  There the next item in parts may begin,
// with its group 0 on that word; but a group that begins in the last CTA has
// one part, which is a group's result already: it counts nowhere
// (group_parts is 1), and every word that does count lies before the CTA in
// which the next item begins.
struct Join {
  int c_first, parts, groups;
  int group, group_parts;      // of this CTA
  QL_HOST_DEVICE bool grouped() const { return groups > 1 && group_parts > 1; }
  QL_HOST_DEVICE int group_counter() const { return kMaxCtas + c_first + group * kJoin; }
  QL_HOST_DEVICE int item_counter() const { return c_first; }
  QL_HOST_DEVICE int item_arrivals() const { return groups > 1 ? groups : parts; }
};
QL_HOST_DEVICE Join join_of(const Work& w, long long item_begin, int per_item, int cta) {
  Join j;
  j.c_first = w.cta_of(item_begin);
  j.parts = w.cta_of(item_begin + per_item - 1) - j.c_first + 1;
  j.groups = (j.parts + kJoin - 1) / kJoin;
  j.group = (cta - j.c_first) / kJoin;
  const int left = j.parts - j.group * kJoin;
  j.group_parts = left < kJoin ? left : kJoin;
  return j;
}

}  // namespace att
}  // namespace ql
