// csrc/overlap.h against a list of every byte, for random layouts of up to four dimensions: "no" must be true. And the layouts of this
// framework must be told apart: heads of the same rows, interleaved heads, column ranges.
#include <stdio.h>
#include <stdlib.h>

#include <set>
#include <vector>

#include "overlap.h"

using ob_overlap::Place;

static uint64_t state = 12345;
static uint64_t rnd(uint64_t n) {
  state = state * 6364136223846793005ull + 1442695040888963407ull;
  return (state >> 33) % n;
}
static std::vector<int64_t> bytes_of(const Place& p) {
  std::vector<int64_t> at{(int64_t)p.at};
  if (p.empty) return {};
  for (int d = 0; d < p.dims; ++d) {
    std::vector<int64_t> next;
    for (int64_t a : at)
      for (int64_t i = 0; i < p.dim[d].size; ++i) next.push_back(a + i * p.dim[d].stride);
    at = next;
  }
  std::vector<int64_t> out;
  for (int64_t a : at)
    for (int64_t i = 0; i < p.item; ++i) out.push_back(a + i);
  return out;
}
static Place make(uintptr_t at, int64_t item, std::vector<std::pair<int64_t, int64_t>> dims) {
  Place p;
  p.at = at, p.item = item;
  for (auto [stride, size] : dims) p.add(stride, size);
  return p;
}

int main(int argc, char** argv) {
  const long rounds = argc > 1 ? atol(argv[1]) : 100000;
  long wrong = 0, missed = 0, overlapping = 0, told = 0;
  for (long r = 0; r < rounds; ++r) {
    Place p[2];
    const int64_t row = 8 + 2 * rnd(40);
    for (auto& x : p) {
      x.at = 1000 + rnd(60), x.item = 1 << rnd(3);
      const int dims = (int)rnd(4);
      for (int d = 0; d < dims; ++d) x.add(rnd(3) == 0 ? row : (int64_t)rnd(24), (int64_t)rnd(5));
    }
    const auto a = bytes_of(p[0]), b = bytes_of(p[1]);
    const std::set<int64_t> sa(a.begin(), a.end());
    bool meet = false;
    for (int64_t x : b) meet |= sa.count(x) > 0;
    const bool says = ob_overlap::may_overlap(p[0], p[1]);
    if (says != ob_overlap::may_overlap(p[1], p[0])) ++wrong;
    if (meet && !says) ++wrong;
    overlapping += meet;
    told += !meet && !says;
    missed += !meet && says;
    if (sa.size() != a.size() && !ob_overlap::may_overlap_itself(p[0])) ++wrong;
  }
  // rows of 12 heads of 64 fp16 values, 9 tokens
  auto heads = [](int first, int count, int step, int d0, int dims) {
    return make(4096 + first * 128 + d0 * 2, 2, {{12 * 128, 9}, {128 * step, count}, {2, dims}});
  };
  struct { Place a, b; bool want; } known[] = {
      {heads(0, 4, 1, 0, 64), heads(4, 4, 1, 0, 64), false}, {heads(0, 4, 1, 0, 64), heads(1, 4, 1, 0, 64), true},
      {heads(0, 6, 2, 0, 64), heads(1, 6, 2, 0, 64), false}, {heads(0, 6, 2, 0, 64), heads(2, 3, 2, 0, 64), true},
      {heads(0, 12, 1, 0, 32), heads(0, 12, 1, 32, 32), false}, {heads(0, 12, 1, 0, 33), heads(0, 12, 1, 32, 32), true},
      {heads(8, 4, 1, 0, 64), heads(0, 8, 1, 0, 64), false}, {heads(8, 4, 1, 0, 64), make(4096 + 11 * 128, 2, {{2, 64}}), true},
      {heads(8, 4, 1, 0, 64), make(4096 + 12 * 128 + 64, 2, {{2, 64}}), false},
      {make(4096, 2, {{0, 9}, {128, 4}, {2, 64}}), make(4096 + 512, 2, {{512, 9}, {2, 256}}), false},      // a broadcast row before the other
      {make(4096, 2, {{0, 9}, {128, 4}, {2, 64}}), make(4096 + 510, 2, {{512, 9}, {2, 256}}), true}};
  for (auto& k : known) wrong += ob_overlap::may_overlap(k.a, k.b) != k.want || ob_overlap::may_overlap(k.b, k.a) != k.want;
  printf("%ld %ld %ld %ld\n", wrong, overlapping, told, missed);
  return wrong != 0;
}
