// Do two strided tensors share memory? Plain C++, also compiled by a host test. Views into a fused projection's rows are the normal
// case here: neither is dense, and their address ranges interleave without a common byte.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace ob_overlap {

constexpr int kMaxDims = 8;

struct Dim { int64_t stride, size; };                     // bytes; steps

// Where the elements of a tensor lie: the dimensions that move, by falling stride. Strides are not negative.
struct Place {
  uintptr_t at = 0;
  int64_t item = 0;                                       // bytes of an element
  bool empty = false;
  int dims = 0;
  Dim dim[kMaxDims];

  void add(int64_t stride_bytes, int64_t size) {          // at most kMaxDims that move
    if (size == 0) empty = true;
    if (size <= 1) return;
    int i = dims++;
    for (; i > 0 && dim[i - 1].stride < stride_bytes; --i) dim[i] = dim[i - 1];
    dim[i] = {stride_bytes, size};
  }
  int64_t extent(int from) const {                        // bytes from the first to behind the last element
    int64_t e = item;
    for (int i = from; i < dims; ++i) e += dim[i].stride * (dim[i].size - 1);
    return e;
  }
};

// False only if every element has bytes of its own.
inline bool may_overlap_itself(const Place& a) {
  if (a.empty) return false;
  for (int i = 0; i < a.dims; ++i)
    if (a.dim[i].stride < a.extent(i + 1)) return true;
  return false;
}

// b begins `off` bytes after a; dimensions before i (of a) and j (of b) are dealt with. Of the rows that the longer stride makes,
// only neighbours can meet: their inner parts decide. Rows that are longer than that stride are taken to meet.
inline bool may_meet(const Place& a, int i, const Place& b, int j, int64_t off) {
  if (off >= a.extent(i) || off <= -b.extent(j)) return false;
  if (i == a.dims && j == b.dims) return true;
  const int64_t s = std::max(i < a.dims ? a.dim[i].stride : 0, j < b.dims ? b.dim[j].stride : 0);
  const bool a_has = i < a.dims && a.dim[i].stride == s, b_has = j < b.dims && b.dim[j].stride == s;
  const int ai = i + a_has, bj = j + b_has;
  const int64_t ea = a.extent(ai), eb = b.extent(bj);
  if (s == 0) return may_meet(a, ai, b, bj, off);         // a broadcast: the same row again
  if (ea > s || eb > s) return true;
  const int64_t last_a = a_has ? a.dim[i].size - 1 : 0, last_b = b_has ? b.dim[j].size - 1 : 0;
  // rows x of a and y of b are off + (y - x) s apart: those closer than a row
  const int64_t nearest = -off / s;
  for (int64_t m = std::max(-last_a, nearest - 2); m <= std::min(last_b, nearest + 2); ++m)
    if (may_meet(a, ai, b, bj, off + m * s)) return true;
  return false;
}

// False only if no byte belongs to both.
inline bool may_overlap(const Place& a, const Place& b) {
  return !a.empty && !b.empty && may_meet(a, 0, b, 0, static_cast<int64_t>(b.at - a.at));
}

}  // namespace ob_overlap
