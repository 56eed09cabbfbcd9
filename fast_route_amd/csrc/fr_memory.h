// Host side: whether two strided arrays of 16-bit elements, or two elements of one, lie in the same place.  Parts of a joint tensor (the heads of a projection's rows, the
// halves of a cache) have ranges of addresses that overlap and no element in common, so the ranges alone do not say.
#pragma once
#include "fr_common.h"

namespace fr {

struct Box {
  const void* at;
  int dims;
  int64_t size[4], stride[4];  // in elements; strides of dimensions with one place: 0
  int64_t first, last;         // addresses of its bytes; first > last: there are none
  Box(const void* p, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t n3, int64_t s3)
      : at(p), dims(4), size{n0, n1, n2, n3}, stride{s0, s1, s2, s3}, first(1), last(0) {
    __int128 low = static_cast<__int128>(reinterpret_cast<uintptr_t>(p)), high = low + 1;
    for (int i = 0; i < dims; ++i) {
      if (size[i] <= 0) return;
      if (size[i] == 1) stride[i] = 0;
      const __int128 reach = static_cast<__int128>(stride[i]) * (size[i] - 1) * 2;
      (reach < 0 ? low : high) += reach;
    }
    constexpr __int128 kEnd = static_cast<__int128>(1) << 62;
    first = static_cast<int64_t>(low < -kEnd ? -kEnd : low);
    last = static_cast<int64_t>(high > kEnd ? kEnd : high);
  }
  Box(const void* p, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2) : Box(p, 1, 0, n0, s0, n1, s1, n2, 1) {}
  bool is_empty() const { return first > last; }
};
// Same place and layout, of arrays of the same sizes.
inline bool is_same(const Box& a, const Box& b) {
  if (a.at != b.at) return false;
  for (int i = 0; i < a.dims; ++i)
    if (a.size[i] != b.size[i] || a.stride[i] != b.stride[i]) return false;
  return true;
}

// Whether sum(stride[i] * x[i]) = distance for whole numbers lo[i] <= x[i] <= hi[i], not all zero if `other`.  Strides positive, descending: what the smaller ones
// reach leaves one or two x where they are nested, as in parts of one tensor.  After kSteps without an answer, and beyond 2^61 elements: yes.
struct Steps {
  static constexpr int kMost = 9, kSteps = 4096;
  int count = 0, left = kSteps;
  int64_t stride[kMost], lo[kMost], hi[kMost], low[kMost + 1], high[kMost + 1];  // low, high: what the strides from i on reach
  bool same = false;  // two strides alike, or one of zero, of more than one place
  void add(int64_t s, int64_t from, int64_t to) {
    if (from == to) return;
    int i = 0;
    while (i < count && stride[i] > s) ++i;
    same = same || s == 0 || (i < count && stride[i] == s);
    if (s == 0) return;
    if (i < count && stride[i] == s) {
      lo[i] += from;
      hi[i] += to;
      return;
    }
    for (int j = count++; j > i; --j) stride[j] = stride[j - 1], lo[j] = lo[j - 1], hi[j] = hi[j - 1];
    stride[i] = s, lo[i] = from, hi[i] = to;
  }
  bool from(int i, int64_t distance, bool other) {
    if (i == count) return distance == 0 && !other;
    if (--left < 0) return true;
    auto down = [](int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); };
    int64_t first = -down(high[i + 1] - distance, stride[i]), last = down(distance - low[i + 1], stride[i]);
    first = first < lo[i] ? lo[i] : first;
    last = last > hi[i] ? hi[i] : last;
    for (int64_t x = first; x <= last; ++x)
      if (from(i + 1, distance - x * stride[i], other && x == 0)) return true;
    return false;
  }
  bool reach(__int128 distance, bool other) {
    constexpr __int128 kFurthest = static_cast<__int128>(1) << 61;
    __int128 under = 0, over = 0;
    low[count] = high[count] = 0;
    for (int i = count - 1; i >= 0; --i) {
      under += static_cast<__int128>(stride[i]) * lo[i];
      over += static_cast<__int128>(stride[i]) * hi[i];
      if (under < -kFurthest || over > kFurthest) return true;
      low[i] = static_cast<int64_t>(under), high[i] = static_cast<int64_t>(over);
    }
    return distance >= under && distance <= over && from(0, static_cast<int64_t>(distance), other);
  }
};
// Two elements of an array in one place.
inline bool meets_itself(const Box& b) {
  if (b.is_empty()) return false;
  bool nested = true;  // every stride beyond what those behind it reach, as most are
  __int128 reach = 0;
  for (int i = b.dims - 1; i >= 0; --i) {
    nested = nested && (b.size[i] == 1 || b.stride[i] > reach);
    reach += static_cast<__int128>(b.stride[i]) * (b.size[i] - 1);
  }
  if (nested) return false;
  Steps steps;
  for (int i = 0; i < b.dims; ++i) steps.add(b.stride[i] < 0 ? -b.stride[i] : b.stride[i], 1 - b.size[i], b.size[i] - 1);
  return steps.same || steps.reach(0, true);
}
// An element of one and an element of the other in one place.
inline bool meets(const Box& a, const Box& b) {
  if (a.is_empty() || b.is_empty() || a.first > b.last || b.first > a.last) return false;
  const int64_t bytes = b.first - a.first;
  Steps steps;
  for (int i = 0; i < a.dims; ++i) steps.add(a.stride[i] < 0 ? -a.stride[i] : a.stride[i], 0, a.size[i] - 1);
  for (int i = 0; i < b.dims; ++i) steps.add(b.stride[i] < 0 ? -b.stride[i] : b.stride[i], 1 - b.size[i], 0);
  const int64_t odd = bytes & 1;  // halves of elements: one place less, too
  steps.add(1, 0, odd);
  return steps.reach((bytes - odd) / 2 + odd, false);
}

}  // namespace fr
