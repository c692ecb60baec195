// overlap.h - whether two strided views share a byte of memory. Host code, used by
// the argument checks: an output may lie in the gaps of an input (the heads of
// one fused projection), so comparing first and last addresses does not do.
#pragma once

#include <algorithm>
#include <cstdint>

namespace pkb200 {

// Up to four axes of `n` places, `stride` bytes apart (not negative), of values of
// `size` bytes.
struct View {
  std::uintptr_t base;
  int axes;
  long long n[4], stride[4];
  long long size;

  bool empty() const { return std::any_of(n, n + axes, [](long long x) { return x == 0; }); }
  // one past the last byte
  std::uintptr_t end() const {
    std::uintptr_t e = base + size;
    for (int i = 0; i < axes; ++i) e += (n[i] - 1) * stride[i];
    return e;
  }
  bool same_places(const View& o) const {
    if (base != o.base || axes != o.axes || size != o.size) return false;
    for (int i = 0; i < axes; ++i)
      if (n[i] != o.n[i] || (n[i] > 1 && stride[i] != o.stride[i])) return false;
    return true;
  }
};

namespace overlap {

// A term of the distance between a byte of one view and a byte of the other: `stride`
// times a whole number of [lo, hi]; `least` and `most` bound the sum of the terms after it.
struct Term {
  long long stride, lo, hi, least, most;
};

inline long long floor_div(long long a, long long b) { return a / b - (a % b < 0); }

// Whether the terms from k on can add up to `want`. Strides fall, and in views
// without overlaps of their own each is beyond the reach of those after it, so
// that only one or two numbers are tried for a term; `tries` bounds the rest.
inline bool reach(const Term* t, int count, int k, long long want, long long& tries) {
  if (k == count) return want == 0;
  const long long first = std::max(t[k].lo, -floor_div(t[k].most - want, t[k].stride));
  const long long last = std::min(t[k].hi, floor_div(want - t[k].least, t[k].stride));
  for (long long c = first; c <= last; ++c) {
    if (--tries < 0) return true;  // not decided: taken for an overlap
    if (reach(t, count, k + 1, want - c * t[k].stride, tries)) return true;
  }
  return false;
}

}  // namespace overlap

inline bool share_memory(const View& a, const View& b) {
  if (a.empty() || b.empty() || a.end() <= b.base || b.end() <= a.base) return false;
  overlap::Term t[10];
  int count = 0;
  auto add = [&](long long stride, long long lo, long long hi) {
    if (stride == 0 || lo == hi) return;
    for (int i = 0; i < count; ++i)
      if (t[i].stride == stride) {
        t[i].lo += lo;
        t[i].hi += hi;
        return;
      }
    t[count++] = {stride, lo, hi, 0, 0};
  };
  for (int i = 0; i < a.axes; ++i) add(a.stride[i], 0, a.n[i] - 1);
  for (int i = 0; i < b.axes; ++i) add(b.stride[i], -(b.n[i] - 1), 0);
  add(1, 0, a.size - 1);
  add(1, -(b.size - 1), 0);
  std::sort(t, t + count, [](const overlap::Term& x, const overlap::Term& y) { return x.stride > y.stride; });
  for (int i = count - 1; i > 0; --i) {
    t[i - 1].least = t[i].least + t[i].stride * t[i].lo;
    t[i - 1].most = t[i].most + t[i].stride * t[i].hi;
  }
  long long tries = 1 << 16;
  return overlap::reach(t, count, 0, static_cast<long long>(b.base - a.base), tries);
}

}  // namespace pkb200
