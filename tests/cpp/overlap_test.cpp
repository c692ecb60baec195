// Compares share_memory with a count of the bytes of both views, over random
// views of one small buffer.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>

#include "../../polykernel_b200/csrc/overlap.h"

using pkb200::View;

static std::set<long long> bytes(const View& v) {
  std::set<long long> s;
  long long at[4];
  long long total = 1;
  for (int i = 0; i < v.axes; ++i) total *= v.n[i];
  for (long long x = 0; x < total; ++x) {
    long long rest = x, place = static_cast<long long>(v.base);
    for (int i = 0; i < v.axes; ++i) {
      at[i] = rest % v.n[i];
      rest /= v.n[i];
      place += at[i] * v.stride[i];
    }
    for (int b = 0; b < v.size; ++b) s.insert(place + b);
  }
  return s;
}

int main() {
  std::mt19937 rng(3);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  long met = 0, apart = 0, gaps = 0;
  for (int round = 0; round < 40000; ++round) {
    View v[2];
    const int strides[] = {0, 2, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 100};
    for (View& x : v) {
      x.base = 1000 + pick(0, 150);
      x.axes = pick(1, 4);
      x.size = 1 << pick(0, 2);
      for (int i = 0; i < 4; ++i) {
        x.n[i] = pick(0, 20) ? pick(1, 5) : 0;
        x.stride[i] = strides[pick(0, 12)];
      }
    }
    if (pick(0, 1)) {  // two slices of one fused buffer
      v[1] = v[0];
      v[1].base += pick(0, 60);
      v[1].n[0] = pick(1, 5);
    }
    const std::set<long long> a = bytes(v[0]), b = bytes(v[1]);
    bool common = false;
    for (long long x : a) common |= b.count(x) != 0;
    if (pkb200::share_memory(v[0], v[1]) != common || pkb200::share_memory(v[1], v[0]) != common) {
      std::printf("round %d: bytes %d\n", round, common);
      return 1;
    }
    (common ? met : apart)++;
    if (!common && !a.empty() && !b.empty() && *a.begin() < *b.rbegin() && *b.begin() < *a.rbegin()) ++gaps;
  }
  if (met < 1000 || apart < 1000 || gaps < 1000) return 2;
  // long views: [rows][heads][128] slices of one projection, and one row further
  View q{0, 3, {100000, 32, 128}, {48 * 256, 256, 2}, 2}, k = q;
  k.base = 32 * 256;
  k.n[1] = 8;
  if (pkb200::share_memory(q, k)) return 3;
  k.base = 40 * 256 + 256 * 4;  // the last four reach the next row's heads
  if (!pkb200::share_memory(q, k)) return 4;
  std::printf("ok %ld met, %ld apart, %ld in gaps\n", met, apart, gaps);
  return 0;
}
