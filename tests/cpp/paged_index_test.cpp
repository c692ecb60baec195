// Feeds random batch descriptions, most of them wrong, to the index arithmetic
// of the paged-cache kernels, walks what a kernel would walk, and checks that
// nothing out of range would be read or written. Prints the number of
// descriptions that were reported as bad.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../polykernel_b200/csrc/paged_index.h"

using namespace pkb200::paged;

#define CHECK(x)                                              \
  do {                                                        \
    if (!(x)) {                                               \
      std::printf("line %d: %s\n", __LINE__, #x);             \
      std::exit(1);                                           \
    }                                                         \
  } while (0)

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int odd[] = {INT_MIN, -1, 0, 1, 7, 63, 64, 65, 1000, INT_MAX - 1, INT_MAX};
  long bad_seqs = 0, good_seqs = 0, misplaced = 0, placed = 0;
  for (int round = 0; round < 20000; ++round) {
    const int B = pick(1, 5), T = pick(0, 40), width = pick(0, 6), page_size = 8 * pick(1, 5);
    const int pages = pick(1, 9), G = pick(1, 9), causal = pick(0, 1), window = causal ? pick(0, 1) * pick(1, 90) : 0;
    std::vector<int> cu(B + 1), lens(B), table(B * width);
    const bool wild = pick(0, 1);
    for (int i = 0, t = 0; i <= B; ++i) {
      cu[i] = wild && pick(0, 2) == 0 ? (pick(0, 1) ? odd[pick(0, 10)] : pick(-5, 50)) : t;
      t = least(T, t + pick(0, 12));
    }
    for (int& x : lens) x = pick(0, 3) == 0 ? odd[pick(0, 10)] : pick(-3, 300);
    for (int& x : table) x = pick(0, 4) == 0 ? odd[pick(0, 10)] : pick(-2, 11);
    const long long capacity = static_cast<long long>(width) * page_size;

    auto read_key = [&](int b, const Seq& s, int key) {  // as the fetching warps do
      if (key >= s.len) return;
      const int slot = key / page_size;
      CHECK(key >= 0 && slot < width);
      const int page = clip_page(table[b * width + slot], pages);
      CHECK(page >= 0 && page <= pages);
    };
    for (int b = 0; b < B; ++b) {
      bool bad;
      const Seq s = clip_seq(cu[b], cu[b + 1], lens[b], T, capacity, bad);
      (bad ? bad_seqs : good_seqs)++;
      CHECK(s.nq >= 0 && s.len >= 0 && s.len <= capacity);
      if (s.nq > 0) CHECK(s.t0 >= 0 && s.t0 + s.nq <= T);
      if (!bad && s.nq > 0) CHECK(s.pos0 >= 0 && s.pos0 + s.nq == lens[b]);
      for (const int kt : {64, 128}) {
        const int tile_rows = kt == 64 ? 16 : 2 * (128 / G) * G;
        const int rows = s.nq * G;
        for (int r0 = 0; r0 < rows; r0 += tile_rows) {
          const int first = r0 / G, last = (least(rows, r0 + tile_rows) - 1) / G;
          int tile0;
          const int n = clip_tiles(s, first, last, causal, window, kt, tile0);
          CHECK(n >= 1 && tile0 >= 0);
          CHECK(n <= capacity / kt + 2);
          for (int key = tile0 * kt; key < (tile0 + n) * kt; ++key) read_key(b, s, key);
          // every key that a row sees is in the tiles
          for (int i = first; i <= last; ++i) {
            const int lo = clip_lo(s, i, window), hi = clip_hi(s, i, causal);
            CHECK(hi <= s.len);
            if (lo < hi) CHECK(lo >= tile0 * kt && hi <= (tile0 + n) * kt);
          }
        }
      }
    }
    for (int t = 0; t < T; ++t) {
      int seq = -1;
      long long position = -1;
      const TokenPlace where = place_token(cu.data(), B, t, [&](int b) { return lens[b]; }, seq, position);
      if (where != kPlaced) {
        misplaced += where == kMisplaced;
        continue;
      }
      ++placed;
      CHECK(seq >= 0 && seq < B && position >= 0);
      CHECK(cu[seq] <= t && t < cu[seq + 1]);
      const long long slot = position / page_size;
      const int page = slot < width ? clip_page(table[seq * width + slot], pages) : pages;
      CHECK(page >= 0 && page <= pages);
      if (page < pages) CHECK(position < capacity);
    }
  }
  CHECK(bad_seqs > 1000 && good_seqs > 1000 && misplaced > 1000 && placed > 1000);
  std::printf("ok %ld bad, %ld good\n", bad_seqs, good_seqs);
  return 0;
}
