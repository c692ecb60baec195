// paged_index.h - the index arithmetic of the paged-cache kernels: which rows,
// keys and pages a batch description leads to, cut off where it would lead out
// of range. Plain functions for device and host code, so that descriptions
// which are wrong can be tried without a GPU.
#pragma once

#ifdef __CUDACC__
#define PKB_INDEX __host__ __device__ __forceinline__
#else
#define PKB_INDEX inline
#endif

namespace pkb200 {
namespace paged {

PKB_INDEX int least(int a, int b) { return a < b ? a : b; }
PKB_INDEX int most(int a, int b) { return a > b ? a : b; }

struct Seq {
  int t0, nq, len, pos0;  // first packed row, new tokens, keys, position of the first new token
};

// A sequence with new tokens [t0, t1) of `tokens` packed rows and `len` keys in a
// table of `capacity` rows. `bad`: it does not fit, and is cut off to what does.
PKB_INDEX Seq clip_seq(int t0, int t1, int len, int tokens, long long capacity, bool& bad) {
  Seq s;
  const bool in_order = t0 >= 0 && t1 >= t0 && t1 <= tokens;
  s.t0 = t0;
  s.nq = in_order ? t1 - t0 : 0;
  if (capacity > 0x7fffffff - 1024) capacity = 0x7fffffff - 1024;  // room to round up to key tiles
  const bool fits = len <= capacity;
  s.len = fits ? most(len, 0) : static_cast<int>(capacity);
  s.pos0 = s.len - s.nq;
  bad = !in_order || (s.nq > 0 && (!fits || len < s.nq));
  return s;
}

// Keys [lo, hi) that new token i of a sequence sees (window 0: none).
PKB_INDEX int clip_hi(const Seq& s, int i, int causal) {
  return causal ? least(s.len, s.pos0 + i + 1) : s.len;
}
PKB_INDEX int clip_lo(const Seq& s, int i, int window) {
  return window && s.pos0 + i >= window ? s.pos0 + i - window + 1 : 0;  // (no step leaves 32 bits)
}

// Key tiles of `kt` keys that hold the keys [lo, hi), from tile0 on: at least one,
// which may be masked throughout, so that rows without keys take the common path.
PKB_INDEX int tiles_of_keys(int lo, int hi, int kt, int& tile0) {
  tile0 = lo / kt;
  return most(1, (hi - tile0 * kt + kt - 1) / kt);
}
// Those that the tokens [first, last] need.
PKB_INDEX int clip_tiles(const Seq& s, int first, int last, int causal, int window, int kt, int& tile0) {
  return tiles_of_keys(clip_lo(s, first, window), clip_hi(s, last, causal), kt, tile0);
}

// A page of the pool, or num_pages (past its end, where tensor-map reads give
// zeros) for one that is not in it.
PKB_INDEX int clip_page(int page, int num_pages) {
  return page >= 0 && page < num_pages ? page : num_pages;
}

// Where the append puts a packed row: a sequence that has it, and its position there. kNoSequence: the row is of none;
// kMisplaced: the offsets are out of order or the sequence is shorter than its
// new tokens.
enum TokenPlace { kPlaced, kNoSequence, kMisplaced };
template <class Lengths>
PKB_INDEX TokenPlace place_token(const int* cu, int num_seqs, long long token, Lengths lens, int& seq,
                                 long long& position) {
  // With one new token each, which is what decoding steps have, it is sequence
  // `token`: looked at first, with loads that do not wait for one another.
  const int guess = token < num_seqs ? static_cast<int>(token) : num_seqs - 1;
  const int begin = cu[0], end = cu[num_seqs], from = cu[guess], to = cu[guess + 1], len = lens(guess);
  if (token < begin || token >= end) return kNoSequence;
  if (token >= from && token < to) {
    seq = guess;
    position = static_cast<long long>(len) - to + token;
    return position >= 0 ? kPlaced : kMisplaced;
  }
  int lo = 0, hi = num_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= token) lo = mid;
    else hi = mid;
  }
  seq = lo;
  position = static_cast<long long>(lens(lo)) - cu[lo + 1] + token;
  return token >= cu[lo] && token < cu[lo + 1] && position >= 0 ? kPlaced : kMisplaced;
}

}  // namespace paged
}  // namespace pkb200
