// The line of tiles of the attention over pages (attention_paged.h): which keys a tile sees, how long it is on the line, and where the line is cut.  Whole
// numbers alone, for the kernels and for a host check.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define MRL_LINE_HD __host__ __device__
#else
#define MRL_LINE_HD
#endif

namespace mrl {
namespace paged {

// A request: its new tokens, their first row, and its length.
struct Request {
  int32_t n, start, length;
};

// What is the same for all tiles of a call.  Div: divides by `group` with div().
template <class Div>
struct Rules {
  Div by_group;
  uint32_t group, bq_log2, block_log2;   // query heads of a key/value head; rows of a tile, keys of a block
  uint32_t capacity, window, overhead;   // keys that a row of the page table has columns for; what a tile costs besides its blocks, in blocks
};

template <class T>
MRL_LINE_HD inline T smaller(T x, T y) { return x < y ? x : y; }
template <class T>
MRL_LINE_HD inline T larger(T x, T y) { return x > y ? x : y; }

// Keys that some row of rows row0 .. row0 + rows - 1 of a request sees lie in [begin, end), in so many blocks; `at`: the place of the request's token 0 among
// its keys (may be below zero).
struct Seen {
  int32_t at;
  uint32_t begin, end, blocks;
};
template <class Div>
MRL_LINE_HD inline Seen seen_of(const Rules<Div> &k, const Request &q, uint32_t row0, uint32_t rows) {
  Seen s;
  const int32_t known = smaller(larger(q.length, int32_t(0)), int32_t(k.capacity));
  s.at = int32_t(larger(int64_t(q.length) - q.n, -(int64_t(1) << 30)));
  const int64_t last = int64_t(s.at) + k.by_group.div(row0 + rows - 1), first = int64_t(s.at) + k.by_group.div(row0);
  s.end = uint32_t(smaller(larger(last + 1, int64_t(0)), int64_t(known)));
  s.begin = k.window ? uint32_t(smaller(larger(first - int64_t(k.window) + 1, int64_t(0)), int64_t(s.end))) : 0;
  s.blocks = s.end > s.begin ? ((s.end - 1) >> k.block_log2) - (s.begin >> k.block_log2) + 1 : 0;
  return s;
}
template <class Div>
MRL_LINE_HD inline uint32_t tiles_of(const Rules<Div> &k, const Request &q) {
  return (uint32_t(q.n) * k.group + (1u << k.bq_log2) - 1) >> k.bq_log2;
}
// Rows of a tile, the last of which may have fewer.
template <class Div>
MRL_LINE_HD inline uint32_t rows_of(const Rules<Div> &k, const Request &q, uint32_t tile) {
  return smaller(uint32_t(q.n) * k.group - (tile << k.bq_log2), 1u << k.bq_log2);
}

// floor(x / y) for x < 2^52 (a quotient that is no whole number is at least 1 / y off one: more than a rounding in 64 bits); 2^32 - 1 for what is more.
MRL_LINE_HD inline uint32_t quotient(uint64_t x, uint64_t y) { return uint32_t(smaller(double(x) / double(y), 4294967295.0)); }
// 1 / x to 22 bits or more.
MRL_LINE_HD inline float reciprocal(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_rcpf(x);
#else
  return 1.0f / x;
#endif
}

// A request's tiles on the line, of one head.
struct Lengths {
  uint32_t tiles;
  uint32_t first, slope, most, grown;   // tile t: first + t * slope / 256 for t below `grown`, then `most`; in the few tiles' way `most` for all

  MRL_LINE_HD uint64_t before(uint32_t t) const {   // of the tiles before tile t
    const uint64_t x = smaller(t, grown);
    return x * first + ((x * (x - (x != 0)) / 2 * slope) >> 8) + uint64_t(t - uint32_t(x)) * most;
  }
  MRL_LINE_HD uint32_t of(uint32_t t) const { return uint32_t(before(t + 1) - before(t)); }
  MRL_LINE_HD uint64_t all() const { return before(tiles); }
};
// A tile has at most (keys it sees) / 2^block_log2 + 2 blocks, and tile t sees at most at + (t + 1) * bq / G + 1 keys, or window + bq / G + 1, or what the table has
// columns for.  (Two more, as the 256ths of `slope` are rounded where they are summed.)
template <class Div>
MRL_LINE_HD inline Lengths lengths_of(const Rules<Div> &k, const Request &q) {
  Lengths l;
  const uint32_t bq = 1u << k.bq_log2, step = bq / k.group + 1, more = 4 + k.overhead;
  const uint32_t at = uint32_t(smaller(larger(int64_t(q.length) - q.n, int64_t(0)), int64_t(k.capacity)));
  l.tiles = tiles_of(k, q);
  l.slope = ((bq * 256 / k.group) >> k.block_log2) + 1;
  l.first = (uint32_t((uint64_t(at) + step) >> k.block_log2)) + more;
  // The first of them grow, the others have as many as a window or the table allows.  Where the one ends and the other begins is rounded in 32 bits: a tile has its blocks on
  // either side.
  const uint32_t keys = k.window ? smaller(k.window, k.capacity) : k.capacity;
  l.most = ((keys + step) >> k.block_log2) + more;
  l.grown = l.first < l.most ? uint32_t(smaller(float(l.most - l.first) * (256.0f * reciprocal(float(l.slope))), 4.0e9f)) + 1 : 0;
  return l;
}
// In the few tiles' way, each as long as the longest can be.
template <class Div>
MRL_LINE_HD inline uint32_t most_blocks(const Rules<Div> &k, const Request &q, uint32_t tiles) {
  const Seen last = seen_of(k, q, (tiles - 1) << k.bq_log2, rows_of(k, q, tiles - 1));
  if (tiles == 1) return larger(last.blocks, 1u);
  return k.window ? smaller(((last.end + 1) >> k.block_log2) + 2, uint32_t((uint64_t(k.window) + (1u << k.bq_log2) / k.group + 1) >> k.block_log2) + 2)
                  : larger(last.blocks, 1u);
}
// .. rounded up to whole shares.
MRL_LINE_HD inline void make_few(Lengths *l, uint32_t most, uint32_t share) { l->grown = 0, l->most = quotient(uint64_t(most) + share - 1, share) * share; }

// A workgroup's share of the line, and whether the tiles lie on it in the few tiles' way.  `tiles`, `line`, `blocks`: of all requests and heads, the last two the line's
// length and the blocks in the few tiles' way; the others are the Work's.
struct Cut {
  uint32_t share;
  bool few;
};
MRL_LINE_HD inline Cut cut_of(uint64_t tiles, uint64_t line, uint64_t blocks, uint64_t workers, uint32_t least, uint32_t second) {
  Cut c = {larger(quotient(line + workers - 1, workers), 1u), false};
  // A piece to each, where that is no longer than equal shares and the second piece that they may come to.  (More than the second product are surely longer, and not divided.)
  if (tiles < workers && blocks <= (uint64_t(c.share) + second) * (workers - tiles)) {
    const uint32_t spare = uint32_t(workers - tiles), single = larger((quotient(blocks + spare - 1, spare) + least - 1) / least, 1u) * least;
    c.few = single <= c.share + second;
    if (c.few) c.share = single;
  }
  return c;
}
// How many workgroups have a piece of a tile of `blocks` behind the one that begins it and whose share ends before block `b1`.
MRL_LINE_HD inline uint32_t pieces_behind(uint32_t blocks, uint32_t b1, uint32_t share) { return 1 + (blocks - 1 - b1) / share; }

// Whether shares of 31 bits cover the line of any batch of so many tokens in all, on at least `units` workgroups: tiles, at most so many, times the longest of them
// (lengths_of: its blocks are of 32 keys or more; up to 11 for what a tile costs besides, and two where the keys of its other tokens come to some).
inline bool line_fits(uint32_t tokens, uint32_t requests, uint32_t group, uint32_t kv_heads, uint64_t capacity, uint32_t units) {
  return (double(tokens) * group / 16 + requests) * kv_heads * (double(capacity) / 32 + 16) < double(units) * double(1u << 31);
}

}  // namespace paged
}  // namespace mrl
