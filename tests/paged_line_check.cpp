// Host check of morello_amd/csrc/paged_line.h: the line of tiles of the attention over pages is cut so that every block of every tile falls to exactly one
// workgroup, in order, and what is noted of a cut tile for the putting together is so; and shares of 32 bits cover every line that the rule lets through.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include <random>
#include <vector>

#include "../morello_amd/csrc/paged_line.h"

using namespace mrl::paged;

struct Div {
  uint32_t d;
  uint32_t div(uint32_t n) const { return n / d; }
};
struct Form {
  const char *name;
  uint32_t bq_log2, block_log2, resident, least, second, overhead;
};
// The forms' numbers: 16 rows (most workgroups to a compute unit, and least) and 32, 128 rows of up to 64 and 128 dims.
constexpr Form FORMS[] = {{"16 rows", 4, 5, 4, 4, 12, 3}, {"16 rows, f32", 4, 5, 1, 4, 12, 3}, {"32 rows", 5, 5, 2, 4, 12, 3}, {"128 rows, 64 dims", 7, 6, 1, 8, 7, 7}, {"128 rows", 7, 6, 1, 8, 7, 4}};

struct Batch {
  Form form;
  uint32_t units, group, kv_heads, capacity, window, tokens;
  std::vector<Request> requests;
};

[[noreturn]] static void fail(const Batch &b, const char *what, long long x, long long y) {
  std::printf("%s, %u units, group %u, %u heads, %u keys, window %u, %u tokens, %zu requests (first: %d new, length %d): %s (%lld, %lld)\n", b.form.name, b.units, b.group,
              b.kv_heads, b.capacity, b.window, b.tokens, b.requests.size(), b.requests.empty() ? 0 : b.requests[0].n, b.requests.empty() ? 0 : b.requests[0].length, what, x, y);
  std::exit(1);
}

struct Line {
  Rules<Div> rules;
  uint64_t tiles = 0, blocks = 0, workers;
  long double length = 0;   // (not in the kernels' 64 bits)
  Cut cut;
};

static Line line_of(const Batch &b) {
  Line l = {{{b.group}, b.group, b.form.bq_log2, b.form.block_log2, b.capacity, b.window, b.form.overhead}, 0, 0, uint64_t(b.units) * b.form.resident, 0, {}};
  uint64_t sum = 0;
  for (const Request &q : b.requests) {
    if (!q.n) continue;
    const Lengths of = lengths_of(l.rules, q);
    l.tiles += uint64_t(of.tiles) * b.kv_heads, l.blocks += uint64_t(of.tiles) * most_blocks(l.rules, q, of.tiles) * b.kv_heads;
    sum += of.all() * b.kv_heads, l.length += (long double)of.all() * b.kv_heads;
  }
  l.cut = cut_of(l.tiles, sum, l.blocks, l.workers, b.form.least, b.form.second);
  return l;
}

// Shares cover the line: equal ones its length, those of the few tiles' way a piece each.
static void check_shares(const Batch &b) {
  const Line l = line_of(b);
  if (l.tiles == 0) return;
  long double most = l.length;
  if (l.cut.few) {
    most = 0;
    for (const Request &q : b.requests) {
      if (!q.n) continue;
      Lengths of = lengths_of(l.rules, q);
      make_few(&of, most_blocks(l.rules, q, of.tiles), l.cut.share);
      most += (long double)of.all() * b.kv_heads;
    }
  }
  if ((long double)l.cut.share * l.workers < most) fail(b, l.cut.few ? "few tiles: shares do not cover the line" : "equal shares do not cover the line", l.cut.share, (long long)most);
}

// Every tile, a workgroup's part after the other, as the kernels' Worker goes.
static bool check_dealing(const Batch &b) {
  const Line l = line_of(b);
  const uint64_t share = l.cut.share;
  struct Places {
    int begun = 0, carried = 0;   // pieces left in place 1, in place 0
  };
  std::vector<Places> places(l.workers);
  uint64_t at = 0;
  bool cut = false;
  for (const Request &q : b.requests) {
    if (!q.n) continue;
    Lengths of = lengths_of(l.rules, q);
    if (l.cut.few) make_few(&of, most_blocks(l.rules, q, of.tiles), l.cut.share);
    for (uint32_t head = 0; head < b.kv_heads; head++)
      for (uint32_t tile = 0; tile < of.tiles; tile++) {
        const Seen seen = seen_of(l.rules, q, tile << b.form.bq_log2, rows_of(l.rules, q, tile));
        const uint64_t length = of.of(tile);
        if (length < seen.blocks || length == 0) fail(b, "a tile is shorter on the line than its blocks", (long long)length, seen.blocks);
        uint32_t done = 0, pieces = 0, noted = 0;
        uint64_t last = 0;
        for (uint64_t w = at / share; w <= (at + length - 1) / share; w++) {
          const uint64_t from = w * share > at ? w * share - at : 0, to = (w + 1) * share < at + length ? (w + 1) * share - at : length;
          const uint32_t b0 = uint32_t(smaller<uint64_t>(from, seen.blocks)), b1 = uint32_t(smaller<uint64_t>(to, seen.blocks));
          if (!(b0 < b1 || (seen.blocks == 0 && from == 0))) continue;
          if (w >= l.workers) fail(b, "work past the last workgroup", (long long)w, (long long)l.workers);
          if (b0 != done) fail(b, "a block is dealt twice or not at all", b0, done);
          if (pieces && w != last + 1) fail(b, "a tile's pieces are not with neighbours", (long long)w, (long long)last);
          const bool whole = b0 == 0 && b1 == seen.blocks;
          if (!whole && b0 == 0) noted = pieces_behind(seen.blocks, b1, l.cut.share), places[w].begun++;
          if (!whole && b0 != 0) places[w].carried++;
          if (places[w].begun > 1 || places[w].carried > 1) fail(b, "two pieces in a place", (long long)w, 0);
          done = b1, pieces++, last = w;
        }
        if (done != seen.blocks || pieces == 0) fail(b, "blocks that nobody has", done, seen.blocks);
        if (pieces - 1 != noted) fail(b, "other pieces than noted", pieces - 1, noted);
        cut = cut || (pieces > 1 && !l.cut.few);
        at += length;
      }
  }
  return cut;
}

int main() {
  std::mt19937_64 rng(1);
  auto pick = [&](std::initializer_list<uint32_t> from) { return from.begin()[rng() % from.size()]; };
  auto upto = [&](uint32_t n) { return uint32_t(rng() % (uint64_t(n) + 1)); };

  int equal = 0;
  for (int i = 0; i < 12000; i++) {
    Batch b = {FORMS[rng() % 5], pick({32, 256, 256}), pick({1, 1, 2, 3, 4, 7, 8, 16, 40}), pick({1, 2, 3, 8}), pick({16, 48, 592, 4096, 40000}), pick({0, 0, 1, 20, 100, 1024, 0xffffffffu}), 0, {}};
    const uint32_t requests = 1 + upto(pick({0, 3, 20, 150})), longest = pick({1, 1, 8, 100, 1500});
    for (uint32_t r = 0; r < requests; r++) {
      const int32_t n = int32_t(upto(pick({1, longest, longest})));
      // lengths that the table holds, past it, below the new tokens
      const int32_t length = rng() % 8 ? int32_t(upto(b.capacity)) + n : rng() % 2 ? int32_t(upto(3 * b.capacity)) : int32_t(upto(20)) - 10;
      b.requests.push_back({n, int32_t(b.tokens), length}), b.tokens += uint32_t(n);
    }
    check_shares(b);
    equal += check_dealing(b);
  }
  if (equal < 1000) std::printf("cut tiles on a line of equal shares in %d batches only\n", equal), std::exit(1);

  // As many new tokens as there may be, over tables of any size; as long as the rule for the tiles lets through.
  int let = 0;
  for (const Form &form : FORMS)
    for (uint32_t units : {32u, 64u, 256u})
      for (uint32_t group : {1u, 2u, 4u, 16u, 128u, 255u})
        for (uint32_t kv_heads : {1u, 8u, 128u, 4096u, 65535u})
          for (uint32_t capacity : {16u, 4096u, 1u << 20, 0x7fff0000u})
            for (uint32_t window : {0u, 4096u, 1u << 22, 0xffffffffu})
              for (uint32_t tokens : {1u, 8000u, 1u << 20, 1u << 23})
                for (uint32_t requests : {1u, 3u, 15u, 1000u}) {
                  if (requests > tokens || uint64_t(tokens) * group >= 1u << 31 || !line_fits(tokens, requests, group, kv_heads, capacity, units)) continue;
                  let++;
                  Batch b = {form, units, group, kv_heads, capacity, window, tokens, {}};
                  const int32_t n = int32_t(tokens / requests);
                  for (int32_t length : {n, int32_t(capacity), 0x7fffffff}) {   // a prompt that begins, one that fills the table, one far past it
                    b.requests.assign(requests, {n, 0, length});
                    check_shares(b);
                  }
                  // few tiles of long requests, nearly as many as there are workgroups
                  const uint32_t few = units * form.resident / smaller(kv_heads, 1000u);
                  if (tokens == 1 && few && line_fits(few, few, group, kv_heads, capacity, units)) {
                    b.tokens = few, b.requests.assign(few, {1, 0, int32_t(capacity)});
                    check_shares(b);
                    b.tokens = few - 1, b.requests.pop_back();
                    check_shares(b);
                  }
                }
  if (let < 1000) std::printf("%d sizes let through only\n", let), std::exit(1);
  std::printf("paged line ok\n");
}
