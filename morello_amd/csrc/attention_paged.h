// What the kernels of the attention over pages share: the tiles of query rows, how work is dealt to workgroups, and where partial results go
// (attention_paged.hip, attention_paged_keys.hip, attention_paged_chunk.hip).
//
// A TILE is up to 16, 32 or 128 query rows of one request that read the same key/value head: row i of a request is its token i / G at query head i % G of the
// G = q_heads / kv_heads that share it, so that keys and values are fetched once for all of them.  A tile's keys come in BLOCKS; how many it has
// follows from the lengths, which are on the device.  The host chooses a number of workgroups, and each finds its own share from the lengths before it begins.
//
// All tiles lie on a line, request by request, head by head (what shares a head's keys and values runs beside each other, on one XCD, and finds them in its
// L2), and the line is cut in equal shares:
//   few tiles for the workgroups: a tile's length on the line is its request's most blocks rounded up to the share, and the share so small that the
//     pieces are at most as many as workgroups: each has one piece;
//   else: a tile's length is its blocks and some for what a tile costs besides.  Tile t's keys end bq / G tokens behind tile t - 1's, so lengths grow evenly up to what
//     a window or the table allows; taken as that (at least the tile's blocks), the place of any tile is a formula (paged_line.h), and no list of tiles is needed.
// A workgroup's share may begin and end inside a tile: there it leaves a partial result (O, m, l: the sum of the values, the reference in the
// exponent's base of two, the denominator) instead of the tile's rows, one for the tile it does not begin (place 0) and one for the tile it
// begins and does not end (place 1).  Who begins a tile and does not end it describes it for a last launch, which puts the pieces together in their order.  No
// atomics: results do not depend on who is first.  Where a table holds so few keys that a workgroup does a request's head in some rounds, there is
// one to each and nothing is shared out (`direct`).
//
// Tried and left: the dealing in a launch of its own that notes every tile's place (9 us and a gap in front of a decoding step; here 3 us of the kernel); pieces off a
// queue, whoever is free (no faster where memory bounds them: of equal shares of a decoding step's keys the first was done after 115 us, the last after
// 157, but whoever is done leaves its bandwidth to the others; slower where pieces are short).
#pragma once
#include "attention.h"
#include "paged.h"
#include "paged_line.h"

namespace mrl {
namespace paged {

struct Work {
  bool once;                     // no request is expected to have more than a tile: its keys and values are read once
  bool direct;                   // a workgroup to each (request, head): nothing is dealt
  uint32_t workers;
  uint32_t bq_log2, block_log2;  // of a tile's rows, of a block's keys
  uint32_t least;                // the least blocks that a tile is cut to where workgroups are to spare
  uint32_t overhead, second;     // what a tile costs besides its blocks, in blocks, where the chip has all it can do; what a second piece costs a workgroup that has no other
  uint32_t *merges;              // [workers][8]: see describe()
  float *partials;               // [workers][2][rows of a tile][row_floats]
};

// A kernel's arguments.  They are read again where they are wanted (kernargs()): kept in scalar registers over the loops, they would push the loops' own
// numbers out (an early form had 400 of them moved to lanes of vector registers, and those to memory).
struct Kernargs {
  PagedAttnArgs p;
  Work w;
  FastDiv by_group, by_page16;
  float c;   // scale * log2 e
};
__device__ inline const Kernargs &kernargs() {
  typedef const __attribute__((address_space(4))) void *Segment;
  Segment s = (Segment)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(s));
  return *(const Kernargs *)s;
}

// attn::dma16_ordered for what is read once: it leaves the caches to others.
__device__ inline void dma16_once(__amdgpu_buffer_rsrc_t from, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" : : "s"(lds_addr), "v"(voff), "s"(from) : "memory");
}

__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline uint64_t uniform(uint64_t x) { return uint64_t(uniform(uint32_t(x >> 32))) << 32 | uniform(uint32_t(x)); }

// Of values' bits (two of bf16, one of f32): something but zero where one is infinite or no number: an exponent of ones runs over into the sign's bit.
template <bool BF16>
__device__ inline uint32_t not_finite(attn::v4i x) {
  constexpr uint32_t EXPONENT = BF16 ? 0x7f807f80 : 0x7f800000, ONE = BF16 ? 0x00800080 : 0x00800000;
  uint32_t over = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) over |= (uint32_t(x[j]) & EXPONENT) + ONE;
  return over & (BF16 ? 0x80008000u : 0x80000000u);
}

__device__ inline Rules<FastDiv> rules(const Kernargs &k) { return {k.by_group, k.p.group, k.w.bq_log2, k.w.block_log2, k.p.width * k.p.page_size, k.p.window, k.w.overhead}; }

__device__ inline Request read_request(const PagedAttnArgs &p, uint32_t r) {
  const int32_t most = int32_t(p.tokens);
  const int32_t s0 = min(max(p.starts[r], 0), most), s1 = min(max(p.starts[r + 1], 0), most);
  return {max(s1 - s0, 0), s0, p.lengths[r]};
}

// One tile's piece, in scalar registers.
struct Piece {
  uint32_t request, head, row0, rows;   // rows row0 .. row0 + rows - 1 of the request, at key/value head `head`
  int32_t start, at;                    // the tensors' row of the request's token 0, and its place among the keys (may be below zero)
  uint32_t begin, end, blocks;          // keys that some row of the tile sees lie in [begin, end), in so many blocks
  uint32_t b0, b1;                      // the piece's, counted from the one that holds `begin`
  __device__ bool whole() const { return b0 == 0 && b1 == blocks; }
};
// Tile `tile` of a request, as a whole.
__device__ inline Piece tile_of(const Kernargs &k, const Request &q, uint32_t tile) {
  Piece t = {};
  const auto r = rules(k);
  t.row0 = tile << r.bq_log2, t.rows = rows_of(r, q, tile), t.start = q.start;
  const Seen s = seen_of(r, q, t.row0, t.rows);
  t.at = s.at, t.begin = s.begin, t.end = s.end, t.blocks = t.b1 = s.blocks;
  return t;
}

__device__ inline uint32_t of_lane(uint32_t x, int lane) { return uint32_t(__builtin_amdgcn_readlane(int(x), lane)); }
__device__ inline uint64_t of_lane(uint64_t x, int lane) { return uint64_t(of_lane(uint32_t(x >> 32), lane)) << 32 | of_lane(uint32_t(x), lane); }

// A workgroup's way along its share of the line; every wave goes it for itself, so that no wave waits for another.
struct Worker {
  uint32_t number = xcd_run(blockIdx.x, gridDim.x);
  uint32_t request = 0xffffffffu, head = 0, tile = 0, at = 0;   // where it stands
  Request q = {0, 0, 0};                                        // the request there, and its tiles
  Lengths l = {};
  uint32_t share = 1, left = 0;
  bool few = false, described = false;

  __device__ Lengths lengths(const Kernargs &k, const Request &q) const {
    const auto r = rules(k);
    Lengths l = lengths_of(r, q);
    if (few) make_few(&l, most_blocks(r, q, l.tiles), share);
    return l;
  }

  // Takes the request that lane `it` has, of those from `first` on.
  __device__ void stand(const Request &mine, const Lengths &of_mine, uint32_t first, int it) {
    request = first + it;
    q = {int32_t(of_lane(uint32_t(mine.n), it)), int32_t(of_lane(uint32_t(mine.start), it)), int32_t(of_lane(uint32_t(mine.length), it))};
    l = {of_lane(of_mine.tiles, it), of_lane(of_mine.first, it), of_lane(of_mine.slope, it), of_lane(of_mine.most, it), of_lane(of_mine.grown, it)};
  }

  // Finds its start, a lane to a request.
  __device__ Worker(const Kernargs &k) {
    const uint32_t lane = threadIdx.x & 63, requests = k.p.requests;
    const uint64_t heads = k.p.kv_heads, workers = k.w.workers;
    // How many tiles, how long the line, how many blocks in the few tiles' way.
    uint64_t tiles = 0, line = 0, blocks = 0;
    Request mine = {0, 0, 0};
    for (uint32_t r = lane; r < requests; r += 64) {
      mine = read_request(k.p, r);
      if (!mine.n) continue;
      const auto rule = rules(k);
      const Lengths l = lengths_of(rule, mine);
      tiles += l.tiles, line += l.all(), blocks += uint64_t(l.tiles) * most_blocks(rule, mine, l.tiles);
    }
    tiles = of_lane(sums_up_to(tiles), 63) * heads, line = of_lane(sums_up_to(line), 63) * heads, blocks = of_lane(sums_up_to(blocks), 63) * heads;
    const Cut cut = cut_of(tiles, line, blocks, workers, k.w.least, k.w.second);
    share = uniform(cut.share), few = uniform(uint32_t(cut.few));
    // The request that holds its start.
    const uint64_t from = uint64_t(share) * number;
    uint64_t base = 0;
    for (uint32_t r0 = 0; r0 < requests; r0 += 64) {
      if (requests > 64) {
        mine = {0, 0, 0};
        if (r0 + lane < requests) mine = read_request(k.p, r0 + lane);
      }
      Lengths of_mine = {};
      uint64_t length = 0;
      if (mine.n) of_mine = lengths(k, mine), length = of_mine.all();
      const uint64_t sum = sums_up_to(length * heads), off = base + sum - length * heads;
      const bool here = mine.n && from >= off && from < base + sum;
      const uint64_t where = __ballot(here);
      if (where) {
        const int it = __builtin_ctzll(where);
        stand(mine, of_mine, r0, it);
        const uint64_t all = of_lane(length, it), in_request = from - of_lane(off, it);
        head = min(uniform(quotient(in_request, all)), k.p.kv_heads - 1), left = share;   // (past it only where starts that fall make a line that 64 bits do not hold)
        // The tile that holds the place in the head: the last that begins at or before it, found among 64 at a time.
        const uint64_t in_head = in_request - head * all;
        uint32_t step = 1;
        while (step * 64 < l.tiles) step *= 64;
        for (;; step /= 64) {
          const uint32_t t = tile + lane * step;
          tile += (__builtin_popcountll(__ballot(t < l.tiles && l.before(t) <= in_head)) - 1) * step;   // (of tiles that rise: the first lanes)
          if (step == 1) break;
        }
        at = uniform(uint32_t(in_head - l.before(tile)));
        break;
      }
      base += of_lane(sum, 63);
    }
  }

  // The next piece that has something to do; false: there is none.
  __device__ bool next(const Kernargs &k, Piece *out) {
    while (left) {
      const uint32_t length = uniform(l.of(tile));
      Piece t = tile_of(k, q, tile);
      t.request = request, t.head = head, t.b0 = min(at, t.blocks), t.b1 = min(at + min(left, length - at), t.blocks);
      const bool any = t.b0 < t.b1 || (t.blocks == 0 && at == 0);
      left -= min(left, length - at), at = 0, tile++;
      if (tile == l.tiles) {
        tile = 0, head++;
        if (head == k.p.kv_heads && left) {   // the next request with new tokens
          head = 0;
          const uint32_t lane = threadIdx.x & 63;
          uint64_t some = 0;
          Request mine = {0, 0, 0};
          for (request++; request < k.p.requests; request += 64) {
            mine = {0, 0, 0};
            if (request + lane < k.p.requests) mine = read_request(k.p, request + lane);
            some = __ballot(mine.n != 0);
            if (some) break;
          }
          left = some ? left : 0;
          if (some) stand(mine, mine.n ? lengths(k, mine) : Lengths{}, request, __builtin_ctzll(some));
        }
      }
      if (any) {
        *out = t;
        out->start = uniform(t.start), out->at = uniform(t.at), out->begin = uniform(t.begin), out->end = uniform(t.end), out->blocks = uniform(t.blocks);
        out->b0 = uniform(t.b0), out->b1 = uniform(t.b1), out->row0 = uniform(t.row0), out->rows = uniform(t.rows);
        return true;
      }
    }
    return false;
  }
  // Where a piece that is not its tile leaves its partial result.
  __device__ float *place(const Work &w, const Piece &t, uint32_t piece_floats) const { return w.partials + (uint64_t(number) * 2 + (t.b0 == 0)) * piece_floats; }
  // By one thread, of a tile that this workgroup begins and others end: how many of them, and which rows.  (Its share ends behind block b1 - 1.)
  __device__ void describe(const Work &w, const Piece &t) const {
    uint32_t *d = w.merges + number * 8;
    d[0] = pieces_behind(t.blocks, t.b1, share), d[1] = uint32_t(t.start), d[2] = t.row0, d[3] = t.rows, d[4] = t.head;
  }
};

// In a `direct` launch: a request's head to a workgroup, tile after tile (one, where max_new says what is so).
struct DirectWorker {
  uint32_t request, head, tile = 0;
  Request q;
  __device__ DirectWorker(const Kernargs &k) {
    const uint32_t worker = xcd_run(blockIdx.x, gridDim.x);
    request = worker / k.p.kv_heads, head = worker - request * k.p.kv_heads;
    q = read_request(k.p, request);
    q.n = uniform(q.n), q.start = uniform(q.start), q.length = uniform(q.length);
  }
  __device__ bool next(const Kernargs &k, Piece *out) {
    if (uint64_t(tile) << k.w.bq_log2 >= uint64_t(q.n) * k.p.group) return false;
    *out = tile_of(k, q, tile++);
    out->request = request, out->head = head;
    return true;
  }
};

// Floats of a row of a partial result: O of the head dim the kernels are built for, reference, denominator, and two that are not used.
inline uint32_t kernel_dims(const PagedAttnArgs &a) { return a.head_dim <= 64 ? 64 : a.dtype == MRL_F32 && a.head_dim <= 96 ? (a.head_dim <= 80 ? 80 : 96) : 128; }
inline uint32_t row_floats(const PagedAttnArgs &a) { return kernel_dims(a) + 4; }
// attention_paged_chunk.hip: tiles of 128 rows, bf16.  The Work's fixed numbers, and the launch.
void chunk_work(const PagedAttnArgs &a, Work *w);
hipError_t launch_chunk(const PagedAttnArgs &a, const Work &work, hipStream_t stream);
// attention_paged_keys.hip, for qb = 1 or 2: tiles of 16 or 32 rows.
void keys_work(const PagedAttnArgs &a, int qb, Work *w);
hipError_t launch_keys(const PagedAttnArgs &a, const Work &work, int qb, hipStream_t stream);

}  // namespace paged
}  // namespace mrl
