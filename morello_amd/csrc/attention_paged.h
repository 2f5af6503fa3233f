// What the kernels of the attention over pages share: the tiles of query rows, how work is dealt to workgroups, and where partial results go
// (attention_paged.hip, attention_paged_keys.hip, attention_paged_chunk.hip).
//
// A TILE is up to 16, 32 or 128 query rows of one request that read the same key/value head: row i of a request is its token i / G at query head i % G of the
// G = q_heads / kv_heads that share it, so that keys and values are fetched once for all of them.  A tile's keys come in BLOCKS; how many it has
// follows from the lengths, which are on the device.  So a launch of one workgroup (k_paged_attn_deal) lays the tiles on a line, request by request, head by
// head (what shares a head's keys and values runs beside each other, on one XCD, and finds them in its L2), and cuts the line in equal shares:
//   few tiles for the workgroups: a tile's length on the line is its blocks rounded up to the share, and the share so small that
//     the pieces are at most as many as workgroups: each has one piece;
//   else: a tile's length is its blocks and some for what a tile costs besides, the share what all come to over the workgroups.
// A workgroup's share may begin and end inside a tile: there it leaves a partial result (O, m, l: the sum of the values, the reference in the
// exponent's base of two, the denominator) instead of the tile's rows, one for the tile it does not begin (place 0) and one for the tile it
// begins and does not end (place 1).  Who begins a tile and does not end it describes it for a last launch, which puts the pieces together in their order.  No
// atomics: results do not depend on who is first.  Where a table holds so few keys that a workgroup does a request's head in some rounds, there is
// one to each and nothing is dealt (`direct`).
// (Pieces off a queue, whoever is free: no faster where memory bounds them -- of equal shares of a decoding step's keys the first was done after 115 us, the last
// after 157, but whoever is done leaves its bandwidth to the others -- and slower where pieces are short.)
#pragma once
#include "attention.h"
#include "paged.h"

namespace mrl {
namespace paged {

constexpr uint32_t MOST_WORKERS = 1024;   // threads of the dealing's workgroup

// What the dealing leaves in the workspace.
struct Line {
  uint64_t share;      // of each workgroup
  uint32_t tiles;      // that are noted (of all heads together one)
  uint32_t unused[5];
};
struct Start {         // of a workgroup's share: tile, head, place in the tile
  uint32_t tile, head, at, unused;
};
struct Tile {
  uint32_t request, row0, rows;      // rows row0 .. row0 + rows - 1 of the request
  int32_t start, at;                 // the tensors' row of the request's token 0, and its place among the keys (may be below zero)
  uint32_t begin, end;               // keys that some row sees lie in [begin, end)
  uint32_t blocks, length;           // their blocks, and the tile's length on the line
  uint32_t first, behind;            // tiles of its request (of those noted together): these follow each other once for every head
  uint32_t unused[5];
};

struct Work {
  uint32_t min_rows, max_rows;   // requests of so many query rows; others' are left to another kernel
  bool direct;                   // a workgroup to each (request, head): nothing is dealt
  uint32_t workers;
  uint32_t bq_log2, block_log2;  // of a tile's rows, of a block's keys
  uint32_t least;                // the least blocks that a tile is cut to where workgroups are to spare
  uint32_t overhead, second;     // what a tile costs besides its blocks, in blocks, where the chip has all it can do; what a second piece costs a workgroup that has no other
  uint32_t most_tiles;           // that there is room to note
  Line *line;
  Start *starts;                 // [workers]
  Tile *tiles;                   // [most_tiles]
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

__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline uint64_t uniform(uint64_t x) { return uint64_t(uniform(uint32_t(x >> 32))) << 32 | uniform(uint32_t(x)); }

// A request: its new tokens (0: none of this kernel's), their first row, and its length.
struct Request {
  int32_t n, start, length;
};
__device__ inline Request read_request(const PagedAttnArgs &p, const Work &w, uint32_t r) {
  const int32_t most = int32_t(p.tokens);
  const int32_t s0 = min(max(p.starts[r], 0), most), s1 = min(max(p.starts[r + 1], 0), most);
  Request q = {max(s1 - s0, 0), s0, p.lengths[r]};
  const uint32_t rows = uint32_t(q.n) * p.group;
  if (rows < w.min_rows || rows > w.max_rows) q.n = 0;
  return q;
}

// The keys that a tile sees, and their blocks.
__device__ inline Tile measure(const PagedAttnArgs &p, FastDiv by_group, const Request &q, uint32_t row0, uint32_t rows, uint32_t block_log2) {
  Tile t = {};
  const int32_t known = min(max(q.length, 0), int32_t(p.width * p.page_size));
  t.row0 = row0, t.rows = rows, t.start = q.start, t.at = int32_t(max(int64_t(q.length) - q.n, -(int64_t(1) << 30)));
  const int64_t last = int64_t(t.at) + by_group.div(row0 + rows - 1), first = int64_t(t.at) + by_group.div(row0);
  t.end = uint32_t(min(max(last + 1, int64_t(0)), int64_t(known)));
  t.begin = p.window ? uint32_t(min(max(first - int64_t(p.window) + 1, int64_t(0)), int64_t(t.end))) : 0;
  t.blocks = t.end > t.begin ? ((t.end - 1) >> block_log2) - (t.begin >> block_log2) + 1 : 0;
  return t;
}

// floor(x / y) for x < 2^52 and a quotient below 2^32 (a quotient that is no whole number is at least 1 / y off one: more than a rounding in 64 bits).
__device__ inline uint32_t quotient(uint64_t x, uint64_t y) { return uint32_t(double(x) / double(y)); }

// One tile's piece, in scalar registers.
struct Piece {
  uint32_t request, head, row0, rows;
  int32_t start, at;
  uint32_t begin, end, blocks;
  uint32_t b0, b1;   // its blocks, counted from the one that holds `begin`
  __device__ bool whole() const { return b0 == 0 && b1 == blocks; }
};

// A workgroup's way along its share of the line; everybody calls it.
struct Worker {
  uint32_t number = xcd_run(blockIdx.x, gridDim.x);
  uint32_t tile, head, at;   // where it stands
  uint32_t left;             // of its share
  bool described = false;

  __device__ Worker(const Work &w) {
    const volatile Start *s = w.starts + number;
    tile = uniform(s->tile), head = uniform(s->head), at = uniform(s->at), left = uniform(uint32_t(w.line->share));
  }
  // The next piece that has something to do; false: there is none.
  __device__ bool next(const Kernargs &k, Piece *out) {
    const uint32_t tiles = uniform(k.w.line->tiles);
    while (left && tile < tiles) {
      const volatile Tile *t = k.w.tiles + tile;
      const uint32_t blocks = uniform(t->blocks), length = uniform(t->length), first = uniform(t->first), behind = uniform(t->behind);
      out->request = uniform(t->request), out->head = head, out->row0 = uniform(t->row0), out->rows = uniform(t->rows), out->start = uniform(int32_t(t->start));
      out->at = uniform(int32_t(t->at)), out->begin = uniform(t->begin), out->end = uniform(t->end), out->blocks = blocks;
      out->b0 = min(at, blocks), out->b1 = min(at + min(left, length - at), blocks);
      const bool any = out->b0 < out->b1 || (blocks == 0 && at == 0);
      left -= min(left, length - at), at = 0, tile++;
      if (tile == behind && head + 1 < k.p.kv_heads) tile = first, head++;
      else if (tile == behind) head = 0;
      if (any) return true;
    }
    return false;
  }
  // Where a piece that is not its tile leaves its partial result.
  __device__ float *place(const Work &w, const Piece &t, uint32_t piece_floats) const { return w.partials + (uint64_t(number) * 2 + (t.b0 == 0)) * piece_floats; }
  // By one thread, of a tile that this workgroup begins and others end: how many of them, and which rows.  Its last block lies `b1 .. blocks` behind this share's end, but
  // for the last share's.
  __device__ void describe(const Work &w, const Piece &t) const {
    uint32_t *d = w.merges + number * 8;
    d[0] = 1 + quotient(t.blocks - 1 - t.b1, w.line->share), d[1] = uint32_t(t.start), d[2] = t.row0, d[3] = t.rows, d[4] = t.head;
  }
};

// In a `direct` launch: the workgroup's one tile, as a whole; false: it has none.
__device__ inline bool direct_piece(const Kernargs &k, Piece *out) {
  const uint32_t worker = xcd_run(blockIdx.x, gridDim.x), request = worker / k.p.kv_heads;
  Request q = read_request(k.p, k.w, request);
  q.n = uniform(q.n), q.start = uniform(q.start), q.length = uniform(q.length);
  if (!q.n) return false;
  const Tile t = measure(k.p, k.by_group, q, 0, uint32_t(q.n) * k.p.group, k.w.block_log2);
  *out = {request, worker - request * k.p.kv_heads, t.row0, t.rows, t.start, t.at, t.begin, t.end, t.blocks, 0, t.blocks};
  return true;
}

// Floats of a row of a partial result: O of the head dim the kernels are built for, reference, denominator, and two that are not used.
inline uint32_t row_floats(const PagedAttnArgs &a) { return (a.head_dim <= 64 ? 64 : 128) + 4; }
// attention_paged_chunk.hip: tiles of 128 rows, bf16.  The Work's fixed numbers, and the launch.
void chunk_work(const PagedAttnArgs &a, Work *w);
hipError_t launch_chunk(const PagedAttnArgs &a, const Work &work, hipStream_t stream);
// attention_paged_keys.hip, for qb = 1 or 2: tiles of 16 or 32 rows.
void keys_work(const PagedAttnArgs &a, int qb, Work *w);
hipError_t launch_keys(const PagedAttnArgs &a, const Work &work, int qb, hipStream_t stream);

}  // namespace paged
}  // namespace mrl
