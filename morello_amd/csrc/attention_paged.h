// What the kernels of the attention over pages share: the tiles of query rows, how work is dealt to workgroups, and where
// partial results go (attention_paged.hip, attention_paged_keys.hip).
//
// A TILE is up to `BQ` query rows of one request that read the same key/value head: row i of a request is its token i / G at query head
// i % G of the G = q_heads / kv_heads that share it, so that keys and values are fetched once for all of them.  A tile's keys come in
// BLOCKS; how many it has follows from the lengths, which are on the device.
//
// The host chooses a number of workgroups; each finds its own share by itself, from the same lengths (some thousand bytes out of a cache,
// no launch before the kernel).  Shares are equal runs of one line on which the tiles lie, request by request, tile by tile, head by head:
//   few tiles for the workgroups: a tile's length on the line is its blocks rounded up to the share, and the share so small that
//     the pieces are just as many as workgroups: each has one piece, a tile's pieces meet in the merging launch;
//   else: a tile's length is its blocks and some for what a tile costs besides, the share what all come to over the workgroups.
// A workgroup's run may begin and end inside a tile: there it leaves a partial result (O, m, l: the sum of the values, the reference in the
// exponent's base of two, the denominator) instead of the tile's rows, one for the tile it does not begin (place 0) and one for the tile it
// does not end (place 1).  Who begins a tile and does not end it describes it for the merging launch.  No atomics: results do not
// depend on who is first.
#pragma once
#include "attention.h"
#include "paged.h"

namespace mrl {
namespace paged {

constexpr uint32_t OVERHEAD_KEYS = 96;   // what a tile costs besides its blocks, as keys: the trips to memory before its first block, and its results

struct Work {
  uint32_t min_rows, max_rows;   // requests of so many query rows; others' are left to another kernel
  bool single;                   // no such request has more than a tile
  bool direct;                   // a workgroup to each (request, head): nothing is shared out
  uint32_t workers;
  uint32_t round_blocks;         // blocks that a workgroup does at a time
  float *partials;               // [worker][2][BQ][row_floats]
  uint32_t *tiles;               // [worker][8]: see describe()
};

// One tile's piece for this workgroup.
struct Piece {
  uint32_t request, head, row0, rows;   // rows row0 .. row0 + rows - 1 of the request, at key/value head `head`
  int32_t start, at;                    // the tensors' row of the request's token 0, and its place among the keys (may be below zero)
  uint32_t begin, end;                  // keys that some row sees lie in [begin, end)
  uint32_t first_block, blocks;         // their blocks, and of them
  uint32_t b0, b1;                      // this piece's, counted from first_block
  uint32_t v0, v1;                      // workers that have pieces of it
};

__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// floor(x / y) for x < 2^52 and a quotient below 2^32 (a quotient that is no whole number is at least 1 / y off one: more than a rounding in 64 bits).
__device__ inline uint32_t quotient(uint64_t x, uint64_t y) { return uint32_t(double(x) / double(y)); }

template <int TH, int BQ, int BK>
struct Dealer {
  // Shared memory of the dealing: used between pieces only.
  struct Shared {
    uint64_t wave_sums[TH / 64];
    uint32_t piece[16];
    uint32_t first[TH];                 // the first tile of each request of a chunk, and what is known of it
    int32_t n[TH], start[TH], length[TH];
  };

  const PagedAttnArgs &p;
  const Work &w;
  const FastDiv by_group;
  Shared *sh;
  const uint32_t worker;
  // The chunk of tiles, one to a thread.
  uint32_t r0 = 0, t0 = 0, chunk_tiles = 0, chunk_requests = 0;
  bool started = false;
  uint32_t request = 0, tile = 0, begin = 0, end = 0, blocks = 0;
  int32_t n = 0, start = 0, at = 0;
  // The line.
  uint64_t cur = 0, stop = 0, chunk_begin = 0, chunk_end = 0, off = 0, share = 1;
  uint32_t length_on_line = 0;
  bool few = false, done = false;

  __device__ Dealer(const PagedAttnArgs &p_, const Work &w_, FastDiv by_group_, Shared *sh_) : p(p_), w(w_), by_group(by_group_), sh(sh_), worker(xcd_run(blockIdx.x, gridDim.x)) {}

  __device__ uint64_t scan(uint64_t &x) {   // x: the sum over the threads before; returns the sum over all
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint64_t below = __shfl_up(sum, d);
      if (lane >= d) sum += below;
    }
    __syncthreads();
    if (lane == 63) sh->wave_sums[wave] = sum;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < TH / 64; i++) {
      if (i < wave) before += sh->wave_sums[i];
      all += sh->wave_sums[i];
    }
    x = before + sum - x;
    return all;
  }

  // New tokens, their first row, and the length of a request of this kernel's (n = 0: none of it).
  __device__ void read_request(uint32_t r, int32_t &n_, int32_t &start_, int32_t &length_) const {
    const int32_t most = int32_t(p.tokens);
    const int32_t s0 = min(max(p.starts[r], 0), most), s1 = min(max(p.starts[r + 1], 0), most);
    n_ = max(s1 - s0, 0), start_ = s0, length_ = p.lengths[r];
    const uint32_t rows = uint32_t(n_) * p.group;
    if (rows < w.min_rows || rows > w.max_rows) n_ = 0;
  }

  // Keys and blocks of a tile: `at` and the rest from n, length and the tile's number.
  __device__ void measure(int32_t length) {
    const uint32_t rows = uint32_t(n) * p.group, row0 = tile * BQ;
    const int32_t capacity = int32_t(p.width * p.page_size);
    const int32_t known = min(max(length, 0), capacity);
    at = int32_t(max(int64_t(length) - n, -(int64_t(1) << 30)));
    const int64_t last = int64_t(at) + by_group.div(min(row0 + BQ, rows) - 1), first = int64_t(at) + by_group.div(row0);
    end = uint32_t(min(max(last + 1, int64_t(0)), int64_t(known)));
    begin = p.window ? uint32_t(min(max(first - int64_t(p.window) + 1, int64_t(0)), int64_t(end))) : 0;
    blocks = end > begin ? (end - 1) / BK - begin / BK + 1 : 0;
  }

  // The next tiles, one to a thread (n = 0 on threads without one).
  __device__ bool next_chunk() {
    const uint32_t tid = threadIdx.x;
    if (w.single) {
      if (started) r0 += TH;
      started = true;
      if (r0 >= p.requests) return false;
      request = r0 + tid, tile = 0, n = 0, blocks = 0;
      int32_t length = 0;
      if (request < p.requests) read_request(request, n, start, length);
      if (n) measure(length);
      return true;
    }
    for (;;) {
      if (started && t0 + TH < chunk_tiles) {
        t0 += TH;
      } else {
        if (started) r0 += TH;
        started = true;
        if (r0 >= p.requests) return false;
        int32_t n_ = 0, start_ = 0, length_ = 0;
        if (r0 + tid < p.requests) read_request(r0 + tid, n_, start_, length_);
        uint64_t first = (uint32_t(n_) * p.group + BQ - 1) / BQ;
        chunk_tiles = uint32_t(scan(first));
        sh->first[tid] = uint32_t(first), sh->n[tid] = n_, sh->start[tid] = start_, sh->length[tid] = length_;
        __syncthreads();
        t0 = 0;
        if (chunk_tiles == 0) continue;
      }
      const uint32_t i = t0 + tid;
      n = 0, blocks = 0;
      if (i < chunk_tiles) {
        uint32_t lo = 0, hi = TH;   // first[lo] <= i < first[hi]: the last request that begins at i or before (those without tiles lie before it)
        while (hi - lo > 1) {
          const uint32_t mid = (lo + hi) / 2;
          if (sh->first[mid] <= i) lo = mid;
          else hi = mid;
        }
        request = r0 + lo, tile = i - sh->first[lo], n = sh->n[lo], start = sh->start[lo];
        measure(sh->length[lo]);
      }
      return true;
    }
  }

  __device__ void begin_line() {
    // All tiles and blocks there are.
    uint64_t tiles = 0, sum = 0;
    const bool one = w.single && p.requests <= TH;
    while (next_chunk()) {
      tiles += n != 0, sum += blocks;
      if (one) break;
    }
    const uint64_t all_tiles = scan(tiles) * p.kv_heads, all_blocks = scan(sum) * p.kv_heads;
    few = all_tiles * 4 < uint64_t(w.workers) * 3;
    const uint64_t round = w.round_blocks;
    if (few) {
      const uint64_t spare = w.workers - all_tiles;
      share = (all_blocks + spare - 1) / spare;
      share = max((share + round - 1) / round * round, round);
    } else {
      share = (all_blocks + all_tiles * (1 + OVERHEAD_KEYS / BK) + w.workers - 1) / w.workers;
    }
    cur = share * worker, stop = cur + share;
    if (!one) r0 = t0 = chunk_tiles = 0, started = false;
    else lay();
  }

  // The chunk's tiles on the line.
  __device__ void lay() {
    length_on_line = 0;
    if (n) length_on_line = few ? uint32_t((uint64_t(max(blocks, 1u)) + share - 1) / share * share) : blocks + 1 + OVERHEAD_KEYS / BK;
    off = uint64_t(length_on_line) * p.kv_heads;
    const uint64_t all = scan(off);
    off += chunk_end;
    chunk_begin = chunk_end, chunk_end += all;
  }

  // The workgroup's next piece; false: it has no more.
  __device__ bool next(Piece &out) {
    if (w.direct) {
      if (done) return false;
      done = true;
      request = worker / p.kv_heads, tile = 0;
      int32_t length;
      read_request(request, n, start, length);
      n = uniform(n);
      if (!n) return false;
      measure(uniform(length));
      out.request = request, out.head = worker - request * p.kv_heads, out.row0 = 0, out.rows = uint32_t(n) * p.group;
      out.start = uniform(start), out.at = uniform(at), out.begin = uniform(begin), out.end = uniform(end);
      out.first_block = out.begin / BK, out.blocks = out.b1 = uniform(blocks), out.b0 = out.v0 = out.v1 = 0;
      return true;
    }
    if (!done) {
      done = true;
      begin_line();
    }
    while (cur < stop) {
      while (cur >= chunk_end) {
        if ((w.single && p.requests <= TH) || !next_chunk()) return false;
        lay();
      }
      __syncthreads();   // (what was shared of the piece before has been read)
      if (length_on_line && cur >= off && cur < off + uint64_t(length_on_line) * p.kv_heads) {
        const uint32_t head = quotient(cur - off, length_on_line);
        const uint64_t from = off + uint64_t(head) * length_on_line;
        uint32_t *s = sh->piece;
        s[0] = request, s[1] = head, s[2] = tile * BQ, s[3] = min(uint32_t(BQ), uint32_t(n) * p.group - tile * BQ);
        s[4] = uint32_t(start), s[5] = uint32_t(at), s[6] = begin, s[7] = end, s[8] = blocks;
        s[9] = uint32_t(cur - from), s[10] = uint32_t(min(stop - from, uint64_t(length_on_line)));
        s[11] = quotient(from, share), s[12] = blocks ? quotient(from + blocks - 1, share) : s[11];
        s[13] = length_on_line;
      }
      __syncthreads();
      const uint32_t *s = sh->piece;
      out.request = uniform(s[0]), out.head = uniform(s[1]), out.row0 = uniform(s[2]), out.rows = uniform(s[3]);
      out.start = int32_t(uniform(s[4])), out.at = int32_t(uniform(s[5])), out.begin = uniform(s[6]), out.end = uniform(s[7]);
      out.blocks = uniform(s[8]), out.first_block = out.begin / BK;
      const uint32_t u0 = uniform(s[9]), u1 = uniform(s[10]);
      out.v0 = uniform(s[11]), out.v1 = uniform(s[12]);
      cur += uniform(s[13]) - u0;   // (the tile's end; past `stop` where the tile goes on)
      out.b0 = min(u0, out.blocks), out.b1 = min(u1, out.blocks);
      if (out.b0 < out.b1 || (out.blocks == 0 && u0 == 0)) return true;
    }
    return false;
  }

  __device__ static bool whole(const Piece &t) { return t.b0 == 0 && t.b1 == t.blocks; }
  // Where a piece of a tile leaves its partial result: rows of `row_floats`.
  __device__ float *place(const Piece &t, uint32_t row_floats) const { return w.partials + (uint64_t(worker) * 2 + (t.b0 == 0)) * BQ * row_floats; }
  // What the merging launch has to know of a tile that this workgroup begins and others end; called by one thread.
  __device__ void describe(const Piece &t) {
    uint32_t *d = w.tiles + worker * 8;
    d[0] = t.v1 - worker, d[1] = uint32_t(t.start), d[2] = t.row0, d[3] = t.rows, d[4] = t.head;
  }
  // After the last piece, by the thread that described: a workgroup that began no such tile says so.
  __device__ void finish(bool described_) const {
    if (!w.direct && !described_) w.tiles[worker * 8] = 0;
  }
};

// attention_paged_keys.hip, for qb = 1 or 2 (16 or 32 rows of a tile): workgroups that fill the chip, floats of a row of a partial result, the launch.
uint32_t keys_workers(const PagedAttnArgs &a, int qb);
uint32_t keys_row_floats(const PagedAttnArgs &a);
hipError_t launch_keys(const PagedAttnArgs &a, const Work &work, int qb, hipStream_t stream);

}  // namespace paged
}  // namespace mrl
