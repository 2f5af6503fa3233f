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
//     the pieces are at most as many as workgroups: each has one piece, a tile's pieces meet in the merging launch;
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

struct Work {
  uint32_t min_rows, max_rows;   // requests of so many query rows; others' are left to another kernel
  bool single;                   // no such request has more than a tile
  bool direct;                   // a workgroup to each (request, head): nothing is shared out
  uint32_t workers;
  uint32_t round_blocks;         // the least blocks of a piece where a tile is cut because workgroups are to spare
  float *partials;               // [worker][2][rows of a tile][row_floats]
  uint32_t *tiles;               // [worker][8]: see describe()
  uint32_t *lists;               // [worker][LIST][16]: a workgroup's own notes
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

// One tile's piece for this workgroup.
struct Piece {
  uint32_t request, head, row0, rows;   // rows row0 .. row0 + rows - 1 of the request, at key/value head `head`
  int32_t start, at;                    // the tensors' row of the request's token 0, and its place among the keys (may be below zero)
  uint32_t begin, end;                  // keys that some row sees lie in [begin, end)
  uint32_t blocks;                      // their blocks, and of them
  uint32_t b0, b1;                      // this piece's, counted from the one that holds `begin`
  uint32_t more;                        // workgroups behind this one that have pieces of the tile, if this one begins it
  __device__ bool whole() const { return b0 == 0 && b1 == blocks; }
};

__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline uint64_t uniform(uint64_t x) { return uint64_t(uniform(uint32_t(x >> 32))) << 32 | uniform(uint32_t(x)); }

// floor(x / y) for x < 2^52 and a quotient below 2^32 (a quotient that is no whole number is at least 1 / y off one: more than a rounding in 64 bits).
__device__ inline uint32_t quotient(uint64_t x, uint64_t y) { return uint32_t(double(x) / double(y)); }

constexpr int LIST = 16;   // pieces that a workgroup notes at a time

// What a tile costs besides its blocks (the trips to memory before its first one, its results), in blocks: OVERHEAD where the chip has all it can do, START
// where a workgroup waits for nothing but its own loads.
template <int TH, int BQ, int BK, int OVERHEAD, int START>
struct Dealer {
  // Shared memory of the dealing: nothing in it is kept over a piece.
  struct Shared {
    uint64_t wave_sums[TH / 64];
    uint64_t next;
    uint32_t first[TH];                 // the first tile of each request of a chunk, and what is known of it
    int32_t n[TH], start[TH], length[TH];
  };

  const Kernargs &k;
  Shared *sh;
  // The chunk of tiles, one to a thread.
  uint32_t r0 = 0, t0 = 0, chunk_tiles = 0;
  bool started = false;
  uint32_t request = 0, tile = 0, begin = 0, end = 0, blocks = 0;
  int32_t n = 0, start = 0, at = 0;

  __device__ Dealer(const Kernargs &k_, Shared *sh_) : k(k_), sh(sh_) {}

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
    return uniform(all);
  }

  // New tokens, their first row, and the length of a request of this kernel's (n = 0: none of it).
  __device__ void read_request(uint32_t r, int32_t &n_, int32_t &start_, int32_t &length_) const {
    const int32_t most = int32_t(k.p.tokens);
    const int32_t s0 = min(max(k.p.starts[r], 0), most), s1 = min(max(k.p.starts[r + 1], 0), most);
    n_ = max(s1 - s0, 0), start_ = s0, length_ = k.p.lengths[r];
    const uint32_t rows = uint32_t(n_) * k.p.group;
    if (rows < k.w.min_rows || rows > k.w.max_rows) n_ = 0;
  }

  // Keys and blocks of a tile: from n, length and the tile's number.
  __device__ void measure(int32_t length) {
    const uint32_t rows = uint32_t(n) * k.p.group, row0 = tile * BQ;
    const int32_t known = min(max(length, 0), int32_t(k.p.width * k.p.page_size));
    at = int32_t(max(int64_t(length) - n, -(int64_t(1) << 30)));
    const int64_t last = int64_t(at) + k.by_group.div(min(row0 + BQ, rows) - 1), first = int64_t(at) + k.by_group.div(row0);
    end = uint32_t(min(max(last + 1, int64_t(0)), int64_t(known)));
    begin = k.p.window ? uint32_t(min(max(first - int64_t(k.p.window) + 1, int64_t(0)), int64_t(end))) : 0;
    blocks = end > begin ? (end - 1) / BK - begin / BK + 1 : 0;
  }

  // The next tiles, one to a thread (n = 0 on threads without one).
  __device__ bool next_chunk() {
    const uint32_t tid = threadIdx.x;
    if (k.w.single) {
      if (started) r0 += TH;
      started = true;
      if (r0 >= k.p.requests) return false;
      request = r0 + tid, tile = 0, n = 0, blocks = 0;
      int32_t length = 0;
      if (request < k.p.requests) read_request(request, n, start, length);
      if (n) measure(length);
      return true;
    }
    for (;;) {
      if (started && t0 + TH < chunk_tiles) t0 += TH;
      else if (started) r0 += TH, t0 = 0;
      started = true;
      if (r0 >= k.p.requests) return false;
      int32_t n_ = 0, start_ = 0, length_ = 0;
      if (r0 + tid < k.p.requests) read_request(r0 + tid, n_, start_, length_);
      uint64_t first = (uint32_t(n_) * k.p.group + BQ - 1) / BQ;
      chunk_tiles = uint32_t(scan(first));
      sh->first[tid] = uint32_t(first), sh->n[tid] = n_, sh->start[tid] = start_, sh->length[tid] = length_;
      __syncthreads();
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
      __syncthreads();
      if (chunk_tiles) return true;
    }
  }

  __device__ void note(uint32_t *to, uint32_t head, uint32_t b0, uint32_t b1, uint32_t more) const {
    to[0] = request, to[1] = head, to[2] = tile * BQ, to[3] = min(uint32_t(BQ), uint32_t(n) * k.p.group - tile * BQ);
    to[4] = uint32_t(start), to[5] = uint32_t(at), to[6] = begin, to[7] = end, to[8] = blocks, to[9] = b0, to[10] = b1, to[11] = more;
  }

  // Notes the workgroup's next pieces in `list` ([LIST][16]) and returns how many; `cur`: 0 at first, and then what the call before left (all ones: there are
  // no more).  Everybody calls it, and passes a barrier before reading.
  __device__ uint32_t deal(uint32_t worker, uint32_t *list, uint64_t &cur) {
    const uint64_t DONE = ~uint64_t(0);
    if (k.w.direct) {
      cur = DONE;
      request = worker / k.p.kv_heads, tile = 0;
      int32_t length;
      read_request(request, n, start, length);
      n = uniform(n);
      if (!n) return 0;
      measure(length);
      if (threadIdx.x == 0) note(list, worker - request * k.p.kv_heads, 0, blocks, 0);
      return 1;
    }
    // All tiles and blocks there are.
    const bool one = k.w.single && k.p.requests <= TH;
    uint64_t tiles = 0, sum = 0;
    while (next_chunk()) {
      tiles += n != 0, sum += blocks;
      if (one) break;
    }
    const uint64_t heads = k.p.kv_heads, workers = k.w.workers, all_tiles = scan(tiles) * heads, all_blocks = scan(sum) * heads;
    uint64_t share = max(uint64_t(quotient(all_blocks + all_tiles * (1 + OVERHEAD) + workers - 1, workers)), uint64_t(1));
    bool few = false;
    if (all_tiles < workers) {   // a piece to each, where that is no longer than equal shares and the second start that they cost
      const uint64_t spare = workers - all_tiles, round = k.w.round_blocks;
      const uint64_t single = max((uint64_t(quotient(all_blocks + spare - 1, spare)) + round - 1) / round * round, round);
      few = single <= share + START;
      if (few) share = single;
    }
    const uint64_t stop = share * (worker + 1);
    cur = max(cur, share * worker);
    if (!one) r0 = t0 = chunk_tiles = 0, started = false;
    uint32_t count = 0;
    uint64_t chunk_end = 0;
    while (one || next_chunk()) {
      // The chunk's tiles on the line.
      uint32_t length = 0;
      if (n) length = few ? uint32_t((uint64_t(max(blocks, 1u)) + share - 1) / share * share) : blocks + 1 + OVERHEAD;
      uint64_t off = uint64_t(length) * heads;
      const uint64_t all = scan(off);
      off += chunk_end, chunk_end += all;
      // Of this thread's tile, heads h0 .. h1 - 1 have pieces in [cur, stop).
      uint32_t h0 = 0, h1 = 0;
      if (length && off < stop && off + length * heads > cur) {
        h0 = cur > off ? quotient(cur - off, length) : 0;
        h1 = stop - off >= length * heads ? uint32_t(heads) : quotient(stop - off + length - 1, length);
        const uint64_t from = off + uint64_t(h0) * length;
        if (cur > from && cur - from >= blocks) h0++;   // (nothing but the overhead is left of it)
      }
      uint64_t place = h1 - min(h0, h1);
      const uint64_t pieces = scan(place);
      for (uint32_t h = h0; h < h1 && count + place < LIST; h++, place++) {
        const uint64_t from = off + uint64_t(h) * length;
        const uint32_t b0 = cur > from ? uint32_t(cur - from) : 0, b1 = uint32_t(min(stop - from, uint64_t(blocks)));
        note(list + (count + place) * 16, h, b0, b1, blocks ? quotient(from + blocks - 1, share) - worker : 0);
        if (count + place == LIST - 1) sh->next = from + length;
      }
      count += uint32_t(min(pieces, uint64_t(LIST - count)));
      if (one || count == LIST || chunk_end >= stop) break;
    }
    __syncthreads();
    cur = count == LIST ? uniform(sh->next) : DONE;
    if (cur >= stop) cur = DONE;
    return count;
  }

  // A noted piece, in scalar registers.
  __device__ static Piece read(const uint32_t *list, uint32_t i) {
    const uint32_t *s = list + i * 16;
    Piece t;
    t.request = uniform(s[0]), t.head = uniform(s[1]), t.row0 = uniform(s[2]), t.rows = uniform(s[3]), t.start = int32_t(uniform(s[4])), t.at = int32_t(uniform(s[5]));
    t.begin = uniform(s[6]), t.end = uniform(s[7]), t.blocks = uniform(s[8]), t.b0 = uniform(s[9]), t.b1 = uniform(s[10]), t.more = uniform(s[11]);
    return t;
  }
};

// Where a piece of a tile leaves its partial result: rows of `row_floats`.
__device__ inline float *partial_place(const Work &w, uint32_t worker, const Piece &t, uint32_t bq, uint32_t row_floats) {
  return w.partials + (uint64_t(worker) * 2 + (t.b0 == 0)) * bq * row_floats;
}
// What the merging launch has to know of a tile that this workgroup begins and others end; a workgroup that begins no such tile says so (tiles[worker][0] = 0).
__device__ inline void describe(const Work &w, uint32_t worker, const Piece &t) {
  uint32_t *d = w.tiles + worker * 8;
  d[0] = t.more, d[1] = uint32_t(t.start), d[2] = t.row0, d[3] = t.rows, d[4] = t.head;
}

// Floats of a row of a partial result: O of the head dim the kernels are built for, reference, denominator, and two that are not used.
inline uint32_t row_floats(const PagedAttnArgs &a) { return (a.head_dim <= 64 ? 64 : 128) + 4; }
// attention_paged_chunk.hip: tiles of 128 rows, bf16.
constexpr int CHUNK_ROWS = 128;
uint32_t chunk_workers(const PagedAttnArgs &a);
hipError_t launch_chunk(const PagedAttnArgs &a, const Work &work, hipStream_t stream);
// attention_paged_keys.hip, for qb = 1 or 2 (16 or 32 rows of a tile): workgroups that fill the chip, and the launch.
uint32_t keys_workers(const PagedAttnArgs &a, int qb);
hipError_t launch_keys(const PagedAttnArgs &a, const Work &work, int qb, hipStream_t stream);

}  // namespace paged
}  // namespace mrl
