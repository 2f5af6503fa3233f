// Attention of requests' new tokens over their pages of keys and values.
#include <algorithm>
#include <cmath>

#include "attention_paged.h"

namespace mrl {
namespace {

// Any head dim, page size, stride and alignment: a workgroup per token and query head, 256 keys at a time.  A thread forms
// one key's score, the statistics of the softmax run along (m, l: the largest score so far and the sum of exponentials against it), then a
// thread takes dims d, d + 256, .. of the sum over the keys' values.  A hidden key's slot is not read.
typedef unsigned short u16;
__device__ inline float to_f32(u16 x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float to_f32(float x) { return x; }
constexpr int THREADS = 256, MOST_DIMS = 1024;

template <class T>
__global__ __launch_bounds__(THREADS) void k_paged_attn_generic(PagedAttnArgs p, FastDiv by_page) {
  __shared__ float q_row[MOST_DIMS], weight[THREADS];
  __shared__ int64_t value_at[THREADS];
  __shared__ float shared_max[THREADS / 64], shared_sum[THREADS / 64];
  const uint32_t token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  // The token's request: the one whose [start, end) holds it, found by halving (starts do not fall; where they do, a request that ends
  // before it starts has no tokens and whichever request is found is checked to hold the token).
  uint32_t lo = 0, hi = p.requests;   // starts[lo] <= token < starts[hi], if any
  if (int64_t(p.starts[0]) > int64_t(token)) return;
  if (int64_t(p.starts[p.requests]) <= int64_t(token)) return;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (int64_t(p.starts[mid]) <= int64_t(token)) lo = mid;
    else hi = mid;
  }
  const int64_t start = max(p.starts[lo], 0), end = min(int64_t(p.starts[lo + 1]), int64_t(p.tokens));
  const int64_t length = p.lengths[lo], at = length - (end - start) + (int64_t(token) - start);
  const int64_t last = min(min(at + 1, length), int64_t(p.width) * p.page_size);   // one behind the last key
  const int64_t first = p.window ? max(at - int64_t(p.window) + 1, int64_t(0)) : 0;
  const T *q = (const T *)p.q + int64_t(token) * p.q_t + int64_t(head) * p.q_h;
  for (uint32_t d = tid; d < p.head_dim; d += THREADS) q_row[d] = to_f32(q[d]) * p.scale;
  const uint32_t kv = head / p.group;
  const T *keys = (const T *)p.keys + int64_t(kv) * p.key_h, *values = (const T *)p.values + int64_t(kv) * p.val_h;
  constexpr int EACH = MOST_DIMS / THREADS;
  float sum[EACH] = {0, 0, 0, 0}, m = -__builtin_inff(), l = 0;
  for (int64_t k0 = first; k0 < last; k0 += THREADS) {
    const int64_t key = k0 + tid;
    float s = -__builtin_inff();
    int64_t from_value = -1;
    __syncthreads();
    if (key < last) {
      const uint32_t column = by_page.div(uint32_t(key)), place = uint32_t(key) - column * p.page_size;
      const int32_t page = p.table[uint64_t(lo) * p.width + column];
      if (page >= 0 && uint32_t(page) < p.pages) {
        const T *k = keys + int64_t(page) * p.key_p + int64_t(place) * p.key_s;
        s = 0;
        for (uint32_t d = 0; d < p.head_dim; d++) s = __builtin_fmaf(q_row[d], to_f32(k[d]), s);
        from_value = int64_t(page) * p.val_p + int64_t(place) * p.val_s;
      }
    }
    value_at[tid] = from_value;
    float most = s;
    for (int d = 32; d; d /= 2) most = fmaxf(most, __shfl_xor(most, d));
    if ((tid & 63) == 0) shared_max[tid >> 6] = most;
    __syncthreads();
    most = m;
    for (int w = 0; w < THREADS / 64; w++) most = fmaxf(most, shared_max[w]);
    const float e = from_value < 0 ? 0.0f : most == -__builtin_inff() ? (s != s ? s : 0.0f) : expf(s - most);
    weight[tid] = e;
    float part = e;
    for (int d = 32; d; d /= 2) part += __shfl_xor(part, d);
    if ((tid & 63) == 0) shared_sum[tid >> 6] = part;
    __syncthreads();
    const float old = m == -__builtin_inff() ? 0.0f : expf(m - most);
    l *= old;
    for (int w = 0; w < THREADS / 64; w++) l += shared_sum[w];
    m = most;
    const int count = int(min(int64_t(THREADS), last - k0));
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const uint32_t d = tid + i * THREADS;
      if (d >= p.head_dim) break;
      float x = sum[i] * old;
      for (int j = 0; j < count; j++)
        if (value_at[j] >= 0) x = __builtin_fmaf(weight[j], to_f32(values[value_at[j] + d]), x);
      sum[i] = x;
    }
  }
  T *out = (T *)p.out + int64_t(token) * p.o_t + int64_t(head) * p.o_h;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t d = tid + i * THREADS;
    if (d >= p.head_dim) break;
    const float x = l == 0.0f ? 0.0f : sum[i] / l;
    if constexpr (sizeof(T) == 2) out[d] = __builtin_bit_cast(u16, (__bf16)x);
    else out[d] = x;
  }
}

template <class T>
hipError_t launch_generic(const PagedAttnArgs &a, hipStream_t stream) {
  const double capacity = double(a.width) * a.page_size;
  plan::work(plan::UNIT_VALU, 4.0 * a.tokens * a.q_heads * a.head_dim * capacity, 2.0 * sizeof(T) * a.tokens * double(a.q_heads) * a.head_dim);
  MRL_LAUNCH(k_paged_attn_generic<T>, dim3(a.tokens, a.q_heads), dim3(THREADS), 0, stream, a, FastDiv(a.page_size));
  return plan::last_error();
}

// ---- Dealing: the tiles on a line, its shares (attention_paged.h). ----
struct DealArgs {
  PagedAttnArgs p;
  FastDiv by_group;
  paged::Work work[2];   // a workgroup to each
};
constexpr int DEAL = int(paged::MOST_WORKERS), DEAL_WAVES = DEAL / 64;

// x: the sum over the threads before this one; returns the sum over all.
__device__ inline uint64_t scan(uint64_t &x, uint64_t *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t sum = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t below = __shfl_up(sum, d);
    if (lane >= d) sum += below;
  }
  __syncthreads();   // (the sums of the scan before have been read)
  if (lane == 63) wave_sums[wave] = sum;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < DEAL_WAVES; w++) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  x = before + sum - x;
  return all;
}
// The last of 1024 ascending numbers that is at most x (the first one is).
template <class N>
__device__ inline uint32_t last_up_to(const N *numbers, N x) {
  uint32_t lo = 0;
#pragma unroll
  for (uint32_t step = DEAL / 2; step; step /= 2)
    if (numbers[lo + step] <= x) lo += step;
  return lo;
}

// Requests 1024 at a time, their tiles 1024 at a time, a thread each; once for how much there is (and once more where that was more than one such chunk), then to note them.
// Of a chunk, request r's tiles lie at heads * (lengths of the tiles before r's) + head * (lengths of r's) + (lengths of r's before it).
__global__ __launch_bounds__(DEAL) void k_paged_attn_deal(DealArgs a) {
  using namespace paged;
  __shared__ uint64_t wave_sums[DEAL_WAVES];
  __shared__ uint32_t first[DEAL], tiles_of[DEAL];          // of a request: its first tile in the chunk of requests, how many
  __shared__ int32_t n_of[DEAL], start_of[DEAL], length_of[DEAL];
  __shared__ uint64_t line[DEAL + 1];                       // lengths of the chunk's tiles before a tile
  __shared__ uint32_t request_of[DEAL];
  const Work &w = a.work[blockIdx.x];
  const uint32_t tid = threadIdx.x, heads = a.p.kv_heads;
  uint32_t r0 = 0, t0 = 0, tiles = 0, left = 0, request = 0, noted = 0;
  Tile t = {};
  // The next chunk: a tile to a thread (t.rows = 0: none).
  auto next_chunk = [&](bool start) {
    if (start) r0 = t0 = tiles = 0, left = w.most_tiles;   // (starts that do not fall never come to more; others are cut off here)
    else t0 += DEAL;
    while (t0 >= tiles) {
      if (!start) r0 += DEAL;
      start = false;
      if (r0 >= a.p.requests || !left) return false;
      Request q = {0, 0, 0};
      if (r0 + tid < a.p.requests) q = read_request(a.p, w, r0 + tid);
      const uint32_t mine = (uint32_t(q.n) * a.p.group + (1u << w.bq_log2) - 1) >> w.bq_log2;
      uint64_t at = mine;
      tiles = uint32_t(min(scan(at, wave_sums), uint64_t(left))), t0 = 0, left -= tiles;
      first[tid] = uint32_t(at), tiles_of[tid] = mine, n_of[tid] = q.n, start_of[tid] = q.start, length_of[tid] = q.length;
      __syncthreads();
    }
    t.rows = 0, t.blocks = 0;
    if (t0 + tid < tiles) {
      request = last_up_to(first, t0 + tid);
      const Request q = {n_of[request], start_of[request], length_of[request]};
      const uint32_t row0 = (t0 + tid - first[request]) << w.bq_log2;
      t = measure(a.p, a.by_group, q, row0, min(uint32_t(q.n) * a.p.group - row0, 1u << w.bq_log2), w.block_log2);
    }
    return true;
  };
  uint64_t sum_tiles = 0, sum_blocks = 0;
  uint32_t chunks = 0;
  for (bool more = next_chunk(true); more; more = next_chunk(false)) {
    sum_tiles += t.rows != 0, sum_blocks += t.blocks, chunks++;
    if (tiles <= DEAL && a.p.requests <= DEAL) break;
  }
  const uint64_t all_tiles = scan(sum_tiles, wave_sums) * heads, all_blocks = scan(sum_blocks, wave_sums) * heads, workers = w.workers;
  uint64_t share = quotient(all_blocks + all_tiles * (1 + w.overhead) + workers - 1, workers);
  bool few = false;
  if (all_tiles < workers) {   // a piece to each, where that is no longer than equal shares and the second piece that they may come to
    const uint32_t spare = uint32_t(workers - all_tiles), single = max((quotient(all_blocks + spare - 1, spare) + w.least - 1) / w.least, 1u) * w.least;
    few = single <= share + w.second;
    if (few) share = single;
  }
  share = max(share, uint64_t(1));
  uint64_t base = 0;   // of the chunk, on the line
  const uint64_t my_start = share * tid;
  bool open = tid < w.workers;   // this workgroup's start is not found yet
  const bool again = !(chunks == 1 && tiles <= DEAL && a.p.requests <= DEAL);
  for (bool more = again ? next_chunk(true) : chunks == 1; more; more = again && next_chunk(false)) {
    if (t.rows) t.length = few ? (quotient(max(t.blocks, 1u) + share - 1, share)) * uint32_t(share) : t.blocks + 1 + w.overhead;
    uint64_t at = t.rows ? t.length : 0;
    const uint64_t all = scan(at, wave_sums);   // (its barriers: what the chunk before noted has been read)
    line[tid] = at, request_of[tid] = request;
    if (tid == 0) line[DEAL] = all;
    __syncthreads();
    const uint32_t count = min(tiles - t0, uint32_t(DEAL));
    if (t.rows) {
      t.request = r0 + request;
      t.first = noted + max(first[request], t0) - t0, t.behind = noted + min(first[request] + tiles_of[request] - t0, count);
      w.tiles[noted + tid] = t;
    }
    if (open && my_start < base + all * heads) {
      const uint64_t here = my_start - base;
      const uint32_t of = request_of[last_up_to(line, uint64_t(quotient(here, heads)))];
      const uint32_t lo = max(first[of], t0) - t0, hi = min(first[of] + tiles_of[of] - t0, count);
      const uint64_t rest = here - line[lo] * heads, each = line[hi] - line[lo];
      const uint32_t head = quotient(rest, each);
      const uint64_t in_head = line[lo] + (rest - head * each);
      const uint32_t x = last_up_to(line, in_head);
      w.starts[tid] = {noted + x, head, uint32_t(in_head - line[x]), 0};
      open = false;
    }
    base += all * heads, noted += count;
  }
  if (open) w.starts[tid] = {0xffffffffu, 0, 0, 0};
  if (tid == 0) w.line->share = share, w.line->tiles = noted;
}

// ---- Tiles in pieces: out = sum_v O_v 2^(m_v - M) / sum_v l_v 2^(m_v - M), M the largest m_v, over the pieces in their order (the parts formula of
// morello/src/spec.rs:107-132 in base 2). ----
struct MergeArgs {
  struct {
    const uint32_t *merges;
    const float *partials;
    uint32_t workers, bq;
  } of[2];
  uint32_t row_floats;
  FastDiv by_group, by_quads;
};
// U: pieces asked for at a time.
template <class T, uint32_t U>
__device__ inline void merge_rows(const PagedAttnArgs &p, const MergeArgs &a, const float *partials, uint32_t more, uint32_t piece_floats, int32_t start, uint32_t row0, uint32_t rows,
                                  uint32_t kv) {
  const uint32_t quads = (p.head_dim + 3) / 4, stat = a.row_floats - 4;
  for (uint32_t x = blockIdx.y * THREADS + threadIdx.x; x < rows * quads; x += gridDim.y * THREADS) {
    const uint32_t i = a.by_quads.div(x), dim = (x - i * quads) * 4;
    // piece 0 lies in the first workgroup's place 1, the others in place 0 of those behind it
    auto piece = [&](uint32_t v) { return partials + (2 * uint64_t(v) + (v == 0)) * piece_floats + i * a.row_floats; };
    float m = -3.0e38f, l = 0;
    attn::v4f sum = {0, 0, 0, 0};
    for (uint32_t v0 = 0; v0 <= more; v0 += U) {
      float ms[U], ls[U];
      attn::v4f os[U];
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
        const float *from = piece(min(v0 + u, more));
        ms[u] = from[stat], ls[u] = from[stat + 1], os[u] = *(const attn::v4f *)(from + dim);
      }
      float most = m;
#pragma unroll
      for (uint32_t u = 0; u < U; u++) most = fmaxf(most, ms[u]);
      const float old = __builtin_amdgcn_exp2f(m - most);
      sum *= old, l *= old, m = most;
#pragma unroll
      for (uint32_t u = 0; u < U; u++)
        if (v0 + u <= more) {
          const float f = __builtin_amdgcn_exp2f(ms[u] - m);
          sum += os[u] * f, l += ls[u] * f;
        }
    }
    sum *= l == 0.0f ? 0.0f : 1.0f / l;
    const uint32_t row = row0 + i, token = a.by_group.div(row), head = kv * p.group + (row - token * p.group);
    T *out = (T *)p.out + int64_t(start + int32_t(token)) * p.o_t + int64_t(head) * p.o_h + dim;
    if constexpr (sizeof(T) == 2) {
      typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
      *(v4bf *)out = v4bf{(__bf16)sum[0], (__bf16)sum[1], (__bf16)sum[2], (__bf16)sum[3]};
    } else {
      *(attn::v4f *)out = sum;
    }
  }
}
// blockIdx.x: the workgroup that begins the tile, those of the first kernel before those of the second; blockIdx.y: a share of its rows.
template <class T>
__global__ __launch_bounds__(THREADS) void k_paged_attn_merge(PagedAttnArgs p, MergeArgs a) {
  const uint32_t second = blockIdx.x >= a.of[0].workers, worker = blockIdx.x - (second ? a.of[0].workers : 0);
  const uint32_t *d = a.of[second].merges + worker * 8;
  const uint32_t piece_floats = a.of[second].bq * a.row_floats, more = d[0], row0 = d[2], rows = d[3], kv = d[4];
  const int32_t start = int32_t(d[1]);
  if (!more) return;
  const float *const partials = a.of[second].partials + 2 * uint64_t(worker) * piece_floats;
  if (more < 2) merge_rows<T, 2>(p, a, partials, more, piece_floats, start, row0, rows, kv);
  else if (more < 4) merge_rows<T, 4>(p, a, partials, more, piece_floats, start, row0, rows, kv);
  else merge_rows<T, 16>(p, a, partials, more, piece_floats, start, row0, rows, kv);
}

constexpr uint32_t DIRECT_KEYS = 1024;

// How a call runs, by sizes, types and strides: on tiles of 16 * qb rows, of 128, or small requests on the former and the others on the latter.
struct Choice {
  bool tiled = false;                 // else the generic kernel
  int qb = 0;                         // 0: no tiles of 16 or 32 rows
  paged::Work keys = {}, chunk = {};  // workers = 0: none of them
  size_t keys_at[5] = {}, chunk_at[5] = {}, bytes = 0;   // what the Work points at, in the workspace; all of it
};

void lay_out(const PagedAttnArgs &a, paged::Work &w, size_t *at, size_t *bytes) {
  const uint64_t bq = uint64_t(1) << w.bq_log2;
  w.most_tiles = uint32_t(((uint64_t(a.tokens) * a.group + bq - 1) >> w.bq_log2) + a.requests);
  auto take = [&](size_t n) {
    const size_t from = *bytes;
    *bytes += (n + 255) & ~size_t(255);
    return from;
  };
  at[0] = take(sizeof(paged::Line)), at[1] = take(w.workers * sizeof(paged::Start)), at[2] = take(w.most_tiles * sizeof(paged::Tile)), at[3] = take(w.workers * 32);
  at[4] = take(2 * w.workers * bq * paged::row_floats(a) * sizeof(float));
}
void place(paged::Work &w, const size_t *at, uint8_t *workspace) {
  w.line = reinterpret_cast<paged::Line *>(workspace + at[0]), w.starts = reinterpret_cast<paged::Start *>(workspace + at[1]);
  w.tiles = reinterpret_cast<paged::Tile *>(workspace + at[2]), w.merges = reinterpret_cast<uint32_t *>(workspace + at[3]);
  w.partials = reinterpret_cast<float *>(workspace + at[4]);
}

Choice choose(const PagedAttnArgs &a) {
  Choice c;
  const int size = a.dtype == MRL_BF16 ? 2 : 4;
  auto chunks = [&](int64_t n) { return n * size % 16 == 0; };
  const double scale = std::fabs(a.scale);
  // Pages of whole sixteens of slots, heads and strides of whole 16-byte chunks, 16 slots of a page within what an offset of 31 bits reaches; a line of blocks that
  // 256 shares of 32 bits cover.
  c.tiled = a.page_size % 16 == 0 && a.head_dim <= 128 && chunks(a.head_dim) && chunks(a.q_t) && chunks(a.q_h) && chunks(a.o_t) && chunks(a.o_h) && chunks(a.key_p) &&
            chunks(a.key_s) && chunks(a.key_h) && chunks(a.val_p) && chunks(a.val_s) && chunks(a.val_h) && a.key_s < (1 << 24) && a.val_s < (1 << 24) &&
            uint64_t(a.tokens) * a.group < (1u << 31) &&
            (double(a.tokens) * a.group / 16 + a.requests) * a.kv_heads * (double(a.width) * a.page_size / 32 + 16) < double(1ull << 39) && scale > 1e-30 && scale < 1e30;
  if (!c.tiled) return c;
  const uint64_t rows = uint64_t(a.max_new) * a.group;
  const bool chunk = a.dtype == MRL_BF16 && rows > 32;
  if (!chunk) c.qb = rows <= 16 ? 1 : 2;
  else if (a.requests > 1) c.qb = 1;
  if (c.qb) {
    paged::Work &w = c.keys;
    paged::keys_work(a, c.qb, &w);
    w.min_rows = 1, w.max_rows = chunk ? 16 : 0x7fffffff;
    // Tables of some hundred keys at most: a workgroup to each request and head does them in some rounds, with nothing to find out before and no launch behind.
    // (max_new is the program's word: a request of more tokens would have more tiles than one)
    w.direct = !chunk && uint64_t(a.tokens) * a.group <= 16u * c.qb && uint64_t(a.width) * a.page_size <= DIRECT_KEYS;
    if (!w.direct) lay_out(a, w, c.keys_at, &c.bytes);
  }
  if (chunk) {
    paged::chunk_work(a, &c.chunk);
    c.chunk.min_rows = c.qb ? 17 : 1, c.chunk.max_rows = 0x7fffffff;
    lay_out(a, c.chunk, c.chunk_at, &c.bytes);
  }
  return c;
}

hipError_t launch_deal(const PagedAttnArgs &a, const Choice &c, hipStream_t stream) {
  DealArgs d;
  d.p = a, d.by_group = FastDiv(a.group);
  int n = 0;
  if (c.chunk.workers) d.work[n++] = c.chunk;
  if (c.keys.workers) d.work[n++] = c.keys;
  plan::work(plan::UNIT_STREAM, 0, 12.0 * a.requests + 64.0 * (c.chunk.most_tiles + c.keys.most_tiles));
  MRL_LAUNCH(k_paged_attn_deal, dim3(n), dim3(DEAL), 0, stream, d);
  return plan::last_error();
}

template <class T>
hipError_t launch_merge(const PagedAttnArgs &a, const Choice &c, hipStream_t stream) {
  MergeArgs m;
  m.of[0] = {c.chunk.merges, c.chunk.partials, c.chunk.workers, 1u << c.chunk.bq_log2};
  m.of[1] = {c.keys.merges, c.keys.partials, c.keys.workers, 1u << c.keys.bq_log2};
  m.row_floats = paged::row_floats(a), m.by_group = FastDiv(a.group), m.by_quads = FastDiv((a.head_dim + 3) / 4);
  plan::work(plan::UNIT_STREAM, 0, double(c.bytes) / 2);
  MRL_LAUNCH(k_paged_attn_merge<T>, dim3(c.chunk.workers + c.keys.workers, c.chunk.workers ? 8 : 2), dim3(THREADS), 0, stream, a, m);
  return plan::last_error();
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnArgs &a) { return choose(a).bytes; }

hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream) {
  const bool bf16 = a.dtype == MRL_BF16;
  auto aligned = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  Choice c = choose(a);
  if (!c.tiled || !aligned(a.q) || !aligned(a.keys) || !aligned(a.values) || !aligned(a.out))
    return bf16 ? launch_generic<u16>(a, stream) : launch_generic<float>(a, stream);
  if (c.keys.direct) return paged::launch_keys(a, c.keys, c.qb, stream);
  place(c.keys, c.keys_at, a.workspace), place(c.chunk, c.chunk_at, a.workspace);
  hipError_t e = launch_deal(a, c, stream);
  if (e == hipSuccess && c.chunk.workers) e = paged::launch_chunk(a, c.chunk, stream);
  if (e == hipSuccess && c.keys.workers) e = paged::launch_keys(a, c.keys, c.qb, stream);
  if (e != hipSuccess) return e;
  return bf16 ? launch_merge<u16>(a, c, stream) : launch_merge<float>(a, c, stream);
}

}  // namespace mrl
