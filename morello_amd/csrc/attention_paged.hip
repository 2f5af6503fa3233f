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

// ---- Tiles in pieces: out = sum_v O_v 2^(m_v - M) / sum_v l_v 2^(m_v - M), M the largest m_v, over the pieces in their order (the parts formula of
// morello/src/spec.rs:107-132 in base 2). ----
struct MergeArgs {
  const uint32_t *merges;
  const float *partials;
  uint32_t bq, row_floats;   // rows of a tile
  FastDiv by_group, by_quads;
};
// Pieces put together so far.
struct Sum {
  float m, l;
  attn::v4f o;
};
constexpr Sum NOTHING = {-3.0e38f, 0, {0, 0, 0, 0}};
// Pieces first .. last of four dims of a row, U asked for at a time; from(v): the row's of piece v.
template <uint32_t U, class F>
__device__ inline Sum sum_of(uint32_t first, uint32_t last, uint32_t stat, uint32_t dim, F from) {
  Sum s = NOTHING;
  for (uint32_t v0 = first; v0 <= last; v0 += U) {
    float ms[U], ls[U];
    attn::v4f os[U];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      const float *x = from(min(v0 + u, last));
      ms[u] = x[stat], ls[u] = x[stat + 1], os[u] = *(const attn::v4f *)(x + dim);
    }
    float most = s.m;
#pragma unroll
    for (uint32_t u = 0; u < U; u++) most = fmaxf(most, ms[u]);
    const float old = __builtin_amdgcn_exp2f(s.m - most);
    s.o *= old, s.l *= old, s.m = most;
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
      if (v0 + u <= last) {
        const float f = __builtin_amdgcn_exp2f(ms[u] - s.m);
        s.o += os[u] * f, s.l += ls[u] * f;
      }
  }
  return s;
}
constexpr uint32_t MANY = 4;   // pieces from which on the waves of a workgroup share them
// blockIdx.x: the workgroup that begins the tile; blockIdx.y: a share of its rows' dims, four to a thread.  What it takes is latency: a descriptor, then all pieces of a
// thread at once.
template <class T>
__global__ __launch_bounds__(THREADS) void k_paged_attn_merge(PagedAttnArgs p, MergeArgs a) {
  constexpr uint32_t WAVES = THREADS / 64;
  __shared__ Sum met[WAVES][64];
  const uint32_t *d = a.merges + blockIdx.x * 8;
  // (as many as there are workgroups behind: starts that fall could make a line that its shares do not cover)
  const uint32_t piece_floats = a.bq * a.row_floats, more = min(d[0], gridDim.x - 1 - blockIdx.x), row0 = d[2], rows = d[3], kv = d[4];
  const int32_t start = int32_t(d[1]);
  if (!more) return;
  const float *const partials = a.partials + 2 * uint64_t(blockIdx.x) * piece_floats;
  const uint32_t quads = (p.head_dim + 3) / 4, stat = a.row_floats - 4, all = rows * quads;
  auto store = [&](const Sum &s, uint32_t i, uint32_t dim) {
    const attn::v4f y = s.o * (s.l == 0.0f ? 0.0f : 1.0f / s.l);
    const uint32_t row = row0 + i, token = a.by_group.div(row), head = kv * p.group + (row - token * p.group);
    T *out = (T *)p.out + int64_t(start + int32_t(token)) * p.o_t + int64_t(head) * p.o_h + dim;
    if constexpr (sizeof(T) == 2) {
      typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
      *(v4bf *)out = v4bf{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
    } else {
      *(attn::v4f *)out = y;
    }
  };
  // (piece 0 lies in the first workgroup's place 1, the others in place 0 of those behind it)
  if (more < MANY) {
    for (uint32_t x = blockIdx.y * THREADS + threadIdx.x; x < all; x += gridDim.y * THREADS) {
      const uint32_t i = a.by_quads.div(x), dim = (x - i * quads) * 4;
      auto from = [&](uint32_t v) { return partials + (2 * uint64_t(v) + (v == 0)) * piece_floats + i * a.row_floats; };
      store(more < 2 ? sum_of<2>(0, more, stat, dim, from) : sum_of<MANY>(0, more, stat, dim, from), i, dim);
    }
    return;
  }
  const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64, each = more / WAVES + 1, first = wave * each, last = min(first + each - 1, more);
  for (uint32_t x0 = blockIdx.y * 64; x0 < all; x0 += gridDim.y * 64) {
    const uint32_t x = min(x0 + lane, all - 1), i = a.by_quads.div(x), dim = (x - i * quads) * 4;
    auto from = [&](uint32_t v) { return partials + (2 * uint64_t(v) + (v == 0)) * piece_floats + i * a.row_floats; };
    met[wave][lane] = first <= more ? sum_of<8>(first, last, stat, dim, from) : NOTHING;
    __syncthreads();
    if (wave == 0 && x0 + lane < all) {
      Sum s = met[0][lane];
#pragma unroll
      for (uint32_t w = 1; w < WAVES; w++) {
        const Sum &y = met[w][lane];
        const float most = fmaxf(s.m, y.m), old = __builtin_amdgcn_exp2f(s.m - most), f = __builtin_amdgcn_exp2f(y.m - most);
        s.o = s.o * old + y.o * f, s.l = s.l * old + y.l * f, s.m = most;
      }
      store(s, i, dim);
    }
    __syncthreads();
  }
}

// How a call runs, by sizes, types and strides.
struct Choice {
  bool tiled = false;        // else the generic kernel
  int qb = 0;                // on tiles of 16 * qb rows; 0: of 128
  paged::Work work = {};
  size_t partial_bytes = 0, bytes = 0;   // of partial results in the workspace, of all of it (the descriptions lie behind)
};

Choice choose(const PagedAttnArgs &a) {
  Choice c;
  const int size = a.dtype == MRL_BF16 ? 2 : 4;
  auto chunks = [&](int64_t n) { return n * size % 16 == 0; };
  const double scale = std::fabs(a.scale);
  // Pages of whole sixteens of slots, heads and strides of whole 16-byte chunks, the slots of a page, and neighbouring pages, within 2 GB; places of
  // keys that some blocks more do not take past 31 bits; a line of blocks that its shares cover.
  c.tiled = a.page_size % 16 == 0 && a.head_dim <= 128 && chunks(a.head_dim) && chunks(a.q_t) && chunks(a.q_h) && chunks(a.o_t) && chunks(a.o_h) && chunks(a.key_p) &&
            chunks(a.key_s) && chunks(a.key_h) && chunks(a.val_p) && chunks(a.val_s) && chunks(a.val_h) && a.key_s < (1 << 24) && a.val_s < (1 << 24) &&
            a.key_p < (1 << 29) && a.val_p < (1 << 29) && a.key_s * a.page_size < (1 << 29) && a.val_s * a.page_size < (1 << 29) &&
            uint64_t(a.tokens) * a.group < (1u << 31) && uint64_t(a.width) * a.page_size <= 0x7fff0000u &&
            paged::line_fits(a.tokens, a.requests, a.group, a.kv_heads, uint64_t(a.width) * a.page_size, g_compute_units) && scale > 1e-30 && scale < 1e30;
  if (!c.tiled) return c;
  const uint64_t rows = uint64_t(a.max_new) * a.group;
  paged::Work &w = c.work;
  const bool near = a.q_t < (1 << 22) && a.q_h < (1 << 28) / int64_t(a.group);   // (a tile's queries within 2 GB of its first)
  if (a.dtype == MRL_BF16 && rows > 32 && near) {
    // us, on tiles of 128 rows and of 32, recorded into a graph.  48 rows: 16 requests to 16384 keys, 8 heads of 128 dims, 81 and 121; 4 requests to 2000 keys 25 and 36;
    // 48 requests to 8000 keys, 2 heads, 48 and 62; 24 requests to 5000 keys, 2 heads of 64 dims, 23.7 and 24.1.  24 rows, the first two 76 and 79, 23.7 and 29.5; 32 rows, the last 21.4 and
    // 27.0: of those of 17 to 32 rows that were measured the 128-row tiles are the faster, too (the border was set before).  Four rows:
    // a decoding step of 48 requests to 16384 keys 171, on tiles of 16 rows 146.
    // Requests of few rows among others go the same way: a tile of 128 rows streams its keys at what memory delivers, too (18 such requests beside 6 chunks in a launch
    // of their own on tiles of 16 rows: 53 us, 39 together).
    paged::chunk_work(a, &w);
  } else {
    c.qb = rows <= 16 ? 1 : 2;
    paged::keys_work(a, c.qb, &w);
    w.once = rows <= 16u * c.qb;
    // Tables of some hundred keys: a request's head to a workgroup, with nothing to find out before and no launch behind.  us, so and shared out: bf16, 4 requests and 16 heads of
    // 128 dims 9.1 and 14.0 at 512 keys, 15.3 and 18.2 at 1024, 27.5 and 22.3 at 2048; 16 requests and 8 such heads 10.2 and 17.6, 17.0 and 21.3, 30.0 and 33.9; 2 requests and a
    // head of 64 dims 5.8 and 9.7, 8.7 and 10.0, 12.9 and 10.3; f32, the first 20.2 and 19.8 at 512, 33.9 and 24.4 at 1024.
    // (A million workgroups are still a launch.)
    w.direct = w.once && uint64_t(a.width) * a.page_size <= (a.dtype == MRL_BF16 ? 1024u : 512u) && uint64_t(a.requests) * a.kv_heads <= 1u << 20;
  }
  if (!w.direct) {
    c.partial_bytes = (size_t(2 * w.workers) << w.bq_log2) * paged::row_floats(a) * sizeof(float);
    c.bytes = c.partial_bytes + w.workers * 32;
  }
  return c;
}

template <class T>
hipError_t launch_merge(const PagedAttnArgs &a, const Choice &c, hipStream_t stream) {
  const MergeArgs m = {c.work.merges, c.work.partials, 1u << c.work.bq_log2, paged::row_floats(a), FastDiv(a.group), FastDiv((a.head_dim + 3) / 4)};
  plan::work(plan::UNIT_STREAM, 0, double(c.bytes) / 2);
  MRL_LAUNCH(k_paged_attn_merge<T>, dim3(c.work.workers, c.qb ? 2 : 8), dim3(THREADS), 0, stream, a, m);
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
  c.work.partials = reinterpret_cast<float *>(a.workspace), c.work.merges = reinterpret_cast<uint32_t *>(a.workspace + c.partial_bytes);
  const hipError_t e = c.qb ? paged::launch_keys(a, c.work, c.qb, stream) : paged::launch_chunk(a, c.work, stream);
  if (e != hipSuccess || c.work.direct) return e;
  return bf16 ? launch_merge<u16>(a, c, stream) : launch_merge<float>(a, c, stream);
}

}  // namespace mrl
