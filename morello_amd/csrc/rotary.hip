// Rotary positions: each pair (x, y) of a head's dims turned by its token's angle, queries to queries, keys (and the values as
// they are) to a dense tensor or into the slots of a cache of pages.
//     angle = positions[axis(i)][t] * frequencies[i],   (x, y) -> (x cos - y sin, y cos + x sin)
// A position past 2^24 is not a 32-bit float, and of a large product nothing but the part behind the last whole turn counts: the
// angle is formed in turns, in 64 bits, and what is left of it, at most half a turn, goes to sine and cosine in 32 as the nearest
// float and the rest behind it, which enters to first order (a half turn's rounding alone would be 1.9e-7 of a sine).
//
// A token to a workgroup, or to up to four where it has more than 256 threads' worth of heads: its angles' sines and cosines once, in LDS, for all heads; then 16 bytes of
// either half of a pair to a thread.  What bounds it: q, k and v read once and written once.  4101 tokens of 32 + 8 + 8 heads of 128 dims in bf16, three axes, into pages: 100.8 MB in
// 21.6 us, 4.7 TB/s (a copy of 1 GiB: 5.0); 2048 tokens of 32 heads of 80 dims in f32: 42 MB in 11 us; a decoding step of 32 tokens: 3.4 us, a launch.
#include <cmath>

#include "paged.h"

namespace mrl {
namespace {

constexpr int THREADS = 256;

typedef unsigned short u16;
__device__ inline float to_f32(u16 x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float to_f32(float x) { return x; }
template <class T>
__device__ inline T from_f32(float x);
template <>
__device__ inline u16 from_f32<u16>(float x) { return __builtin_bit_cast(u16, (__bf16)x); }
template <>
__device__ inline float from_f32<float>(float x) { return x; }

template <class T, int V>
struct Chunk {
  T x[V];
} __attribute__((aligned(sizeof(T) * V)));

// V: elements a thread moves at once (16 bytes), or 1 where sizes, strides or addresses do not allow that.
template <class T, int V, bool ADJACENT>
__global__ __launch_bounds__(THREADS) void k_rotary(RotaryArgs p, uint32_t items, FastDiv by_turned, FastDiv by_chunks, FastDiv by_page) {
  extern __shared__ float2 turns[];   // [pair]: cosine, sine
  const uint32_t t = blockIdx.x;
  for (uint32_t pair = threadIdx.x; pair < p.pairs; pair += THREADS) {
    uint32_t axis = 0;
#pragma unroll
    for (int a = 0; a < MRL_MAX_AXES - 1; a++) axis += pair >= p.section_end[a];
    constexpr double TURNS = 0.15915494309189533577;   // 1 / (2 pi)
    const double all = double(p.positions[uint64_t(axis) * p.tokens + t]) * (double(p.frequencies[pair]) * TURNS);
    const double part = all - rint(all);
    const float near = float(part), rest = float((part - double(near)) * 6.283185307179586477);
    float s, c;
    sincospif(2.0f * near, &s, &c);
    const float sine = s + c * rest;
    turns[pair] = float2{c - s * rest, p.inverse ? -sine : sine};
  }
  __syncthreads();
  // A token's items: of each query and key head the chunks of its pairs' first halves (ADJACENT: of its pairs) and of the dims behind
  // the pairs, then of each value head its chunks.
  const uint32_t whole = p.head_dim / V, first = ADJACENT ? 2 * p.pairs / V : p.pairs / V, turned = whole - (ADJACENT ? 0 : first);
  const bool paged = p.page_size != 0;
  const uint32_t heads = p.q_heads + p.kv_heads;
  typedef Chunk<T, V> C;
  for (uint32_t item = blockIdx.y * THREADS + threadIdx.x; item < items; item += THREADS * gridDim.y) {
    int64_t to_key = 0, to_value = 0;
    bool kept = true;
    if (item >= p.q_heads * turned) {
      if (paged) {
        const int32_t slot = p.slots[t];
        kept = slot >= 0 && uint32_t(slot) < p.slot_count;
        const uint32_t page = kept ? by_page.div(uint32_t(slot)) : 0, place = kept ? uint32_t(slot) - page * p.page_size : 0;
        to_key = int64_t(page) * p.key_p + int64_t(place) * p.key_s, to_value = int64_t(page) * p.val_p + int64_t(place) * p.val_s;
      } else {
        to_key = int64_t(t) * p.key_s;
      }
      if (!kept) continue;
    }
    if (item >= heads * turned) {
      const uint32_t j = item - heads * turned, head = by_chunks.div(j), chunk = j - head * whole;
      const C x = *(const C *)((const T *)p.v + int64_t(t) * p.v_t + int64_t(head) * p.v_h + chunk * V);
      *(C *)((T *)p.values + to_value + int64_t(head) * p.val_h + chunk * V) = x;
      continue;
    }
    const uint32_t head = by_turned.div(item);
    uint32_t chunk = item - head * turned;
    const bool query = head < p.q_heads;
    const T *from = query ? (const T *)p.q + int64_t(t) * p.q_t + int64_t(head) * p.q_h : (const T *)p.k + int64_t(t) * p.k_t + int64_t(head - p.q_heads) * p.k_h;
    T *to = query ? (T *)p.q_out + int64_t(t) * p.qo_t + int64_t(head) * p.qo_h : (T *)p.keys + to_key + int64_t(head - p.q_heads) * p.key_h;
    if (chunk >= first) {   // behind the pairs
      if (!ADJACENT) chunk += first;
      *(C *)(to + chunk * V) = *(const C *)(from + chunk * V);
      continue;
    }
    if constexpr (ADJACENT && V > 1) {
      C x = *(const C *)(from + chunk * V);
      const float2 *turn = turns + chunk * (V / 2);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 w = turn[e / 2];
        const float a = to_f32(x.x[e]), b = to_f32(x.x[e + 1]);
        x.x[e] = from_f32<T>(a * w.x - b * w.y), x.x[e + 1] = from_f32<T>(b * w.x + a * w.y);
      }
      *(C *)(to + chunk * V) = x;
    } else {
      // (ADJACENT with single elements: `chunk` is one of 2 * pairs, the even ones do the pair)
      if (ADJACENT && chunk % 2) continue;
      const uint32_t lo = chunk * V, hi = ADJACENT ? lo + 1 : lo + p.pairs;
      C x = *(const C *)(from + lo), y = *(const C *)(from + hi);
      const float2 *turn = turns + (ADJACENT ? chunk / 2 : lo);
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float2 w = turn[e];
        const float a = to_f32(x.x[e]), b = to_f32(y.x[e]);
        x.x[e] = from_f32<T>(a * w.x - b * w.y), y.x[e] = from_f32<T>(b * w.x + a * w.y);
      }
      *(C *)(to + lo) = x;
      *(C *)(to + hi) = y;
    }
  }
}

template <class T, int V, bool ADJACENT>
hipError_t launch_one(const RotaryArgs &a, hipStream_t stream) {
  const uint32_t whole = a.head_dim / V, turned = whole - (ADJACENT ? 0 : a.pairs / V);
  const uint64_t items = uint64_t(a.q_heads + a.kv_heads) * turned + (a.page_size ? uint64_t(a.kv_heads) * whole : 0);
  const uint32_t split = uint32_t(std::max<uint64_t>(1, std::min<uint64_t>((items + THREADS - 1) / THREADS, 4)));
  const double bytes = 2.0 * sizeof(T) * a.tokens * double(a.q_heads + (a.page_size ? 2 : 1) * a.kv_heads) * a.head_dim;
  plan::work(plan::UNIT_STREAM, 0, bytes);
  MRL_LAUNCH((k_rotary<T, V, ADJACENT>), dim3(a.tokens, split), dim3(THREADS), a.pairs * sizeof(float2), stream, a, uint32_t(items), FastDiv(turned), FastDiv(whole), FastDiv(a.page_size ? a.page_size : 1));
  return plan::last_error();
}

template <class T>
hipError_t launch_for(const RotaryArgs &a, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  auto whole = [](int64_t n) { return n % V == 0; };
  auto aligned = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool wide = whole(a.head_dim) && whole(a.adjacent ? 2 * a.pairs : a.pairs) && whole(a.q_t) && whole(a.q_h) && whole(a.k_t) && whole(a.k_h) && whole(a.v_t) &&
                    whole(a.v_h) && whole(a.qo_t) && whole(a.qo_h) && whole(a.key_p) && whole(a.key_s) && whole(a.key_h) && whole(a.val_p) && whole(a.val_s) &&
                    whole(a.val_h) && aligned(a.q) && aligned(a.k) && aligned(a.v) && aligned(a.q_out) && aligned(a.keys) && aligned(a.values);
  if (a.adjacent) return wide ? launch_one<T, V, true>(a, stream) : launch_one<T, 1, true>(a, stream);
  return wide ? launch_one<T, V, false>(a, stream) : launch_one<T, 1, false>(a, stream);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs &a, hipStream_t stream) {
  return a.dtype == MRL_BF16 ? launch_for<u16>(a, stream) : launch_for<float>(a, stream);
}

}  // namespace mrl
