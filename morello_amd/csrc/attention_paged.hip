// Attention of requests' new tokens over their pages of keys and values.
#include <algorithm>
#include <cmath>

#include "paged.h"

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

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnArgs &) { return 0; }

hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream) {
  return a.dtype == MRL_BF16 ? launch_generic<u16>(a, stream) : launch_generic<float>(a, stream);
}

}  // namespace mrl
