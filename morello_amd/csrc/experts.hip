// A layer of experts for a few tokens:
//     p = softmax(router x),  the top_k largest p_e chosen,  out = sum of share_e down_e (silu(gate_e x) * up_e x)  over a token's chosen e.
//
// What bounds it is reading the wanted experts' weights, once each.  They go from memory into registers in the order in which the matrix
// instructions take them: 16 rows of weights against up to 16 of the expert's tokens, 128 bytes of each row at a time, a lane 32 of them.
// Each of the steps needs all of the one before, a launch each: logits; choice (with few tokens and experts every workgroup of the next launch makes it for itself);
// gate and up to h, a workgroup to 16 rows of one expert; down, a workgroup to 16 rows of all experts, so that a token's sum over
// its experts is formed in one place and in one order.  A choice is known by its number i = token * top_k + j; no lists go through memory but the chosen experts.
#include <algorithm>

#include "blocks_device.h"

namespace mrl {
namespace {
using namespace blocks;

// What the launches of a call leave each other in the workspace.
struct Places {
  double *logits;       // [tokens][experts]
  int32_t *chosen;      // [tokens][top_k]
  float *shares;        // [tokens][top_k]
  uint16_t *h;          // [tokens * top_k][h_s]
  uint32_t h_s;
};
size_t places(const ExpertsArgs &a, Places *to) {
  Places w = {};
  const size_t choices = size_t(a.tokens) * a.top_k;
  w.h_s = (a.inter + 63) / 64 * 64;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t *p = a.workspace ? a.workspace + at : nullptr;
    at += (bytes + 127) / 128 * 128;
    return p;
  };
  w.logits = (double *)take(sizeof(double) * a.tokens * a.experts);
  w.chosen = (int32_t *)take(4 * choices);
  w.shares = (float *)take(4 * choices);
  w.h = (uint16_t *)take(2 * choices * w.h_s);
  if (to) *to = w;
  return at;
}

__device__ inline uint32_t live_rows(const ExpertsArgs &p) { return p.rows ? uint32_t(min(max(*p.rows, 0), int32_t(p.tokens))) : p.tokens; }

__device__ inline float lo_f32(int x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float hi_f32(int x) { return __uint_as_float(uint32_t(x) & 0xffff0000u); }

// ---- Logits: a workgroup to an expert and ROUTER_TOKENS tokens, in 64 bits (a product of two bf16 numbers is exact in 32), so that which experts are chosen
// does not hang on the order of a sum. ----
constexpr int ROUTER_TOKENS = 4, ROUTER_THREADS = 256;
__global__ __launch_bounds__(ROUTER_THREADS) void k_experts_logits(ExpertsArgs p, Places w) {
  __shared__ double part[ROUTER_THREADS / 64][ROUTER_TOKENS];
  const uint32_t lane = threadIdx.x & 63, expert = blockIdx.x, t0 = blockIdx.y * ROUTER_TOKENS, rows = live_rows(p);
  if (t0 >= rows) return;
  const uint8_t *from = (const uint8_t *)(p.router + int64_t(expert) * p.router_s);
  const int count = int(min(uint32_t(ROUTER_TOKENS), rows - t0));
  double sum[ROUTER_TOKENS] = {};
  for (uint32_t k = threadIdx.x * 8; k < p.hidden; k += ROUTER_THREADS * 8) {
    const int bytes = int(p.hidden - k) * 2;
    const v4i r = chunk_up_to(from + int64_t(k) * 2, bytes);
#pragma unroll
    for (int t = 0; t < ROUTER_TOKENS; t++) {
      if (t >= count) break;
      const v4i x = chunk_up_to((const uint8_t *)(p.x + int64_t(t0 + t) * p.x_s + k), bytes);
#pragma unroll
      for (int i = 0; i < 4; i++) sum[t] += double(lo_f32(r[i]) * lo_f32(x[i])), sum[t] += double(hi_f32(r[i]) * hi_f32(x[i]));
    }
  }
#pragma unroll
  for (int t = 0; t < ROUTER_TOKENS; t++) {
    if (t >= count) break;
    for (int d = 32; d; d /= 2) sum[t] += __shfl_xor(sum[t], d);
    if (lane == 0) part[threadIdx.x / 64][t] = sum[t];
  }
  __syncthreads();
  if (int(threadIdx.x) < count) {
    double all = 0;
#pragma unroll
    for (int v = 0; v < ROUTER_THREADS / 64; v++) all += part[v][threadIdx.x];
    w.logits[uint64_t(t0 + threadIdx.x) * p.experts + expert] = all;
  }
}

// ---- Choice of a token's experts by a workgroup: the j-th is the one that j others are before ----
template <int THREADS>
struct Choice {
  double key[MOST_EXPERTS];   // logits; NaN as the lowest value
  double most;
  float sums[THREADS / 64], e[MOST_CHOSEN];
  int32_t expert[MOST_CHOSEN];
};
// Ends on a barrier: expert[0 .. top_k) are there; returns their number tid's share (for tid < top_k).
template <int THREADS>
__device__ inline float choose(const ExpertsArgs &p, const Places &w, uint32_t token, Choice<THREADS> &c) {
  constexpr int EACH = MOST_EXPERTS / THREADS;
  static_assert(MOST_EXPERTS % THREADS == 0, "");
  const uint32_t tid = threadIdx.x;
  double value[EACH], key[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t e = tid + i * THREADS;
    if (e >= p.experts) break;
    value[i] = w.logits[uint64_t(token) * p.experts + e];
    key[i] = value[i] == value[i] ? value[i] : -__builtin_inf();
    c.key[e] = key[i];
  }
  __syncthreads();
  uint32_t before[EACH] = {};
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t e = tid + i * THREADS;
    if (e >= p.experts) break;
#pragma unroll 8
    for (uint32_t o = 0; o < p.experts; o++) {
      const double k = c.key[o];
      before[i] += (k > key[i] || (k == key[i] && o < e)) ? 1 : 0;
    }
    if (before[i] == 0) c.most = key[i];
  }
  __syncthreads();
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t e = tid + i * THREADS;
    if (e >= p.experts) break;
    const float x = expf(float(value[i] - c.most));
    sum += x;
    if (before[i] < p.top_k) c.expert[before[i]] = int32_t(e), c.e[before[i]] = x;
  }
  for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
  if (tid % 64 == 0) c.sums[tid / 64] = sum;
  __syncthreads();
  sum = 0.0f;
  if (p.renormalise) {
    for (uint32_t j = 0; j < p.top_k; j++) sum += c.e[j];
  } else {
#pragma unroll
    for (int v = 0; v < THREADS / 64; v++) sum += c.sums[v];
  }
  return tid < p.top_k ? c.e[tid] / sum : 0.0f;
}
template <int THREADS>
__device__ inline void keep(const ExpertsArgs &p, const Places &w, uint32_t token, const Choice<THREADS> &c, float share) {
  if (threadIdx.x >= p.top_k) return;
  const uint32_t i = token * p.top_k + threadIdx.x;
  w.chosen[i] = c.expert[threadIdx.x], w.shares[i] = share;
  if (p.chosen) p.chosen[i] = c.expert[threadIdx.x];
  if (p.shares) p.shares[i] = share;
}
constexpr int CHOOSE_THREADS = 256;
__global__ __launch_bounds__(CHOOSE_THREADS) void k_experts_choose(ExpertsArgs p, Places w) {
  __shared__ Choice<CHOOSE_THREADS> c;
  if (blockIdx.x >= live_rows(p)) return;
  keep(p, w, blockIdx.x, c, choose(p, w, blockIdx.x, c));
}

// ---- Products with experts' weights: 16 rows from `row` on (this lane's: row + lane % 16), steps s0 .. s1 - 1 of 128 bytes a row ----
template <bool F8>
struct Weights {
  static constexpr int STEP = F8 ? 128 : 64;   // elements
  const uint8_t *row;
  const float *scales;
  __device__ inline Weights(const Stack &s, uint32_t expert, uint32_t row0, uint32_t rows) {
    const uint32_t r = min(row0 + (threadIdx.x & 15), rows - 1);
    row = s.w + (int64_t(expert) * s.w_e + int64_t(r) * s.w_s) * (F8 ? 1 : 2);
    scales = F8 ? s.scales + int64_t(expert) * s.scales_e + int64_t(row0 / BLOCK) * s.scales_s : nullptr;
  }
};
// A lane's 32 bytes of a row of weights and the x that they meet, of one step.
template <bool F8, int N>
struct Step {
  v4i q[N][2], y[F8 ? 4 : 2];
};
template <bool F8, int N>
__device__ inline void multiply(v4f (&acc)[N], const Step<F8, N> &t, const Weights<F8> (&of)[N], uint32_t s) {
#pragma unroll
  for (int n = 0; n < N; n++) {
    if constexpr (F8) {
      v4f part = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        int u[4];
        widen4(t.q[n][i / 2][i % 2 * 2], u[0], u[1]);
        widen4(t.q[n][i / 2][i % 2 * 2 + 1], u[2], u[3]);
        part = mma_bf16(v4i{u[0], u[1], u[2], u[3]}, t.y[i], part);
      }
      acc[n] += part * of[n].scales[s];
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) acc[n] = mma_bf16(t.q[n][i], t.y[i], acc[n]);
    }
  }
}
// acc[i] += of[i]'s rows against the lane's token's x (nullptr: zeros), k elements in all.  AHEAD steps' loads are asked for together.
template <bool F8, int N, int AHEAD>
__device__ inline void products(v4f (&acc)[N], const Weights<F8> (&of)[N], const uint16_t *x, uint32_t s0, uint32_t s1, int k) {
  constexpr int STEP = Weights<F8>::STEP, EACH = STEP / 4, SIZE = F8 ? 1 : 2;   // elements of a lane, bytes of one
  const int lg = (threadIdx.x & 63) >> 4;
  const uint32_t whole = min(s1, uint32_t(k / STEP));
  uint32_t s = s0;
  for (; s + AHEAD <= whole; s += AHEAD) {
    Step<F8, N> t[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      const int64_t at = int64_t(s + a) * STEP + lg * EACH;
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) t[a].q[n][i] = chunk_at(of[n].row + at * SIZE + i * 16);
#pragma unroll
      for (int i = 0; i < EACH / 8; i++) t[a].y[i] = v4i{0, 0, 0, 0};
    }
    if (x) {
#pragma unroll
      for (int a = 0; a < AHEAD; a++)
#pragma unroll
        for (int i = 0; i < EACH / 8; i++) t[a].y[i] = chunk_at((const uint8_t *)(x + int64_t(s + a) * STEP + lg * EACH + i * 8));
    }
#pragma unroll
    for (int a = 0; a < AHEAD; a++) multiply<F8, N>(acc, t[a], of, s + a);
  }
  for (; s < s1; s++) {   // the steps left, and the one that holds the rows' ends
    Step<F8, N> t;
    const int at = int(s) * STEP + lg * EACH;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < 2; i++) t.q[n][i] = chunk_up_to(of[n].row + at * SIZE + i * 16, (k - at) * SIZE - i * 16);
#pragma unroll
    for (int i = 0; i < EACH / 8; i++) t.y[i] = x ? chunk_up_to((const uint8_t *)(x + at + i * 8), (k - at - i * 8) * 2) : v4i{0, 0, 0, 0};
    multiply<F8, N>(acc, t, of, s);
  }
}

// ---- Gate and up.  blockIdx.x: an expert, or where there are fewer choices than experts a choice, which stands for its expert if no earlier one does.
// FUSED: from logits, the choices made here. ----
constexpr int UP_WAVES = 4;
constexpr uint32_t FUSED_TOKENS = 4;
template <bool F8, bool FUSED>
__global__ __launch_bounds__(UP_WAVES * 64) void k_experts_up(ExpertsArgs p, Places w) {
  __shared__ v4f part[UP_WAVES][2][64];
  __shared__ uint16_t choices[MOST_TOKENS];   // of this expert, ascending
  __shared__ int32_t chosen[FUSED ? FUSED_TOKENS * MOST_CHOSEN : 1];
  const uint32_t lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const uint32_t row0 = blockIdx.y * 16, rows = live_rows(p), all = rows * p.top_k;
  if constexpr (FUSED) {
    __shared__ Choice<UP_WAVES * 64> c;
    for (uint32_t t = 0; t < rows; t++) {
      const float share = choose(p, w, t, c);
      if (threadIdx.x < p.top_k) chosen[t * p.top_k + threadIdx.x] = c.expert[threadIdx.x];
      if (blockIdx.x == 0 && blockIdx.y == 0) keep(p, w, t, c, share);
      __syncthreads();
    }
  }
  const int32_t *const of_choice = FUSED ? chosen : w.chosen;
  uint32_t expert = blockIdx.x;
  if (p.tokens * p.top_k < p.experts) {
    if (expert >= all) return;
    expert = uint32_t(of_choice[blockIdx.x]);
  }
  // Every wave goes through the choices; the first writes down the expert's.
  uint32_t count = 0;
  for (uint32_t i0 = 0; i0 < all; i0 += 64) {
    const uint32_t i = i0 + lane;
    const bool mine = i < all && uint32_t(of_choice[i]) == expert;
    const uint64_t mask = __ballot(mine);
    if (mine && wave == 0) choices[count + __popcll(mask & ((1ull << lane) - 1))] = uint16_t(i);
    count += __popcll(mask);
  }
  if (count == 0) return;
  __syncthreads();
  if (p.tokens * p.top_k < p.experts && choices[0] != blockIdx.x) return;
  const Weights<F8> of[2] = {{p.gate, expert, row0, p.inter}, {p.up, expert, row0, p.inter}};
  const uint32_t steps = (p.hidden + Weights<F8>::STEP - 1) / Weights<F8>::STEP;
  for (uint32_t c0 = 0; c0 < count; c0 += 16) {
    const bool mine = c0 + li < count;
    const uint32_t choice = choices[min(c0 + li, count - 1)];
    v4f acc[2] = {};
    products<F8, 2, F8 ? 2 : 4>(acc, of, mine ? p.x + int64_t(choice / p.top_k) * p.x_s : nullptr, steps * wave / UP_WAVES, steps * (wave + 1) / UP_WAVES, int(p.hidden));
    if (c0) __syncthreads();
    part[wave][0][lane] = acc[0], part[wave][1][lane] = acc[1];
    __syncthreads();
    if (wave == 0 && mine) {
      v4f g = part[0][0][lane], u = part[0][1][lane], h;
#pragma unroll
      for (int v = 1; v < UP_WAVES; v++) g += part[v][0][lane], u += part[v][1][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) h[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
      const uint32_t row = row0 + lg * 4;
      if (row < p.inter) store4(w.h + uint64_t(choice) * w.h_s + row, h, int(p.inter - row));
    }
  }
}

// ---- Down: blockIdx.x: 16 rows; blockIdx.y: DOWN_TOKENS tokens ----
constexpr int DOWN_WAVES = 16, DOWN_TOKENS = 64;
constexpr int DOWN_THREADS = DOWN_WAVES * 64;
template <bool F8>
__global__ __launch_bounds__(DOWN_THREADS) void k_experts_down(ExpertsArgs p, Places w, uint32_t tokens_here, uint32_t words) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dynamic[];
  v4f *const sums = (v4f *)dynamic;                                                       // [DOWN_WAVES][tokens_here][4]
  uint32_t *const wants = (uint32_t *)(sums + DOWN_WAVES * tokens_here * 4);              // [experts][words] a bit for each token of this workgroup's
  uint16_t *const choices = (uint16_t *)(wants + p.experts * words);                      // [tokens_here * top_k] expert after expert
  __shared__ uint16_t expert_of[MOST_EXPERTS], first[MOST_EXPERTS + 1], first_of[MOST_EXPERTS];
  __shared__ int32_t totals[2][MOST_EXPERTS / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const uint32_t row0 = blockIdx.x * 16, t0 = blockIdx.y * DOWN_TOKENS, rows = live_rows(p);
  if (t0 >= rows) return;
  const uint32_t here = min(tokens_here, rows - t0), all = here * p.top_k;
  const int32_t *const chosen = w.chosen + t0 * p.top_k;
  for (uint32_t i = tid; i < p.experts * words; i += DOWN_THREADS) wants[i] = 0;
  for (uint32_t i = lane; i < here * 4; i += 64) sums[wave * tokens_here * 4 + i] = v4f{0, 0, 0, 0};
  __syncthreads();
  for (uint32_t i = tid; i < all; i += DOWN_THREADS) {
    const uint32_t t = i / p.top_k;
    atomicOr(&wants[uint32_t(chosen[i]) * words + t / 32], 1u << (t % 32));
  }
  __syncthreads();
  // Wanted experts, and choices, before each expert.
  int32_t count = 0;
  if (tid < p.experts)
    for (uint32_t j = 0; j < words; j++) count += __popc(wants[tid * words + j]);
  int32_t before = count, slot = count > 0;
  if (tid < MOST_EXPERTS) {
    for (int d = 1; d < 64; d *= 2) {
      const int32_t x = __shfl_up(before, d), y = __shfl_up(slot, d);
      if (int(lane) >= d) before += x, slot += y;
    }
    if (lane == 63) totals[0][wave] = before, totals[1][wave] = slot;
  }
  __syncthreads();
  uint32_t active = 0;
  for (uint32_t v = 0; v < MOST_EXPERTS / 64; v++) {
    if (v < wave) before += totals[0][v], slot += totals[1][v];
    active += totals[1][v];
  }
  if (tid < p.experts) {
    first_of[tid] = uint16_t(before - count);
    if (count > 0) expert_of[slot - 1] = uint16_t(tid), first[slot - 1] = uint16_t(before - count);
  }
  if (tid == 0) first[active] = uint16_t(all);
  __syncthreads();
  for (uint32_t i = tid; i < all; i += DOWN_THREADS) {
    const uint32_t t = i / p.top_k, e = uint32_t(chosen[i]);
    uint32_t at = first_of[e];
    for (uint32_t j = 0; j < t / 32; j++) at += __popc(wants[e * words + j]);
    choices[at + __popc(wants[e * words + t / 32] & ((1u << (t % 32)) - 1))] = uint16_t(i);
  }
  __syncthreads();
  const uint32_t steps = (p.inter + Weights<F8>::STEP - 1) / Weights<F8>::STEP;
  // All experts' steps in a line, an equal share to each wave.
  const uint32_t line = active * steps, begin = uint32_t(uint64_t(line) * wave / DOWN_WAVES), end = uint32_t(uint64_t(line) * (wave + 1) / DOWN_WAVES);
  for (uint32_t at = begin; at < end;) {
    const uint32_t slot_at = at / steps, s0 = at - slot_at * steps, s1 = min(steps, s0 + (end - at));
    at += s1 - s0;
    const Weights<F8> of[1] = {{p.down, expert_of[slot_at], row0, p.hidden}};
    const uint32_t last = first[slot_at + 1];
    for (uint32_t c0 = first[slot_at]; c0 < last; c0 += 16) {
      const bool mine = c0 + li < last;
      const uint32_t local = choices[min(c0 + li, last - 1)], choice = t0 * p.top_k + local;
      v4f acc[1] = {};
      products<F8, 1, F8 ? 2 : 4>(acc, of, mine ? w.h + uint64_t(choice) * w.h_s : nullptr, s0, s1, int(p.inter));
      if (mine) sums[(wave * tokens_here + local / p.top_k) * 4 + lg] += acc[0] * w.shares[choice];
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < here * 4; i += DOWN_THREADS) {
    v4f sum = sums[i];
#pragma unroll
    for (uint32_t v = 1; v < DOWN_WAVES; v++) sum += sums[v * tokens_here * 4 + i];
    const uint32_t row = row0 + i % 4 * 4;
    if (row < p.hidden) store4(p.out + int64_t(t0 + i / 4) * p.out_s + row, sum, int(p.hidden - row));
  }
}

template <bool F8>
hipError_t launch(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  const uint32_t choices = a.tokens * a.top_k, slots = std::min(a.experts, choices);
  const double weight = 3.0 * a.inter * a.hidden * (F8 ? 1 : 2) * slots;
  plan::work(plan::UNIT_STREAM, 0, 2.0 * (double(a.experts) + a.tokens) * a.hidden);
  MRL_LAUNCH(k_experts_logits, dim3(a.experts, (a.tokens + ROUTER_TOKENS - 1) / ROUTER_TOKENS), dim3(ROUTER_THREADS), 0, stream, a, w);
  const bool fused = a.tokens <= FUSED_TOKENS && a.tokens * a.experts * a.experts <= 1u << 16;
  if (!fused) {
    plan::work(plan::UNIT_STREAM, 0, 8.0 * a.experts * a.tokens);
    MRL_LAUNCH(k_experts_choose, dim3(a.tokens), dim3(CHOOSE_THREADS), 0, stream, a, w);
  }
  plan::work(plan::UNIT_STREAM, 0, weight * 2 / 3);
  const dim3 up(slots, (a.inter + 15) / 16);
  if (fused) MRL_LAUNCH((k_experts_up<F8, true>), up, dim3(UP_WAVES * 64), 0, stream, a, w);
  else MRL_LAUNCH((k_experts_up<F8, false>), up, dim3(UP_WAVES * 64), 0, stream, a, w);
  const uint32_t here = std::min(a.tokens, uint32_t(DOWN_TOKENS)), words = (here + 31) / 32;
  const size_t lds = size_t(DOWN_WAVES) * here * 64 + size_t(a.experts) * words * 4 + size_t(here) * a.top_k * 2;
  static std::atomic<uint64_t> raised{0};
  if (lds > 48 * 1024 && !plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_experts_down<F8>), 96 * 1024);
    if (e != hipSuccess) return e;
  }
  plan::work(plan::UNIT_STREAM, 0, weight / 3);
  MRL_LAUNCH(k_experts_down<F8>, dim3((a.hidden + 15) / 16, (a.tokens + DOWN_TOKENS - 1) / DOWN_TOKENS), dim3(DOWN_THREADS), lds, stream, a, w, here, words);
  return plan::last_error();
}

}  // namespace

size_t experts_workspace_bytes(const ExpertsArgs &a) { return places(a, nullptr); }

hipError_t launch_experts(const ExpertsArgs &a, hipStream_t stream) {
  Places w;
  places(a, &w);
  return a.weight_dtype == MRL_BF16 ? launch<false>(a, w, stream) : launch<true>(a, w, stream);
}

}  // namespace mrl
