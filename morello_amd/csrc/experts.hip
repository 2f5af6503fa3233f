// A layer of experts for a few tokens:
//     p = softmax(router x),  the top_k largest p_e chosen,  out = sum of share_e down_e (silu(gate_e x) * up_e x)  over a token's chosen e.
//
// What bounds it is reading the wanted experts' weights, once each.  They go from memory into registers in the order in which the matrix
// instructions take them: 16 rows of weights against up to 16 of the expert's tokens, 128 bytes of each row at a time, a lane 32 of them.
// Three dependent things have to be done, a launch for each: logits; choice, and the experts' lists of tokens;
// gate and up to h (a workgroup to 16 rows of one expert); down (a workgroup to 16 rows of all experts, so that a token's sum over
// its experts is formed in one place and in one order).
#include <algorithm>

#include "blocks_device.h"

namespace mrl {
namespace {
using namespace blocks;

// What the launches of a call leave each other in the workspace.
struct Places {
  double *logits;       // [tokens][experts]
  int32_t *active;      // [1] experts that some token chose
  int32_t *expert;      // [slots] which, ascending
  int32_t *first;       // [slots + 1] their first entries; the entries of an expert are its tokens, ascending
  int32_t *token;       // [tokens * top_k] of an entry
  float *share;         // [tokens * top_k]
  uint16_t *h;          // [tokens * top_k][h_s]
  uint32_t slots, h_s;
};
size_t places(const ExpertsArgs &a, Places *to) {
  Places w = {};
  const size_t entries = size_t(a.tokens) * a.top_k;
  w.slots = uint32_t(std::min<size_t>(a.experts, entries));
  w.h_s = (a.inter + 127) / 128 * 128;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t *p = a.workspace ? a.workspace + at : nullptr;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  w.logits = (double *)take(sizeof(double) * a.tokens * a.experts);
  w.active = (int32_t *)take(4);
  w.expert = (int32_t *)take(4 * size_t(w.slots));
  w.first = (int32_t *)take(4 * (size_t(w.slots) + 1));
  w.token = (int32_t *)take(4 * entries);
  w.share = (float *)take(4 * entries);
  w.h = (uint16_t *)take(2 * entries * w.h_s);
  if (to) *to = w;
  return at;
}

__device__ inline uint32_t live_rows(const ExpertsArgs &p) { return p.rows ? uint32_t(min(max(*p.rows, 0), int32_t(p.tokens))) : p.tokens; }

__device__ inline float lo_f32(int x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float hi_f32(int x) { return __uint_as_float(uint32_t(x) & 0xffff0000u); }

// ---- Logits: a wave to an expert and TOKENS tokens, in 64 bits (a product of two bf16 numbers is exact in 32), so that which experts are chosen does not
// hang on the order of a sum. ----
constexpr int ROUTER_TOKENS = 8;
__global__ __launch_bounds__(256) void k_experts_logits(ExpertsArgs p, Places w) {
  const uint32_t lane = threadIdx.x & 63, expert = blockIdx.x * 4 + threadIdx.x / 64, t0 = blockIdx.y * ROUTER_TOKENS, rows = live_rows(p);
  if (expert >= p.experts || t0 >= rows) return;
  const uint8_t *from = (const uint8_t *)(p.router + int64_t(expert) * p.router_s);
  const int count = int(min(uint32_t(ROUTER_TOKENS), rows - t0));
  double sum[ROUTER_TOKENS] = {};
  for (uint32_t k = lane * 8; k < p.hidden; k += 512) {
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
    if (lane == 0) w.logits[uint64_t(t0 + t) * p.experts + expert] = sum[t];
  }
}

// ---- Choice: a wave to a token, then the lists of all experts ----
constexpr int CHOOSE_THREADS = 1024;
__global__ __launch_bounds__(CHOOSE_THREADS) void k_experts_choose(ExpertsArgs p, Places w) {
  constexpr int EACH = MOST_EXPERTS / 64, WORDS = MOST_TOKENS / 32;
  __shared__ uint32_t wants[MOST_EXPERTS][WORDS + 1];   // a bit for each token
  __shared__ int32_t sums[2][CHOOSE_THREADS / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rows = live_rows(p);
  for (uint32_t i = tid; i < MOST_EXPERTS * (WORDS + 1); i += CHOOSE_THREADS) (&wants[0][0])[i] = 0;
  __syncthreads();
  extern __shared__ __attribute__((aligned(16))) uint8_t dynamic[];   // expert and share of each choice
  int32_t *const chosen = (int32_t *)dynamic;
  float *const shares = (float *)(chosen + p.tokens * p.top_k);
  for (uint32_t t = wave; t < rows; t += CHOOSE_THREADS / 64) {
    const double *l = w.logits + uint64_t(t) * p.experts;
    double value[EACH], most = -__builtin_inf();
    uint32_t left = 0;   // a bit for each of the lane's experts that are not chosen yet
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const uint32_t e = lane + i * 64;
      value[i] = e < p.experts ? l[e] : 0.0;
      if (e < p.experts) left |= 1u << i;
      if (e < p.experts && value[i] > most) most = value[i];   // (NaN: not)
    }
    for (int d = 32; d; d /= 2) most = fmax(most, __shfl_xor(most, d));
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; i++)
      if (lane + i * 64 < p.experts) total += expf(float(value[i] - most));
    for (int d = 32; d; d /= 2) total += __shfl_xor(total, d);
    float chosen_total = 0.0f;
    for (uint32_t j = 0; j < p.top_k; j++) {
      // The largest left, of equal ones the lowest; NaN counts as the lowest value.
      double best = -__builtin_inf();
      int32_t which = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        const double v = value[i] == value[i] ? value[i] : -__builtin_inf();
        const int32_t e = int32_t(lane + i * 64);
        if ((left >> i & 1) && (v > best || (v == best && e < which))) best = v, which = e;
      }
      for (int d = 32; d; d /= 2) {
        const double v = __shfl_xor(best, d);
        const int32_t e = __shfl_xor(which, d);
        if (v > best || (v == best && e < which)) best = v, which = e;
      }
      // (top_k is at most the experts: there is one left)
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < EACH; i++)
        if (which == int32_t(lane + i * 64)) left &= ~(1u << i), mine = expf(float(value[i] - most));
      const float e = __shfl(mine, which & 63);
      chosen_total += e;
      if (lane == 0) {
        chosen[t * p.top_k + j] = which, shares[t * p.top_k + j] = e;
        atomicOr(&wants[which][t / 32], 1u << (t % 32));
      }
    }
    const float by = p.renormalise ? chosen_total : total;
    __builtin_amdgcn_wave_barrier();
    for (uint32_t j = lane; j < p.top_k; j += 64) {
      const float s = shares[t * p.top_k + j] / by;
      shares[t * p.top_k + j] = s;
      if (p.chosen) p.chosen[uint64_t(t) * p.top_k + j] = chosen[t * p.top_k + j];
      if (p.shares) p.shares[uint64_t(t) * p.top_k + j] = s;
    }
  }
  __syncthreads();
  // Entries before each expert, and experts with any before it.
  int32_t count = 0;
  if (tid < p.experts)
    for (int i = 0; i < WORDS; i++) count += __popc(wants[tid][i]);
  int32_t before = count, slot = count > 0;
  for (int d = 1; d < 64; d *= 2) {
    const int32_t x = __shfl_up(before, d), y = __shfl_up(slot, d);
    if (int(lane) >= d) before += x, slot += y;
  }
  if (lane == 63) sums[0][wave] = before, sums[1][wave] = slot;
  __syncthreads();
  int32_t all = 0;
  for (uint32_t v = 0; v < CHOOSE_THREADS / 64; v++) {
    if (v < wave) before += sums[0][v], slot += sums[1][v];
    all += sums[1][v];
  }
  before -= count, slot -= count > 0;
  if (tid < p.experts) wants[tid][WORDS] = uint32_t(before);
  if (count > 0) w.expert[slot] = int32_t(tid), w.first[slot] = before;
  if (tid == 0) w.active[0] = all, w.first[all] = int32_t(rows * p.top_k);
  __syncthreads();
  for (uint32_t i = tid; i < rows * p.top_k; i += CHOOSE_THREADS) {
    const uint32_t t = i / p.top_k, e = uint32_t(chosen[i]);
    uint32_t at = wants[e][WORDS];
    for (uint32_t j = 0; j < t / 32; j++) at += __popc(wants[e][j]);
    at += __popc(wants[e][t / 32] & ((1u << (t % 32)) - 1));
    w.token[at] = int32_t(t), w.share[at] = shares[i];
  }
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
// acc[i] += of[i]'s rows against the lane's token's x (nullptr: zeros), k elements in all.
template <bool F8, int N>
__device__ inline void products(v4f (&acc)[N], const Weights<F8> (&of)[N], const uint16_t *x, uint32_t s0, uint32_t s1, int k) {
  constexpr int STEP = Weights<F8>::STEP, EACH = STEP / 4;   // elements of a lane
  const int lg = (threadIdx.x & 63) >> 4;
  for (uint32_t s = s0; s < s1; s++) {
    const int at = int(s) * STEP + lg * EACH;
    v4i y[EACH / 8];
#pragma unroll
    for (int i = 0; i < EACH / 8; i++) y[i] = x ? chunk_up_to((const uint8_t *)(x + at + i * 8), (k - at - i * 8) * 2) : v4i{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < N; n++) {
      if constexpr (F8) {
        v4f part = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const v4i q = chunk_up_to(of[n].row + at + i * 16, k - at - i * 16);
#pragma unroll
          for (int j = 0; j < 2; j++) {
            int u[4];
            widen4(q[2 * j], u[0], u[1]);
            widen4(q[2 * j + 1], u[2], u[3]);
            part = mma_bf16(v4i{u[0], u[1], u[2], u[3]}, y[i * 2 + j], part);
          }
        }
        acc[n] += part * of[n].scales[s];
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) acc[n] = mma_bf16(chunk_up_to(of[n].row + (at + i * 8) * 2, (k - at - i * 8) * 2), y[i], acc[n]);
      }
    }
  }
}

constexpr int UP_WAVES = 4;
template <bool F8>
__global__ __launch_bounds__(UP_WAVES * 64) void k_experts_up(ExpertsArgs p, Places w) {
  __shared__ v4f part[UP_WAVES][2][64];
  const uint32_t slot = blockIdx.x, row0 = blockIdx.y * 16;
  if (slot >= uint32_t(*w.active)) return;
  const uint32_t expert = uint32_t(w.expert[slot]), first = uint32_t(w.first[slot]), end = uint32_t(w.first[slot + 1]);
  const uint32_t lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const Weights<F8> of[2] = {{p.gate, expert, row0, p.inter}, {p.up, expert, row0, p.inter}};
  const uint32_t steps = (p.hidden + Weights<F8>::STEP - 1) / Weights<F8>::STEP;
  for (uint32_t e0 = first; e0 < end; e0 += 16) {
    const uint32_t entry = e0 + li;
    const uint16_t *x = entry < end ? p.x + int64_t(w.token[entry]) * p.x_s : nullptr;
    v4f acc[2] = {};
    products<F8, 2>(acc, of, x, steps * wave / UP_WAVES, steps * (wave + 1) / UP_WAVES, int(p.hidden));
    __syncthreads();
    part[wave][0][lane] = acc[0], part[wave][1][lane] = acc[1];
    __syncthreads();
    if (wave == 0 && entry < end) {
      v4f g = part[0][0][lane], u = part[0][1][lane], h;
#pragma unroll
      for (int v = 1; v < UP_WAVES; v++) g += part[v][0][lane], u += part[v][1][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) h[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
      const uint32_t row = row0 + lg * 4;
      if (row < p.inter) store4(w.h + uint64_t(entry) * w.h_s + row, h, int(p.inter - row));
    }
  }
}

constexpr int DOWN_WAVES = 8, DOWN_TOKENS = 64;   // tokens of a workgroup
template <bool F8>
__global__ __launch_bounds__(DOWN_WAVES * 64) void k_experts_down(ExpertsArgs p, Places w) {
  __shared__ v4f sums[DOWN_WAVES][DOWN_TOKENS][4];
  const uint32_t row0 = blockIdx.x * 16, t0 = blockIdx.y * DOWN_TOKENS, rows = live_rows(p);
  if (t0 >= rows) return;
  const uint32_t t1 = min(t0 + DOWN_TOKENS, rows);
  const uint32_t lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  for (uint32_t i = lane; i < DOWN_TOKENS * 4; i += 64) (&sums[wave][0][0])[i] = v4f{0, 0, 0, 0};
  const uint32_t steps = (p.inter + Weights<F8>::STEP - 1) / Weights<F8>::STEP, active = uint32_t(*w.active);
  // All experts' steps in a line, an equal share to each wave.
  const uint32_t all = active * steps, begin = uint32_t(uint64_t(all) * wave / DOWN_WAVES), end = uint32_t(uint64_t(all) * (wave + 1) / DOWN_WAVES);
  for (uint32_t at = begin; at < end;) {
    const uint32_t slot = at / steps, s0 = at - slot * steps, s1 = min(steps, s0 + (end - at));
    at += s1 - s0;
    const Weights<F8> of[1] = {{p.down, uint32_t(w.expert[slot]), row0, p.hidden}};
    const uint32_t last = uint32_t(w.first[slot + 1]);
    for (uint32_t e0 = uint32_t(w.first[slot]); e0 < last; e0 += 16) {
      const uint32_t entry = e0 + li, token = entry < last ? uint32_t(w.token[entry]) : 0xffffffffu;
      const bool mine = token >= t0 && token < t1;
      if (!__any(mine)) continue;
      v4f acc[1] = {};
      products<F8, 1>(acc, of, mine ? w.h + uint64_t(entry) * w.h_s : nullptr, s0, s1, int(p.inter));
      if (mine) sums[wave][token - t0][lg] += acc[0] * w.share[entry];
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (t1 - t0) * 4; i += DOWN_WAVES * 64) {
    v4f sum = sums[0][i / 4][i % 4];
#pragma unroll
    for (int v = 1; v < DOWN_WAVES; v++) sum += sums[v][i / 4][i % 4];
    const uint32_t row = row0 + i % 4 * 4;
    if (row < p.hidden) store4(p.out + int64_t(t0 + i / 4) * p.out_s + row, sum, int(p.hidden - row));
  }
}

template <bool F8>
hipError_t launch(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  const double weight = 3.0 * a.inter * a.hidden * (F8 ? 1 : 2) * w.slots;
  plan::work(plan::UNIT_STREAM, 0, 2.0 * (double(a.experts) + a.tokens) * a.hidden);
  MRL_LAUNCH(k_experts_logits, dim3((a.experts + 3) / 4, (a.tokens + ROUTER_TOKENS - 1) / ROUTER_TOKENS), dim3(256), 0, stream, a, w);
  plan::work(plan::UNIT_STREAM, 0, 8.0 * a.experts * a.tokens);
  MRL_LAUNCH(k_experts_choose, dim3(1), dim3(CHOOSE_THREADS), 8 * a.tokens * a.top_k, stream, a, w);
  plan::work(plan::UNIT_STREAM, 0, weight * 2 / 3);
  MRL_LAUNCH(k_experts_up<F8>, dim3(w.slots, (a.inter + 15) / 16), dim3(UP_WAVES * 64), 0, stream, a, w);
  plan::work(plan::UNIT_STREAM, 0, weight / 3);
  MRL_LAUNCH(k_experts_down<F8>, dim3((a.hidden + 15) / 16, (a.tokens + DOWN_TOKENS - 1) / DOWN_TOKENS), dim3(DOWN_WAVES * 64), 0, stream, a, w);
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
