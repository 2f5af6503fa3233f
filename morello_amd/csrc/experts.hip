// A layer of experts for a few tokens:
//     p = softmax(router x),  the top_k largest p_e chosen,  out = sum of share_e down_e (silu(gate_e x) * up_e x)  over a token's chosen e.
//
// What bounds it is reading the wanted experts' weights, once each.  They go from memory into registers in the order in which the matrix
// instructions take them: 16 rows of weights against up to 16 of the expert's tokens, 128 bytes of each row at a time, a lane 32 of them.
// Each of the steps needs all of the one before, a launch each: logits; choice (with few tokens and experts every workgroup of the next launch makes it for itself);
// gate and up to h, 16 rows of one expert at a time; down, a workgroup to some rows of all experts, so that a token's sum over
// its experts is formed in one place and in one order (several workgroups to fewer rows than there are compute units for, and a launch that adds up what they have).  us: 16 tokens, 2 of 8 experts of 4096 x 14336 in bf16 475 to 492 (2.8 GB, 5.7 to 5.9 TB/s: up 314, down 157); 32 tokens, 8 of 128 of 2048 x 768 in e4m3 110 to 115 (528 MB, 4.6 to 4.8 TB/s:
// logits and choice 5 each, up 62, down 40); 1 token, 8 of 64 of 2048 x 1024 in bf16 27 (101 MB: 3, 15, 9; each launch begins with 3 to 4 of reading what the one before left).  A choice is known by its number i = token * top_k + j; no lists go through memory but the chosen experts.
#include <algorithm>

#include "blocks_device.h"
#include "paged.h"

namespace mrl {
namespace {
using namespace blocks;

// What the launches of a call leave each other in the workspace.
struct Places {
  double *logits;       // [tokens][experts]
  int32_t *chosen;      // [tokens][top_k]
  float *shares;        // [tokens][top_k]
  uint16_t *h;          // [tokens * top_k][2][h_s]: rounded to bf16, and what that left, rounded
  uint32_t h_s;
  uint32_t down_shares; // workgroups that share some rows of down; of more than one, what each has
  float *sums;          // [down_shares][tokens][hidden_s]
  uint32_t hidden_s;
};
// What is between the products is in two bf16 numbers, sixteen bits of it, so that a result is rounded once, whatever other tokens there are: in one number results are off by 1.4 times as much (rms 0.0024 for 0.0017).  (us of the layer, in
// one and in two, each in the forms that are fastest: 32 tokens through 128 experts of 2048 x 768 in bf16 193 and 197, in e4m3 110 and 114, 16 through 8 of 4096 x 14336 476 and 483, in e4m3 250 and 265, 100 tokens, 8 of 64 of 2048 x 768 150 and 149,
// in e4m3 101 and 106, 128, 4 of 16 of 4096 x 1024 in e4m3 95 and 110: beside the weights every workgroup reads all tokens' h, which is twice as much.)

// Many tokens of each expert, and more than a little of all, go through gate and up in parts of sixteen, others in parts of eight.
bool few_of_each(const ExpertsArgs &a) { return a.tokens <= 8 || a.tokens * a.top_k < 6 * a.experts || uint64_t(a.tokens) * a.top_k * a.inter <= 1u << 13; }
// Through down in parts of four, whose two numbers each leave a matrix instruction room for a pair of runs (PAIRED), or of sixteen.  (us of the layer, 4 and 16: 32 tokens, 8 of 128 experts of 2048 x 768 in bf16 197 and 200, 20 of 64 117 and 119, 1 of 64 of
// 2048 x 1024 29 and 31; 16, 2 of 8 of 4096 x 14336 515 and 483, 48, 8 of 128 of 2048 x 768 in e4m3 133 and 127, 40, 4 of 60 of 1280 x 512 in bf16 66 and 62.)
uint32_t parts_of_down(const ExpertsArgs &a) { return a.tokens <= 4 || a.tokens * a.top_k * 2 <= 5 * a.experts ? 4 : 16; }

// Rows of down to a workgroup at a time.  In parts of four eight where sixteen would leave half of the compute units without any, and in bf16 where these leave the unit with the most of them fewer.  In parts of sixteen sixteen, several workgroups to the
// same rows where units would have none: that halves what all of them read of h.  (us of the layer, 8 and 16: 64 tokens, 8 of 64 experts of 2048 x 768 in bf16 153 and 134, in e4m3 100 and 89, 128, 2 of 8 of 2048 x 1024 61 and 57, 100, 6 of 64 of 640 x 192 in e4m3 47 and 39; in parts of
// four 16, 8 of 128 of 2048 x 768 in bf16 145 and 150.)
uint32_t rows_of_down(const ExpertsArgs &a) {
  if (parts_of_down(a) == 16) return 16;
  auto most_rows = [&](uint32_t h) { return ((a.hidden + h - 1) / h + g_compute_units - 1) / g_compute_units * h; };
  return (a.weight_dtype == MRL_BF16 ? most_rows(8) < most_rows(16) : a.hidden <= 8 * g_compute_units) ? 8 : 16;
}
uint32_t tokens_of_down(const ExpertsArgs &a);   // that a workgroup has sums for
// Workgroups that share some rows of down: as many as find a compute unit, with 50 steps of 2 KiB and more to each.  (us of the layer, one and as many: 94 tokens, 2 of 8 experts of 384 x 11652 in bf16 214 and 103, 1 token,
// 8 of 64 of 384 x 9600 in e4m3 50 and 37, 32 tokens, 8 of 128 of 1024 x 768 in e4m3 75 and 71; with 96 steps and with 48, 128 tokens, 4 of 16 of 512 x 512 in bf16 37 and 31, 100, 6 of 64 of 640 x 192 in e4m3 44.6 and 39.4; with less, 4 tokens, 4 of 64
// of 1024 x 512 in bf16, 23.4 and 24.5.)
uint32_t shares_of_down(const ExpertsArgs &a) {
  const uint32_t height = rows_of_down(a), here = tokens_of_down(a), groups = (a.hidden + height - 1) / height * ((a.tokens + here - 1) / here), choices = a.tokens * a.top_k;
  const uint32_t parts = std::max(std::min(a.experts, choices), choices / parts_of_down(a));   // about
  const uint64_t steps = uint64_t(parts) * ((uint64_t(a.inter) * (a.weight_dtype == MRL_BF16 ? 2 : 1) * height + 2047) / 2048);
  return uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(g_compute_units / groups, steps / 50)));
}
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
  w.down_shares = shares_of_down(a), w.hidden_s = (a.hidden + 3) / 4 * 4;
  if (w.down_shares > 1) w.sums = (float *)take(sizeof(float) * w.down_shares * a.tokens * w.hidden_s);
  w.h = (uint16_t *)take(4 * choices * w.h_s);
  if (to) *to = w;
  return at;
}

__device__ inline uint32_t live_rows(const ExpertsArgs &p) { return p.rows ? uint32_t(min(max(*p.rows, 0), int32_t(p.tokens))) : p.tokens; }

// Over the lanes of a wave, in the last one (the same order whatever the kernel).
__device__ inline double sum_over_wave(double x) {
  return paged::over_lanes_up_to(x, [](double y, auto ctrl, auto rows) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, y);
    const uint32_t lo = uint32_t(paged::moved<ctrl(), rows()>(int32_t(uint32_t(bits)), 0)), hi = uint32_t(paged::moved<ctrl(), rows()>(int32_t(uint32_t(bits >> 32)), 0));
    return y + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
  });
}
__device__ inline float sum_over_wave(float x) {
  return paged::over_lanes_up_to(x, [](float y, auto ctrl, auto rows) { return y + __int_as_float(paged::moved<ctrl(), rows()>(__float_as_int(y), 0)); });
}

__device__ inline float lo_f32(int x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float hi_f32(int x) { return __uint_as_float(uint32_t(x) & 0xffff0000u); }

// ---- Logits: a workgroup to an expert and TOKENS tokens, in 64 bits, products too (of two bf16 numbers they have sixteen bits, but twice the range of 32-bit numbers), so that which experts are chosen
// does not hang on the order of a sum, and finite inputs have finite logits. ----
constexpr int ROUTER_THREADS = 256;
template <int TOKENS>
__global__ __launch_bounds__(ROUTER_THREADS) void k_experts_logits(ExpertsArgs p, Places w) {
  __shared__ double part[ROUTER_THREADS / 64][TOKENS];
  const uint32_t lane = threadIdx.x & 63, expert = blockIdx.x, t0 = blockIdx.y * TOKENS, rows = live_rows(p);
  if (t0 >= rows) return;
  const uint8_t *const from = (const uint8_t *)(p.router + int64_t(expert) * p.router_s), *x[TOKENS];
#pragma unroll
  for (int t = 0; t < TOKENS; t++) x[t] = (const uint8_t *)(p.x + int64_t(min(t0 + t, rows - 1)) * p.x_s);   // (the last again, behind it)
  double sum[TOKENS] = {};
  auto add = [&](v4i r, const v4i (&y)[TOKENS]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const double lo = lo_f32(r[i]), hi = hi_f32(r[i]);
#pragma unroll
      for (int t = 0; t < TOKENS; t++) sum[t] = __builtin_fma(hi, double(hi_f32(y[t][i])), __builtin_fma(lo, double(lo_f32(y[t][i])), sum[t]));
    }
  };
  uint32_t k = threadIdx.x * 8;
  for (; k + 8 <= p.hidden; k += ROUTER_THREADS * 8) {
    v4i y[TOKENS];
    const v4i r = chunk_at(from + k * 2);
#pragma unroll
    for (int t = 0; t < TOKENS; t++) y[t] = chunk_at(x[t] + k * 2);
    add(r, y);
  }
  if (k < p.hidden) {
    v4i y[TOKENS];
    const int bytes = int(p.hidden - k) * 2;
    const v4i r = chunk_up_to(from + k * 2, bytes, int(k) * 2);
#pragma unroll
    for (int t = 0; t < TOKENS; t++) y[t] = chunk_up_to(x[t] + k * 2, bytes, int(k) * 2);
    add(r, y);
  }
#pragma unroll
  for (int t = 0; t < TOKENS; t++) {
    const double all = sum_over_wave(sum[t]);
    if (lane == 63) part[threadIdx.x / 64][t] = all;
  }
  __syncthreads();
  if (threadIdx.x < TOKENS && t0 + threadIdx.x < rows) {
    double all = 0;
#pragma unroll
    for (int v = 0; v < ROUTER_THREADS / 64; v++) all += part[v][threadIdx.x];
    w.logits[uint64_t(t0 + threadIdx.x) * p.experts + expert] = all;
  }
}

// ---- Choice of experts: a token's j-th is the one that j others are before.  Of some tokens by a workgroup: where there are more threads than logits, a logit's threads share the others. ----
// The share of lane j's expert, of the j-th chosen (logits again: a NaN makes all shares of its token NaN).
__device__ inline float share_of(const ExpertsArgs &p, const double *of_token, double most, int32_t chosen) {
  const uint32_t lane = threadIdx.x & 63;
  float sum = 0.0f, mine = 0.0f;
  if (lane < p.top_k) mine = expf(float(of_token[chosen] - most));
  if (p.renormalise) {
    sum = mine;
  } else {
    for (uint32_t e = lane; e < p.experts; e += 64) sum += expf(float(of_token[e] - most));
  }
  return mine / __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum_over_wave(sum)), 63));
}
struct Choice {          // in LDS, for `tokens` tokens
  double *key;           // [tokens][experts] logits; NaN as the lowest value
  double *most;          // [tokens]
  uint32_t *before;      // [tokens][experts]
  int32_t *expert;       // [tokens][top_k]
  float *share;          // [tokens][top_k]
  __device__ inline Choice(uint8_t *at, const ExpertsArgs &p, uint32_t tokens) {
    key = (double *)at, at += tokens * p.experts * 8;
    most = (double *)at, at += tokens * 8;
    before = (uint32_t *)at, at += tokens * p.experts * 4;
    expert = (int32_t *)at, at += tokens * p.top_k * 4;
    share = (float *)at;
  }
};
// Tokens t0 .. t0 + tokens - 1.  Ends on a barrier.
template <int THREADS>
__device__ inline void choose(const ExpertsArgs &p, const Places &w, uint32_t t0, uint32_t tokens, const FastDiv &by_experts, const Choice &c) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, all = tokens * p.experts;
  const double *const logits = w.logits + uint64_t(t0) * p.experts;
  for (uint32_t i = tid; i < all; i += THREADS) {
    const double x = logits[i];
    c.key[i] = x == x ? x : -__builtin_inf();
    c.before[i] = 0;
  }
  __syncthreads();
  const uint32_t span = all <= 64 ? 64 : 1u << (32 - __clz(all - 1)), shared = span < THREADS ? THREADS / span : 1, each = (p.experts + shared - 1) / shared;   // (span: a power of two)
  for (uint32_t i = tid & (span - 1); i < all; i += THREADS) {   // (span below THREADS: one turn, tid / span below shared)
    const uint32_t t = by_experts.div(i), e = i - t * p.experts, o0 = span < THREADS ? tid / span * each : 0, o1 = min(p.experts, o0 + each);
    const double mine = c.key[i], *const others = c.key + t * p.experts;
    uint32_t before = 0;
#pragma unroll 8
    for (uint32_t o = o0; o < o1; o++) {
      const double k = others[o];
      before += (k > mine || (k == mine && o < e)) ? 1 : 0;
    }
    atomicAdd(&c.before[i], before);
  }
  __syncthreads();
  for (uint32_t i = tid; i < all; i += THREADS) {
    const uint32_t t = by_experts.div(i), before = c.before[i];
    if (before == 0) c.most[t] = c.key[i];
    if (before < p.top_k) c.expert[t * p.top_k + before] = int32_t(i - t * p.experts);
  }
  __syncthreads();
  for (uint32_t t = wave; t < tokens; t += THREADS / 64) {
    const float share = share_of(p, logits + t * p.experts, c.most[t], lane < p.top_k ? c.expert[t * p.top_k + lane] : 0);
    if (lane < p.top_k) c.share[t * p.top_k + lane] = share;
  }
  __syncthreads();
}
template <int THREADS>
__device__ inline void keep(const ExpertsArgs &p, const Places &w, uint32_t t0, uint32_t tokens, const Choice &c) {
  for (uint32_t i = threadIdx.x; i < tokens * p.top_k; i += THREADS) {
    const uint32_t to = t0 * p.top_k + i;
    w.chosen[to] = c.expert[i], w.shares[to] = c.share[i];
    if (p.chosen) p.chosen[to] = c.expert[i];
    if (p.shares) p.shares[to] = c.share[i];
  }
}
// Of a token by a workgroup: each wave ranks sixty-four experts among themselves, and the top_k of each are ranked among all of these.  (A rank among all experts takes four times the comparisons, in 64 bits, of
// which 256 experts' take 4 us.)
constexpr uint32_t MOST_CHUNKS = MOST_EXPERTS / 64;
__global__ __launch_bounds__(MOST_EXPERTS) void k_experts_choose(ExpertsArgs p, Places w) {
  __shared__ double keys[MOST_CHUNKS * MOST_CHOSEN], most;
  __shared__ int32_t experts[MOST_CHUNKS * MOST_CHOSEN], chosen[MOST_CHOSEN];
  const uint32_t token = blockIdx.x, e = threadIdx.x, lane = e & 63, chunk = e / 64, chunks = blockDim.x / 64;
  if (token >= live_rows(p)) return;
  const double *const logits = w.logits + uint64_t(token) * p.experts;
  const double x = e < p.experts ? logits[e] : 0.0, mine = e < p.experts && x == x ? x : -__builtin_inf();   // (those that there are not are behind the lowest of those that there are)
  uint32_t before = 0;
#pragma unroll
  for (int o = 0; o < 64; o++) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, mine);
    const double other = __builtin_bit_cast(double, uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits >> 32)), o))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits)), o)));
    before += (other > mine || (other == mine && uint32_t(o) < lane)) ? 1 : 0;
  }
  if (e < p.experts && before < p.top_k) keys[chunk * MOST_CHOSEN + before] = mine, experts[chunk * MOST_CHOSEN + before] = int32_t(e);
  __syncthreads();
  auto of_chunk = [&](uint32_t c) { return min(p.top_k, min(64u, p.experts - c * 64)); };
  const uint32_t c = e / MOST_CHOSEN, rank = e % MOST_CHOSEN;
  if (c < chunks && rank < of_chunk(c)) {
    const double key = keys[e];
    uint32_t place = rank;
    for (uint32_t d = 0; d < chunks; d++) {
      if (d == c) continue;
      for (uint32_t i = 0, n = of_chunk(d); i < n; i++) place += (keys[d * MOST_CHOSEN + i] > key || (keys[d * MOST_CHOSEN + i] == key && d < c)) ? 1 : 0;
    }
    if (place < p.top_k) chosen[place] = experts[e];
    if (place == 0) most = key;
  }
  __syncthreads();
  if (chunk > 0) return;
  const int32_t its = chosen[min(lane, p.top_k - 1)];
  const float share = share_of(p, logits, most, its);
  if (lane >= p.top_k) return;
  const uint32_t to = token * p.top_k + lane;
  w.chosen[to] = its, w.shares[to] = share;
  if (p.chosen) p.chosen[to] = its;
  if (p.shares) p.shares[to] = share;
}
// Whether every workgroup of the next launch makes all choices for itself: up to 128 comparisons a thread.  (us of the layer in a graph, so and with a launch for them, 2048 x 512, tokens and experts: 1 and 64 16.3
// and 17.3, 1 and 128 20.6 and 21.4, 1 and 160 28.5 and 28.3, 1 and 512 49.8 and 38.1, 4 and 32 22.0 and 23.4, 4 and 64 24.1 and 23.8, 8 and 32 27.1 and 27.7, 8 and 128 84.9 and 74.8, 16 and 16 24.0 and 24.2,
// 16 and 32 48.5 and 47.6, 32 and 8 20.5 and 20.7, 32 and 16 26.9 and 24.7.  Outside of graphs a launch is some 4 more.)
constexpr uint32_t MOST_FUSED_TOKENS = 32, MOST_FUSED = 256;   // (logits, and so choices)
bool fused_choice(const ExpertsArgs &a) { return a.tokens <= MOST_FUSED_TOKENS && a.tokens * a.experts <= MOST_FUSED && a.tokens * a.experts * a.experts <= 1u << 15; }

// ---- Products with experts' weights: 16 rows of each of N matrices against the x of a part's tokens, a step of 128 bytes of the rows at a time.  Loads take a row's 128 bytes with eight
// lanes, x's with eight or sixteen, and LDS brings both into the order in which the matrix instructions want them: what bounds such loops else is the rate at which a compute
// unit's address unit takes cache lines, of which a load of 16 bytes of sixteen rows next to each other has four times as many. ----
// ROOM: tokens that a part may have, 8 or 16, or where a token has two numbers for each twice what it may have, 8 or 32: "tokens" below are then a token's first numbers and, next to them, its second.  More than sixteen are
// multiplied sixteen after sixteen by the same rows in registers.  HOW a step fills an instruction: FULL as above; HALF: with eight rows, and nothing for the others; PAIRED, of a ROOM of eight: eight rows and tokens, 256 bytes of the
// rows, whose second 128 go where rows and tokens 8 to 15 would be: the instruction's sums of rows 0 to 7 with tokens 0 to 7, and of 8 to 15 with 8 to 15, are what is wanted.
enum How { FULL = 0, HALF = 1, PAIRED = 2 };
template <bool F8, int ROOM, int HOW>
struct Shape {
  static constexpr int PAIR = HOW == PAIRED ? 2 : 1, SIZE = F8 ? 1 : 2;                 // runs of 128 bytes of a row in a step; bytes of an element
  static constexpr int STEP = (F8 ? 128 : 64) * PAIR, BYTES = 128 * PAIR;               // of a row in a step: elements, bytes
  static constexpr int LANES = BYTES / 16, LOADS = HOW == HALF ? 1 : 2;                 // of a row in a load; loads for all rows
  static constexpr int X_BYTES = STEP * 2, X_CHUNKS = X_BYTES / 16;                     // of a token's x
  static constexpr int X_LOADS = ROOM * X_BYTES / 1024, X_TOKENS = 64 / X_CHUNKS;       // for all tokens; tokens of a load
  static constexpr int GROUPS = ROOM > 16 ? ROOM / 16 : 1, GROUP_LOADS = X_LOADS / GROUPS;  // sixteens that the same rows are multiplied by, one after the other
  static constexpr int IN_LDS = ROOM / GROUPS * PAIR, ROW_BYTES = X_BYTES / PAIR;       // tokens as the instruction has them, and of one of these
  static constexpr int BOUNCE = IN_LDS * ROW_BYTES;
  static_assert(HOW != PAIRED || ROOM == 8, "");
};
constexpr int TILE_BYTES = 16 * 128;   // of LDS of a wave for each matrix
template <bool F8, int ROOM, int N, int HOW>
struct Rows {
  typedef Shape<F8, ROOM, HOW> S;
  const uint8_t *row[N][S::LOADS];   // of the lane: sixteen bytes of step 0 of row lane / LANES, and of that row + 64 / LANES (of the last row, where there is none: its sums are not looked at)
  const float *scale;             // of step 0: the first matrix's for the first half of the lanes, the last's for the others (a tile's rows are of one block of 128); PAIRED: all lanes the one's
  const uint16_t *x[S::X_LOADS];  // of the lane: eight elements of step 0 of token lane / X_CHUNKS, and of those X_TOKENS behind (of the last, where there is none)
  int x_loads;                    // that the part has tokens for
  __device__ inline void matrix(int n, const Stack &s, uint32_t expert, uint32_t row0, uint32_t height) {   // height: rows that there are from row0 on, up to sixteen
    const uint32_t lane = threadIdx.x & 63;
    const uint8_t *const tile = s.w + (int64_t(expert) * s.w_e + int64_t(row0) * s.w_s) * S::SIZE + lane % S::LANES * 16;
#pragma unroll
    for (int i = 0; i < S::LOADS; i++) row[n][i] = tile + int64_t(min(lane / S::LANES + i * (64 / S::LANES), height - 1)) * (s.w_s * S::SIZE);
    if (F8 && (n == 0 || lane >= 32)) scale = s.scales + int64_t(expert) * s.scales_e + int64_t(row0 / BLOCK) * s.scales_s;
  }
  template <class F>
  __device__ inline void tokens(uint32_t count, F first_of) {   // first_of(i): the i-th token's x
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < S::X_LOADS; i++) x[i] = first_of(min(lane / S::X_CHUNKS + i * S::X_TOKENS, count - 1)) + lane % S::X_CHUNKS * 8;
    x_loads = int(count + S::X_TOKENS - 1) / S::X_TOKENS;
  }
};
// Where rows end.  INSIDE a step: its chunks that the end cuts, or that lie behind it, come from the row's last sixteen bytes and are put right before they are used, so that all steps have
// the same loads, without branches; SHORT: rows of weights or of x below sixteen bytes, byte by byte.
enum Tail { WHOLE = 0, INSIDE = 1, SHORT = 2 };
// What a lane has of one step.
template <bool F8, int ROOM, int N, int TAIL, int HOW>
struct Step {
  typedef Shape<F8, ROOM, HOW> S;
  v4i q[N][S::LOADS], y[S::X_LOADS];
  float scale;
  int x_loads;
  int left, x_left;   // INSIDE: bytes of a row from the lane's chunk on
  // k: elements of a row.
  __device__ inline void fetch(const Rows<F8, ROOM, N, HOW> &of, uint32_t s, int k) {
    const int at = int(s) * S::BYTES, x_at = int(s) * S::X_BYTES;   // bytes
    x_loads = of.x_loads;
    // (PAIRED: the first half of the lanes has the sums with the step's first block, the others those with its second; the row's last block again, where that is behind it)
    if constexpr (F8) scale = of.scale[HOW == PAIRED ? min(int(s) * 2 + int(threadIdx.x >> 5 & 1), (k - 1) / int(BLOCK)) : int(s)];
    const int chunk = at + int(threadIdx.x) % S::LANES * 16, x_chunk = x_at + int(threadIdx.x) % S::X_CHUNKS * 16;   // the lane's
    if constexpr (TAIL != SHORT) {
      int back = at, x_back = x_at;
      if constexpr (TAIL == INSIDE) {
        left = k * S::SIZE - chunk, x_left = k * 2 - x_chunk;
        back += min(left - 16, 0), x_back += min(x_left - 16, 0);
      }
#pragma unroll
      for (int i = 0; i < S::LOADS; i++)
#pragma unroll
        for (int n = 0; n < N; n++) q[n][i] = chunk_at(of.row[n][i] + back);
#pragma unroll
      for (int i = 0; i < S::X_LOADS; i++)
        if (i < x_loads) y[i] = chunk_at((const uint8_t *)of.x[i] + x_back);
    } else {
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) q[n][i] = chunk_up_to(of.row[n][i] + at, k * S::SIZE - chunk, chunk);
#pragma unroll
      for (int i = 0; i < S::X_LOADS; i++)
        if (i < x_loads) y[i] = chunk_up_to((const uint8_t *)of.x[i] + x_at, k * 2 - x_chunk, x_chunk);
    }
  }
  // bounce: LDS of this wave's, N tiles and x of IN_LDS tokens.  Chunk c of a row of 128 bytes at c ^ (row / 2 % 8), of 256 bytes at c ^ row: sixteen lanes with a
  // chunk of sixteen rows each reach every bank once.
  __device__ inline void multiply(v4f (&acc)[N][S::GROUPS], uint8_t *bounce) {
    const uint32_t lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    if (TAIL == INSIDE && __any(left < 16 || x_left < 16)) {
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) q[n][i] = last_of_row(q[n][i], left);
#pragma unroll
      for (int i = 0; i < S::X_LOADS; i++) y[i] = last_of_row(y[i], x_left);
      if (F8 && HOW == PAIRED && left + int(lane % S::LANES) * 16 <= int(lane / 32) * 128) scale = 0;   // (no such block; the last one's may be infinite)
    }
    uint8_t *const of_x = bounce + N * TILE_BYTES;
    auto put_x = [&](int g) {
#pragma unroll
      for (int i = 0; i < S::GROUP_LOADS; i++)
        if (g * S::GROUP_LOADS + i < x_loads) {
          constexpr uint32_t CHUNKS = S::ROW_BYTES / 16;
          const uint32_t token = lane / S::X_CHUNKS + i * S::X_TOKENS + lane % S::X_CHUNKS / CHUNKS * 8;
          *(v4i *)(of_x + token * S::ROW_BYTES + (lane % CHUNKS ^ (F8 ? token : token / 2 % 8)) * 16) = y[g * S::GROUP_LOADS + i];
        }
    };
    lanes_meet();   // (over what the step before was multiplied from)
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < S::LOADS; i++) {
        const uint32_t row = lane / S::LANES + i * (64 / S::LANES) + lane % S::LANES / 8 * 8;
        *(v4i *)(bounce + n * TILE_BYTES + row * 128 + (lane % 8 ^ (row / 2 & 7)) * 16) = q[n][i];
      }
    put_x(0);
    lanes_meet();
    const uint32_t mine = li & (S::IN_LDS - 1);
    const uint8_t *const my_x = of_x + mine * S::ROW_BYTES;
    float scales[2] = {0, 0};
    if constexpr (F8 && HOW == PAIRED) scales[0] = scale;
    else if constexpr (F8) scales[0] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(scale))), scales[1] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scale), 32));
    auto weights = [&](int n, int i) { return *(const v4i *)(bounce + n * TILE_BYTES + li * 128 + ((i * 4 + lg) ^ (li >> 1)) * 16); };
    auto next_group = [&](int g) {   // (of a part that has tokens for it)
      lanes_meet();
      put_x(g);
      lanes_meet();
    };
    if constexpr (F8) {
      v4i b[S::GROUPS > 1 ? 2 : 1][2];   // (a group's alone: as they are wanted)
#pragma unroll
      for (int g = 0; g < S::GROUPS; g++) {
        if (g > 0) {
          if (g * S::GROUP_LOADS >= x_loads) break;
          next_group(g);
        }
        v4i u[2][2];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) u[i][j] = *(const v4i *)(my_x + ((i * 8 + lg * 2 + j) ^ mine) * 16);
#pragma unroll
        for (int n = 0; n < N; n++) {
          v4f part = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 2; i++) {
            v4i(&wide)[2] = b[S::GROUPS > 1 ? i : 0];
            if (g == 0) {
              const v4i w = weights(n, i);
#pragma unroll
              for (int j = 0; j < 2; j++) {
                int x[4];
                widen4(w[2 * j], x[0], x[1]);
                widen4(w[2 * j + 1], x[2], x[3]);
                wide[j] = v4i{x[0], x[1], x[2], x[3]};
              }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) part = mma_bf16(wide[j], u[i][j], part);
          }
          acc[n][g] += part * scales[n];
        }
      }
    } else {
      v4i b[2];
#pragma unroll
      for (int g = 0; g < S::GROUPS; g++) {
        if (g > 0) {
          if (g * S::GROUP_LOADS >= x_loads) break;
          next_group(g);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const v4i u = *(const v4i *)(my_x + ((i * 4 + lg) ^ (mine >> 1)) * 16);
          if constexpr (S::GROUPS > 1) {
            if (g == 0) b[i] = weights(0, i);
            acc[0][g] = mma_bf16(b[i], u, acc[0][g]);
          } else {
#pragma unroll
            for (int n = 0; n < N; n++) acc[n][g] = mma_bf16(weights(n, i), u, acc[n][g]);
          }
        }
      }
    }
  }
};

// ---- A workgroup's choices by experts: expert after expert, in parts of up to `room` (8 or 16) ----
struct Part { uint16_t expert, first, count, unused; };
constexpr uint32_t most_parts(uint32_t experts, uint32_t choices, uint32_t room) { return (choices < experts ? choices : experts) + choices / room; }
// What is in LDS, for up to `choices` choices of `experts` experts by tokens of `words` times 32.
struct Lists {
  Part *parts;
  uint16_t *choices;     // expert after expert, a token before the later ones
  uint32_t *wants;       // [experts][words] a bit for each token
  uint16_t *first_of;    // [experts]
  int32_t *totals;       // [2][waves]
  __device__ inline Lists(uint8_t *at, uint32_t experts, uint32_t all, uint32_t words, uint32_t room, uint32_t waves) {
    parts = (Part *)at, at += most_parts(experts, all, room) * sizeof(Part);
    wants = (uint32_t *)at, at += experts * words * 4;
    totals = (int32_t *)at, at += waves * 8;
    choices = (uint16_t *)at, at += all * 2;
    first_of = (uint16_t *)at;
  }
  static size_t bytes(uint32_t experts, uint32_t all, uint32_t words, uint32_t room, uint32_t waves) { return most_parts(experts, all, room) * sizeof(Part) + experts * words * 4 + waves * 8 + all * 2 + experts * 2; }
};
// Returns the number of parts.  `all` choices, of which token i / top_k made the i-th; ends on a barrier.
template <int THREADS>
__device__ inline uint32_t list(const Lists &to, const ExpertsArgs &p, const int32_t *of_choice, uint32_t all, uint32_t words, uint32_t room) {
  constexpr int EACH = MOST_EXPERTS > THREADS ? MOST_EXPERTS / THREADS : 1;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (all <= p.top_k) {   // one token: its experts differ
    if (tid < all) to.parts[tid] = {uint16_t(of_choice[tid]), uint16_t(tid), 1, 0}, to.choices[tid] = uint16_t(tid);
    __syncthreads();
    return all;
  }
  for (uint32_t i = tid; i < p.experts * words; i += THREADS) to.wants[i] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < all; i += THREADS) {
    const uint32_t t = i / p.top_k;
    atomicOr(&to.wants[uint32_t(of_choice[i]) * words + t / 32], 1u << (t % 32));
  }
  __syncthreads();
  // Choices (below 2^14), and parts of them, before each expert, in one number (a thread has EACH neighbours).
  uint32_t count[EACH], mine = 0;
#pragma unroll
  for (int k = 0; k < EACH; k++) {
    const uint32_t e = tid * EACH + k;
    count[k] = 0;
    if (e < p.experts)
      for (uint32_t j = 0; j < words; j++) count[k] += __popc(to.wants[e * words + j]);
    mine += count[k] << 16 | (count[k] + room - 1) / room;
  }
  uint32_t before = paged::over_lanes_up_to(mine, [](uint32_t x, auto ctrl, auto rows) { return x + uint32_t(paged::moved<ctrl(), rows()>(int32_t(x), 0)); });
  if (lane == 63) to.totals[wave] = int32_t(before);
  __syncthreads();
  before -= mine;
  uint32_t parts = 0;
#pragma unroll
  for (uint32_t v = 0; v < THREADS / 64; v++) {
    const uint32_t x = uint32_t(to.totals[v]);
    if (v < wave) before += x;
    parts += x & 0xffff;
  }
#pragma unroll
  for (int k = 0; k < EACH; k++) {
    const uint32_t e = tid * EACH + k;
    if (e < p.experts) {
      to.first_of[e] = uint16_t(before >> 16);
      for (uint32_t c = 0; c < count[k]; c += room) to.parts[before++ & 0xffff] = {uint16_t(e), uint16_t(to.first_of[e] + c), uint16_t(min(room, count[k] - c)), 0};
    }
    before += count[k] << 16;
  }
  __syncthreads();
  for (uint32_t i = tid; i < all; i += THREADS) {
    const uint32_t t = i / p.top_k, e = uint32_t(of_choice[i]);
    uint32_t at = to.first_of[e];
    for (uint32_t j = 0; j < t / 32; j++) at += __popc(to.wants[e * words + j]);
    to.choices[at + __popc(to.wants[e * words + t / 32] & ((1u << (t % 32)) - 1))] = uint16_t(i);
  }
  __syncthreads();
  return parts;
}

// ---- Gate and up.  All parts' tiles of 16 rows lie on a line, of which workgroup b has the tiles b, b + gridDim.x, ..: what is under way at a time lies close together (equal runs of the line for each
// took 10 % longer over 1.9 GB).  The waves share a tile's steps; their loads run AHEAD steps in front, from one tile into the next, and the
// waves' sums meet behind each.  FUSED: from logits, the choices made here. ----
template <bool F8, int ROOM, bool FUSED, int TAIL, int UP_WAVES>
__global__ __launch_bounds__(UP_WAVES * 64, 2) void k_experts_up(ExpertsArgs p, Places w, uint32_t words, FastDiv by_tiles, FastDiv by_experts) {
  constexpr int AHEAD = 3;
  typedef Shape<F8, ROOM, FULL> S;
  extern __shared__ __attribute__((aligned(16))) uint8_t dynamic[];
  __shared__ v4f sums[2][UP_WAVES][2][64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t rows = live_rows(p), all = rows * p.top_k;
  constexpr uint32_t BOUNCE = 2 * TILE_BYTES + S::BOUNCE;
  uint8_t *const bounce = dynamic + wave * BOUNCE;
  const Lists lists(dynamic + UP_WAVES * BOUNCE, p.experts, p.tokens * p.top_k, words, ROOM, UP_WAVES);
  const int32_t *chosen = w.chosen;
  if constexpr (FUSED) {
    const Choice c(dynamic, p, p.tokens);   // (where the waves' tiles will be)
    choose<UP_WAVES * 64>(p, w, 0, rows, by_experts, c);
    if (blockIdx.x == 0) keep<UP_WAVES * 64>(p, w, 0, rows, c);
    chosen = c.expert;
  }
  const uint32_t tiles = (p.inter + 15) / 16, line = tiles * __builtin_amdgcn_readfirstlane(list<UP_WAVES * 64>(lists, p, chosen, all, words, ROOM));
  const uint32_t steps = (p.hidden + S::STEP - 1) / S::STEP, s0 = steps * wave / UP_WAVES, n = steps * (wave + 1) / UP_WAVES - s0;   // this wave's steps of each tile
  Rows<F8, ROOM, 2, FULL> of;
  Step<F8, ROOM, 2, TAIL, FULL> t[AHEAD] = {};
  auto go_to = [&](uint32_t tile) {
    const uint32_t part = by_tiles.div(tile), row0 = (tile - part * tiles) * 16, height = min(16u, p.inter - row0);
    const Part q = lists.parts[part];
    const uint32_t expert = __builtin_amdgcn_readfirstlane(q.expert);
    of.matrix(0, p.gate, expert, row0, height), of.matrix(1, p.up, expert, row0, height);
    of.tokens(__builtin_amdgcn_readfirstlane(q.count), [&](uint32_t i) { return p.x + int64_t(lists.choices[q.first + i] / p.top_k) * p.x_s; });
  };
  if (blockIdx.x < line) {
    go_to(blockIdx.x);
#pragma unroll
    for (int a = 0; a < AHEAD; a++)
      if (uint32_t(a) < n) t[a].fetch(of, s0 + a, int(p.hidden));
  }
  uint32_t turn = 0;
  for (uint32_t tile = blockIdx.x; tile < line; tile += gridDim.x, turn ^= 1) {
    v4f acc[2][1] = {};
    for (uint32_t at = 0; at < n; at += AHEAD) {
      const bool last = at + AHEAD >= n, more = tile + gridDim.x < line;
      if (last && more) go_to(tile + gridDim.x);
#pragma unroll
      for (int a = 0; a < AHEAD; a++) {
        if (at + a < n) t[a].multiply(acc, bounce);
        const uint32_t next = last ? uint32_t(a) : at + a + AHEAD;
        if (next < n && (!last || more)) t[a].fetch(of, s0 + next, int(p.hidden));
      }
    }
    v4f(&here)[UP_WAVES][2][64] = sums[turn];
    here[wave][0][lane] = acc[0][0], here[wave][1][lane] = acc[1][0];
    __syncthreads();   // (the tile before the last has been read: its readers are here)
    if (wave == tile / gridDim.x % UP_WAVES) {
      v4f g = here[0][0][lane], u = here[0][1][lane], h;
#pragma unroll
      for (uint32_t v = 1; v < UP_WAVES; v++) g += here[v][0][lane], u += here[v][1][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) h[i] = g[i] / (1.0f + expf(-g[i])) * u[i];
      const uint32_t part = by_tiles.div(tile), row = (tile - part * tiles) * 16 + lg * 4;
      const Part q = lists.parts[part];
      if (li < q.count && row < p.inter) {
        uint16_t *const to = w.h + uint64_t(lists.choices[q.first + li]) * 2 * w.h_s + row;
        store4(to, h, int(p.inter - row));
        v4f rest;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float r = h[i] - float((__bf16)h[i]);
          rest[i] = fabsf(r) < __builtin_inff() ? r : 0.0f;
        }
        store4(to + w.h_s, rest, int(p.inter - row));
      }
    }
  }
}

// ---- Down: a workgroup to 16 rows, or 8, and behind them those gridDim.x further; blockIdx.y: tokens_here tokens; blockIdx.z: which of those that share the rows.  All parts' steps in a line, cut into pieces of up to
// 1024 bytes of a part's rows, of which a wave has every eighth: a workgroup's waves go through the same rows together, and each asks for the next rows' weights while it multiplies the last of these.  (Eight rows PAIRED
// against HALF, us of the layer: 32 tokens through 128 experts of 2048 x 768 in bf16 199 and 221, in e4m3 114 and 120; 8 of 1024 through 64 40.6 and 42.5.  A workgroup to each rows, 1 token, 2 of 8 of 4992 x 768 in e4m3 23.4
// for 21.0; sixteen waves, with h in one number, 32 tokens as above 194 for 196 in bf16, 110 for 106 in e4m3.) ----
constexpr int DOWN_WAVES = 8;
template <bool F8, int MOST, int TAIL, int HOW>
__global__ __launch_bounds__(DOWN_WAVES * 64) void k_experts_down(ExpertsArgs p, Places w, uint32_t tokens_here, uint32_t words) {
  constexpr int ROOM = MOST * 2, WAVES = DOWN_WAVES, THREADS = WAVES * 64, AHEAD = F8 && ROOM == 32 ? 3 : HOW == PAIRED || ROOM == 32 ? 4 : 6;   // (what registers take: PAIRED has twice a step's bytes, ROOM 32 four times those of x)
  constexpr uint32_t HEIGHT = HOW == FULL ? 16 : 8;
  typedef Shape<F8, ROOM, HOW> S;
  extern __shared__ __attribute__((aligned(16))) uint8_t dynamic[];
  v4f *const sums = (v4f *)dynamic;                            // [WAVES][tokens_here][4]
  float *const shares = (float *)(sums + WAVES * tokens_here * 4);   // [tokens_here * top_k]
  const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr uint32_t BOUNCE = TILE_BYTES + S::BOUNCE;
  uint8_t *const bounces = (uint8_t *)(shares + (tokens_here * p.top_k + 3) / 4 * 4), *const bounce = bounces + wave * BOUNCE;
  const Lists lists(bounces + WAVES * BOUNCE, p.experts, tokens_here * p.top_k, words, MOST, WAVES);
  const uint32_t t0 = blockIdx.y * tokens_here, rows = live_rows(p), groups = (p.hidden + HEIGHT - 1) / HEIGHT;
  if (t0 >= rows) return;
  const uint32_t here = min(tokens_here, rows - t0);
  v4f *const mine = sums + wave * tokens_here * 4;
  for (uint32_t i = lane; i < here * 4; i += 64) mine[i] = v4f{0, 0, 0, 0};
  for (uint32_t i = tid; i < here * p.top_k; i += THREADS) shares[i] = w.shares[t0 * p.top_k + i];
  const uint32_t parts = __builtin_amdgcn_readfirstlane(list<THREADS>(lists, p, w.chosen + t0 * p.top_k, here * p.top_k, words, MOST));
  // Pieces of eight steps, or fewer where a seventh of the waves' last turn would be idle.
  const uint32_t steps = (p.inter + S::STEP - 1) / S::STEP;
  const uint32_t all_waves = WAVES * gridDim.z, first = wave + blockIdx.z * WAVES;
  uint32_t size = 8 / S::PAIR, of_part, pieces;
  for (;; size /= 2) {
    of_part = (steps + size - 1) / size, pieces = parts * of_part;
    if (size == 1 || pieces * 7 >= (pieces + all_waves - 1) / all_waves * all_waves * 6) break;
  }
  // The waves' sums of some rows into one, and on to the next.
  auto finish = [&](uint32_t group) {
    __syncthreads();
    const uint32_t row0 = group * HEIGHT, rows_here = min(HEIGHT, p.hidden - row0);
    for (uint32_t i = tid; i < here * 4; i += THREADS) {
      const uint32_t row = i % 4 * 4;
      if (row >= rows_here) continue;
      v4f sum = sums[i];
#pragma unroll
      for (uint32_t v = 1; v < WAVES; v++) sum += sums[v * tokens_here * 4 + i];
      if (HOW == PAIRED && row < 8) {
#pragma unroll
        for (uint32_t v = 0; v < WAVES; v++) sum += sums[v * tokens_here * 4 + i + 2];
      }
      if (gridDim.z > 1) *(v4f *)(w.sums + (uint64_t(blockIdx.z) * p.tokens + t0 + i / 4) * w.hidden_s + row0 + row) = sum;   // (hidden_s: whole fours)
      else store4(p.out + int64_t(t0 + i / 4) * p.out_s + row0 + row, sum, int(rows_here - row));
    }
    if (group + gridDim.x >= groups) return;
    __syncthreads();
    for (uint32_t i = lane; i < here * 4; i += 64) mine[i] = v4f{0, 0, 0, 0};   // (lanes meet in the next multiply, before any of them adds)
  };
  if (first >= pieces) {   // (of each row the same)
    for (uint32_t group = blockIdx.x; group < groups; group += gridDim.x) finish(group);
    return;
  }
  // The piece to fetch from, and the one to multiply, of which rows.
  uint32_t fetch_group = blockIdx.x, fetch_piece = first, fetch_s = 0, fetch_end = 0, group = blockIdx.x, piece = first, s = 0, end = 0;
  Rows<F8, ROOM, 1, HOW> of;
  Step<F8, ROOM, 1, TAIL, HOW> t[AHEAD] = {};
  auto fetch = [&](Step<F8, ROOM, 1, TAIL, HOW> &to) {
    if (fetch_s == fetch_end) {
      const uint32_t part = fetch_piece / of_part;
      const Part q = lists.parts[part];
      fetch_s = (fetch_piece - part * of_part) * size, fetch_end = min(steps, fetch_s + size);
      of.matrix(0, p.down, __builtin_amdgcn_readfirstlane(q.expert), fetch_group * HEIGHT, min(HEIGHT, p.hidden - fetch_group * HEIGHT));
      of.tokens(__builtin_amdgcn_readfirstlane(q.count) * 2, [&](uint32_t i) { return w.h + (uint64_t(t0 * p.top_k + lists.choices[q.first + i / 2]) * 2 + i % 2) * w.h_s; });
    }
    to.fetch(of, fetch_s, int(p.inter));
    if (++fetch_s == fetch_end && (fetch_piece += all_waves) >= pieces) fetch_piece = first, fetch_group += gridDim.x;
  };
  v4f acc[1][S::GROUPS] = {};
#pragma unroll
  for (int a = 0; a < AHEAD; a++)
    if (fetch_group < groups) fetch(t[a]);
  while (group < groups) {
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      if (group >= groups) break;
      if (s == end) {
        const uint32_t part = piece / of_part;
        s = (piece - part * of_part) * size, end = min(steps, s + size);
      }
      t[a].multiply(acc, bounce);
      if (fetch_group < groups) fetch(t[a]);
      if (++s == end) {
        const Part q = lists.parts[piece / of_part];
#pragma unroll
        for (int g = 0; g < S::GROUPS; g++) {
          const uint32_t column = (HOW == PAIRED ? li - lg / 2 * 8 : li) + g * 16;   // (PAIRED: below 8 where the lane's sums are wanted, or far above)
          v4f both;
#pragma unroll
          for (int e = 0; e < 4; e++) {   // (and the next lane's, but where that is infinity times nothing)
            const float x = acc[0][g][e], rest = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xb1, 0xf, 0xf, true));
            both[e] = fabsf(x) < __builtin_inff() ? x + rest : x;
          }
          if (column % 2 == 0 && column / 2 < q.count) {
            const uint32_t choice = lists.choices[q.first + column / 2];
            sums[(wave * tokens_here + choice / p.top_k) * 4 + lg] += both * shares[choice];
          }
          acc[0][g] = v4f{0, 0, 0, 0};
        }
        if ((piece += all_waves) >= pieces) finish(group), group += gridDim.x, piece = first;
      }
    }
  }
}

// What several workgroups have of the same rows, in their order.
constexpr int JOIN_THREADS = 256;
__global__ __launch_bounds__(JOIN_THREADS) void k_experts_join(ExpertsArgs p, Places w) {
  const uint32_t at = (blockIdx.x * JOIN_THREADS + threadIdx.x) * 4, token = blockIdx.y;
  if (at >= p.hidden || token >= live_rows(p)) return;
  const float *const from = w.sums + uint64_t(token) * w.hidden_s + at;
  v4f sum = *(const v4f *)from;
  for (uint32_t z = 1; z < w.down_shares; z++) sum += *(const v4f *)(from + uint64_t(z) * p.tokens * w.hidden_s);
  store4(p.out + int64_t(token) * p.out_s + at, sum, int(p.hidden - at));
}

template <bool F8, int ROOM, bool FUSED, int TAIL, int UP_WAVES>
hipError_t launch_up_waves(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  // Two workgroups to a compute unit, what their registers allow, or one to a tile.  (us, two with three steps ahead and three with two: 128 tokens through 128 experts of 2048 x 768 in e4m3 155 and
  // 180, 32 tokens 110 and 112, 16 through 8 of 4096 x 14336 254 and 253.)
  const uint32_t tiles = (a.inter + 15) / 16, words = (a.tokens + 31) / 32, choices = a.tokens * a.top_k;
  const uint32_t grid = uint32_t(std::min<uint64_t>(uint64_t(most_parts(a.experts, choices, ROOM)) * tiles, 2 * g_compute_units));
  static_assert(!FUSED || MOST_FUSED * 20 + MOST_FUSED_TOKENS * 8 <= UP_WAVES * (2 * TILE_BYTES + Shape<F8, ROOM, FULL>::BOUNCE), "");
  const size_t lds = UP_WAVES * (2 * TILE_BYTES + Shape<F8, ROOM, FULL>::BOUNCE) + Lists::bytes(a.experts, choices, words, ROOM, UP_WAVES);
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_experts_up<F8, ROOM, FUSED, TAIL, UP_WAVES>), 96 * 1024);
    if (e != hipSuccess) return e;
  }
  MRL_LAUNCH((k_experts_up<F8, ROOM, FUSED, TAIL, UP_WAVES>), dim3(grid), dim3(UP_WAVES * 64), lds, stream, a, w, words, FastDiv(tiles), FastDiv(a.experts));
  return plan::last_error();
}
template <bool F8, int ROOM, bool FUSED, int TAIL>
hipError_t launch_up(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  // Eight waves to a tile where at least half of the compute units have none and its rows are 2 KiB and more.  (us of the layer, four and eight, 1 token: 2 of 8 experts of 4096 x 512 in bf16 18.7 and 16.8, 4 of 64 of
  // 7168 x 512 in e4m3 23.9 and 22.5; 4 of 16 of 4096 x 1024 19.9 and 20.6, of 1024 x 256 12.3 and 12.4.)
  const uint64_t tiles = uint64_t(most_parts(a.experts, a.tokens * a.top_k, ROOM)) * ((a.inter + 15) / 16);
  if constexpr (ROOM == 8 && TAIL != SHORT) {
    if (tiles * 2 <= uint64_t(g_compute_units) && a.hidden * (F8 ? 1 : 2) >= 2048) return launch_up_waves<F8, ROOM, FUSED, TAIL, 8>(a, w, stream);
  }
  return launch_up_waves<F8, ROOM, FUSED, TAIL, 4>(a, w, stream);
}
constexpr size_t MOST_LDS = 160 * 1024;
template <bool F8, int MOST, int HOW>
size_t down_lds(const ExpertsArgs &a, uint32_t here) {
  return size_t(DOWN_WAVES) * here * 64 + size_t(here * a.top_k + 3) / 4 * 16 + DOWN_WAVES * (TILE_BYTES + Shape<F8, MOST * 2, HOW>::BOUNCE) + Lists::bytes(a.experts, here * a.top_k, (here + 31) / 32, MOST, DOWN_WAVES);
}
// Of rows of a single run of 128 bytes there is no pair.  (us of the layer, HALF and PAIRED, in e4m3, 4 tokens, 8 of 64 experts of 2048 x 128 21.1 and 22.9.)
How how_of_down(const ExpertsArgs &a) { return rows_of_down(a) == 16 ? FULL : a.inter * (a.weight_dtype == MRL_BF16 ? 2 : 1) > 128 ? PAIRED : HALF; }
template <bool F8>
size_t down_lds(const ExpertsArgs &a, uint32_t here) {
  const How how = how_of_down(a);
  return how == PAIRED ? down_lds<F8, 4, PAIRED>(a, here) : how == HALF ? down_lds<F8, 4, HALF>(a, here) : parts_of_down(a) == 4 ? down_lds<F8, 4, FULL>(a, here) : down_lds<F8, 16, FULL>(a, here);
}
uint32_t tokens_of_down(const ExpertsArgs &a) {
  uint32_t here = a.tokens;   // all, or as many as LDS has place for
  while ((a.weight_dtype == MRL_BF16 ? down_lds<false>(a, here) : down_lds<true>(a, here)) > MOST_LDS) here -= (here + 31) / 32 > 1 ? here - (here - 1) / 32 * 32 : here / 2;
  return here;
}
template <bool F8, int MOST, int TAIL, int HOW>
hipError_t launch_down(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  constexpr uint32_t HEIGHT = HOW == FULL ? 16 : 8;
  const uint32_t here = tokens_of_down(a);
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_experts_down<F8, MOST, TAIL, HOW>), MOST_LDS);
    if (e != hipSuccess) return e;
  }
  const size_t lds = down_lds<F8, MOST, HOW>(a, here);
  MRL_LAUNCH((k_experts_down<F8, MOST, TAIL, HOW>), dim3(std::min((a.hidden + HEIGHT - 1) / HEIGHT, uint32_t(g_compute_units)), (a.tokens + here - 1) / here, w.down_shares), dim3(DOWN_WAVES * 64), lds, stream, a, w, here, (here + 31) / 32);
  if (w.down_shares > 1) {
    plan::work(plan::UNIT_STREAM, 0, (4.0 * w.down_shares + 2) * a.tokens * a.hidden);
    MRL_LAUNCH(k_experts_join, dim3((a.hidden + JOIN_THREADS * 4 - 1) / (JOIN_THREADS * 4), a.tokens), dim3(JOIN_THREADS), 0, stream, a, w);
  }
  return plan::last_error();
}
// How rows of k elements end.
template <bool F8>
Tail tail_of(uint32_t k, uint32_t step = F8 ? 128 : 64) { return k * (F8 ? 1 : 2) < 16 || k * 2 < 16 ? SHORT : k % step ? INSIDE : WHOLE; }
template <bool F8, int MOST, int HOW>
hipError_t launch_down_how(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  const Tail tail = tail_of<F8>(a.inter, Shape<F8, MOST * 2, HOW>::STEP);
  if constexpr (HOW != PAIRED) {
    if (tail == SHORT) return launch_down<F8, MOST, SHORT, HOW>(a, w, stream);
  }
  return tail == WHOLE ? launch_down<F8, MOST, WHOLE, HOW>(a, w, stream) : launch_down<F8, MOST, INSIDE, HOW>(a, w, stream);
}
template <bool F8, int ROOM, bool FUSED>
hipError_t launch_products(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  const double weight = 3.0 * a.inter * a.hidden * (F8 ? 1 : 2) * std::min(a.experts, a.tokens * a.top_k);
  const Tail up = tail_of<F8>(a.hidden);
  plan::work(plan::UNIT_STREAM, 0, weight * 2 / 3);
  const hipError_t e = up == WHOLE    ? launch_up<F8, ROOM, FUSED, WHOLE>(a, w, stream)
                       : up == INSIDE ? launch_up<F8, ROOM, FUSED, INSIDE>(a, w, stream)
                                      : launch_up<F8, ROOM, FUSED, SHORT>(a, w, stream);
  if (e != hipSuccess) return e;
  plan::work(plan::UNIT_STREAM, 0, weight / 3);
  switch (how_of_down(a)) {
    case PAIRED: return launch_down_how<F8, 4, PAIRED>(a, w, stream);
    case HALF: return launch_down_how<F8, 4, HALF>(a, w, stream);
    default: return parts_of_down(a) == 4 ? launch_down_how<F8, 4, FULL>(a, w, stream) : launch_down_how<F8, 16, FULL>(a, w, stream);
  }
}
template <bool F8>
hipError_t launch(const ExpertsArgs &a, const Places &w, hipStream_t stream) {
  plan::work(plan::UNIT_STREAM, 0, 2.0 * (double(a.experts) + a.tokens) * a.hidden);
  // (a token to a workgroup while these still run side by side: the layer takes 31.5 us so and 32.3 with four for 1 token and 512 experts, 33 and 33 for 16 and 128, 202 and 185 for 200 and 256)
  if (a.experts * a.tokens <= 8 * g_compute_units) MRL_LAUNCH(k_experts_logits<1>, dim3(a.experts, a.tokens), dim3(ROUTER_THREADS), 0, stream, a, w);
  else MRL_LAUNCH(k_experts_logits<4>, dim3(a.experts, (a.tokens + 3) / 4), dim3(ROUTER_THREADS), 0, stream, a, w);
  const bool few = few_of_each(a), fused = few && fused_choice(a);
  if (!fused) {
    plan::work(plan::UNIT_STREAM, 0, 8.0 * a.experts * a.tokens);
    MRL_LAUNCH(k_experts_choose, dim3(a.tokens), dim3((a.experts + 63) / 64 * 64), 0, stream, a, w);
  }
  // Parts of sixteen are what a matrix instruction takes; of eight take less LDS, fewer registers, and less of x where few of an expert's are there.  (us, 16 and 8 for up and down alike, with h in one number, choices an expert: 2 113.6 and 111.6,
  // 4 33.3 and 31.5, 6 149.2 and 150.5, 137 and 145, 8 156 and 172, 91 and 101.)
  return !few ? launch_products<F8, 16, false>(a, w, stream) : fused ? launch_products<F8, 8, true>(a, w, stream) : launch_products<F8, 8, false>(a, w, stream);
}

}  // namespace

size_t experts_workspace_bytes(const ExpertsArgs &a) { return places(a, nullptr); }

hipError_t launch_experts(const ExpertsArgs &a, hipStream_t stream) {
  Places w;
  places(a, &w);
  return a.weight_dtype == MRL_BF16 ? launch<false>(a, w, stream) : launch<true>(a, w, stream);
}

}  // namespace mrl
