// The product of blocks (matmul_blocks.hip) on tiles of 128 x 128 to 64 x 64, for rows of whole 16-byte chunks: what leaves compute units idle on tiles of 256 x 256,
// and results in f32.
//
// Four waves, 2 x 2, or GROUPS of four, each of which has every GROUPS-th block of K: one wave on a SIMD takes some 800 cycles from the barrier over reads from LDS, products and
// sums to the next, of which the products are 128 (64 x 64) to 512, and groups fill them.  A block of all the tile's rows, and a's scales, go straight from memory into a
// ring of DEPTH blocks in LDS that is the group's.  (1024 x 2048 x 4096 18.4 us, 0.93 PFLOP/s.)  Results in f32 pay for bf16: four matrix instructions of 16 cycles for one of 32, and sixteen conversions of each
// sixteen rows for each wave that multiplies them: 1024 x 4096 x 4480 43 us, 0.87 PFLOP/s.
#include "matmul_blocks.h"

namespace mrl {
namespace {
using namespace blocks;

template <int BM, int BN, int GROUPS, int DEPTH, bool SHARED, class OUT>
__global__ __launch_bounds__(GROUPS * 256) void k_product_tile(ProductArgs p, uint32_t tiles_m, uint32_t tiles_n, uint32_t high) {
  constexpr int MT = BM / 32, NT = BN / 32, A_LOADS = BM / 32, B_LOADS = BN / 32, LOADS = A_LOADS + B_LOADS + 1;   // a wave's, a step
  constexpr int SLOT = (BM + BN) * int(BLOCK) + 4 * 256;   // (a's scales: 256 bytes from each wave, BM of them what is wanted)
  constexpr int SCALES = BLOCK % BN == 0 ? 1 : NT;                 // of b, for a wave's sums: one, or one for each sixteen of b's rows
  static_assert((DEPTH - 2) * LOADS < 64 && GROUPS * DEPTH * SLOT <= 160 * 1024 && (GROUPS - 1) * BM * BN * 4 <= GROUPS * DEPTH * SLOT, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int my_group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  // An XCD's tiles in groups of `high` by all of n.
  const uint32_t at = xcd_run(blockIdx.x, gridDim.x), group = at / (high * tiles_n), here = min(high, tiles_m - group * high), in_group = at - group * high * tiles_n;
  const uint32_t tile_n = in_group / here, tile_m = group * high + in_group - tile_n * here;
  const uint32_t m0 = tile_m * BM, n0 = tile_n * BN, wm = wave / 2 * (BM / 2), wn = wave % 2 * (BN / 2);
  const int steps = int((p.k + BLOCK - 1) / BLOCK), all_groups = SHARED ? GROUPS * int(gridDim.y) : GROUPS;
  const int first = SHARED ? int(blockIdx.y) * GROUPS + my_group : my_group, turns = (steps + all_groups - 1) / all_groups, mine = steps > first ? (steps - first + all_groups - 1) / all_groups : 0;   // mine: turns or one less
  // This wave's loads of a step: every fourth eight rows of a and of b, from the wave-th on.  Chunk c of a row at c ^ (row / 2 % 8) of its 128 bytes.
  const uint32_t row0 = wave * 8 + (lane >> 3), chunk = (lane & 7) ^ (row0 >> 1 & 7), a_s = uint32_t(p.a_s), b_s = uint32_t(p.b_s);
  const uint32_t a_off = row0 * a_s + chunk * 16, b_off = row0 * b_s + chunk * 16;
  const uint32_t a_rows = min(uint32_t(BM), p.m - m0), b_rows = min(uint32_t(BN), p.n - n0), left_in_last = p.k - (steps - 1) * BLOCK;
  const uint8_t *const a = p.a + int64_t(m0) * p.a_s, *const b = p.b + int64_t(n0) * p.b_s;
  const uint32_t scale_row = (wave * 64 + lane) % BM, scale_off = scale_row < a_rows ? scale_row * uint32_t(p.as_s) * 4 : OUTSIDE;
  const float *const a_scales = p.a_scales + int64_t(m0) * p.as_s;
  uint8_t *const ring = lds + my_group * (DEPTH * SLOT);
  const uint32_t lds0 = lds_address(ring);
  uint32_t slot_in = 0;   // where the next step goes
  auto fetch = [&](int turn) {
    const int step = turn * all_groups + first;
    const bool none = step == steps - 1 && chunk * 16 >= left_in_last;
    // (up to the last row's end: rows behind it bring zeros, or where rows overlap something, which nobody sees)
    const uint32_t left = p.k - step * BLOCK;
    const v4i from_a = resource(a + step * int(BLOCK), (a_rows - 1) * a_s + left), from_b = resource(b + step * int(BLOCK), (b_rows - 1) * b_s + left);
    const uint32_t to = lds0 + slot_in * SLOT;
    slot_in = slot_in + 1 == DEPTH ? 0 : slot_in + 1;
#pragma unroll
    for (int i = 0; i < A_LOADS; i++) dma16(from_a, none ? OUTSIDE : a_off + i * 32 * a_s, to + (i * 32 + wave * 8) * BLOCK);
#pragma unroll
    for (int i = 0; i < B_LOADS; i++) dma16(from_b, none ? OUTSIDE : b_off + i * 32 * b_s, to + (BM + i * 32 + wave * 8) * BLOCK);
    dma4(resource(a_scales + step, 0x7fffffff), scale_off, to + (BM + BN) * BLOCK + wave * 256);
  };
  typedef const __attribute__((address_space(4))) float const_float;   // (scalar loads: vector ones would be counted with those above)
  const_float *b_scale[SCALES];
#pragma unroll
  for (int u = 0; u < SCALES; u++) b_scale[u] = (const_float *)(p.b_scales + int64_t(min(n0 + wn + u * 16, p.n - 1) / BLOCK) * p.bs_s);
  auto fragment = [&](const uint8_t *row) {   // (rows of a fragment start at a multiple of 16)
    const uint8_t *const mine = row + li * BLOCK;
    const v4i lo = *(const v4i *)(mine + (lg ^ (li >> 1)) * 16), hi = *(const v4i *)(mine + ((lg + 4) ^ (li >> 1)) * 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  v4f acc[MT][NT] = {};
#pragma unroll
  for (int i = 0; i < DEPTH - 1; i++)
    if (i < mine) fetch(i);
  float sb[SCALES];
#pragma unroll
  for (int u = 0; u < SCALES; u++) sb[u] = b_scale[u][min(first, steps - 1)];
  uint32_t slot = 0;
  for (int turn = 0; turn < turns; turn++) {
    if (turn + DEPTH - 1 <= mine) wait_for_all_but<(DEPTH - 2) * LOADS>();   // (DEPTH - 2 steps behind this one are under way)
    else wait_for_all_but<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (turn + DEPTH - 1 < mine) fetch(turn + DEPTH - 1);   // (over the step before this one, which all waves are done with)
    if (GROUPS > 1 && turn >= mine) break;                  // (the last turn, and no barrier behind it in the loop)
    float next[SCALES];
#pragma unroll
    for (int u = 0; u < SCALES; u++) next[u] = b_scale[u][min((turn + 1) * all_groups + first, steps - 1)];
    const uint8_t *const from = ring + slot * SLOT;
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
    const float *const scales = (const float *)(from + (BM + BN) * BLOCK) + wm + li;
    Operand<OUT> w[NT];
#pragma unroll
    for (int u = 0; u < NT; u++) w[u].from(fragment(from + (BM + wn + u * 16) * BLOCK));
#pragma unroll
    for (int t = 0; t < MT; t++) {
      Operand<OUT> x;
      x.from(fragment(from + (wm + t * 16) * BLOCK));
      const float scale = scales[t * 16];
      v4f part[NT];
      products(part, w, x);
#pragma unroll
      for (int u = 0; u < NT; u++) acc[t][u] += part[u] * (scale * sb[SCALES == 1 ? 0 : u]);
    }
#pragma unroll
    for (int u = 0; u < SCALES; u++) sb[u] = next[u];
  }
  if constexpr (GROUPS > 1) {
    // The groups' sums in their order.
    __syncthreads();
    v4f *const parts = (v4f *)lds + (wave * MT * NT) * 64 + lane;   // [GROUPS - 1][4][MT * NT][64]
    if (my_group > 0) {
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int u = 0; u < NT; u++) parts[((my_group - 1) * 4 * MT * NT + t * NT + u) * 64] = acc[t][u];
    }
    __syncthreads();
    if (my_group > 0) return;
#pragma unroll
    for (int g = 0; g < GROUPS - 1; g++)
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int u = 0; u < NT; u++) acc[t][u] += parts[(g * 4 * MT * NT + t * NT + u) * 64];
  }
  if constexpr (GROUPS == 1) __syncthreads();   // (all waves have read their operands)
  else wait_for_lds();                          // (the sums of the others are in; each wave's lie where its own have been)
  if constexpr (SHARED) store_sums<MT, NT, float>(lds + wave * (MT * NT * 1024), acc, part_of(p), m0 + wm, n0 + wn);
  else store_sums<MT, NT, OUT>(lds + wave * (MT * NT * 1024), acc, p, m0 + wm, n0 + wn);
}

template <int BM, int BN, int GROUPS, int DEPTH, class OUT, bool SHARED = false>
hipError_t launch(const ProductArgs &p, hipStream_t stream) {
  constexpr int BYTES = GROUPS * DEPTH * ((BM + BN) * int(BLOCK) + 4 * 256);
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_product_tile<BM, BN, GROUPS, DEPTH, SHARED, OUT>), BYTES);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;
  MRL_LAUNCH((k_product_tile<BM, BN, GROUPS, DEPTH, SHARED, OUT>), dim3(tiles_m * tiles_n, SHARED ? p.shares : 1), dim3(GROUPS * 256), BYTES, stream, p, tiles_m, tiles_n, 512u / BM);
  return plan::last_error();
}

template <class OUT>
hipError_t choose(const ProductArgs &p, hipStream_t stream) {
  auto tiles = [&](uint32_t bm, uint32_t bn) { return uint64_t((p.m + bm - 1) / bm) * ((p.n + bn - 1) / bn); };
  if (p.shares > 1) return launch<64, 64, 3, 3, OUT, true>(p, stream);
  // The smallest tiles that the compute units take in one round, each with a workgroup of several groups; past a round of the largest, two workgroups of one to a unit.  us as 64 x 64
  // in 3 groups, 64 x 96, 128 x 64, 96 x 96, 128 x 96 and 128 x 128 in 2, and 128 x 128 in 1, bf16: 1024 x 1024 x 4096 (256 tiles of 64 x 64) 12.1, .., 18.4, .., .., 24.4, 28; 1024 x 1536 x 4096 22.4,
  // 15.3, 17.7, 18.7, 21.9, 23.6, 27.2; 1500 x 1500 x 2048 19.8, 16.6, 18.7, 12.0, 13.5, 14.8, 16.9; 1300 x 2600 x 2048 .., 23.3, 18.7, 20.6, 23.4, 14.6, 16.3; f32: 1001 x 2050 x 4432 .., 47.9, 58, 35,
  // 40, 44, 53; 1500 x 1500 x 2048 .., 22.6, 26.9, 16.2, 18.5, 20.7, 24.6; 1500 x 3500 x 2048 .., 42.6, 38.8, 41.5, 34.2, 38.4, 35.4.
  if (tiles(64, 64) <= g_compute_units) return launch<64, 64, 3, 3, OUT>(p, stream);
  if (tiles(64, 96) <= g_compute_units) return launch<64, 96, 2, 3, OUT>(p, stream);
  if (tiles(96, 64) <= g_compute_units) return launch<96, 64, 2, 3, OUT>(p, stream);
  if (tiles(128, 64) <= g_compute_units) return launch<128, 64, 2, 3, OUT>(p, stream);
  if (tiles(96, 96) <= g_compute_units) return launch<96, 96, 2, 3, OUT>(p, stream);
  if (tiles(128, 96) <= g_compute_units) return launch<128, 96, 2, 2, OUT>(p, stream);
  if (tiles(128, 128) <= g_compute_units) return launch<128, 128, 2, 2, OUT>(p, stream);
  return launch<128, 128, 1, 2, OUT>(p, stream);
}

}  // namespace

// As many as find a compute unit, of tiles that leave half of them without one, with four blocks and more to each group of waves.  (us, one and as many: 129 x 512 x 4992 12.0 and 9.2, 256 x 1024 x 8192 19.5 and 11.6,
// 600 x 600 x 4096 in f32 15.5 and 13.2, 128 x 4096 x 4096 11.9 and 11.3; with two blocks 128 x 1024 x 2048 6.8 and 7.6.)
uint32_t shares_of_tiles(const ProductArgs &p) {
  const uint64_t tiles = uint64_t((p.m + 63) / 64) * ((p.n + 63) / 64);
  return uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(g_compute_units / tiles, (p.k + BLOCK - 1) / BLOCK / 12)));
}

hipError_t launch_product_tile(const ProductArgs &p, hipStream_t stream) { return p.out_dtype == MRL_BF16 ? choose<uint16_t>(p, stream) : choose<float>(p, stream); }

}  // namespace mrl
