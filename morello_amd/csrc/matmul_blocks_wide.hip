// The product of blocks (matmul_blocks.hip) on tiles of 256 x 256, for rows of whole 16-byte chunks and results in bf16.
//
// Eight waves of 128 rows of a by 64 of b: 128 sums a lane.  (Four waves of 128 x 128 would read a third less from LDS, but their 256 sums leave a wave's vector
// instructions, which reach 256 registers, nothing to work with: every sum takes one of them per block.)  Per block of K a wave has 32 matrix
// instructions of 32 cycles and 128 multiply-adds of 4, in the shadow of the other wave's matrix instructions on the same SIMD.  Operands go
// straight from memory into LDS, two blocks of 64 KiB, the next under this one's products; chunk c of a row at c ^ (row / 2 % 8), so that sixteen lanes with
// a chunk of sixteen rows each reach every bank once.  The products of both scales are formed four blocks ahead by all threads, and lie in LDS by rows of a.
#include "matmul_blocks.h"

namespace mrl {
namespace {
using namespace blocks;

constexpr int SIDE = 256, THREADS = 512, AHEAD = 4;            // AHEAD: blocks whose scales are formed together
constexpr int SLOT = 2 * SIDE * int(BLOCK), SCALES = AHEAD * 2 * SIDE * 4;
constexpr int LDS_BYTES = 2 * SLOT + 2 * SCALES;
constexpr int HIGH = 4;                                         // tiles of m that go together

__global__ __launch_bounds__(THREADS, 2) void k_product_wide(ProductArgs p, uint32_t tiles_m, uint32_t tiles_n) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
  // An XCD's tiles in groups of HIGH by all of n.
  const uint32_t at = xcd_run(blockIdx.x, gridDim.x), group = at / (HIGH * tiles_n), high = min(uint32_t(HIGH), tiles_m - group * HIGH), in_group = at - group * HIGH * tiles_n;
  const uint32_t tile_n = in_group / high, tile_m = group * HIGH + in_group - tile_n * high;
  const uint32_t m0 = tile_m * SIDE, n0 = tile_n * SIDE;
  const int steps = int((p.k + BLOCK - 1) / BLOCK);

  // This wave's eight loads of a step: 64 rows of a (waves 0 to 3) or of b, eight to a load.
  const bool of_a = wave < 4;
  const uint32_t first = (wave & 3) * 64, stride = uint32_t(of_a ? p.a_s : p.b_s), rows = of_a ? min(uint32_t(SIDE), p.m - m0) : min(uint32_t(SIDE), p.n - n0);
  const uint8_t *const tile = of_a ? p.a + int64_t(m0) * p.a_s : p.b + int64_t(n0) * p.b_s;
  const uint32_t row8 = lane >> 3, even = (lane & 7) ^ (row8 >> 1), odd = even ^ 4;   // chunks of even and odd loads
  const uint32_t off_even = (first + row8) * stride + even * 16, off_odd = (first + 8 + row8) * stride + odd * 16;
  const uint32_t lds0 = lds_address(lds), to0 = lds0 + (of_a ? 0 : SIDE * BLOCK) + first * BLOCK;
  const uint32_t left_in_last = p.k - (steps - 1) * BLOCK;
  auto fetch = [&](int step) {
    // (up to the last row's end: rows behind it bring zeros, or where rows overlap something, which nobody sees)
    const v4i from = resource(tile + step * int(BLOCK), (rows - 1) * stride + (p.k - step * BLOCK));
    const bool last = step == steps - 1;
    const uint32_t e = last && even * 16 >= left_in_last ? OUTSIDE : off_even, o = last && odd * 16 >= left_in_last ? OUTSIDE : off_odd;
    const uint32_t to = to0 + (step & 1) * SLOT;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      dma16(from, e + i * 8 * stride, to + i * 1024);
      dma16(from, o + i * 8 * stride, to + (i + 1) * 1024);
    }
  };
  // The products of scales of AHEAD steps: [slot][step][half of n][row of a].
  float *const scales = (float *)(lds + 2 * SLOT);
  const float *const a_scale = p.a_scales + int64_t(min(m0 + (tid & 255), p.m - 1)) * p.as_s;
  const float *const b_scale = p.b_scales + int64_t(min(n0 / BLOCK + (tid >> 8), (p.n - 1) / BLOCK)) * p.bs_s;
  float sa[AHEAD], sb[AHEAD];
  auto fetch_scales = [&](int step) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++) sa[i] = a_scale[min(step + i, steps - 1)], sb[i] = b_scale[min(step + i, steps - 1)];
  };
  auto keep_scales = [&](int slot) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++) scales[((slot * AHEAD + i) * 2 + (tid >> 8)) * SIDE + (tid & 255)] = sa[i] * sb[i];
  };
  auto fragment = [&](const uint8_t *row) {   // (rows of a fragment start at a multiple of 16)
    const uint8_t *const mine = row + li * BLOCK;
    const v4i lo = *(const v4i *)(mine + (lg ^ (li >> 1)) * 16), hi = *(const v4i *)(mine + ((lg + 4) ^ (li >> 1)) * 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  v4f acc[8][4] = {};
  fetch_scales(0);
  fetch(0);
  keep_scales(0);
  for (int step = 0; step < steps; step++) {
    wait_for_all_but<0>();
    if (step % AHEAD == 1 && step + AHEAD - 1 < steps) keep_scales((step / AHEAD + 1) & 1);   // (asked for a step ago)
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (step % AHEAD == 0 && step + AHEAD < steps) fetch_scales(step + AHEAD);
    if (step + 1 < steps) fetch(step + 1);
    const uint8_t *const a = lds + (step & 1) * SLOT + wm * 128 * BLOCK, *const b = lds + (step & 1) * SLOT + (SIDE + wn * 64) * BLOCK;
    const float *const scale = scales + ((step / AHEAD & 1) * AHEAD * 2 + step % AHEAD * 2 + (wn >> 1)) * SIDE + wm * 128 + li;
    v8i w[4], x[2];
    v4f part[2][4];
    float s[2];
    x[0] = fragment(a), s[0] = scale[0];
#pragma unroll
    for (int u = 0; u < 4; u++) w[u] = fragment(b + u * 16 * BLOCK);
    // A sixteen of a's rows under the multiply-adds of the one before; its operands are read one ahead.
#pragma unroll
    for (int t = 0; t < 9; t++) {
      if (t < 7) x[(t + 1) & 1] = fragment(a + (t + 1) * 16 * BLOCK);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (t < 8) part[t & 1][u] = mma_e4m3(w[u], x[t & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (t > 0) acc[t - 1][u] += part[(t - 1) & 1][u] * s[(t - 1) & 1];
      }
      if (t < 7) s[(t + 1) & 1] = scale[(t + 1) * 16];
    }
  }
#pragma unroll
  for (int t = 0; t < 8; t++) {
    const uint32_t row = m0 + wm * 128 + t * 16 + li;
    if (row >= p.m) continue;
    uint16_t *const out = (uint16_t *)p.out + int64_t(row) * p.out_s;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t col = n0 + wn * 64 + u * 16 + lg * 4;
      store4(out + col, acc[t][u], int(p.n) - int(col));
    }
  }
}

}  // namespace

hipError_t launch_product_wide(const ProductArgs &p, hipStream_t stream) {
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_product_wide), LDS_BYTES);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_m = (p.m + SIDE - 1) / SIDE, tiles_n = (p.n + SIDE - 1) / SIDE;
  MRL_LAUNCH(k_product_wide, dim3(tiles_m * tiles_n), dim3(THREADS), LDS_BYTES, stream, p, tiles_m, tiles_n);
  return plan::last_error();
}

}  // namespace mrl
