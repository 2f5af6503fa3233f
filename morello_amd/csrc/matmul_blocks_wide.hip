// The product of blocks (matmul_blocks.hip) on tiles of 256 x 256, for rows of whole 16-byte chunks and results in bf16.
//
// Eight waves of 128 rows of a by 64 of b: 128 sums a lane.  (Four waves of 128 x 128 would read a third less from LDS, but their 256 sums leave a wave's vector
// instructions, which reach 256 registers, nothing to work with: every sum takes one of them per block.)  Per block of K a wave has 32 matrix
// instructions of 32 cycles and 128 multiply-adds of 4, in the shadow of the other wave's matrix instructions on the same SIMD.  Operands go
// straight from memory into LDS, which holds two blocks of 64 KiB; chunk c of a row at c ^ (row / 2 % 8), so that sixteen lanes with
// a chunk of sixteen rows each reach every bank once.  What bounds it is the way of 64 KiB into each compute unit, some 3500 cycles from the first load to the last byte where the products take
// 2048: a block's last operands are read into registers halfway through its products, and the block after the next is asked for then, over it.  8192^3 478 to 490 us
// (2.25 to 2.3 PFLOP/s, the clock at 2.0 GHz), 4096^3 62 us (2.2 PFLOP/s); the loop without its loads 396, its matrix instructions alone 324 (the clock at 1.6).
#include "matmul_blocks.h"

namespace mrl {
namespace {
using namespace blocks;

constexpr int SIDE = 256, THREADS = 512;
constexpr int SLOT = 2 * SIDE * int(BLOCK), LOADS = 8;          // a's rows and b's; a wave's loads, a step
constexpr int GROUP = 8, SCALES = GROUP * SIDE * 4;             // a's scales, of a group of steps
constexpr int LDS_BYTES = 2 * SLOT + 2 * SCALES;
constexpr int HIGH = 4;                                         // tiles of m that go together

template <bool CHUNKS>   // a's scales are whole 16-byte chunks
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
  // a's scales of a group of steps, with the first of them: 32 rows from each wave, two lanes to a row's 32 bytes, to [row][step]; where they are not whole chunks four bytes of a row at a time, from the
  // first four waves 64 rows each, to [step][row].
  const uint32_t a_rows = min(uint32_t(SIDE), p.m - m0);
  const uint32_t scale_row = CHUNKS ? wave * 32 + lane / 2 : (wave & 3) * 64 + lane, scale_off = scale_row < a_rows ? scale_row * uint32_t(p.as_s) * 4 + (CHUNKS ? lane % 2 * 16 : 0) : OUTSIDE;
  const float *const a_scales = p.a_scales + int64_t(m0) * p.as_s;
  auto fetch_scales = [&](int step) {
    const uint32_t to = lds0 + 2 * SLOT + (step / GROUP & 1) * SCALES;
    if constexpr (CHUNKS) {
      dma16(resource(a_scales + step, 0x7fffffff), step + lane % 2 * 4 < steps ? scale_off : OUTSIDE, to + wave * 1024);
    } else if (wave < 4) {
      for (int i = 0; i < GROUP && step + i < steps; i++) dma4(resource(a_scales + step + i, 0x7fffffff), scale_off, to + i * (SIDE * 4) + wave * 256);
    }
  };
  // What of the others depends on the step; the i-th of them.  (Behind the last step: zeros that nobody reads, rather than branches.)
  v4i from;
  uint32_t even_off, odd_off, slot_in;
  auto begin_fetch = [&](int step) {
    // (up to the last row's end: rows behind it bring zeros, or where rows overlap something, which nobody sees)
    from = resource(tile + step * int(BLOCK), step < steps ? (rows - 1) * stride + (p.k - step * BLOCK) : 0);
    const bool last = step == steps - 1;
    even_off = last && even * 16 >= left_in_last ? OUTSIDE : off_even, odd_off = last && odd * 16 >= left_in_last ? OUTSIDE : off_odd;
    slot_in = (step & 1) * SLOT;
  };
  auto fetch = [&](int i) { dma16(from, (i & 1 ? odd_off : even_off) + (i & ~1) * 8 * stride, to0 + slot_in + i * 1024); };
  typedef const __attribute__((address_space(4))) float const_float;   // (scalar loads: vector ones would be counted with those above)
  const_float *const b_scale = (const_float *)(p.b_scales + int64_t(min(n0 + wn * 64, p.n - 1) / BLOCK) * p.bs_s);
  auto fragment = [&](const uint8_t *row) {   // (rows of a fragment start at a multiple of 16)
    const uint8_t *const mine = row + li * BLOCK;
    const v4i lo = *(const v4i *)(mine + (lg ^ (li >> 1)) * 16), hi = *(const v4i *)(mine + ((lg + 4) ^ (li >> 1)) * 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  v4f acc[8][4] = {};
#pragma unroll
  for (int ahead = 0; ahead < 2; ahead++) {
    if (ahead == 0) fetch_scales(0);
    begin_fetch(ahead);
#pragma unroll
    for (int i = 0; i < LOADS; i++) fetch(i);
  }
  float sb = b_scale[0];
  for (int step = 0; step < steps; step++) {
    wait_for_all_but<LOADS>();   // (those of the step behind this one; scales are asked for in front of them)
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if ((step + 1) % GROUP == 0 && step + 1 < steps) fetch_scales(step + 1);
    const uint8_t *const slot = lds + (step & 1) * SLOT, *const a = slot + wm * 128 * BLOCK, *const b = slot + (SIDE + wn * 64) * BLOCK;
    const float *const scale = (const float *)(lds + 2 * SLOT + (step / GROUP & 1) * SCALES) + (CHUNKS ? (wm * 128 + li) * GROUP + step % GROUP : step % GROUP * SIDE + wm * 128 + li);
    const float next = b_scale[min(step + 1, steps - 1)];
    // A sixteen of a's rows under the multiply-adds of the one before; its operands are read three ahead.
    v8i w[4], x[4];
    v4f part[2][4];
    float s[8];
    x[0] = fragment(a);
#pragma unroll
    for (int u = 0; u < 4; u++) w[u] = fragment(b + u * 16 * BLOCK);
#pragma unroll
    for (int t = 1; t < 3; t++) x[t] = fragment(a + t * 16 * BLOCK);
#pragma unroll
    for (int t = 0; t < 8; t++) s[t] = scale[t * 16 * (CHUNKS ? GROUP : 1)];
#pragma unroll
    for (int t = 0; t < 9; t++) {
      if (t < 5) x[(t + 3) & 3] = fragment(a + (t + 3) * 16 * BLOCK);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (t < 8) part[t & 1][u] = mma_e4m3(w[u], x[t & 3]);
        __builtin_amdgcn_sched_barrier(0);
        if (t > 0) acc[t - 1][u] += part[(t - 1) & 1][u] * (s[t - 1] * sb);
      }
      if (t == 4) {   // the slot has been read
        wait_for_lds();
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
        begin_fetch(step + 2);
      }
#pragma unroll
      for (int i = 0; i < 3; i++)
        if (t >= 5 && t < 8 && (t - 5) * 3 + i < LOADS) fetch((t - 5) * 3 + i);
    }
    sb = next;
  }
  wait_for_all_but<0>();   // (what is under way goes into this workgroup's LDS)
  __syncthreads();
  // Through LDS, where a wave's sums take 16 KiB, into whole rows of 128 bytes: eight columns, which are sixteen bytes, at c ^ (row % 8).  (In 32-byte pieces of rows 8192^3 takes 2 % longer,
  // 4096 x 4096 x 1024 15 %; store_sums, which does the same, 1.5 %.)
  uint8_t *const mine = lds + wave * 16384;
#pragma unroll
  for (int t = 0; t < 8; t++)
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const v4f &x = acc[t][u];
      *(v4bf *)(mine + (t * 16 + li) * 128 + ((u * 2 + lg / 2) ^ (li & 7)) * 16 + lg % 2 * 8) = v4bf{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
    }
  lanes_meet();
  const uint32_t col = n0 + wn * 64 + (lane & 7) * 8, row_end = min(128u, p.m - min(p.m, m0 + wm * 128));
  uint16_t *const out = (uint16_t *)p.out + int64_t(m0 + wm * 128) * p.out_s + col;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const uint32_t row = i * 8 + row8;
    const v4i x = *(const v4i *)(mine + row * 128 + ((lane & 7) ^ row8) * 16);
    if (row < row_end && col < p.n) {
      if (col + 8 <= p.n) *(v4i_any *)(out + int64_t(row) * p.out_s) = x;
      else
        for (uint32_t e = 0; e < p.n - col; e++) out[int64_t(row) * p.out_s + e] = uint16_t(uint32_t(x[e / 2]) >> (e % 2 * 16));
    }
  }
}

template <bool CHUNKS>
hipError_t launch(const ProductArgs &p, hipStream_t stream) {
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_product_wide<CHUNKS>), LDS_BYTES);
    if (e != hipSuccess) return e;
  }
  const uint32_t tiles_m = (p.m + SIDE - 1) / SIDE, tiles_n = (p.n + SIDE - 1) / SIDE;
  MRL_LAUNCH(k_product_wide<CHUNKS>, dim3(tiles_m * tiles_n), dim3(THREADS), LDS_BYTES, stream, p, tiles_m, tiles_n);
  return plan::last_error();
}

}  // namespace

hipError_t launch_product_wide(const ProductArgs &p, hipStream_t stream) {
  return (reinterpret_cast<uintptr_t>(p.a_scales) & 15) == 0 && p.as_s % 4 == 0 && (p.k + BLOCK - 1) / BLOCK % 4 == 0 ? launch<true>(p, stream) : launch<false>(p, stream);
}

}  // namespace mrl
