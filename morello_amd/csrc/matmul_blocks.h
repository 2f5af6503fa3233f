// What the kernels of products of blocks share (matmul_blocks.hip, matmul_blocks_wide.hip).
#pragma once
#include <algorithm>

#include "blocks_device.h"

namespace mrl {
namespace blocks {

// Results in bf16 come from products in e4m3, whose cuts, 2^-13 of a block's largest product each, came to 2^-12.2 of it at worst on normal data: as much as the result's own rounding where products cancel to some 2^-4 of the
// largest, and more below that (128 cuts that all go one way would be 2^-6 of it); results in f32 from the same numbers in bf16.
template <class OUT> struct Operand;
template <> struct Operand<uint16_t> {
  v8i x;
  __device__ inline void from(v8i q) { x = q; }
};
template <> struct Operand<float> {
  Wide x;
  __device__ inline void from(v8i q) { x = widen(q); }
};
// sums[i] = a block's products of w[i] and x.  (In bf16 four instructions to a sum, each of which waits for the one before: N sums side by side.)
template <int N>
__device__ inline void products(v4f (&sums)[N], const Operand<uint16_t> (&w)[N], const Operand<uint16_t> &x) {
#pragma unroll
  for (int i = 0; i < N; i++) sums[i] = mma_e4m3(w[i].x, x.x);
}
template <int N>
__device__ inline void products(v4f (&sums)[N], const Operand<float> (&w)[N], const Operand<float> &x) {
#pragma unroll
  for (int i = 0; i < N; i++) sums[i] = v4f{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < N; i++) sums[i] = mma_bf16(w[i].x.x[j], x.x.x[j], sums[i]);
}

constexpr uint32_t OUTSIDE = 0x80000000u;   // an offset that no resource here holds
typedef __attribute__((address_space(3))) void lds_void;
__device__ inline uint32_t lds_address(const void *p) { return uint32_t(reinterpret_cast<uintptr_t>((lds_void *)p)); }
// 64 lanes x 16 bytes from `off` (of each lane) behind `from` into the KiB at LDS address `to`, lane l to its l-th sixteen; offsets past the resource bring zeros.  Assembly, so
// that the compiler does not wait for it; M0 is set in the same statement.
__device__ inline void dma16(v4i from, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(off), "s"(from), "s"(to) : "memory");
}
// The same with 4 bytes a lane: 256 bytes.
__device__ inline void dma4(v4i from, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" : : "v"(off), "s"(from), "s"(to) : "memory");
}
__device__ inline v4i resource(const void *base, uint32_t bytes) {
  const uint64_t b = reinterpret_cast<uintptr_t>(base);
  return v4i{int(uint32_t(b)), int(uint32_t(b >> 32)), int(bytes), 0x00020000};
}
// All but the newest N loads have landed, and every LDS access of this wave is done.
template <int N>
__device__ inline void wait_for_all_but() {
  asm volatile("" : : : "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  asm volatile("" : : : "memory");
}

// Every LDS access of this wave is done.
__device__ inline void wait_for_lds() {
  asm volatile("" : : : "memory");
  __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);
  asm volatile("" : : : "memory");
}

// Rows of whole 16-byte chunks, 256 of them within 2 GB.
inline bool rows_of_chunks(const void *p, int64_t stride, uint32_t k) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 16 == 0 && k % 16 == 0 && stride < (1 << 23);
}

// A wave's sums of MT x NT sixteens, the first of row `row0` and column `col0`, through `lds` (16 * MT * 16 * NT elements) into whole rows: chunk c of a row at c ^ row, as far as
// that stays in the row.
template <int MT, int NT, class OUT>
__device__ inline void store_sums(uint8_t *lds, const v4f (&acc)[MT][NT], const ProductArgs &p, uint32_t row0, uint32_t col0) {
  constexpr int SIZE = sizeof(OUT), EACH = 16 / SIZE, ROW = NT * 16 * SIZE, CHUNKS = ROW / 16, TURNED = (CHUNKS & -CHUNKS) - 1, ALL = MT * 16 * CHUNKS;
  const uint32_t lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int t = 0; t < MT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) {
      const v4f &x = acc[t][u];
      const uint32_t byte = (u * 16 + lg * 4) * SIZE;
      uint8_t *const to = lds + (t * 16 + li) * ROW + (byte / 16 ^ (li & TURNED)) * 16 + byte % 16;
      if constexpr (SIZE == 2) *(v4bf *)to = v4bf{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
      else *(v4f *)to = x;
    }
  lanes_meet();
  const uint32_t row_end = p.m - min(p.m, row0);
  OUT *const out = (OUT *)p.out + int64_t(row0) * p.out_s + col0;
#pragma unroll
  for (int i = 0; i < (ALL + 63) / 64; i++) {
    const uint32_t at = i * 64 + lane, row = at / CHUNKS, chunk = at % CHUNKS, col = col0 + chunk * EACH;
    if ((ALL % 64 == 0 || at < ALL) && row < row_end && col < p.n) {
      const v4i x = *(const v4i *)(lds + row * ROW + (chunk ^ (row & TURNED)) * 16);
      OUT *const to = out + int64_t(row) * p.out_s + chunk * EACH;
      if (col + EACH <= p.n) *(v4i_any *)to = x;
      else
#pragma unroll
        for (int e = 0; e < EACH; e++)
          if (col + e < p.n) {
            if constexpr (SIZE == 2) to[e] = uint16_t(uint32_t(x[e / 2]) >> (e % 2 * 16));
            else to[e] = __int_as_float(x[e]);
          }
    }
  }
}

// This workgroup's part, where several share K.
__device__ inline ProductArgs part_of(const ProductArgs &p) {
  ProductArgs q = p;
  q.out = p.parts + uint64_t(blockIdx.y) * p.m * p.parts_s, q.out_s = p.parts_s;
  return q;
}

}  // namespace blocks

hipError_t launch_product_wide(const ProductArgs &p, hipStream_t stream);
hipError_t launch_product_tile(const ProductArgs &p, hipStream_t stream);
// Rows of whole chunks, scales of a within 2 GB.  (us, so and on tiles: 80 x 8192 x 8192 19.4 and 20.4, 96 x 4096 x 4096 10.4 and 11.8, 128 x 8192 x 8192 41.8 and 21.3, 128 x 4096 x 4096 13.4 and 12.0.)
constexpr uint32_t MOST_FEW = 96;
hipError_t launch_product_few(const ProductArgs &p, hipStream_t stream);
// Workgroups that share the K of a tile; of more than one, sums go to parts.
uint32_t shares_of_tiles(const ProductArgs &p);

}  // namespace mrl
