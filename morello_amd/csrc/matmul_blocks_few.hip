// The product of blocks (matmul_blocks.hip) for up to 96 rows of a, of whole 16-byte chunks.
//
// What bounds it is reading b once.  A workgroup has 16 NT of b's rows and all of a's (16 MT), its waves every WAVES-th block of K each: a block's 128 bytes
// of all these rows, and a's scales, go straight from memory into a ring of DEPTH blocks in LDS that is the wave's own, so that no wave waits for another
// before the end, and what is under way is bounded by LDS and not by registers.  Eight lanes take a row's 128 bytes: sixteen cycles for an instruction's KiB, where the order in
// which the matrix instructions want them (a lane of sixteen different rows next to each other) would take 64.
// 8 x 4096 x 4096 5.1 us (17 MB; 5.8 with cold caches), 96 x 8192 x 8192 20.5 us (68 MB, 3.3 TB/s), 67 x 6144 x 4096 8.2 us: of a workgroup's 460 KB there 330 are a, which every one of them reads from L2.
#include "matmul_blocks.h"

namespace mrl {
namespace {
using namespace blocks;

template <int MT, int NT, int WAVES, int DEPTH, class OUT>
__global__ __launch_bounds__(WAVES * 64) void k_product_few(ProductArgs p) {
  constexpr int ROWS = (MT + NT) * 16, SCALE_LOADS = (MT + 3) / 4, LOADS = (MT + NT) * 2 + SCALE_LOADS;
  constexpr int SLOT = ROWS * int(BLOCK) + SCALE_LOADS * 256;
  static_assert((DEPTH - 1) * LOADS < 64 && WAVES * DEPTH * SLOT <= 160 * 1024 && MT * NT <= 2 * DEPTH * SLOT / 2048, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n0 = blockIdx.x * (16 * NT);
  const int steps = int((p.k + BLOCK - 1) / BLOCK), mine = steps > wave ? (steps - wave + WAVES - 1) / WAVES : 0;
  uint8_t *const ring = lds + wave * (DEPTH * SLOT);
  const uint32_t ring_at = lds_address(ring);
  // Chunk c of a row at c ^ (row / 2 % 8) of its 128 bytes; eight rows to a load.
  const uint32_t row8 = lane >> 3, even = (lane & 7) ^ (row8 >> 1), odd = even ^ 4, a_s = uint32_t(p.a_s), b_s = uint32_t(p.b_s);
  const uint32_t left_in_last = p.k - (steps - 1) * BLOCK, b_rows = min(uint32_t(16 * NT), p.n - n0);
  const uint8_t *const b = p.b + int64_t(n0) * p.b_s;
  uint32_t scale_off[SCALE_LOADS];
#pragma unroll
  for (int i = 0; i < SCALE_LOADS; i++) scale_off[i] = uint32_t(i * 64 + lane) < p.m ? uint32_t(i * 64 + lane) * uint32_t(p.as_s) * 4 : OUTSIDE;
  auto fetch = [&](int i) {   // the wave's i-th block
    const int step = wave + i * WAVES;
    const bool last = step == steps - 1;
    const bool no_even = last && even * 16 >= left_in_last, no_odd = last && odd * 16 >= left_in_last;
    // (up to the last row's end: rows behind it bring zeros, or where rows overlap something, which nobody sees)
    const uint32_t left = p.k - step * BLOCK;
    const v4i from_b = resource(b + step * int(BLOCK), (b_rows - 1) * b_s + left), from_a = resource(p.a + step * int(BLOCK), (p.m - 1) * a_s + left);
    const v4i from_scales = resource(p.a_scales + step, 0x7fffffff);
    const uint32_t to = ring_at + uint32_t(i % DEPTH) * SLOT;
#pragma unroll
    for (int j = 0; j < NT * 2; j++) dma16(from_b, (j & 1 ? no_odd : no_even) ? OUTSIDE : (j * 8 + row8) * b_s + (j & 1 ? odd : even) * 16, to + j * 1024);
#pragma unroll
    for (int j = 0; j < MT * 2; j++) dma16(from_a, (j & 1 ? no_odd : no_even) ? OUTSIDE : (j * 8 + row8) * a_s + (j & 1 ? odd : even) * 16, to + (NT * 2 + j) * 1024);
#pragma unroll
    for (int j = 0; j < SCALE_LOADS; j++) dma4(from_scales, scale_off[j], to + ROWS * BLOCK + j * 256);
  };
  typedef const __attribute__((address_space(4))) float const_float;   // (scalar loads: vector ones would be counted with those above)
  const_float *const b_scale = (const_float *)(p.b_scales + int64_t(n0 / BLOCK) * p.bs_s);
  auto fragment = [&](const uint8_t *row) {
    const uint8_t *const at = row + li * BLOCK;
    const v4i lo = *(const v4i *)(at + (lg ^ (li >> 1)) * 16), hi = *(const v4i *)(at + ((lg + 4) ^ (li >> 1)) * 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  v4f acc[MT][NT] = {};
#pragma unroll
  for (int i = 0; i < DEPTH - 1; i++)
    if (i < mine) fetch(i);
  float sb = mine ? b_scale[wave] : 0.0f;
  for (int i = 0; i < mine; i++) {
    if (i + DEPTH - 1 < mine) {
      fetch(i + DEPTH - 1);   // (over the block before this one, whose reads the last iteration ended on)
      wait_for_all_but<(DEPTH - 1) * LOADS>();
    } else {
      wait_for_all_but<0>();
    }
    const float next = i + 1 < mine ? b_scale[wave + (i + 1) * WAVES] : 0.0f;
    const uint8_t *const slot = ring + i % DEPTH * SLOT;
    const float *const scales = (const float *)(slot + ROWS * BLOCK);
    Operand<OUT> w[NT];
#pragma unroll
    for (int u = 0; u < NT; u++) w[u].from(fragment(slot + u * 16 * BLOCK));
#pragma unroll
    for (int t = 0; t < MT; t++) {
      Operand<OUT> x;
      x.from(fragment(slot + (NT + t) * 16 * BLOCK));
      const float scale = scales[t * 16 + li] * sb;
      v4f part[NT];
      products(part, w, x);
#pragma unroll
      for (int u = 0; u < NT; u++) acc[t][u] += part[u] * scale;
    }
    sb = next;
    wait_for_lds();
  }
  __syncthreads();
  v4f *const part = (v4f *)lds;   // [WAVES][MT * NT][64]
#pragma unroll
  for (int t = 0; t < MT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) part[(wave * MT * NT + t * NT + u) * 64 + lane] = acc[t][u];
  __syncthreads();
  for (int x = wave; x < MT * NT; x += WAVES) {
    v4f sum = part[x * 64 + lane];
#pragma unroll
    for (int v = 1; v < WAVES; v++) sum += part[(v * MT * NT + x) * 64 + lane];
    const uint32_t row = x / NT * 16 + li, col = n0 + x % NT * 16 + lg * 4;
    if (row < p.m && col < p.n) store4((OUT *)p.out + int64_t(row) * p.out_s + col, sum, int(p.n - col));
  }
}

template <int MT, int NT, int WAVES, int DEPTH, class OUT>
hipError_t launch(const ProductArgs &p, hipStream_t stream) {
  constexpr int BYTES = WAVES * DEPTH * ((MT + NT) * 16 * int(BLOCK) + (MT + 3) / 4 * 256);
  static std::atomic<uint64_t> raised{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(raised, reinterpret_cast<const void *>(&k_product_few<MT, NT, WAVES, DEPTH, OUT>), BYTES);
    if (e != hipSuccess) return e;
  }
  MRL_LAUNCH((k_product_few<MT, NT, WAVES, DEPTH, OUT>), dim3((p.n + 16 * NT - 1) / (16 * NT)), dim3(WAVES * 64), BYTES, stream, p);
  return plan::last_error();
}

template <class OUT>
hipError_t choose(const ProductArgs &p, hipStream_t stream) {
  // 32 of b's rows to a workgroup where these still keep three in four compute units busy.  (us, 16 and 32: 48 x 4096 x 4096 7.5 and 7.7, 96 x 4096 x 4096 10.4 and 11.0, 48 x 6144 x 4096 11.5 and 8.2,
  // 96 x 6144 x 4096 18.0 and 11.6.)
  const bool pairs = p.n >= 32 * g_compute_units * 3 / 4;
  switch ((p.m + 15) / 16) {
    case 1: return launch<1, 1, 8, 4, OUT>(p, stream);
    case 2: return launch<2, 1, 8, 3, OUT>(p, stream);
    case 3: return pairs ? launch<3, 2, 4, 3, OUT>(p, stream) : launch<3, 1, 8, 2, OUT>(p, stream);
    case 4: return pairs ? launch<4, 2, 4, 3, OUT>(p, stream) : launch<4, 1, 4, 3, OUT>(p, stream);
    case 5: return pairs ? launch<5, 2, 4, 2, OUT>(p, stream) : launch<5, 1, 6, 2, OUT>(p, stream);
    default: return pairs ? launch<6, 2, 4, 2, OUT>(p, stream) : launch<6, 1, 4, 2, OUT>(p, stream);
  }
}

}  // namespace

hipError_t launch_product_few(const ProductArgs &p, hipStream_t stream) { return p.out_dtype == MRL_BF16 ? choose<uint16_t>(p, stream) : choose<float>(p, stream); }

}  // namespace mrl
