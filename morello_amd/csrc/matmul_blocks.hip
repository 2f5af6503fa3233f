// out[m][n] = sum over blocks j of K of sa[m][j] sb[n / 128][j] (sum over the block's 128 k of a[m][k] b[n][k]),  a and b in e4m3.
//
// A matrix instruction takes a whole block of K (16 x 16 x 128), so that a block's sums come out of it against zero and are added
// to the running ones, in 32 bits, by one multiplication with both scales: as many vector instructions as sums, beside one matrix instruction
// for every four of them per lane.  b's rows are the instruction's first operand: a lane then holds four neighbouring n of one m, whose scales it
// has as one number.
#include <algorithm>

#include "matmul_blocks.h"

namespace mrl {
namespace {
using namespace blocks;

// ---- Tiles of BM x BN, the waves 2 x 2 ----
constexpr int TILE_THREADS = 256;
template <int BM, int BN, class OUT>
__global__ __launch_bounds__(TILE_THREADS) void k_product_tile_any(ProductArgs p, uint32_t tiles_m) {
  constexpr int A_EACH = BM * 8 / TILE_THREADS, B_EACH = BN * 8 / TILE_THREADS, MT = BM / 32, NT = BN / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][(BM + BN) * BLOCK];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tile_n = blockIdx.x / tiles_m, tile_m = blockIdx.x - tile_n * tiles_m;
  const uint32_t m0 = tile_m * BM, n0 = tile_n * BN, wm = wave / 2 * (BM / 2), wn = wave % 2 * (BN / 2);
  const int steps = int((p.k + BLOCK - 1) / BLOCK), k = int(p.k);
  // Chunk c of a row lies at c ^ (row % 8) of its 128 bytes.
  const int chunk = tid & 7, row0 = tid >> 3;
  const uint32_t put = row0 * BLOCK + (chunk ^ (row0 & 7)) * 16;
  v4i a_reg[A_EACH], b_reg[B_EACH];
  auto fetch = [&](int step) {
    const int at = step * int(BLOCK) + chunk * 16;
#pragma unroll
    for (int i = 0; i < A_EACH; i++) a_reg[i] = chunk_up_to(p.a + int64_t(min(m0 + row0 + i * 32, p.m - 1)) * p.a_s + at, k - at, at);
#pragma unroll
    for (int i = 0; i < B_EACH; i++) b_reg[i] = chunk_up_to(p.b + int64_t(min(n0 + row0 + i * 32, p.n - 1)) * p.b_s + at, k - at, at);
  };
  auto keep = [&](int slot) {
#pragma unroll
    for (int i = 0; i < A_EACH; i++) *(v4i *)(lds[slot] + put + i * 32 * BLOCK) = a_reg[i];
#pragma unroll
    for (int i = 0; i < B_EACH; i++) *(v4i *)(lds[slot] + BM * BLOCK + put + i * 32 * BLOCK) = b_reg[i];
  };
  auto fragment = [&](const uint8_t *row) {   // (rows of a fragment start at a multiple of 16)
    const v4i lo = *(const v4i *)(row + li * BLOCK + ((2 * lg) ^ (li & 7)) * 16), hi = *(const v4i *)(row + li * BLOCK + ((2 * lg + 1) ^ (li & 7)) * 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  const float *a_scale[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) a_scale[t] = p.a_scales + int64_t(min(m0 + wm + t * 16 + li, p.m - 1)) * p.as_s;
  const float *b_scale = p.b_scales + int64_t(min(n0 + wn, p.n - 1) / BLOCK) * p.bs_s;
  v4f acc[MT][NT] = {};
  fetch(0);
  for (int step = 0; step < steps; step++) {
    keep(step & 1);
    float scale[MT];
    const float sb = b_scale[step];
#pragma unroll
    for (int t = 0; t < MT; t++) scale[t] = a_scale[t][step] * sb;
    __syncthreads();
    if (step + 1 < steps) fetch(step + 1);
    const uint8_t *from = lds[step & 1];
    Operand<OUT> b[NT];
#pragma unroll
    for (int u = 0; u < NT; u++) b[u].from(fragment(from + (BM + wn + u * 16) * BLOCK));
#pragma unroll
    for (int t = 0; t < MT; t++) {
      Operand<OUT> a;
      a.from(fragment(from + (wm + t * 16) * BLOCK));
      v4f part[NT];
      products(part, b, a);
#pragma unroll
      for (int u = 0; u < NT; u++) acc[t][u] += part[u] * scale[t];
    }
  }
#pragma unroll
  for (int t = 0; t < MT; t++) {
    const uint32_t row = m0 + wm + t * 16 + li;
    if (row >= p.m) continue;
    OUT *out = (OUT *)p.out + int64_t(row) * p.out_s;
#pragma unroll
    for (int u = 0; u < NT; u++) {
      const uint32_t col = n0 + wn + u * 16 + lg * 4;
      store4(out + col, acc[t][u], int(p.n) - int(col));
    }
  }
}

constexpr uint32_t MOST_FEW_ANY = 32;
// ---- Few rows: 16 of b's rows to a workgroup, whose waves share K.  Memory bounds it, so that the products are in bf16 whatever the result's type. ----
template <int MT, int WAVES, class OUT>
__global__ __launch_bounds__(WAVES * 64) void k_product_few_any(ProductArgs p) {
  __shared__ v4f part[WAVES][MT][64];
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const uint32_t n0 = blockIdx.x * 16;
  const int steps = int((p.k + BLOCK - 1) / BLOCK), k = int(p.k);
  const uint8_t *b = p.b + int64_t(min(n0 + li, p.n - 1)) * p.b_s;
  const float *b_scale = p.b_scales + int64_t(n0 / BLOCK) * p.bs_s;
  const uint8_t *a[MT];
  const float *a_scale[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) {
    const int64_t row = min(uint32_t(t * 16 + li), p.m - 1);
    a[t] = p.a + row * p.a_s, a_scale[t] = p.a_scales + row * p.as_s;
  }
  v4f acc[MT] = {};
  auto thirty_two = [&](const uint8_t *row, int at) {
    const v4i lo = chunk_up_to(row + at, k - at, at), hi = chunk_up_to(row + at + 16, k - at - 16, at + 16);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  for (int step = wave; step < steps; step += WAVES) {
    const int at = step * int(BLOCK) + lg * 32;
    Operand<float> x[1], y;
    x[0].from(thirty_two(b, at));
    const float sb = b_scale[step];
#pragma unroll
    for (int t = 0; t < MT; t++) {
      v4f part[1];
      y.from(thirty_two(a[t], at));
      products(part, x, y);
      acc[t] += part[0] * (a_scale[t][step] * sb);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; t++) part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int x = threadIdx.x; x < MT * 64; x += WAVES * 64) {
    const uint32_t row = x / 64 * 16 + li, col = n0 + lg * 4;
    v4f sum = part[0][x / 64][lane];
#pragma unroll
    for (int w = 1; w < WAVES; w++) sum += part[w][x / 64][lane];
    if (row < p.m && col < p.n) store4((OUT *)p.out + int64_t(row) * p.out_s + col, sum, int(p.n - col));
  }
}

// What several workgroups have of the same sums, in their order.
template <class OUT>
__global__ __launch_bounds__(TILE_THREADS) void k_product_join(ProductArgs p, FastDiv by_fours) {
  const uint32_t at = blockIdx.x * TILE_THREADS + threadIdx.x, row = by_fours.div(at), col = (at - row * (p.parts_s / 4)) * 4;
  if (row >= p.m) return;
  const float *const from = p.parts + uint64_t(row) * p.parts_s + col;
  v4f sum = *(const v4f *)from;
  for (uint32_t z = 1; z < p.shares; z++) sum += *(const v4f *)(from + uint64_t(z) * p.m * p.parts_s);
  store4((OUT *)p.out + int64_t(row) * p.out_s + col, sum, int(p.n - col));
}
template <class OUT>
hipError_t launch_join(const ProductArgs &p, hipStream_t stream) {
  const uint32_t fours = p.parts_s / 4;
  plan::work(plan::UNIT_STREAM, 0, double(p.m) * p.n * (4.0 * p.shares + sizeof(OUT)));
  MRL_LAUNCH(k_product_join<OUT>, dim3((p.m * fours + TILE_THREADS - 1) / TILE_THREADS), dim3(TILE_THREADS), 0, stream, p, FastDiv(fours));
  return plan::last_error();
}

template <class OUT>
hipError_t launch(const ProductArgs &p, hipStream_t stream) {
  plan::work(plan::UNIT_MFMA_I8, 2.0 * p.m * double(p.n) * p.k, (double(p.m) + p.n) * p.k + double(p.m) * p.n * sizeof(OUT), 0, 0, sizeof(OUT) == 2 ? 1.4 : 0.7);
  if (rows_of_chunks(p.a, p.a_s, p.k) && rows_of_chunks(p.b, p.b_s, p.k) && p.as_s < (1 << 21)) {
    if (p.m <= MOST_FEW) return launch_product_few(p, stream);
    if (p.shares > 1) {
      const hipError_t e = launch_product_tile(p, stream);
      return e == hipSuccess ? launch_join<OUT>(p, stream) : e;
    }
    // Tiles of 256 x 256 where they make one round over the compute units and those of 128 x 128, of which a unit takes two at a time, more than one; in more rounds, and where rows of the result are off 16 bytes and cost the
    // larger tiles' stores, all at one time, more, where the last round is not too empty.  us, so and on the smaller ones: 2048 x 4096 x 4096 (128 tiles, 512 of the smaller) 54.3 and 48.7, 2304 x 4096 x 4096 (144, 576) 54.5 and 65.7,
    // 2304 x 4096 x 1040 23.6 and 25.0, 2944 x 2944 x 2048 (144, 529) 31.5 and 34.7, 130 x 40000 x 2048 (157, 626) 33.3 and 40.4, 4096 x 4096 x 512 (256) 17.6 and 18.9; off 16 bytes 2900 x 2950 x 1040 (144) 28.1 and 25.0, 3300 x 3300 x 1024 (169) 24.0 and 21.0,
    // 2304 x 4090 x 4096 57.1 and 64.3, 4000 x 4001 x 1040 (256) 26.3 and 32.1; two rounds 4608 x 4096 x 4096 (288) 111.6 and 106.1, 5120 x 4096 x 4096 (320) 111.9 and 112.5, 5632 x 4096 x 4096 (352) 112.8 and 126.
    const uint64_t wide = uint64_t((p.m + 255) / 256) * ((p.n + 255) / 256), small = uint64_t((p.m + 127) / 128) * ((p.n + 127) / 128), rounds = (wide + g_compute_units - 1) / g_compute_units;
    const bool few_rounds = rounds == 1 && p.out_s % 8 == 0 ? small > 2 * g_compute_units : wide * 100 >= 62 * rounds * g_compute_units;
    return sizeof(OUT) == 2 && few_rounds ? launch_product_wide(p, stream) : launch_product_tile(p, stream);
  }
  if (p.m <= 16) MRL_LAUNCH((k_product_few_any<1, 8, OUT>), dim3((p.n + 15) / 16), dim3(512), 0, stream, p);
  else if (p.m <= MOST_FEW_ANY) MRL_LAUNCH((k_product_few_any<2, 8, OUT>), dim3((p.n + 15) / 16), dim3(512), 0, stream, p);
  else {
    const uint32_t tiles_m = (p.m + 127) / 128, tiles_n = (p.n + 127) / 128;
    MRL_LAUNCH((k_product_tile_any<128, 128, OUT>), dim3(tiles_m * tiles_n), dim3(TILE_THREADS), 0, stream, p, tiles_m);
  }
  return plan::last_error();
}

// Operands whose rows are not whole 16-byte chunks are copied into ones that are, with zeros behind K, but for one or two rows and small products of few.  (us, with and without: 1 x 4095 x 4095 12.5 and 10.1,
// 4 12.4 and 13.1, 16 12.9 and 17.7, 33 13.7 and 48, 128 19 and 57; 1 x 16383 x 16383 150 and 124, 8 152 and 193; 16 x 1001 x 1001 4.9 and 4.0, 40 x 600 x 601 5.1 and 10.7; 1000 x 8191 x 2047 36 and 55.)
struct Copies {
  bool a = false, b = false;
  uint32_t ld = 0;
  size_t a_bytes = 0, b_bytes = 0;
};
Copies copies(const ProductArgs &p) {
  Copies c;
  if (p.m <= 2 || (p.m <= 16 && uint64_t(p.n) * p.k <= 1u << 21)) return c;
  c.a = p.k % 16 != 0 || p.a_s % 16 != 0, c.b = p.k % 16 != 0 || p.b_s % 16 != 0;
  c.ld = (p.k + 127) / 128 * 128;
  if (c.a) c.a_bytes = size_t(p.m) * c.ld;
  if (c.b) c.b_bytes = size_t(p.n) * c.ld;
  if (std::max(c.a_bytes, c.b_bytes) >= (size_t(1) << 34)) return Copies();   // (numbered in chunks of 16 bytes below 2^31)
  return c;
}
PadRows rows_of(const void *from, uint32_t rows, uint32_t k, int64_t stride, void *to, uint32_t ld) {
  PadRows r = {};
  r.src.ptr = const_cast<void *>(from), r.src.dtype = MRL_U8, r.src.rank = 3;
  r.src.shape[0] = 1, r.src.shape[1] = rows, r.src.shape[2] = k;
  r.src.stride[0] = 0, r.src.stride[1] = stride, r.src.stride[2] = 1;
  r.dst = to, r.dst_ld = ld, r.dst_rows = rows, r.elem_size = 1;
  return r;
}

}  // namespace

// Workgroups that share K, by sizes and strides alone.
uint32_t shares(const ProductArgs &p, const Copies &c) {
  const bool a = c.a || (p.k % 16 == 0 && p.a_s % 16 == 0), b = c.b || (p.k % 16 == 0 && p.b_s % 16 == 0);
  return p.m > MOST_FEW && a && b ? shares_of_tiles(p) : 1;
}

size_t product_workspace_bytes(const ProductArgs &p) {
  const Copies c = copies(p);
  const uint32_t z = shares(p, c);
  return c.a_bytes + c.b_bytes + (z > 1 ? sizeof(float) * z * p.m * ((p.n + 3) / 4 * 4) : 0);
}

hipError_t launch_product(const ProductArgs &given, hipStream_t stream) {
  ProductArgs p = given;
  const Copies c = copies(p);
  p.shares = shares(p, c), p.parts = (float *)(p.workspace + c.a_bytes + c.b_bytes), p.parts_s = (p.n + 3) / 4 * 4;
  // (an operand that keeps its rows has to have them at such addresses, too)
  auto aligned = [](const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if ((c.a || c.b) && (c.a || aligned(p.a)) && (c.b || aligned(p.b))) {
    const PadRows a = rows_of(p.a, p.m, p.k, p.a_s, p.workspace, c.ld), b = rows_of(p.b, p.n, p.k, p.b_s, p.workspace + c.a_bytes, c.ld);
    const hipError_t e = c.a && c.b ? launch_pad_rows_pair(a, b, stream) : launch_pad_rows(c.a ? a : b, stream);
    if (e != hipSuccess) return e;
    if (c.a) p.a = p.workspace, p.a_s = c.ld;
    if (c.b) p.b = p.workspace + c.a_bytes, p.b_s = c.ld;
    p.k = (p.k + 15) / 16 * 16;
  }
  return p.out_dtype == MRL_BF16 ? launch<uint16_t>(p, stream) : launch<float>(p, stream);
}

}  // namespace mrl
