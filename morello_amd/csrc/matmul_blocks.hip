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
__global__ __launch_bounds__(TILE_THREADS) void k_product_tile(ProductArgs p, uint32_t tiles_m) {
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
#pragma unroll
      for (int u = 0; u < NT; u++) acc[t][u] += b[u].by(a) * scale[t];
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
    const Wide x = widen(thirty_two(b, at));
    const float sb = b_scale[step];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] += mma_wide(x, widen(thirty_two(a[t], at))) * (a_scale[t][step] * sb);
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

template <class OUT>
hipError_t launch(const ProductArgs &p, hipStream_t stream) {
  const double ops = 2.0 * p.m * double(p.n) * p.k, bytes = (double(p.m) + p.n) * p.k + double(p.m) * p.n * sizeof(OUT);
  plan::work(plan::UNIT_MFMA_I8, ops, bytes);
  const bool chunks = rows_of_chunks(p.a, p.a_s, p.k) && rows_of_chunks(p.b, p.b_s, p.k);
  if (chunks && p.m <= MOST_FEW && p.as_s < (1 << 21)) return launch_product_few(p, stream);
  if (p.m <= 16) MRL_LAUNCH((k_product_few_any<1, 8, OUT>), dim3((p.n + 15) / 16), dim3(512), 0, stream, p);
  else if (p.m <= 32) MRL_LAUNCH((k_product_few_any<2, 8, OUT>), dim3((p.n + 15) / 16), dim3(512), 0, stream, p);
  else if (sizeof(OUT) == 2 && p.m > 512 && p.n > 512 && chunks) return launch_product_wide(p, stream);
  else {
    const uint32_t tiles_m = (p.m + 127) / 128, tiles_n = (p.n + 127) / 128;
    MRL_LAUNCH((k_product_tile<128, 128, OUT>), dim3(tiles_m * tiles_n), dim3(TILE_THREADS), 0, stream, p, tiles_m);
  }
  return plan::last_error();
}

}  // namespace

size_t product_workspace_bytes(const ProductArgs &) { return 0; }

hipError_t launch_product(const ProductArgs &p, hipStream_t stream) { return p.out_dtype == MRL_BF16 ? launch<uint16_t>(p, stream) : launch<float>(p, stream); }

}  // namespace mrl
