// Rows of bf16 or f32 -> e4m3 with a scale for each block of 128, or of 128 x 128.
//
// With a the largest size in a block, at least 2^-110: scale = a / 448 (448 is e4m3's largest number), values x (448 / a), rounded to nearest
// even; both quotients are correctly rounded divisions in 32 bits, so that the same tensor gives the same bytes anywhere.  2^-110 keeps
// 448 / a within 32 bits.  A NaN is a NaN again; an infinity has the scale infinity, under which the block's other numbers are 0 (0 times infinity: they read
// back as NaN).
//
// Memory bounds it: 4101 x 8192 in bf16 behind a gate 30 us (169 MB, 5.6 TB/s; a copy of 1 GiB reaches 5.1), 8100 x 4110 in f32 in blocks of 128 x 128 36 us (166 MB, 4.6 TB/s).
#include "blocks_device.h"

namespace mrl {
namespace {
using namespace blocks;

constexpr float LEAST = 0x1p-110f, LARGEST = 448.0f;
constexpr int THREADS = 256;

__device__ inline float to_f32(uint16_t x) { return __uint_as_float(uint32_t(x) << 16); }
__device__ inline float to_f32(float x) { return x; }

struct Eight { float x[8]; };
// Elements col .. col + 7 of a row of `cols`, zeros behind its end.
template <class T>
__device__ inline Eight eight_at(const T *row, uint32_t col, uint32_t cols) {
  Eight e;
  if (col + 8 <= cols) {
    const uint8_t *p = (const uint8_t *)(row + col);
    if constexpr (sizeof(T) == 2) {
      const v4i u = chunk_at(p);
#pragma unroll
      for (int i = 0; i < 4; i++) e.x[2 * i] = __uint_as_float(uint32_t(u[i]) << 16), e.x[2 * i + 1] = __uint_as_float(uint32_t(u[i]) & 0xffff0000u);
    } else {
      const v4i u = chunk_at(p), w = chunk_at(p + 16);
#pragma unroll
      for (int i = 0; i < 4; i++) e.x[i] = __int_as_float(u[i]), e.x[4 + i] = __int_as_float(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) e.x[i] = col + i < cols ? to_f32(row[col + i]) : 0.0f;
  }
  return e;
}
// silu(gate) * up, in some ten instructions where the library's exponential and division take forty, which would bound the kernel: exp(-g) = 2^t with t = -g log2 e in two parts, of which the
// small one joins behind the exponential; good to 3e-7 like those (rms 5.6e-8 and 4.9e-8).
__device__ inline float gated(float g, float u) {
  constexpr float L = 1.44269504088896340736f, L_REST = 1.925963033500893e-08f /* log2 e - L */, LN2 = 0.69314718055994530942f, OVERFLOWS = -88.5f;
  const float x = __builtin_amdgcn_fmed3f(g, OVERFLOWS, 100.0f), t = x * -L;
  const float rest = __builtin_fmaf(x, -L_REST, __builtin_fmaf(x, -L, -t)), e = __builtin_amdgcn_exp2f(t);
  const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, rest * LN2, e));
  return g * (g < OVERFLOWS ? 0.0f : r) * u;
}
__device__ inline Eight gated(const Eight &g, const Eight &u) {
  Eight e;
#pragma unroll
  for (int i = 0; i < 8; i++) e.x[i] = gated(g.x[i], u.x[i]);
  return e;
}
__device__ inline float largest(const Eight &e) {
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) a = fmaxf(a, fabsf(e.x[i]));
  return a;
}
__device__ inline void store_eight(uint8_t *row, uint32_t col, uint32_t cols, const Eight &e, float factor) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float *x = e.x + 4 * i;
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * factor, x[1] * factor, 0, false);
    w[i] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * factor, x[3] * factor, lo, true));
  }
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  typedef v2u v2u_any __attribute__((aligned(1)));
  if (col + 8 <= cols) {
    *(v2u_any *)(row + col) = v2u{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (col + i < cols) row[col + i] = uint8_t(w[i / 4] >> (i % 4 * 8));
  }
}
template <int CTRL>
__device__ inline float moved(float x) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)); }
// Over the sixteen lanes that a lane is one of: rotations by 8, 4, 2, 1.
__device__ inline float largest_of_16(float x) {
  x = fmaxf(x, moved<0x128>(x));
  x = fmaxf(x, moved<0x124>(x));
  x = fmaxf(x, moved<0x122>(x));
  return fmaxf(x, moved<0x121>(x));
}

// A block of a row to sixteen lanes, eight elements each.
template <class T, bool GATED>
__global__ __launch_bounds__(THREADS) void k_cast_rows(CastArgs p, uint32_t blocks, FastDiv by_blocks) {
  const uint32_t at = (blockIdx.x * THREADS + threadIdx.x) / 16;   // (below 2^31)
  const uint32_t row = by_blocks.div(at), block = at - row * blocks;
  if (row >= p.rows) return;
  const uint32_t col = block * BLOCK + threadIdx.x % 16 * 8;
  const T *x = (const T *)p.x + int64_t(row) * p.x_s;
  Eight e = eight_at(x, col, p.cols);
  if constexpr (GATED) e = gated(e, eight_at(x + p.cols, col, p.cols));
  const float a = fmaxf(largest_of_16(largest(e)), LEAST);
  if (threadIdx.x % 16 == 0) p.scales[int64_t(row) * p.scale_s + block] = a / LARGEST;
  store_eight(p.out + int64_t(row) * p.out_s, col, p.cols, e, LARGEST / a);
}

// 128 rows of 128 elements to a workgroup, sixteen lanes to a row, kept in registers between the two passes.  (us, 256 and 512 threads: 8192 x 4096 in f32 34.5 and 33.8, in bf16 23.7 and 25.8.)
template <class T, bool GATED, int THREADS>
__global__ __launch_bounds__(THREADS) void k_cast_squares(CastArgs p, uint32_t blocks, FastDiv by_blocks) {
  __shared__ float of_wave[THREADS / 64];
  constexpr int EACH = BLOCK / (THREADS / 16);
  const uint32_t at = xcd_run(blockIdx.x, gridDim.x);   // (blocks whose rows share cache lines, of an XCD)
  const uint32_t block_row = by_blocks.div(at), block = at - block_row * blocks;
  const uint32_t row0 = block_row * BLOCK + threadIdx.x / 16, col = block * BLOCK + threadIdx.x % 16 * 8;
  Eight e[EACH];
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t row = row0 + i * (THREADS / 16);
    if (row < p.rows) {
      const T *x = (const T *)p.x + int64_t(row) * p.x_s;
      e[i] = eight_at(x, col, p.cols);
      if constexpr (GATED) e[i] = gated(e[i], eight_at(x + p.cols, col, p.cols));
      a = fmaxf(a, largest(e[i]));
    }
  }
  a = largest_of_16(a);
  a = fmaxf(a, __shfl_xor(a, 16));
  a = fmaxf(a, __shfl_xor(a, 32));
  if (threadIdx.x % 64 == 0) of_wave[threadIdx.x / 64] = a;
  __syncthreads();
  a = LEAST;
#pragma unroll
  for (int w = 0; w < THREADS / 64; w++) a = fmaxf(a, of_wave[w]);
  if (threadIdx.x == 0) p.scales[int64_t(block_row) * p.scale_s + block] = a / LARGEST;
  const float factor = LARGEST / a;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t row = row0 + i * (THREADS / 16);
    if (row < p.rows) store_eight(p.out + int64_t(row) * p.out_s, col, p.cols, e[i], factor);
  }
}

template <class T, bool GATED>
hipError_t launch(const CastArgs &a, hipStream_t stream) {
  const uint32_t blocks = (a.cols + BLOCK - 1) / BLOCK;
  const double elements = double(a.rows) * a.cols;
  plan::work(plan::UNIT_STREAM, 0, elements * (1 + sizeof(T) * (GATED ? 2 : 1)) + 4.0 * blocks * ((a.rows + a.block_rows - 1) / a.block_rows));
  if (a.block_rows == 1) {
    MRL_LAUNCH((k_cast_rows<T, GATED>), dim3(uint32_t((uint64_t(a.rows) * blocks + THREADS / 16 - 1) / (THREADS / 16))), dim3(THREADS), 0, stream, a, blocks, FastDiv(blocks));
  } else {
    constexpr int SQUARE = sizeof(T) == 4 ? 512 : 256;
    MRL_LAUNCH((k_cast_squares<T, GATED, SQUARE>), dim3(blocks * ((a.rows + BLOCK - 1) / BLOCK)), dim3(SQUARE), 0, stream, a, blocks, FastDiv(blocks));
  }
  return plan::last_error();
}

}  // namespace

hipError_t launch_cast_blocks(const CastArgs &a, hipStream_t stream) {
  if (a.dtype == MRL_BF16) return a.gated ? launch<uint16_t, true>(a, stream) : launch<uint16_t, false>(a, stream);
  return a.gated ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
}

}  // namespace mrl
