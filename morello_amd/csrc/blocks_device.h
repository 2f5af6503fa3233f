// Loads of rows that begin on any byte and end inside a step, and the matrix instructions on them (matmul_blocks.hip, experts.hip).
#pragma once
#include "blocks.h"

namespace mrl {
namespace blocks {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
// On any byte: the memory path takes such addresses for vector accesses.
typedef v4i v4i_any __attribute__((aligned(1)));
typedef v4f v4f_any __attribute__((aligned(4)));
typedef v4bf v4bf_any __attribute__((aligned(2)));

// What lanes of a wave have written to LDS is there for its others, and what they have read may be written over: a wave's LDS accesses complete in order, and this keeps the compiler from changing theirs.
__device__ inline void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

__device__ inline v4i chunk_at(const uint8_t *p) { return *(const v4i_any *)p; }
// A row's last sixteen bytes moved down to where its last n of them belong, zeros behind them (n: 0 or less: zeros; 16 and more: as they are).
__device__ inline v4i last_of_row(v4i x, int n) {
  typedef unsigned __int128 u128;
  return n >= 16 ? x : n <= 0 ? v4i{0, 0, 0, 0} : __builtin_bit_cast(v4i, __builtin_bit_cast(u128, x) >> ((16 - n) * 8));
}
// The first n bytes of sixteen, zeros behind them (n may be negative, or more); `before`: bytes of the same row in front of p.
__device__ inline v4i chunk_up_to(const uint8_t *p, int n, int before) {
  if (n >= 16) return chunk_at(p);
  v4i x = {0, 0, 0, 0};
  if (n <= 0) return x;
  if (n + before >= 16) return last_of_row(chunk_at(p + n - 16), n);
#pragma unroll
  for (int d = 0; d < 4; d++)
    for (int i = 0; i < 4 && d * 4 + i < n; i++) x[d] |= int(uint32_t(p[d * 4 + i]) << (i * 8));
  return x;
}

template <class T>
__device__ inline void store4(T *to, v4f x, int n) {   // the first n of four
  if constexpr (sizeof(T) == 2) {
    if (n >= 4) { *(v4bf_any *)to = v4bf{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]}; return; }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) to[i] = __builtin_bit_cast(uint16_t, (__bf16)x[i]);
  } else {
    if (n >= 4) { *(v4f_any *)to = x; return; }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) to[i] = x[i];
  }
}

// 16 x 16 sums over 128 products of e4m3: lane l gives a's and b's row l % 16, thirty-two elements of the l / 16-th quarter (which ones does not
// matter as long as a and b have the same), and gets rows 4 (l / 16) .. + 3 of a against row l % 16 of b.  The instruction cuts products at some 2^-13 of the
// largest among its 128 (measured: 2^-12.2 of it off at worst on normal data, 1.5e-5 of the result in the mean); on the same numbers in bf16 the instructions keep 32 bits (8.5e-9).
__device__ inline v4f mma_e4m3(v8i a, v8i b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ inline v4f mma_bf16(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// Four e4m3 numbers as bf16, which holds them all.
__device__ inline void widen4(int x, int &lo, int &hi) {
  lo = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
  hi = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true));
}
// A lane's thirty-two elements in bf16, eight to an instruction.
struct Wide { v4i x[4]; };
__device__ inline Wide widen(v8i q) {
  Wide w;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    int u[4];
    widen4(q[2 * i], u[0], u[1]);
    widen4(q[2 * i + 1], u[2], u[3]);
    w.x[i] = v4i{u[0], u[1], u[2], u[3]};
  }
  return w;
}
}  // namespace blocks
}  // namespace mrl
