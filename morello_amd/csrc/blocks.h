// Tensors in e4m3 with a scale for each block of 128, and layers of experts: what the host side (api.hip) hands to cast_blocks.hip, matmul_blocks.hip and experts.hip.
#pragma once
#include "kernels.h"

namespace mrl {

constexpr uint32_t BLOCK = 128;   // elements of a row that share a scale

struct CastArgs {
  const void *x;
  uint8_t *out;
  float *scales;
  uint32_t rows, cols, block_rows;
  int dtype;
  bool gated;
  int64_t x_s, out_s, scale_s;   // strides of a row in elements
};
hipError_t launch_cast_blocks(const CastArgs &a, hipStream_t stream);

struct ProductArgs {
  const uint8_t *a, *b;
  const float *a_scales, *b_scales;
  void *out;
  uint8_t *workspace;
  float *parts;         // [shares][m][parts_s], where several workgroups share K
  uint32_t m, n, k, shares, parts_s;
  int out_dtype;
  int64_t a_s, as_s, b_s, bs_s, out_s;   // strides of a row in elements (of a row of blocks for b's scales)
};
// By sizes, types and strides alone, without pointers.
size_t product_workspace_bytes(const ProductArgs &p);
hipError_t launch_product(const ProductArgs &p, hipStream_t stream);

// One of the three stacks of matrices of a layer of experts.
struct Stack {
  const uint8_t *w;
  const float *scales;                  // nullptr: bf16
  int64_t w_e, w_s, scales_e, scales_s;   // strides in elements: of an expert, of a row (of blocks)
};
struct ExpertsArgs {
  const uint16_t *x, *router;
  Stack gate, up, down;
  const int32_t *rows;                  // nullptr: all tokens
  uint16_t *out;
  int32_t *chosen;                      // nullptr: not wanted, like shares
  float *shares;
  uint8_t *workspace;
  uint32_t tokens, hidden, inter, experts, top_k;
  int weight_dtype;
  bool renormalise;
  int64_t x_s, out_s, router_s;
};
constexpr uint32_t MOST_TOKENS = 256, MOST_EXPERTS = 512, MOST_CHOSEN = 32, MOST_DIMS = 1u << 17;
size_t experts_workspace_bytes(const ExpertsArgs &a);
hipError_t launch_experts(const ExpertsArgs &a, hipStream_t stream);

}  // namespace mrl
