// The cache of keys and values in pages: what the host side (api.hip) hands to page_tables.hip, rotary.hip and the
// attention over pages (attention_paged*.hip).
#pragma once
#include "kernels.h"

namespace mrl {

namespace paged {
// Another lane's x, by DPP control CTRL and for the sixteens of lanes in ROWS; `none` where there is no such lane.
template <int CTRL, int ROWS>
__device__ inline int32_t moved(int32_t x, int32_t none) { return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false); }
// x over the lanes up to each, f(x, control, rows) being x with what is moved to it; all lanes take part.  (No trips through LDS, as shuffles make.)
template <class T, class F>
__device__ inline T over_lanes_up_to(T x, F f) {
  x = f(x, std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());   // row_shr 1, 2, 4, 8: within sixteens
  x = f(x, std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  x = f(x, std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  x = f(x, std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  x = f(x, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());   // row_bcast 15, 31: the last of a sixteen, of a half, to those behind
  return f(x, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
}
__device__ inline uint64_t sums_up_to(uint64_t x) {
  return over_lanes_up_to(x, [](uint64_t y, auto ctrl, auto rows) {
    const uint32_t lo = moved<ctrl(), rows()>(int32_t(uint32_t(y)), 0), hi = moved<ctrl(), rows()>(int32_t(uint32_t(y >> 32)), 0);
    return y + (uint64_t(hi) << 32 | lo);
  });
}
__device__ inline int32_t largest_up_to(int32_t x, int32_t least) {
  return over_lanes_up_to(x, [=](int32_t y, auto ctrl, auto rows) { return max(y, moved<ctrl(), rows()>(y, least)); });
}
}  // namespace paged

struct PageTablesArgs {
  const int32_t *cached, *added, *free_list, *free_count;
  int32_t *table, *starts, *lengths, *slots, *positions, *free_left;
  uint32_t requests, width, page_size, pages, tokens, free_pages;
};
hipError_t launch_page_tables(const PageTablesArgs &a, hipStream_t stream);

struct RotaryArgs {
  const void *q, *k, *v;
  const int32_t *positions;
  const float *frequencies;
  const int32_t *slots;
  void *q_out, *keys, *values;
  uint32_t tokens, q_heads, kv_heads, head_dim, pairs;
  uint32_t section_end[MRL_MAX_AXES];   // the pair behind each axis's last, `pairs` from the last axis on
  int dtype;
  bool adjacent, inverse;
  uint32_t page_size, slot_count;       // 0 and 0: dense keys
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h, key_p, key_s, key_h, val_p, val_s, val_h;   // strides in elements
};
hipError_t launch_rotary(const RotaryArgs &a, hipStream_t stream);

struct PagedAttnArgs {
  const void *q, *keys, *values;
  const int32_t *table, *starts, *lengths;
  void *out;
  uint8_t *workspace;
  uint32_t tokens, requests, q_heads, kv_heads, group, head_dim, page_size, pages, width, max_new, window;
  int dtype;
  float scale;
  int64_t q_t, q_h, o_t, o_h, key_p, key_s, key_h, val_p, val_s, val_h;   // strides in elements
};
// By sizes, types and strides alone, without pointers (a call whose pointers are not 16-byte aligned takes the generic kernel, which wants none).
size_t paged_attn_workspace_bytes(const PagedAttnArgs &a);
hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream);

}  // namespace mrl
