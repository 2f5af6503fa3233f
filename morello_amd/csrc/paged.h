// The cache of keys and values in pages: what the host side (api.hip) hands to page_tables.hip, rotary.hip and the
// attention over pages (attention_paged*.hip).
#pragma once
#include "kernels.h"

namespace mrl {

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
