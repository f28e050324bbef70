// What the planner hands the head norm and rotation kernels by value (plain
// fields at their natural alignment; the host packs the same struct).
#pragma once

#include <stdint.h>

struct TilerHeads {
  uint64_t tokens;
  uint32_t q_heads, kv_heads, head_dim, rotary;
  uint32_t neighbours;  // pairs (2 p, 2 p + 1), else (p, p + rotary / 2)
  uint32_t norm;        // 0: no norm
  float eps;
  uint32_t page;        // of the cache; 0: none
  uint32_t each;        // tokens that a workgroup takes at a time (the forms in units)
  uint32_t q_groups;    // workgroups of the queries' gradients, the first ones
  uint64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements from token to token
  uint64_t slots, page_stride, token_stride, head_stride;             // the cache: pages * page, elements
};
