// What the planner hands the attention sublayer's kernels by value, and the
// division of a key's position by the page size.  Plain fields at their natural
// alignment: the host packs the same struct (runtime/attention.cpp).
#pragma once

#include <stdint.h>

// n / d for n below 2^31 and d from 1 to 2^31: (mulhi(n, multiplier) + n) >> shift.
struct TilerDivisor {
  uint32_t divisor, multiplier, shift;
};

struct TilerAttentionShape {
  uint32_t tokens, sequences, kv_heads, group;  // group: query heads a key/value head
  uint32_t head_dim, pages, width, splits;      // width: pages a row of the table
  uint32_t window, sinks;
  float scale;                                  // of the logits, times log2(e)
  TilerDivisor page, groups;
  uint32_t page_stride, token_stride;           // of the cache, elements; a page's tokens span less than 2^32
  uint32_t whole;                               // of the tiles: the first workgroups, which take all keys; the others' keys are split
  uint64_t q_stride, out_stride;                // elements from token to token
  uint64_t head_stride;
};
