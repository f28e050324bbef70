// 16-byte pieces of memory at any alignment (global memory takes unaligned
// vector accesses).
#pragma once

#include "common.h"

namespace tiler_pieces {

typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// A piece without its first `missing` (1 to 15) bytes: the rest moves to the
// front, zeros follow.
__device__ __forceinline__ u32x4 drop_bytes(u32x4 v, uint32_t missing) {
  uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
  if (missing >= 8u) {
    lo = hi >> (8u * (missing - 8u));
    hi = 0;
  } else {
    lo = lo >> (8u * missing) | hi << (64u - 8u * missing);
    hi >>= 8u * missing;
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// Sixteen bytes from `p` of which the first `valid` (at least 1) exist; the
// rest zero.  `start` is where the operand starts: a short piece is the end of
// the 16 bytes before its end, or, next to the operand's start, read by bytes.
__device__ __forceinline__ u32x4 guarded_piece(const uint8_t* p, uint32_t valid, const uint8_t* start) {
  if (valid >= 16u) return *reinterpret_cast<const u32x4_any*>(p);
  const uint32_t missing = 16u - valid;
  if ((uint64_t)(p - start) >= missing) return drop_bytes(*reinterpret_cast<const u32x4_any*>(p - missing), missing);
  uint64_t lo = 0, hi = 0;
#pragma unroll 1
  for (uint32_t e = valid; e-- > 0;) {
    hi = hi << 8 | lo >> 56;
    lo = lo << 8 | p[e];
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

}  // namespace tiler_pieces
