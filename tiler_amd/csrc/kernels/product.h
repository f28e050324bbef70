// The tile product behind the gated contraction, its gradients and the 8-bit
// contraction: D[i, j] = sum over the depth of A(i, .) B(j, .) on MFMA, for
// operands stored depth-contiguous ("row" layout, [i][depth]) or transposed
// ("column" layout, [depth][i]).
//
// A tile of an operand in LDS is one depth slice of 128 bytes (64 bf16, 128
// i8) over TILE rows, in its own layout, in 16-byte pieces:
// * row layout: TILE rows of 128 bytes; piece c of row r sits at
//   c ^ ((r >> 1) & 7), so the 16 rows of a fragment read cover all 64 banks.
//   A lane reads its fragment (16 bytes of one row) at once.
// * column layout (bf16): 64 depth rows of 2 TILE bytes; the 32-byte block c
//   (16 columns) of depth row d sits at c ^ f(d), f(d) = (d & 3) | (d >> 1 & 4):
//   a transposing read (ds_read_b64_tr_b16) of 16 lanes takes 32 bytes of 4
//   depth rows d, d + 1, d + 2, d + 3, its neighbour those of d + 8 ..., and f
//   spreads the eight over the banks.  Lane i of the 16 receives column i's
//   four elements; two such reads make the fragment.  No operand is ever
//   transposed in memory.
// Both layouts deal a lane the same depth elements, so they mix freely.
#pragma once

#include "common.h"

namespace tiler_product {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_bytes;
// 16 bytes at any byte address (global memory takes unaligned vector accesses)
typedef u32x4 u32x4_any __attribute__((aligned(1)));

constexpr uint32_t kSlice = 128;  // bytes of depth per tile

struct Bf16 {
  using Acc = f32x4;
  static constexpr uint32_t kBytes = 2;
  static __device__ __forceinline__ Acc zero() { return Acc{0.0f, 0.0f, 0.0f, 0.0f}; }
  static __device__ __forceinline__ Acc mfma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
};
struct I8 {
  using Acc = i32x4;
  static constexpr uint32_t kBytes = 1;
  static __device__ __forceinline__ Acc zero() { return Acc{0, 0, 0, 0}; }
  static __device__ __forceinline__ Acc mfma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

// Byte offset of 16-byte piece `id` of an operand tile in LDS, and which
// piece of the operand it is: (row, piece along the depth) in row layout,
// (depth row, 8-column piece) in column layout.
template <uint32_t TILE, bool kCol>
__device__ __forceinline__ uint32_t piece_offset(uint32_t outer, uint32_t inner) {
  if constexpr (kCol) return outer * (TILE * 2u) + (((inner >> 1) ^ ((outer & 3u) | ((outer >> 1) & 4u))) << 5) + ((inner & 1u) << 4);
  else return outer * kSlice + ((inner ^ ((outer >> 1) & 7u)) << 4);
}
template <uint32_t TILE, bool kCol>
struct Pieces {
  static constexpr uint32_t kPerOuter = kCol ? TILE / 8u : 8u;  // pieces of one row / depth row
  static constexpr uint32_t kCount = TILE * 8u;
};

// A lane's fragments of BLOCKS 16-row blocks starting at row `row0` of a tile.
template <uint32_t TILE, bool kCol, int BLOCKS>
struct Fragments {
  uint32_t at[kCol ? BLOCKS : 2];  // byte offsets in the tile
  __device__ __forceinline__ Fragments(uint32_t row0, uint32_t lane) {
    const uint32_t i = lane & 15u, g = lane >> 4;
    if constexpr (kCol) {
      const uint32_t f = (i >> 2) | ((g & 1u) << 2);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
        at[b] = (8u * g + (i >> 2)) * (TILE * 2u) + (((row0 / 16u + b) ^ f) << 5) + ((i & 3u) << 3);
    } else {
      const uint32_t swz = (i >> 1) & 7u;
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (row0 + i) * kSlice + (((uint32_t)s * 4u + g) ^ swz) * 16u;
    }
  }
  __device__ __forceinline__ void read(const uint8_t* tile, int step, u32x4 (&v)[BLOCKS]) const {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      if constexpr (kCol) {
        const uint8_t* p = tile + at[b] + (uint32_t)step * 32u * TILE * 2u;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4u * TILE * 2u));
        const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
        v[b] = u32x4{l.x, l.y, h.x, h.y};
      } else {
        v[b] = *reinterpret_cast<const u32x4*>(tile + at[step] + b * 16u * kSlice);
      }
    }
  }
};

// Sixteen bytes from `p` of which the first `valid` (at least 1) exist; the
// rest zero.  `start` is where the operand starts: a short piece is the end of
// the 16 bytes before its end, or, next to the operand's start, read by bytes.
__device__ __forceinline__ u32x4 guarded_piece(const uint8_t* p, uint32_t valid, const uint8_t* start) {
  if (valid >= 16u) return *reinterpret_cast<const u32x4_any*>(p);
  uint64_t lo = 0, hi = 0;
  const uint32_t missing = 16u - valid;
  if ((uint64_t)(p - start) >= missing) {
    const u32x4 v = *reinterpret_cast<const u32x4_any*>(p - missing);
    lo = (uint64_t)v.y << 32 | v.x;
    hi = (uint64_t)v.w << 32 | v.z;
    if (missing >= 8u) {
      lo = hi >> (8u * (missing - 8u));
      hi = 0;
    } else {
      lo = lo >> (8u * missing) | hi << (64u - 8u * missing);
      hi >>= 8u * missing;
    }
  } else {
#pragma unroll 1
    for (uint32_t e = valid; e-- > 0;) {
      hi = hi << 8 | lo >> 56;
      lo = lo << 8 | p[e];
    }
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// An operand in memory: `rows` indices of the result, `depth` contracted ones,
// `ld` elements between consecutive rows (row layout) or depth rows (column).
struct Operand {
  const uint8_t* base;
  uint64_t ld;
  uint32_t rows, depth;
};

// Piece (outer, inner) of the tile at (row0, depth0), zero outside the operand.
template <typename E, bool kCol>
__device__ __forceinline__ u32x4 operand_piece(const Operand& o, uint32_t row0, uint32_t depth0, uint32_t outer,
                                               uint32_t inner) {
  constexpr uint32_t kPer = 16u / E::kBytes;
  const uint32_t major = (kCol ? depth0 : row0) + outer, major_end = kCol ? o.depth : o.rows;
  const uint32_t minor = (kCol ? row0 : depth0) + inner * kPer, minor_end = kCol ? o.rows : o.depth;
  if (major >= major_end || minor >= minor_end) return u32x4{0, 0, 0, 0};
  const uint64_t left = (uint64_t)(minor_end - minor) * E::kBytes;
  return guarded_piece(o.base + (major * o.ld + minor) * E::kBytes, left < 16u ? (uint32_t)left : 16u, o.base);
}

// The guarded product, for any sizes and alignments: pieces come through
// registers (zero outside the operand), one slice ahead of the products.
// WM x WN waves of MB x NB blocks of 16 x 16; piece_a(t, outer, inner) and
// piece_b fetch a piece of slice t.
template <typename E, bool kACol, bool kBCol, int WM, int WN, int MB, int NB, typename FA, typename FB>
__device__ __forceinline__ void guarded_product(uint8_t* smem, uint32_t slices, FA piece_a, FB piece_b,
                                                typename E::Acc (&acc)[MB][NB]) {
  constexpr uint32_t kThreads = 64u * WM * WN, kRowsA = WM * MB * 16u, kRowsB = WN * NB * 16u;
  constexpr uint32_t kLoadsA = kRowsA * 8u / kThreads, kLoadsB = kRowsB * 8u / kThreads;
  constexpr uint32_t kStage = (kRowsA + kRowsB) * kSlice;
  static_assert(kRowsA * 8u % kThreads == 0 && kRowsB * 8u % kThreads == 0, "whole pieces per thread");
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const Fragments<kRowsA, kACol, MB> ra((wave / WN) * MB * 16u, lane);
  const Fragments<kRowsB, kBCol, NB> rb((wave % WN) * NB * 16u, lane);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = E::zero();
  u32x4 pa[kLoadsA], pb[kLoadsB];
  constexpr uint32_t kOuterA = Pieces<kRowsA, kACol>::kPerOuter, kOuterB = Pieces<kRowsB, kBCol>::kPerOuter;
  auto load = [&](uint32_t t) {
#pragma unroll
    for (uint32_t q = 0; q < kLoadsA; ++q) {
      const uint32_t id = threadIdx.x + q * kThreads;
      pa[q] = piece_a(t, id / kOuterA, id % kOuterA);
    }
#pragma unroll
    for (uint32_t q = 0; q < kLoadsB; ++q) {
      const uint32_t id = threadIdx.x + q * kThreads;
      pb[q] = piece_b(t, id / kOuterB, id % kOuterB);
    }
  };
  auto store = [&](uint32_t stage) {
    uint8_t* at = smem + stage * kStage;
#pragma unroll
    for (uint32_t q = 0; q < kLoadsA; ++q) {
      const uint32_t id = threadIdx.x + q * kThreads;
      *reinterpret_cast<u32x4*>(at + piece_offset<kRowsA, kACol>(id / kOuterA, id % kOuterA)) = pa[q];
    }
#pragma unroll
    for (uint32_t q = 0; q < kLoadsB; ++q) {
      const uint32_t id = threadIdx.x + q * kThreads;
      *reinterpret_cast<u32x4*>(at + kRowsA * kSlice + piece_offset<kRowsB, kBCol>(id / kOuterB, id % kOuterB)) = pb[q];
    }
  };
  load(0);
  store(0);
  __syncthreads();
  for (uint32_t t = 0; t < slices; ++t) {
    if (t + 1 < slices) load(t + 1);
    const uint8_t* at = smem + (t & 1u) * kStage;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[MB], fb[NB];
      ra.read(at, s, fa);
      rb.read(at + kRowsA * kSlice, s, fb);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = E::mfma(fa[i], fb[j], acc[i][j]);
    }
    if (t + 1 < slices) store((t & 1u) ^ 1u);
    __syncthreads();
  }
}

}  // namespace tiler_product
