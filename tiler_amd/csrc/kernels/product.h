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

#include "pieces.h"

namespace tiler_product {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_bytes;
using tiler_pieces::guarded_piece;
using tiler_pieces::u32x4_any;

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

// Byte offset of a row's 16-byte piece in a row-layout tile.
__device__ __forceinline__ uint32_t piece_offset(uint32_t row, uint32_t piece) {
  return row * kSlice + ((piece ^ ((row >> 1) & 7u)) << 4);
}

// f(d) changes the places of at most eight blocks, four in a tile of 64.
template <uint32_t TILE>
constexpr uint32_t kBlockMask = TILE / 16u < 8u ? TILE / 16u - 1u : 7u;

// A lane's fragments of BLOCKS 16-row blocks starting at row `row0` of a tile.
template <uint32_t TILE, bool kCol, int BLOCKS>
struct Fragments {
  uint32_t at[kCol ? BLOCKS : 2];  // byte offsets in the tile
  __device__ __forceinline__ Fragments(uint32_t row0, uint32_t lane) {
    const uint32_t i = lane & 15u, g = lane >> 4;
    if constexpr (kCol) {
      const uint32_t f = ((i >> 2) | ((g & 1u) << 2)) & kBlockMask<TILE>;
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

// A row-layout operand in memory: `rows` rows of `depth` elements, one after
// another.
struct Operand {
  const uint8_t* base;
  uint32_t rows, depth;
};

// The guarded product, for any sizes and alignments: pieces come through
// registers, two slices ahead of the products.  A loader's load is free of
// branches, so that nothing waits between the loads: a piece that would pass
// its row's end is the last whole one inside it, a row past the last is the last
// one again.  store puts the pieces into LDS and, in the last slice, moves their
// elements into place and clears what lies past the depth; rows past the last
// only reach results that are not stored.
template <typename E, uint32_t TILE, uint32_t THREADS>
struct GuardedLoader {
  static constexpr uint32_t kLoads = TILE * 8u / THREADS;
  static_assert(TILE * 8u % THREADS == 0, "whole pieces per thread");
  Operand o;
  uint32_t row0, row_bytes;
  __device__ __forceinline__ GuardedLoader(const Operand& o_, uint32_t row0_)
      : o(o_), row0(row0_), row_bytes(o_.depth * E::kBytes) {}
  // `base`: the operand's storage (either weight's, in the gated product).
  __device__ __forceinline__ void load(const uint8_t* base, uint32_t t, u32x4 (&v)[kLoads]) const {
    const uint8_t* from = base + (uint64_t)row0 * row_bytes;
    const uint32_t last = o.rows - 1u - row0, in_last = row_bytes - 16u;
#pragma unroll
    for (uint32_t q = 0; q < kLoads; ++q) {
      const uint32_t id = threadIdx.x + q * THREADS, row = id / 8u, in = t * kSlice + id % 8u * 16u;
      v[q] = *reinterpret_cast<const u32x4_any*>(from + (row < last ? row : last) * row_bytes + (in < in_last ? in : in_last));
    }
  }
  __device__ __forceinline__ void store(uint32_t t, uint8_t* tile, u32x4 (&v)[kLoads]) const {
    const bool cut = (t + 1u) * kSlice > row_bytes;
#pragma unroll
    for (uint32_t q = 0; q < kLoads; ++q) {
      const uint32_t id = threadIdx.x + q * THREADS;
      if (cut) {
        const uint32_t end = t * kSlice + id % 8u * 16u + 16u;
        if (end > row_bytes) v[q] = end - row_bytes >= 16u ? u32x4{0, 0, 0, 0} : tiler_pieces::drop_bytes(v[q], end - row_bytes);
      }
      *reinterpret_cast<u32x4*>(tile + piece_offset(id / 8u, id % 8u)) = v[q];
    }
  }
};
// The same for rows of less than a piece (one slice): checked piece by piece.
template <typename E, uint32_t TILE, uint32_t THREADS>
struct TinyLoader {
  static constexpr uint32_t kLoads = TILE * 8u / THREADS;
  Operand o;
  uint32_t row0;
  __device__ __forceinline__ TinyLoader(const Operand& o_, uint32_t row0_) : o(o_), row0(row0_) {}
  __device__ __forceinline__ void load(const uint8_t* base, uint32_t, u32x4 (&v)[kLoads]) const {
    const uint32_t bytes = o.depth * E::kBytes;
#pragma unroll 1
    for (uint32_t q = 0; q < kLoads; ++q) {
      const uint32_t id = threadIdx.x + q * THREADS, row = row0 + id / 8u;
      u32x4 p = {0, 0, 0, 0};
      if (row < o.rows && id % 8u == 0) p = guarded_piece(base + (uint64_t)row * bytes, bytes, base);
#pragma unroll
      for (uint32_t x = 0; x < kLoads; ++x)
        if (x == q) v[x] = p;
    }
  }
  __device__ __forceinline__ void store(uint32_t, uint8_t* tile, const u32x4 (&v)[kLoads]) const {
#pragma unroll
    for (uint32_t q = 0; q < kLoads; ++q) {
      const uint32_t id = threadIdx.x + q * THREADS;
      *reinterpret_cast<u32x4*>(tile + piece_offset(id / 8u, id % 8u)) = v[q];
    }
  }
};

// load_a(t, pieces) and load_b fetch a slice, store_a(t, tile, pieces) and
// store_b put it into LDS; WM x WN waves of MB x NB blocks of 16 x 16.
template <typename E, int WM, int WN, int MB, int NB, typename LA, typename LB, typename SA, typename SB>
__device__ __forceinline__ void guarded_product(uint8_t* smem, uint32_t slices, LA load_a, LB load_b, SA store_a,
                                                SB store_b, typename E::Acc (&acc)[MB][NB]) {
  constexpr uint32_t kThreads = 64u * WM * WN, kRowsA = WM * MB * 16u, kRowsB = WN * NB * 16u;
  constexpr uint32_t kLoadsA = kRowsA * 8u / kThreads, kLoadsB = kRowsB * 8u / kThreads;
  constexpr uint32_t kStage = (kRowsA + kRowsB) * kSlice;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const Fragments<kRowsA, false, MB> ra((wave / WN) * MB * 16u, lane);
  const Fragments<kRowsB, false, NB> rb((wave % WN) * NB * 16u, lane);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = E::zero();
  u32x4 pa[2][kLoadsA], pb[2][kLoadsB];
  auto load = [&](uint32_t t, auto slot) {
    load_a(t, pa[decltype(slot)::value]);
    load_b(t, pb[decltype(slot)::value]);
  };
  auto store = [&](uint32_t t, auto slot) {
    uint8_t* at = smem + (t & 1u) * kStage;
    store_a(t, at, pa[decltype(slot)::value]);
    store_b(t, at + kRowsA * kSlice, pb[decltype(slot)::value]);
  };
  auto multiply = [&](uint32_t t) {
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
  };
  // Slice t in LDS, slice t + 1 in registers (slot (t + 1) % 2): requests slice
  // t + 2, multiplies slice t, puts slice t + 1 into LDS.  Two turns a round
  // without a condition in them, so that a wait counts only the loads before it.
  auto turn = [&](uint32_t t, auto next, auto after) {
    load(t + 2 < slices ? t + 2 : slices - 1, after);
    __builtin_amdgcn_sched_barrier(0);
    multiply(t);
    store(t + 1, next);
    __syncthreads();
  };
  constexpr tiler::Step<0> even{};
  constexpr tiler::Step<1> odd{};
  load(0, even);
  load(slices > 1 ? 1 : 0, odd);
  store(0, even);
  __syncthreads();
  uint32_t t = 0;
  for (; t + 2 < slices; t += 2) {
    turn(t, odd, even);
    turn(t + 1, even, odd);
  }
  multiply(t);
  if (t + 1 < slices) {
    store(t + 1, odd);
    __syncthreads();
    multiply(t + 1);
  }
  __syncthreads();  // the caller may use the LDS
}

// ---------------------------------------------------------------------------
// The staged product: pieces move global -> LDS with buffer_load_dwordx4 ...
// lds, S slices in LDS, for operands whose rows (depth rows, in column
// layout) start on 16 bytes.
//
// A loader issues its wave's share of one slice of one operand.  The buffer
// resource starts at the slice (64-bit scalar arithmetic, so an operand may
// have any size; a tile's own span stays below 2^31 bytes) and ends with the
// operand, so what lies past the last row, or past the last depth row of a
// column operand, loads as zeros; pieces past the depth of a row operand,
// which lie in the next row, are sent past the resource's end instead.
// Columns past the last of a column operand load whatever follows: they only
// reach results that are not stored.
constexpr uint32_t kPastEnd = 0x80000000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
}

// TILE rows from `base`, `rows` of them real; `wave_rows` where this wave's
// LOADS * 8 rows start in memory and `wave_lds` where they go in the tile (the
// gated product's weights interleave two matrices).  Where the waves' rows are
// more than the tile's, the loads past it bring zeros to `spare` (1024 bytes),
// so that every wave counts the same loads.
template <typename E, int LOADS, uint32_t TILE = ~0u>
struct RowLoader {
  const uint8_t* base;
  uint32_t span, depth_bytes, lds0;
  uint8_t* spare;
  uint32_t voff[LOADS], piece[2];
  __device__ __forceinline__ RowLoader(const uint8_t* base_, uint64_t ld, uint32_t rows, uint32_t depth,
                                       uint32_t wave_rows, uint32_t wave_lds, uint32_t lane, uint8_t* spare_ = nullptr)
      : base(base_), span((uint32_t)(rows * ld * E::kBytes)), depth_bytes(depth * E::kBytes), lds0(wave_lds * kSlice),
        spare(spare_) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint32_t in = (lane & 7u) ^ (((wave_lds + j * 8u + (lane >> 3)) >> 1) & 7u);
      if (j < 2) piece[j] = in * 16u;
      voff[j] = past(j) ? kPastEnd : (wave_rows + j * 8u + (lane >> 3)) * (uint32_t)(ld * E::kBytes) + in * 16u;
    }
  }
  __device__ __forceinline__ bool past(int j) const { return TILE != ~0u && lds0 + j * 1024u >= TILE * kSlice; }
  __device__ __forceinline__ lds_bytes* place(uint8_t* tile, int j) const {
    return (lds_bytes*)(past(j) ? spare : tile + lds0 + j * 1024u);
  }
  __device__ __forceinline__ void issue(uint32_t t, uint8_t* tile) const { issue(base, t, tile); }
  __device__ __forceinline__ void issue(const uint8_t* from, uint32_t t, uint8_t* tile) const {
    const uint32_t at = t * kSlice, left = depth_bytes - at;
    const __amdgpu_buffer_rsrc_t panel = resource(from + at, span - at);
    if (left >= kSlice) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(panel, place(tile, j), 16, voff[j], 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(panel, place(tile, j), 16,
                                                 piece[j & 1] < left ? voff[j] : kPastEnd, 0, 0, 0);
    }
  }
};

// A slice of 64 depth rows of TILE columns (bf16) from `base`, which points at
// the tile's first column of depth row 0; `before` columns of the row lie
// before it.
template <uint32_t TILE, int LOADS>
struct ColumnLoader {
  const uint8_t* base;
  uint64_t row_bytes;
  uint32_t depth, before_bytes, lds0;
  uint32_t voff[LOADS];
  __device__ __forceinline__ ColumnLoader(const uint8_t* base_, uint64_t ld, uint32_t before, uint32_t depth_,
                                          uint32_t wave, uint32_t lane)
      : base(base_), row_bytes(ld * 2u), depth(depth_), before_bytes(before * 2u), lds0(wave * LOADS * 1024u) {
    constexpr uint32_t kPer = TILE / 8u;
    static_assert(TILE >= 64 && (TILE & (TILE - 1u)) == 0, "blocks of a row change places");
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint32_t id = (wave * LOADS + j) * 64u + lane, outer = id / kPer, slot = id % kPer;
      const uint32_t block = (slot >> 1) ^ (((outer & 3u) | ((outer >> 1) & 4u)) & kBlockMask<TILE>);
      voff[j] = outer * (uint32_t)row_bytes + block * 32u + (slot & 1u) * 16u;
    }
  }
  __device__ __forceinline__ void issue(uint32_t t, uint8_t* tile) const { issue(base, t, tile); }
  __device__ __forceinline__ void issue(const uint8_t* from, uint32_t t, uint8_t* tile) const {
    const uint32_t left = depth - t * 64u, rows = left < 64u ? left : 64u;
    const __amdgpu_buffer_rsrc_t panel =
        resource(from + t * 64u * row_bytes, rows * (uint32_t)row_bytes - before_bytes);
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(panel, (lds_bytes*)(tile + lds0 + j * 1024u), 16, voff[j], 0, 0, 0);
  }
};

// vmcnt(n) alone (gfx9 layout: vmcnt [3:0] and [15:14], expcnt [6:4], lgkmcnt [11:8]).
constexpr int wait_loads(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }
constexpr int kWaitLds = 0xC07F;  // lgkmcnt(0) alone

// issue_a(t, tile) and issue_b request slice t, kLoads loads of a wave in all.
// A slice is two depth steps; the fragments of the next step are read while
// the products of the current one run, across slices too, so the only
// wait a wave takes is the barrier in the middle of a slice: behind it every
// wave's reads of the slice are done (its buffer takes slice t + S) and every
// wave's share of the next slice has landed.  The reads are
// dealt out among the products (4096 x 14336 x 4096, dx 745 -> 715 us, the
// weights' gradients 800 -> 750, against all reads of a step first).
template <typename E, bool kACol, bool kBCol, int WM, int WN, int MB, int NB, int kLoads, int S, typename IA, typename IB>
__device__ __forceinline__ void staged_product(uint8_t* smem, uint32_t slices, IA issue_a, IB issue_b,
                                               typename E::Acc (&acc)[MB][NB]) {
  constexpr uint32_t kRowsA = WM * MB * 16u, kRowsB = WN * NB * 16u, kTileA = kRowsA * kSlice;
  constexpr uint32_t kStage = (kRowsA + kRowsB) * kSlice;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Fragments<kRowsA, kACol, MB> ra((wave / WN) * MB * 16u, lane);
  const Fragments<kRowsB, kBCol, NB> rb((wave % WN) * NB * 16u, lane);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = E::zero();
  static_assert((S - 1) * kLoads < 64, "the loads in flight fit the wait counter");
  auto issue = [&](uint32_t t, uint32_t stage) {
    uint8_t* at = smem + stage * kStage;
    issue_a(t, at);
    issue_b(t, at + kTileA);
  };
  u32x4 fa[2][MB], fb[2][NB];
  auto read = [&](uint32_t stage, int s) {
    const uint8_t* at = smem + stage * kStage;
    ra.read(at, s, fa[s]);
    rb.read(at + kTileA, s, fb[s]);
  };
  auto products = [&](int s) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = E::mfma(fa[s][i], fb[s][j], acc[i][j]);
  };
  if (slices == 0) return;
#pragma unroll
  for (uint32_t t = 0; t < (uint32_t)S; ++t)
    if (t < slices) issue(t, t);
  if (slices >= (uint32_t)S) __builtin_amdgcn_s_waitcnt(wait_loads((S - 1) * kLoads));
  else __builtin_amdgcn_s_waitcnt(wait_loads(0));
  asm volatile("s_barrier" ::: "memory");
  read(0, 0);
  constexpr int kReads = (kACol ? 2 * MB : MB) + (kBCol ? 2 * NB : NB), kEach = MB * NB / kReads;
  auto deal = [&]() {  // one LDS read (0x100), kEach products (0x008), and so on; the products left over
#pragma unroll
    for (int q = 0; q < kReads; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MB * NB - kEach * kReads, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t stage = 0;  // slice t's
  for (uint32_t t = 0; t + 1 < slices; ++t) {
    const uint32_t next = stage + 1u == (uint32_t)S ? 0u : stage + 1u;
    read(stage, 1);
    products(0);
    deal();
    // slice t + 1 has landed (behind it, where S > 2, S - 2 more are in flight)
    if (S == 2 || t + S > slices) __builtin_amdgcn_s_waitcnt(wait_loads(0));
    else __builtin_amdgcn_s_waitcnt(wait_loads((S - 2) * kLoads));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLds);  // satisfied: tells the compiler so
    if (t + S < slices) issue(t + S, stage);
    read(next, 0);
    products(1);
    deal();
    stage = next;
  }
  read(stage, 1);
  products(0);
  products(1);
}

// Every wave's partial tile to LDS, then finish(total): total(q) is block q's
// sum (row block q / NB, column block q % NB), the waves' parts in ascending order.
template <typename E, int MB, int NB, int W, typename F>
__device__ __forceinline__ void fold_waves(uint8_t* smem, const typename E::Acc (&acc)[MB][NB], F finish) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  __syncthreads();
  typename E::Acc* const part = reinterpret_cast<typename E::Acc*>(smem);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) part[(wave * MB * NB + i * NB + j) * 64u + lane] = acc[i][j];
  __syncthreads();
  auto total = [&](uint32_t q) {
    typename E::Acc v = part[q * 64u + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const typename E::Acc o = part[(w * MB * NB + q) * 64u + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += o[r];
    }
    return v;
  };
  finish(total);
}
// The product for few rows: a workgroup of W waves owns MB x NB blocks of
// 16 x 16 results, and wave w the depth slices w, w + W, ...: it moves a slice's
// rows into a slot of its own (issue(t, slot)), reads its fragments, requests
// its next slice into the same slot and multiplies while that lands.  No barrier
// until the end, so nearly W slots a workgroup stay in flight; then fold_waves.
template <typename E, int MB, int NB, int W, typename I, typename F>
__device__ __forceinline__ void few_rows_product(uint8_t* smem, uint32_t slices, I issue, F finish) {
  constexpr uint32_t kSlot = (MB + NB) * 16u * kSlice;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Fragments<MB * 16u, false, MB> ra(0, lane);
  const Fragments<NB * 16u, false, NB> rb(0, lane);
  typename E::Acc acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = E::zero();
  uint8_t* const slot = smem + wave * kSlot;
  if (wave < slices) issue(wave, slot);
  for (uint32_t t = wave; t < slices; t += W) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    u32x4 fa[2][MB], fb[2][NB];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      ra.read(slot, s, fa[s]);
      rb.read(slot + MB * 16u * kSlice, s, fb[s]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + W < slices) issue(t + W, slot);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = E::mfma(fa[s][i], fb[s][j], acc[i][j]);
  }
  fold_waves<E, MB, NB, W>(smem, acc, finish);
}
template <int MB, int NB, int W>
constexpr uint32_t few_rows_lds() {
  return W * (MB + NB) * 16u * kSlice > W * MB * NB * 1024u ? W * (MB + NB) * 16u * kSlice : W * MB * NB * 1024u;
}

// Tile `id` of a tiles_m x tiles_n grid.  Workgroups go round robin over the
// 8 XCDs: each XCD takes a contiguous run of an order that walks groups of
// 8 tile rows column by column, so the tiles an XCD runs together (32 CUs)
// share 8 row panels and a few column panels in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  const uint32_t total = tiles_m * tiles_n, xcd = id & 7u, per = total >> 3, rest = total & 7u;
  const uint32_t at = xcd * per + (xcd < rest ? xcd : rest) + (id >> 3);
  const uint32_t group = at / (8u * tiles_n), in = at % (8u * tiles_n);
  const uint32_t height = tiles_m - group * 8u < 8u ? tiles_m - group * 8u : 8u;
  tm = group * 8u + in % height;
  tn = in / height;
}

// The tile of the few-row products: column panels in groups of eight, one per
// XCD, whose tiles run one after another there (tn may lie past the last panel).
__device__ __forceinline__ void panel_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  if (tiles_n >= 8u) {
    tm = (id >> 3) % tiles_m;
    tn = (id >> 3) / tiles_m * 8u + (id & 7u);
  } else {
    tm = id % tiles_m;
    tn = id / tiles_m;
  }
}

// A pair of adjacent result rows (v0: row r, v1: row r + 1) of this lane's
// column, and the neighbouring lane's of its column: row r's two columns on
// even lanes, row r + 1's on odd ones, narrowed to bf16 (NaN canonical).
__device__ __forceinline__ uint32_t column_pair(float v0, float v1, bool odd) {
  const uint32_t p = tiler::bf16_pack2_rne(v0, v1);
  const uint32_t q = (uint32_t)__builtin_amdgcn_mov_dpp((int)p, 0xB1, 0xF, 0xF, true);  // quad_perm [1,0,3,2]
  return __builtin_amdgcn_perm(q, p, odd ? 0x03020706u : 0x05040100u);
}

// Stores a tile of bf16 results through LDS: value(i, j)[r] is this lane's
// result of row 16 i + 4 (lane / 16) + r, column 16 j + lane % 16 of its wave's
// (row0, col0) part of the ROWS x COLS tile; the tile is at (m0, n0) of the
// m x n result.  16-byte stores of whole row pieces, at any alignment; kStream:
// past the caches, for results that wait for another pass.  The caller's waves are
// done with the LDS.
template <uint32_t ROWS, uint32_t COLS, uint32_t THREADS, int MB, int NB, bool kStream, typename F>
__device__ __forceinline__ void store_tile_bf16(uint8_t* smem, uint32_t row0, uint32_t col0, uint16_t* out, uint32_t m,
                                                uint32_t n, uint32_t m0, uint32_t n0, F value) {
  constexpr uint32_t kRow = COLS * 2u, kPer = COLS / 8u;
  const uint32_t lane = threadIdx.x & 63u;
  const bool odd = lane & 1u;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const f32x4 v = value(i, j);
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const uint32_t row = row0 + i * 16u + (lane >> 4) * 4u + r + (odd ? 1u : 0u);
        const uint32_t col = col0 + j * 16u + (lane & 14u);
        *reinterpret_cast<uint32_t*>(smem + row * kRow + (((col >> 3) ^ (((row & 7u) << 1) & (kPer - 1u))) << 4) + ((col & 7u) << 1)) =
            column_pair(v[r], v[r + 1], odd);
      }
    }
  __syncthreads();
#pragma unroll 4
  for (uint32_t id = threadIdx.x; id < ROWS * kPer; id += THREADS) {
    const uint32_t row = id / kPer, piece = id % kPer, col = n0 + piece * 8u;
    if (m0 + row >= m || col >= n) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(smem + row * kRow + ((piece ^ (((row & 7u) << 1) & (kPer - 1u))) << 4));
    uint16_t* to = out + (uint64_t)(m0 + row) * n + col;
    if (n - col >= 8u) {
      if constexpr (kStream) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(to));
      else *reinterpret_cast<u32x4_any*>(to) = v;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 7u; ++e)
        if (e < n - col) to[e] = (uint16_t)(v[e >> 1] >> (16u * (e & 1u)));
    }
  }
}

}  // namespace tiler_product
