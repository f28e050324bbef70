// Attention of new tokens over a paged cache: for query i of sequence s, at
// position p = length - new + i, over the keys j <= p that its window (j > p -
// window) or the first `sinks` tokens leave visible,
//   o = sum_j e^(scale q k_j - m) v_j / sum_j e^(scale q k_j - m)
// in one pass over the keys with the running maximum m and sum in binary32.
//
// Both products run on MFMA, transposed: S^T = K Q^T leaves each lane with one
// query's logits (the keys in its registers), so that the softmax needs one
// exchange across lanes a step, and its weights are, as they lie, the right
// operand of O^T = V^T P^T: the matrix unit sums over the keys in whatever order
// both operands name them.  The weights are rounded to bf16, the matrix unit's
// operand type; their sum, in binary32, is of the rounded ones, so that the
// rounding errors of equal weights cancel.
//
// The query heads that share a key/value head are rows of one tile (row =
// token * group + head of the group), so the cache is read once for all.
//
// A key's row comes through the page table: 64-bit offsets, any page size.
// Keys that no row of a tile sees are not read (zeros, so that what lies there
// cannot turn a weight of zero into a NaN); an entry that names no page of the
// cache reads as zeros too.
#pragma once

#include "attention.h"
#include "pieces.h"
#include "row_pieces.h"

namespace tiler_attention {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_bytes;
typedef const __attribute__((address_space(1))) void global_bytes;
using tiler_pieces::u32x2_any;
using tiler_pieces::u32x4_any;

constexpr float kHidden = -__builtin_huge_valf();
// What is read in place of a key's or value's row that is not there.
__device__ const u32x4 kZeroRow[32] = {};
__device__ __forceinline__ uint64_t zero_row() {
  uint64_t at = (uint64_t)(const void*)kZeroRow;
  asm("" : "+v"(at));  // an address like the others: no branch around their loads
  return at;
}
// 16 bytes a lane from `from` + kFrom, one after another to `to` (the instruction's
// own offset counts on both sides).
template <int kFrom = 0>
__device__ __forceinline__ void load_to_lds(uint64_t from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_bytes*)from, (lds_bytes*)(to - kFrom), 16, kFrom, 0);
}
constexpr int kWaitAll = 0x0070;    // s_waitcnt vmcnt(0) lgkmcnt(0)
constexpr int kWaitLds = 0xC07F;    // lgkmcnt(0)
constexpr int kWaitLoads = 0x0F70;  // vmcnt(0)

__device__ __forceinline__ uint32_t divide(const TilerDivisor& d, uint32_t n) {
  return (__umulhi(n, d.multiplier) + n) >> d.shift;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((tiler::f32x2_pair{a, b}), tiler::bf16x2_pair));
}
// sum + the two weights of a packed pair, as the values' product takes them.
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
  const tiler::bf16x2_pair ones = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(tiler::bf16x2_pair, pair), ones, sum, false);
}
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// A sequence's rows and keys, from the device's lists.  Lists that break their
// contract are cut to what exists: starts to the tokens, lengths to the table.
struct Sequence {
  uint32_t first, fresh;  // its rows of q and out
  int32_t kept;           // position of its first new token (below zero: the list says fewer tokens than are new)
  __device__ __forceinline__ Sequence(const TilerAttentionShape& a, const int32_t* starts, const int32_t* lengths, uint32_t s)
      : Sequence(a, starts[s], starts[s + 1], lengths[s]) {}
  __device__ __forceinline__ Sequence(const TilerAttentionShape& a, int32_t start, int32_t next, int32_t length) {
    const int32_t most = (int32_t)a.tokens;
    auto cut = [&](int32_t v) { return v < 0 ? 0 : v > most ? most : v; };
    const int32_t b = cut(start), e = cut(next);
    first = (uint32_t)b;
    fresh = e > b ? (uint32_t)(e - b) : 0u;
    kept = (length < 0 ? 0 : length) - (int32_t)fresh;
  }
};

// Which rows a tile of kRows has.  Sequence s has the tiles from starts[s] * group /
// kRows + s on: as many as its rows need, or one more.  Its lists' entries come
// along with the search.
template <uint32_t kRows>
struct Tile {
  uint32_t before = 0, in = 0;  // sequence s = before - 1 (0: none), and its tile
  int32_t start = 0, next = 0, length = 0;
  __device__ __forceinline__ Tile(const TilerAttentionShape& a, const int32_t* starts, const int32_t* lengths, uint32_t tile) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += 64u) {
      const uint32_t n = s0 + lane, at = n < a.sequences ? n : a.sequences - 1u;
      const int32_t starts_here = starts[at], next_here = starts[at + 1u], length_here = lengths[at];
      const int32_t cut = starts_here < 0 ? 0 : starts_here > (int32_t)a.tokens ? (int32_t)a.tokens : starts_here;
      const uint32_t from = (uint32_t)cut * a.group / kRows + n;
      const uint64_t mask = __ballot(n < a.sequences && from <= tile);
      if (mask) {
        const int last = 63 - __builtin_clzll(mask);
        in = tile - (uint32_t)__builtin_amdgcn_readlane(from, last);
        start = __builtin_amdgcn_readlane(starts_here, last);
        next = __builtin_amdgcn_readlane(next_here, last);
        length = __builtin_amdgcn_readlane(length_here, last);
      }
      before += __popcll(mask);
      if (mask != ~0ull) break;
    }
  }
};

// What a workgroup of the tiles does: with `whole` zero, every tile's keys in `splits`
// parts, a tile's and head's parts one after another; else the first `whole` tiles (times
// heads) whole, and the others' keys in parts, every first part before every second.
// Either way a head's workgroups are a multiple of the heads apart, on as few XCDs as can be.
struct Work {
  uint32_t head, tile, split = 0, splits = 1, part = 0;  // part: the split tile's number among them
  __device__ __forceinline__ Work(const TilerAttentionShape& a, uint32_t block, uint32_t rest) {
    uint32_t at = block;
    if (block >= a.whole) {
      const uint32_t in = block - a.whole;
      splits = a.splits;
      split = a.whole ? in / rest : in / a.kv_heads % splits;
      part = a.whole ? in % rest : in / (a.kv_heads * splits) * a.kv_heads + in % a.kv_heads;
      at = a.whole + part;
    }
    head = at % a.kv_heads;
    tile = (a.whole + rest) / a.kv_heads - 1u - at / a.kv_heads;
  }
};

// The keys a run of rows sees, in steps of `kStep`: first the steps of the
// sinks before the window, then those from the window's first key on.
template <uint32_t kStep>
struct Keys {
  uint32_t low, high, sinks;        // seen by any row: [low, high) and [0, sinks)
  uint32_t sink_steps, skip, steps;  // step t < sink_steps is t, else t + skip
  // p_first and p_last: the rows' first and last position
  __device__ __forceinline__ Keys(const TilerAttentionShape& a, int32_t p_first, int32_t p_last) {
    const uint32_t most = a.width * a.page.divisor;
    high = p_last < 0 ? 0u : (uint32_t)p_last + 1u;
    high = high < most ? high : most;
    low = a.window && p_first >= 0 && (uint32_t)p_first >= a.window ? (uint32_t)p_first - a.window + 1u : 0u;
    low = low < high ? low : high;
    sinks = a.window ? (a.sinks < low ? a.sinks : low) : 0u;
    const uint32_t from = low / kStep;
    sink_steps = (sinks + kStep - 1u) / kStep;
    sink_steps = sink_steps < from ? sink_steps : from;
    skip = from - sink_steps;
    steps = (high + kStep - 1u) / kStep - skip;
  }
  __device__ __forceinline__ uint32_t base(uint32_t t) const { return (t < sink_steps ? t : t + skip) * kStep; }
  __device__ __forceinline__ bool read(uint32_t key) const { return (key < high) & ((key >= low) | (key < sinks)); }
};

// The keys that one row sees: key <= limit and (key > floor or key < sinks).
struct Sight {
  int32_t limit, floor;
  __device__ __forceinline__ Sight(const TilerAttentionShape& a, uint32_t high, int32_t p) {
    limit = p < (int32_t)high - 1 ? p : (int32_t)high - 1;
    limit = limit > -1 ? limit : -1;
    const int64_t behind = (int64_t)p - (int64_t)a.window;
    floor = a.window && behind > -1 ? (int32_t)behind : -1;
    floor = floor < limit ? floor : limit;
  }
};
// Byte offset of a key's row in the cache, or -1 where none is read.
__device__ __forceinline__ int64_t row_offset(const TilerAttentionShape& a, bool read, int32_t entry, uint32_t key, uint32_t head) {
  const uint32_t in = key - divide(a.page, key) * a.page.divisor;
  const uint64_t at = (uint64_t)(uint32_t)entry * a.page_stride + (uint64_t)in * a.token_stride + (uint64_t)head * a.head_stride;
  return (read & ((uint32_t)entry < a.pages)) ? (int64_t)(at * 2u) : -1;
}

// Place of a 16-byte piece in a value row of D elements in LDS.  The transposing
// read takes 32-byte blocks of 8 or 16 rows at once; the block's place changes
// with the row so that those lie on all banks, each as often.
template <int D>
__device__ __forceinline__ uint32_t value_piece(uint32_t key, uint32_t piece) {
  return piece ^ ((D == 64 ? (key >> 1) & 3u : key & 7u) << 1);
}

// ---------------------------------------------------------------------------
// Few rows: a tile of 16 rows, four waves that take the steps of 32 keys in turn,
// each on its own (keys to registers, values to LDS, one step ahead of the
// products, no barrier), and a join of the waves at the end.  16 rows fill the smaller
// matrix instruction; eight waves and no parts to join afterwards are slower (15.4 us
// against 14.3).  A long decode step is bound by the cache's bytes: 8 sequences of 20000 to
// 32000 tokens, 8 heads of 128, 148 us (5.6 TB/s; 164 when each step waits for its
// loads).  A short one is bound by five trips to memory in a row (arguments, lists, table,
// keys, results): 16 sequences of 100 to 1000 tokens 11 us traced and 3 for the join.
template <int NC, int WAVES>
struct FewSpace {
  static constexpr int D = 32 * NC;
  static constexpr uint32_t kRow = D * 2, kStage = 32 * kRow;
  union {
    uint8_t stage[WAVES][2][kStage];
    float o[WAVES][16][D + 4];
  };
  float m[WAVES][16], l[WAVES][16];
};

template <int NC, int WAVES>
__device__ __forceinline__ void few(const TilerAttentionShape& a, const uint16_t* __restrict__ q, const uint8_t* __restrict__ k,
                                    const uint8_t* __restrict__ v, const int32_t* __restrict__ table,
                                    const int32_t* __restrict__ starts, const int32_t* __restrict__ lengths,
                                    uint16_t* __restrict__ out, float* __restrict__ part_o,
                                    tiler::f32x2_pair* __restrict__ part_ml, FewSpace<NC, WAVES>& space) {
  using Space = FewSpace<NC, WAVES>;
  constexpr int D = Space::D, NB = 2 * NC;  // blocks of 16 elements
  constexpr uint32_t kPieces = D / 8, kValueLoads = Space::kStage / 1024u;
  constexpr int kLoads = kValueLoads + 2 * NC + 1;  // of a step, with the next one's entry
  static_assert(kLoads < 64, "a step's loads fit the wait counter");
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 15u, g = lane >> 4;
  const uint32_t split = blockIdx.x / a.kv_heads % a.splits, head = blockIdx.x % a.kv_heads;
  const uint32_t s = blockIdx.x / (a.kv_heads * a.splits);
  const Sequence seq(a, starts, lengths, s);
  const uint32_t rows = seq.fresh * a.group;
  const int32_t* const pages = table + (uint64_t)s * a.width;
  const uint32_t real_pieces = a.head_dim / 8u;
  const uint64_t zero = zero_row();
  for (uint32_t row0 = 0; row0 < rows; row0 += 16u) {
    const uint32_t row = row0 + col, last = row0 + 15u < rows - 1u ? row0 + 15u : rows - 1u;
    const uint32_t token = divide(a.groups, row < rows ? row : rows - 1u);
    const uint32_t in_group = (row < rows ? row : rows - 1u) - token * a.group;
    const int32_t p = seq.kept + (int32_t)token;
    const int32_t p_first = seq.kept + (int32_t)divide(a.groups, row0), p_last = seq.kept + (int32_t)divide(a.groups, last);
    const Keys<32> keys(a, p_first, p_last);
    const uint32_t begin = (uint32_t)((uint64_t)keys.steps * split / a.splits) + wave;
    const uint32_t end = (uint32_t)((uint64_t)keys.steps * (split + 1u) / a.splits);
    const Sight sight(a, keys.high, p);
    const int32_t sinks = a.sinks < 0x7fffffffu ? (int32_t)a.sinks : 0x7fffffff;
    auto look_up = [&](uint32_t t) {
      const uint32_t key = keys.base(t) + (lane & 31u);
      return pages[((t < end) & keys.read(key)) ? divide(a.page, key) : 0u];
    };
    // Step t's values on their way to the stage, its keys to kf.
    auto request = [&](uint32_t t, int32_t entry, uint8_t* stage, u32x4 (&kf)[2][NC]) {
      const uint32_t key = keys.base(t) + (lane & 31u);
      const int64_t off = row_offset(a, keys.read(key), entry, key, head);
      auto of = [&](uint32_t r) {  // row r's offset
        const uint32_t lo = __builtin_amdgcn_ds_bpermute((int)(r * 4u), (int)(uint32_t)off);
        const uint32_t hi = __builtin_amdgcn_ds_bpermute((int)(r * 4u), (int)(uint32_t)(off >> 32));
        return (int64_t)((uint64_t)hi << 32 | lo);
      };
#pragma unroll
      for (uint32_t i = 0; i < kValueLoads; ++i) {
        const uint32_t id = i * 64u + lane, r = id / kPieces, piece = value_piece<D>(r, id % kPieces);
        const int64_t at = of(r);
        load_to_lds(at >= 0 && piece < real_pieces ? (uint64_t)v + at + piece * 16u : zero, stage + i * 1024u);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t at = of(16u * b + col);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint32_t piece = 4u * c + g;
          kf[b][c] = *reinterpret_cast<const u32x4*>(at >= 0 && piece < real_pieces ? (uint64_t)k + at + piece * 16u : zero);
        }
      }
    };
    u32x4 even[2][NC], odd[2][NC], qf[NC];
    int32_t entry = -1;
    if (begin < end) {
      entry = look_up(begin);
      const int32_t next = look_up(begin + WAVES);
      request(begin, entry, space.stage[wave][0], even);
      entry = next;
    }
    {
      const uint16_t* at = q + (uint64_t)(seq.first + token) * a.q_stride + (uint64_t)(head * a.group + in_group) * a.head_dim;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        qf[c] = 4u * c + g < real_pieces ? *reinterpret_cast<const u32x4_any*>(at + 32 * c + 8 * g) : u32x4{0, 0, 0, 0};
    }
    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    float m = kHidden, l = 0.0f;
    // Step t with the keys in kf, the next one's into next.
    auto step = [&](uint32_t t, uint32_t at, const u32x4 (&kf)[2][NC], u32x4 (&next)[2][NC]) {
      if (t + WAVES < end) {
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // the stage is read
        asm volatile("" ::: "memory");
        request(t + WAVES, entry, space.stage[wave][at ^ 1u], next);
        entry = look_up(t + 2 * WAVES);
        asm volatile("" ::: "memory");  // all of them requested: the wait counts them
        __builtin_amdgcn_s_waitcnt((kLoads & 15) | (kLoads >> 4) << 14 | 0x0F70);
      } else {
        __builtin_amdgcn_s_waitcnt(kWaitLoads);
      }
      asm volatile("" ::: "memory");  // step t's values have landed
      f32x4 sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        sc[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; ++c) sc[b] = mfma16(kf[b][c], qf[c], sc[b]);
      }
      const uint32_t base = keys.base(t);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int32_t key = (int32_t)(base + 16u * b + 4u * g + r);
          const bool seen = (key <= sight.limit) & ((key > sight.floor) | (key < sinks));
          sc[b][r] = seen ? sc[b][r] : kHidden;
        }
      float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                        fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      top = fmaxf(top, m);
      const float shift = top == kHidden ? 0.0f : -top * a.scale;  // a row that has seen nothing keeps weights of zero
      const float alpha = exp2_fast(__builtin_fmaf(m, a.scale, shift));
      m = top;
      u32x4 pf;
      float sum = 0.0f;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = exp2_fast(__builtin_fmaf(sc[b][r], a.scale, shift));
        pf[2 * b] = narrow2(w[0], w[1]);
        pf[2 * b + 1] = narrow2(w[2], w[3]);
        sum = add_pair(pf[2 * b + 1], add_pair(pf[2 * b], sum));
      }
      l = __builtin_fmaf(l, alpha, sum);
      const uint8_t* const stage = space.stage[wave][at];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= alpha;
        u32x2 h[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t key = 16u * b + 4u * g + (col >> 2);
          const uint8_t* from = stage + key * Space::kRow + value_piece<D>(key, 2u * i + ((col & 3u) >> 1)) * 16u + (col & 1u) * 8u;
          h[b] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)from));
        }
        o[i] = mfma16(u32x4{h[0].x, h[0].y, h[1].x, h[1].y}, pf, o[i]);
      }
    };
    for (uint32_t t = begin; t < end; t += 2 * WAVES) {
      step(t, 0, even, odd);
      if (t + WAVES < end) step(t + WAVES, 1, odd, even);
    }
    // the four lanes of a row hold its sum in parts, the waves its keys
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the stages are read
    if (g == 0) space.m[wave][col] = m, space.l[wave][col] = l;
#pragma unroll
    for (int i = 0; i < NB; ++i) *reinterpret_cast<f32x4*>(&space.o[wave][col][16 * i + 4 * g]) = o[i];
    __syncthreads();
    for (uint32_t id = threadIdx.x; id < 16u * (D / 4); id += 64u * WAVES) {
      const uint32_t r = id / (D / 4), d = id % (D / 4) * 4u, flat = row0 + r;
      if (flat >= rows || d >= a.head_dim) continue;
      float top = kHidden, total = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, space.m[w][r]);
      const float shift = top == kHidden ? 0.0f : -top * a.scale;
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float weight = exp2_fast(__builtin_fmaf(space.m[w][r], a.scale, shift));
        total += weight * space.l[w][r];
        sum += weight * *reinterpret_cast<const f32x4*>(&space.o[w][r][d]);
      }
      const uint32_t t = divide(a.groups, flat), h = head * a.group + (flat - t * a.group);
      const uint64_t token_row = seq.first + t;
      if (a.splits > 1u) {
        const uint64_t at = (token_row * (a.kv_heads * a.group) + h) * a.splits + split;
        *reinterpret_cast<f32x4*>(part_o + at * a.head_dim + d) = sum;
        if (d == 0) part_ml[at] = tiler::f32x2_pair{top, total};
      } else {
        const float by = total == 0.0f ? 0.0f : 1.0f / total;
        u32x2 y = {narrow2(sum[0] * by, sum[1] * by), narrow2(sum[2] * by, sum[3] * by)};
        *reinterpret_cast<u32x2_any*>(out + token_row * a.out_stride + (uint64_t)h * a.head_dim + d) = y;
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Many rows: four or eight waves of 32 rows each over steps of 64 keys, two steps
// of keys and values in LDS, brought there directly, one while the other is worked
// on.  Four waves bring a step; of eight, four take turns with the other four.
//
// LDS holds a step as 4 groups of 16 keys, each as NS segments of 32 elements, each
// as 16 keys of 64 bytes: a wave brings one group, each lane a piece of one key for
// every segment, so that it looks up one page a step.  Of the keys, piece c of a
// segment sits at c ^ (key / 4 & 3): the 16 keys of a fragment read then cover all
// banks.  A transposing read of the values takes 8 keys of one segment, 512 bytes
// in a row.
//
// The running maximum moves only where a logit passes it by kSlack (a factor of
// 2^8 in the weights, far inside binary32 and bf16): most steps rescale nothing.
//
// Heads of 128 are bound by the matrix pipe under the card's power limit: two prompts
// of 4096 tokens, 32 heads on 8, 283 to 295 us from card to card or 930 to 972 TFLOP/s,
// four fifths of a library product of 8192^3 (1209); the products alone, without the
// softmax, take 221.  512 tokens over 8512 keys: 73 to 81 us and 7 for the join.  Heads of
// 64 have half the products for the same exponentials, and the vector pipe bounds them:
// 700 TFLOP/s on the same prompts (heads of 96, 879).  Heads of 192 and 256 leave a CU one
// workgroup (674 and 655 TFLOP/s); at 256 some 160 bytes a lane do not fit the 512
// registers.
// Slower, us on the prompts: 64 rows a wave 356; three or four steps in LDS with the
// table's entries brought along 300; table lookups dealt out among the products 300; the
// keys' products before the values' (registers spill), and so two steps unrolled.
constexpr float kSlack = 8.0f;

template <int I, int N, typename F>
__device__ __forceinline__ void unroll(F f) {
  if constexpr (I < N) {
    f(tiler::Step<I>{});
    unroll<I + 1, N>(f);
  }
}

template <int NS>
struct TileSpace {
  static constexpr uint32_t kOperand = 64u * NS * 64u;
  uint8_t keys[2][kOperand], values[2][kOperand];
};

template <int NS, int WAVES>
__device__ __forceinline__ void tile(const TilerAttentionShape& a, const uint16_t* __restrict__ q, const uint8_t* __restrict__ k, const uint8_t* __restrict__ v,
                                     const int32_t* __restrict__ table, const int32_t* __restrict__ starts, const int32_t* __restrict__ lengths, uint16_t* __restrict__ out,
                                     float* __restrict__ part_o, tiler::f32x2_pair* __restrict__ part_ml, TileSpace<NS>& space) {
  constexpr uint32_t kRows = 32u * WAVES, kTurns = WAVES / 4;
  constexpr int NC = 2 * NS;  // depth steps of 16 elements
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 31u, h = lane >> 5;
  const Work work(a, blockIdx.x, (gridDim.x - a.whole) / a.splits);
  const uint32_t head = work.head, split = work.split, splits = work.splits;
  const Tile<kRows> place(a, starts, lengths, work.tile);
  if (place.before == 0) return;
  const uint32_t s = place.before - 1u, tile_in = place.in;
  const Sequence seq(a, place.start, place.next, place.length);
  const uint32_t rows = seq.fresh * a.group, row0 = tile_in * kRows;
  if (row0 >= rows) return;
  const int32_t* const pages = table + (uint64_t)s * a.width;
  const uint32_t real_pieces = a.head_dim / 8u;
  auto position = [&](uint32_t row) { return seq.kept + (int32_t)divide(a.groups, row < rows ? row : rows - 1u); };
  const Keys<64> keys(a, position(row0), position(row0 + kRows - 1u));
  const uint32_t begin = (uint32_t)((uint64_t)keys.steps * split / splits);
  const uint32_t end = (uint32_t)((uint64_t)keys.steps * (split + 1u) / splits);
  const uint32_t wave_row = row0 + wave * 32u;
  const bool works = wave_row < rows;
  const int32_t p_first = position(wave_row), p_last = position(wave_row + 31u);
  const uint32_t row = wave_row + col, real = row < rows ? row : rows - 1u;
  const uint32_t token = divide(a.groups, real), hq = head * a.group + (real - token * a.group);
  const int32_t p = seq.kept + (int32_t)token;
  u32x4 qf[NC];
  {
    const uint16_t* at = q + (uint64_t)(seq.first + token) * a.q_stride + (uint64_t)hq * a.head_dim;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      qf[c] = 2u * c + h < real_pieces ? *reinterpret_cast<const u32x4_any*>(at + 16 * c + 8 * h) : u32x4{0, 0, 0, 0};
  }
  // This lane's key of a step, and the piece of a segment that it brings; pieces
  // past the head's end are zeros.
  const uint32_t key_in = wave % 4u * 16u + (lane >> 2), turn = wave / 4u, value_in = lane & 3u, key_piece = value_in ^ ((lane >> 4) & 3u);
  const uint64_t zero = zero_row();
  const uint64_t keys_from = (uint64_t)k + head * a.head_stride * 2u + key_piece * 16u;
  const uint64_t values_from = (uint64_t)v + head * a.head_stride * 2u + value_in * 16u;
  // The page of this lane's key, the key's place in it (elements) and the entry of
  // the table: looked up a step ahead, and stepped without a division.
  const uint32_t page_span = a.page.divisor * a.token_stride;
  const uint32_t step_pages = divide(a.page, 64u * kTurns), step_span = (64u * kTurns - step_pages * a.page.divisor) * a.token_stride;
  uint32_t index = 0, in_page = 0, in_found = 0;
  int32_t entry = -1;
  uint64_t found = 0;  // a bit a lane
  auto go_to = [&](uint32_t t) {
    const uint32_t key = keys.base(t) + key_in;
    index = divide(a.page, key);
    in_page = (key - index * a.page.divisor) * a.token_stride;
  };
  auto look_up = [&](uint32_t t) {  // of step t, and on to this wave's next
    const uint32_t base = keys.base(t), key = base + key_in;
    uint32_t at = index;
    found = ~0ull;
    if (t >= end || base < keys.low || base + 63u >= keys.high) {
      found = t < end ? __ballot(keys.read(key)) : 0ull;
      at = found >> lane & 1u ? index : 0u;
      asm volatile("" : "+v"(at));
    }
    entry = pages[at];
    in_found = in_page;
    if (t < keys.sink_steps && t + kTurns >= keys.sink_steps) {
      go_to(t + kTurns);
    } else {
      in_page += step_span;
      const bool wraps = in_page >= page_span || in_page < step_span;
      index += step_pages + (wraps ? 1u : 0u);
      in_page -= wraps ? page_span : 0u;
    }
  };
  struct Row {
    uint64_t at, there;  // elements; a bit a lane
  };
  auto row_found = [&] {
    return Row{(uint64_t)(uint32_t)entry * a.page_stride + in_found, found & __ballot((uint32_t)entry < a.pages)};
  };
  uint8_t* const to = space.keys[0] + wave % 4u * (NS * 1024u);
  auto request = [&](const Row& r, uint64_t from, uint32_t piece, uint8_t* at) {
    // Branches, not selections: the asm keeps the usual case free of them.
    uint64_t src = from + r.at * 2u;
    if (r.there != ~0ull) {
      src = r.there >> lane & 1u ? src : zero;
      asm volatile("" : "+v"(src));
    }
    unroll<0, NS>([&](auto n) {
      if (4u * n.value + 4u > real_pieces) {
        uint64_t some = 4u * n.value + piece < real_pieces ? src : zero;
        asm volatile("" : "+v"(some));
        load_to_lds<n.value * 64>(some, at + n.value * 1024);
      } else {
        load_to_lds<n.value * 64>(src, at + n.value * 1024);
      }
    });
  };
  auto request_keys = [&](const Row& r, uint32_t buffer) { request(r, keys_from, key_piece, to + buffer * TileSpace<NS>::kOperand); };
  auto request_values = [&](const Row& r, uint32_t buffer) {
    request(r, values_from, value_in, to + (2u + buffer) * TileSpace<NS>::kOperand);
  };
  auto landed = [&] {  // everything this wave requested; behind the barrier, every wave's
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitAll);
    asm volatile("s_barrier" ::: "memory");
  };
  f32x16 o[NS], sc[2];
  float m = kHidden, l = 0.0f, most = kHidden;  // most: of this lane's first 16 logits of a step
  u32x4 pf[4];  // the last step's weights
#pragma unroll
  for (int n = 0; n < NS; ++n) o[n] = f32x16{};
  // Byte offsets of this lane's fragments: keys 32 kb + col, piece 2 c + h; values
  // of keys 16 kc + 4 h + (lane / 4 & 3) (and 8 on), elements 32 n + 16 (lane / 16 & 1) + 4 (lane & 3).
  const uint32_t key_at = (col >> 4) * (NS * 1024u) + (col & 15u) * 64u, key_swap = (col >> 2) & 3u;
  const uint32_t value_at = (4u * h + ((lane >> 2) & 3u)) * 64u + ((lane >> 4) & 1u) * 32u + (lane & 3u) * 8u;
  const Sight first(a, keys.high, p_first), last(a, keys.high, p_last), sight(a, keys.high, p);
  const int32_t sinks = a.sinks < 0x7fffffffu ? (int32_t)a.sinks : 0x7fffffff;
  auto read_key = [&](uint32_t buffer, int kb, int c) {
    return *reinterpret_cast<const u32x4*>(space.keys[buffer] + key_at + kb * (2u * NS * 1024u) + (c >> 1) * 1024u +
                                           ((((c & 1u) * 2u + h) ^ key_swap) << 4));
  };
  auto read_value = [&](uint32_t buffer, int kc, int n) {
    const uint8_t* at = space.values[buffer] + value_at + kc * (NS * 1024u) + n * 1024u;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 512)));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };
  // What the last step's maximum made of the results before that step's values.
  bool moved = false;
  float alpha = 1.0f;
  auto rescale = [&] {
    if (moved) {
#pragma unroll
      for (int n = 0; n < NS; ++n) o[n] *= alpha;
    }
  };
  Row rows_of[3 - kTurns] = {};  // whose values are still to come: of this wave's steps before t + 2
  // Step t, of which sc holds the logits: its weights to pf, while the matrix unit
  // takes in the values of step t - 1 (unless t is the first) and makes the logits of
  // step t + 1 in the place of these (unless t is the last).
  auto step = [&](uint32_t t, auto is_first, auto is_last) {
    const uint32_t buffer = (t - begin) & 1u;
    const int32_t base = (int32_t)keys.base(t), top_key = base > 0x7fffffff - 63 ? 0x7fffffff : base + 63;
    const bool cut_above = top_key > first.limit, cut_below = base <= last.floor && top_key >= sinks;
    if (cut_above || cut_below) {  // not every row sees every key
      const int32_t from = base + 4 * (int32_t)h;
      auto show = [&](auto seen) {
        most = kHidden;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          sc[i >> 4][i & 15] = seen(8 * (i >> 2) + (i & 3)) ? sc[i >> 4][i & 15] : kHidden;
          if (i < 16) most = fmaxf(most, sc[0][i]);
        }
      };
      if (!cut_below || top_key < (int32_t)keys.low) {  // one bound: the row's own key, or the sinks before every window
        const int32_t limit = (cut_below ? sinks - 1 : sight.limit) - from;
        show([&](int32_t key) { return key <= limit; });
      } else if (base >= sinks) {  // a window: one comparison of what lies above its floor
        const uint32_t below = (uint32_t)(from - 1 - sight.floor), count = (uint32_t)(sight.limit - sight.floor);
        show([&](int32_t key) { return below + (uint32_t)key < count; });
      } else {
        const int32_t limit = sight.limit - from, floor = sight.floor - from, sink = sinks - from;
        show([&](int32_t key) { return (key <= limit) & ((key > floor) | (key < sink)); });
      }
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(most, sc[1][i]), sc[1][i + 1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
    const float top = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    rescale();
    moved = __any((top - m) * a.scale > kSlack);  // also at the first key: m is -infinity
    if (moved) {
      const float to = fmaxf(top, m);
      alpha = to == kHidden ? 1.0f : exp2_fast((m - to) * a.scale);
      m = to;
      l *= alpha;
    }
    const float shift = m == kHidden ? 0.0f : -m * a.scale;
    most = kHidden;
    u32x4 weights[4];
    float sums[2] = {0.0f, 0.0f}, one = 0.0f;
    auto weigh = [&](int i) {  // logit i of the step's 32
      const float w = exp2_fast(__builtin_fmaf(sc[i >> 4][i & 15], a.scale, shift));
      if (i % 2 == 0) {
        one = w;
        asm volatile("" : "+v"(one));  // made here, not where it is used
        return;
      }
      uint32_t both = narrow2(one, w);
      float sum = add_pair(both, sums[(i >> 1) & 1]);
      asm volatile("" : "+v"(both), "+v"(sum));
      sums[(i >> 1) & 1] = sum;
      weights[i >> 3][(i >> 1) & 3] = both;
    };
    // The products one by one: three quarters of the values' with the weights of the
    // first 32 keys, whose logits' place the next first 32 take then, with the rest
    // of the values' beside the other weights; then the next other 32 keys'.  With
    // each product go its share of the weights (at the end, of the next maximum) and
    // the fragment of a later product.  Nothing moves from one such group to another:
    // left to itself the compiler puts all weights before the products.
    constexpr int kA = is_first.value ? 0 : 3 * NS, kB = kA + (is_last.value ? 0 : 2 * NS), kC = kB + (is_first.value ? 0 : NS);
    constexpr int kProducts = kC + (is_last.value ? 0 : 2 * NS), kBatch = 2;
    auto fragment = [&](int u) {
      const int p = u < kA ? u : u - (kB - kA);  // of the values
      return u < kA || (u >= kB && u < kC) ? read_value(buffer ^ 1u, p / NS, p % NS)
                                           : read_key(buffer ^ 1u, u >= kC, u < kB ? u - kA : u - kC);
    };
    auto weighed = [&](int u) {  // logits before product u
      if (is_last.value) return kProducts ? 32 * u / (kProducts ? kProducts : 1) : 32;
      return u < kA ? 16 * u / (kA ? kA : 1) : u < kC ? 16 + 16 * (u - kA) / (kC - kA) : 32;
    };
#pragma unroll
    for (int i = 0; i < weighed(0); ++i) weigh(i);
    u32x4 f[2][kBatch];
#pragma unroll
    for (int u = 0; u < kBatch && u < kProducts; ++u) f[0][u] = fragment(u);
    unroll<0, kProducts>([&](auto product) {
      constexpr int u = product.value;
      const u32x4 at = f[u / kBatch % 2][u % kBatch];
      const int p = u < kA ? u : u - (kB - kA);
      if (u < kA || (u >= kB && u < kC)) o[p % NS] = mfma32(at, pf[p / NS], o[p % NS]);
      else if (u < kB) sc[0] = mfma32(at, qf[u - kA], u == kA ? f32x16{} : sc[0]);
      else sc[1] = mfma32(at, qf[u - kC], u == kC ? f32x16{} : sc[1]);
      if (u % kBatch == 0) {  // this batch's fragments are there: the next one's
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = u + kBatch; j < u + 2 * kBatch && j < kProducts; ++j) f[j / kBatch % 2][j % kBatch] = fragment(j);
      }
#pragma unroll
      for (int i = weighed(u); i < weighed(u + 1); ++i) weigh(i);
      if (u >= kC) {
#pragma unroll
        for (int i = (u - kC) * 8 / (2 * NS); i < (u - kC + 1) * 8 / (2 * NS); ++i) {
          most = fmaxf(fmaxf(most, sc[0][2 * i]), sc[0][2 * i + 1]);
          asm volatile("" : "+v"(most));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    l += sums[0] + sums[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = weights[i];
  };
  if (begin < end) {
    using No = tiler::Step<0>;
    using Yes = tiler::Step<1>;
    go_to(begin + turn);
    look_up(begin + turn);
    for (uint32_t i = 0; i < 3u - kTurns; ++i) {
      rows_of[i] = row_found();
      look_up(begin + turn + (i + 1u) * kTurns);
    }
    if (turn == 0) request_keys(rows_of[0], 0);
    landed();
    if (kTurns == 1) request_keys(rows_of[2 - kTurns], 1);
    else if (turn == 1) request_keys(rows_of[0], 1);
    if (works) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int c = 0; c < NC; ++c) sc[kb] = mfma32(read_key(0, kb, c), qf[c], c == 0 ? f32x16{} : sc[kb]);
#pragma unroll
      for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(most, sc[0][i]), sc[0][i + 1]);
    }
    // Before step t: the keys of step t + 1 and the values of step t - 1 have landed,
    // and every wave has read those of steps t and t - 2, whose places the next ones take.
    auto advance = [&](uint32_t t) {
      landed();
      const uint32_t buffer = (t - begin) & 1u;
      if (kTurns > 1 && buffer != turn) return;
      const Row r = row_found();
      look_up(t + 2u + kTurns);
      if (t + 2u < end) request_keys(r, buffer);
      request_values(rows_of[0], buffer);
      if (kTurns == 1) rows_of[0] = rows_of[2 - kTurns];
      rows_of[2 - kTurns] = r;
    };
    uint32_t t = begin;
    advance(t);
    if (end - begin == 1u) {
      if (works) step(t, Yes{}, Yes{});
    } else {
      if (works) step(t, Yes{}, No{});
      for (++t; t + 1u < end; ++t) {
        advance(t);
        if (works) step(t, No{}, No{});
      }
      advance(t);
      if (works) step(t, No{}, Yes{});
    }
    landed();  // the last values
    if (works) {
      rescale();
#pragma unroll
      for (int kc = 0; kc < 4; ++kc)
#pragma unroll
        for (int n = 0; n < NS; ++n) o[n] = mfma32(read_value((end - 1u - begin) & 1u, kc, n), pf[kc], o[n]);
    }
  }
  if (row >= rows) return;
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float total = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
  const uint64_t token_row = seq.first + token;
  if (splits > 1u) {
    const uint64_t at = (a.whole ? (uint64_t)work.part * kRows + (row - row0) : token_row * (a.kv_heads * a.group) + hq) * splits + split;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint32_t d = 32u * n + 2u * i + 4u * h;
        if (d < a.head_dim) *reinterpret_cast<f32x4*>(part_o + at * a.head_dim + d) = f32x4{o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]};
      }
    if (h == 0) part_ml[at] = tiler::f32x2_pair{m, total};
  } else {
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const at = out + token_row * a.out_stride + (uint64_t)hq * a.head_dim;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint32_t d = 32u * n + 2u * i + 4u * h;
        if (d < a.head_dim)
          *reinterpret_cast<u32x2_any*>(at + d) = u32x2{narrow2(o[n][i] * by, o[n][i + 1] * by), narrow2(o[n][i + 2] * by, o[n][i + 3] * by)};
      }
  }
}

// Four elements of a row from its parts, in order, four parts at a time: their sums
// and results are read at once, ahead of the maximum that weighs them.
__device__ __forceinline__ u32x2 joined(const TilerAttentionShape& a, const tiler::f32x2_pair* ml, const float* from) {
  float m = kHidden, total = 0.0f;
  f32x4 sum = {0, 0, 0, 0};
  for (uint32_t z0 = 0; z0 < a.splits; z0 += 4u) {
    tiler::f32x2_pair of[4];
    f32x4 o[4];
#pragma unroll
    for (uint32_t z = 0; z < 4u; ++z) {
      const uint32_t at = z0 + z < a.splits ? z0 + z : a.splits - 1u;
      of[z] = ml[at];
      o[z] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(from + (uint64_t)at * a.head_dim));
    }
    float top = m;
#pragma unroll
    for (uint32_t z = 0; z < 4u; ++z) {
      const bool there = z0 + z < a.splits;
      of[z] = there ? of[z] : tiler::f32x2_pair{kHidden, 0.0f};
      o[z] = there ? o[z] : f32x4{0, 0, 0, 0};
      top = fmaxf(top, of[z].x);
    }
    const float shift = top == kHidden ? 0.0f : -top * a.scale;
    const float before = exp2_fast(__builtin_fmaf(m, a.scale, shift));
    m = top;
    total *= before;
    sum *= before;
#pragma unroll
    for (uint32_t z = 0; z < 4u; ++z) {
      const float weight = exp2_fast(__builtin_fmaf(of[z].x, a.scale, shift));
      total += weight * of[z].y;
      sum += weight * o[z];
    }
  }
  const float by = total == 0.0f ? 0.0f : 1.0f / total;
  return u32x2{narrow2(sum[0] * by, sum[1] * by), narrow2(sum[2] * by, sum[3] * by)};
}

// All rows' parts, four elements a thread, read ahead of the list that says which rows
// are any sequence's.
__device__ __forceinline__ void join(const TilerAttentionShape& a, const int32_t* __restrict__ starts,
                                     const float* __restrict__ part_o, const tiler::f32x2_pair* __restrict__ part_ml,
                                     uint16_t* __restrict__ out) {
  const uint32_t heads = a.kv_heads * a.group, quads = a.head_dim / 4u;
  const int32_t first = starts[0], said = starts[a.sequences];
  const uint64_t all = (uint64_t)a.tokens * heads * quads;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256u) {
    const uint32_t row = (uint32_t)(i / quads), d = (uint32_t)(i - (uint64_t)row * quads) * 4u;
    const uint64_t at = (uint64_t)row * a.splits;
    const u32x2 y = joined(a, part_ml + at, part_o + at * a.head_dim + d);
    const uint32_t token = row / heads, h = row - token * heads;
    if ((int32_t)token < first || (int32_t)token >= said) continue;
    *reinterpret_cast<u32x2_any*>(out + (uint64_t)token * a.out_stride + (uint64_t)h * a.head_dim + d) = y;
  }
}

// The split tiles' behind the whole ones: a workgroup takes 32 rows of one.
template <uint32_t kRows>
__device__ __forceinline__ void join_tail(const TilerAttentionShape& a, const int32_t* __restrict__ starts,
                                          const int32_t* __restrict__ lengths, const float* __restrict__ part_o,
                                          const tiler::f32x2_pair* __restrict__ part_ml, uint16_t* __restrict__ out) {
  const Work work(a, a.whole + blockIdx.x, gridDim.x);
  const Tile<kRows> place(a, starts, lengths, work.tile);
  if (place.before == 0) return;
  const Sequence seq(a, place.start, place.next, place.length);
  const uint32_t rows = seq.fresh * a.group, quads = a.head_dim / 4u;
  for (uint32_t i = threadIdx.x; i < 32u * quads; i += 256u) {
    const uint32_t in = blockIdx.y * 32u + i / quads, d = i % quads * 4u, row = place.in * kRows + in;
    if (row >= rows) return;
    const uint64_t at = ((uint64_t)work.part * kRows + in) * a.splits;
    const u32x2 y = joined(a, part_ml + at, part_o + at * a.head_dim + d);
    const uint32_t token = divide(a.groups, row), h = work.head * a.group + (row - token * a.group);
    *reinterpret_cast<u32x2_any*>(out + (uint64_t)(seq.first + token) * a.out_stride + (uint64_t)h * a.head_dim + d) = y;
  }
}

}  // namespace tiler_attention

#define TILER_ATTENTION_FEW(NAME, NC, WAVES)                                                                        \
  extern "C" __global__ void __launch_bounds__(64 * WAVES) NAME(                                                    \
      TilerAttentionShape a, const uint16_t* q, const uint8_t* k, const uint8_t* v, const int32_t* table,           \
      const int32_t* starts, const int32_t* lengths, uint16_t* out, float* part_o, tiler::f32x2_pair* part_ml) {    \
    __shared__ __attribute__((aligned(16))) tiler_attention::FewSpace<NC, WAVES> space;                             \
    tiler_attention::few<NC, WAVES>(a, q, k, v, table, starts, lengths, out, part_o, part_ml, space);               \
  }
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few64, 2, 4)
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few128, 4, 4)
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few256, 8, 4)
#undef TILER_ATTENTION_FEW

#define TILER_ATTENTION_TILE(NAME, NS, WAVES, EACH)                                                                 \
  extern "C" __global__ void __launch_bounds__(64 * WAVES, EACH) NAME(                                              \
      TilerAttentionShape a, const uint16_t* q, const uint8_t* k, const uint8_t* v, const int32_t* table,           \
      const int32_t* starts, const int32_t* lengths, uint16_t* out, float* part_o, tiler::f32x2_pair* part_ml) {    \
    __shared__ __attribute__((aligned(16))) tiler_attention::TileSpace<NS> space;                                   \
    tiler_attention::tile<NS, WAVES>(a, q, k, v, table, starts, lengths, out, part_o, part_ml, space);              \
  }
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t128_d64, 2, 4, 2)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t128_d96, 3, 4, 2)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t128_d128, 4, 4, 2)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t128_d192, 6, 4, 1)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t128_d256, 8, 4, 1)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t256_d64, 2, 8, 2)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t256_d96, 3, 8, 2)
TILER_ATTENTION_TILE(tiler_paged_attention_bf16_t256_d128, 4, 8, 2)
#undef TILER_ATTENTION_TILE

extern "C" __global__ void __launch_bounds__(256)
    tiler_paged_attention_bf16_join(TilerAttentionShape a, const int32_t* starts, const float* part_o,
                                    const tiler::f32x2_pair* part_ml, uint16_t* out) {
  tiler_attention::join(a, starts, part_o, part_ml, out);
}
extern "C" __global__ void __launch_bounds__(256)
    tiler_paged_attention_bf16_join_t128(TilerAttentionShape a, const int32_t* starts, const int32_t* lengths, const float* part_o,
                                         const tiler::f32x2_pair* part_ml, uint16_t* out) {
  tiler_attention::join_tail<128>(a, starts, lengths, part_o, part_ml, out);
}
extern "C" __global__ void __launch_bounds__(256)
    tiler_paged_attention_bf16_join_t256(TilerAttentionShape a, const int32_t* starts, const int32_t* lengths, const float* part_o,
                                         const tiler::f32x2_pair* part_ml, uint16_t* out) {
  tiler_attention::join_tail<256>(a, starts, lengths, part_o, part_ml, out);
}
