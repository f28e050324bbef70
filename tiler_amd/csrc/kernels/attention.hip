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
// operand type; their sum is taken before that, in binary32.
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
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

__device__ __forceinline__ uint32_t divide(const TilerDivisor& d, uint32_t n) {
  return (__umulhi(n, d.multiplier) + n) >> d.shift;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((tiler::f32x2_pair{a, b}), tiler::bf16x2_pair));
}
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// A sequence's rows and keys, from the device's lists.  Lists that break their
// contract are cut to what exists: starts to the tokens, lengths to the table.
struct Sequence {
  uint32_t first, fresh;  // its rows of q and out
  int32_t kept;           // position of its first new token (below zero: the list says fewer tokens than are new)
  __device__ __forceinline__ Sequence(const TilerAttentionShape& a, const int32_t* starts, const int32_t* lengths, uint32_t s) {
    const int32_t most = (int32_t)a.tokens;
    auto cut = [&](int32_t v) { return v < 0 ? 0 : v > most ? most : v; };
    const int32_t b = cut(starts[s]), e = cut(starts[s + 1]), length = lengths[s];
    first = (uint32_t)b;
    fresh = e > b ? (uint32_t)(e - b) : 0u;
    kept = (length < 0 ? 0 : length) - (int32_t)fresh;
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
  __device__ __forceinline__ bool read(uint32_t key) const { return key < high && (key >= low || key < sinks); }
};

// Byte offset of a key's row in the cache, or all ones where none is read.
__device__ __forceinline__ uint64_t row_offset(const TilerAttentionShape& a, bool read, int32_t entry, uint32_t key, uint32_t head) {
  const uint32_t in = key - divide(a.page, key) * a.page.divisor;
  const uint64_t at = (uint64_t)(uint32_t)entry * a.page_stride + (uint64_t)in * a.token_stride + (uint64_t)head * a.head_stride;
  return read && (uint32_t)entry < a.pages ? at * 2u : ~0ull;
}

// Place of a 16-byte piece in a value row of D elements in LDS.  The transposing
// read takes 32-byte blocks of 8 or 16 rows at once; the block's place changes
// with the row so that those lie on all banks, each as often.
template <int D>
__device__ __forceinline__ uint32_t value_piece(uint32_t key, uint32_t piece) {
  return piece ^ ((D == 64 ? (key >> 1) & 3u : key & 7u) << 1);
}

// ---------------------------------------------------------------------------
// Few rows: a tile of 16 rows, four waves that each take every fourth step of
// 32 keys on their own (keys to registers, values to LDS, one step ahead), and a
// join of the waves at the end.  A decode step is bound by the cache's bytes.
template <int NC>
struct FewSpace {
  static constexpr int D = 32 * NC;
  static constexpr uint32_t kRow = D * 2, kStage = 32 * kRow, kWaves = 4;
  union {
    uint8_t stage[kWaves][2][kStage];
    struct {
      float o[kWaves][16][D + 4];
    } join;
  };
  float m[kWaves][16], l[kWaves][16];
};

template <int NC>
__device__ __forceinline__ void few(const TilerAttentionShape& a, const uint16_t* q, const uint8_t* k, const uint8_t* v,
                                    const int32_t* table, const int32_t* starts, const int32_t* lengths, uint16_t* out,
                                    float* part_o, tiler::f32x2_pair* part_ml, FewSpace<NC>& space) {
  using Space = FewSpace<NC>;
  constexpr int D = Space::D, NB = 2 * NC;  // blocks of 16 elements
  constexpr uint32_t kPieces = D / 8;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 15u, g = lane >> 4;
  const uint32_t split = blockIdx.x / a.kv_heads % a.splits, head = blockIdx.x % a.kv_heads;
  const uint32_t s = blockIdx.x / (a.kv_heads * a.splits);
  const Sequence seq(a, starts, lengths, s);
  const uint32_t rows = seq.fresh * a.group;
  const int32_t* const pages = table + (uint64_t)s * a.width;
  const uint32_t real_pieces = a.head_dim / 8u;
  for (uint32_t row0 = 0; row0 < rows; row0 += 16u) {
    const uint32_t row = row0 + col, last = row0 + 15u < rows - 1u ? row0 + 15u : rows - 1u;
    const uint32_t token = divide(a.groups, row < rows ? row : rows - 1u);
    const uint32_t in_group = (row < rows ? row : rows - 1u) - token * a.group;
    const int32_t p = seq.kept + (int32_t)token;
    const int32_t p_first = seq.kept + (int32_t)divide(a.groups, row0), p_last = seq.kept + (int32_t)divide(a.groups, last);
    const Keys<32> keys(a, p_first, p_last);
    u32x4 qf[NC];
    {
      const uint16_t* at = q + (uint64_t)(seq.first + token) * a.q_stride + (uint64_t)(head * a.group + in_group) * a.head_dim;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        qf[c] = 4u * c + g < real_pieces ? *reinterpret_cast<const u32x4_any*>(at + 32 * c + 8 * g) : u32x4{0, 0, 0, 0};
    }
    const uint32_t begin = (uint32_t)((uint64_t)keys.steps * split / a.splits);
    const uint32_t end = (uint32_t)((uint64_t)keys.steps * (split + 1u) / a.splits);
    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    float m = kHidden, l = 0.0f;
    u32x4 kf[2][NC];
    int32_t entry = -1;
    auto look_up = [&](uint32_t t) {
      const uint32_t key = keys.base(t) + (lane & 31u);
      entry = t < end && keys.read(key) ? pages[divide(a.page, key)] : -1;
    };
    // Step t's keys into kf, its values on their way to the stage.
    auto request = [&](uint32_t t, uint32_t stage) {
      const uint32_t key = keys.base(t) + (lane & 31u);
      const uint64_t off = row_offset(a, keys.read(key), entry, key, head);
      auto of = [&](uint32_t r) {  // row r's offset
        const uint32_t lo = __builtin_amdgcn_ds_bpermute((int)(r * 4u), (int)(uint32_t)off);
        const uint32_t hi = __builtin_amdgcn_ds_bpermute((int)(r * 4u), (int)(uint32_t)(off >> 32));
        return (uint64_t)hi << 32 | lo;
      };
#pragma unroll
      for (uint32_t i = 0; i < Space::kStage / 1024u; ++i) {
        const uint32_t id = i * 64u + lane, r = id / kPieces, piece = value_piece<D>(r, id % kPieces);
        const uint64_t at = of(r);
        const uint8_t* from = at != ~0ull && piece < real_pieces ? v + at + piece * 16u : (const uint8_t*)&kZeroPiece;
        __builtin_amdgcn_global_load_lds((global_bytes*)from, (lds_bytes*)(space.stage[wave][stage] + i * 1024u), 16, 0, 0);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint64_t at = of(16u * b + col);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint32_t piece = 4u * c + g;
          const uint8_t* from = at != ~0ull && piece < real_pieces ? k + at + piece * 16u : (const uint8_t*)&kZeroPiece;
          kf[b][c] = *reinterpret_cast<const u32x4*>(from);
        }
      }
    };
    for (uint32_t t = begin + wave; t < end; t += Space::kWaves) {
      look_up(t);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      request(t, 0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
          const uint32_t key = base + 16u * b + 4u * g + r;
          const bool seen = key < keys.high && (int32_t)key <= p &&
                            (!a.window || (int64_t)key > (int64_t)p - (int64_t)a.window || key < a.sinks);
          if (!seen) sc[b][r] = kHidden;
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
        sum += (w[0] + w[1]) + (w[2] + w[3]);
        pf[2 * b] = narrow2(w[0], w[1]);
        pf[2 * b + 1] = narrow2(w[2], w[3]);
      }
      l = __builtin_fmaf(l, alpha, sum);
      const uint8_t* const stage = space.stage[wave][0];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        o[i] *= alpha;
        u32x2 h[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t key = 16u * b + 4u * g + (col >> 2);
          const uint8_t* at = stage + key * Space::kRow + value_piece<D>(key, 2u * i + ((col & 3u) >> 1)) * 16u + (col & 1u) * 8u;
          h[b] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
        }
        o[i] = mfma16(u32x4{h[0].x, h[0].y, h[1].x, h[1].y}, pf, o[i]);
      }
    }
    // the four lanes of a row hold its sum in parts, the four waves its keys
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the stages are read
    if (g == 0) space.m[wave][col] = m, space.l[wave][col] = l;
#pragma unroll
    for (int i = 0; i < NB; ++i) *reinterpret_cast<f32x4*>(&space.join.o[wave][col][16 * i + 4 * g]) = o[i];
    __syncthreads();
    for (uint32_t id = threadIdx.x; id < 16u * (D / 4); id += 256u) {
      const uint32_t r = id / (D / 4), d = id % (D / 4) * 4u, flat = row0 + r;
      if (flat >= rows || d >= a.head_dim) continue;
      float top = kHidden, total = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, space.m[w][r]);
      const float shift = top == kHidden ? 0.0f : -top * a.scale;
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float weight = exp2_fast(__builtin_fmaf(space.m[w][r], a.scale, shift));
        total += weight * space.l[w][r];
        sum += weight * *reinterpret_cast<const f32x4*>(&space.join.o[w][r][d]);
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

// A row's splits joined, in order: a wave a row.
__device__ __forceinline__ void join(const TilerAttentionShape& a, const int32_t* starts, const float* part_o,
                                     const tiler::f32x2_pair* part_ml, uint16_t* out) {
  const uint32_t lane = threadIdx.x & 63u, heads = a.kv_heads * a.group;
  const int32_t said = starts[a.sequences];
  const uint64_t tokens = said < 0 ? 0u : (uint32_t)said < a.tokens ? (uint32_t)said : a.tokens;
  for (uint64_t row = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6); row < tokens * heads; row += (uint64_t)gridDim.x * 4u) {
    const tiler::f32x2_pair* ml = part_ml + row * a.splits;
    float top = kHidden, total = 0.0f;
    for (uint32_t z = 0; z < a.splits; ++z) top = fmaxf(top, ml[z].x);
    const float shift = top == kHidden ? 0.0f : -top * a.scale;
    for (uint32_t z = 0; z < a.splits; ++z) total += exp2_fast(__builtin_fmaf(ml[z].x, a.scale, shift)) * ml[z].y;
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    const uint64_t token = row / heads, h = row % heads;
    for (uint32_t d = lane * 4u; d < a.head_dim; d += 256u) {
      f32x4 sum = {0, 0, 0, 0};
      for (uint32_t z = 0; z < a.splits; ++z) {
        const float weight = exp2_fast(__builtin_fmaf(ml[z].x, a.scale, shift));
        sum += weight * *reinterpret_cast<const f32x4*>(part_o + (row * a.splits + z) * a.head_dim + d);
      }
      u32x2 y = {narrow2(sum[0] * by, sum[1] * by), narrow2(sum[2] * by, sum[3] * by)};
      *reinterpret_cast<u32x2_any*>(out + token * a.out_stride + h * a.head_dim + d) = y;
    }
  }
}

}  // namespace tiler_attention

#define TILER_ATTENTION_FEW(NAME, NC)                                                                               \
  extern "C" __global__ void __launch_bounds__(256) NAME(                                                           \
      TilerAttentionShape a, const uint16_t* q, const uint8_t* k, const uint8_t* v, const int32_t* table,           \
      const int32_t* starts, const int32_t* lengths, uint16_t* out, float* part_o, tiler::f32x2_pair* part_ml) {              \
    __shared__ __attribute__((aligned(16))) tiler_attention::FewSpace<NC> space;                                    \
    tiler_attention::few<NC>(a, q, k, v, table, starts, lengths, out, part_o, part_ml, space);                      \
  }
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few64, 2)
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few128, 4)
TILER_ATTENTION_FEW(tiler_paged_attention_bf16_few256, 8)
#undef TILER_ATTENTION_FEW

extern "C" __global__ void __launch_bounds__(256)
    tiler_paged_attention_bf16_join(TilerAttentionShape a, const int32_t* starts, const float* part_o,
                                    const tiler::f32x2_pair* part_ml, uint16_t* out) {
  tiler_attention::join(a, starts, part_o, part_ml, out);
}
