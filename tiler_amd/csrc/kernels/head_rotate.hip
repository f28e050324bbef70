// The norm of each query and key head and the position rotation, in one pass:
//   u = x w / sqrt(mean(x^2) + eps)          (or x, without a norm)
//   y_i = u_i cos a_p - u_j sin a_p, y_j = u_j cos a_p + u_i sin a_p
// for pair p = (i, j) of the head's first `rotary` elements, a_p = position *
// frequency_p; the elements behind them pass.  Its gradients turn dy back,
// g = R^T dy, and with xh = x r and gw = g w
//   dx = r (gw - xh mean(gw xh)), dw = sum over tokens and heads of g xh.
//
// Angles are products in 64 bits, reduced to a quarter turn in 64 bits; sine and
// cosine of what remains are sums in binary32.  In binary32 a position of 10^6
// radians would be off by 0.03.  A token's angles are made once for all its heads.
#pragma once

#include "common.h"
#include "head_rotate.h"
#include "row_pieces.h"

namespace tiler_heads {

// (cos, sin) of an angle below 2^62.  Its quarter turns come off in 64 bits, by pi / 2
// in two parts (a fused product is exact before its one rounding), and once more from an
// angle beyond 2^40, whose quotient may itself be off by turns.  The series for what
// remains, |r| <= pi / 4, go to r^9 and r^10 and leave out less than 3e-8 of it.
__device__ __forceinline__ tiler::f32x2_pair turn_of(double angle) {
  const double quarters = __builtin_rint(angle * 0.63661977236758134308);
  double left = __builtin_fma(-quarters, 1.57079632679489655800, angle);
  left = __builtin_fma(-quarters, 6.12323399573676603587e-17, left);
  uint32_t turn = (uint32_t)(long long)quarters;
  if (__builtin_fabs(angle) > 0x1p40) {
    const double more = __builtin_rint(left * 0.63661977236758134308);
    left = __builtin_fma(-more, 1.57079632679489655800, left);
    left = __builtin_fma(-more, 6.12323399573676603587e-17, left);
    turn += (uint32_t)(int)more;
  }
  const float r = (float)left, r2 = r * r;
  float s = __builtin_fmaf(r2, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = __builtin_fmaf(r2, s, 1.0f / 120.0f);
  s = __builtin_fmaf(r2, s, -1.0f / 6.0f);
  s = __builtin_fmaf(r * r2, s, r);
  float c = __builtin_fmaf(r2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = __builtin_fmaf(r2, c, -1.0f / 720.0f);
  c = __builtin_fmaf(r2, c, 1.0f / 24.0f);
  c = __builtin_fmaf(r2, c, -0.5f);
  c = __builtin_fmaf(r2, c, 1.0f);
  turn &= 3u;
  const float a = turn & 1u ? s : c, b = turn & 1u ? c : s;
  return tiler::f32x2_pair{turn == 1u || turn == 2u ? -a : a, turn >= 2u ? -b : b};
}

template <typename T>
__device__ __forceinline__ float widened(T v) {
  if constexpr (sizeof(T) == 2) return __uint_as_float((uint32_t)v << 16);
  else return v;
}
template <typename T>
__device__ __forceinline__ T narrowed(float v) {
  if constexpr (sizeof(T) == 2) return (T)__builtin_bit_cast(uint16_t, (__bf16)v);
  else return v;
}

constexpr uint32_t kMostPairs = 512;  // of a head of 1024 elements

// Elements of a head's pairs: lane's pairs are p, p + 64 ...
__device__ __forceinline__ uint32_t pair_first(const TilerHeads& a, uint32_t p) { return a.neighbours ? 2u * p : p; }
__device__ __forceinline__ uint32_t pair_second(const TilerHeads& a, uint32_t p) {
  return a.neighbours ? 2u * p + 1u : p + a.rotary / 2u;
}

__device__ __forceinline__ float wave_sum(float v) {
  return tiler_rows::wave_fold(v, [](float x, float y) { return x + y; });
}

// Any head size, rotation and alignment: a workgroup a token, a wave a head, an
// element a load; the head is read twice.  Latency bounds it: 8192 tokens of 32 and 8
// heads of 80, 20 elements rotated, 164 us and 301 for the gradients (32 rotated, in
// units, 27 and 44).
template <typename T>
__device__ __forceinline__ void rotate_any(const TilerHeads& a, const T* q, const T* k, const T* v, const T* wq,
                                           const T* wk, const int32_t* positions, const double* frequencies, T* q_out,
                                           T* k_out, T* k_cache, T* v_cache, const int32_t* slots) {
  __shared__ tiler::f32x2_pair turns[kMostPairs];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, pairs = a.rotary / 2u;
  const uint32_t heads = a.q_heads + a.kv_heads + (v ? a.kv_heads : 0u);
  for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    __syncthreads();  // the turns before are read
    for (uint32_t p = threadIdx.x; p < pairs; p += 256u) turns[p] = turn_of((double)positions[token] * frequencies[p]);
    __syncthreads();
    const int64_t slot = slots ? slots[token] : -1;
    const bool stored = slot >= 0 && (uint64_t)slot < a.slots;
    const uint64_t at = stored ? (uint64_t)((uint32_t)slot / a.page) * a.page_stride + (uint64_t)((uint32_t)slot % a.page) * a.token_stride : 0;
    for (uint32_t n = wave; n < heads; n += 4u) {
      const bool is_q = n < a.q_heads, is_k = !is_q && n < a.q_heads + a.kv_heads;
      const uint32_t head = is_q ? n : is_k ? n - a.q_heads : n - a.q_heads - a.kv_heads;
      const uint64_t in_cache = at + head * a.head_stride;
      if (!is_q && !is_k) {
        const T* from = v + token * a.v_stride + (uint64_t)head * a.head_dim;
        if (stored)
          for (uint32_t i = lane; i < a.head_dim; i += 64u) v_cache[in_cache + i] = from[i];
        continue;
      }
      const T* const x = (is_q ? q + token * a.q_stride : k + token * a.k_stride) + (uint64_t)head * a.head_dim;
      const T* const w = is_q ? wq : wk;
      T* const y = is_q ? q_out + token * a.q_out_stride + (uint64_t)head * a.head_dim
                        : k_out ? k_out + token * a.k_out_stride + (uint64_t)head * a.head_dim : nullptr;
      T* const also = !is_q && stored ? k_cache + in_cache : nullptr;
      float r = 1.0f;
      if (a.norm) {
        float sum = 0.0f;
        for (uint32_t i = lane; i < a.head_dim; i += 64u) {
          const float e = widened(x[i]);
          sum = __builtin_fmaf(e, e, sum);
        }
        r = 1.0f / __builtin_sqrtf(wave_sum(sum) / (float)a.head_dim + a.eps);
      }
      auto normed = [&](uint32_t i) {
        const float e = widened(x[i]);
        return !a.norm ? e : w ? e * r * widened(w[i]) : e * r;
      };
      auto put = [&](uint32_t i, float e) {
        const T o = narrowed<T>(e);
        if (y) y[i] = o;
        if (also) also[i] = o;
      };
      for (uint32_t p = lane; p < pairs; p += 64u) {
        const uint32_t i = pair_first(a, p), j = pair_second(a, p);
        const float ui = normed(i), uj = normed(j);
        const tiler::f32x2_pair cs = turns[p];
        put(i, __builtin_fmaf(ui, cs.x, -(uj * cs.y)));
        put(j, __builtin_fmaf(uj, cs.x, ui * cs.y));
      }
      for (uint32_t i = a.rotary + lane; i < a.head_dim; i += 64u) put(i, normed(i));
    }
  }
}

// Its gradients, in the same manner; the first q_groups workgroups take the
// queries', the others the keys'.  A lane adds up its own elements of dw in LDS, its wave's share, and the
// workgroup writes one row of partial sums.
template <typename T>
__device__ __forceinline__ void rotate_grad_any(const TilerHeads& a, const T* dq_out, const T* dk_out, const T* q,
                                                const T* k, const T* wq, const T* wk, const int32_t* positions,
                                                const double* frequencies, T* dq, T* dk, float* partials_q, float* partials_k) {
  __shared__ tiler::f32x2_pair turns[kMostPairs];
  __shared__ float sums[4][2 * kMostPairs];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, pairs = a.rotary / 2u;
  const bool is_q = blockIdx.x < a.q_groups;
  const uint32_t block = is_q ? blockIdx.x : blockIdx.x - a.q_groups, blocks = is_q ? a.q_groups : gridDim.x - a.q_groups;
  const uint32_t heads = is_q ? a.q_heads : a.kv_heads;
  const uint64_t x_stride = is_q ? a.q_stride : a.k_stride, dy_stride = is_q ? a.q_out_stride : a.k_out_stride;
  const T *const xs = is_q ? q : k, *const dys = is_q ? dq_out : dk_out, *const w = is_q ? wq : wk;
  T* const dxs = is_q ? dq : dk;
  float* const partials = is_q ? partials_q : partials_k;
  if (!dxs && !partials) return;
  for (uint32_t i = lane; i < a.head_dim; i += 64u) sums[wave][i] = 0.0f;
  for (uint64_t token = block; token < a.tokens; token += blocks) {
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < pairs; p += 256u) turns[p] = turn_of((double)positions[token] * frequencies[p]);
    __syncthreads();
    for (uint32_t head = wave; head < heads; head += 4u) {
      const T* const dy = dys + token * dy_stride + (uint64_t)head * a.head_dim;
      const T* const x = a.norm ? xs + token * x_stride + (uint64_t)head * a.head_dim : nullptr;
      T* const dx = dxs ? dxs + token * x_stride + (uint64_t)head * a.head_dim : nullptr;
      auto weight = [&](uint32_t i) { return w ? widened(w[i]) : 1.0f; };
      // each element with its gradient of the rotation's input
      auto each = [&](auto f) {
        for (uint32_t p = lane; p < pairs; p += 64u) {
          const uint32_t i = pair_first(a, p), j = pair_second(a, p);
          const float di = widened(dy[i]), dj = widened(dy[j]);
          const tiler::f32x2_pair cs = turns[p];
          f(i, __builtin_fmaf(di, cs.x, dj * cs.y));
          f(j, __builtin_fmaf(dj, cs.x, -(di * cs.y)));
        }
        for (uint32_t i = a.rotary + lane; i < a.head_dim; i += 64u) f(i, widened(dy[i]));
      };
      if (!a.norm) {
        each([&](uint32_t i, float g) { dx[i] = narrowed<T>(g); });
        continue;
      }
      float squares = 0.0f, along = 0.0f;
      each([&](uint32_t i, float g) {
        const float e = widened(x[i]);
        squares = __builtin_fmaf(e, e, squares);
        along = __builtin_fmaf(g * weight(i), e, along);
      });
      const float r = 1.0f / __builtin_sqrtf(wave_sum(squares) / (float)a.head_dim + a.eps);
      const float mean = wave_sum(along) * r / (float)a.head_dim;
      each([&](uint32_t i, float g) {
        const float xh = widened(x[i]) * r;
        if (dx) dx[i] = narrowed<T>(r * __builtin_fmaf(-xh, mean, g * weight(i)));
        if (partials) sums[wave][i] = __builtin_fmaf(g, xh, sums[wave][i]);
      });
    }
  }
  if (!partials) return;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.head_dim; i += 256u)
    partials[(uint64_t)block * a.head_dim + i] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// Heads in registers: a unit is two 16-byte pieces of a head, a lane's, and L lanes
// hold a head (2 L pieces at least; lanes past its end idle).  In the rotated part a
// unit is kVec pairs whichever way they lie: pieces u and u + rotary / (2 kVec), or 2 u
// and 2 u + 1; behind it, the next two pieces.  Any alignment: memory takes unaligned
// vectors.  A token's angles are made once, by the workgroup, into LDS.
template <typename T, bool kNeighbours>
struct Unit {
  static constexpr uint32_t V = tiler_rows::kVec<T>;
  uint32_t first, second;  // elements; second past the head where there is no second piece
  uint32_t pair;           // the unit's first pair
  bool rotated, there, both;
  __device__ __forceinline__ Unit(const TilerHeads& a, uint32_t u) {
    const uint32_t turned = a.rotary / (2u * V);
    rotated = u < turned;
    pair = u * V;
    first = !rotated ? a.rotary + (u - turned) * 2u * V : kNeighbours ? 2u * u * V : u * V;
    second = rotated && !kNeighbours ? first + a.rotary / 2u : first + V;
    there = first < a.head_dim;
    both = there && second < a.head_dim;
  }
};

template <typename T>
struct Pieces {
  static constexpr int V = tiler_rows::kVec<T>;
  u32x4 a, b;
  template <typename U>
  __device__ __forceinline__ void load(const T* head, const U& u) {
    a = b = u32x4{0, 0, 0, 0};
    if (u.there) a = *reinterpret_cast<const tiler_rows::u32x4_any*>(head + u.first);
    if (u.both) b = *reinterpret_cast<const tiler_rows::u32x4_any*>(head + u.second);
  }
  template <typename U>
  __device__ __forceinline__ void store(T* head, const U& u) const {
    if (u.there) *reinterpret_cast<tiler_rows::u32x4_any*>(head + u.first) = a;
    if (u.both) *reinterpret_cast<tiler_rows::u32x4_any*>(head + u.second) = b;
  }
  __device__ __forceinline__ void widen(float (&x)[2 * V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = tiler_rows::element<T>(a, e), x[V + e] = tiler_rows::element<T>(b, e);
  }
  __device__ __forceinline__ void narrow(const float (&x)[2 * V]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 2) {
        a[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((tiler::f32x2_pair{x[2 * e], x[2 * e + 1]}), tiler::bf16x2_pair));
        b[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((tiler::f32x2_pair{x[V + 2 * e], x[V + 2 * e + 1]}), tiler::bf16x2_pair));
      } else {
        a[e] = __float_as_uint(x[e]);
        b[e] = __float_as_uint(x[V + e]);
      }
    }
  }
};

// The unit's pairs turned, by the angle or back.
template <int V, bool kNeighbours>
__device__ __forceinline__ void turn(float (&x)[2 * V], const tiler::f32x2_pair* turns, bool back) {
  tiler::f32x2_pair cs[V];
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const f32x4 two = *reinterpret_cast<const f32x4*>(turns + e);
    cs[e] = tiler::f32x2_pair{two.x, back ? -two.y : two.y};
    cs[e + 1] = tiler::f32x2_pair{two.z, back ? -two.w : two.w};
  }
  if constexpr (kNeighbours) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float i = x[2 * e], j = x[2 * e + 1];
      x[2 * e] = __builtin_fmaf(i, cs[e].x, -(j * cs[e].y));
      x[2 * e + 1] = __builtin_fmaf(j, cs[e].x, i * cs[e].y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float i = x[e], j = x[V + e];
      x[e] = __builtin_fmaf(i, cs[e].x, -(j * cs[e].y));
      x[V + e] = __builtin_fmaf(j, cs[e].x, i * cs[e].y);
    }
  }
}

// Sum over groups of L lanes, in every lane of the group.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  auto moved = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += moved(v, tiler::Step<0xB1>{});                         // quad_perm [1,0,3,2]
  v += moved(v, tiler::Step<0x4E>{});                         // quad_perm [2,3,0,1]
  if constexpr (L >= 8) v += moved(v, tiler::Step<0x141>{});  // row_half_mirror
  if constexpr (L >= 16) v += moved(v, tiler::Step<0x140>{}); // row_mirror
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

constexpr uint32_t kTurnPairs = 2048;  // angles a workgroup holds: of 4 tokens of 512 pairs

// Head n of a token: of its queries, its keys or its values.
template <typename T>
__device__ __forceinline__ const T* head_at(const TilerHeads& a, const T* q, const T* k, const T* v, uint64_t token, uint32_t n) {
  if (n < a.q_heads) return q + token * a.q_stride + (uint64_t)n * a.head_dim;
  n -= a.q_heads;
  if (n < a.kv_heads) return k + token * a.k_stride + (uint64_t)n * a.head_dim;
  return v + token * a.v_stride + (uint64_t)(n - a.kv_heads) * a.head_dim;
}

// The workgroup's tokens are `each` at a time; their tasks, heads, go round the groups
// of L lanes of the blockIdx.y workgroups that share them (few tokens: one task a group).
// A task's head is read ahead, the first one before the angles.  HBM bounds it: 8192
// tokens of 32 and 8 heads of 128 bf16 take 35 us on changing inputs (4.8 TB/s; f32 70),
// 173 in the form of any size; their gradients 56 (4.5 TB/s) and 5 for the sum of the
// partials (f32 107 in all), 334 in the form of any size; 4096 tokens and their values
// stored 24 (4.3 TB/s).  Inputs that lie in the last cache take 28 and 45.
template <typename T, int L, bool kNeighbours>
__device__ __forceinline__ void rotate_units(const TilerHeads& a, const T* __restrict__ q, const T* __restrict__ k,
                                             const T* __restrict__ v, const T* __restrict__ wq, const T* __restrict__ wk,
                                             const int32_t* __restrict__ positions, const double* __restrict__ frequencies,
                                             T* __restrict__ q_out, T* __restrict__ k_out, T* __restrict__ k_cache,
                                             T* __restrict__ v_cache, const int32_t* __restrict__ slots) {
  constexpr int V = tiler_rows::kVec<T>;
  constexpr uint32_t kGroups = 256 / L;
  __shared__ __attribute__((aligned(16))) tiler::f32x2_pair turns[kTurnPairs];
  const uint32_t group = blockIdx.y * kGroups + threadIdx.x / L, step = gridDim.y * kGroups, pairs = a.rotary / 2u, each = a.each;
  const uint32_t heads = a.q_heads + a.kv_heads + (v ? a.kv_heads : 0u);
  const Unit<T, kNeighbours> unit(a, threadIdx.x % L);
  Pieces<T> of_q, of_k;
  if (wq) of_q.load(wq, unit);
  if (wk) of_k.load(wk, unit);
  for (uint64_t token0 = (uint64_t)blockIdx.x * each; token0 < a.tokens; token0 += (uint64_t)gridDim.x * each) {
    const uint32_t count = a.tokens - token0 < each ? (uint32_t)(a.tokens - token0) : each;
    uint32_t in = group / heads, n = group - in * heads;  // the task's token, and its head
    Pieces<T> ahead{};
    if (in < count) ahead.load(head_at(a, q, k, v, token0 + in, n), unit);
    if (token0 != (uint64_t)blockIdx.x * each) __syncthreads();  // the turns before are read
    for (uint32_t i = threadIdx.x; i < count * pairs; i += 256u) {
      const uint32_t t = i / pairs;
      turns[i] = turn_of((double)positions[token0 + t] * frequencies[i - t * pairs]);
    }
    __syncthreads();
    while (in < count) {
      const uint64_t token = token0 + in;
      const uint32_t of = in;
      const bool is_q = n < a.q_heads, is_k = !is_q && n < a.q_heads + a.kv_heads;
      const uint32_t head = is_q ? n : is_k ? n - a.q_heads : n - a.q_heads - a.kv_heads;
      Pieces<T> x = ahead;
      const int64_t slot = slots && !is_q ? slots[token] : -1;
      n += step;
      while (n >= heads) n -= heads, ++in;
      if (in < count) ahead.load(head_at(a, q, k, v, token0 + in, n), unit);
      if (is_q || is_k) {
        float u[2 * V];
        x.widen(u);
        if (a.norm) {
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) sum = __builtin_fmaf(u[e], u[e], sum);
          const float r = 1.0f / __builtin_sqrtf(group_sum<L>(sum) / (float)a.head_dim + a.eps);
          const bool weighted = is_q ? wq != nullptr : wk != nullptr;
          float w[2 * V];
          Pieces<T> wp;
#pragma unroll
          for (int e = 0; e < 4; ++e) wp.a[e] = is_q ? of_q.a[e] : of_k.a[e], wp.b[e] = is_q ? of_q.b[e] : of_k.b[e];
          wp.widen(w);
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) u[e] = weighted ? u[e] * r * w[e] : u[e] * r;
        }
        if (unit.rotated) turn<V, kNeighbours>(u, turns + of * pairs + unit.pair, false);
        x.narrow(u);
      }
      if (is_q) x.store(q_out + token * a.q_out_stride + (uint64_t)head * a.head_dim, unit);
      if (is_k && k_out) x.store(k_out + token * a.k_out_stride + (uint64_t)head * a.head_dim, unit);
      if (slot >= 0 && (uint64_t)slot < a.slots) {
        const uint32_t page = (uint32_t)slot / a.page, place = (uint32_t)slot - page * a.page;
        x.store((is_k ? k_cache : v_cache) + (uint64_t)page * a.page_stride + (uint64_t)place * a.token_stride + (uint64_t)head * a.head_stride, unit);
      }
    }
  }
}

// Its gradients.  The first a.q_groups workgroups have the queries' heads, the others
// the keys'.
template <typename T, int L, bool kNeighbours>
__device__ __forceinline__ void rotate_grad_units(const TilerHeads& a, const T* __restrict__ dq_out, const T* __restrict__ dk_out,
                                                  const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ wq,
                                                  const T* __restrict__ wk, const int32_t* __restrict__ positions,
                                                  const double* __restrict__ frequencies, T* __restrict__ dq, T* __restrict__ dk,
                                                  float* __restrict__ partials_q, float* __restrict__ partials_k) {
  constexpr int V = tiler_rows::kVec<T>;
  constexpr uint32_t kGroups = 256 / L;
  __shared__ __attribute__((aligned(16))) union {
    tiler::f32x2_pair turns[kTurnPairs];
    float sums[kGroups][2 * V * L];
  } space;
  const bool is_q = blockIdx.x < a.q_groups;
  const uint32_t block = is_q ? blockIdx.x : blockIdx.x - a.q_groups, blocks = is_q ? a.q_groups : gridDim.x - a.q_groups;
  const uint32_t group = threadIdx.x / L, pairs = a.rotary / 2u, each = a.each, heads = is_q ? a.q_heads : a.kv_heads;
  const uint64_t x_stride = is_q ? a.q_stride : a.k_stride, dy_stride = is_q ? a.q_out_stride : a.k_out_stride;
  const T *const xs = is_q ? q : k, *const dys = is_q ? dq_out : dk_out, *const w = is_q ? wq : wk;
  T* const dxs = is_q ? dq : dk;
  float* const partials = is_q ? partials_q : partials_k;
  const Unit<T, kNeighbours> unit(a, threadIdx.x % L);
  float weight[2 * V], dw[2 * V];
  {
    Pieces<T> of;
    if (w) of.load(w, unit);
    of.widen(weight);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) weight[e] = w ? weight[e] : 1.0f, dw[e] = 0.0f;
  }
  for (uint64_t token0 = (uint64_t)block * each; token0 < a.tokens; token0 += (uint64_t)blocks * each) {
    const uint32_t count = a.tokens - token0 < each ? (uint32_t)(a.tokens - token0) : each;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count * pairs; i += 256u) {
      const uint32_t t = i / pairs;
      space.turns[i] = turn_of((double)positions[token0 + t] * frequencies[i - t * pairs]);
    }
    __syncthreads();
    uint32_t in = group / heads, n = group - in * heads;
    while (in < count) {
      const uint64_t token = token0 + in;
      Pieces<T> dy, x;
      dy.load(dys + token * dy_stride + (uint64_t)n * a.head_dim, unit);
      if (a.norm) x.load(xs + token * x_stride + (uint64_t)n * a.head_dim, unit);
      float g[2 * V];
      dy.widen(g);
      if (unit.rotated) turn<V, kNeighbours>(g, space.turns + in * pairs + unit.pair, true);
      if (a.norm) {
        float e_x[2 * V], squares = 0.0f, along = 0.0f;
        x.widen(e_x);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          squares = __builtin_fmaf(e_x[e], e_x[e], squares);
          along = __builtin_fmaf(g[e] * weight[e], e_x[e], along);
        }
        const float r = 1.0f / __builtin_sqrtf(group_sum<L>(squares) / (float)a.head_dim + a.eps);
        const float mean = group_sum<L>(along) * r / (float)a.head_dim;
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const float xh = e_x[e] * r;
          dw[e] = __builtin_fmaf(g[e], xh, dw[e]);
          g[e] = r * __builtin_fmaf(-xh, mean, g[e] * weight[e]);
        }
      }
      if (dxs) {
        dy.narrow(g);
        dy.store(dxs + token * x_stride + (uint64_t)n * a.head_dim, unit);
      }
      n += kGroups;
      while (n >= heads) n -= heads, ++in;
    }
  }
  if (!partials) return;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (unit.there) space.sums[group][unit.first + e] = dw[e];
    if (unit.both) space.sums[group][unit.second + e] = dw[V + e];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.head_dim; i += 256u) {
    float s = 0.0f;
    for (uint32_t n = 0; n < kGroups; ++n) s += space.sums[n][i];
    partials[(uint64_t)block * a.head_dim + i] = s;
  }
}

// dw from the rows of partial sums: sixteen elements a workgroup, whose 64 groups
// of sixteen lanes each add every 64th row.  blockIdx.y: the queries' (0) or the keys'.
template <typename T>
__device__ __forceinline__ void rotate_sums(const float* partials_q, const float* partials_k, uint32_t count_q,
                                            uint32_t count_k, uint32_t head_dim, T* dwq, T* dwk) {
  __shared__ float waves[16][16];
  const float* const partials = blockIdx.y ? partials_k : partials_q;
  const uint32_t count = blockIdx.y ? count_k : count_q;
  T* const dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, i = blockIdx.x * 16u + (lane & 15u);
  float s = 0.0f;
  if (i < head_dim)
#pragma unroll 8
    for (uint32_t p = threadIdx.x >> 4; p < count; p += 64u) s += partials[(uint64_t)p * head_dim + i];
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if (lane < 16u) waves[wave][lane] = s;
  __syncthreads();
  if (threadIdx.x < 16u && i < head_dim) {
#pragma unroll
    for (int n = 1; n < 16; ++n) s += waves[n][lane];
    dw[i] = narrowed<T>(s);
  }
}

}  // namespace tiler_heads

#define TILER_NORM_ROTATE(TY, T)                                                                                      \
  extern "C" __global__ void __launch_bounds__(256) tiler_norm_rotate_##TY##_any(                                     \
      TilerHeads a, const T* q, const T* k, const T* v, const T* wq, const T* wk, const int32_t* positions,           \
      const double* frequencies, T* q_out, T* k_out, T* k_cache, T* v_cache, const int32_t* slots) {                  \
    tiler_heads::rotate_any<T>(a, q, k, v, wq, wk, positions, frequencies, q_out, k_out, k_cache, v_cache, slots);    \
  }                                                                                                                   \
  extern "C" __global__ void __launch_bounds__(256) tiler_norm_rotate_grad_##TY##_any(                                \
      TilerHeads a, const T* dq_out, const T* dk_out, const T* q, const T* k, const T* wq, const T* wk,               \
      const int32_t* positions, const double* frequencies, T* dq, T* dk, float* partials_q, float* partials_k) {      \
    tiler_heads::rotate_grad_any<T>(a, dq_out, dk_out, q, k, wq, wk, positions, frequencies, dq, dk, partials_q,      \
                                    partials_k);                                                                      \
  }                                                                                                                   \
  extern "C" __global__ void __launch_bounds__(1024) tiler_norm_rotate_sum_##TY(                                      \
      const float* partials_q, const float* partials_k, uint32_t count_q, uint32_t count_k, uint32_t head_dim,        \
      T* dwq, T* dwk) {                                                                                               \
    tiler_heads::rotate_sums<T>(partials_q, partials_k, count_q, count_k, head_dim, dwq, dwk);                        \
  }
TILER_NORM_ROTATE(bf16, uint16_t)
TILER_NORM_ROTATE(f32, float)
#undef TILER_NORM_ROTATE

#define TILER_NORM_ROTATE_UNITS(TY, T, L, FORM, NEIGHBOURS)                                                           \
  extern "C" __global__ void __launch_bounds__(256) tiler_norm_rotate_##TY##_##FORM(                                  \
      TilerHeads a, const T* q, const T* k, const T* v, const T* wq, const T* wk, const int32_t* positions,           \
      const double* frequencies, T* q_out, T* k_out, T* k_cache, T* v_cache, const int32_t* slots) {                  \
    tiler_heads::rotate_units<T, L, NEIGHBOURS>(a, q, k, v, wq, wk, positions, frequencies, q_out, k_out, k_cache,    \
                                                v_cache, slots);                                                      \
  }                                                                                                                   \
  extern "C" __global__ void __launch_bounds__(256) tiler_norm_rotate_grad_##TY##_##FORM(                             \
      TilerHeads a, const T* dq_out, const T* dk_out, const T* q, const T* k, const T* wq, const T* wk,               \
      const int32_t* positions, const double* frequencies, T* dq, T* dk, float* partials_q, float* partials_k) {      \
    tiler_heads::rotate_grad_units<T, L, NEIGHBOURS>(a, dq_out, dk_out, q, k, wq, wk, positions, frequencies, dq, dk, \
                                                     partials_q, partials_k);                                         \
  }
#define TILER_NORM_ROTATE_FORMS(TY, T, L)             \
  TILER_NORM_ROTATE_UNITS(TY, T, L, h##L, false)      \
  TILER_NORM_ROTATE_UNITS(TY, T, L, n##L, true)
#define TILER_NORM_ROTATE_LANES(L)          \
  TILER_NORM_ROTATE_FORMS(bf16, uint16_t, L) \
  TILER_NORM_ROTATE_FORMS(f32, float, L)
TILER_NORM_ROTATE_LANES(4)
TILER_NORM_ROTATE_LANES(8)
TILER_NORM_ROTATE_LANES(16)
TILER_NORM_ROTATE_LANES(32)
TILER_NORM_ROTATE_LANES(64)
#undef TILER_NORM_ROTATE_LANES
#undef TILER_NORM_ROTATE_FORMS
#undef TILER_NORM_ROTATE_UNITS
