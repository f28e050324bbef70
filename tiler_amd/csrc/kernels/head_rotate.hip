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

// (cos, sin) of an angle.  Its quarter turns come off in 64 bits, by pi / 2 in two
// parts (a fused product is exact before its one rounding); the series for what
// remains, |r| <= pi / 4, go to r^9 and r^10 and leave out less than 3e-8 of it.
__device__ __forceinline__ tiler::f32x2_pair turn_of(double angle) {
  const double quarters = __builtin_rint(angle * 0.63661977236758134308);
  double left = __builtin_fma(-quarters, 1.57079632679489655800, angle);
  left = __builtin_fma(-quarters, 6.12323399573676603587e-17, left);
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
  const uint32_t turn = (uint32_t)(long long)quarters & 3u;
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
// element a load; the head is read twice.
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

// Its gradients, in the same manner; blockIdx.y: the queries' (0) or the keys'.
// A lane adds up its own elements of dw in LDS, its wave's share, and the
// workgroup writes one row of partial sums.
template <typename T>
__device__ __forceinline__ void rotate_grad_any(const TilerHeads& a, const T* dq_out, const T* dk_out, const T* q,
                                                const T* k, const T* wq, const T* wk, const int32_t* positions,
                                                const double* frequencies, T* dq, T* dk, float* partials_q, float* partials_k) {
  __shared__ tiler::f32x2_pair turns[kMostPairs];
  __shared__ float sums[4][2 * kMostPairs];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, pairs = a.rotary / 2u;
  const bool is_q = blockIdx.y == 0;
  const uint32_t heads = is_q ? a.q_heads : a.kv_heads;
  const uint64_t x_stride = is_q ? a.q_stride : a.k_stride, dy_stride = is_q ? a.q_out_stride : a.k_out_stride;
  const T *const xs = is_q ? q : k, *const dys = is_q ? dq_out : dk_out, *const w = is_q ? wq : wk;
  T* const dxs = is_q ? dq : dk;
  float* const partials = is_q ? partials_q : partials_k;
  if (!dxs && !partials) return;
  for (uint32_t i = threadIdx.x; i < 4u * 2u * kMostPairs; i += 256u) (&sums[0][0])[i] = 0.0f;
  for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
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
    partials[(uint64_t)blockIdx.x * a.head_dim + i] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// dw from the rows of partial sums: 64 elements a workgroup, sixteen waves that
// each add every sixteenth row.  blockIdx.y: the queries' (0) or the keys'.
template <typename T>
__device__ __forceinline__ void rotate_sums(const float* partials_q, const float* partials_k, uint32_t count_q,
                                            uint32_t count_k, uint32_t head_dim, T* dwq, T* dwk) {
  __shared__ float waves[16][64];
  const float* const partials = blockIdx.y ? partials_k : partials_q;
  const uint32_t count = blockIdx.y ? count_k : count_q;
  T* const dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, i = blockIdx.x * 64u + lane;
  float s = 0.0f;
  if (i < head_dim)
#pragma unroll 8
    for (uint32_t p = wave; p < count; p += 16u) s += partials[(uint64_t)p * head_dim + i];
  waves[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && i < head_dim) {
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
