// Rows held in registers by a group of WAVES waves, 16-byte pieces at any
// alignment: piece c of thread t of the group starts at element
// (c 64 WAVES + t) kVec of its row (kVec = 8 bf16 or 4 f32), so each load
// instruction of a wave covers 1 KiB of contiguous row.
#pragma once

#include "pieces.h"

namespace tiler_rows {

using tiler_pieces::u32_any;
using tiler_pieces::u32x2_any;
using tiler_pieces::u32x4_any;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// Element e of a piece, widened.
template <typename T>
__device__ __forceinline__ float element(const u32x4& v, int e) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
  else return __uint_as_float(v[e]);
}

// How many of the elements from `at` lie in the row.
template <typename T>
__device__ __forceinline__ uint32_t valid_from(uint32_t at, uint32_t extent) {
  return at >= extent ? 0u : extent - at < (uint32_t)kVec<T> ? extent - at : (uint32_t)kVec<T>;
}

// A thread's CH pieces of a row (of at least kVec elements) in two steps, so
// that no branch stands between the loads: load_row reads a whole piece each,
// those that would pass the row's end the last one inside it; settle_row moves
// their elements into place and clears what lies past the end.  kStream: read
// once, past the caches.
template <typename T, int WAVES, int CH, bool kStream>
__device__ __forceinline__ void load_row(const T* row, uint32_t t, uint32_t extent, u32x4 (&v)[CH]) {
  constexpr uint32_t V = kVec<T>;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t at = (c * 64u * WAVES + t) * V;
    const u32x4_any* p = reinterpret_cast<const u32x4_any*>(row + (at + V <= extent ? at : extent - V));
    v[c] = kStream ? __builtin_nontemporal_load(p) : *p;
  }
}
template <typename T, int WAVES, int CH>
__device__ __forceinline__ void settle_row(uint32_t t, uint32_t extent, u32x4 (&v)[CH]) {
  constexpr uint32_t V = kVec<T>;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t at = (c * 64u * WAVES + t) * V;
    if (at + V > extent) v[c] = at >= extent ? u32x4{0, 0, 0, 0}
                                             : tiler_pieces::drop_bytes(v[c], (at + V - extent) * (uint32_t)sizeof(T));
  }
}

// Narrows and stores the piece's elements inside the row.  A NaN is looked for
// two values at a time (an unordered comparison) and made canonical where there
// is one.
template <typename T>
__device__ __forceinline__ void store_piece(T* row, uint32_t at, uint32_t extent, float (&o)[kVec<T>]) {
  const uint32_t valid = valid_from<T>(at, extent);
  bool nan = false;
#pragma unroll
  for (int e = 0; e < kVec<T>; e += 2) nan |= __builtin_isunordered(o[e], o[e + 1]);
  if (nan) {
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) o[e] = tiler::canon(o[e]);
  }
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 2)
      v[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((tiler::f32x2_pair{o[2 * e], o[2 * e + 1]}), tiler::bf16x2_pair));
    else v[e] = __float_as_uint(o[e]);
  }
  if (valid == (uint32_t)kVec<T>) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(row + at));
    return;
  }
#pragma unroll
  for (int e = 0; e < kVec<T> - 1; ++e)
    if ((uint32_t)e < valid) {
      if constexpr (sizeof(T) == 2) row[at + e] = (T)(v[e >> 1] >> (16 * (e & 1)));
      else row[at + e] = __uint_as_float(v[e]);
    }
}

// Sum of a kVec run, in pairs.
template <int N>
__device__ __forceinline__ float pairwise(const float (&v)[N]) {
  if constexpr (N == 8) return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  else return (v[0] + v[1]) + (v[2] + v[3]);
}

// A wave's fold of v under f, the same value in every lane: within each row of
// 16 lanes by four data-parallel moves (lanes i ^ 1, i ^ 2, 7 - i, 15 - i), then
// the four rows' values, read through scalar registers.  No LDS round trips.
template <typename V, typename F>
__device__ __forceinline__ V wave_fold(V v, F f) {
  auto moved = [](V x, auto ctrl) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = f(v, moved(v, tiler::Step<0xB1>{}));   // quad_perm [1,0,3,2]
  v = f(v, moved(v, tiler::Step<0x4E>{}));   // quad_perm [2,3,0,1]
  v = f(v, moved(v, tiler::Step<0x141>{}));  // row_half_mirror
  v = f(v, moved(v, tiler::Step<0x140>{}));  // row_mirror
  auto lane = [&](int l) { return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
  return f(f(lane(0), lane(16)), f(lane(32), lane(48)));
}

// Two sums over a group of WAVES waves, the same values in every lane.  The
// waves of one workgroup all call it; `slots` holds 2 floats per wave, and a
// caller alternates between two such arrays from call to call, so that one
// barrier a call is enough.
template <int WAVES>
__device__ __forceinline__ void group_sums(float& a, float& b, float* slots) {
  auto add = [](float p, float q) { return p + q; };
  a = wave_fold(a, add);
  b = wave_fold(b, add);
  if constexpr (WAVES > 1) {
    const uint32_t wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
    if ((threadIdx.x & 63u) == 0) {
      slots[2u * wave] = a;
      slots[2u * wave + 1u] = b;
    }
    __syncthreads();
    float sa[WAVES], sb[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      sa[w] = slots[2u * (first + w)];
      sb[w] = slots[2u * (first + w) + 1u];
    }
#pragma unroll
    for (int s = 1; s < WAVES; s *= 2)
#pragma unroll
      for (int w = 0; w + s < WAVES; w += 2 * s) {
        sa[w] += sa[w + s];
        sb[w] += sb[w + s];
      }
    a = sa[0];
    b = sb[0];
  }
}

}  // namespace tiler_rows
