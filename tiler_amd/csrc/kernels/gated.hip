// The gated feed-forward product and its gradients for gfx950, bf16 on MFMA
// with f32 accumulation:
//
//   G = x Wg^T, U = x Wu^T, h = silu(G) U          (x [m, k]; Wg, Wu [n, k])
//   dU = dh silu(G), dG = dh U s (1 + G (1 - s))    s = 1 / (1 + e^-G)
//   dx = dG Wg + dU Wu, dWg = dG^T x, dWu = dU^T x
//
// Forward: one kernel reads x once for both projections; a wave's columns are
// half gate, half up (the same 32 of each), so both sums of an output meet in
// one lane's registers and the activation and the product need no exchange.
// h is taken from the f32 sums and rounded once; G and U, where kept, are the
// same sums rounded once.
//
// Backward: dG and dU are formed once per element from the kept G and U and
// rounded to bf16 (the matrix pipe's operand type; one rounding of each term
// of a sum, as independent as the terms), then dx contracts them with the
// weights as they lie (the weights' rows are its depth) and dWg, dWu with x
// over the tokens (both operands in column layout).
//
// us, 4096 x 14336 x 4096, by the card: forward with G and U kept 750 .. 767 (1.26
// .. 1.28 PFLOP/s: the matrix pipe under the power limit, as a plain library product
// of the size), its gradients 1515 .. 1552, of them dG and dU 96 (587 MB, 6 TB/s),
// dx and the weights' gradients half the rest each.  16 tokens 45: the weights'
// 235 MB.
#include "product.h"

namespace {

using tiler_product::Bf16;
using tiler_product::Operand;
using tiler_product::kSlice;

// e^-G by the hardware exponential; 1 / (1 + e) by the hardware reciprocal.  The
// exponent rounds twice, so that the relative error grows as |G| 2^-24: a few
// binary32 steps near zero, 17 bits left at G = -80.  +-inf and NaN as the formula
// gives them.
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -0x1.715476p+0f));
}
// From here down e^-G nears the end of binary32's range (it passes it at -88.7, where
// silu(G) v need not be small): there s is e^G to the last bit, 1 - s is 1, and s
// goes into the products as e^(G / 2) twice.  That is zero below G = -174.7 (silu(G)
// 10^-74).  Tested for an element, or for the largest bits of four or eight: 4096 x
// 14336 x 4096 with G and U kept 759.5 -> 762.5 us, the gradients as before; all
// elements by e^(-|G| / 2), without a test, 1% more.
constexpr float kFarGate = -80.0f;
constexpr uint32_t kFarGateBits = 0xc2a00000u;  // below kFarGate, negative: larger bits (a NaN's too)
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float far_factor(float g) { return __builtin_amdgcn_exp2f(g * 0x1.715476p-1f); }
__device__ __forceinline__ float far_silu_times(float g, float v) {
  const float f = far_factor(g);
  return g * f * (f * v);
}
// silu(G) v
__device__ __forceinline__ float silu_times(float g, float v) {
  return g < kFarGate ? far_silu_times(g, v) : g * sigmoid(g) * v;
}
__device__ __forceinline__ f32x4 silu_times(const f32x4& g, const f32x4& v) {
  f32x4 h;
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = g[e] * sigmoid(g[e]) * v[e];
  const u32x4 bits = __builtin_bit_cast(u32x4, g);
  if (larger(larger(larger(bits[0], bits[1]), bits[2]), bits[3]) > kFarGateBits) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (g[e] < kFarGate) h[e] = far_silu_times(g[e], v[e]);
  }
  return h;
}

// Guarded form: 128 (or 64) tokens x (64 gate + 64 up) columns, any sizes and
// alignments.  Row r of the B tile: gate (r & 32 == 0) or up row
// (r >> 6) * 32 + (r & 31) of the 64-column tile.
constexpr int kW = 2, kNB = 4;  // 2 x 2 waves of MB x 4 blocks, MB 4 or 2

// Rows of dG and dU, and of the copies of x and the weights in the backward pass.
__device__ __forceinline__ uint32_t row_of_mid(uint32_t n) { return (n + 63u) & ~63u; }
__device__ __forceinline__ uint32_t row_of_copy(uint32_t k) { return (k + 7u) & ~7u; }
__device__ __forceinline__ uint64_t quotient(uint64_t v, uint32_t by) {  // a 64-bit division costs five of 32
  return v >> 32 ? v / by : (uint32_t)v / by;
}

template <int MB>
__device__ __forceinline__ void gated_guarded(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,
                                              const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k,
                                              uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                                              uint16_t* __restrict__ up) {
  constexpr uint32_t kRows = kW * MB * 16u;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2u * (kRows + 128u) * kSlice];
  const uint32_t m0 = blockIdx.y * kRows, n0 = blockIdx.x * 64u;
  // thread t's pieces of B are rows t / 8 + 32 q of its tile: gate rows for even q, up rows for odd
  const Operand a{reinterpret_cast<const uint8_t*>(x), m, k}, b{reinterpret_cast<const uint8_t*>(wg), n, k};
  f32x4 acc[MB][kNB];
  // (lb fetches 64 rows of either weight, whole lays the 128 of the tile out)
  auto product = [&](const auto& la, const auto& lb, const auto& whole) {
    tiler_product::guarded_product<Bf16, kW, kW, MB, kNB>(
        smem, (k + 63u) / 64u, [&](uint32_t t, u32x4(&v)[MB]) { la.load(a.base, t, v); },
        [&](uint32_t t, u32x4(&v)[4]) {
          u32x4 g[2], u[2];
          lb.load(reinterpret_cast<const uint8_t*>(wg), t, g);
          lb.load(reinterpret_cast<const uint8_t*>(wu), t, u);
          v[0] = g[0], v[1] = u[0], v[2] = g[1], v[3] = u[1];
        },
        [&](uint32_t t, uint8_t* tile, u32x4(&v)[MB]) { la.store(t, tile, v); },
        [&](uint32_t t, uint8_t* tile, u32x4(&v)[4]) { whole.store(t, tile, v); },
        acc);
  };
  using tiler_product::GuardedLoader;
  using tiler_product::TinyLoader;
  if (k >= 8u)
    product(GuardedLoader<Bf16, kRows, 256>(a, m0), GuardedLoader<Bf16, 64, 256>(b, n0),
            GuardedLoader<Bf16, 128, 256>(b, n0));
  else
    product(TinyLoader<Bf16, kRows, 256>(a, m0), TinyLoader<Bf16, 64, 256>(b, n0),
            TinyLoader<Bf16, 128, 256>(b, n0));
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t row = m0 + (wave / kW) * MB * 16u + i * 16u + (lane >> 4) * 4u + r;
        const uint32_t col = n0 + (wave % kW) * 32u + j * 16u + (lane & 15u);
        if (row >= m || col >= n) continue;
        const float g = acc[i][j][r], u = acc[i][j + 2][r];
        const uint64_t at = (uint64_t)row * n + col;
        h[at] = (uint16_t)tiler::bf16_narrow(silu_times(g, u));
        if (gate) {
          gate[at] = (uint16_t)tiler::bf16_narrow(g);
          up[at] = (uint16_t)tiler::bf16_narrow(u);
        }
      }
}

}  // namespace

// Tiles of 128 and of 64 tokens.
extern "C" __global__ void __launch_bounds__(256, 2)
tiler_gated_bf16_g128(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg, const uint16_t* __restrict__ wu,
                      uint32_t m, uint32_t n, uint32_t k, uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                      uint16_t* __restrict__ up) {
  gated_guarded<4>(x, wg, wu, m, n, k, h, gate, up);
}
extern "C" __global__ void __launch_bounds__(256, 2)
tiler_gated_bf16_g64(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg, const uint16_t* __restrict__ wu,
                     uint32_t m, uint32_t n, uint32_t k, uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                     uint16_t* __restrict__ up) {
  gated_guarded<2>(x, wg, wu, m, n, k, h, gate, up);
}

// dG and dU (behind dG) of one row's eight columns per item, into rows of n
// rounded up to 64 (the columns past n are written as zeros): the first `forming`
// workgroups; the others copy.  Where the rows of
// x or of the weights do not start on 16 bytes, they are copied to rows that do,
// of k rounded up to 8, so that the products always run staged: gradients of
// 4096 x 14336 x 4095, us, 226 + 712 + 741; with the products' operands through
// registers instead (as the forward pass's guarded form) 112 + 1395 + 1349.
extern "C" __global__ void __launch_bounds__(256)
tiler_gated_bf16_grad(const uint16_t* __restrict__ gate, const uint16_t* __restrict__ up,
                      const uint16_t* __restrict__ dh, const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,
                      const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k, uint32_t forming,
                      uint16_t* __restrict__ dg, uint16_t* __restrict__ to_x, uint16_t* __restrict__ to_w) {
  using tiler_pieces::guarded_piece;
  using tiler_pieces::u32x4_any;
  const uint32_t ld = row_of_mid(n), per = ld / 8u, ldk = row_of_copy(k), per_k = ldk / 8u;
  const uint64_t mids = (uint64_t)m * per, copies = ((to_x ? (uint64_t)m : 0u) + (to_w ? 2ull * n : 0u)) * per_k;
  if (blockIdx.x >= forming) {
    for (uint64_t id = (blockIdx.x - forming) * 256ull + threadIdx.x; id < copies; id += (gridDim.x - forming) * 256ull) {
      uint64_t row = quotient(id, per_k);
      const uint32_t col = (uint32_t)(id - row * per_k) * 8u;
      const uint16_t* from = x;
      uint16_t* to = to_x;
      if (!to_x || row >= m) {
        if (to_x) row -= m;
        from = row >= n ? wu : wg;
        to = to_w + (row >= n ? (uint64_t)n * ldk : 0u);
        if (row >= n) row -= n;
      }
      const uint32_t valid = k - col < 8u ? (k - col) * 2u : 16u;
      *reinterpret_cast<u32x4*>(to + row * ldk + col) = guarded_piece(
          reinterpret_cast<const uint8_t*>(from + row * k + col), valid, reinterpret_cast<const uint8_t*>(from));
    }
    return;
  }
  for (uint64_t id = blockIdx.x * 256ull + threadIdx.x; id < mids; id += forming * 256ull) {
    const uint32_t row = (uint32_t)quotient(id, per), col = (uint32_t)(id - (uint64_t)row * per) * 8u;
    const uint64_t at = (uint64_t)row * n + col;
    const uint32_t valid = col >= n ? 0u : n - col < 8u ? (n - col) * 2u : 16u;
    u32x4 vg = {0, 0, 0, 0}, vu = vg, vd = vg;
    if (valid == 16u) {
      vg = *reinterpret_cast<const u32x4_any*>(gate + at);
      vu = *reinterpret_cast<const u32x4_any*>(up + at);
      vd = *reinterpret_cast<const u32x4_any*>(dh + at);
    } else if (valid) {
      auto piece = [&](const uint16_t* q) {
        return guarded_piece(reinterpret_cast<const uint8_t*>(q + at), valid, reinterpret_cast<const uint8_t*>(q));
      };
      vg = piece(gate);
      vu = piece(up);
      vd = piece(dh);
    }
    u32x4 og, ou;
    auto value = [](const u32x4& v, int e) { return tiler::bf16_widen((v[e >> 1] >> (16 * (e & 1))) & 0xffffu); };
    float g2[8], u2[8];
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float g = value(vg, e), u = value(vu, e), d = value(vd, e), s = sigmoid(g);
      g2[e] = d * u * s * (1.0f + g * (1.0f - s));
      u2[e] = d * g * s;
      bits = larger(bits, __float_as_uint(g));
    }
    if (bits > kFarGateBits) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = value(vg, e), d = value(vd, e), f = far_factor(g);
        if (g < kFarGate) {
          g2[e] = f * d * value(vu, e) * (f * (1.0f + g));
          u2[e] = far_silu_times(g, d);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      og[e] = tiler::bf16_pack2_rne(g2[2 * e], g2[2 * e + 1]);
      ou[e] = tiler::bf16_pack2_rne(u2[2 * e], u2[2 * e + 1]);
    }
    const uint64_t to = (uint64_t)row * ld + col;
    *reinterpret_cast<u32x4*>(dg + to) = og;
    *reinterpret_cast<u32x4*>(dg + (uint64_t)m * ld + to) = ou;
  }
}

// Where the depth is split over `splits` workgroups a tile (blockIdx.y): this
// one's slices.
__device__ __forceinline__ void split_range(uint32_t slices, uint32_t splits, uint32_t s, uint32_t& t0, uint32_t& t1) {
  t0 = (uint32_t)((uint64_t)slices * s / splits);
  t1 = (uint32_t)((uint64_t)slices * (s + 1u) / splits);
}

// A wave's blocks as binary32 partials of the m x n result.
template <int MB, int NB>
__device__ __forceinline__ void store_partial(const f32x4 (&acc)[MB][NB], float* out, uint32_t m, uint32_t n, uint32_t row0,
                                              uint32_t col0) {
  const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t row = row0 + i * 16u + (lane >> 4) * 4u + r, col = col0 + j * 16u + (lane & 15u);
        if (row < m && col < n) out[(uint64_t)row * n + col] = acc[i][j][r];
      }
}

// Gradients from the partials of the products whose depth is split, each in
// ascending order: `count_x` elements of dx, `count_w` of either weight's
// gradient (0: not split).  Four to a thread.
extern "C" __global__ void __launch_bounds__(256)
tiler_gated_bf16_sum(const float* __restrict__ of_x, uint32_t splits_x, uint64_t count_x, uint16_t* __restrict__ dx,
                     const float* __restrict__ of_w, uint32_t splits_w, uint64_t count_w, uint16_t* __restrict__ dwg,
                     uint16_t* __restrict__ dwu) {
  const uint64_t pieces_x = (count_x + 3u) / 4u, pieces_w = (count_w + 3u) / 4u, total = pieces_x + 2u * pieces_w;
  for (uint64_t id = blockIdx.x * 256ull + threadIdx.x; id < total; id += gridDim.x * 256ull) {
    const bool is_x = id < pieces_x, second = !is_x && id - pieces_x >= pieces_w;
    const uint64_t at = (is_x ? id : id - pieces_x - (second ? pieces_w : 0u)) * 4u, count = is_x ? count_x : count_w;
    const uint64_t stride = is_x ? count_x : 2u * count_w;
    const uint32_t splits = is_x ? splits_x : splits_w;
    const float* from = (is_x ? of_x : of_w + (second ? count_w : 0u)) + at;
    uint16_t* to = (is_x ? dx : second ? dwu : dwg) + at;
    if (count - at >= 4u) {
      f32x4 s = __builtin_bit_cast(f32x4, *reinterpret_cast<const tiler_pieces::u32x4_any*>(from));
#pragma unroll 4
      for (uint32_t p = 1; p < splits; ++p) {
        const f32x4 v = __builtin_bit_cast(f32x4, *reinterpret_cast<const tiler_pieces::u32x4_any*>(from + p * stride));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
      }
      *reinterpret_cast<tiler_pieces::u32x2_any*>(to) = u32x2{tiler::bf16_pack2_rne(s[0], s[1]), tiler::bf16_pack2_rne(s[2], s[3])};
    } else {
      for (uint64_t e = 0; e < count - at; ++e) {
        float s = from[e];
        for (uint32_t p = 1; p < splits; ++p) s += from[p * stride + e];
        to[e] = (uint16_t)tiler::bf16_narrow(s);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Staged forms: rows that start on 16 bytes.  WM x WN waves
// of MB x 4 blocks.
namespace {

template <int WM, int WN, int MB, int S>
__device__ __forceinline__ void gated_staged(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,
                                             const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k,
                                             uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                                             uint16_t* __restrict__ up) {
  constexpr uint32_t kRowsA = WM * MB * 16u, kRowsB = WN * 64u, kCols = kRowsB / 2u, kThreads = 64u * WM * WN;
  constexpr int kLoadsA = (kRowsA / 8 + WM * WN - 1) / (WM * WN), kLoadsB = kRowsB / 8 / (WM * WN);
  static_assert(kLoadsB == 4 || kLoadsB == 2, "a wave's rows of B lie in one of the two weights");
  constexpr bool kUneven = kRowsA % (8 * WM * WN) != 0;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * (kRowsA + kRowsB) * kSlice + (kUneven ? 1024u : 0u)];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t tm, tn;
  tiler_product::tile_of(blockIdx.x, (m + kRowsA - 1u) / kRowsA, (n + kCols - 1u) / kCols, tm, tn);
  const uint32_t m0 = tm * kRowsA, n0 = tn * kCols;
  const tiler_product::RowLoader<Bf16, kLoadsA, kUneven ? kRowsA : ~0u> la(
      reinterpret_cast<const uint8_t*>(x + (uint64_t)m0 * k), k, m - m0 < kRowsA ? m - m0 : kRowsA, k, wave * kLoadsA * 8u,
                                                   wave * kLoadsA * 8u, lane, smem + S * (kRowsA + kRowsB) * kSlice);
  // B's LDS rows 64 c .. 64 c + 31 are columns 32 c .. of the gate's weight, the next 32 of the up projection's
  const uint32_t b0 = wave * kLoadsB * 8u;
  const tiler_product::RowLoader<Bf16, kLoadsB> lb(
      reinterpret_cast<const uint8_t*>(((b0 & 32u) ? wu : wg) + (uint64_t)n0 * k), k, n - n0 < kCols ? n - n0 : kCols,
      k, (b0 >> 6) * 32u + (b0 & 31u), b0, lane);
  f32x4 acc[MB][4];
  tiler_product::staged_product<Bf16, false, false, WM, WN, MB, 4, kLoadsA + kLoadsB, S>(
      smem, (k + 63u) / 64u, [&](uint32_t t, uint8_t* at) { la.issue(t, at); },
      [&](uint32_t t, uint8_t* at) { lb.issue(t, at); }, acc);
  const uint32_t row0 = (wave / WN) * MB * 16u, col0 = (wave % WN) * 32u;
  // h for the next product, from the caches; G and U, as the weights' gradients, past
  // them: too large to be kept until they are read (4096 x 14336 x 4096: 746 -> 735
  // us, the weights' gradients 735 -> 710)
  auto store = [&](auto stream, uint16_t* out, auto value) {
    __syncthreads();
    tiler_product::store_tile_bf16<kRowsA, kCols, kThreads, MB, 2, decltype(stream)::value != 0>(smem, row0, col0, out, m, n,
                                                                                            m0, n0, value);
  };
  store(tiler::Step<0>{}, h, [&](int i, int j) { return silu_times(acc[i][j], acc[i][j + 2]); });
  if (gate) {
    store(tiler::Step<1>{}, gate, [&](int i, int j) { return acc[i][j]; });
    store(tiler::Step<1>{}, up, [&](int i, int j) { return acc[i][j + 2]; });
  }
}

// dx [m, k] = dG Wg + dU Wu: depth n twice (dG with Wg, then dU with Wu), the
// weights in column layout, their rows ldk long (wu null: Wu is behind Wg).  With
// splits > 1 each split's sums go to partials[split], binary32 [m, k].
template <int WM, int WN, int MB, int S>
__device__ __forceinline__ void gated_dx_staged(const uint16_t* __restrict__ dg, const uint16_t* __restrict__ wg,
                                                const uint16_t* __restrict__ wu, uint32_t ldk, uint32_t m, uint32_t n,
                                                uint32_t k, uint16_t* __restrict__ dx, uint32_t splits,
                                                float* __restrict__ partials) {
  constexpr uint32_t kRowsA = WM * MB * 16u, kCols = WN * 64u, kThreads = 64u * WM * WN;
  constexpr int kLoadsA = kRowsA / 8 / (WM * WN), kLoadsB = kCols / 8 / (WM * WN);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * (kRowsA + kCols) * kSlice];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t tm, tn, t0, t1;
  tiler_product::tile_of(blockIdx.x, (m + kRowsA - 1u) / kRowsA, (k + kCols - 1u) / kCols, tm, tn);
  const uint32_t m0 = tm * kRowsA, c0 = tn * kCols, ld = row_of_mid(n), per = ld / 64u;
  split_range(2u * per, splits, blockIdx.y, t0, t1);
  // dG's rows hold zeros from n to ld, the weights' depth rows load as zeros there
  const tiler_product::RowLoader<Bf16, kLoadsA> la(reinterpret_cast<const uint8_t*>(dg + (uint64_t)m0 * ld), ld,
                                                   m - m0 < kRowsA ? m - m0 : kRowsA, ld, wave * kLoadsA * 8u,
                                                   wave * kLoadsA * 8u, lane);
  const tiler_product::ColumnLoader<kCols, kLoadsB> lb(reinterpret_cast<const uint8_t*>(wg + c0), ldk, c0, n, wave, lane);
  const uint8_t* const a2 = reinterpret_cast<const uint8_t*>(dg + ((uint64_t)m + m0) * ld);
  const uint8_t* const b2 = reinterpret_cast<const uint8_t*>((wu ? wu : wg + (uint64_t)n * ldk) + c0);
  f32x4 acc[MB][4];
  tiler_product::staged_product<Bf16, false, true, WM, WN, MB, 4, kLoadsA + kLoadsB, S>(
      smem, t1 - t0,
      [&](uint32_t t, uint8_t* at) {
        const bool first = t + t0 < per;
        la.issue(first ? la.base : a2, first ? t + t0 : t + t0 - per, at);
      },
      [&](uint32_t t, uint8_t* at) {
        const bool first = t + t0 < per;
        lb.issue(first ? lb.base : b2, first ? t + t0 : t + t0 - per, at);
      },
      acc);
  const uint32_t row0 = (wave / WN) * MB * 16u, col0 = (wave % WN) * 64u;
  if (splits > 1) {
    store_partial(acc, partials + (uint64_t)blockIdx.y * m * k, m, k, m0 + row0, c0 + col0);
    return;
  }
  __syncthreads();
  tiler_product::store_tile_bf16<kRowsA, kCols, kThreads, MB, 4, false>(smem, row0, col0, dx, m, k, m0, c0,
                                                                 [&](int i, int j) { return acc[i][j]; });
}

// dWg [n, k] = dG^T x and dWu = dU^T x: depth m, both operands in column
// layout, x's rows ldk long.  With splits > 1 each split's sums go to
// partials[split], binary32 [2, n, k].
template <int WM, int WN, int MB, int S>
__device__ __forceinline__ void gated_dw_staged(const uint16_t* __restrict__ dg, const uint16_t* __restrict__ x,
                                                uint32_t ldk, uint32_t m, uint32_t n, uint32_t k,
                                                uint16_t* __restrict__ dwg, uint16_t* __restrict__ dwu, uint32_t splits,
                                                float* __restrict__ partials) {
  constexpr uint32_t kRowsA = WM * MB * 16u, kCols = WN * 64u, kThreads = 64u * WM * WN;
  constexpr int kLoadsA = kRowsA / 8 / (WM * WN), kLoadsB = kCols / 8 / (WM * WN);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * (kRowsA + kCols) * kSlice];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = (n + kRowsA - 1u) / kRowsA;
  uint32_t tm, tn;
  tiler_product::tile_of(blockIdx.x, 2u * tiles, (k + kCols - 1u) / kCols, tm, tn);
  const bool second = tm >= tiles;
  const uint32_t j0 = (second ? tm - tiles : tm) * kRowsA, c0 = tn * kCols, ld = row_of_mid(n);
  const tiler_product::ColumnLoader<kRowsA, kLoadsA> la(reinterpret_cast<const uint8_t*>(dg + (second ? (uint64_t)m * ld : 0u) + j0), ld, j0,
                                                        m, wave, lane);
  const tiler_product::ColumnLoader<kCols, kLoadsB> lb(reinterpret_cast<const uint8_t*>(x + c0), ldk, c0, m, wave, lane);
  f32x4 acc[MB][4];
  uint32_t t0, t1;
  split_range((m + 63u) / 64u, splits, blockIdx.y, t0, t1);
  tiler_product::staged_product<Bf16, true, true, WM, WN, MB, 4, kLoadsA + kLoadsB, S>(
      smem, t1 - t0, [&](uint32_t t, uint8_t* at) { la.issue(t0 + t, at); },
      [&](uint32_t t, uint8_t* at) { lb.issue(t0 + t, at); }, acc);
  const uint32_t row0 = (wave / WN) * MB * 16u, col0 = (wave % WN) * 64u;
  if (splits > 1) {
    store_partial(acc, partials + ((uint64_t)blockIdx.y * 2u + (second ? 1u : 0u)) * n * k, n, k, j0 + row0, c0 + col0);
    return;
  }
  __syncthreads();
  tiler_product::store_tile_bf16<kRowsA, kCols, kThreads, MB, 4, true>(smem, row0, col0, second ? dwu : dwg, n, k, j0, c0,
                                                                 [&](int i, int j) { return acc[i][j]; });
}

}  // namespace

// Four waves: two workgroups to a CU; eight: one.  Two waves a SIMD in either.
// What LDS holds decides what is in flight, and that a slice's time where the
// weights come from memory: eight waves with three slices of a smaller tile (_n:
// 64 columns of each projection, _w: 128) against two of a larger, us, 256 x
// 14336 x 4096: 66 (256_n; with two slices 89) / 104 (256); 301 of them: 80
// (160_w) / 90 (192).  The deep forms (_d), four waves and one workgroup to a
// CU, are for grids that give a CU one workgroup in any case.  (Their bound of 512
// threads, of which 256 run, keeps the compiler to 256 registers: given 512, it
// spreads them over the accumulation registers and copies them back and forth.)
#define TILER_GATED_TILES(NAME, WM, WN, MB, S)                                                                          \
  extern "C" __global__ void __launch_bounds__(S > 2 ? 512 : 64 * WM * WN, 2)                                       \
      tiler_gated_bf16_t##NAME(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,                     \
                               const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k,                 \
                               uint16_t* __restrict__ h, uint16_t* __restrict__ gate, uint16_t* __restrict__ up) {  \
    gated_staged<WM, WN, MB, S>(x, wg, wu, m, n, k, h, gate, up);                                                    \
  }
#define TILER_GATED_DX_STAGED(NAME, WN, MB, S)                                                                        \
  extern "C" __global__ void __launch_bounds__(S > 2 ? 512 : 128 * WN, 2)                                                         \
      tiler_gated_bf16_dx_t##NAME(const uint16_t* __restrict__ dg, const uint16_t* __restrict__ wg,                 \
                                  const uint16_t* __restrict__ wu, uint32_t ldk, uint32_t m, uint32_t n,            \
                                  uint32_t k, uint16_t* __restrict__ dx, uint32_t splits,                           \
                                  float* __restrict__ partials) {                                                   \
    gated_dx_staged<2, WN, MB, S>(dg, wg, wu, ldk, m, n, k, dx, splits, partials);                                     \
  }
#define TILER_GATED_DW_STAGED(NAME, WN, MB, S)                                                                        \
  extern "C" __global__ void __launch_bounds__(S > 2 ? 512 : 128 * WN, 2)                                                         \
      tiler_gated_bf16_dw_t##NAME(const uint16_t* __restrict__ dg, const uint16_t* __restrict__ x, uint32_t ldk,    \
                                  uint32_t m, uint32_t n, uint32_t k, uint16_t* __restrict__ dwg,                   \
                                  uint16_t* __restrict__ dwu, uint32_t splits, float* __restrict__ partials) {      \
    gated_dw_staged<2, WN, MB, S>(dg, x, ldk, m, n, k, dwg, dwu, splits, partials);                                    \
  }
TILER_GATED_TILES(96, 2, 2, 3, 2)
TILER_GATED_TILES(128, 2, 2, 4, 2)
TILER_GATED_TILES(192, 2, 4, 6, 2)
TILER_GATED_TILES(256, 2, 4, 8, 2)
TILER_GATED_TILES(192_n, 4, 2, 3, 3)
TILER_GATED_TILES(256_n, 4, 2, 4, 3)
TILER_GATED_TILES(160_w, 2, 4, 5, 3)
TILER_GATED_TILES(64_d, 2, 2, 2, 6)
TILER_GATED_TILES(96_d, 2, 2, 3, 5)
TILER_GATED_TILES(128_d, 2, 2, 4, 4)
TILER_GATED_DX_STAGED(64_d, 2, 2, 6)
TILER_GATED_DX_STAGED(128, 2, 4, 2)
TILER_GATED_DX_STAGED(256, 4, 8, 2)
TILER_GATED_DW_STAGED(64_d, 2, 2, 6)
TILER_GATED_DW_STAGED(128, 2, 4, 2)
TILER_GATED_DW_STAGED(256, 4, 8, 2)

// ---------------------------------------------------------------------------
// Few tokens: the weights' bytes.  A workgroup takes 16 MB tokens and 16 P
// columns of both projections, its 8 waves the depth in turn.
namespace {

// The results of MB x P blocks from their gate and up sums (a row of blocks: P
// gate blocks, then P up blocks).
template <int MB, int P, typename T>
__device__ __forceinline__ void gated_finish(T total, uint32_t m, uint32_t n, uint32_t m0, uint32_t n0,
                                             uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                                             uint16_t* __restrict__ up) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  for (uint32_t q = wave; q < (uint32_t)(MB * P); q += 8u) {
    const uint32_t i = q / P, j = q % P;
    const f32x4 g = total(i * 2u * P + j), u = total(i * 2u * P + P + j);
    const uint32_t col = n0 + j * 16u + (lane & 15u);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t row = m0 + i * 16u + (lane >> 4) * 4u + r;
      if (row >= m || col >= n) continue;
      const uint64_t at = (uint64_t)row * n + col;
      h[at] = (uint16_t)tiler::bf16_narrow(silu_times(g[r], u[r]));
      if (gate) {
        gate[at] = (uint16_t)tiler::bf16_narrow(g[r]);
        up[at] = (uint16_t)tiler::bf16_narrow(u[r]);
      }
    }
  }
}

template <int MB, int P>
__device__ __forceinline__ void gated_few(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,
                                          const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k,
                                          uint16_t* __restrict__ h, uint16_t* __restrict__ gate,
                                          uint16_t* __restrict__ up) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[tiler_product::few_rows_lds<MB, 2 * P, 8>()];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t tm, tn;
  tiler_product::panel_of(blockIdx.x, (m + MB * 16u - 1u) / (MB * 16u), (n + P * 16u - 1u) / (P * 16u), tm, tn);
  if (tn * P * 16u >= n) return;
  const uint32_t m0 = tm * MB * 16u, n0 = tn * P * 16u, cols = n - n0 < P * 16u ? n - n0 : P * 16u;
  const tiler_product::RowLoader<Bf16, 2 * MB> la(reinterpret_cast<const uint8_t*>(x + (uint64_t)m0 * k), k,
                                                  m - m0 < MB * 16u ? m - m0 : MB * 16u, k, 0, 0, lane);
  const tiler_product::RowLoader<Bf16, 2 * P> lg(reinterpret_cast<const uint8_t*>(wg + (uint64_t)n0 * k), k, cols, k, 0, 0,
                                                 lane);
  const uint8_t* const u0 = reinterpret_cast<const uint8_t*>(wu + (uint64_t)n0 * k);
  tiler_product::few_rows_product<Bf16, MB, 2 * P, 8>(
      smem, (k + 63u) / 64u,
      [&](uint32_t t, uint8_t* slot) {
        lg.issue(t, slot + MB * 16u * kSlice);
        lg.issue(u0, t, slot + (MB + P) * 16u * kSlice);
        la.issue(t, slot);
      },
      [&](auto total) { gated_finish<MB, P>(total, m, n, m0, n0, h, gate, up); });
}

}  // namespace

#define TILER_GATED_FEW(MB, P)                                                                                     \
  extern "C" __global__ void __launch_bounds__(512)                                                                \
      tiler_gated_bf16_few##MB##x##P(const uint16_t* __restrict__ x, const uint16_t* __restrict__ wg,              \
                                     const uint16_t* __restrict__ wu, uint32_t m, uint32_t n, uint32_t k,          \
                                     uint16_t* __restrict__ h, uint16_t* __restrict__ gate,                        \
                                     uint16_t* __restrict__ up) {                                                  \
    gated_few<MB, P>(x, wg, wu, m, n, k, h, gate, up);                                                             \
  }
TILER_GATED_FEW(1, 1)
TILER_GATED_FEW(2, 1)
TILER_GATED_FEW(4, 1)
TILER_GATED_FEW(4, 2)
