// The 8-bit linear layer for gfx950: rows quantized to int8 with one binary32
// scale each, and the product of two such operands,
//
//   C[i, j] = (sum over k of a_ik b_jk) sa_i sb_j     (a [m, k], b [n, k])
//
// on v_mfma_i32_16x16x64_i8.  The integer sum is exact (k <= 131071 keeps
// |sum| <= 2^31 - 2^14 for every pair of codes, -128 included); it is rounded
// to binary32, multiplied by sa_i, then by sb_j, and narrowed to bf16 where C is bf16.
//
// us: rows of 4096 x 4096 bf16 quantized 11 (50 MB, 4.6 TB/s: read once), the
// product 4096 x 4096 x 4096 59 (2.3 P operations/s, the matrix pipe; the forms of
// few rows and small grids are bound by what LDS keeps in flight): 16 x 4096 x
// 4096 5.3, 301 rows 15.6; 257 x 5001 x 1111 (rows off 16 bytes) 15.
#include "product.h"
#include "row_pieces.h"

namespace {

using tiler_product::I8;
using tiler_product::Operand;
using tiler_product::i32x4;
using tiler_product::kSlice;

// s = max(max |x| / 127, 2^-126), the quotient correctly rounded; q = x / s to
// the nearest integer, ties to even, exactly: the candidate r = rint(x (1 / s))
// is at most one off, next to a tie; d = x - r s is exact in one FMA (a
// multiple of s's last place below 2 s, or x itself when r = 0), so comparing
// it with the exact s / 2 decides.  |x| <= 127 s (1 + 2^-24), so |q| <= 127.
__device__ __forceinline__ float row_scale(float largest) {
  const float s = largest / 127.0f;
  return s < 0x1p-126f ? 0x1p-126f : s;
}
__device__ __forceinline__ int32_t code_of(float x, float s, float inverse) {
  float r = __builtin_rintf(x * inverse);
  const float d = __builtin_fmaf(-r, s, x), half = 0.5f * s;
  const bool odd = ((int32_t)r) & 1;
  if (d > half || (odd && d == half)) r += 1.0f;
  else if (-d > half || (odd && -d == half)) r -= 1.0f;
  return (int32_t)r;
}

// Four codes, a byte each.  The candidates come as the low bits of
// x (1 / s) + 1.5 2^23 (one FMA, rounded to an integer by the sum); where some
// |x - r s| reaches s / 2, a tie or a candidate that is off, the exact rule.
constexpr float kRound = 12582912.0f;
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float s, float inverse) {
  uint32_t bits[4];
  bool check = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float m = __builtin_fmaf(x[e], inverse, kRound);
    bits[e] = __float_as_uint(m);
    check |= __builtin_fabsf(__builtin_fmaf(-(m - kRound), s, x[e])) >= 0.5f * s;
  }
  if (check) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bits[e] = (uint32_t)code_of(x[e], s, inverse);
  }
  const uint32_t lo = __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits[3], bits[2], 0x04000c0cu);
  return lo | hi;
}

// |x| and whether it is not finite, folded over a row: the magnitude's bits
// order as the magnitudes do, infinity and NaN last.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest magnitude of a group of WAVES waves, in every lane.
template <int WAVES>
__device__ __forceinline__ uint32_t group_top(uint32_t top, uint32_t* slots) {
  top = tiler_rows::wave_fold(top, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
  if constexpr (WAVES > 1) {
    __syncthreads();  // a row before is done with the slots
    if ((threadIdx.x & 63u) == 0) slots[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = slots[w] > top ? slots[w] : top;
  }
  return top;
}

// A group of WAVES waves per row, CH pieces a thread held in registers between
// the maximum and the codes: x read once.  8 codes (bf16) or 4 (f32) leave in
// one store.
template <typename T, int WAVES, int CH>
__device__ __forceinline__ void quantize_rows(const T* __restrict__ x, uint64_t rows, uint32_t extent,
                                              int8_t* __restrict__ q, float* __restrict__ scales) {
  using namespace tiler_rows;
  constexpr int V = kVec<T>;
  __shared__ uint32_t slots[WAVES];
  const uint32_t t = threadIdx.x % (64u * WAVES);
  const uint64_t row = (uint64_t)blockIdx.x * (WAVES == 1 ? 4 : 1) + threadIdx.x / (64u * WAVES);
  if (row >= rows) return;  // whole groups
  x += row * extent;
  q += row * extent;
  u32x4 v[CH];
  load_row<T, WAVES, CH, true>(x, t, extent, v);
  settle_row<T, WAVES, CH>(t, extent, v);
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t b = magnitude(element<T>(v[c], i));
      top = b > top ? b : top;
    }
  top = group_top<WAVES>(top, slots);
#pragma unroll
  for (int c = 0; c < CH; ++c) asm volatile("" : "+v"(v[c]));  // widened again below, not kept widened
  const bool finite = top < 0x7f800000u;
  const float s = finite ? row_scale(__uint_as_float(top)) : __uint_as_float(TILER_CANONICAL_F32_NAN);
  const float inverse = 1.0f / s;
  if (t == 0) scales[row] = s;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t at = (c * 64u * WAVES + t) * V, valid = valid_from<T>(at, extent);
    if (valid == 0) continue;
    uint32_t words[V / 4];
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      float four[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) four[e] = element<T>(v[c], 4 * h + e);
      const uint32_t word = codes_of(four, s, inverse);
      words[h] = finite ? word : 0u;
    }
    if (valid == (uint32_t)V) {
      if constexpr (V == 8) *reinterpret_cast<u32x2_any*>(q + at) = u32x2{words[0], words[1]};
      else *reinterpret_cast<u32_any*>(q + at) = words[0];
    } else {
#pragma unroll
      for (int e = 0; e < V - 1; ++e)
        if ((uint32_t)e < valid) q[at + e] = (int8_t)(words[e >> 2] >> (8 * (e & 3)));
    }
    __builtin_amdgcn_sched_barrier(0);  // one piece's temporaries at a time
  }
}

// Any number of rows of any extent: one workgroup per row at a time, the row
// read twice, the second time from the caches.
template <typename T>
__device__ __forceinline__ void quantize_stream(const T* __restrict__ x, uint64_t rows, uint64_t extent,
                                                int8_t* __restrict__ q, float* __restrict__ scales) {
  __shared__ uint32_t slots[4];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * extent;
    int8_t* qr = q + row * extent;
    auto value = [&](uint64_t i) {
      if constexpr (sizeof(T) == 2) return tiler::bf16_widen(xr[i]);
      else return xr[i];
    };
    uint32_t top = 0;
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) {
      const uint32_t b = magnitude(value(i));
      top = b > top ? b : top;
    }
    top = group_top<4>(top, slots);
    const bool finite = top < 0x7f800000u;
    const float s = finite ? row_scale(__uint_as_float(top)) : __uint_as_float(TILER_CANONICAL_F32_NAN);
    const float inverse = 1.0f / s;
    if (threadIdx.x == 0) scales[row] = s;
    for (uint64_t i = threadIdx.x; i < extent; i += 256u)
      qr[i] = finite ? (int8_t)code_of(value(i), s, inverse) : (int8_t)0;
  }
}

}  // namespace

#define TILER_QUANTIZE_ROWS(TY, T, WAVES, CH)                                                              \
  extern "C" __global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, 4)                            \
      tiler_quantize_rows_i8_##TY##_w##WAVES##c##CH(const T* __restrict__ x, uint64_t rows, uint64_t extent, \
                                                    int8_t* __restrict__ q, float* __restrict__ scales) {  \
    quantize_rows<T, WAVES, CH>(x, rows, (uint32_t)extent, q, scales);                                     \
  }
#define TILER_QUANTIZE_FORMS(TY, T)                                                                        \
  extern "C" __global__ void __launch_bounds__(256)                                                        \
      tiler_quantize_rows_i8_##TY##_s(const T* __restrict__ x, uint64_t rows, uint64_t extent,             \
                                      int8_t* __restrict__ q, float* __restrict__ scales) {                \
    quantize_stream<T>(x, rows, extent, q, scales);                                                        \
  }                                                                                                        \
  TILER_QUANTIZE_ROWS(TY, T, 1, 1)                                                                         \
  TILER_QUANTIZE_ROWS(TY, T, 1, 2)                                                                         \
  TILER_QUANTIZE_ROWS(TY, T, 4, 1)                                                                         \
  TILER_QUANTIZE_ROWS(TY, T, 4, 2)                                                                         \
  TILER_QUANTIZE_ROWS(TY, T, 4, 4)                                                                         \
  TILER_QUANTIZE_ROWS(TY, T, 16, 1)                                                                        \
  TILER_QUANTIZE_ROWS(TY, T, 16, 2)                                                                        \
  TILER_QUANTIZE_ROWS(TY, T, 16, 4)
TILER_QUANTIZE_FORMS(bf16, uint16_t)
TILER_QUANTIZE_FORMS(f32, float)
TILER_QUANTIZE_ROWS(f32, float, 1, 4)

namespace {

__device__ __forceinline__ float scaled(int32_t sum, float sa, float sb) { return tiler::canon((float)sum * sa * sb); }

// Guarded form: 128 x 128 (or 64 x 128) tiles, any sizes and alignments.
template <int MB, bool kBf16>
__device__ __forceinline__ void contract_i8_guarded(const int8_t* __restrict__ a, const int8_t* __restrict__ b,
                                                    const float* __restrict__ sa, const float* __restrict__ sb,
                                                    uint32_t m, uint32_t n, uint32_t k, void* __restrict__ c) {
  constexpr uint32_t kRows = 2u * MB * 16u;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2u * (kRows + 128u) * kSlice];
  const uint32_t m0 = blockIdx.y * kRows, n0 = blockIdx.x * 128u;
  const Operand oa{reinterpret_cast<const uint8_t*>(a), m, k}, ob{reinterpret_cast<const uint8_t*>(b), n, k};
  i32x4 acc[MB][4];
  auto product = [&](const auto& la, const auto& lb) {
    tiler_product::guarded_product<I8, 2, 2, MB, 4>(
        smem, (k + 127u) / 128u, [&](uint32_t t, u32x4(&v)[MB]) { la.load(oa.base, t, v); },
        [&](uint32_t t, u32x4(&v)[4]) { lb.load(ob.base, t, v); },
        [&](uint32_t t, uint8_t* tile, u32x4(&v)[MB]) { la.store(t, tile, v); },
        [&](uint32_t t, uint8_t* tile, u32x4(&v)[4]) { lb.store(t, tile, v); }, acc);
  };
  if (k >= 16u) product(tiler_product::GuardedLoader<I8, kRows, 256>(oa, m0), tiler_product::GuardedLoader<I8, 128, 256>(ob, n0));
  else product(tiler_product::TinyLoader<I8, kRows, 256>(oa, m0), tiler_product::TinyLoader<I8, 128, 256>(ob, n0));
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t col = n0 + (wave & 1u) * 64u + j * 16u + (lane & 15u);
    if (col >= n) continue;
    const float cs = sb[col];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t row = m0 + (wave >> 1) * MB * 16u + i * 16u + (lane >> 4) * 4u + r;
        if (row >= m) continue;
        const float v = scaled(acc[i][j][r], sa[row], cs);
        const uint64_t at = (uint64_t)row * n + col;
        if constexpr (kBf16) static_cast<uint16_t*>(c)[at] = (uint16_t)tiler::bf16_narrow(v);
        else static_cast<float*>(c)[at] = v;
      }
  }
}

}  // namespace

#define TILER_CONTRACT_I8_GUARDED(TY, BF16, TILE, MB)                                                              \
  extern "C" __global__ void __launch_bounds__(256, 2)                                                             \
      tiler_contract_i8_##TY##_g##TILE(const int8_t* __restrict__ a, const int8_t* __restrict__ b,                 \
                                       const float* __restrict__ sa, const float* __restrict__ sb, uint32_t m,     \
                                       uint32_t n, uint32_t k, void* __restrict__ c) {                             \
    contract_i8_guarded<MB, BF16>(a, b, sa, sb, m, n, k, c);                                                       \
  }
TILER_CONTRACT_I8_GUARDED(bf16, true, 128, 4)
TILER_CONTRACT_I8_GUARDED(f32, false, 128, 4)
TILER_CONTRACT_I8_GUARDED(bf16, true, 64, 2)
TILER_CONTRACT_I8_GUARDED(f32, false, 64, 2)

// ---------------------------------------------------------------------------
// Staged form: k a multiple of 16 and 16-byte aligned operands.
namespace {

template <int WM, int WN, int MB, int S, bool kBf16>
__device__ __forceinline__ void contract_i8_staged(const int8_t* __restrict__ a, const int8_t* __restrict__ b,
                                                   const float* __restrict__ sa, const float* __restrict__ sb,
                                                   uint32_t m, uint32_t n, uint32_t k, void* __restrict__ c) {
  constexpr uint32_t kRowsA = WM * MB * 16u, kRowsB = WN * 64u, kThreads = 64u * WM * WN;
  constexpr int kLoadsA = kRowsA / 8 / (WM * WN), kLoadsB = kRowsB / 8 / (WM * WN);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * (kRowsA + kRowsB) * kSlice];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t tm, tn;
  tiler_product::tile_of(blockIdx.x, (m + kRowsA - 1u) / kRowsA, (n + kRowsB - 1u) / kRowsB, tm, tn);
  const uint32_t m0 = tm * kRowsA, n0 = tn * kRowsB;
  const tiler_product::RowLoader<I8, kLoadsA> la(reinterpret_cast<const uint8_t*>(a + (uint64_t)m0 * k), k,
                                                 m - m0 < kRowsA ? m - m0 : kRowsA, k, wave * kLoadsA * 8u,
                                                 wave * kLoadsA * 8u, lane);
  const tiler_product::RowLoader<I8, kLoadsB> lb(reinterpret_cast<const uint8_t*>(b + (uint64_t)n0 * k), k,
                                                 n - n0 < kRowsB ? n - n0 : kRowsB, k, wave * kLoadsB * 8u,
                                                 wave * kLoadsB * 8u, lane);
  i32x4 acc[MB][4];
  tiler_product::staged_product<I8, false, false, WM, WN, MB, 4, kLoadsA + kLoadsB, S>(
      smem, (k + 127u) / 128u, [&](uint32_t t, uint8_t* at) { la.issue(t, at); },
      [&](uint32_t t, uint8_t* at) { lb.issue(t, at); }, acc);
  const uint32_t row0 = (wave / WN) * MB * 16u, col0 = (wave % WN) * 64u;
  float rows[MB][4], cols[4];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t row = m0 + row0 + i * 16u + (lane >> 4) * 4u + r;
      rows[i][r] = sa[row < m ? row : m - 1u];
    }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t col = n0 + col0 + j * 16u + (lane & 15u);
    cols[j] = sb[col < n ? col : n - 1u];
  }
  if constexpr (kBf16) {
    __syncthreads();
    tiler_product::store_tile_bf16<kRowsA, kRowsB, kThreads, MB, 4, false>(
        smem, row0, col0, static_cast<uint16_t*>(c), m, n, m0, n0,
        [&](int i, int j) {
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][j][r] * rows[i][r] * cols[j];
          return v;
        });
  } else {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t row = m0 + row0 + i * 16u + (lane >> 4) * 4u + r, col = n0 + col0 + j * 16u + (lane & 15u);
          if (row < m && col < n)
            static_cast<float*>(c)[(uint64_t)row * n + col] = scaled(acc[i][j][r], rows[i][r], cols[j]);
        }
  }
}

}  // namespace

// Four waves: two workgroups to a CU; eight: one.  Two waves a SIMD in either.
// The deep forms (_d) keep as many slices in LDS as it holds, for the grids that
// give a CU one workgroup.
#define TILER_CONTRACT_I8_STAGED(TY, BF16, NAME, WN, MB, S)                                                        \
  extern "C" __global__ void __launch_bounds__(S > 2 ? 512 : 128 * WN, 2)                                       \
      tiler_contract_i8_##TY##_t##NAME(const int8_t* __restrict__ a, const int8_t* __restrict__ b,                 \
                                       const float* __restrict__ sa, const float* __restrict__ sb, uint32_t m,     \
                                       uint32_t n, uint32_t k, void* __restrict__ c) {                             \
    contract_i8_staged<2, WN, MB, S, BF16>(a, b, sa, sb, m, n, k, c);                                              \
  }
#define TILER_CONTRACT_I8_TILES(TY, BF16)             \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 96, 2, 3, 2)     \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 128, 2, 4, 2)    \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 192, 4, 6, 2)    \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 256, 4, 8, 2)    \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 64_d, 2, 2, 6)   \
  TILER_CONTRACT_I8_STAGED(TY, BF16, 96_d, 2, 3, 5)
TILER_CONTRACT_I8_TILES(bf16, true)
TILER_CONTRACT_I8_TILES(f32, false)

// ---------------------------------------------------------------------------
// Few rows: the bytes of b.  A workgroup takes 16 MB rows and 16 NB columns, its
// 8 waves the depth in turn.
namespace {

// The results of MB x NB blocks from their sums.
template <int MB, int NB, bool kBf16, typename T>
__device__ __forceinline__ void contract_i8_finish(T total, const float* __restrict__ sa, const float* __restrict__ sb,
                                                   uint32_t m, uint32_t n, uint32_t m0, uint32_t n0,
                                                   void* __restrict__ c) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  for (uint32_t q = wave; q < (uint32_t)(MB * NB); q += 8u) {
    const i32x4 v = total(q);
    const uint32_t col = n0 + q % NB * 16u + (lane & 15u);
    if (col >= n) continue;
    const float cs = sb[col];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t row = m0 + q / NB * 16u + (lane >> 4) * 4u + r;
      if (row >= m) continue;
      const float f = scaled(v[r], sa[row], cs);
      const uint64_t at = (uint64_t)row * n + col;
      if constexpr (kBf16) static_cast<uint16_t*>(c)[at] = (uint16_t)tiler::bf16_narrow(f);
      else static_cast<float*>(c)[at] = f;
    }
  }
}

template <int MB, int NB, bool kBf16>
__device__ __forceinline__ void contract_i8_few(const int8_t* __restrict__ a, const int8_t* __restrict__ b,
                                                const float* __restrict__ sa, const float* __restrict__ sb, uint32_t m,
                                                uint32_t n, uint32_t k, void* __restrict__ c) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[tiler_product::few_rows_lds<MB, NB, 8>()];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t tm, tn;
  tiler_product::panel_of(blockIdx.x, (m + MB * 16u - 1u) / (MB * 16u), (n + NB * 16u - 1u) / (NB * 16u), tm, tn);
  if (tn * NB * 16u >= n) return;
  const uint32_t m0 = tm * MB * 16u, n0 = tn * NB * 16u;
  const tiler_product::RowLoader<I8, 2 * MB> la(reinterpret_cast<const uint8_t*>(a + (uint64_t)m0 * k), k,
                                                m - m0 < MB * 16u ? m - m0 : MB * 16u, k, 0, 0, lane);
  const tiler_product::RowLoader<I8, 2 * NB> lb(reinterpret_cast<const uint8_t*>(b + (uint64_t)n0 * k), k,
                                                n - n0 < NB * 16u ? n - n0 : NB * 16u, k, 0, 0, lane);
  tiler_product::few_rows_product<I8, MB, NB, 8>(
      smem, (k + 127u) / 128u,
      [&](uint32_t t, uint8_t* slot) {
        lb.issue(t, slot + MB * 16u * kSlice);
        la.issue(t, slot);
      },
      [&](auto total) { contract_i8_finish<MB, NB, kBf16>(total, sa, sb, m, n, m0, n0, c); });
}

}  // namespace

#define TILER_CONTRACT_I8_FEW(TY, BF16, MB, NB)                                                                    \
  extern "C" __global__ void __launch_bounds__(512)                                                                \
      tiler_contract_i8_##TY##_few##MB##x##NB(const int8_t* __restrict__ a, const int8_t* __restrict__ b,          \
                                              const float* __restrict__ sa, const float* __restrict__ sb,          \
                                              uint32_t m, uint32_t n, uint32_t k, void* __restrict__ c) {          \
    contract_i8_few<MB, NB, BF16>(a, b, sa, sb, m, n, k, c);                                                       \
  }
#define TILER_CONTRACT_I8_FEW_FORMS(TY, BF16) \
  TILER_CONTRACT_I8_FEW(TY, BF16, 1, 1)       \
  TILER_CONTRACT_I8_FEW(TY, BF16, 2, 1)       \
  TILER_CONTRACT_I8_FEW(TY, BF16, 2, 2)       \
  TILER_CONTRACT_I8_FEW(TY, BF16, 4, 2)       \
  TILER_CONTRACT_I8_FEW(TY, BF16, 4, 4)
TILER_CONTRACT_I8_FEW_FORMS(bf16, true)
TILER_CONTRACT_I8_FEW_FORMS(f32, false)
