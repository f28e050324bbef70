// Layer normalization over the last axis and its gradients for gfx950, f32 and
// bf16 storage, binary32 arithmetic (binary64 sums where a row is streamed):
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b
//   xh = (x - mu) r, g = dy w:
//   dx = r (g - mean(g) - xh mean(g xh)), dw = sum over rows of dy xh, db = of dy
//
// Memory bounds all of it, so a row is read once and held in registers between
// its sums and its results, and the gradients' workgroups keep dw's and db's sums
// over their rows in registers.  us, and a copy of the same bytes: 8192 x 4096
// bf16 with statistics 27 / 26, its gradients 46 and 4.6 for the partials' sum /
// 39; the same in f32 48 / 52 and 79 / 78; 16 x 4096, a launch, 6; gradients of
// 1237 x 1023 f32 6.9 and 4.2 / 3.  Gradients of rows longer than registers hold
// read dy and x twice, an element a load: 4096 x 12288 f32 341 / 117.
#include "row_pieces.h"

namespace {

template <typename T>
__device__ __forceinline__ float norm_load(const T* p, uint64_t i) {
  if constexpr (sizeof(T) == 2) return tiler::bf16_widen(p[i]);
  else return p[i];
}
template <typename T>
__device__ __forceinline__ void norm_store(T* p, uint64_t i, float v) {
  if constexpr (sizeof(T) == 2) p[i] = (T)tiler::bf16_narrow(v);
  else p[i] = tiler::canon(v);
}

// Columns of a partial: dw's sums, then db's, each from a 32-byte boundary.
__device__ __forceinline__ uint64_t partial_ld(uint64_t extent) { return (extent + 7u) / 8u * 8u; }

// Sum over a 256-thread workgroup, the same value in every thread.
__device__ __forceinline__ double block_sum(double v, double* waves) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  return (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// Any extent and alignment: one workgroup streams a row.
template <typename T>
__device__ __forceinline__ void layer_norm_stream(const T* __restrict__ x, const T* __restrict__ w,
                                                  const T* __restrict__ b, uint64_t rows, uint64_t extent, float eps,
                                                  T* __restrict__ y, float* __restrict__ mean,
                                                  float* __restrict__ rstd) {
  __shared__ double waves[4];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * extent;
    T* yr = y + row * extent;
    double s = 0.0;
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) s += norm_load(xr, i);
    const double mu = block_sum(s, waves) / (double)extent;
    s = 0.0;
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) {
      const double d = norm_load(xr, i) - mu;
      s += d * d;
    }
    const double r = 1.0 / __builtin_sqrt(block_sum(s, waves) / (double)extent + (double)eps);
    if (threadIdx.x == 0 && mean) {
      mean[row] = (float)mu;
      rstd[row] = (float)r;
    }
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) {
      const float xh = (float)((norm_load(xr, i) - mu) * r);
      norm_store(yr, i, (w ? xh * norm_load(w, i) : xh) + (b ? norm_load(b, i) : 0.0f));
    }
  }
}

template <typename T>
__device__ __forceinline__ void layer_norm_grad_stream(const T* __restrict__ dy, const T* __restrict__ x,
                                                       const T* __restrict__ w, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, uint64_t rows,
                                                       uint64_t extent, T* __restrict__ dx) {
  __shared__ double waves[4];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const uint64_t at = row * extent;
    const float mu = mean[row], r = rstd[row];
    double s1 = 0.0, s2 = 0.0;
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) {
      const float g = w ? norm_load(dy, at + i) * norm_load(w, i) : norm_load(dy, at + i);
      s1 += g;
      s2 += (double)g * ((norm_load(x, at + i) - mu) * r);
    }
    const float c1 = (float)(block_sum(s1, waves) / (double)extent);
    const float c2 = (float)(block_sum(s2, waves) / (double)extent);
    for (uint64_t i = threadIdx.x; i < extent; i += 256u) {
      const float g = w ? norm_load(dy, at + i) * norm_load(w, i) : norm_load(dy, at + i);
      norm_store(dx, at + i, r * (g - c1 - (norm_load(x, at + i) - mu) * r * c2));
    }
  }
}

// ---------------------------------------------------------------------------
// Rows in registers.

// Forward: a group of WAVES waves per row, CH pieces a thread.  The mean first,
// then the squares of the differences from it.  The binary32 mean is off by its
// roundings, |mu| 2^-24 and more, which a row far from zero or nearly constant
// would carry into its results, so what it is off by (`shift`) is taken off the
// differences too, in the FMA that scales them.  f32 rows: the mean of the
// differences.  bf16 rows: the remainder of the division; their sum is all but
// exact (8 bits a value, where the values are of one size) and the sum of the
// differences would cost a tenth of the kernel.  Of f32 rows 10^5 deviations
// from zero y is off by 5e-7, by 1e-2 with the mean alone; 8192 x 4096 bf16 27.2
// us, with the mean alone 27.05.
template <typename T, int WAVES, int CH>
__device__ __forceinline__ void layer_norm_rows(const T* __restrict__ x, const T* __restrict__ w,
                                                const T* __restrict__ b, uint64_t rows, uint32_t extent, float eps,
                                                T* __restrict__ y, float* __restrict__ mean,
                                                float* __restrict__ rstd) {
  using namespace tiler_rows;
  constexpr int V = kVec<T>;
  constexpr bool kCorrect = sizeof(T) == 4;
  constexpr uint32_t kGroups = WAVES == 1 ? 4 : 1, kSpan = 64u * WAVES * V;
  __shared__ float slots[2][2 * (WAVES == 1 ? 1 : WAVES)];
  const uint32_t t = threadIdx.x % (64u * WAVES);
  const uint64_t row = (uint64_t)blockIdx.x * kGroups + threadIdx.x / (64u * WAVES);
  if (row >= rows) return;  // whole groups
  x += row * extent;
  y += row * extent;
  u32x4 v[CH];
  load_row<T, WAVES, CH, true>(x, t, extent, v);
  settle_row<T, WAVES, CH>(t, extent, v);
  const float count = (float)extent, inverse = 1.0f / count;
  float s = 0.0f, none = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = element<T>(v[c], i);
    s += pairwise(e);
  }
  group_sums<WAVES>(s, none, slots[0]);
  // opaque: widened again below, not kept widened across the sums
#pragma unroll
  for (int c = 0; c < CH; ++c) asm volatile("" : "+v"(v[c]));
  const float mu = s / count;  // divided: a constant row's is exact
  float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float d[V], q = 0.0f;
    if ((c + 1u) * kSpan <= extent) {  // uniform: every thread's piece is whole
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = element<T>(v[c], i) - mu;
    } else {
      const uint32_t valid = valid_from<T>((c * 64u * WAVES + t) * V, extent);
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = (uint32_t)i < valid ? element<T>(v[c], i) - mu : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) q = __builtin_fmaf(d[i], d[i], q);
    if constexpr (kCorrect) s1 += pairwise(d);
    s2 += q;
  }
  group_sums<WAVES>(s2, s1, slots[1]);
#pragma unroll
  for (int c = 0; c < CH; ++c) asm volatile("" : "+v"(v[c]));
  const float shift = (kCorrect ? s1 : __builtin_fmaf(-mu, count, s)) * inverse;
  float var = __builtin_fmaf(-shift, shift, s2 * inverse);
  var = var < 0.0f ? 0.0f : var;
  const float r = 1.0f / __builtin_sqrtf(var + eps), off = -(shift * r);
  if (t == 0 && mean) {
    mean[row] = mu + shift;
    rstd[row] = r;
  }
  // w and b a few pieces at a time: they come from the caches
  constexpr int kBatch = CH < 4 ? CH : 4;
#pragma unroll
  for (int c0 = 0; c0 < CH; c0 += kBatch) {
    const uint32_t t0 = c0 * 64u * WAVES + t;  // as pieces 0.. of a thread further on
    u32x4 wv[kBatch], bv[kBatch];
    if (w) {
      load_row<T, WAVES, kBatch, false>(w, t0, extent, wv);
      settle_row<T, WAVES, kBatch>(t0, extent, wv);
    }
    if (b) {
      load_row<T, WAVES, kBatch, false>(b, t0, extent, bv);
      settle_row<T, WAVES, kBatch>(t0, extent, bv);
    }
#pragma unroll
    for (int c = 0; c < kBatch; ++c) {
      const uint32_t at = (c * 64u * WAVES + t0) * V;
      if (at >= extent) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        o[i] = __builtin_fmaf(element<T>(v[c0 + c], i) - mu, r, off);
        if (w && b) o[i] = __builtin_fmaf(o[i], element<T>(wv[c], i), element<T>(bv[c], i));
        else if (w) o[i] = o[i] * element<T>(wv[c], i);
        else if (b) o[i] = o[i] + element<T>(bv[c], i);
      }
      store_piece<T>(y, at, extent, o);
    }
  }
}

// Waves of a gradient workgroup: 8, two workgroups to a CU (each waits at its
// own barriers); 16 where a row takes them all.
template <int WAVES>
constexpr int kGradWaves = WAVES == 16 ? 16 : 8;

// Gradients, one read of dy and x: a workgroup holds kGradWaves / WAVES
// rows at a time and walks the rows with a stride of the whole grid; a thread
// keeps the column sums of its own pieces over all of its rows, the groups meet
// in LDS, and each workgroup leaves one partial (dw's sums, then db's), or the
// results themselves where it is the only one.  The next rows are loaded
// before the current ones are reduced.
template <typename T, int WAVES, int CH>
__device__ __forceinline__ void layer_norm_grad_rows(const T* __restrict__ dy, const T* __restrict__ x,
                                                     const T* __restrict__ w, const float* __restrict__ mean,
                                                     const float* __restrict__ rstd, uint64_t rows, uint32_t extent,
                                                     T* __restrict__ dx, float* __restrict__ partials,
                                                     T* __restrict__ dw, T* __restrict__ db) {
  using namespace tiler_rows;
  constexpr int V = kVec<T>;
  constexpr bool kAhead = CH * V <= 8;  // beyond, the next rows' pieces do not fit the registers
  constexpr uint32_t kGroups = kGradWaves<WAVES> / WAVES, kSpan = CH * 64u * WAVES * V;  // elements a group's pieces cover
  __shared__ float slots[2][2 * kGradWaves<WAVES>];
  __shared__ float columns[kGroups > 1 ? 2 * kSpan : 1];
  const uint32_t t = threadIdx.x % (64u * WAVES), group = threadIdx.x / (64u * WAVES);
  const bool sums = partials || dw || db;
  float aw[CH][V], ab[CH][V];
  u32x4 wv[CH], xv[CH], dv[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    wv[c] = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i) aw[c][i] = ab[c][i] = 0.0f;
  }
  if (w) {
    load_row<T, WAVES, CH, false>(w, t, extent, wv);
    settle_row<T, WAVES, CH>(t, extent, wv);
  }
  const uint64_t step = (uint64_t)gridDim.x * kGroups;
  uint64_t row = (uint64_t)blockIdx.x * kGroups + group;
  const uint64_t rounds = (rows - (uint64_t)blockIdx.x * kGroups + step - 1) / step;  // the first group's: the same for all
  float mu = 0.0f, r = 0.0f;
  // A group past the last row reads the last one; its terms are dropped.
  auto load = [&](uint64_t at_row, u32x4(&xo)[CH], u32x4(&dyo)[CH], float& muo, float& ro) {
    const uint64_t here = at_row < rows ? at_row : rows - 1u;
    muo = mean[here];
    ro = rstd[here];
    load_row<T, WAVES, CH, true>(x + here * extent, t, extent, xo);
    load_row<T, WAVES, CH, true>(dy + here * extent, t, extent, dyo);
  };
  // One round: the next rows' pieces are requested (past the last rows, the
  // last one again), then the current ones are reduced and stored.
  auto turn = [&](uint64_t k, u32x4(&xc)[CH], u32x4(&dc)[CH], float mu, float r, u32x4(&xn)[CH], u32x4(&dn)[CH],
                  float& mun, float& rn) {
    if constexpr (kAhead) load(row + step, xn, dn, mun, rn);
    settle_row<T, WAVES, CH>(t, extent, xc);
    settle_row<T, WAVES, CH>(t, extent, dc);
    if (row >= rows) {  // whole groups, in the last round
#pragma unroll
      for (int c = 0; c < CH; ++c) xc[c] = dc[c] = u32x4{0, 0, 0, 0};
      mu = r = 0.0f;
    }
    float s1 = 0.0f, s2 = 0.0f, xh[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float g[V], q = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // past the row's end dy is zero, and so are the terms
        const float d = element<T>(dc[c], i);
        xh[c][i] = (element<T>(xc[c], i) - mu) * r;
        g[i] = w ? d * element<T>(wv[c], i) : d;
        q = __builtin_fmaf(g[i], xh[c][i], q);
        aw[c][i] = __builtin_fmaf(d, xh[c][i], aw[c][i]);
        ab[c][i] += d;
        asm volatile("" : "+v"(aw[c][i]), "+v"(ab[c][i]));  // added here, not past the barrier with its terms kept
      }
      s1 += pairwise(g);
      s2 += q;
      __builtin_amdgcn_sched_barrier(0);  // one piece's temporaries at a time
    }
    // opaque: widened again below, not kept widened across the sums
#pragma unroll
    for (int c = 0; c < CH; ++c) asm volatile("" : "+v"(xc[c]), "+v"(dc[c]), "+v"(wv[c]));
    if (dx) {  // uniform: every wave takes the same barriers
      group_sums<WAVES>(s1, s2, slots[k & 1u]);
      // dx = r g - (xh (r c2) + r c1), xh kept where the registers hold it (8192 x
      // 4096 bf16 48.7 us, formed again 50.0).  As an FMA of x with mu in the constant
      // (49.3) the row's distance from zero would round into dx: f32 rows 10^5
      // deviations from zero 4e-4 of the largest dx instead of 5e-8; and r^2 leaves
      // binary32 where a row's deviation is below 10^-19.
      const float c1 = s1 / (float)extent, c2 = s2 / (float)extent, a = -(r * c2), z = -(r * c1);
      if (row < rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const uint32_t at = (c * 64u * WAVES + t) * V;
          if (at >= extent) continue;
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float d = element<T>(dc[c], i), g = w ? d * element<T>(wv[c], i) : d;
            o[i] = __builtin_fmaf(g, r, __builtin_fmaf(kAhead ? xh[c][i] : (element<T>(xc[c], i) - mu) * r, a, z));
          }
          store_piece<T>(dx + row * extent, at, extent, o);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    row += step;
    if constexpr (!kAhead) {
      if (k + 1 < rounds) load(row, xn, dn, mun, rn);
    }
  };
  load(row, xv, dv, mu, r);
  u32x4 xo[CH], dyo[CH];
  float muo = 0.0f, ro = 0.0f;
#pragma unroll 1
  for (uint64_t k = 0; k < rounds; k += 2) {  // two rounds, so that no piece moves between registers
    turn(k, xv, dv, mu, r, xo, dyo, muo, ro);
    if (k + 1 < rounds) turn(k + 1, xo, dyo, muo, ro, xv, dv, mu, r);
  }
  if (!sums) return;
  // The groups' columns, added in ascending order of the groups.
  if constexpr (kGroups > 1) {
    for (uint32_t q = 1; q < kGroups; ++q) {
      __syncthreads();
      if (group == q) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            columns[(c * V + i) * 64u * WAVES + t] = aw[c][i];
            columns[kSpan + (c * V + i) * 64u * WAVES + t] = ab[c][i];
          }
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            aw[c][i] += columns[(c * V + i) * 64u * WAVES + t];
            ab[c][i] += columns[kSpan + (c * V + i) * 64u * WAVES + t];
          }
      }
    }
    if (group != 0) return;
  }
  const bool alone = gridDim.x == 1;
  const uint32_t ld = partial_ld(extent);
  float* out = alone ? nullptr : partials + (uint64_t)blockIdx.x * 2u * ld;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t at = (c * 64u * WAVES + t) * V;
    if (at >= extent) continue;
    if (alone) {
      if (dw) store_piece<T>(dw, at, extent, aw[c]);
      if (db) store_piece<T>(db, at, extent, ab[c]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        *reinterpret_cast<f32x4*>(out + at + i) = f32x4{aw[c][i], aw[c][i + 1], aw[c][i + 2], aw[c][i + 3]};
        *reinterpret_cast<f32x4*>(out + ld + at + i) = f32x4{ab[c][i], ab[c][i + 1], ab[c][i + 2], ab[c][i + 3]};
      }
    }
  }
}

// Column sums over a strip of rows: blockIdx.x takes 256 columns at a time,
// blockIdx.y rows [y * strip, ...); partial y holds dw's sums, then db's.
template <typename T>
__device__ __forceinline__ void layer_norm_columns(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                   uint64_t rows, uint64_t extent, uint64_t strip,
                                                   float* __restrict__ partials) {
  const uint64_t r0 = blockIdx.y * strip, r1 = r0 + strip < rows ? r0 + strip : rows;
  const uint64_t ld = partial_ld(extent);
  float* out = partials + (uint64_t)blockIdx.y * 2u * ld;
  for (uint64_t col = blockIdx.x * 256ull + threadIdx.x; col < extent; col += gridDim.x * 256ull) {
    float sw = 0.0f, sb = 0.0f;
    for (uint64_t r = r0; r < r1; ++r) {
      const float d = norm_load(dy, r * extent + col);
      sw += d * ((norm_load(x, r * extent + col) - mean[r]) * rstd[r]);
      sb += d;
    }
    out[col] = sw;
    out[ld + col] = sb;
  }
}

// dw (blockIdx.y 0) and db (1) from `count` partials: 64 columns a workgroup at
// a time, wave q the partials q, q + 16, ... in ascending order, the waves' sums
// in ascending order.
template <typename T>
__device__ __forceinline__ void layer_norm_columns_final(const float* __restrict__ partials, uint32_t count,
                                                         uint64_t extent, T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float waves[16][64];
  T* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t ld = partial_ld(extent);
  for (uint64_t first = blockIdx.x * 64ull; first < extent; first += gridDim.x * 64ull) {  // the same for every wave
    const uint64_t col = first + lane;
    float s = 0.0f;
    if (col < extent) {
      const float* at = partials + blockIdx.y * ld + col;
#pragma unroll 8
      for (uint32_t p = wave; p < count; p += 16u) s += at[(uint64_t)p * 2u * ld];
    }
    if (first != blockIdx.x * 64ull) __syncthreads();  // the columns before are read
    waves[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < extent) {
#pragma unroll
      for (int q = 1; q < 16; ++q) s += waves[q][lane];
      norm_store(out, col, s);
    }
  }
}

}  // namespace

#define TILER_LAYER_NORM(TY, T)                                                                           \
  extern "C" __global__ void __launch_bounds__(256)                                                       \
      tiler_layer_norm_##TY##_s(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, \
                                uint64_t rows, uint64_t extent, float eps, T* __restrict__ y,             \
                                float* __restrict__ mean, float* __restrict__ rstd) {                     \
    layer_norm_stream<T>(x, w, b, rows, extent, eps, y, mean, rstd);                                      \
  }                                                                                                       \
  extern "C" __global__ void __launch_bounds__(256)                                                       \
      tiler_layer_norm_grad_##TY##_s(const T* __restrict__ dy, const T* __restrict__ x,                   \
                                     const T* __restrict__ w, const float* __restrict__ mean,             \
                                     const float* __restrict__ rstd, uint64_t rows, uint64_t extent,      \
                                     T* __restrict__ dx) {                                                \
    layer_norm_grad_stream<T>(dy, x, w, mean, rstd, rows, extent, dx);                                    \
  }                                                                                                       \
  extern "C" __global__ void __launch_bounds__(256)                                                       \
      tiler_layer_norm_columns_##TY(const T* __restrict__ dy, const T* __restrict__ x,                    \
                                    const float* __restrict__ mean, const float* __restrict__ rstd,       \
                                    uint64_t rows, uint64_t extent, uint64_t strip,                       \
                                    float* __restrict__ partials) {                                       \
    layer_norm_columns<T>(dy, x, mean, rstd, rows, extent, strip, partials);                              \
  }                                                                                                       \
  extern "C" __global__ void __launch_bounds__(1024)                                                      \
      tiler_layer_norm_columns_final_##TY(const float* __restrict__ partials, uint32_t count,             \
                                          uint64_t extent, T* __restrict__ dw, T* __restrict__ db) {      \
    layer_norm_columns_final<T>(partials, count, extent, dw, db);                                         \
  }
TILER_LAYER_NORM(bf16, uint16_t)
TILER_LAYER_NORM(f32, float)

#define TILER_LAYER_NORM_ROWS(TY, T, WAVES, CH)                                                            \
  extern "C" __global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, 4)                            \
      tiler_layer_norm_##TY##_w##WAVES##c##CH(const T* __restrict__ x, const T* __restrict__ w,            \
                                              const T* __restrict__ b, uint64_t rows, uint64_t extent,     \
                                              float eps, T* __restrict__ y, float* __restrict__ mean,      \
                                              float* __restrict__ rstd) {                                  \
    layer_norm_rows<T, WAVES, CH>(x, w, b, rows, (uint32_t)extent, eps, y, mean, rstd);                    \
  }
#define TILER_LAYER_NORM_GRAD_ROWS(TY, T, WAVES, CH)                                                        \
  extern "C" __global__ void __launch_bounds__(64 * kGradWaves<WAVES>)                                     \
      tiler_layer_norm_grad_##TY##_w##WAVES##c##CH(                                                        \
          const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w,                      \
          const float* __restrict__ mean, const float* __restrict__ rstd, uint64_t rows, uint64_t extent,  \
          T* __restrict__ dx, float* __restrict__ partials, T* __restrict__ dw, T* __restrict__ db) {      \
    layer_norm_grad_rows<T, WAVES, CH>(dy, x, w, mean, rstd, rows, (uint32_t)extent, dx, partials, dw, db); \
  }
#define TILER_LAYER_NORM_FORMS(TY, T)      \
  TILER_LAYER_NORM_ROWS(TY, T, 1, 1)       \
  TILER_LAYER_NORM_ROWS(TY, T, 1, 2)       \
  TILER_LAYER_NORM_ROWS(TY, T, 1, 4)       \
  TILER_LAYER_NORM_ROWS(TY, T, 4, 1)       \
  TILER_LAYER_NORM_ROWS(TY, T, 4, 2)       \
  TILER_LAYER_NORM_ROWS(TY, T, 4, 4)       \
  TILER_LAYER_NORM_ROWS(TY, T, 16, 1)      \
  TILER_LAYER_NORM_ROWS(TY, T, 16, 2)      \
  TILER_LAYER_NORM_ROWS(TY, T, 16, 4)      \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 1, 1) \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 2, 1) \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 4, 1) \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 8, 1) \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 16, 1) \
  TILER_LAYER_NORM_GRAD_ROWS(TY, T, 16, 2)
TILER_LAYER_NORM_FORMS(bf16, uint16_t)
TILER_LAYER_NORM_FORMS(f32, float)
