// Layer normalization over the last axis and its gradients for gfx950, f32 and
// bf16 storage, binary32 arithmetic (binary64 sums where a row is streamed):
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r w + b
//   xh = (x - mu) r, g = dy w:
//   dx = r (g - mean(g) - xh mean(g xh)), dw = sum over rows of dy xh, db = of dy
#include "common.h"

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

// Column sums over a strip of rows: blockIdx.x takes 256 columns, blockIdx.y
// rows [y * strip, ...); partial y holds dw's sums, then db's.
template <typename T>
__device__ __forceinline__ void layer_norm_columns(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                   uint64_t rows, uint64_t extent, uint64_t strip,
                                                   float* __restrict__ partials) {
  const uint64_t col = blockIdx.x * 256ull + threadIdx.x;
  if (col >= extent) return;
  const uint64_t r0 = blockIdx.y * strip, r1 = r0 + strip < rows ? r0 + strip : rows;
  float sw = 0.0f, sb = 0.0f;
  for (uint64_t r = r0; r < r1; ++r) {
    const float d = norm_load(dy, r * extent + col);
    sw += d * ((norm_load(x, r * extent + col) - mean[r]) * rstd[r]);
    sb += d;
  }
  float* out = partials + (uint64_t)blockIdx.y * 2u * extent;
  out[col] = sw;
  out[extent + col] = sb;
}

// dw and db from `count` partials, in ascending order of the strips.
template <typename T>
__device__ __forceinline__ void layer_norm_columns_final(const float* __restrict__ partials, uint32_t count,
                                                         uint64_t extent, T* __restrict__ dw, T* __restrict__ db) {
  const uint64_t i = blockIdx.x * 256ull + threadIdx.x;
  if (i >= 2u * extent) return;
  float s = 0.0f;
  for (uint32_t p = 0; p < count; ++p) s += partials[(uint64_t)p * 2u * extent + i];
  T* out = i < extent ? dw : db;
  if (out) norm_store(out, i < extent ? i : i - extent, s);
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
  extern "C" __global__ void __launch_bounds__(256)                                                       \
      tiler_layer_norm_columns_final_##TY(const float* __restrict__ partials, uint32_t count,             \
                                          uint64_t extent, T* __restrict__ dw, T* __restrict__ db) {      \
    layer_norm_columns_final<T>(partials, count, extent, dw, db);                                         \
  }
TILER_LAYER_NORM(bf16, uint16_t)
TILER_LAYER_NORM(f32, float)
