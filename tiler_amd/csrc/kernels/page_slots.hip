// Page tables and cache slots of a batch's new tokens from the sequences'
// lengths: running sums over the sequences (of new tokens, and of pages to take
// from the free list), then one thread a token.
//
// Every workgroup makes the sums itself, 1024 sequences at a time, and places the
// 1024 tokens that are its own: one launch, nothing to wait for but the lengths
// (a few KB from L2).  A token's sequence is found among the block's sums in LDS.
// The token that opens a page enters the page into the table; pages before that
// are read from it, new ones computed from the list, so no workgroup reads what
// another writes.  Latency bounds it: 64 sequences of a token each 4.6 us traced, 512
// of up to 130 tokens 6.2, and a launch from the host takes 4.4.
#pragma once

#include "common.h"
#include "page_slots.h"

namespace tiler_slots {

constexpr uint32_t kThreads = 1024;

// Inclusive sums over the workgroup's threads of two values at once.
__device__ __forceinline__ void block_sums(int64_t& a, int64_t& b, int64_t (&waves)[2][16]) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (uint32_t step = 1; step < 64u; step <<= 1) {
    const int64_t x = __shfl_up((long long)a, step), y = __shfl_up((long long)b, step);
    if (lane >= step) a += x, b += y;
  }
  if (lane == 63u) waves[0][wave] = a, waves[1][wave] = b;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) a += waves[0][w], b += waves[1][w];
}

// n / d for n from 0 on: in 32 bits where n fits, as it nearly always does.
__device__ __forceinline__ int64_t divided(int64_t n, uint32_t d) {
  return (uint64_t)n >> 32 ? n / d : (int64_t)((uint32_t)n / d);
}
__device__ __forceinline__ int32_t saturated(int64_t v) { return v > 0x7fffffff ? 0x7fffffff : (int32_t)v; }

}  // namespace tiler_slots

extern "C" __global__ void __launch_bounds__(1024)
    tiler_page_slots(TilerPageSlots a, const int32_t* kept_of, const int32_t* fresh_of, const int32_t* free_pages,
                     int32_t* table, int32_t* starts, int32_t* lengths, int32_t* positions, int32_t* slots, int32_t* taken) {
  using namespace tiler_slots;
  __shared__ int64_t waves[2][16];
  __shared__ int64_t ends[kThreads], bases[kThreads];  // of the block's sequences
  __shared__ int32_t kept_at[kThreads], fresh_at[kThreads];
  const uint64_t t = (uint64_t)blockIdx.x * kThreads + threadIdx.x;  // this thread's token
  const bool first = blockIdx.x == 0;
  const uint64_t after = ((uint64_t)blockIdx.x + 1u) * kThreads;
  bool placed = t >= a.tokens;
  int64_t tokens = 0, pages = 0;  // of the blocks before
  for (uint64_t s0 = 0; s0 < a.sequences; s0 += kThreads) {
    const uint64_t s = s0 + threadIdx.x;
    const bool is = s < a.sequences;
    const int32_t kept = is ? max(kept_of[s], 0) : 0, fresh = is ? max(fresh_of[s], 0) : 0;
    const int64_t length = (int64_t)kept + fresh;
    const int64_t have = divided((int64_t)kept + a.page - 1, a.page), need = divided(length + a.page - 1, a.page);
    const int64_t most = need < (int64_t)a.width ? need : (int64_t)a.width, fresh_pages = most > have ? most - have : 0;
    int64_t end = fresh, page_end = fresh_pages;
    block_sums(end, page_end, waves);
    end += tokens;
    page_end += pages;
    ends[threadIdx.x] = end;
    bases[threadIdx.x] = page_end - fresh_pages;
    kept_at[threadIdx.x] = kept;
    fresh_at[threadIdx.x] = fresh;
    if (first && is) {
      starts[s + 1] = saturated(end);
      lengths[s] = saturated(length);
    }
    __syncthreads();
    tokens = ends[kThreads - 1];
    if (!placed && (int64_t)t < tokens) {
      uint32_t low = 0, high = kThreads - 1;  // the first sequence that ends past the token
      while (low < high) {
        const uint32_t mid = (low + high) / 2u;
        if (ends[mid] > (int64_t)t) high = mid;
        else low = mid + 1u;
      }
      const int64_t position = (int64_t)kept_at[low] + ((int64_t)t - (ends[low] - fresh_at[low]));
      const int64_t j = divided(position, a.page), in = position - j * a.page;
      const int64_t opened = divided((int64_t)kept_at[low] + a.page - 1, a.page);
      int32_t entry = -1;
      if (j < (int64_t)a.width) {
        int32_t* const at = table + (s0 + low) * a.width + j;
        if (j >= opened) {
          const int64_t take = bases[low] + j - opened;
          entry = take < (int64_t)a.free_count ? free_pages[take] : -1;
          if (in == 0) *at = entry;
        } else {
          entry = *at;
        }
      }
      const int64_t slot = entry < 0 ? -1 : (int64_t)entry * a.page + in;
      positions[t] = saturated(position);
      slots[t] = slot > 0x7fffffff ? -1 : (int32_t)slot;
      placed = true;
    }
    // of all threads: the last one's pages
    if (threadIdx.x == kThreads - 1) waves[1][15] = page_end;
    __syncthreads();
    pages = waves[1][15];
    __syncthreads();
    if (!first && tokens >= (int64_t)after) break;  // every token of this workgroup is placed
  }
  if (first && threadIdx.x == 0) {
    starts[0] = 0;
    taken[0] = saturated(pages);
  }
  if (!placed) positions[t] = 0, slots[t] = -1;  // behind the last sequence
}
