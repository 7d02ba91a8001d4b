// Pieces shared by the kernels of the 128-value block format: the scale rule, and how rows sorted by expert are cut up.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "mx_common.cuh"

namespace mxb200 {

constexpr int kBlock = 128;  // values per scale along the quantized axis
constexpr int kMaxExperts = 1024;
constexpr int64_t kMostSize = int64_t{1} << 30;  // of a dimension, and of a launch's tiles

constexpr int64_t blocks_up(int64_t n, int64_t d) {
  return (n + d - 1) / d;
}

// Biased exponent of the scale of a block: the smallest power of two with max|block| <= 448 scale, as for MX, but not below
// 2^-126, so that the scale is a normal fp32 number (the reciprocal is one up to 2^126).
__device__ __forceinline__ int block_exponent(uint32_t amax_bits) {
  return max(mx_exponent(amax_bits, false), 1);
}

// Rows sorted by expert: expert e has rows [end(e - 1), end(e)), end(e) = ends[e] held to [end(e - 1), rows], so that no value
// of ends leads out of the matrix. Writes into shared memory, for e = 0 .. experts, the first row and the number of `tile`-row
// tiles of all experts before e. Rows behind the last expert's are nobody's. ends null: one expert that has all rows.
// The whole block calls it (`tmp`: experts words); ends with __syncthreads().
__device__ __forceinline__ void scan_experts(const int32_t* ends, int experts, int rows, int tile, int* first_row,
                                             int* first_tile, int* tmp) {
  if (ends == nullptr) {
    if (threadIdx.x == 0) {
      first_row[0] = 0, first_row[1] = rows;
      first_tile[0] = 0, first_tile[1] = (rows + tile - 1) / tile;
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < experts; e += blockDim.x)
    tmp[e] = min(max(ends[e], 0), rows);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int row = 0, tiles = 0;  // carried from one group of 32 experts to the next
    if (lane == 0)
      first_row[0] = 0, first_tile[0] = 0;
    for (int base = 0; base < experts; base += 32) {
      const int e = base + lane;
      int end = e < experts ? tmp[e] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, end, d);
        end = lane >= d ? max(end, o) : end;
      }
      end = max(end, row);
      int before = __shfl_up_sync(0xffffffffu, end, 1);
      before = lane == 0 ? row : before;
      int t = (end - before + tile - 1) / tile;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, t, d);
        t += lane >= d ? o : 0;
      }
      t += tiles;
      if (e < experts)
        first_row[e + 1] = end, first_tile[e + 1] = t;
      row = __shfl_sync(0xffffffffu, end, 31);
      tiles = __shfl_sync(0xffffffffu, t, 31);
    }
  }
  __syncthreads();
}

// The expert whose tiles hold tile t < first_tile[experts]: the last e with first_tile[e] <= t.
__device__ __forceinline__ int expert_of_tile(const int* first_tile, int experts, int t) {
  int lo = 0, hi = experts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

}  // namespace mxb200
