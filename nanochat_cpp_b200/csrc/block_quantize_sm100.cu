// Quantizers of the 128-value block format: E4M3 with one fp32 power-of-two scale per block.
//
//   rows     128 values of a row (activations and gradients on their way into the forward and the input gradient)
//   tokens   128 rows of a column, blocks starting over at every expert's first row (both operands of a weight gradient)
//   weight   128 x 128 values
//
// Scale = the smallest power of two s >= 2^-126 with max|block| <= 448 s, so x / s is exact and E4M3 rounds once. NaN does not
// count in the maximum and stays NaN; Inf saturates to 448 s.
//
// All three work on 128 x 128 tiles, 256 threads: 16 lanes hold a row's 128 values, 8 each, and a thread 8 rows 16 apart, all
// loaded before the first is used. A row's maximum is taken by shuffles over 16 lanes, a column's through shared memory. Bound by
// memory: 2 bytes read and 1 written per value and layout; both layouts of an activation come from one read. Data never leaves
// transposed, since the matrix product reads either orientation.
#include <algorithm>
#include <cstdint>

#include <cuda_bf16.h>

#include "bf16x2_sm100.cuh"
#include "block_common.cuh"
#include "internal.h"
#include "ptx_sm100.cuh"

namespace mxb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerThread = 8;

struct QuantizeParams {
  const void* x;
  int64_t ld;           // values between rows
  int64_t x_expert;     // weight: values between experts
  int64_t rows, cols;
  const int32_t* ends;  // tokens: rows by expert
  int experts;
  uint8_t* row_data;    // rows: (rows, cols); null where they are not wanted
  float* row_scale;     // (cols / 128, rows)
  uint8_t* col_data;    // tokens: (token blocks * 128, cols); weight: (experts, rows, cols)
  float* col_scale;     // weight: (experts, rows / 128, cols / 128)
  uint32_t* col_scale_words;  // tokens: (token blocks, cols / 128, 128); weight: (experts, rows / 128, cols / 128, 128) or null
  uint32_t* row_scale_words;  // rows in the experts' token blocks: (token blocks, cols / 128, 128)
};

struct Values {
  float v[8];
};

template <bool kBf16>
__device__ __forceinline__ Values load_values(const void* x, int64_t at) {
  Values r;
  if constexpr (kBf16) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(x) + at);
    r.v[0] = lo_f32(w.x), r.v[1] = hi_f32(w.x), r.v[2] = lo_f32(w.y), r.v[3] = hi_f32(w.y);
    r.v[4] = lo_f32(w.z), r.v[5] = hi_f32(w.z), r.v[6] = lo_f32(w.w), r.v[7] = hi_f32(w.w);
  } else {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 a = q[0], b = q[1];
    r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w, r.v[4] = b.x, r.v[5] = b.y, r.v[6] = b.z, r.v[7] = b.w;
  }
  return r;
}

__device__ __forceinline__ float scale_of(int exponent) {
  return __uint_as_float(static_cast<uint32_t>(exponent) << 23);
}

__device__ __forceinline__ float multiplier_of(int exponent) {
  return __uint_as_float(mx_multiplier_bits(exponent));
}

__device__ __forceinline__ int exponent_of(float amax) {
  return block_exponent(__float_as_uint(amax));
}

// 8 rows 16 apart of the tile from `row` on (rows_left of them exist), 8 columns at `at`.
template <bool kBf16>
__device__ __forceinline__ void load_tile(const void* x, int64_t at, int64_t ld, int row, int rows_left, bool col_ok, Values (&v)[kRowsPerThread]) {
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i) {
    if (col_ok && row + 16 * i < rows_left)
      v[i] = load_values<kBf16>(x, at + 16 * i * ld);
    else
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[i].v[k] = 0.f;
  }
}

// What the threads of a block share of an activation's tile.
struct TileShared {
  uint16_t row_by[kBlock];                                  // bf16 multipliers of the tile's rows; a warp reads its own rows' only
  uint8_t row_exponent[kBlock];
  __align__(16) uint32_t col_max[kThreads / 32][kBlock / 2];  // packed bf16: the warps' maxima of two columns
  __align__(16) uint32_t col_by[kBlock / 2];                  // packed bf16 multipliers of two columns
};

__device__ __forceinline__ uint16_t by_of(int exponent) {
  return static_cast<uint16_t>(mx_multiplier_bits(exponent) >> 16);
}

// A block of rows at a time, its column tiles with a stride of gridDim.y. The values stay packed bf16: maxima by
// max.xorsign.abs.bf16x2, the product with the scale's reciprocal (a power of two, a bf16 number) by fma.rn.f32.bf16.
enum Rows : int { kNoRows, kRowsInPlace, kRowsInBlocks };

template <int kRows, bool kTokens>
__device__ __forceinline__ void quantize_activation(const QuantizeParams& p, TileShared* s, int* first_row, int* first_tile, int* tmp) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lane16 = lane & 15, row = threadIdx.x >> 4;
  int64_t row0 = static_cast<int64_t>(blockIdx.x) * kBlock;
  int rows_left;
  if constexpr (kTokens) {
    scan_experts(p.ends, p.experts, static_cast<int>(p.rows), kBlock, first_row, first_tile, tmp);
    if (static_cast<int>(blockIdx.x) >= first_tile[p.experts])
      return;
    const int e = expert_of_tile(first_tile, p.experts, blockIdx.x);
    const int r = first_row[e] + (static_cast<int>(blockIdx.x) - first_tile[e]) * kBlock;
    row0 = r;
    rows_left = min(kBlock, first_row[e + 1] - r);
  } else {
    rows_left = static_cast<int>(min(static_cast<int64_t>(kBlock), p.rows - row0));
  }
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + (row0 + row) * p.ld;
  uint8_t* row_out = p.row_data + ((kRows == kRowsInBlocks ? static_cast<int64_t>(blockIdx.x) * kBlock : row0) + row) * p.cols;
  const int tiles = static_cast<int>((p.cols + kBlock - 1) / kBlock);
  for (int t = blockIdx.y; t < tiles; t += gridDim.y) {
    const int64_t col = static_cast<int64_t>(t) * kBlock + 8 * lane16;
    const bool col_ok = col < p.cols;
    uint4 v[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i)
      v[i] = col_ok && row + 16 * i < rows_left ? *reinterpret_cast<const uint4*>(x + 16 * i * p.ld + col) : make_uint4(0, 0, 0, 0);
    if constexpr (kTokens) {
      uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kRowsPerThread; ++i) {
        m[0] = max_abs_skip_nan_bf16x2(m[0], v[i].x), m[1] = max_abs_skip_nan_bf16x2(m[1], v[i].y);
        m[2] = max_abs_skip_nan_bf16x2(m[2], v[i].z), m[3] = max_abs_skip_nan_bf16x2(m[3], v[i].w);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        m[k] = max_abs_skip_nan_bf16x2(m[k], __shfl_xor_sync(0xffffffffu, m[k], 16));
      if (lane < 16)
        *reinterpret_cast<uint4*>(&s->col_max[warp][4 * lane]) = make_uint4(m[0], m[1], m[2], m[3]);
    }
    if constexpr (kRows != kNoRows) {
      // eight rows' maxima over 16 lanes: each exchange halves the rows that a lane goes on with
      uint32_t m[kRowsPerThread];
#pragma unroll
      for (int i = 0; i < kRowsPerThread; ++i) {
        const uint32_t w = max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(0u, v[i].x), v[i].y), v[i].z), v[i].w) & 0x7fff7fffu;
        m[i] = max(w & 0xffffu, w >> 16);
      }
#pragma unroll
      for (int n = 4, d = 8; n > 0; n >>= 1, d >>= 1) {
        const bool upper = (lane & d) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const uint32_t sent = upper ? m[i] : m[i + n], kept = upper ? m[i + n] : m[i];
          m[i] = max(kept, __shfl_xor_sync(0xffffffffu, sent, d));
        }
      }
      m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
      const int e = block_exponent(m[0] << 16);
      // lanes with bit 0 clear: row i of this half warp, i from lane bits 3, 2, 1
      const int i = ((lane >> 3) & 1) * 4 + ((lane >> 2) & 1) * 2 + ((lane >> 1) & 1);
      __syncwarp();  // the previous tile's multipliers have been read
      if ((lane & 1) == 0)
        s->row_by[row + 16 * i] = by_of(e), s->row_exponent[row + 16 * i] = static_cast<uint8_t>(e);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kRowsPerThread; ++k)
        if (col_ok && (kRows == kRowsInBlocks || row + 16 * k < rows_left)) {
          const uint16_t by = s->row_by[row + 16 * k];
          *reinterpret_cast<uint2*>(row_out + 16 * k * p.cols + col) =
                make_uint2(e4m3x4_scaled_fma(v[k].x, v[k].y, by, by), e4m3x4_scaled_fma(v[k].z, v[k].w, by, by));
        }
    }
    __syncthreads();
    if (kRows == kRowsInPlace && threadIdx.x < rows_left)
      p.row_scale[static_cast<int64_t>(t) * p.rows + row0 + threadIdx.x] = scale_of(s->row_exponent[threadIdx.x]);
    if (kRows == kRowsInBlocks && threadIdx.x < kBlock)
      p.row_scale_words[(static_cast<int64_t>(blockIdx.x) * tiles + t) * kBlock + (threadIdx.x & 31) * 4 + (threadIdx.x >> 5)] =
            s->row_exponent[threadIdx.x] * 0x01010101u;
    if constexpr (kTokens) {
      if (threadIdx.x < kBlock / 2) {
        uint32_t m = s->col_max[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w)
          m = max_abs_skip_nan_bf16x2(m, s->col_max[w][threadIdx.x]);
        m &= 0x7fff7fffu;
        const int e[2] = {block_exponent(m << 16), block_exponent(m & 0xffff0000u)};
        s->col_by[threadIdx.x] = by_of(e[0]) | static_cast<uint32_t>(by_of(e[1])) << 16;
        // a tile of 128 columns' scale bytes, each four times, in the order that the copy to tensor memory takes
        uint32_t* words = p.col_scale_words + (static_cast<int64_t>(blockIdx.x) * tiles + t) * kBlock;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = 2 * threadIdx.x + k;
          words[(c & 31) * 4 + (c >> 5)] = static_cast<uint32_t>(e[k]) * 0x01010101u;
        }
      }
      __syncthreads();
      if (col_ok) {
        const uint4 by = *reinterpret_cast<const uint4*>(&s->col_by[4 * lane16]);
        uint8_t* out = p.col_data + (static_cast<int64_t>(blockIdx.x) * kBlock + row) * p.cols + col;
#pragma unroll
        for (int k = 0; k < kRowsPerThread; ++k)  // rows that do not exist are zeros: they count in the product
          *reinterpret_cast<uint2*>(out + 16 * k * p.cols) =
                make_uint2(e4m3x4_scaled_each(v[k].x, v[k].y, by.x, by.y), e4m3x4_scaled_each(v[k].z, v[k].w, by.z, by.w));
      }
    } else if (gridDim.y < tiles) {
      __syncthreads();  // the scales have been read
    }
  }
}

template <bool kBf16>
__device__ __forceinline__ void quantize_weight(const QuantizeParams& p, float* partial) {
  grid_dependency_wait();
  const int lane16 = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t tiles_n = (p.cols + kBlock - 1) / kBlock, tiles_m = (p.rows + kBlock - 1) / kBlock;
  const int64_t tile = blockIdx.x;
  const int64_t e = tile / (tiles_m * tiles_n), tm = tile / tiles_n % tiles_m, tn = tile % tiles_n;
  const int64_t row0 = tm * kBlock, col = tn * kBlock + 8 * lane16;
  const int rows_left = static_cast<int>(min(static_cast<int64_t>(kBlock), p.rows - row0));
  const bool col_ok = col < p.cols;
  Values v[kRowsPerThread];
  load_tile<kBf16>(p.x, e * p.x_expert + (row0 + row) * p.ld + col, p.ld, row, rows_left, col_ok, v);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m = fmaxf(m, fabsf(v[i].v[k]));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if ((threadIdx.x & 31) == 0)
    partial[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w)
    m = fmaxf(m, partial[w]);
  const int ex = exponent_of(m);
  const float f = multiplier_of(ex);
#pragma unroll
  for (int i = 0; i < kRowsPerThread; ++i)
    if (col_ok && row + 16 * i < rows_left)
      *reinterpret_cast<uint2*>(p.col_data + (e * p.rows + row0 + row + 16 * i) * p.cols + col) =
            make_uint2(e4m3x4_from_f32(v[i].v[0] * f, v[i].v[1] * f, v[i].v[2] * f, v[i].v[3] * f),
                       e4m3x4_from_f32(v[i].v[4] * f, v[i].v[5] * f, v[i].v[6] * f, v[i].v[7] * f));
  if (p.col_scale_words == nullptr) {
    if (threadIdx.x == 0)
      p.col_scale[tile] = scale_of(ex);
  } else if (threadIdx.x < kBlock) {
    p.col_scale_words[tile * kBlock + threadIdx.x] = static_cast<uint32_t>(ex) * 0x01010101u;
  }
}

}  // namespace
}  // namespace mxb200

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_rows(const __grid_constant__ mxb200::QuantizeParams p) {
  __shared__ mxb200::TileShared s;
  mxb200::quantize_activation<mxb200::kRowsInPlace, false>(p, &s, nullptr, nullptr, nullptr);
}

template <int kRows>
__device__ __forceinline__ void quantize_tokens(const mxb200::QuantizeParams& p) {
  __shared__ int first_row[mxb200::kMaxExperts + 1], first_tile[mxb200::kMaxExperts + 1];
  __shared__ union {
    int tmp[mxb200::kMaxExperts];
    mxb200::TileShared tile;
  } u;
  mxb200::quantize_activation<kRows, true>(p, &u.tile, first_row, first_tile, u.tmp);
}

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_tokens(const __grid_constant__ mxb200::QuantizeParams p) {
  quantize_tokens<mxb200::kNoRows>(p);
}

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_both(const __grid_constant__ mxb200::QuantizeParams p) {
  quantize_tokens<mxb200::kRowsInPlace>(p);
}

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_both_in_blocks(const __grid_constant__ mxb200::QuantizeParams p) {
  quantize_tokens<mxb200::kRowsInBlocks>(p);
}

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_weight_bf16(const __grid_constant__ mxb200::QuantizeParams p) {
  __shared__ float partial[mxb200::kThreads / 32];
  mxb200::quantize_weight<true>(p, partial);
}

__global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_quantize_weight_f32(const __grid_constant__ mxb200::QuantizeParams p) {
  __shared__ float partial[mxb200::kThreads / 32];
  mxb200::quantize_weight<false>(p, partial);
}

namespace mxb200 {
namespace {

// Null or misaligned pointers among those that are needed.
int check_pointers(std::initializer_list<const void*> pointers) {
  for (const void* q : pointers) {
    if (q == nullptr)
      return MXB200_ERR_NULL;
    if (!aligned16(q))
      return MXB200_ERR_ALIGNMENT;
  }
  return MXB200_OK;
}

}  // namespace
}  // namespace mxb200

extern "C" int mxb200_block_quantize(const void* x, int64_t rows, int64_t cols, int64_t ld, const int32_t* ends, int experts,
                                     void* row_data, void* row_scale, int rows_in_blocks, void* token_data, uint32_t* token_scale, void* stream) {
  using namespace mxb200;
  if (rows < 0 || rows > kMostSize || cols <= 0 || cols > kMostSize || cols % 16 || ld < cols || ld % 8 || experts < 1 || experts > kMaxExperts)
    return MXB200_ERR_SHAPE;
  if (ends == nullptr && experts != 1)
    return MXB200_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(ends) & 3) != 0)
    return MXB200_ERR_ALIGNMENT;
  if (rows == 0)
    return MXB200_OK;
  const bool want_rows = row_data != nullptr, want_tokens = token_data != nullptr;
  if (!want_rows && !want_tokens)
    return MXB200_ERR_NULL;
  if (rows_in_blocks != 0 && !(want_rows && want_tokens))
    return MXB200_ERR_ARGUMENT;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  if (int st = check_pointers({x}); st != MXB200_OK)
    return st;
  if (int st = want_rows ? check_pointers({row_data, row_scale}) : MXB200_OK; st != MXB200_OK)
    return st;
  if (int st = want_tokens ? check_pointers({token_data, token_scale}) : MXB200_OK; st != MXB200_OK)
    return st;
  QuantizeParams p{};
  p.x = x, p.ld = ld, p.rows = rows, p.cols = cols, p.ends = ends, p.experts = experts;
  p.row_data = static_cast<uint8_t*>(row_data);
  if (rows_in_blocks != 0)
    p.row_scale_words = static_cast<uint32_t*>(row_scale);
  else
    p.row_scale = static_cast<float*>(row_scale);
  p.col_data = static_cast<uint8_t*>(token_data), p.col_scale_words = token_scale;
  // enough blocks to fill the machine; beyond that a block goes on to its rows' next columns, with its experts looked up once
  const int64_t blocks = want_tokens ? mxb200_block_token_blocks(rows, experts) : blocks_up(rows, kBlock);
  const int64_t parts = std::min<int64_t>(blocks_up(cols, kBlock), std::max<int64_t>(1, blocks_up(8 * dev.sms, blocks)));
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<int64_t>(parts, 65535)));
  const auto kernel = !want_tokens     ? mxb200_block_quantize_rows
                      : rows_in_blocks ? mxb200_block_quantize_both_in_blocks
                      : want_rows      ? mxb200_block_quantize_both
                                       : mxb200_block_quantize_tokens;
  return launch_kernel(kernel, grid, kThreads, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int mxb200_block_quantize_weight(const void* w, int w_bf16, int experts, int64_t rows, int64_t cols, void* data,
                                            void* scale, int in_tiles, void* stream) {
  using namespace mxb200;
  if (rows <= 0 || rows > kMostSize || cols <= 0 || cols > kMostSize || rows % 16 || cols % 16 || experts < 1 || experts > kMaxExperts)
    return MXB200_ERR_SHAPE;
  const int64_t tiles = experts * blocks_up(rows, kBlock) * blocks_up(cols, kBlock);
  if (tiles > kMostSize)
    return MXB200_ERR_SHAPE;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  if (int st = check_pointers({w, data, scale}); st != MXB200_OK)
    return st;
  QuantizeParams p{w, cols, rows * cols, rows, cols, nullptr, experts, nullptr, nullptr, static_cast<uint8_t*>(data), in_tiles ? nullptr : static_cast<float*>(scale),
                   in_tiles ? static_cast<uint32_t*>(scale) : nullptr, nullptr};
  return launch_kernel(w_bf16 ? mxb200_block_quantize_weight_bf16 : mxb200_block_quantize_weight_f32, static_cast<unsigned>(tiles),
                       kThreads, 0, static_cast<cudaStream_t>(stream), p);
}
