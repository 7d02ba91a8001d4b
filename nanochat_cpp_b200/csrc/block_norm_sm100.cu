// RMS norm behind a residual add, its result in the 128-value block format, and its backward.
//
//   res = bf16(x + r),  rstd = 1 / sqrt(mean(res^2) + eps),  n = bf16(res rstd gain),  (q, scale) = rows of n in blocks of 128
//   d = dn gain,  hat = res rstd,  dx = bf16(rstd (d - hat mean(d hat)) + dres)  (of x and of r),  dgain = sum over rows of dn hat
//
// A row stays with its threads from load to store, in registers (beyond 8192 columns the backward spills 280 bytes a thread), so
// every tensor is read or written once; both kernels are bound by memory. Forward: a row of up to 2048 columns belongs to one warp, whose sums are shuffles, a wider one (up to 16384)
// to 256 threads; 16 lanes hold 128 consecutive values, one scale block. Backward: a block's threads own columns and go through
// its rows, several at a time. Sums, rstd and the gain's gradient are fp32.
//
// The gain's gradient: every CTA adds up its rows in a fixed order in registers and writes one row of partial sums; a second
// kernel adds those rows in order. No atomics: the same bits every time.
#include <algorithm>
#include <cstdint>
#include <mutex>

#include <cuda_bf16.h>

#include "bf16x2_sm100.cuh"
#include "block_common.cuh"
#include "internal.h"
#include "ptx_sm100.cuh"

namespace mxb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpCols = 2048, kMaxCols = 16384;

struct ForwardParams {
  const void* x;
  const void* r;
  const void* gain;
  void* res;
  void* n;
  uint8_t* q;
  float* scale;
  float* rstd;
  int64_t rows;
  int cols;
  int gain_bf16;
  float eps;
};

struct BackwardParams {
  const void* dn;
  const void* dres;
  const void* res;
  const float* rstd;
  const void* gain;
  void* dx;
  float* partial;  // (gridDim.x, cols); null: no gradient of the gain
  int64_t rows;
  int cols;
  int gain_bf16;
};

__device__ __forceinline__ void unpack(const uint4& w, float (&f)[8]) {
  f[0] = lo_f32(w.x), f[1] = hi_f32(w.x), f[2] = lo_f32(w.y), f[3] = hi_f32(w.y);
  f[4] = lo_f32(w.z), f[5] = hi_f32(w.z), f[6] = lo_f32(w.w), f[7] = hi_f32(w.w);
}

__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  return make_uint4(pack_bf16x2_rn(f[0], f[1]), pack_bf16x2_rn(f[2], f[3]), pack_bf16x2_rn(f[4], f[5]), pack_bf16x2_rn(f[6], f[7]));
}

__device__ __forceinline__ uint4 load16(const void* p, int64_t at) {
  return *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at);
}

__device__ __forceinline__ void store16(void* p, int64_t at, const uint4& w) {
  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at) = w;
}

__device__ __forceinline__ void load_gain(const void* gain, int gain_bf16, int col, float (&g)[8]) {
  if (gain == nullptr) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      g[k] = 1.f;
  } else if (gain_bf16) {
    unpack(load16(gain, col), g);
  } else {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(gain) + col);
    const float4 a = q[0], b = q[1];
    g[0] = a.x, g[1] = a.y, g[2] = a.z, g[3] = a.w, g[4] = b.x, g[5] = b.y, g[6] = b.z, g[7] = b.w;
  }
}

// Sum over the threads of a row: a warp, or all of the block (`parts`: a word per warp). Every thread gets it.
template <int kPerRow>
__device__ __forceinline__ float row_sum(float v, float* parts) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kPerRow > 32) {
    __syncthreads();  // the previous row's parts have been read
    if ((threadIdx.x & 31) == 0)
      parts[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kPerRow / 32; ++w)
      v += parts[w];
  }
  return v;
}

template <int kPerRow, int kVecs>
__device__ __forceinline__ void norm_forward(const ForwardParams& p) {
  __shared__ float parts[kThreads / 32];
  grid_dependency_wait();
  const int at = threadIdx.x % kPerRow;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kPerRow) + threadIdx.x / kPerRow;
  if (row >= p.rows)
    return;  // whole warps: a row of 256 threads is the whole block's
  uint4 v[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (i * kPerRow + at);
    v[i] = col < p.cols ? load16(p.x, row * p.cols + col) : make_uint4(0, 0, 0, 0);
  }
  if (p.r != nullptr) {
    uint4 r[kVecs];  // all on their way before the first store
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (i * kPerRow + at);
      r[i] = col < p.cols ? load16(p.r, row * p.cols + col) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int col = 8 * (i * kPerRow + at);
      v[i] = make_uint4(add_bf16x2(v[i].x, r[i].x), add_bf16x2(v[i].y, r[i].y), add_bf16x2(v[i].z, r[i].z), add_bf16x2(v[i].w, r[i].w));
      if (col < p.cols)
        store16(p.res, row * p.cols + col, v[i]);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float f[8];
    unpack(v[i], f);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      sum = fmaf(f[k], f[k], sum);
  }
  sum = row_sum<kPerRow>(sum, parts);
  const float rstd = __frsqrt_rn(sum / static_cast<float>(p.cols) + p.eps);
  if (at == 0)
    p.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (i * kPerRow + at);
    const bool in = col < p.cols;
    float f[8], g[8];
    if (in)
      load_gain(p.gain, p.gain_bf16, col, g);
    unpack(v[i], f);
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f[k] = in ? f[k] * rstd * g[k] : 0.f;
    const uint4 w = pack(f);
    if (in && p.n != nullptr)
      store16(p.n, row * p.cols + col, w);
    unpack(w, f);  // what is quantized is the bf16 n
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m = fmaxf(m, fabsf(f[k]));
#pragma unroll
    for (int d = 8; d > 0; d >>= 1)
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const int e = block_exponent(__float_as_uint(m));
    const float by = __uint_as_float(mx_multiplier_bits(e));
    if (in) {
      *reinterpret_cast<uint2*>(p.q + row * p.cols + col) =
            make_uint2(e4m3x4_from_f32(f[0] * by, f[1] * by, f[2] * by, f[3] * by),
                       e4m3x4_from_f32(f[4] * by, f[5] * by, f[6] * by, f[7] * by));
      if ((at & 15) == 0)
        p.scale[(col / kBlock) * p.rows + row] = __uint_as_float(static_cast<uint32_t>(e) << 23);
    }
  }
}

// A block's threads own columns (8 kVecs each) and go through its rows kRows at a time, so that the gain's sums of a thread are
// few and its loads many. One barrier per step: the rows' sums of one step are gathered while the other half of `parts` may still
// be read.
template <int kVecs, int kRows>
__device__ __forceinline__ void norm_backward(const BackwardParams& p) {
  __shared__ float parts[2][kRows][kThreads / 32];
  grid_dependency_wait();
  const int threads = blockDim.x, warps = threads / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float gain[kVecs][8], dgain[kVecs][8];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (i * threads + threadIdx.x);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      gain[i][k] = 1.f, dgain[i][k] = 0.f;
    if (col < p.cols)
      load_gain(p.gain, p.gain_bf16, col, gain[i]);
  }
  // the next step's rows are on their way while this one's are worked on, as long as registers hold them
  constexpr bool kAhead = kVecs < 8;
  uint4 v[1 + kAhead][kRows][kVecs], d[1 + kAhead][kRows][kVecs], o[1 + kAhead][kRows][kVecs];
  float rstd[1 + kAhead][kRows];
  const auto load = [&](int64_t row, int to) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool there = row + r < p.rows;
      rstd[to][r] = there ? p.rstd[row + r] : 0.f;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = 8 * (i * threads + threadIdx.x);
        const int64_t at = (row + r) * p.cols + col;
        const bool in = there && col < p.cols;
        v[to][r][i] = in ? load16(p.res, at) : make_uint4(0, 0, 0, 0);
        d[to][r][i] = in ? load16(p.dn, at) : make_uint4(0, 0, 0, 0);
        o[to][r][i] = in && p.dres != nullptr ? load16(p.dres, at) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  const auto work = [&](int64_t row, int at) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        float f[8], h[8];
        unpack(v[at][r][i], h);
        unpack(d[at][r][i], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = f[k] * (h[k] * rstd[at][r]);
          dgain[i][k] += t;
          sum = fmaf(t, gain[i][k], sum);
        }
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (lane == 0)
        parts[at][r][warp] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float mean = 0.f;
      for (int w = 0; w < warps; ++w)
        mean += parts[at][r][w];
      mean /= static_cast<float>(p.cols);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int col = 8 * (i * threads + threadIdx.x);
        float f[8], h[8], e[8];
        unpack(v[at][r][i], h);
        unpack(d[at][r][i], f);
        unpack(o[at][r][i], e);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          f[k] = rstd[at][r] * (f[k] * gain[i][k] - h[k] * rstd[at][r] * mean) + e[k];
        if (row + r < p.rows && col < p.cols)
          store16(p.dx, (row + r) * p.cols + col, pack(f));
      }
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows;
  if constexpr (kAhead) {
    load(row, 0);
    for (; row < p.rows; row += 2 * step) {
      load(row + step, 1);
      work(row, 0);
      if (row + step >= p.rows)
        break;
      load(row + 2 * step, 0);
      work(row + step, 1);
    }
  } else {
    for (; row < p.rows; row += step) {
      load(row, 0);
      work(row, 0);
      __syncthreads();  // the rows' sums have been read
    }
  }
  if (p.partial == nullptr)
    return;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int col = 8 * (i * threads + threadIdx.x);
    if (col < p.cols) {
      float4* out = reinterpret_cast<float4*>(p.partial + static_cast<int64_t>(blockIdx.x) * p.cols + col);
      out[0] = make_float4(dgain[i][0], dgain[i][1], dgain[i][2], dgain[i][3]);
      out[1] = make_float4(dgain[i][4], dgain[i][5], dgain[i][6], dgain[i][7]);
    }
  }
}

}  // namespace
}  // namespace mxb200

// kVecs: 8-value vectors per thread
#define MXB200_NORM_KERNEL(per_row, vecs)                                                                                             \
  __global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_norm_##per_row##x##vecs(const __grid_constant__ mxb200::ForwardParams p) { \
    mxb200::norm_forward<per_row, vecs>(p);                                                                                           \
  }
#define MXB200_NORM_BACKWARD_KERNEL(vecs, rows)                                                                                       \
  __global__ void __launch_bounds__(mxb200::kThreads) mxb200_block_norm_bwd_##vecs##x##rows(const __grid_constant__ mxb200::BackwardParams p) { \
    mxb200::norm_backward<vecs, rows>(p);                                                                                             \
  }
MXB200_NORM_KERNEL(32, 2)
MXB200_NORM_KERNEL(32, 4)
MXB200_NORM_KERNEL(32, 6)
MXB200_NORM_KERNEL(32, 8)
MXB200_NORM_KERNEL(256, 2)
MXB200_NORM_KERNEL(256, 4)
MXB200_NORM_KERNEL(256, 8)
MXB200_NORM_BACKWARD_KERNEL(1, 2)
MXB200_NORM_BACKWARD_KERNEL(2, 1)
MXB200_NORM_BACKWARD_KERNEL(4, 1)
MXB200_NORM_BACKWARD_KERNEL(8, 1)

// The rows of partial sums: 32 columns per block, whose 32 warps each add every 32nd row in order, then the warps' sums in order.
__global__ void __launch_bounds__(1024) mxb200_block_norm_sum_gain(const float* partial, int parts, int cols, void* out, int out_bf16) {
  __shared__ float share[32][32];
  mxb200::grid_dependency_wait();
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, g = threadIdx.x >> 5;
  float sum = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int i = g; i < parts; i += 32)
      sum += partial[static_cast<int64_t>(i) * cols + c];
  }
  share[g][lane] = sum;
  __syncthreads();
  if (g != 0 || c >= cols)
    return;
#pragma unroll
  for (int i = 1; i < 32; ++i)
    sum += share[i][lane];
  if (out_bf16)
    static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(sum);
  else
    static_cast<float*>(out)[c] = sum;
}

namespace mxb200 {
namespace {

struct Forward {
  void (*kernel)(ForwardParams);
  int rows_per_block;
};

// One warp per row as long as its registers hold it (64 values per lane), then the whole block.
Forward forward_of(int cols) {
  const int vecs = cols / 8;
  if (cols <= kWarpCols) {
    if (vecs <= 64)
      return {mxb200_block_norm_32x2, kThreads / 32};
    if (vecs <= 128)
      return {mxb200_block_norm_32x4, kThreads / 32};
    if (vecs <= 192)
      return {mxb200_block_norm_32x6, kThreads / 32};
    return {mxb200_block_norm_32x8, kThreads / 32};
  }
  if (vecs <= 512)
    return {mxb200_block_norm_256x2, 1};
  if (vecs <= 1024)
    return {mxb200_block_norm_256x4, 1};
  return {mxb200_block_norm_256x8, 1};
}

constexpr int kBackwards = 4;

struct Backward {
  int id;
  void (*kernel)(BackwardParams);
  int threads, rows_per_step;
  int blocks_per_sm;  // at most; resident() says how many there is room for
};

// As many threads as a row has vectors of 8, up to 256, then more vectors per thread.
Backward backward_of(int cols) {
  const int vecs = cols / 8;
  const auto threads = [&](int per_thread) { return ((vecs + per_thread - 1) / per_thread + 31) / 32 * 32; };
  if (vecs <= kThreads)
    return {0, mxb200_block_norm_bwd_1x2, threads(1), 2, std::min(8, 512 / threads(1))};
  if (vecs <= 2 * kThreads)
    return {1, mxb200_block_norm_bwd_2x1, threads(2), 1, 2};
  if (vecs <= 4 * kThreads)
    return {2, mxb200_block_norm_bwd_4x1, threads(4), 1, 2};
  return {3, mxb200_block_norm_bwd_8x1, threads(8), 1, 1};
}

int check_shape(int64_t rows, int32_t cols) {
  return rows < 0 || rows > kMostSize || cols <= 0 || cols > kMaxCols || cols % 16 ? MXB200_ERR_SHAPE : MXB200_OK;
}

// needed pointers first, then optional ones
int check_pointers(std::initializer_list<const void*> needed, std::initializer_list<const void*> optional) {
  for (const void* q : needed)
    if (q == nullptr)
      return MXB200_ERR_NULL;
  for (const auto* list : {&needed, &optional})
    for (const void* q : *list)
      if (!aligned16(q))
        return MXB200_ERR_ALIGNMENT;
  return MXB200_OK;
}

// How many of the kernel's blocks an SM of this device holds, asked once for each size of block. 0: the question failed.
int resident(const Backward& v, const DeviceInfo& dev) {
  static std::mutex mu;
  static int known[64][kBackwards][kThreads / 32];
  std::lock_guard<std::mutex> lock(mu);
  int local = 0;
  int& blocks = dev.device < 64 ? known[dev.device][v.id][v.threads / 32 - 1] : local;
  if (blocks == 0 &&
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, reinterpret_cast<const void*>(v.kernel), v.threads, 0) != cudaSuccess) {
    cudaGetLastError();
    blocks = 0;
  }
  return blocks;
}

// CTAs of the backward: one round of what the SMs hold, fewer where there are not the rows; 0: not known. A second round
// fills its pipeline anew and writes as many partial sums again: 4096 x 8192 takes 49.9 us in one round of 148 CTAs and 53.4 in
// two, 509 x 5040 9.7 and 11.5. (Without the loads ahead an SM has room for two of these CTAs; they take 64.4 and 12.8.)
int64_t backward_blocks(int64_t rows, const Backward& v, const DeviceInfo& dev) {
  const int64_t at_once = static_cast<int64_t>(std::min(v.blocks_per_sm, resident(v, dev))) * dev.sms;
  return std::min<int64_t>(std::max<int64_t>(1, (rows + v.rows_per_step - 1) / v.rows_per_step), at_once);
}

}  // namespace
}  // namespace mxb200

extern "C" int mxb200_block_norm_fwd(const mxb200_block_norm_args* a, void* stream) {
  using namespace mxb200;
  if (a == nullptr)
    return MXB200_ERR_NULL;
  if (int st = check_shape(a->rows, a->cols); st != MXB200_OK)
    return st;
  if (a->rows == 0)
    return MXB200_OK;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  if (int st = check_pointers({a->x, a->rstd, a->q, a->scale}, {a->r, a->gain, a->res, a->n}); st != MXB200_OK)
    return st;
  if ((a->r == nullptr) != (a->res == nullptr))
    return MXB200_ERR_ARGUMENT;
  const Forward v = forward_of(a->cols);
  const ForwardParams p{a->x, a->r, a->gain, a->res, a->n, static_cast<uint8_t*>(a->q), a->scale, a->rstd,
                        a->rows, a->cols, a->gain_bf16, a->eps};
  return launch_kernel(v.kernel, static_cast<unsigned>((a->rows + v.rows_per_block - 1) / v.rows_per_block), kThreads, 0,
                       static_cast<cudaStream_t>(stream), p);
}

extern "C" size_t mxb200_block_norm_workspace_bytes(int64_t rows, int32_t cols) {
  using namespace mxb200;
  DeviceInfo dev;
  if (check_shape(rows, cols) != MXB200_OK || current_device(&dev) != MXB200_OK)
    return 0;
  return static_cast<size_t>(backward_blocks(rows, backward_of(cols), dev)) * cols * sizeof(float);
}

extern "C" int mxb200_block_norm_bwd(const mxb200_block_norm_bwd_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mxb200;
  if (a == nullptr)
    return MXB200_ERR_NULL;
  if (int st = check_shape(a->rows, a->cols); st != MXB200_OK)
    return st;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  const auto s = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {
    if (a->dgain != nullptr && cudaMemsetAsync(a->dgain, 0, a->cols * (a->gain_bf16 ? size_t{2} : size_t{4}), s) != cudaSuccess)
      return MXB200_ERR_LAUNCH;
    return MXB200_OK;
  }
  if (int st = check_pointers({a->dn, a->res, a->rstd, a->dx}, {a->dres, a->gain, a->dgain, workspace}); st != MXB200_OK)
    return st;
  if (a->dgain != nullptr && a->gain == nullptr)
    return MXB200_ERR_ARGUMENT;
  if (a->dgain != nullptr && (workspace == nullptr || workspace_bytes < mxb200_block_norm_workspace_bytes(a->rows, a->cols)))
    return MXB200_ERR_WORKSPACE;
  const Backward v = backward_of(a->cols);
  const int blocks = static_cast<int>(backward_blocks(a->rows, v, dev));
  if (blocks == 0)
    return MXB200_ERR_LAUNCH;
  float* partial = a->dgain != nullptr ? static_cast<float*>(workspace) : nullptr;
  const BackwardParams p{a->dn, a->dres, a->res, a->rstd, a->gain, a->dx, partial, a->rows, a->cols, a->gain_bf16};
  if (int st = launch_kernel(v.kernel, static_cast<unsigned>(blocks), v.threads, 0, s, p); st != MXB200_OK || partial == nullptr)
    return st;
  return launch_kernel(mxb200_block_norm_sum_gain, static_cast<unsigned>((a->cols + 31) / 32), 1024, 0, s,
                       static_cast<const float*>(partial), blocks, static_cast<int>(a->cols), a->dgain, static_cast<int>(a->gain_bf16));
}
