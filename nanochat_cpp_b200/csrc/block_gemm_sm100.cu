// Matrix products of E4M3 operands with one fp32 scale for 128 values along the contraction, dense and by expert.
//
//   forward       y[t, n]  = sum over blocks b of sx[b, t] sw[n / 128, b]  * sum over k in b of xq[t, k] wq[n, k]
//   input grad    dx[t, k] = sum over blocks b of sg[b, t] sw[b, k / 128]  * sum over n in b of gq[t, n] wq[n, k]
//   weight grad   dw[n, k] = sum over token blocks b of sg[b, n] sx[b, k]  * sum over t in b of gq[t, n] xq[t, k]
//
// Rows (tokens) may be sorted by expert; each expert has its own weight, and token blocks never cross experts.
//
// The scales are any fp32 numbers, so they cannot ride on the tensor core's own block scales (powers of two): the tensor core
// makes the plain fp32 product of one block (K = 128: four MMAs) in tensor memory, and the epilogue warps take it from there
// with one fused multiply-add per value into accumulators in registers, while the next block's MMAs fill another tensor
// memory buffer. The rows of the tensor core's tile (its lanes) are the weight's, the columns are tokens: few tokens then
// cost few columns, not a tile of 128 rows, and an expert's last tile is as narrow as its last rows.
//
// No operand is ever transposed in memory. The input gradient contracts over the weight's rows and the weight gradient over
// tokens; both read their operands as they lie, row-contiguous, through the tensor core's MN-major form.
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <mutex>

#include "bf16x2_sm100.cuh"
#include "block_common.cuh"
#include "internal.h"
#include "ptx_sm100.cuh"

namespace mxb200 {

// Non-zero after a bounded wait ran out: 0x20000000 | CTA << 8 | site.
__device__ uint32_t g_block_gemm_watchdog_word;

namespace {

constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr uint32_t kTmemCols = 512;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kStages = 5;
constexpr int kScaleSlots = 8;
constexpr uint32_t kABytes = 128 * 128, kBBytes = 128 * 128;
constexpr uint32_t kBBoxBytes = 32 * 128;  // tokens' rows come 32 at a time, as many as the tile has
constexpr int kPanel = 8;                  // weight tiles per raster panel

enum Mode : int { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };

enum WaitSite : uint32_t {
  kSiteStageEmpty = 1,
  kSiteScaleEmpty = 2,
  kSiteStageFull = 3,
  kSiteAccEmpty = 4,
  kSiteAccFull = 5,
  kSiteScaleFull = 6,
};

template <int kCtas>
struct Tile {
  static constexpr int kM = 128 * kCtas;
  static constexpr int kN = 128 * kCtas;
  static constexpr int kPartN = kN / 2;           // columns per epilogue warp: two warps share a tensor memory quarter
  static constexpr int kChunks = kPartN / 32;
  static constexpr int kAccBuffers = kTmemCols / kN;
};

// What the columns' scales and, for the weight gradient, the rows' are to one block.
struct ScaleSlot {
  float col[256];
  float row[128];  // [0] alone holds the weight's scale in the other two modes
};

constexpr uint32_t kStageRowBytes = 80;  // 32 bf16 and 16 bytes that put 8 rows' 16-byte pieces into different banks
constexpr uint32_t kOutBytes = 32 * kStageRowBytes;

struct Shared {
  ScaleSlot scales[kScaleSlots];
  unsigned char out[kEpilogueWarps][kOutBytes];
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[4], acc_empty[4];
  uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
  uint32_t tmem_base;
  uint32_t abort_flag;
  int first_row[kMaxExperts + 2];
  int first_tile[kMaxExperts + 2];
};

constexpr size_t kSmemBytes = 1024 + kStages * static_cast<size_t>(kABytes + kBBytes) + sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");
static_assert(kStages * kABytes >= kMaxExperts * 4, "the operand stages hold the scan's copy of ends");

struct Params {
  const float* col_scale;  // (blocks, col_ld)
  const float* row_scale;  // weight gradient: (blocks, row_ld); else the weight's (experts, ., .)
  int64_t col_ld, row_ld;
  int64_t w_scale_expert;
  int w_scale_m, w_scale_b;  // strides of the weight's scale over row tiles of 128 and over blocks
  void* d;
  const int32_t* ends;
  int experts;     // 1 where ends is null
  int rows;        // tokens
  int m, n;        // rows of the A operand; columns of the output of a weight gradient
  int blocks;      // contraction blocks (forward, input grad)
  int out_bf16;
};

struct Unit {
  int expert;
  int m0, n0;        // first row of A; first token, or first column of dw
  int cols;          // columns that exist
  int block0, blocks;
};

__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, Shared* s, uint32_t site) {
  bool ok = true;
  if (!mbar_try_wait(bar, parity)) {
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (!mbar_try_wait(bar, parity)) {
      if ((++spins & 63u) == 0) {
        if (*reinterpret_cast<volatile uint32_t*>(&s->abort_flag) != 0) {
          ok = false;
          break;
        }
        if (global_timer_ns() - t0 > kWaitLimitNs) {
          *reinterpret_cast<volatile uint32_t*>(&s->abort_flag) = 1;
          atomicCAS(&g_block_gemm_watchdog_word, 0u, 0x20000000u | (blockIdx.x << 8) | site);
          ok = false;
          break;
        }
      }
    }
  }
  return __all_sync(0xffffffffu, ok) != 0;
}

__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t pair_u32(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

__device__ __forceinline__ uint64_t pair_f32(float lo, float hi) {
  return pair_u32(__float_as_uint(lo), __float_as_uint(hi));
}

__device__ __forceinline__ float2 both(uint64_t v) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}

// The position a walk over units has in (expert, weight tile, token tile): all of a panel's weight tiles for one token tile,
// then for the next, so that the CTAs at work at one time share operands in L2.
template <int kMode, int kCtas>
__device__ __forceinline__ Unit unit_at(const Params& p, const Shared* s, int u) {
  using T = Tile<kCtas>;
  const int mt = (p.m + T::kM - 1) / T::kM;
  Unit x;
  int nt, v;
  if constexpr (kMode == kWeightGrad) {
    nt = (p.n + T::kN - 1) / T::kN;
    x.expert = u / (mt * nt);
    v = u - x.expert * mt * nt;
    x.block0 = s->first_tile[x.expert];
    x.blocks = s->first_tile[x.expert + 1] - x.block0;
  } else {
    const int t = u / mt;  // token tiles before this one, over all experts
    x.expert = expert_of_tile(s->first_tile, p.experts + (p.ends != nullptr), t);
    nt = s->first_tile[x.expert + 1] - s->first_tile[x.expert];
    v = u - s->first_tile[x.expert] * mt;
    x.block0 = 0;
    x.blocks = x.expert < p.experts ? p.blocks : 0;  // rows of no expert: zeros
  }
  const int panel = v / (kPanel * nt);
  v -= panel * kPanel * nt;
  const int width = min(kPanel, mt - panel * kPanel);
  const int n = v / width;
  x.m0 = (panel * kPanel + v - n * width) * T::kM;
  x.n0 = n * T::kN;
  if constexpr (kMode == kWeightGrad) {
    x.cols = min(T::kN, p.n - x.n0);
  } else {
    x.n0 += s->first_row[x.expert];
    x.cols = min(T::kN, s->first_row[x.expert + 1] - x.n0);
  }
  return x;
}

// ---------------------------------------------------------------------------------------------------- producer

template <int kMode, int kCtas>
__device__ __forceinline__ void produce(const Params& p, const CUtensorMap* map_a, const CUtensorMap* map_b, Shared* s,
                                        uint32_t a0, uint32_t b0, int rank, int first, int step, int units, int lane) {
  using T = Tile<kCtas>;
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t empty0 = smem_u32(&s->empty[0]), full0 = smem_u32(&s->full[0]);
  const uint32_t full_leader0 = kCtas == 2 ? map_to_cta(full0, 0) : full0;
  const uint32_t scale_full0 = smem_u32(&s->scale_full[0]), scale_empty0 = smem_u32(&s->scale_empty[0]);
  uint32_t stage = 0, phase = 0, slot = 0, slot_phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kMode, kCtas>(p, s, u);
    const int half = (x.cols + 16 * kCtas - 1) / (16 * kCtas) * 16;  // columns of the tile that this CTA brings
    const int row_a = x.m0 + rank * 128, col_b = x.n0 + rank * half;
    const int boxes = kMode == kWeightGrad ? 4 : (half + 31) / 32;
    const uint32_t bytes = kABytes + boxes * kBBoxBytes;
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(empty0 + stage * 8, phase ^ 1u, s, kSiteStageEmpty))
        return;
      const int k = (x.block0 + b) * kBlock;
      const uint32_t full = full_leader0 + stage * 8;
      if (rank == 0)
        mbar_arrive_expect_tx(el, full0 + stage * 8, bytes * kCtas);
      const int ax = kMode == kForward ? k : row_a, ay = kMode == kForward ? row_a : k;
      const int az = kMode == kWeightGrad ? 0 : x.expert;
      if constexpr (kCtas == 2)
        tma_load_3d_pair(el, a0 + stage * kABytes, map_a, full, ax, ay, az);
      else
        tma_load_3d(el, a0 + stage * kABytes, map_a, full, ax, ay, az);
      for (int i = 0; i < boxes; ++i) {
        const int bx = kMode == kWeightGrad ? col_b : k, by = (kMode == kWeightGrad ? k : col_b) + 32 * i;
        const uint32_t dst = b0 + stage * kBBytes + i * kBBoxBytes;
        if constexpr (kCtas == 2)
          tma_load_3d_pair(el, dst, map_b, full, bx, by, 0);
        else
          tma_load_3d(el, dst, map_b, full, bx, by, 0);
      }
      if (++stage == kStages)
        stage = 0, phase ^= 1u;

      // the block's scales
      if (!wait_bounded(scale_empty0 + slot * 8, slot_phase ^ 1u, s, kSiteScaleEmpty))
        return;
      const uint32_t dst = smem_u32(&s->scales[slot]);
      const float* col = p.col_scale + (x.block0 + b) * p.col_ld + x.n0;
      for (int i = lane; i < x.cols; i += 32)
        cp_async_4(dst + 4 * i, col + i);
      const uint32_t row_dst = dst + static_cast<uint32_t>(offsetof(ScaleSlot, row));
      if constexpr (kMode == kWeightGrad) {
        const float* row = p.row_scale + (x.block0 + b) * p.row_ld + row_a;
        for (int i = lane; i < 128; i += 32)
          if (row_a + i < p.m)
            cp_async_4(row_dst + 4 * i, row + i);
      } else if (lane == 0 && row_a < p.m) {
        cp_async_4(row_dst, p.row_scale + x.expert * p.w_scale_expert + (row_a >> 7) * static_cast<int64_t>(p.w_scale_m) +
                                  (x.block0 + b) * static_cast<int64_t>(p.w_scale_b));
      }
      cp_async_arrive(scale_full0 + slot * 8);
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
  }
}

// ---------------------------------------------------------------------------------------------------- MMA issuer

template <int kMode, int kCtas>
__device__ __forceinline__ void issue_mmas(const Params& p, Shared* s, uint32_t a0, uint32_t b0, uint32_t tmem_base, int first,
                                           int step, int units) {
  using T = Tile<kCtas>;
  constexpr bool kAMn = kMode != kForward, kBMn = kMode == kWeightGrad;
  // 128-byte swizzle, groups of 8 rows of 128 bytes 1024 apart. K-major: K = 32 is 32 bytes within a row; MN-major: 32 rows.
  constexpr uint32_t kAStep = kAMn ? 4096 >> 4 : 32 >> 4, kBStep = kBMn ? 4096 >> 4 : 32 >> 4;
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t empty0 = smem_u32(&s->empty[0]), full0 = smem_u32(&s->full[0]);
  const uint64_t a_desc0 = make_smem_desc(a0, 1024, 1024, 2), b_desc0 = make_smem_desc(b0, 1024, 1024, 2);
  uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kMode, kCtas>(p, s, u);
    const uint32_t n = (x.cols + 16 * kCtas - 1) / (16 * kCtas) * (16 * kCtas);
    const uint32_t idesc = make_idesc_f8(T::kM, n, kAMn, kBMn);
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(smem_u32(&s->acc_empty[buf]), buf_phase ^ 1u, s, kSiteAccEmpty) ||
          !wait_bounded(full0 + stage * 8, phase, s, kSiteStageFull))
        return;
      tcgen05_fence_after_sync();
      const uint32_t acc = tmem_base + buf * T::kN;
      const uint64_t a = a_desc0 + stage * (kABytes >> 4), bd = b_desc0 + stage * (kBBytes >> 4);
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        if constexpr (kCtas == 2)
          tcgen05_mma_f8_pair(el, acc, a + k * kAStep, bd + k * kBStep, idesc, k > 0);
        else
          tcgen05_mma_f8(el, acc, a + k * kAStep, bd + k * kBStep, idesc, k > 0);
      }
      if constexpr (kCtas == 2) {
        tcgen05_commit_pair(el, empty0 + stage * 8, 3);
        tcgen05_commit_pair(el, &s->acc_full[buf], 3);
      } else {
        tcgen05_commit(el, &s->empty[stage]);
        tcgen05_commit(el, &s->acc_full[buf]);
      }
      if (++stage == kStages)
        stage = 0, phase ^= 1u;
      if (++buf == T::kAccBuffers)
        buf = 0, buf_phase ^= 1u;
    }
  }
}

// ---------------------------------------------------------------------------------------------------- epilogue

// 32 columns of this warp's 32 rows to the output. v[j][i]: 8-column group j, row 8 i + lane / 4, columns 2 (lane % 4), + 1.
template <int kMode>
__device__ __forceinline__ void store_chunk(const Params& p, const Unit& x, unsigned char* stage, int lane, int row0, int c0,
                                            const uint64_t (&v)[4][4]) {
  const uint32_t st = smem_u32(stage);
  if (kMode == kWeightGrad && !p.out_bf16) {
    float* d = static_cast<float*>(p.d) + static_cast<int64_t>(x.expert) * p.m * p.n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 8 * i + (lane >> 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + 8 * j + 2 * (lane & 3);
        if (row < p.m && c < x.cols)
          *reinterpret_cast<float2*>(d + static_cast<int64_t>(row) * p.n + x.n0 + c) = both(v[j][i]);
      }
    }
    return;
  }
  __syncwarp();  // the previous chunk has been read out
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(v[j][i]);
      h[i] = pack_bf16x2_rn(f.x, f.y);
    }
    if constexpr (kMode == kWeightGrad)  // a row of the stage: 32 columns of one row of dw
      stmatrix_x4(st + lane * kStageRowBytes + j * 16, h[0], h[1], h[2], h[3]);
    else  // ... 32 features of one token
      stmatrix_x4_trans(st + (8 * j + (lane & 7)) * kStageRowBytes + (lane >> 3) * 16, h[0], h[1], h[2], h[3]);
  }
  __syncwarp();
  uint16_t* d = static_cast<uint16_t*>(p.d);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2), piece = lane & 3;
    const uint4 w = *reinterpret_cast<const uint4*>(stage + r * kStageRowBytes + piece * 16);
    if constexpr (kMode == kWeightGrad) {
      const int64_t row = static_cast<int64_t>(x.expert) * p.m + row0 + r;
      if (row0 + r < p.m && c0 + piece * 8 < x.cols)
        *reinterpret_cast<uint4*>(d + row * p.n + x.n0 + c0 + piece * 8) = w;
    } else {
      if (c0 + r < x.cols && row0 + piece * 8 < p.m)
        *reinterpret_cast<uint4*>(d + static_cast<int64_t>(x.n0 + c0 + r) * p.m + row0 + piece * 8) = w;
    }
  }
}

template <int kMode, int kCtas>
__device__ __forceinline__ void accumulate(const Params& p, Shared* s, uint32_t tmem_base, int rank, int first, int step, int units,
                                           int warp, int lane) {
  using T = Tile<kCtas>;
  const int quarter = warp & 3, part = (warp - 2) >> 2;  // a warp may read the tensor memory lanes 32 (warp % 4) on
  const int part0 = part * T::kPartN;
  const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
  const uint32_t acc_empty0 = kCtas == 2 ? map_to_cta(smem_u32(&s->acc_empty[0]), 0) : smem_u32(&s->acc_empty[0]);
  unsigned char* stage = s->out[warp - 2];
  uint32_t buf = 0, buf_phase = 0, slot = 0, slot_phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kMode, kCtas>(p, s, u);
    uint64_t acc[T::kChunks][4][4];
#pragma unroll
    for (int c = 0; c < T::kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[c][j][i] = 0;
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(smem_u32(&s->scale_full[slot]), slot_phase, s, kSiteScaleFull) ||
          !wait_bounded(smem_u32(&s->acc_full[buf]), buf_phase, s, kSiteAccFull))
        return;
      tcgen05_fence_after_sync();
      const ScaleSlot& sc = s->scales[slot];
      uint64_t row_scale[4];
      if constexpr (kMode == kWeightGrad) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = sc.row[quarter * 32 + 8 * i + (lane >> 2)];
          row_scale[i] = pair_f32(f, f);
        }
      } else {
        row_scale[0] = pair_f32(sc.row[0], sc.row[0]);
      }
      const uint32_t t = tmem_base + lane_base + buf * T::kN + part0;
#pragma unroll
      for (int c = 0; c < T::kChunks; ++c) {
        if (part0 + 32 * c >= x.cols)
          break;
        uint32_t lo[16], hi[16];
        tmem_ld_16x256b_x4(t + 32 * c, lo);
        tmem_ld_16x256b_x4(t + 32 * c + (16u << 16), hi);
        uint64_t col[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = *reinterpret_cast<const float2*>(&sc.col[part0 + 32 * c + 8 * j + 2 * (lane & 3)]);
          col[j] = pair_f32(f.x, f.y);
          if constexpr (kMode != kWeightGrad)
            col[j] = mul_f32x2(col[j], row_scale[0]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k)
          asm volatile("" : "+r"(lo[k]), "+r"(hi[k]));
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t v = i < 2 ? pair_u32(lo[4 * j + 2 * i], lo[4 * j + 2 * i + 1])
                                     : pair_u32(hi[4 * j + 2 * i - 4], hi[4 * j + 2 * i - 3]);
            const uint64_t f = kMode == kWeightGrad ? mul_f32x2(col[j], row_scale[i]) : col[j];
            acc[c][j][i] = fma_f32x2(v, f, acc[c][j][i]);
          }
      }
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kCtas == 2)
          mbar_arrive_cluster(acc_empty0 + buf * 8);
        else
          mbar_arrive(&s->acc_empty[buf]);
        mbar_arrive(&s->scale_empty[slot]);
      }
      if (++buf == T::kAccBuffers)
        buf = 0, buf_phase ^= 1u;
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
    const int row0 = x.m0 + rank * 128 + quarter * 32;
#pragma unroll
    for (int c = 0; c < T::kChunks; ++c)
      if (part0 + 32 * c < x.cols && row0 < p.m)
        store_chunk<kMode>(p, x, stage, lane, row0, part0 + 32 * c, acc[c]);
  }
}

// ---------------------------------------------------------------------------------------------------- kernel

template <int kMode, int kCtas>
__device__ __forceinline__ void block_gemm_body(const Params& p, const CUtensorMap* map_a, const CUtensorMap* map_b) {
  using T = Tile<kCtas>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t a0 = smem_u32(base), b0 = a0 + kStages * kABytes;
  Shared* s = reinterpret_cast<Shared*>(base + kStages * (kABytes + kBBytes));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCtas == 2 ? static_cast<int>(cluster_ctarank()) : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    for (int i = 0; i < T::kAccBuffers; ++i) {
      mbar_init(&s->acc_full[i], 1);
      mbar_init(&s->acc_empty[i], kEpilogueWarps * kCtas);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(&s->scale_full[i], 32);
      mbar_init(&s->scale_empty[i], kEpilogueWarps);
    }
    s->abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(map_a);
    prefetch_tensormap(map_b);
  }
  if (warp == 1) {
    if constexpr (kCtas == 2) {
      tmem_alloc_pair(&s->tmem_base, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&s->tmem_base, kTmemCols);
      tmem_relinquish();
    }
  }
  tcgen05_fence_before_sync();
  grid_dependency_wait();
  scan_experts(p.ends, p.experts, p.rows, kMode == kWeightGrad ? kBlock : T::kN, s->first_row, s->first_tile,
               reinterpret_cast<int*>(base));
  if (kMode != kWeightGrad && p.ends != nullptr) {
    // the rows behind the last expert's, as one more expert without a weight
    if (threadIdx.x == 0) {
      s->first_row[p.experts + 1] = p.rows;
      s->first_tile[p.experts + 1] = s->first_tile[p.experts] + (p.rows - s->first_row[p.experts] + T::kN - 1) / T::kN;
    }
    __syncthreads();
  }
  // the scan's words lie where operands are loaded to
  fence_proxy_async_smem();
  __syncthreads();
  if constexpr (kCtas == 2) {
    cluster_arrive();  // the peer's barriers exist before anything is credited to them
    cluster_wait();
  }
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);

  const int mt = (p.m + T::kM - 1) / T::kM;
  const int units = kMode == kWeightGrad ? p.experts * mt * ((p.n + T::kN - 1) / T::kN)
                                         : s->first_tile[p.experts + (p.ends != nullptr)] * mt;
  const int first = blockIdx.x / kCtas, step = gridDim.x / kCtas;
  if (warp == 0) {
    produce<kMode, kCtas>(p, map_a, map_b, s, a0, b0, rank, first, step, units, lane);
  } else if (warp == 1) {
    if (rank == 0)
      issue_mmas<kMode, kCtas>(p, s, a0, b0, tmem_base, first, step, units);
  } else {
    accumulate<kMode, kCtas>(p, s, tmem_base, rank, first, step, units, warp, lane);
  }
  __syncwarp();

  // on an abort, copies and MMAs in flight get time to land before shared and tensor memory go away
  if (*reinterpret_cast<volatile uint32_t*>(&s->abort_flag) != 0) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if constexpr (kCtas == 2) {
    cluster_arrive();  // neither CTA leaves while the other can still read its shared memory or signal its barriers
    cluster_wait();
  }
  if (warp == 1) {
    tcgen05_fence_after_sync();
    if constexpr (kCtas == 2)
      tmem_dealloc_pair(tmem_base, kTmemCols);
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

struct Launch {
  CUtensorMap a, b;
  Params p;
};

}  // namespace
}  // namespace mxb200

#define MXB200_BLOCK_KERNEL(name, mode)                                                                                     \
  __global__ void __launch_bounds__(mxb200::kThreads, 1) name(const __grid_constant__ mxb200::Launch args) {                \
    mxb200::block_gemm_body<mode, 1>(args.p, &args.a, &args.b);                                                             \
  }
MXB200_BLOCK_KERNEL(mxb200_block_gemm_forward_128x128, mxb200::kForward)
MXB200_BLOCK_KERNEL(mxb200_block_gemm_input_grad_128x128, mxb200::kInputGrad)
MXB200_BLOCK_KERNEL(mxb200_block_gemm_weight_grad_128x128, mxb200::kWeightGrad)

namespace mxb200 {
namespace {

// (z, y, x) bytes, x contiguous; box 128 x box_y x 1, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int box_y) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr)
    return MXB200_ERR_DRIVER;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(x), static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(x), static_cast<cuuint64_t>(x * y)};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_y), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MXB200_OK : MXB200_ERR_DRIVER;
}

int64_t up(int64_t n, int64_t d) {
  return (n + d - 1) / d;
}

using Kernel = void (*)(Launch);

int block_gemm(const mxb200_block_gemm_args& g, cudaStream_t stream) {
  if (g.kind < MXB200_BLOCK_FORWARD || g.kind > MXB200_BLOCK_WEIGHT_GRAD ||
      (g.out_kind != MXB200_OUT_BF16 && (g.out_kind != MXB200_OUT_F32 || g.kind != MXB200_BLOCK_WEIGHT_GRAD)))
    return MXB200_ERR_ARGUMENT;
  constexpr int64_t kMost = int64_t{1} << 30;
  if (g.tokens < 0 || g.tokens > kMost || g.in_features <= 0 || g.in_features > kMost || g.out_features <= 0 ||
      g.out_features > kMost || g.in_features % 16 || g.out_features % 16 || g.experts < 1 || g.experts > kMaxExperts)
    return MXB200_ERR_SHAPE;
  if (g.ends == nullptr && g.experts != 1)
    return MXB200_ERR_NULL;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  const bool wgrad = g.kind == MXB200_BLOCK_WEIGHT_GRAD;
  if (g.tokens == 0) {
    if (!wgrad)
      return MXB200_OK;
    if (g.d == nullptr)
      return MXB200_ERR_NULL;
    const size_t bytes = static_cast<size_t>(g.experts) * g.out_features * g.in_features * (g.out_kind == MXB200_OUT_F32 ? 4 : 2);
    return cudaMemsetAsync(g.d, 0, bytes, stream) == cudaSuccess ? MXB200_OK : MXB200_ERR_LAUNCH;
  }
  if (g.a == nullptr || g.a_scale == nullptr || g.b == nullptr || g.b_scale == nullptr || g.d == nullptr)
    return MXB200_ERR_NULL;
  if (!aligned16(g.a) || !aligned16(g.b) || !aligned16(g.d) ||
      ((reinterpret_cast<uintptr_t>(g.a_scale) | reinterpret_cast<uintptr_t>(g.b_scale) | reinterpret_cast<uintptr_t>(g.ends)) & 3) != 0)
    return MXB200_ERR_ALIGNMENT;
  const int64_t in = g.in_features, out = g.out_features;
  const int64_t capacity = mxb200_block_token_blocks(g.tokens, g.experts) * kBlock;
  Launch l;
  Params& p = l.p;
  p.col_scale = g.b_scale, p.row_scale = g.a_scale;
  p.d = g.d, p.ends = g.ends, p.experts = g.experts, p.rows = static_cast<int>(g.tokens);
  p.out_bf16 = g.out_kind == MXB200_OUT_BF16;
  p.w_scale_expert = up(out, kBlock) * up(in, kBlock);
  p.row_ld = 0, p.blocks = 0, p.n = 0;
  int st;
  switch (g.kind) {
    case MXB200_BLOCK_FORWARD:
      p.m = static_cast<int>(out), p.blocks = static_cast<int>(up(in, kBlock)), p.col_ld = g.tokens;
      p.w_scale_m = static_cast<int>(up(in, kBlock)), p.w_scale_b = 1;
      st = make_map(&l.a, g.a, in, out, g.experts, 128);
      st = st != MXB200_OK ? st : make_map(&l.b, g.b, in, g.tokens, 1, 32);
      break;
    case MXB200_BLOCK_INPUT_GRAD:
      p.m = static_cast<int>(in), p.blocks = static_cast<int>(up(out, kBlock)), p.col_ld = g.tokens;
      p.w_scale_m = 1, p.w_scale_b = static_cast<int>(up(in, kBlock));
      st = make_map(&l.a, g.a, in, out, g.experts, 128);
      st = st != MXB200_OK ? st : make_map(&l.b, g.b, out, g.tokens, 1, 32);
      break;
    default:
      p.m = static_cast<int>(out), p.n = static_cast<int>(in), p.col_ld = in, p.row_ld = out;
      p.w_scale_m = p.w_scale_b = 0;
      st = make_map(&l.a, g.a, out, capacity, 1, 128);
      st = st != MXB200_OK ? st : make_map(&l.b, g.b, in, capacity, 1, 32);
  }
  if (st != MXB200_OK)
    return st;
  const int ctas = 1;
  const int64_t tile = 128 * ctas;
  // token tiles are known on the device only; this many at most
  const int64_t token_tiles = g.ends == nullptr ? up(g.tokens, tile) : (g.tokens + (tile - 1) * std::min<int64_t>(g.experts + 1, g.tokens)) / tile;
  const int64_t units = up(p.m, tile) * (wgrad ? g.experts * up(p.n, tile) : token_tiles);
  if (units > kMost)
    return MXB200_ERR_SHAPE;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, dev.sms / ctas)) * ctas;
  static const Kernel kernels[3] = {mxb200_block_gemm_forward_128x128, mxb200_block_gemm_input_grad_128x128,
                                    mxb200_block_gemm_weight_grad_128x128};
  const Kernel kernel = kernels[g.kind];
  {
    static std::mutex mu;
    static bool configured[3][64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (dev.device >= 64 || !configured[g.kind][dev.device]) {
      if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess) {
        cudaGetLastError();
        return MXB200_ERR_LAUNCH;
      }
      if (dev.device < 64)
        configured[g.kind][dev.device] = true;
    }
  }
  return launch_kernel(kernel, grid, kThreads, kSmemBytes, stream, l);
}

}  // namespace

uint32_t take_block_gemm_watchdog_word() {
  uint32_t w = 0;
  if (cudaMemcpyFromSymbol(&w, g_block_gemm_watchdog_word, sizeof(w)) != cudaSuccess)
    return 0;
  if (w != 0) {
    const uint32_t zero = 0;
    cudaMemcpyToSymbol(g_block_gemm_watchdog_word, &zero, sizeof(zero));
  }
  return w;
}

}  // namespace mxb200

extern "C" int64_t mxb200_block_token_blocks(int64_t tokens, int experts) {
  if (tokens <= 0 || experts <= 0)
    return 0;
  return (tokens + 127 * std::min<int64_t>(experts, tokens)) / 128;
}

extern "C" int mxb200_block_gemm(const mxb200_block_gemm_args* args, void* stream) {
  if (args == nullptr)
    return MXB200_ERR_NULL;
  return mxb200::block_gemm(*args, static_cast<cudaStream_t>(stream));
}
