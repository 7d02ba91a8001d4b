// Matrix products of E4M3 operands with one fp32 scale for 128 values along the contraction, dense and by expert.
//
//   forward       y[t, n]  = sum over blocks b of sx[b, t] sw[n / 128, b]  * sum over k in b of xq[t, k] wq[n, k]
//   input grad    dx[t, k] = sum over blocks b of sg[b, t] sw[b, k / 128]  * sum over n in b of gq[t, n] wq[n, k]
//   weight grad   dw[n, k] = sum over token blocks b of sg[b, n] sx[b, k]  * sum over t in b of gq[t, n] xq[t, k]
//
// Rows (tokens) may be sorted by expert; each expert has its own weight, and token blocks never cross experts. No operand is
// ever transposed in memory: the input gradient contracts over the weight's rows and the weight gradient over tokens, and both
// read their operands as they lie, row-contiguous, through the tensor core's MN-major form.
//
// Forward and input gradient take any fp32 scales, which cannot ride on the tensor core's own block scales (powers of two): the
// tensor core makes the plain fp32 product of one block (K = 128: four MMAs) in tensor memory, and the epilogue warps take it
// from there with one fused multiply-add per value into accumulators in registers, while the next block's MMAs fill another
// tensor memory buffer. Two kernels:
//   * many tokens: a CTA pair, 256 tokens (the tensor core's rows, tensor memory's lanes) x 256 features. A thread has one
//     token and 128 features of one weight block, so one scale, the product of the two, serves all its values: 64 packed
//     multiply-adds per block and nothing else.
//   * few tokens: one CTA, 128 features (rows) x up to 128 tokens (columns). Few tokens cost few columns, not a tile of 128
//     rows, and an expert's last tile is as narrow as its last rows. Scales differ by column: fragments (16x256b) give a thread
//     8 columns of 4 rows each 32, so that a scale read from shared memory serves 4 values.
//
// Where all scales are this library's own, powers of two, the tensor core applies them itself (kind::mxf8f6f4, the four K = 32
// steps of a block under the same scale byte) and sums up in tensor memory: the weight gradient, always, and the other two in
// training passes of many tokens. The tensor core cuts its running sums off. The weight gradient, which may leave in fp32, is
// therefore taken out in segments (kSegment); forward and input gradient are rounded to bf16, up to 2^-8 of a value, beside which
// the 1e-6 that a sum over 16384 loses is nothing, but may differ in a last bit from the kernels for any scales.
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <mutex>

#include "bf16x2_sm100.cuh"
#include "block_common.cuh"
#include "internal.h"
#include "ptx_sm100.cuh"
#include "register_split.h"

namespace mxb200 {

// Non-zero after a bounded wait ran out: 0x20000000 | CTA << 8 | site.
__device__ uint32_t g_block_gemm_watchdog_word;

namespace {

constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr uint32_t kTmemCols = 512;
constexpr int kEpilogueWarps = 8;
// Warps 0 to 2 load operands, issue MMAs and load scales, warp 3 idles; 4 to 11 are the epilogue. The epilogue warps of `many`
// and of the long weight gradient need more registers than an even share (168 of 384 threads): they draw on the first four
// warps'. The sum, 128 x 72 + 256 x 216, is what a block of 168 a thread is launched with; configure() refuses a build in which
// the compiler gave those kernels fewer.
constexpr int kFirstEpilogueWarp = 4;
constexpr int kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps);
constexpr int kFewRegisters = 72, kManyRegisters = 216;
constexpr RegisterSplit kTraded{kFirstEpilogueWarp, kFewRegisters, kEpilogueWarps, kManyRegisters}, kNotTraded{};
static_assert(kTraded.needed() * kThreads <= 65536, "registers of an SM");
constexpr int kScaleSlots = 8;
constexpr uint32_t kABytes = 128 * 128, kBBytes = 128 * 128;
constexpr uint32_t kBBoxBytes = 32 * 128;  // few tokens' rows come 32 at a time, as many as the tile has
constexpr int kPanel = 8;                  // feature tiles per raster panel

enum Mode : int { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };

enum WaitSite : uint32_t {
  kSiteStageEmpty = 1,
  kSiteScaleEmpty = 2,
  kSiteStageFull = 3,
  kSiteAccEmpty = 4,
  kSiteAccFull = 5,
  kSiteScaleFull = 6,
  kSiteOverlap = 7,
  kSitePartialEmpty = 8,
  kSitePartialFull = 9,
};

// Barriers and what the roles of a CTA share. kStages: operand stages of kABytes + kBBytes.
template <int kStages_>
struct Common {
  static constexpr int kStages = kStages_;
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[4], acc_empty[4];
  uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
  uint64_t overlap_free;
  uint32_t tmem_base;
  uint32_t abort_flag;
  int first_row[kMaxExperts + 2];
  int first_tile[kMaxExperts + 2];
};

struct Params {
  const float* token_scale;   // (blocks, token_ld)
  const float* weight_scale;  // (experts, ., .)
  int64_t token_ld;
  int64_t w_scale_expert;
  int w_scale_f, w_scale_b;   // strides of the weight's scale over feature tiles of 128 and over blocks
  int w_scale_rows;           // scales in the tensor core: rows of scale tiles of an expert's weight
  void* d;
  const int32_t* ends;
  int experts;   // 1 where ends is null
  int rows;      // tokens
  int features;  // of the output; weight gradient: its rows
  int n;         // weight gradient: its columns
  int blocks;    // contraction blocks (forward, input grad)
  int out_bf16;
  int splits;    // few tokens: CTAs of a cluster that share a unit's blocks
  const void* input;    // few tokens, quantized on the way: bf16 rows token_ld values apart, of `input_cols` values
  int input_cols;
};

struct Maps {
  CUtensorMap a, b;
  CUtensorMap a_scale, b_scale;  // scales in the tensor core
  CUtensorMap d;                 // many tokens: the output, 32 tokens x 64 features
};

// A warp's wait for a barrier phase, given up after kWaitLimitNs; its lanes agree on the outcome. kCluster: what other CTAs of
// the cluster wrote before they arrived is visible.
template <bool kCluster = false>
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, uint32_t* abort_flag, uint32_t site) {
  const auto done = [&] { return kCluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
  bool ok = true;
  if (!done()) {
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (!done()) {
      if ((++spins & 63u) == 0) {
        if (*reinterpret_cast<volatile uint32_t*>(abort_flag) != 0) {
          ok = false;
          break;
        }
        if (global_timer_ns() - t0 > kWaitLimitNs) {
          *reinterpret_cast<volatile uint32_t*>(abort_flag) = 1;
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

struct SetUp {
  uint32_t full_arrivals, empty_arrivals;  // of an operand stage
  uint32_t acc_empty_arrivals;
  int acc_buffers;
  uint32_t scale_arrivals;
  int tile_rows;       // of the tiles that experts' rows are cut into
  bool rest_is_a_tile; // the rows behind the last expert's, as one more expert without a weight
};

// Barriers, tensor memory and the experts' rows; the operand stages at `base` hold the scan's words meanwhile. All threads.
// kCtas: that share tensor memory operations. cluster: the CTAs of a cluster signal one another.
// first_block: where given, the blocks of 128 tokens before each expert's.
template <int kCtas, typename S>
__device__ __forceinline__ uint32_t set_up(const Params& p, const CUtensorMap* map_a, const CUtensorMap* map_b, S* s, unsigned char* base,
                                           int warp, const SetUp& set, bool cluster, int* first_block = nullptr) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&s->full[i], set.full_arrivals);
      mbar_init(&s->empty[i], set.empty_arrivals);
    }
    for (int i = 0; i < set.acc_buffers; ++i) {
      mbar_init(&s->acc_full[i], 1);
      mbar_init(&s->acc_empty[i], set.acc_empty_arrivals);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(&s->scale_full[i], set.scale_arrivals);
      mbar_init(&s->scale_empty[i], set.acc_empty_arrivals / kCtas);
    }
    mbar_init(&s->overlap_free, 4 * kCtas);
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
  scan_experts(p.ends, p.experts, p.rows, set.tile_rows, s->first_row, s->first_tile, reinterpret_cast<int*>(base));
  if (first_block != nullptr)
    scan_experts(p.ends, p.experts, p.rows, kBlock, s->first_row, first_block, reinterpret_cast<int*>(base));
  if (set.rest_is_a_tile && p.ends != nullptr && threadIdx.x == 0) {
    s->first_row[p.experts + 1] = p.rows;
    s->first_tile[p.experts + 1] = s->first_tile[p.experts] + (p.rows - s->first_row[p.experts] + set.tile_rows - 1) / set.tile_rows;
  }
  fence_proxy_async_smem();  // operands are loaded over the scan's words
  __syncthreads();
  if (cluster) {
    cluster_arrive();  // the others' barriers exist before anything is credited to them
    cluster_wait();
  }
  tcgen05_fence_after_sync();
  return *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);
}

template <int kCtas, typename S>
__device__ __forceinline__ void tear_down(S* s, uint32_t tmem_base, int warp, bool cluster) {
  __syncwarp();
  // on an abort, copies and MMAs in flight get time to land before shared and tensor memory go away
  if (*reinterpret_cast<volatile uint32_t*>(&s->abort_flag) != 0) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (cluster) {
    cluster_arrive();  // no CTA leaves while another can still read its shared memory or signal its barriers
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

// Where a walk over the units of forward or input gradient is: token tiles (kTokens rows) x feature tiles (kFeatures). Within an
// expert all of a panel's feature tiles for one token tile, then for the next, so that what runs at one time shares operands in
// L2.
struct Unit {
  int expert;
  int row0, rows;  // tokens
  int f0;          // first feature
  int blocks;      // 0: rows of no expert, zeros
};

template <int kTokens, int kFeatures, typename S>
__device__ __forceinline__ Unit unit_at(const Params& p, const S* s, int u) {
  const int ft = (p.features + kFeatures - 1) / kFeatures;
  const int t = u / ft;  // token tiles before this one, over all experts
  Unit x;
  x.expert = expert_of_tile(s->first_tile, p.experts + (p.ends != nullptr), t);
  x.blocks = x.expert < p.experts ? p.blocks : 0;
  const int tiles = s->first_tile[x.expert + 1] - s->first_tile[x.expert];
  int v = u - s->first_tile[x.expert] * ft;
  const int panel = v / (kPanel * tiles);
  v -= panel * kPanel * tiles;
  const int width = min(kPanel, ft - panel * kPanel);
  const int n = v / width;
  x.f0 = (panel * kPanel + v - n * width) * kFeatures;
  x.row0 = s->first_row[x.expert] + n * kTokens;
  x.rows = min(kTokens, s->first_row[x.expert + 1] - x.row0);
  return x;
}

template <typename S>
__device__ __forceinline__ int units_of(const Params& p, const S* s, int features_per_tile) {
  return s->first_tile[p.experts + (p.ends != nullptr)] * ((p.features + features_per_tile - 1) / features_per_tile);
}

// Output of a thread's row, 128 bytes at a time, through shared memory: a row per lane goes in, four whole rows (128-byte lines)
// per store instruction come out. Written straight from the rows' owners, 16 bytes in each of 32 rows per instruction, the
// stores took longer than the products of up to 20 blocks.
constexpr uint32_t kLineRowBytes = 144;  // 128 and 16 that put 8 rows' 16-byte pieces into different banks
struct __align__(16) LineStage {
  unsigned char bytes[32 * kLineRowBytes];
};

// piece(q): this lane's 16 bytes q of 8. rows, bytes: what exists of the 32 rows and of the line.
template <typename Piece>
__device__ __forceinline__ void store_lines(LineStage* stage, int lane, unsigned char* d, int64_t row_bytes, int rows, int bytes, Piece piece) {
  __syncwarp();  // the previous lines have been read out
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<uint4*>(stage->bytes + lane * kLineRowBytes + q * 16) = piece(q);
  __syncwarp();
  const int at = (lane & 7) * 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    const uint4 w = *reinterpret_cast<const uint4*>(stage->bytes + r * kLineRowBytes + at);
    if (r < rows && at < bytes)
      *reinterpret_cast<uint4*>(d + r * row_bytes + at) = w;
  }
}

// ==================================================================================================== few tokens
//
// Rows of the tensor core's tile are features (the weight is operand A), columns tokens. Where the output has fewer tiles than
// the machine SMs, a cluster of up to 8 CTAs shares one: each contracts a share of the blocks, leaves its fp32 tile in shared
// memory, and adds up every n-th token of all of them, always in the cluster's order.
//
// kQuantize: the input comes in bf16 and is quantized on its way into shared memory, by the four warps that would accumulate
// the second half of the columns. That spares a launch, about 2 us on the device and as much on the host; every CTA's repeating
// it costs 0.6 us for one token and 1.9 for 16 (1536 -> 1536), 2.2 for 32 rows over 64 experts and 5.9 for 64.
//
// Blocks go through the barriers in pairs, and of a pair 32 tokens come from tensor memory with one wait: what a warp spends on a
// block besides its bytes (two barriers, the way to tensor memory and back) is as long as the block's way into shared memory. 64
// rows over 64 experts (1536 -> 2048) take 20.4 us by pairs, 23.1 one by one and 20.8 by fours; one token of 6144 -> 24576 29.7,
// 36.3 and 30.9; 128 tokens of 1536 -> 6144 in large tiles 7.9 and 8.9.

namespace few {

constexpr int kTileF = 128;
constexpr uint32_t kStageRowBytes = 80;  // 32 bf16 and 16 bytes that put 8 rows' 16-byte pieces into different banks
constexpr int kPartialRow = 132;         // floats of a token's 128 features: fragments' rows fall into different banks

// kTile: tokens of a unit, 128 or 32; fewer are done with their columns sooner and leave room for more stages of the weight.
template <int kTile, bool kQuantize_>
struct Config {
  static constexpr bool kQuantize = kQuantize_;
  static constexpr int kTileT = kTile;
  static constexpr int kWarps = kTile == 32 ? 4 : 8;  // that accumulate
  static constexpr int kParts = kWarps / 4;           // columns are shared by the warps of a tensor memory quarter
  static constexpr int kPartT = kTile / kParts;
  static constexpr int kChunks = kPartT / 32;
  static constexpr int kTurn = 2;                     // blocks that the barriers pass on at a time
  static constexpr int kAccBuffers = kTmemCols / (kTurn * kTile) < 4 ? kTmemCols / (kTurn * kTile) : 4;

  struct __align__(16) ScaleSlot {  // tokens' scales are read in pairs
    float token[kTileT];
    float weight;
  };

  struct Shared : Common<(kTile == 32 ? 8 : 4) / kTurn> {
    uint64_t partial_full, partial_empty;
    ScaleSlot scales[kScaleSlots][kTurn];
    union {
      __align__(16) unsigned char out[kWarps][32 * kStageRowBytes];
      __align__(16) float partial[kPartT][kPartialRow];
    };
  };
  static constexpr uint32_t kBlockBBytes = kTileT * kBlock, kStageABytes = kTurn * kABytes, kStageBBytes = kTurn * kBlockBBytes;
  static constexpr size_t kSmemBytes = 1024 + Shared::kStages * static_cast<size_t>(kStageABytes + kStageBBytes) + sizeof(Shared);
  static_assert(kSmemBytes <= 232448, "shared memory of one CTA");
  static_assert(Shared::kStages * kStageABytes >= kMaxExperts * 4, "the operand stages hold the scan's copy of ends");
};

// Which CTA of which cluster this is, and its share of a unit's blocks.
struct Place {
  int rank, splits, cluster, clusters;
  __device__ Place(int n) : rank(static_cast<int>(cluster_ctarank())), splits(n), cluster(blockIdx.x / n), clusters(gridDim.x / n) {}
  __device__ int begin(int blocks) const { return blocks * rank / splits; }
  __device__ int end(int blocks) const { return blocks * (rank + 1) / splits; }
};

template <int kMode, typename C>
__device__ __forceinline__ void load_operands(const Params& p, const CUtensorMap* map_w, const CUtensorMap* map_t, typename C::Shared* s,
                                              uint32_t a0, uint32_t b0, const Place& at, int units) {
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t empty0 = smem_u32(&s->empty[0]), full0 = smem_u32(&s->full[0]);
  uint32_t stage = 0, phase = 0;
  for (int u = at.cluster; u < units; u += at.clusters) {
    const Unit x = unit_at<C::kTileT, kTileF>(p, s, u);
    const int boxes = C::kQuantize ? 0 : (x.rows + 31) / 32;
    const int end = at.end(x.blocks);
    for (int b = at.begin(x.blocks); b < end; b += C::kTurn) {
      const int turn = min(C::kTurn, end - b);
      if (!wait_bounded(empty0 + stage * 8, phase ^ 1u, &s->abort_flag, kSiteStageEmpty))
        return;
      const uint32_t full = full0 + stage * 8;
      mbar_arrive_expect_tx(el, full, turn * (kABytes + boxes * kBBoxBytes));
      for (int n = 0; n < turn; ++n) {
        const int k = (b + n) * kBlock;
        tma_load_3d(el, a0 + stage * C::kStageABytes + n * kABytes, map_w, full, kMode == kForward ? k : x.f0, kMode == kForward ? x.f0 : k, x.expert);
        for (int i = 0; i < boxes; ++i)
          tma_load_3d(el, b0 + stage * C::kStageBBytes + n * C::kBlockBBytes + i * kBBoxBytes, map_t, full, k, x.row0 + 32 * i, 0);
      }
      if (++stage == C::Shared::kStages)
        stage = 0, phase ^= 1u;
    }
  }
}

__device__ __forceinline__ const float* weight_scale(const Params& p, const Unit& x, int b) {
  return p.weight_scale + x.expert * p.w_scale_expert + (x.f0 >> 7) * static_cast<int64_t>(p.w_scale_f) + b * static_cast<int64_t>(p.w_scale_b);
}

// A block's scales by 4-byte copies: an expert's tokens start at any row.
template <typename C>
__device__ __forceinline__ void load_scales(const Params& p, typename C::Shared* s, const Place& at, int units, int lane) {
  const uint32_t scale_full0 = smem_u32(&s->scale_full[0]), scale_empty0 = smem_u32(&s->scale_empty[0]);
  uint32_t slot = 0, slot_phase = 0;
  for (int u = at.cluster; u < units; u += at.clusters) {
    const Unit x = unit_at<C::kTileT, kTileF>(p, s, u);
    const int end = at.end(x.blocks);
    for (int b = at.begin(x.blocks); b < end; b += C::kTurn) {
      if (!wait_bounded(scale_empty0 + slot * 8, slot_phase ^ 1u, &s->abort_flag, kSiteScaleEmpty))
        return;
      for (int n = 0; n < min(C::kTurn, end - b); ++n) {
        auto& to = s->scales[slot][n];
        const float* token = p.token_scale + (b + n) * p.token_ld + x.row0;
        for (int i = lane; i < x.rows; i += 32)
          cp_async_4(smem_u32(&to.token[i]), token + i);
        if (lane == 0)
          cp_async_4(smem_u32(&to.weight), weight_scale(p, x, b + n));
      }
      cp_async_arrive(scale_full0 + slot * 8);
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
  }
}

// The input's blocks from bf16 into shared memory as a TMA load would leave them (128-byte swizzle), and their scales. Each of
// the four warps has every fourth block to itself, 16 lanes per token, so that the way of one block (maxima, scale, proxy fence)
// is covered by the others'; with all four at one block a block took 0.47 us instead of 0.33. The values are
// block_quantize_sm100.cu's.
template <typename C>
__device__ __forceinline__ void quantize(const Params& p, typename C::Shared* s, unsigned char* b_stages, const Place& at, int units, int warp,
                                         int lane) {
  static_assert(C::kTurn == 2, "pairs of blocks");
  constexpr int kPasses = C::kTileT / 2;
  const uint32_t full0 = smem_u32(&s->full[0]), empty0 = smem_u32(&s->empty[0]);
  const uint32_t scale_full0 = smem_u32(&s->scale_full[0]), scale_empty0 = smem_u32(&s->scale_empty[0]);
  const int lane16 = lane & 15, token0 = lane >> 4;
  const int in = p.input_cols;
  const uint16_t* input = static_cast<const uint16_t*>(p.input);
  uint4 ahead[kPasses];
  float weight_ahead = 0.f;
  const auto fetch = [&](const Unit& x, int b) {
    const int col = b * kBlock + 8 * lane16;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = token0 + 2 * i;
      ahead[i] = t < x.rows && col < in ? *reinterpret_cast<const uint4*>(input + (x.row0 + t) * p.token_ld + col) : make_uint4(0, 0, 0, 0);
    }
    weight_ahead = *weight_scale(p, x, b);
  };
  uint32_t before = 0;  // blocks of the units before this one, in whole pairs
  for (int u = at.cluster; u < units; u += at.clusters) {
    const Unit x = unit_at<C::kTileT, kTileF>(p, s, u);
    const int begin = at.begin(x.blocks), end = at.end(x.blocks);
    int b = begin + static_cast<int>(((warp & 3) - before) & 3u);
    uint32_t n = before + (b - begin);
    if (b < end)
      fetch(x, b);
    for (; b < end; b += 4, n += 4) {
      const uint32_t pair = n >> 1, of_pair = n & 1, stage = pair % C::Shared::kStages, slot = pair % kScaleSlots;
      if (!wait_bounded(empty0 + stage * 8, (pair / C::Shared::kStages & 1u) ^ 1u, &s->abort_flag, kSiteStageEmpty) ||
          !wait_bounded(scale_empty0 + slot * 8, (pair / kScaleSlots & 1u) ^ 1u, &s->abort_flag, kSiteScaleEmpty))
        return;
      unsigned char* to = b_stages + stage * C::kStageBBytes + of_pair * C::kBlockBBytes;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (2 * i >= x.rows)
          break;
        const int t = token0 + 2 * i;
        const uint32_t w[4] = {ahead[i].x, ahead[i].y, ahead[i].z, ahead[i].w};
        uint32_t m = max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(max_abs_skip_nan_bf16x2(0u, w[0]), w[1]), w[2]), w[3]);
        m &= 0x7fff7fffu;
        m = max(m & 0xffffu, m >> 16);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
          m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        const int e = block_exponent(m << 16);
        const uint16_t by = static_cast<uint16_t>(mx_multiplier_bits(e) >> 16);
        *reinterpret_cast<uint2*>(to + t * kBlock + (((lane16 >> 1) ^ (t & 7)) << 4) + (lane16 & 1) * 8) =
              make_uint2(e4m3x4_scaled_fma(w[0], w[1], by, by), e4m3x4_scaled_fma(w[2], w[3], by, by));
        if (lane16 == 0)
          s->scales[slot][of_pair].token[t] = __uint_as_float(static_cast<uint32_t>(e) << 23);
      }
      if (lane == 0)
        s->scales[slot][of_pair].weight = weight_ahead;
      if (b + 4 < end)
        fetch(x, b + 4);
      fence_proxy_async_smem();
      __syncwarp();
      // a last block without a second one arrives for both
      if (lane < (of_pair == 0 && b + 1 == end ? 2 : 1)) {
        mbar_arrive_addr(full0 + stage * 8);
        mbar_arrive_addr(scale_full0 + slot * 8);
      }
    }
    before += static_cast<uint32_t>((end - begin + 1) & ~1);
  }
}

template <int kMode, typename C>
__device__ __forceinline__ void issue_mmas(const Params& p, typename C::Shared* s, uint32_t a0, uint32_t b0, uint32_t tmem_base, const Place& at,
                                           int units) {
  constexpr bool kAMn = kMode == kInputGrad;
  // 128-byte swizzle, groups of 8 rows of 128 bytes 1024 apart. K-major: K = 32 is 32 bytes within a row; MN-major: 32 rows.
  constexpr uint32_t kAStep = kAMn ? 4096 >> 4 : 32 >> 4, kBStep = 32 >> 4;
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t full0 = smem_u32(&s->full[0]);
  const uint64_t a_desc0 = make_smem_desc(a0, 1024, 1024, 2), b_desc0 = make_smem_desc(b0, 1024, 1024, 2);
  uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
  for (int u = at.cluster; u < units; u += at.clusters) {
    const Unit x = unit_at<C::kTileT, kTileF>(p, s, u);
    const uint32_t idesc = make_idesc_f8(kTileF, (x.rows + 15) / 16 * 16, kAMn, false);
    const int end = at.end(x.blocks);
    for (int b = at.begin(x.blocks); b < end; b += C::kTurn) {
      if (!wait_bounded(smem_u32(&s->acc_empty[buf]), buf_phase ^ 1u, &s->abort_flag, kSiteAccEmpty) ||
          !wait_bounded(full0 + stage * 8, phase, &s->abort_flag, kSiteStageFull))
        return;
      tcgen05_fence_after_sync();
      const uint64_t a = a_desc0 + stage * (C::kStageABytes >> 4), bd = b_desc0 + stage * (C::kStageBBytes >> 4);
      const uint32_t d = tmem_base + buf * (C::kTurn * C::kTileT);
#pragma unroll
      for (int n = 0; n < C::kTurn; ++n) {
        if (b + n >= end)
          break;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          tcgen05_mma_f8(el, d + n * C::kTileT, a + n * (kABytes >> 4) + k * kAStep, bd + n * (C::kBlockBBytes >> 4) + k * kBStep, idesc, k > 0);
      }
      tcgen05_commit(el, &s->empty[stage]);
      tcgen05_commit(el, &s->acc_full[buf]);
      if (++stage == C::Shared::kStages)
        stage = 0, phase ^= 1u;
      if (++buf == C::kAccBuffers)
        buf = 0, buf_phase ^= 1u;
    }
  }
}

// 32 tokens of this warp's 32 features to the output. v[j][i]: tokens 8 j + 2 (lane % 4), + 1, feature 8 i + lane / 4.
__device__ __forceinline__ void store_chunk(const Params& p, const Unit& x, unsigned char* stage, int lane, int feature0, int t0,
                                            const uint64_t (&v)[4][4]) {
  const uint32_t st = smem_u32(stage);
  __syncwarp();  // the previous chunk has been read out
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(v[j][i]);
      h[i] = pack_bf16x2_rn(f.x, f.y);
    }
    // a row of the stage: 32 features of one token
    stmatrix_x4_trans(st + (8 * j + (lane & 7)) * kStageRowBytes + (lane >> 3) * 16, h[0], h[1], h[2], h[3]);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2), piece = lane & 3;
    const uint4 w = *reinterpret_cast<const uint4*>(stage + r * kStageRowBytes + piece * 16);
    if (t0 + r < x.rows && feature0 + piece * 8 < p.features)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.d) + static_cast<int64_t>(x.row0 + t0 + r) * p.features + feature0 + piece * 8) = w;
  }
}

template <typename C>
__device__ __forceinline__ void accumulate(const Params& p, typename C::Shared* s, uint32_t tmem_base, const Place& at, int units, int warp,
                                           int lane) {
  const int quarter = warp & 3, part = (warp - kFirstEpilogueWarp) >> 2, part0 = part * C::kPartT;  // tensor memory lanes 32 (warp % 4) on
  const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
  unsigned char* stage = s->out[warp - kFirstEpilogueWarp];
  uint32_t buf = 0, buf_phase = 0, slot = 0, slot_phase = 0, partial_phase = 0;
  for (int u = at.cluster; u < units; u += at.clusters) {
    const Unit x = unit_at<C::kTileT, kTileF>(p, s, u);
    uint64_t acc[C::kChunks][4][4];
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[c][j][i] = 0;
    const int end = at.end(x.blocks);
    for (int b = at.begin(x.blocks); b < end; b += C::kTurn) {
      if (!wait_bounded(smem_u32(&s->scale_full[slot]), slot_phase, &s->abort_flag, kSiteScaleFull) ||
          !wait_bounded(smem_u32(&s->acc_full[buf]), buf_phase, &s->abort_flag, kSiteAccFull))
        return;
      tcgen05_fence_after_sync();
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        if (part0 + 32 * c >= x.rows)
          break;
        // a last block without a second one: that one's are read and not used
        uint32_t lo[C::kTurn][16], hi[C::kTurn][16];
        uint64_t scale[C::kTurn][4];
#pragma unroll
        for (int n = 0; n < C::kTurn; ++n) {
          const uint32_t t = tmem_base + lane_base + (buf * C::kTurn + n) * C::kTileT + part0 + 32 * c;
          tmem_ld_16x256b_x4(t, lo[n]);
          tmem_ld_16x256b_x4(t + (16u << 16), hi[n]);
        }
#pragma unroll
        for (int n = 0; n < C::kTurn; ++n) {
          const auto& sc = s->scales[slot][n];
          const uint64_t weight = pair_f32(sc.weight, sc.weight);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = *reinterpret_cast<const float2*>(&sc.token[part0 + 32 * c + 8 * j + 2 * (lane & 3)]);
            scale[n][j] = mul_f32x2(pair_f32(f.x, f.y), weight);
          }
        }
        tmem_ld_wait();
#pragma unroll
        for (int n = 0; n < C::kTurn; ++n) {
          if (b + n >= end)
            break;
#pragma unroll
          for (int k = 0; k < 16; ++k)
            asm volatile("" : "+r"(lo[n][k]), "+r"(hi[n][k]));
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t v = i < 2 ? pair_u32(lo[n][4 * j + 2 * i], lo[n][4 * j + 2 * i + 1])
                                       : pair_u32(hi[n][4 * j + 2 * i - 4], hi[n][4 * j + 2 * i - 3]);
              acc[c][j][i] = fma_f32x2(v, scale[n][j], acc[c][j][i]);
            }
        }
      }
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s->acc_empty[buf]);
        mbar_arrive(&s->scale_empty[slot]);
      }
      if (++buf == C::kAccBuffers)
        buf = 0, buf_phase ^= 1u;
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
    if (at.splits == 1) {
      const int feature0 = x.f0 + quarter * 32;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        if (part0 + 32 * c < x.rows && feature0 < p.features)
          store_chunk(p, x, stage, lane, feature0, part0 + 32 * c, acc[c]);
      continue;
    }
    for (int h = 0; h < C::kParts; ++h) {
      const int first = h * C::kPartT, rows = min(C::kPartT, x.rows - first);
      if (rows <= 0)
        break;
      // this CTA's share of these columns into its shared memory, once the cluster has read the last ones ...
      if (!wait_bounded<true>(smem_u32(&s->partial_empty), partial_phase ^ 1u, &s->abort_flag, kSitePartialEmpty))
        return;
      if (h == part) {
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          if (32 * c >= rows)
            break;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = both(acc[c][j][i]);
              float* to = &s->partial[32 * c + 8 * j + 2 * (lane & 3)][quarter * 32 + 8 * i + (lane >> 2)];
              to[0] = f.x, to[kPartialRow] = f.y;
            }
        }
      }
      __syncwarp();
      if (lane < at.splits)
        mbar_arrive_release_cluster(map_to_cta(smem_u32(&s->partial_full), lane));
      // ... and the sum of every splits-th token from all of them
      if (!wait_bounded<true>(smem_u32(&s->partial_full), partial_phase, &s->abort_flag, kSitePartialFull))
        return;
      for (int t = at.rank + at.splits * (warp - kFirstEpilogueWarp); t < rows; t += at.splits * C::kWarps) {
        const uint32_t from = smem_u32(&s->partial[t][4 * lane]);
        float4 sum = load_cluster(map_to_cta(from, 0));
        for (int r = 1; r < at.splits; ++r) {
          const float4 f = load_cluster(map_to_cta(from, r));
          sum.x += f.x, sum.y += f.y, sum.z += f.z, sum.w += f.w;
        }
        if (x.f0 + 4 * lane < p.features)
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.d) + static_cast<int64_t>(x.row0 + first + t) * p.features + x.f0 + 4 * lane) =
                make_uint2(pack_bf16x2_rn(sum.x, sum.y), pack_bf16x2_rn(sum.z, sum.w));
      }
      __syncwarp();
      if (lane < at.splits)
        mbar_arrive_release_cluster(map_to_cta(smem_u32(&s->partial_empty), lane));
      partial_phase ^= 1u;
    }
  }
}

template <int kMode, typename C>
__device__ __forceinline__ void body(const Params& p, const CUtensorMap* map_w, const CUtensorMap* map_t) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* b_stages = base + C::Shared::kStages * C::kStageABytes;
  const uint32_t a0 = smem_u32(base), b0 = smem_u32(b_stages);
  auto* s = reinterpret_cast<typename C::Shared*>(b_stages + C::Shared::kStages * C::kStageBBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Place at(p.splits);
  if (threadIdx.x == 0) {
    mbar_init(&s->partial_full, C::kWarps * p.splits);
    mbar_init(&s->partial_empty, C::kWarps * p.splits);
  }
  SetUp set{1, 1, C::kWarps, C::kAccBuffers, C::kQuantize ? 2u : 32u, C::kTileT, true};
  if (C::kQuantize)
    set.full_arrivals = 3;  // the weights' load and the blocks' warps
  const uint32_t tmem_base = set_up<1>(p, map_w, map_t, s, base, warp, set, p.splits > 1);
  const int units = units_of(p, s, kTileF);
  if (warp == 0)
    load_operands<kMode, C>(p, map_w, map_t, s, a0, b0, at, units);
  else if (warp == 1)
    issue_mmas<kMode, C>(p, s, a0, b0, tmem_base, at, units);
  else if (warp >= kFirstEpilogueWarp && warp < kFirstEpilogueWarp + C::kWarps)
    accumulate<C>(p, s, tmem_base, at, units, warp, lane);
  else if constexpr (C::kQuantize) {
    if (warp >= kFirstEpilogueWarp)
      quantize<C>(p, s, b_stages, at, units, warp, lane);
  } else if (warp == 2) {
    load_scales<C>(p, s, at, units, lane);
  }
  tear_down<1>(s, tmem_base, warp, p.splits > 1);
}

using Tile128 = Config<128, false>;
using Tile32 = Config<32, false>;
using Quantizing = Config<32, true>;

}  // namespace few

// ==================================================================================================== many tokens
//
// Rows of the tensor core's tile are tokens (operand A, 128 per CTA), columns features: each CTA brings its tokens and half of
// the features' rows of the weight.

namespace many {

constexpr int kTileT = 256, kTileF = 256;
constexpr int kAccBuffers = kTmemCols / kTileF;
constexpr int kChunks = 4;  // of 32 features: an epilogue warp has 32 tokens and the 128 features of one weight block

struct __align__(16) ScaleSlot {
  float token[128];
  float weight[2];
};

// A warp's output on its way: 32 tokens x 64 features in the 128-byte swizzle of a TMA store.
constexpr uint32_t kOutStageBytes = 32 * 128;

struct Shared : Common<5> {
  ScaleSlot scales[kScaleSlots];
};

constexpr size_t kOperandBytes = Shared::kStages * static_cast<size_t>(kABytes + kBBytes);
constexpr size_t kSmemBytes = 1024 + kOperandBytes + kEpilogueWarps * kOutStageBytes + sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");

template <int kMode>
__device__ __forceinline__ void load_operands(const Params& p, const CUtensorMap* map_t, const CUtensorMap* map_w, Shared* s, uint32_t a0,
                                              uint32_t b0, int rank, int first, int step, int units) {
  const uint32_t el = elect_one() ? 1u : 0u, el_leader = rank == 0 ? el : 0u;
  const uint32_t empty0 = smem_u32(&s->empty[0]), full0 = smem_u32(&s->full[0]);
  const uint32_t full_leader0 = map_to_cta(full0, 0);
  uint32_t stage = 0, phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kTileT, kTileF>(p, s, u);
    const int row = x.row0 + rank * 128, feature = x.f0 + rank * 128;
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(empty0 + stage * 8, phase ^ 1u, &s->abort_flag, kSiteStageEmpty))
        return;
      mbar_arrive_expect_tx(el_leader, full0 + stage * 8, 2 * (kABytes + kBBytes));
      const uint32_t full = full_leader0 + stage * 8;
      const int k = b * kBlock;
      tma_load_3d_pair(el, a0 + stage * kABytes, map_t, full, k, row, 0);
      tma_load_3d_pair(el, b0 + stage * kBBytes, map_w, full, kMode == kForward ? k : feature, kMode == kForward ? feature : k, x.expert);
      if (++stage == Shared::kStages)
        stage = 0, phase ^= 1u;
    }
  }
}

__device__ __forceinline__ void load_scales(const Params& p, Shared* s, int rank, int first, int step, int units, int lane) {
  const uint32_t scale_full0 = smem_u32(&s->scale_full[0]), scale_empty0 = smem_u32(&s->scale_empty[0]);
  uint32_t slot = 0, slot_phase = 0;
  const int weight_tiles = (p.features + kBlock - 1) / kBlock;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kTileT, kTileF>(p, s, u);
    const int row = rank * 128;
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(scale_empty0 + slot * 8, slot_phase ^ 1u, &s->abort_flag, kSiteScaleEmpty))
        return;
      const float* token = p.token_scale + b * p.token_ld + x.row0 + row;
#pragma unroll
      for (int i = lane; i < 128; i += 32)
        if (row + i < x.rows)
          cp_async_4(smem_u32(&s->scales[slot].token[i]), token + i);
      if (lane < 2 && (x.f0 >> 7) + lane < weight_tiles)
        cp_async_4(smem_u32(&s->scales[slot].weight[lane]),
                   p.weight_scale + x.expert * p.w_scale_expert + ((x.f0 >> 7) + lane) * static_cast<int64_t>(p.w_scale_f) +
                         b * static_cast<int64_t>(p.w_scale_b));
      cp_async_arrive(scale_full0 + slot * 8);
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
  }
}

template <int kMode>
__device__ __forceinline__ void issue_mmas(const Params& p, Shared* s, uint32_t a0, uint32_t b0, uint32_t tmem_base, int first, int step,
                                           int units) {
  constexpr bool kBMn = kMode == kInputGrad;
  constexpr uint32_t kAStep = 32 >> 4, kBStep = kBMn ? 4096 >> 4 : 32 >> 4;
  constexpr uint32_t idesc = make_idesc_f8(kTileT, kTileF, false, kBMn);
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t full0 = smem_u32(&s->full[0]), empty0 = smem_u32(&s->empty[0]);
  const uint64_t a_desc0 = make_smem_desc(a0, 1024, 1024, 2), b_desc0 = make_smem_desc(b0, 1024, 1024, 2);
  uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
  for (int u = first; u < units; u += step) {
    const int blocks = unit_at<kTileT, kTileF>(p, s, u).blocks;
    for (int b = 0; b < blocks; ++b) {
      if (!wait_bounded(smem_u32(&s->acc_empty[buf]), buf_phase ^ 1u, &s->abort_flag, kSiteAccEmpty) ||
          !wait_bounded(full0 + stage * 8, phase, &s->abort_flag, kSiteStageFull))
        return;
      tcgen05_fence_after_sync();
      const uint64_t a = a_desc0 + stage * (kABytes >> 4), bd = b_desc0 + stage * (kBBytes >> 4);
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        tcgen05_mma_f8_pair(el, tmem_base + buf * kTileF, a + k * kAStep, bd + k * kBStep, idesc, k > 0);
      tcgen05_commit_pair(el, empty0 + stage * 8, 3);
      tcgen05_commit_pair(el, &s->acc_full[buf], 3);
      if (++stage == Shared::kStages)
        stage = 0, phase ^= 1u;
      if (++buf == kAccBuffers)
        buf = 0, buf_phase ^= 1u;
    }
  }
}

__device__ __forceinline__ void accumulate(const Params& p, const CUtensorMap* map_d, Shared* s, unsigned char* out, uint32_t tmem_base, int rank,
                                           int first, int step, int units, int warp, int lane) {
  const int quarter = warp & 3, part = (warp - kFirstEpilogueWarp) >> 2;
  const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + part * 128;
  const uint32_t acc_empty0 = map_to_cta(smem_u32(&s->acc_empty[0]), 0);
  uint32_t buf = 0, buf_phase = 0, slot = 0, slot_phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kTileT, kTileF>(p, s, u);
    uint64_t acc[kChunks][16];
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        acc[c][j] = 0;
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(smem_u32(&s->scale_full[slot]), slot_phase, &s->abort_flag, kSiteScaleFull))
        return;
      const float f = s->scales[slot].token[quarter * 32 + lane] * s->scales[slot].weight[part];
      const uint64_t scale = pair_f32(f, f);
      if (!wait_bounded(smem_u32(&s->acc_full[buf]), buf_phase, &s->abort_flag, kSiteAccFull))
        return;
      tcgen05_fence_after_sync();
      const uint32_t t = t0 + buf * kTileF;
      uint32_t v[2][32];
      tmem_ld_32x32b_x32(t, v[0]);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        tmem_ld_wait(v[c & 1]);
        if (c + 1 < kChunks)
          tmem_ld_32x32b_x32(t + 32 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          acc[c][j] = fma_f32x2(pair_u32(v[c & 1][2 * j], v[c & 1][2 * j + 1]), scale, acc[c][j]);
      }
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_cluster(acc_empty0 + buf * 8);
        mbar_arrive(&s->scale_empty[slot]);
      }
      if (++buf == kAccBuffers)
        buf = 0, buf_phase ^= 1u;
      if (++slot == kScaleSlots)
        slot = 0, slot_phase ^= 1u;
    }
    const int row = rank * 128 + quarter * 32, feature = x.f0 + part * 128;
    unsigned char* stage = out + (warp - kFirstEpilogueWarp) * kOutStageBytes;
#pragma unroll
    for (int c = 0; c < kChunks; c += 2) {
      if (lane == 0)
        tma_store_wait_read<0>();  // the stage has been read out
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 o = both(acc[c + (q >> 2)][4 * (q & 3) + j]);
          h[j] = pack_bf16x2_rn(o.x, o.y);
        }
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      const int left = p.features - feature - 32 * c;  // columns that exist
      if (row + 32 <= x.rows) {
        // all tokens there: handed to the copy engine, and the next unit's blocks are taken up meanwhile
        if (lane == 0 && left > 0) {
          tma_store_2d(map_d, stage, feature + 32 * c, x.row0 + row);
          tma_store_commit();
        }
      } else {
        // the tile ends within the warp's tokens, behind which lie another expert's
#pragma unroll 1
        for (int r = lane >> 3; r < x.rows - row; r += 4) {
          const int q = lane & 7;
          const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 128 + ((q ^ (r & 7)) << 4));
          if (8 * q < left)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.d) + static_cast<int64_t>(x.row0 + row + r) * p.features + feature + 32 * c + 8 * q) = w;
        }
      }
    }
  }
  if (lane == 0)
    tma_store_wait_all<0>();
}

template <int kMode>
__device__ __forceinline__ void body(const Params& p, const CUtensorMap* map_t, const CUtensorMap* map_w, const CUtensorMap* map_d) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t a0 = smem_u32(base), b0 = a0 + Shared::kStages * kABytes;
  unsigned char* out = base + kOperandBytes;
  Shared* s = reinterpret_cast<Shared*>(out + kEpilogueWarps * kOutStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const SetUp set{1, 1, 2 * kEpilogueWarps, kAccBuffers, 32, kTileT, true};
  const uint32_t tmem_base = set_up<2>(p, map_t, map_w, s, base, warp, set, true);
  const int units = units_of(p, s, kTileF), first = blockIdx.x / 2, step = gridDim.x / 2;
  if (warp < kFirstEpilogueWarp) {
    set_max_registers_down<kFewRegisters>();
    if (warp == 0)
      load_operands<kMode>(p, map_t, map_w, s, a0, b0, rank, first, step, units);
    else if (warp == 1 && rank == 0)
      issue_mmas<kMode>(p, s, a0, b0, tmem_base, first, step, units);
    else if (warp == 2)
      load_scales(p, s, rank, first, step, units, lane);
  } else {
    set_max_registers_up<kManyRegisters>();
    accumulate(p, map_d, s, out, tmem_base, rank, first, step, units, warp, lane);
  }
  tear_down<2>(s, tmem_base, warp, true);
}

}  // namespace many

// ==================================================================================================== scales in the tensor core
//
// All three products where every scale is this library's own, a power of two: a CTA pair, 256 x 256. Operand A has the output's
// rows (tokens; a weight gradient's features), 128 per CTA, B its columns, each CTA half of them. Scale tiles (512 bytes: a word
// for each of 128 rows or columns, the E8M0 byte four times, in the order of the copy to tensor memory) go through shared into
// tensor memory. Two accumulator buffers share 32 columns, so that the scales find room beside them: [0, 256), [224, 480),
// scales at [480, 492); the epilogue drains the shared columns first.

namespace scaled {

constexpr int kTile = 256;
constexpr uint32_t kScaleTile = 512, kScaleBytes = 3 * kScaleTile;
constexpr uint32_t kAcc1 = 224;  // the second accumulator buffer; the first is at 0
constexpr uint32_t kScaleA = 480, kScaleB = 484;

// Blocks that a weight gradient sums up in tensor memory at a time; longer sums go on in registers. The tensor core cuts its sums
// off instead of rounding them, which shortens them by a part of each step's last bit: with all 16384 tokens in one sum dw was
// 1.1e-6 off (2-norm), with 4096 2.1e-7. The other two products are rounded to bf16.
constexpr int kSegment = 32;

struct Shared : Common<5> {
  int first_block[kMaxExperts + 2];  // blocks of 128 tokens before an expert's
  LineStage out[kEpilogueWarps];
};

constexpr size_t kStageBytes = kABytes + kBBytes + kScaleBytes;
constexpr size_t kSmemBytes = 1024 + Shared::kStages * kStageBytes + sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");

struct Unit {
  int expert;
  int block0, blocks;  // weight gradient: the expert's token blocks; else the tile's first token block, and the blocks of the contraction
  int m0, rows;        // first row of the output (of the expert's dw), and how many there are
  int n0;              // first column
};

template <int kMode>
__device__ __forceinline__ Unit unit_at(const Params& p, const Shared* s, int u) {
  Unit x;
  if constexpr (kMode == kWeightGrad) {
    const int mt = (p.features + kTile - 1) / kTile, nt = (p.n + kTile - 1) / kTile;
    x.expert = u / (mt * nt);
    int v = u - x.expert * mt * nt;
    const int panel = v / (kPanel * nt);
    v -= panel * kPanel * nt;
    const int width = min(kPanel, mt - panel * kPanel);
    x.n0 = v / width * kTile;
    x.m0 = (panel * kPanel + v % width) * kTile;
    x.rows = min(kTile, p.features - x.m0);
    x.block0 = s->first_block[x.expert];
    x.blocks = s->first_block[x.expert + 1] - x.block0;
  } else {
    const mxb200::Unit y = mxb200::unit_at<kTile, kTile>(p, s, u);
    x.expert = y.expert;
    x.n0 = y.f0;
    x.m0 = y.row0;
    x.rows = y.rows;
    x.blocks = y.blocks;
    x.block0 = y.blocks > 0 ? s->first_block[y.expert] + (y.row0 - s->first_row[y.expert]) / kBlock : 0;
  }
  return x;
}

template <int kMode>
__device__ __forceinline__ void load_operands(const Params& p, const Maps& maps, Shared* s, uint32_t a0, int rank, int first, int step, int units) {
  const uint32_t el = elect_one() ? 1u : 0u, el_leader = rank == 0 ? el : 0u;
  const uint32_t empty0 = smem_u32(&s->empty[0]), full0 = smem_u32(&s->full[0]);
  const uint32_t full_leader0 = map_to_cta(full0, 0);
  const uint32_t b0 = a0 + Shared::kStages * kABytes, sf0 = b0 + Shared::kStages * kBBytes;
  uint32_t stage = 0, phase = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kMode>(p, s, u);
    for (int b = 0; b < x.blocks; ++b) {
      if (!wait_bounded(empty0 + stage * 8, phase ^ 1u, &s->abort_flag, kSiteStageEmpty))
        return;
      mbar_arrive_expect_tx(el_leader, full0 + stage * 8, 2 * kStageBytes);
      const uint32_t full = full_leader0 + stage * 8, a = a0 + stage * kABytes, bs = b0 + stage * kBBytes, sf = sf0 + stage * kScaleBytes;
      if constexpr (kMode == kWeightGrad) {
        const int block = x.block0 + b;
        tma_load_3d_pair(el, a, &maps.a, full, x.m0 + rank * 128, block * kBlock, 0);
        tma_load_3d_pair(el, bs, &maps.b, full, x.n0 + rank * 128, block * kBlock, 0);
        tma_load_3d_pair(el, sf, &maps.a_scale, full, 0, (x.m0 >> 7) + rank, block);
        tma_load_3d_pair(el, sf + kScaleTile, &maps.b_scale, full, 0, x.n0 >> 7, block);
      } else {
        const int k = b * kBlock, block = x.block0 + rank, feature = x.n0 + rank * 128;
        const int weight0 = x.expert * p.w_scale_rows;  // the expert's first row of scale tiles
        tma_load_3d_pair(el, a, &maps.a, full, k, block * kBlock, 0);
        tma_load_3d_pair(el, bs, &maps.b, full, kMode == kForward ? k : feature, kMode == kForward ? feature : k, x.expert);
        tma_load_3d_pair(el, sf, &maps.a_scale, full, 0, b, block);
        tma_load_3d_pair(el, sf + kScaleTile, &maps.b_scale, full, 0, kMode == kForward ? b : x.n0 >> 7,
                         weight0 + (kMode == kForward ? x.n0 >> 7 : b));
      }
      if (++stage == Shared::kStages)
        stage = 0, phase ^= 1u;
    }
  }
}

template <int kMode>
__device__ __forceinline__ void issue_mmas(const Params& p, Shared* s, uint32_t a0, uint32_t tmem_base, int first, int step, int units) {
  constexpr bool kAMn = kMode == kWeightGrad, kBMn = kMode != kForward;
  // K = 32: 32 bytes within K-major rows, 32 rows of MN-major ones
  constexpr uint32_t kAStep = kAMn ? 4096 >> 4 : 32 >> 4, kBStep = kBMn ? 4096 >> 4 : 32 >> 4;
  constexpr uint32_t idesc = make_idesc_mxf8(kTile, kTile) | (kAMn ? kIdescAMn : 0u) | (kBMn ? kIdescBMn : 0u);
  const uint32_t el = elect_one() ? 1u : 0u;
  const uint32_t full0 = smem_u32(&s->full[0]), empty0 = smem_u32(&s->empty[0]);
  const uint32_t b0 = a0 + Shared::kStages * kABytes, sf0 = b0 + Shared::kStages * kBBytes;
  const uint64_t a_desc0 = make_smem_desc(a0, 1024, 1024, 2), b_desc0 = make_smem_desc(b0, 1024, 1024, 2);
  const uint64_t sf_desc0 = make_smem_desc(sf0, 0, 128, 0);
  const uint32_t sfa = tmem_base + kScaleA, sfb = tmem_base + kScaleB;
  uint32_t stage = 0, phase = 0, local = 0;
  for (int u = first; u < units; u += step) {
    const int blocks = unit_at<kMode>(p, s, u).blocks;
    for (int b = 0; b < blocks;) {
      const uint32_t buf = local & 1u;
      if (!wait_bounded(smem_u32(&s->acc_empty[buf]), ((local >> 1) & 1u) ^ 1u, &s->abort_flag, kSiteAccEmpty) ||
          (local > 0 && !wait_bounded(smem_u32(&s->overlap_free), (local - 1) & 1u, &s->abort_flag, kSiteOverlap)))
        return;
      ++local;
      const int begin = b, end = kMode == kWeightGrad ? min(b + kSegment, blocks) : blocks;
      for (; b < end; ++b) {
        if (!wait_bounded(full0 + stage * 8, phase, &s->abort_flag, kSiteStageFull))
          return;
        tcgen05_fence_after_sync();
        const uint64_t sf = sf_desc0 + stage * (kScaleBytes >> 4);
        tcgen05_cp_32x128b_warpx4_pair(el, sfa, sf);
        tcgen05_cp_32x128b_warpx4_pair(el, sfb, sf + (kScaleTile >> 4));
        tcgen05_cp_32x128b_warpx4_pair(el, sfb + 4, sf + 2 * (kScaleTile >> 4));
        const uint64_t a = a_desc0 + stage * (kABytes >> 4), bd = b_desc0 + stage * (kBBytes >> 4);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          tcgen05_mma_mxf8_pair(el, tmem_base + buf * kAcc1, a + k * kAStep, bd + k * kBStep, idesc, sfa, sfb, b > begin || k > 0);
        tcgen05_commit_pair(el, empty0 + stage * 8, 3);
        if (++stage == Shared::kStages)
          stage = 0, phase ^= 1u;
      }
      tcgen05_commit_pair(el, &s->acc_full[buf], 3);
    }
  }
}

// kLong: weight gradients whose sums may take more than a segment.
template <int kMode, bool kLong>
__device__ __forceinline__ void store(const Params& p, Shared* s, uint32_t tmem_base, int rank, int first, int step, int units, int warp, int lane) {
  const int quarter = warp & 3, part = (warp - kFirstEpilogueWarp) >> 2;
  const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t acc_empty0 = map_to_cta(smem_u32(&s->acc_empty[0]), 0), overlap_free = map_to_cta(smem_u32(&s->overlap_free), 0);
  const int columns = kMode == kWeightGrad ? p.n : p.features;
  const bool bf16 = kMode != kWeightGrad || p.out_bf16;
  LineStage* stage = &s->out[warp - kFirstEpilogueWarp];
  uint32_t local = 0;
  for (int u = first; u < units; u += step) {
    const Unit x = unit_at<kMode>(p, s, u);
    const int row = rank * 128 + quarter * 32, rows = x.rows - row;
    const int64_t line = static_cast<int64_t>(columns) * (bf16 ? 2 : 4);
    unsigned char* d = static_cast<unsigned char*>(p.d) + ((kMode == kWeightGrad ? static_cast<int64_t>(x.expert) * p.features : 0) + x.m0 + row) * line +
                       static_cast<int64_t>(x.n0) * (bf16 ? 2 : 4);
    if constexpr (kLong) {
      float sum[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 32; ++k)
          sum[c][k] = 0.f;
      for (int b = 0; b < x.blocks; b += kSegment, ++local) {
        const uint32_t buf = local & 1u;
        if (!wait_bounded(smem_u32(&s->acc_full[buf]), (local >> 1) & 1u, &s->abort_flag, kSiteAccFull))
          return;
        tcgen05_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t0 + buf * kAcc1 + 128 * part + 32 * c, v);
          tmem_ld_wait(v);
          if (c == 0 || c == 3) {
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0 && c == (buf == 0 ? 3 : 0) && part == static_cast<int>(1 - buf))
              mbar_arrive_cluster(overlap_free);
            if (lane == 0 && c == 3)
              mbar_arrive_cluster(acc_empty0 + buf * 8);
          }
#pragma unroll
          for (int k = 0; k < 32; ++k)
            sum[c][k] += __uint_as_float(v[k]);
        }
      }
      if (!bf16) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          store_lines(stage, lane, d + 128 * (c + 4 * part), line, rows, (columns - x.n0 - 32 * (c + 4 * part)) * 4, [&](int q) {
            return make_uint4(__float_as_uint(sum[c][4 * q]), __float_as_uint(sum[c][4 * q + 1]), __float_as_uint(sum[c][4 * q + 2]),
                              __float_as_uint(sum[c][4 * q + 3]));
          });
      } else {
#pragma unroll
        for (int c = 0; c < 4; c += 2)
          store_lines(stage, lane, d + 64 * (c + 4 * part), line, rows, (columns - x.n0 - 32 * (c + 4 * part)) * 2, [&](int q) {
            const float* f = &sum[c + (q >> 2)][8 * (q & 3)];
            return make_uint4(pack_bf16x2_rn(f[0], f[1]), pack_bf16x2_rn(f[2], f[3]), pack_bf16x2_rn(f[4], f[5]), pack_bf16x2_rn(f[6], f[7]));
          });
      }
      continue;
    }
    const uint32_t buf = local & 1u;
    if (x.blocks > 0) {
      if (!wait_bounded(smem_u32(&s->acc_full[buf]), (local >> 1) & 1u, &s->abort_flag, kSiteAccFull))
        return;
      tcgen05_fence_after_sync();
      ++local;
    }
    uint32_t half[16];  // bf16: the first 32 columns of a line
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      // the columns that the buffers share, [224, 256), first: the last chunk of part 1 in buffer 0, the first of part 0 in 1.
      // A line of bf16 is two chunks: 3, 2, then 1, 0; or 0, 1, then 2, 3.
      const int c = (buf == 0 ? 3 - i : i) + 4 * part;
      uint32_t v[32];
      if (x.blocks > 0) {
        tmem_ld_32x32b_x32(t0 + buf * kAcc1 + 32 * c, v);
        tmem_ld_wait(v);
        if (i == 0 && part == static_cast<int>(1 - buf)) {
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0)
            mbar_arrive_cluster(overlap_free);
        }
        if (i == 3) {
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0)
            mbar_arrive_cluster(acc_empty0 + buf * 8);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          v[k] = 0;
      }
      if (!bf16) {
        store_lines(stage, lane, d + 128 * c, line, rows, (columns - x.n0 - 32 * c) * 4,
                    [&](int q) { return make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]); });
        continue;
      }
      uint32_t h[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        h[j] = pack_bf16x2_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
      if ((i & 1) == 0) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          half[j] = h[j];
      } else {
        const bool swapped = buf == 0;
        store_lines(stage, lane, d + 64 * (c & ~1), line, rows, (columns - x.n0 - 32 * (c & ~1)) * 2,
                    [&](int q) {
                      const int k = 4 * (q & 3);
                      const bool from_half = (q < 4) != swapped;
                      return make_uint4(from_half ? half[k] : h[k], from_half ? half[k + 1] : h[k + 1],
                                        from_half ? half[k + 2] : h[k + 2], from_half ? half[k + 3] : h[k + 3]);
                    });
      }
    }
  }
}

template <int kMode, bool kLong>
__device__ __forceinline__ void body(const Params& p, const Maps& maps) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t a0 = smem_u32(base);
  Shared* s = reinterpret_cast<Shared*>(base + Shared::kStages * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const SetUp set{1, 1, 2 * kEpilogueWarps, 2, 1, kTile, kMode != kWeightGrad};
  const uint32_t tmem_base = set_up<2>(p, &maps.a, &maps.b, s, base, warp, set, true, s->first_block);
  const int units = kMode == kWeightGrad ? p.experts * ((p.features + kTile - 1) / kTile) * ((p.n + kTile - 1) / kTile) : units_of(p, s, kTile);
  const int first = blockIdx.x / 2, step = gridDim.x / 2;
  if (warp < kFirstEpilogueWarp) {
    if constexpr (kLong)
      set_max_registers_down<kFewRegisters>();
    if (warp == 0)
      load_operands<kMode>(p, maps, s, a0, rank, first, step, units);
    else if (warp == 1 && rank == 0)
      issue_mmas<kMode>(p, s, a0, tmem_base, first, step, units);
  } else {
    if constexpr (kLong)
      set_max_registers_up<kManyRegisters>();
    store<kMode, kLong>(p, s, tmem_base, rank, first, step, units, warp, lane);
  }
  tear_down<2>(s, tmem_base, warp, true);
}

}  // namespace scaled

struct Launch {
  Maps maps;
  Params p;
};

}  // namespace
}  // namespace mxb200

__global__ void __launch_bounds__(mxb200::kThreads, 1) mxb200_block_gemm_forward_few(const __grid_constant__ mxb200::Launch args) {
  mxb200::few::body<mxb200::kForward, mxb200::few::Tile128>(args.p, &args.maps.a, &args.maps.b);
}
__global__ void __launch_bounds__(mxb200::kThreads, 1) mxb200_block_gemm_forward_32(const __grid_constant__ mxb200::Launch args) {
  mxb200::few::body<mxb200::kForward, mxb200::few::Tile32>(args.p, &args.maps.a, &args.maps.b);
}
__global__ void __launch_bounds__(mxb200::kThreads, 1) mxb200_block_gemm_quantize_few(const __grid_constant__ mxb200::Launch args) {
  mxb200::few::body<mxb200::kForward, mxb200::few::Quantizing>(args.p, &args.maps.a, &args.maps.b);
}
__global__ void __launch_bounds__(mxb200::kThreads, 1) mxb200_block_gemm_input_grad_few(const __grid_constant__ mxb200::Launch args) {
  mxb200::few::body<mxb200::kInputGrad, mxb200::few::Tile128>(args.p, &args.maps.a, &args.maps.b);
}
__global__ void __launch_bounds__(mxb200::kThreads, 1) mxb200_block_gemm_input_grad_32(const __grid_constant__ mxb200::Launch args) {
  mxb200::few::body<mxb200::kInputGrad, mxb200::few::Tile32>(args.p, &args.maps.a, &args.maps.b);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_forward_many(const __grid_constant__ mxb200::Launch args) {
  mxb200::many::body<mxb200::kForward>(args.p, &args.maps.a, &args.maps.b, &args.maps.d);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_input_grad_many(const __grid_constant__ mxb200::Launch args) {
  mxb200::many::body<mxb200::kInputGrad>(args.p, &args.maps.a, &args.maps.b, &args.maps.d);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_weight_grad(const __grid_constant__ mxb200::Launch args) {
  mxb200::scaled::body<mxb200::kWeightGrad, false>(args.p, args.maps);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_weight_grad_long(const __grid_constant__ mxb200::Launch args) {
  mxb200::scaled::body<mxb200::kWeightGrad, true>(args.p, args.maps);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_forward_scaled(const __grid_constant__ mxb200::Launch args) {
  mxb200::scaled::body<mxb200::kForward, false>(args.p, args.maps);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxb200::kThreads, 1)
      mxb200_block_gemm_input_grad_scaled(const __grid_constant__ mxb200::Launch args) {
  mxb200::scaled::body<mxb200::kInputGrad, false>(args.p, args.maps);
}

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

// The (tokens, features) bf16 output, 32 tokens x 64 features at a time, 128-byte swizzle.
int make_output_map(CUtensorMap* map, void* base, int64_t features, int64_t tokens) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr)
    return MXB200_ERR_DRIVER;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(features), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(features) * 2};
  const cuuint32_t box[2] = {64, 32};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MXB200_OK : MXB200_ERR_DRIVER;
}

// (z, y) scale tiles of 128 words, `box_z` x `box_y` at a time.
int make_scale_map(CUtensorMap* map, const void* base, int64_t y, int64_t z, int box_y, int box_z) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr)
    return MXB200_ERR_DRIVER;
  const cuuint64_t dims[3] = {kBlock, static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z)};
  const cuuint64_t strides[2] = {kBlock * 4, static_cast<cuuint64_t>(y) * kBlock * 4};
  const cuuint32_t box[3] = {kBlock, static_cast<cuuint32_t>(box_y), static_cast<cuuint32_t>(box_z)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MXB200_OK : MXB200_ERR_DRIVER;
}

using Kernel = void (*)(Launch);

struct Variant {
  const char* name;
  Kernel kernel;
  size_t smem;
  int ctas;             // per unit
  int tokens, features; // of a unit
  RegisterSplit registers = kNotTraded;
};

enum VariantId : int { kForwardFew, kForward32, kForwardMany, kForwardQuantizing, kInputGradFew, kInputGrad32, kInputGradMany, kWeightGradPair, kWeightGradLong, kForwardScaled, kInputGradScaled, kVariants };

const Variant& variant(VariantId id) {
  static const Variant variants[kVariants] = {
        {"forward_few", mxb200_block_gemm_forward_few, few::Tile128::kSmemBytes, 1, few::Tile128::kTileT, few::kTileF},
        {"forward_32", mxb200_block_gemm_forward_32, few::Tile32::kSmemBytes, 1, few::Tile32::kTileT, few::kTileF},
        {"forward_many", mxb200_block_gemm_forward_many, many::kSmemBytes, 2, many::kTileT, many::kTileF, kTraded},
        {"quantize_few", mxb200_block_gemm_quantize_few, few::Quantizing::kSmemBytes, 1, few::Quantizing::kTileT, few::kTileF},
        {"input_grad_few", mxb200_block_gemm_input_grad_few, few::Tile128::kSmemBytes, 1, few::Tile128::kTileT, few::kTileF},
        {"input_grad_32", mxb200_block_gemm_input_grad_32, few::Tile32::kSmemBytes, 1, few::Tile32::kTileT, few::kTileF},
        {"input_grad_many", mxb200_block_gemm_input_grad_many, many::kSmemBytes, 2, many::kTileT, many::kTileF, kTraded},
        {"weight_grad", mxb200_block_gemm_weight_grad, scaled::kSmemBytes, 2, scaled::kTile, scaled::kTile},
        {"weight_grad_long", mxb200_block_gemm_weight_grad_long, scaled::kSmemBytes, 2, scaled::kTile, scaled::kTile, kTraded},
        {"forward_scaled", mxb200_block_gemm_forward_scaled, scaled::kSmemBytes, 2, scaled::kTile, scaled::kTile},
        {"input_grad_scaled", mxb200_block_gemm_input_grad_scaled, scaled::kSmemBytes, 2, scaled::kTile, scaled::kTile}};
  return variants[id];
}

// Token tiles that are expected: how the rows spread over experts is not known here, so every expert is taken to have some, with
// half a tile left over. Rows that all go to a few experts find tiles that are too small for them: 4096 rows (1536 -> 2048) on 4
// experts take 18.7 us among 4 or 16, 26.4 among 64 and 46.9 among 128; 1024 rows 12.2, 10.0, 15.8 and 16.3.
int64_t expected_tiles(int64_t tokens, int experts, int tile) {
  const int64_t used = std::min<int64_t>(experts, tokens);
  return experts == 1 ? blocks_up(tokens, tile) : std::max(used, tokens / tile + used / 2);
}

constexpr int kMostSplits = 8;

// What the current device does with a kernel, looked up once: its registers, its shared memory, and how many clusters of 1 to 8 of its CTAs
// find room at a time (a cluster stays within one of the GPU's groups of SMs: 15 clusters of 8, 33 of 4, 45 of 3).
struct Configured {
  bool done = false;
  int clusters[kMostSplits + 1] = {};
};

int configure(VariantId id, const DeviceInfo& dev, Configured* out) {
  static std::mutex mu;
  static Configured known[64][kVariants];
  std::lock_guard<std::mutex> lock(mu);
  Configured local;
  Configured& c = dev.device < 64 ? known[dev.device][id] : local;
  if (!c.done) {
    const Variant& v = variant(id);
    const void* const kernel = reinterpret_cast<const void*>(v.kernel);
    cudaFuncAttributes built{};
    bool ok = cudaFuncGetAttributes(&built, kernel) == cudaSuccess && v.registers.served_by(built.numRegs) &&
              cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(v.smem)) == cudaSuccess;
    for (int n = 2; ok && v.ctas == 1 && n <= kMostSplits; ++n) {
      cudaLaunchAttribute attribute{};
      attribute.id = cudaLaunchAttributeClusterDimension;
      attribute.val.clusterDim.x = n, attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(n), config.blockDim = dim3(kThreads), config.dynamicSmemBytes = v.smem;
      config.attrs = &attribute, config.numAttrs = 1;
      ok = cudaOccupancyMaxActiveClusters(&c.clusters[n], kernel, &config) == cudaSuccess;
    }
    if (!ok) {
      cudaGetLastError();
      return MXB200_ERR_LAUNCH;
    }
    c.clusters[1] = dev.sms / v.ctas;
    c.done = true;
  }
  *out = c;
  return MXB200_OK;
}

int tile_tokens(int64_t tokens, int experts, int tile) {
  return static_cast<int>(std::min<int64_t>(tile, blocks_up(tokens, experts)));
}

// Few tokens: CTAs that share a unit's blocks, what is expected to take least among those of which all units' clusters find room at
// once. A block takes a CTA 0.17 us of a small tile and 0.3 of a large one or
// where it is quantized (up to 16 tokens go by that, so that the result does not depend on who quantizes them), the exchange 2.5 us
// and 0.02 for each of the tile's tokens. One token of 6144 -> 1536: 16.6 us in one CTA per unit and 7.5 in eight; 32 tokens of
// 1536 -> 1536 5.1 in one and 6.2 in eight.
int share_blocks(int64_t units, int blocks, int tile, int tokens, const Configured& c) {
  const double block = tile == few::Tile32::kTileT && tokens > 16 ? 0.17 : 0.3;
  int best = 1;
  double least = block * blocks;
  for (int n = 2; n <= std::min(kMostSplits, blocks) && units <= c.clusters[n]; ++n)
    if (const double t = block * static_cast<double>(blocks_up(blocks, n)) + 2.5 + 0.02 * tokens; t < least)
      best = n, least = t;
  return best;
}

struct Plan {
  VariantId id;
  int splits;
  int64_t units;  // expected
};

// The kernel that a product of `blocks` contraction blocks to `features` features takes: the one that is expected to be done first.
// With all SMs at work a block of their tile takes about 0.2 us (32 tokens), 0.33 (128) and 0.37 (a pair's 256 x 256), a unit's
// output costs as much as 2 to 4 blocks. In small, large and pairs' tiles: 256 x 1536 -> 1536 5.4, 7.9 and 9.2 us; 512 x 1536 ->
// 6144 18.8, 13.5 and 10.2; 1111 x 1040 -> 2000 -, 8.3 and 8.9; 16384 x 1536 -> 1536 -, 59.7 and 41.2; 16 rows for each of 64 experts
// (1536 -> 2048) 35.5, 38.5 and 54, 48 rows for each 48.4, 46.0 and -; 1024 rows over 8 experts (2048 -> 2048) -, 19.7 and 14.9.
int plan_product(int64_t tokens, int experts, int features, int blocks, bool forward, const DeviceInfo& dev, Plan* plan) {
  struct Kind {
    VariantId id;
    double start, output_blocks, block;
  };
  const Kind kinds[3] = {{forward ? kForward32 : kInputGrad32, 3, 2, 0.2}, {forward ? kForwardFew : kInputGradFew, 4, 3, 0.33}, {forward ? kForwardMany : kInputGradMany, 4.5, 4, 0.37}};
  double least = 0;
  for (const Kind& kind : kinds) {
    const Variant& v = variant(kind.id);
    Configured c;
    if (const int st = configure(kind.id, dev, &c); st != MXB200_OK)
      return st;
    const int64_t units = expected_tiles(tokens, experts, v.tokens) * blocks_up(features, v.features);
    const int of_tile = tile_tokens(tokens, experts, v.tokens);
    const int splits = v.ctas == 1 ? share_blocks(units, blocks, v.tokens, of_tile, c) : 1;
    const double t = kind.start + (splits > 1 ? 2.5 + 0.02 * of_tile : 0) +
                     static_cast<double>(blocks_up(units, dev.sms / v.ctas)) * (blocks_up(blocks, splits) + kind.output_blocks) * kind.block;
    if (least == 0 || t < least)
      *plan = {kind.id, splits, units}, least = t;
  }
  return MXB200_OK;
}

// Whether a forward product of bf16 input takes less than the quantizer's launch and the product of its output, which is 2 to 3 us
// and as much on the host: every CTA's repeating it costs about 0.014 us for a token of a block and 0.03 a block. One token of 1536
// -> 6144: 6.6 us in one launch and 5.0 + 1.9 in two; 16 tokens 9.3 and 5.0 + 1.9; one token of 6144 -> 24576 35.2 and 29.6 + 1.9;
// 16 rows over 16 experts (1536 -> 2048) 8.5 and 7.0 + 1.9, 64 rows over 64 experts 26.3 and 20.4 + 1.9.
bool quantizes(int64_t tokens, int experts, int blocks, const DeviceInfo& dev, const Plan& plan) {
  return plan.id == kForward32 && blocks_up(plan.units, dev.sms) * blocks_up(blocks, plan.splits) *
                                        (tile_tokens(tokens, experts, few::Quantizing::kTileT) + 2) <= 140;
}

int check_sizes(const mxb200_block_gemm_args& g) {
  if (g.kind < MXB200_BLOCK_FORWARD || g.kind > MXB200_BLOCK_INPUT_GRAD_SCALED ||
      (g.out_kind != MXB200_OUT_BF16 && (g.out_kind != MXB200_OUT_F32 || g.kind != MXB200_BLOCK_WEIGHT_GRAD)))
    return MXB200_ERR_ARGUMENT;
  if (g.tokens < 0 || g.tokens > kMostSize || g.in_features <= 0 || g.in_features > kMostSize || g.out_features <= 0 ||
      g.out_features > kMostSize || g.in_features % 16 || g.out_features % 16 || g.experts < 1 || g.experts > kMaxExperts)
    return MXB200_ERR_SHAPE;
  if (g.b_ld != 0 && g.kind != MXB200_BLOCK_FORWARD)
    return MXB200_ERR_ARGUMENT;
  if (g.b_ld != 0 && (g.b_ld < g.in_features || g.b_ld % 8))
    return MXB200_ERR_SHAPE;
  return MXB200_OK;
}

struct Choice {
  VariantId id;
  int splits;  // few tokens: CTAs that share a unit's blocks
  Configured configured;
};

// The kernel of a call with checked sizes and at least one token.
int choose(const mxb200_block_gemm_args& g, const DeviceInfo& dev, Choice* out) {
  const bool forward = g.kind == MXB200_BLOCK_FORWARD || g.kind == MXB200_BLOCK_FORWARD_SCALED;
  out->splits = 1;
  if (g.kind == MXB200_BLOCK_WEIGHT_GRAD) {
    // The host does not know an expert's rows, only that none has more than there are. Where more are there and no expert's sum is
    // long after all, the kernel for long ones takes as long or a little longer: 16384 rows over 16 experts (1536 -> 2048) 69.1 us
    // and 64.6 in the other, 8192 over 32 83.9 and 83.1, 16384 over 64 160 and 166.
    out->id = g.tokens <= scaled::kSegment * kBlock ? kWeightGradPair : kWeightGradLong;
    return configure(out->id, dev, &out->configured);
  }
  if (g.kind == MXB200_BLOCK_FORWARD_SCALED || g.kind == MXB200_BLOCK_INPUT_GRAD_SCALED) {
    out->id = forward ? kForwardScaled : kInputGradScaled;
    return configure(out->id, dev, &out->configured);
  }
  const int blocks = static_cast<int>(blocks_up(forward ? g.in_features : g.out_features, kBlock));
  const int features = static_cast<int>(forward ? g.out_features : g.in_features);
  Plan plan;
  if (const int st = plan_product(g.tokens, g.experts, features, blocks, forward, dev, &plan); st != MXB200_OK)
    return st;
  out->id = g.b_ld != 0 ? kForwardQuantizing : plan.id;
  const Variant& v = variant(out->id);
  if (const int st = configure(out->id, dev, &out->configured); st != MXB200_OK)
    return st;
  if (v.ctas == 1)
    out->splits = share_blocks(expected_tiles(g.tokens, g.experts, v.tokens) * blocks_up(features, v.features), blocks, v.tokens,
                               tile_tokens(g.tokens, g.experts, v.tokens), out->configured);
  return MXB200_OK;
}

int block_gemm(const mxb200_block_gemm_args& g, cudaStream_t stream) {
  if (const int st = check_sizes(g); st != MXB200_OK)
    return st;
  if (g.ends == nullptr && g.experts != 1)
    return MXB200_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(g.ends) & 3) != 0)
    return MXB200_ERR_ALIGNMENT;
  DeviceInfo dev;
  if (int st = current_device(&dev); st != MXB200_OK)
    return st;
  const bool wgrad = g.kind == MXB200_BLOCK_WEIGHT_GRAD;
  const bool scaled = g.kind == MXB200_BLOCK_FORWARD_SCALED || g.kind == MXB200_BLOCK_INPUT_GRAD_SCALED;
  if (g.tokens == 0) {
    if (!wgrad)
      return MXB200_OK;
    if (g.d == nullptr)
      return MXB200_ERR_NULL;
    const size_t bytes = static_cast<size_t>(g.experts) * g.out_features * g.in_features * (g.out_kind == MXB200_OUT_F32 ? 4 : 2);
    return cudaMemsetAsync(g.d, 0, bytes, stream) == cudaSuccess ? MXB200_OK : MXB200_ERR_LAUNCH;
  }
  const bool quantize = g.b_ld != 0;
  if (g.a == nullptr || g.a_scale == nullptr || g.b == nullptr || (g.b_scale == nullptr && !quantize) || g.d == nullptr)
    return MXB200_ERR_NULL;
  const auto bits = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  if (!aligned16(g.a) || !aligned16(g.b) || !aligned16(g.d) ||
      ((bits(g.a_scale) | bits(g.b_scale)) & (wgrad || scaled ? 15 : 3)) != 0)
    return MXB200_ERR_ALIGNMENT;
  const int64_t in = g.in_features, out = g.out_features;
  const bool forward = g.kind == MXB200_BLOCK_FORWARD || g.kind == MXB200_BLOCK_FORWARD_SCALED;
  const int from = static_cast<int>(forward ? in : out), to = static_cast<int>(forward ? out : in);
  const int blocks = static_cast<int>(blocks_up(from, kBlock));
  Launch l{};
  Params& p = l.p;
  p.d = g.d, p.ends = g.ends, p.experts = g.experts, p.rows = static_cast<int>(g.tokens);
  p.out_bf16 = g.out_kind == MXB200_OUT_BF16;
  // token tiles are known on the device only; this many at most
  const auto most_tiles = [&](int64_t tile) {
    return g.ends == nullptr ? blocks_up(g.tokens, tile) : (g.tokens + (tile - 1) * std::min<int64_t>(g.experts + 1, g.tokens)) / tile;
  };
  Choice choice;
  int st = choose(g, dev, &choice);
  if (st != MXB200_OK)
    return st;
  const Variant& v = variant(choice.id);
  p.splits = choice.splits;
  int64_t units;
  if (wgrad) {
    const int64_t capacity = mxb200_block_token_blocks(g.tokens, g.experts) * kBlock;
    p.features = static_cast<int>(out), p.n = static_cast<int>(in);
    units = g.experts * blocks_up(out, mxb200::scaled::kTile) * blocks_up(in, mxb200::scaled::kTile);
    st = make_map(&l.maps.a, g.a, out, capacity, 1, 128);
    st = st != MXB200_OK ? st : make_map(&l.maps.b, g.b, in, capacity, 1, 128);
    st = st != MXB200_OK ? st : make_scale_map(&l.maps.a_scale, g.a_scale, blocks_up(out, kBlock), capacity / kBlock, 1, 1);
    st = st != MXB200_OK ? st : make_scale_map(&l.maps.b_scale, g.b_scale, blocks_up(in, kBlock), capacity / kBlock, 2, 1);
  } else if (scaled) {
    const int64_t capacity = mxb200_block_token_blocks(g.tokens, g.experts) * kBlock;
    p.features = to, p.blocks = blocks, p.w_scale_rows = static_cast<int>(blocks_up(out, kBlock));
    units = most_tiles(mxb200::scaled::kTile) * blocks_up(to, mxb200::scaled::kTile);
    st = make_map(&l.maps.a, g.b, from, capacity, 1, 128);
    st = st != MXB200_OK ? st : make_map(&l.maps.b, g.a, in, out, g.experts, 128);
    st = st != MXB200_OK ? st : make_scale_map(&l.maps.a_scale, g.b_scale, blocks, capacity / kBlock, 1, 1);
    st = st != MXB200_OK ? st : make_scale_map(&l.maps.b_scale, g.a_scale, blocks_up(in, kBlock), blocks_up(out, kBlock) * g.experts, forward ? 1 : 2, forward ? 2 : 1);
  } else {
    const bool many = v.ctas == 2;
    p.weight_scale = static_cast<const float*>(g.a_scale), p.token_scale = static_cast<const float*>(g.b_scale);
    p.token_ld = quantize ? g.b_ld : g.tokens, p.features = to, p.blocks = blocks;
    p.input = g.b, p.input_cols = from;
    p.w_scale_expert = blocks_up(out, kBlock) * blocks_up(in, kBlock);
    p.w_scale_f = forward ? static_cast<int>(blocks_up(in, kBlock)) : 1, p.w_scale_b = forward ? 1 : static_cast<int>(blocks_up(in, kBlock));
    units = most_tiles(v.tokens) * blocks_up(to, v.features);
    CUtensorMap *weight = many ? &l.maps.b : &l.maps.a, *token = many ? &l.maps.a : &l.maps.b;
    st = make_map(weight, g.a, in, out, g.experts, 128);
    st = st != MXB200_OK || quantize ? st : make_map(token, g.b, from, g.tokens, 1, many ? 128 : 32);
    st = st != MXB200_OK || !many ? st : make_output_map(&l.maps.d, g.d, to, g.tokens);
  }
  if (st != MXB200_OK)
    return st;
  if (units > kMostSize)
    return MXB200_ERR_SHAPE;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, choice.configured.clusters[p.splits])) * std::max(v.ctas, p.splits);
  return launch_kernel_clusters(p.splits > 1 ? p.splits : 0, v.kernel, grid, kThreads, v.smem, stream, l);
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

// A training pass's two row products by the scaled kernels, which always go by pairs, against the kernels for any scales with the
// quantizers of each, in us: 2048 x 1536 -> 1536 26.7 and 28.3, 2048 x 1536 -> 6144 56.0 and 64.1, 5001 x 640 ->
// 1552 29.9 and 33.1, 16384 x 6144 -> 1536 339 and 384, 16384 x 144 -> 4112 132 and 131, 8192 rows over 32 experts (1536 -> 2048) 112
// and 128. Where the others would not take pairs for both: 1111 x 1040 -> 2000 26.9 and 25.3, 4096 x 512 -> 512 18.8 and 17.5, 1024 x
// 2048 -> 2048 26.0 and 26.2, 1024 x 6144 -> 1536 42.0 and 45.8, the most that the rule gives away.
extern "C" int mxb200_block_scaled(int64_t tokens, int64_t in_features, int64_t out_features, int experts) {
  using namespace mxb200;
  DeviceInfo dev;
  if (tokens <= 0 || in_features <= 0 || out_features <= 0 || experts <= 0 || current_device(&dev) != MXB200_OK)
    return 0;
  const int in_blocks = static_cast<int>(blocks_up(in_features, kBlock)), out_blocks = static_cast<int>(blocks_up(out_features, kBlock));
  Plan plan;
  return plan_product(tokens, experts, static_cast<int>(out_features), in_blocks, true, dev, &plan) == MXB200_OK && plan.id == kForwardMany &&
         plan_product(tokens, experts, static_cast<int>(in_features), out_blocks, false, dev, &plan) == MXB200_OK && plan.id == kInputGradMany;
}

extern "C" int mxb200_block_quantizes(int64_t tokens, int64_t in_features, int64_t out_features, int experts) {
  using namespace mxb200;
  DeviceInfo dev;
  if (tokens <= 0 || in_features <= 0 || out_features <= 0 || experts <= 0 || current_device(&dev) != MXB200_OK)
    return 0;
  const int blocks = static_cast<int>(blocks_up(in_features, kBlock));
  Plan plan;
  return plan_product(tokens, experts, static_cast<int>(out_features), blocks, true, dev, &plan) == MXB200_OK &&
         quantizes(tokens, experts, blocks, dev, plan);
}

extern "C" const char* mxb200_block_gemm_kernel(const mxb200_block_gemm_args* args, int* splits) {
  using namespace mxb200;
  DeviceInfo dev;
  Choice choice;
  if (args == nullptr || check_sizes(*args) != MXB200_OK || args->tokens == 0 || current_device(&dev) != MXB200_OK ||
      choose(*args, dev, &choice) != MXB200_OK)
    return nullptr;
  if (splits != nullptr)
    *splits = choice.splits;
  return variant(choice.id).name;
}

extern "C" int mxb200_block_gemm(const mxb200_block_gemm_args* args, void* stream) {
  if (args == nullptr)
    return MXB200_ERR_NULL;
  return mxb200::block_gemm(*args, static_cast<cudaStream_t>(stream));
}
