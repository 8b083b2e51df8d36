// Products of microscaled 4-bit matrices (include/xse_mx.h,
// include/xse_experts.h) on the fifth-generation tensor cores.
//
//   y[r][f] = act(sum_k x[r][k] w[f][k] + bias[f])
//
// with x and w as E2M1 codes and one power-of-two scale per 32 elements of k.
// tcgen05.mma kind::mxf4 multiplies the codes, applies both scales of each
// block of 32 and accumulates in fp32 in tensor memory.
//
// Roles. The weights are the MMA's A operand (128 features, the lanes of the
// accumulator) and the rows its B operand (kN rows, the accumulator's columns)
// for every size: a handful of rows then wastes no tensor-core rows, and the
// epilogue's warps hold 32 neighbouring features of a row, so that y is
// written in whole sectors without a transposition.
//
// One block per SM runs over its tiles: warp 0 copies stages of 256 elements
// of k with TMA (codes, 128-byte swizzled; scales, 512-byte tiles as they lie
// in memory), warp 1 moves the scales to tensor memory and issues the MMAs,
// warps 2 to 9 write the results, which overlaps with the next tile's MMAs.
//
// Few rows: warps 10 to 17 read and quantise the rows themselves, into a buffer
// that holds all of a row tile's k. A block takes neighbouring feature tiles,
// so it does that once for a row tile; a second buffer holds the next one. (In
// the stages, anew for every feature tile, the rows' latency bounded the
// kernel: 64 tokens' 4 choices of 64 experts 2048 -> 1024, 23.8 us.)
//
// Few tiles: a cluster of `split` blocks shares a tile, each taking a part of
// k; the parts are added in block order over distributed shared memory.
//
// Every wait is bounded. One that runs out sets a flag that the other roles
// see and g_wait_failed, which xse_mxfp4_check reports.

#include <cuda.h>

#include <type_traits>

#include "../../include/xse_dlrm.h"
#include "xse_mx_internal.h"

namespace xse {
namespace {

constexpr int kM = 128;            // features of a tile
constexpr int kStageK = 256;       // elements of k per stage (128 bytes)
constexpr int kEpilogueWarps = 8;  // two per quarter of the lanes
constexpr int kQuantizeWarps = 8;  // where the product quantises its rows
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr int kThreadsWithRows = kThreads + 32 * kQuantizeWarps;
constexpr int kABytes = kM * kStageK / 2;
constexpr int kScaleBytes = 2 * kMxTileBytes;  // a tile row's, per stage
constexpr int kSharedBytes = 216 * 1024;  // for stages and rows
constexpr int kMostStages = 10;
constexpr long long kWaitCycles = 4000000000ll;  // about two seconds

__device__ int g_wait_failed;

template <int kN>
struct Config {
  static constexpr int kBBytes = kN * kStageK / 2;
  static_assert(kN <= kMxTileRows, "one scale tile of b");
  static constexpr int kStageBytes = kABytes + kBBytes + 2 * kScaleBytes;
  static constexpr int kMost = kSharedBytes / kStageBytes;
  static constexpr int kStages = kMost > kMostStages ? kMostStages : kMost;
  // Where the product quantises its rows: a stage holds weights alone, and a
  // buffer of rows kRowStageBytes for every stage of k.
  static constexpr int kWeightStageBytes = kABytes + kScaleBytes;
  static constexpr int kRowStageBytes = kBBytes + kScaleBytes;
  // Tensor memory columns: accumulators, then each stage's scales.
  static constexpr int kAccColumns = kN < 32 ? 32 : kN;
  static constexpr int kAccs = 2;
  static constexpr int kScaleColumns = 16;
  // Columns that an epilogue warp takes (with 16 rows the second warp of a
  // quarter has none).
  static constexpr int kPart = kN < 32 ? 16 : kN / 2;
  static_assert(kAccs * kAccColumns + kStages * kScaleColumns <= 512,
                "tensor memory");
};

struct GemmParams {
  CUtensorMap a;  // weights [groups][out][row bytes]
  CUtensorMap b;  // rows [rows][row bytes]
  CUtensorMap a_scale_map, b_scale_map;  // [tiles][128 words], pairs only
  const uint8_t* a_scales;
  const uint8_t* b_scales;
  const float* bias;
  void* y;
  const int32_t* offsets;  // expert rows, or NULL for one group of all rows
  const void* x;           // unquantised rows
  const int32_t* order;    // x's row of a sorted row is order[row] / topk; NULL
  int64_t x_stride;        //   for the row itself
  int32_t topk;
  int32_t x_aligned;       // rows of x begin on 16-byte boundaries
  int64_t y_stride;
  int64_t rows;            // of b (and y)
  int64_t b_tiles;         // scale tiles of b, of kN rows or more
  int32_t groups;
  int32_t out;
  int32_t k;
  int32_t k_tiles;
  int32_t k_stages;
  int32_t m_tiles;
  int32_t m_pairs;         // of feature tiles
  int32_t activation;
  int32_t paired;          // bf16 y: 4-byte aligned pairs of features
  int32_t split;           // blocks of a cluster that share a tile's k
  int32_t stages;          // of the ring
  int32_t row_buffers;     // 1 or 2 buffers of quantised rows
  int32_t row_stages;      // stages of k that one holds
};

// ---------------------------------------------------------------- PTX forms

__device__ __forceinline__ uint32_t SharedAddress(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// True in one lane of a converged warp. The compiler knows it to be one, so
// the operands of what that lane issues stay in uniform registers (8192 x 8192
// x 8192: 394 us with a test of the lane's index, 256 us with this).
__device__ __forceinline__ bool Elect() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void BarrierInit(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)
               : "memory");
}

__device__ __forceinline__ void BarrierExpect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                   bar), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void BarrierArrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

__device__ __forceinline__ bool BarrierTry(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// False when the wait ran out, here or (as `failed` tells) in another role.
__device__ __forceinline__ bool BarrierWait(uint32_t bar, uint32_t parity,
                                            volatile int* failed) {
  if (BarrierTry(bar, parity)) return true;
  const long long begin = clock64();
  while (!BarrierTry(bar, parity)) {
    if (*failed) return false;
    if (clock64() - begin > kWaitCycles) {
      *failed = 1;
      g_wait_failed = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void TmaLoad3(uint32_t dst, const CUtensorMap* map,
                                         int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void TmaLoad2(uint32_t dst, const CUtensorMap* map,
                                         int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void BulkLoad(uint32_t dst, const void* src,
                                         uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void FenceAfterSync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void FenceBeforeSync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

// Arrives at `bar` once the MMAs and copies issued so far are done.
__device__ __forceinline__ void Commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 "
      "[%0];" ::"r"(bar)
      : "memory");
}

// 512 bytes of scales (32 rows of 16 bytes, in shared memory as 8-row groups
// of 128 bytes) to four columns, repeated for each warp's lanes.
__device__ __forceinline__ void CopyScales(uint32_t column, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(column),
               "l"(desc)
               : "memory");
}

__device__ __forceinline__ void Mma(uint32_t acc, uint64_t a, uint64_t b,
                                    uint32_t idesc, uint32_t a_scales,
                                    uint32_t b_scales, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X "
      "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"(a_scales), "r"(b_scales),
      "r"(accumulate ? 1u : 0u)
      : "memory");
}

// 16 columns of the calling warp's 32 lanes; complete after WaitLoads.
__device__ __forceinline__ void LoadColumns(uint32_t address, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, "
      "%8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
        "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(address)
      : "memory");
}

__device__ __forceinline__ void WaitLoads() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The forms of a pair of blocks (one on each SM of a pair): issued by its first
// block for both, arrivals in both.
__device__ __forceinline__ void CommitPair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
      "multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void CopyScalesPair(uint32_t column, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(column),
               "l"(desc)
               : "memory");
}
__device__ __forceinline__ void MmaPair(uint32_t acc, uint64_t a, uint64_t b,
                                        uint32_t idesc, uint32_t a_scales,
                                        uint32_t b_scales, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X "
      "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"(a_scales), "r"(b_scales),
      "r"(accumulate ? 1u : 0u)
      : "memory");
}

// Copies into this block's memory that count at a barrier of either block.
__device__ __forceinline__ void TmaLoad3Pair(uint32_t dst,
                                             const CUtensorMap* map, int x,
                                             int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void TmaLoad2Pair(uint32_t dst,
                                             const CUtensorMap* map, int x,
                                             int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::"
      "complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t AddressAt(uint32_t address, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"(address), "r"(rank));
  return at;
}

// Arrives at the barrier at `bar` of block `rank` of the cluster.
__device__ __forceinline__ void BarrierArriveAt(uint32_t bar, int rank) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(
                   AddressAt(bar, rank))
               : "memory");
}

__device__ __forceinline__ void ClusterSync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float LoadPeer(uint32_t address, int rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(remote)
               : "r"(address), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote)
               : "memory");
  return v;
}

// Shared memory descriptors (addresses and strides in 16-byte units, version
// 1): K-major rows of 128 bytes with the 128-byte swizzle, 1024 bytes between
// groups of 8 rows; and unswizzled 8 x 16-byte groups, 128 bytes apart.
__device__ __forceinline__ uint64_t SwizzledDesc(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3fff) | (1ull << 16) |
         (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t ScaleDesc(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3fff) | (1ull << 16) |
         (8ull << 32) | (1ull << 46);
}

// Instruction descriptor of kind::mxf4: E2M1 x E2M1, E8M0 scales, K-major
// operands, dense; `half` selects the scale bytes 0-1 or 2-3 of a column.
template <int kN, int kRowsOfA = kM>
__device__ __forceinline__ uint32_t InstructionDesc(uint32_t half) {
  const uint32_t id = half * 2;
  return (id << 4) | (1u << 7) | (1u << 10) |
         (static_cast<uint32_t>(kN / 8) << 17) | (1u << 23) |
         (static_cast<uint32_t>(kRowsOfA / 16) << 24) | (id << 29);
}

// -------------------------------------------------------------------- tiles

struct Tile {
  int group;       // weights' group
  int64_t row;     // first row of b and y
  int rows;        // of the tile that exist
  int m;           // feature tile
  int64_t b_tile;  // first scale tile of b
};

// Groups' first row tiles (a running count) and rows in shared memory.
template <int kN>
__device__ __forceinline__ Tile TileOf(const GemmParams& p, int m_tiles,
                                       int item, const int* tile_begin,
                                       const int* row_begin) {
  Tile t;
  const int n = item / m_tiles;
  t.m = item - n * m_tiles;
  t.group = 0;
  int64_t at = n;
  int64_t first = 0, count = p.rows;
  if (p.offsets != nullptr) {
    int low = 0, high = p.groups - 1;  // the last group that begins by n
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (tile_begin[mid] <= n) {
        low = mid;
      } else {
        high = mid - 1;
      }
    }
    t.group = low;
    at = n - tile_begin[low];
    first = row_begin[low];
    count = row_begin[low + 1] - first;
  }
  t.row = first + at * kN;
  const int64_t left = count - at * kN;
  t.rows = static_cast<int>(left < kN ? left : kN);
  // ExpertScaleTiles; with one group a tile of rows' own. A tile of 256 rows
  // has two scale tiles.
  t.b_tile = (first / kN + t.group + at) * (kN > kMxTileRows ? 2 : 1);
  return t;
}

// The plan's offsets, held to [0, rows], and a scan of the row tiles; called by
// the whole block, which meets once more before it reads them.
template <int kN>
__device__ __forceinline__ void ScanOffsets(const GemmParams& p, int warp,
                                            int lane, int* tile_begin,
                                            int* row_begin) {
  // Nothing before this touches global memory: this block may have begun under
  // the end of the launch before.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.offsets == nullptr) return;
  if (warp >= 2) {
    for (int i = threadIdx.x - 64; i <= p.groups; i += blockDim.x - 64) {
      row_begin[i] =
          min(max(__ldg(p.offsets + i), 0), static_cast<int>(p.rows));
    }
  }
  __syncthreads();
  if (warp != 2) return;
  int carry = 0;
  for (int base = 0; base <= p.groups; base += 32) {
    const int i = base + lane;
    const int count = i < p.groups ? row_begin[i + 1] - row_begin[i] : 0;
    const int tiles = count > 0 ? (count + kN - 1) / kN : 0;
    int scan = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (i <= p.groups) tile_begin[i] = carry + scan - tiles;
    carry += __shfl_sync(0xffffffffu, scan, 31);
  }
}

// After a failure the copies in flight still have to land: waits (bounded) for
// the last ones issued before `stage` of `phase`.
__device__ __forceinline__ void DrainStages(uint64_t* full_bar, int stage,
                                            uint32_t phase, int64_t issued,
                                            int stages) {
  volatile int ignored = 0;
  for (int64_t i = 0; i < issued && i < stages; ++i) {
    if (--stage < 0) {
      stage = stages - 1;
      phase ^= 1;
    }
    if (!BarrierWait(SharedAddress(full_bar + stage), phase, &ignored)) break;
  }
}

__device__ __forceinline__ float Activate(float v, int activation) {
  if (activation == XSE_ACT_RELU) return v < 0.0f ? 0.0f : v;  // keeps NaN
  if (activation == XSE_ACT_SIGMOID) return 1.0f / (1.0f + expf(-v));
  return v;
}

__device__ __forceinline__ void Store(float* p, float v) { *p = v; }
__device__ __forceinline__ void Store(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// 16 rows of y from the lane's accumulator columns: lane l holds feature l of
// every row. `y` points at the first row's element of this lane; `rows` of the
// 16 exist; `mine`: the feature does.
template <typename T>
__device__ __forceinline__ void StoreRows(T* y, int64_t stride,
                                          const uint32_t* r, float bias,
                                          int activation, int rows, bool mine,
                                          bool paired, int lane) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) + bias;
  if (activation == XSE_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
  } else if (activation == XSE_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = Activate(v[i], XSE_ACT_SIGMOID);
  }
  const bool whole = __all_sync(0xffffffffu, mine) && rows >= 16;
  if constexpr (sizeof(T) == 2) {
    // Two features a store: even lanes take the even rows of a pair of lanes,
    // odd lanes the odd ones. All exchanges come before the first store.
    if (paired) {
      const bool odd = lane & 1;
      uint32_t pair[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float got =
            __shfl_xor_sync(0xffffffffu, odd ? v[2 * i] : v[2 * i + 1], 1);
        const __nv_bfloat162 b = __floats2bfloat162_rn(
            odd ? got : v[2 * i], odd ? v[2 * i + 1] : got);
        __builtin_memcpy(&pair[i], &b, 4);
      }
      y += odd ? stride - 1 : 0;
      rows -= odd ? 1 : 0;
      if (whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          *reinterpret_cast<uint32_t*>(y) = pair[i];
          y += 2 * stride;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (mine && 2 * i < rows) *reinterpret_cast<uint32_t*>(y) = pair[i];
          y += 2 * stride;
        }
      }
      return;
    }
  }
  if (whole) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      Store(y, v[i]);
      y += stride;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (mine && i < rows) Store(y, v[i]);
      y += stride;
    }
  }
}

// Zeros in the rows behind the last group's, by the epilogue's warps.
template <typename T>
__device__ __forceinline__ void ZeroRowsBehind(const GemmParams& p,
                                               const int* row_begin) {
  if (p.offsets == nullptr) return;
  const int64_t kept = row_begin[p.groups];
  const int64_t total = (p.rows - kept) * p.out;
  constexpr int kStep = 32 * kEpilogueWarps;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kStep + threadIdx.x - 64;
       i < total; i += static_cast<int64_t>(gridDim.x) * kStep) {
    const int64_t r = i / p.out;
    Store(static_cast<T*>(p.y) + (kept + r) * p.y_stride + (i - r * p.out),
          0.0f);
  }
}

// The 32 elements of a block of x in registers.
template <typename X>
struct XBlock {
  static constexpr int kWords = 8 * sizeof(X);
  uint4 v[kWords / 4];

  // Elements [col, col + 32) of the row at x, zeros from cols on.
  __device__ void Load(const X* x, int col, int cols, bool aligned) {
    if (aligned && col + 32 <= cols) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        v[i] = __ldg(reinterpret_cast<const uint4*>(x + col) + i);
      }
    } else {
      uint32_t* w = &v[0].x;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const X e = col + i < cols ? x[col + i] : static_cast<X>(0.0f);
        if constexpr (sizeof(X) == 2) {
          const uint32_t bits = __bfloat16_as_ushort(e);
          w[i / 2] = i % 2 ? w[i / 2] | bits << 16 : bits;
        } else {
          w[i] = __float_as_uint(e);
        }
      }
    }
  }
};

// One lane's block of a row tile's buffer: `block` counts 32 columns from the
// first stage of this block's part of k.
template <int kN, typename X>
__device__ __forceinline__ void StoreBlock(uint8_t* buffer, int row, int block,
                                           const XBlock<X>& x) {
  using C = Config<kN>;
  const uint32_t* w = &x.v[0].x;
  const uint32_t s = MxScaleByte(MxLargest<X, XBlock<X>::kWords>(w));
  uint4 c;
  MxEncode<X, 4>(w, s, &c.x);
  uint8_t* codes = buffer + (block >> 3) * C::kRowStageBytes;
  const int b = block & 7;
  // The 128-byte swizzle: 16-byte piece b of row r at b ^ (r % 8).
  *reinterpret_cast<uint4*>(codes + row * 128 + ((b ^ (row & 7)) * 16)) = c;
  codes[C::kBBytes + (b >> 2) * kMxTileBytes + row * 16 + (b & 3)] =
      static_cast<uint8_t>(s);
}

// The row tiles of this block's items, quantised one after another.
template <int kN, typename X>
__device__ __forceinline__ void QuantizeTiles(
    const GemmParams& p, int thread, int first_item, int last_item,
    int k_begin, int k_end, const int* tile_begin, const int* row_begin,
    uint8_t* buffers, uint64_t* rows_full_bar, uint64_t* rows_empty_bar,
    volatile int* failed) {
  using C = Config<kN>;
  constexpr int kQuantizeThreads = 32 * kQuantizeWarps;
  const int blocks = (k_end - k_begin) * 8;
  int buffer = 0;
  uint32_t phase = 0;
  for (int item = first_item; item < last_item;
       item = (item / p.m_tiles + 1) * p.m_tiles) {
    const Tile t = TileOf<kN>(p, p.m_tiles, item, tile_begin, row_begin);
    const bool ok = BarrierWait(SharedAddress(rows_empty_bar + buffer),
                                phase ^ 1, failed);
    if (!__all_sync(0xffffffffu, ok)) break;
    uint8_t* to = buffers + buffer * p.row_stages * C::kRowStageBytes;
    const int total = t.rows * blocks;
    const auto load = [&](int i, XBlock<X>& x) {
      const int row = i / blocks, block = i - row * blocks;
      int64_t r = t.row + row;
      if (p.order != nullptr) {
        const int pair = __ldg(p.order + r);
        r = pair < 0 || pair >= p.rows ? 0 : pair / p.topk;
      }
      x.Load(static_cast<const X*>(p.x) + r * p.x_stride,
             k_begin * kStageK + block * 32, p.k, p.x_aligned);
    };
    constexpr int kAtOnce = sizeof(X) == 2 ? 2 : 1;  // registers hold so many
    for (int i = thread; i < total; i += kAtOnce * kQuantizeThreads) {
      XBlock<X> x[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (i + j * kQuantizeThreads < total) load(i + j * kQuantizeThreads, x[j]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int at = i + j * kQuantizeThreads;
        if (at < total) StoreBlock<kN, X>(to, at / blocks, at % blocks, x[j]);
      }
    }
    // Generic stores, read by the MMA's proxy.
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((thread & 31) == 0) BarrierArrive(SharedAddress(rows_full_bar + buffer));
    if (++buffer == p.row_buffers) {
      buffer = 0;
      phase ^= 1;
    }
  }
}

// X: the type of rows that the kernel quantises itself, void where they come
// as codes and scales.
template <int kN, typename T, typename X>
__global__ void
__launch_bounds__(std::is_void_v<X> ? kThreads : kThreadsWithRows, 1)
    MxGemmKernel(const __grid_constant__ GemmParams p) {
  using C = Config<kN>;
  constexpr bool kRows = !std::is_void_v<X>;
  extern __shared__ uint8_t raw[];
  // Stages' bytes; with rows quantised here, the host gives the ring what the
  // rows' buffers leave.
  constexpr int kStageBytes = kRows ? C::kWeightStageBytes : C::kStageBytes;
  const int num_stages = kRows ? p.stages : C::kStages;
  __shared__ alignas(8) uint64_t full_bar[kMostStages];
  __shared__ alignas(8) uint64_t empty_bar[kMostStages];
  __shared__ alignas(8) uint64_t rows_full_bar[2];
  __shared__ alignas(8) uint64_t rows_empty_bar[2];
  __shared__ alignas(8) uint64_t acc_full_bar[2];
  __shared__ alignas(8) uint64_t acc_empty_bar[2];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int failed;

  uint8_t* stages = raw + (1024 - (SharedAddress(raw) & 1023)) % 1024;
  uint8_t* row_buffers = stages + num_stages * kStageBytes;
  int* tile_begin = reinterpret_cast<int*>(
      row_buffers +
      (kRows ? p.row_buffers * p.row_stages * C::kRowStageBytes : 0));
  int* row_begin = tile_begin + (p.groups + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split;

  if (threadIdx.x == 0) {
    for (int i = 0; i < num_stages; ++i) {
      BarrierInit(SharedAddress(full_bar + i), 1);
      BarrierInit(SharedAddress(empty_bar + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      BarrierInit(SharedAddress(rows_full_bar + i), kQuantizeWarps);
      BarrierInit(SharedAddress(rows_empty_bar + i), 1);
      BarrierInit(SharedAddress(acc_full_bar + i), 1);
      BarrierInit(SharedAddress(acc_empty_bar + i), kEpilogueWarps);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
        ::"r"(SharedAddress(&tmem_base))
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;"
                 ::: "memory");
  }
  if (warp == 0 && Elect()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.a) : "memory");
    if constexpr (!kRows) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&p.b) : "memory");
    }
  }
  ScanOffsets<kN>(p, warp, lane, tile_begin, row_begin);
  FenceBeforeSync();
  __syncthreads();
  FenceAfterSync();
  const uint32_t tmem = tmem_base;
  // Fewer than 2^31: y would not fit the memory otherwise.
  const int row_tiles = p.offsets != nullptr
                            ? tile_begin[p.groups]
                            : static_cast<int>((p.rows + kN - 1) / kN);
  const int items = row_tiles * p.m_tiles;
  // A block's (a cluster's) items: every item_step-th, or, where it quantises
  // their rows, neighbouring ones.
  const int sharers = gridDim.x / p.split, sharer = blockIdx.x / p.split;
  int first_item = sharer, last_item = items, item_step = sharers;
  if constexpr (kRows) {
    const int each = items / sharers, more = items % sharers;
    first_item = each * sharer + min(sharer, more);
    last_item = first_item + each + (sharer < more ? 1 : 0);
    item_step = 1;
  }
  // This block's part of k, in stages.
  const int k_begin = p.k_stages * rank / p.split;
  const int k_end = p.k_stages * (rank + 1) / p.split;
  const uint32_t stage_base = SharedAddress(stages);

  if (warp == 0) {
    // The whole warp follows the loop; one lane issues.
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int64_t issued = 0;
    for (int item = first_item; ok && item < last_item;
         item += item_step) {
      const Tile t = TileOf<kN>(p, p.m_tiles, item, tile_begin, row_begin);
      const uint8_t* a_scales =
          p.a_scales + (static_cast<int64_t>(t.group) * p.m_tiles + t.m) *
                           p.k_tiles * kMxTileBytes;
      const uint8_t* b_scales =
          p.b_scales + t.b_tile * p.k_tiles * kMxTileBytes;
      const bool b_there = !kRows && t.b_tile < p.b_tiles;
      for (int s = k_begin; s < k_end; ++s) {
        ok = BarrierWait(SharedAddress(empty_bar + stage), phase ^ 1, &failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (Elect()) {
          const uint32_t bar = SharedAddress(full_bar + stage);
          const uint32_t at = stage_base + stage * kStageBytes;
          const uint32_t scales = at + kABytes + (kRows ? 0 : C::kBBytes);
          const uint32_t bytes =
              2 * s + 1 < p.k_tiles ? kScaleBytes : kMxTileBytes;
          BarrierExpect(bar, kABytes + (kRows ? 0 : C::kBBytes) +
                                 bytes * (1 + b_there));
          TmaLoad3(at, &p.a, s * (kStageK / 2), t.m * kM, t.group, bar);
          if constexpr (!kRows) {
            TmaLoad2(at + kABytes, &p.b, s * (kStageK / 2),
                     static_cast<int>(t.row), bar);
          }
          const int64_t k_at = static_cast<int64_t>(2 * s) * kMxTileBytes;
          BulkLoad(scales, a_scales + k_at, bytes, bar);
          if (b_there) {
            BulkLoad(scales + kScaleBytes, b_scales + k_at, bytes, bar);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == num_stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) DrainStages(full_bar, stage, phase, issued, num_stages);
  } else if (warp == 1) {
    int stage = 0, acc = 0, rows = 0;
    uint32_t phase = 0, acc_phase = 0, rows_phase = 0;
    bool new_rows = true, ok = true;
    for (int item = first_item; ok && item < last_item;
         item += item_step) {
      ok = BarrierWait(SharedAddress(acc_empty_bar + acc), acc_phase ^ 1,
                       &failed);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (kRows && new_rows) {
        ok = BarrierWait(SharedAddress(rows_full_bar + rows), rows_phase,
                         &failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      const uint32_t d = tmem + acc * C::kAccColumns;
      for (int s = k_begin; s < k_end; ++s) {
        ok = BarrierWait(SharedAddress(full_bar + stage), phase, &failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        FenceAfterSync();
        if (Elect()) {
          const uint32_t at = stage_base + stage * kStageBytes;
          const uint32_t b_at =
              kRows ? SharedAddress(row_buffers) +
                          (rows * p.row_stages + s - k_begin) *
                              C::kRowStageBytes
                    : at + kABytes;
          // The stage's own columns: they are free once its last MMAs are
          // done, which the stage's empty barrier has shown.
          const uint32_t a_col =
              tmem + C::kAccs * C::kAccColumns + stage * C::kScaleColumns;
          const uint32_t b_col = a_col + 8;
          const uint64_t a_desc = SwizzledDesc(at);
          const uint64_t b_desc = SwizzledDesc(b_at);
          const uint64_t a_scales =
              ScaleDesc(at + kABytes + (kRows ? 0 : C::kBBytes));
          const uint64_t b_scales =
              kRows ? ScaleDesc(b_at + C::kBBytes)
                    : a_scales + kScaleBytes / 16;
          const int left = p.k - s * kStageK;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h * 128 >= left) break;
            // Descriptors count 16 bytes.
            CopyScales(a_col + h * 4, a_scales + h * (kMxTileBytes / 16));
            CopyScales(b_col + h * 4, b_scales + h * (kMxTileBytes / 16));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j * 64 >= left) break;
            Mma(d, a_desc + j * 2, b_desc + j * 2, InstructionDesc<kN>(j & 1),
                a_col + (j >> 1) * 4, b_col + (j >> 1) * 4,
                s > k_begin || j > 0);
          }
          Commit(SharedAddress(empty_bar + stage));
        }
        __syncwarp();
        if (++stage == num_stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      // The last item of a row tile gives its buffer back.
      const int then = item + item_step;
      new_rows = kRows &&
                 (then >= last_item || then / p.m_tiles != item / p.m_tiles);
      if (Elect()) {
        Commit(SharedAddress(acc_full_bar + acc));
        if (new_rows) Commit(SharedAddress(rows_empty_bar + rows));
      }
      __syncwarp();
      if (new_rows && ++rows == p.row_buffers) {
        rows = 0;
        rows_phase ^= 1;
      }
      if (++acc == C::kAccs) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else if (kRows && warp >= 2 + kEpilogueWarps) {
    if constexpr (kRows) {
      QuantizeTiles<kN, X>(p, threadIdx.x - kThreads, first_item, last_item,
                           k_begin, k_end, tile_begin, row_begin, row_buffers,
                           rows_full_bar, rows_empty_bar, &failed);
    }
  } else {
    // Tensor memory lanes [32 q, 32 q + 32) belong to warps with warp % 4 = q.
    // A warp takes its columns into registers and gives the accumulator back
    // before it stores them, so that the next tile's MMAs wait for the reads
    // alone.
    const int quarter = warp & 3;
    const int first_column = (warp - 2) / 4 * C::kPart;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int item = first_item; item < last_item; item += item_step) {
      const Tile t = TileOf<kN>(p, p.m_tiles, item, tile_begin, row_begin);
      const int feature = t.m * kM + quarter * 32 + lane;
      const bool mine = feature < p.out;
      const float bias =
          p.bias != nullptr && mine
              ? __ldg(p.bias + static_cast<int64_t>(t.group) * p.out + feature)
              : 0.0f;
      const bool ok = BarrierWait(SharedAddress(acc_full_bar + acc), acc_phase,
                                  &failed);
      if (!__all_sync(0xffffffffu, ok)) break;
      FenceAfterSync();
      const uint32_t d = tmem + acc * C::kAccColumns + first_column +
                         (static_cast<uint32_t>(quarter * 32) << 16);
      const bool some = first_column < kN && first_column < t.rows;
      uint32_t r[C::kPart];
      if (some) {
#pragma unroll
        for (int c = 0; c < C::kPart; c += 16) LoadColumns(d + c, r + c);
        WaitLoads();
      }
      FenceBeforeSync();
      __syncwarp();
      if (lane == 0) BarrierArrive(SharedAddress(acc_empty_bar + acc));
      if (++acc == C::kAccs) {
        acc = 0;
        acc_phase ^= 1;
      }
      if (!some) continue;
      if (p.split == 1) {
        T* y = static_cast<T*>(p.y) +
               (t.row + first_column) * p.y_stride + feature;
        const int rows = t.rows - first_column;
#pragma unroll
        for (int c = 0; c < C::kPart; c += 16) {
          if (c >= rows) break;
          StoreRows(y + c * p.y_stride, p.y_stride, r + c, bias, p.activation,
                    rows - c, mine, p.paired, lane);
        }
      } else {
        // This block's part, [column][feature], over the stages (all read).
        float* part = reinterpret_cast<float*>(stages) + first_column * kM +
                      quarter * 32 + lane;
#pragma unroll
        for (int c = 0; c < C::kPart; ++c) {
          part[c * kM] = k_end > k_begin ? __uint_as_float(r[c]) : 0.0f;
        }
      }
    }
    ZeroRowsBehind<T>(p, row_begin);
  }
  if (p.split > 1) {
    // One tile per cluster; all its blocks come here, also without a tile.
    __syncwarp();
    ClusterSync();
    if (warp >= 2 && warp < 2 + kEpilogueWarps && first_item < last_item &&
        !failed) {
      const Tile t = TileOf<kN>(p, p.m_tiles, first_item, tile_begin, row_begin);
      const int lane_feature = (warp & 3) * 32 + lane;
      const int feature = t.m * kM + lane_feature;
      const float bias =
          p.bias != nullptr && feature < p.out
              ? __ldg(p.bias + static_cast<int64_t>(t.group) * p.out + feature)
              : 0.0f;
      for (int c = rank * 2 + (warp - 2) / 4; c < t.rows; c += 2 * p.split) {
        const uint32_t at = stage_base + (c * kM + lane_feature) * 4;
        float sum = 0.0f;
        for (int b = 0; b < p.split; ++b) sum += LoadPeer(at, b);
        if (feature < p.out) {
          Store(static_cast<T*>(p.y) + (t.row + c) * p.y_stride + feature,
                Activate(sum + bias, p.activation));
        }
      }
    }
    __syncwarp();
    ClusterSync();
  }
  __syncwarp();
  FenceBeforeSync();
  __syncthreads();
  if (warp == 1) {
    FenceAfterSync();
    asm volatile(
        "tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem)
        : "memory");
  }
}

// ------------------------------------------------------------ pairs of blocks

// Many rows: the blocks of a pair of SMs share tiles of 256 features x 256
// rows. Each holds the weights of its 128 features and half of the rows, and
// the pair's MMAs (issued by its first block) read both halves. An SM takes in
// 64 bytes a cycle from L2 and moves 128 through its shared memory, and both
// bound the products: the pair's 35 KB a stage need 560 cycles against its
// MMAs' 512, a block by itself 51 KB for 128 x 256 (8192 x 4096 -> 8192 under the
// power cap: 114 us, in pairs 104 us; off it, at 1.9 GHz, the pairs take 93 us).
// Every block has its own accumulator, scales and epilogue.
struct Pair {
  static constexpr int kN = 256;
  static constexpr int kBBytes = kN / 2 * kStageK / 2;
  static constexpr int kStageBytes = kABytes + kBBytes + 3 * kScaleBytes;
  static constexpr int kStages = (217 * 1024) / kStageBytes;
  // Tensor memory: the accumulator, then the scales of every stage, free once
  // its last MMAs are done, which the stage's empty barrier has shown.
  static constexpr int kScaleColumns = 24;
  static_assert(kN + kStages * kScaleColumns <= 512, "tensor memory");
  static constexpr int kPart = kN / 2;
  // A tile's MMAs take 128 rows where no more exist: a group's last tile.
  __device__ static int RowsFor(const Tile& t) {
    return t.rows <= kN / 2 ? kN / 2 : kN;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    MxPairKernel(const __grid_constant__ GemmParams p) {
  using C = Pair;
  constexpr int kN = C::kN;
  extern __shared__ uint8_t raw[];
  __shared__ alignas(8) uint64_t full_bar[C::kStages];
  __shared__ alignas(8) uint64_t empty_bar[C::kStages];
  __shared__ alignas(8) uint64_t acc_full_bar;
  __shared__ alignas(8) uint64_t acc_empty_bar;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int failed;

  uint8_t* stages = raw + (1024 - (SharedAddress(raw) & 1023)) % 1024;
  int* tile_begin =
      reinterpret_cast<int*>(stages + C::kStages * C::kStageBytes);
  int* row_begin = tile_begin + (p.groups + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      BarrierInit(SharedAddress(full_bar + i), 1);
      BarrierInit(SharedAddress(empty_bar + i), 1);
    }
    BarrierInit(SharedAddress(&acc_full_bar), 1);
    BarrierInit(SharedAddress(&acc_empty_bar), 2 * kEpilogueWarps);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0 && Elect()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.b) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.a_scale_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.b_scale_map) : "memory");
  }
  ScanOffsets<kN>(p, warp, lane, tile_begin, row_begin);
  // Both blocks' barriers are there before either's copies, and both blocks
  // before the pair's allocation.
  __syncwarp();
  ClusterSync();
  if (warp == 1) {
    asm volatile(
        "tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;"
        ::"r"(SharedAddress(&tmem_base))
        : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;"
                 ::: "memory");
  }
  FenceBeforeSync();
  __syncthreads();
  FenceAfterSync();
  __syncwarp();
  ClusterSync();  // both blocks' tensor memory is there
  const uint32_t tmem = tmem_base;
  const int row_tiles = p.offsets != nullptr
                            ? tile_begin[p.groups]
                            : static_cast<int>((p.rows + kN - 1) / kN);
  const int items = row_tiles * p.m_pairs;
  const int first_item = blockIdx.x / 2, item_step = gridDim.x / 2;
  const uint32_t stage_base = SharedAddress(stages);

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int64_t issued = 0;
    for (int item = first_item; ok && item < items; item += item_step) {
      const Tile t = TileOf<kN>(p, p.m_pairs, item, tile_begin, row_begin);
      // A pair's second block may lie behind the last features (its codes then
      // read as zeros, its scales are some other tile's), and a tile's second
      // scales behind the last ones: no result depends on them.
      const int m = t.m * 2 + rank;
      const int a_tile = (t.group * p.m_tiles + m) * p.k_tiles;
      const int b_tile = static_cast<int>(t.b_tile) * p.k_tiles;
      for (int s = 0; s < p.k_stages; ++s) {
        ok = BarrierWait(SharedAddress(empty_bar + stage), phase ^ 1, &failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (Elect()) {
          // All copies of both blocks count at the first block's barrier.
          const uint32_t bar = AddressAt(SharedAddress(full_bar + stage), 0);
          const uint32_t at = stage_base + stage * C::kStageBytes;
          const uint32_t scales = at + kABytes + C::kBBytes;
          if (rank == 0) {
            BarrierExpect(SharedAddress(full_bar + stage),
                          2 * C::kStageBytes);
          }
          TmaLoad3Pair(at, &p.a, s * (kStageK / 2), m * kM, t.group, bar);
          TmaLoad2Pair(at + kABytes, &p.b, s * (kStageK / 2),
                       static_cast<int>(t.row) + rank * (C::RowsFor(t) / 2),
                       bar);
          TmaLoad2Pair(scales, &p.a_scale_map, 0, a_tile + 2 * s, bar);
          TmaLoad2Pair(scales + kScaleBytes, &p.b_scale_map, 0, b_tile + 2 * s,
                       bar);
          TmaLoad2Pair(scales + 2 * kScaleBytes, &p.b_scale_map, 0,
                       b_tile + p.k_tiles + 2 * s, bar);
        }
        __syncwarp();
        ++issued;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && rank == 0) {
      DrainStages(full_bar, stage, phase, issued, C::kStages);
    }
  } else if (warp == 1 && rank == 0) {
    int stage = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int item = first_item; ok && item < items; item += item_step) {
      const bool half_rows =
          C::RowsFor(TileOf<kN>(p, p.m_pairs, item, tile_begin, row_begin)) <
          kN;
      ok = BarrierWait(SharedAddress(&acc_empty_bar), acc_phase ^ 1, &failed);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      for (int s = 0; s < p.k_stages; ++s) {
        ok = BarrierWait(SharedAddress(full_bar + stage), phase, &failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        FenceAfterSync();
        if (Elect()) {
          const uint32_t at = stage_base + stage * C::kStageBytes;
          const uint32_t a_col = tmem + kN + stage * C::kScaleColumns;
          const uint32_t b_col = a_col + 8;
          const uint64_t a_desc = SwizzledDesc(at);
          const uint64_t b_desc = SwizzledDesc(at + kABytes);
          const uint64_t scales = ScaleDesc(at + kABytes + C::kBBytes);
          const int left = p.k - s * kStageK;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h * 128 >= left) break;
            const uint64_t half = scales + h * (kMxTileBytes / 16);
            CopyScalesPair(a_col + h * 4, half);
            CopyScalesPair(b_col + h * 8, half + kScaleBytes / 16);
            CopyScalesPair(b_col + h * 8 + 4, half + 2 * kScaleBytes / 16);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j * 64 >= left) break;
            MmaPair(tmem, a_desc + j * 2, b_desc + j * 2,
                    half_rows ? InstructionDesc<kN / 2, 2 * kM>(j & 1)
                              : InstructionDesc<kN, 2 * kM>(j & 1),
                    a_col + (j >> 1) * 4, b_col + (j >> 1) * 8,
                    s > 0 || j > 0);
          }
          CommitPair(SharedAddress(empty_bar + stage));
        }
        __syncwarp();
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      if (Elect()) CommitPair(SharedAddress(&acc_full_bar));
      __syncwarp();
      acc_phase ^= 1;
    }
  } else if (warp >= 2) {
    const int quarter = warp & 3;
    const int first_column = (warp - 2) / 4 * C::kPart;
    uint32_t acc_phase = 0;
    for (int item = first_item; item < items; item += item_step) {
      const Tile t = TileOf<kN>(p, p.m_pairs, item, tile_begin, row_begin);
      const int feature = (t.m * 2 + rank) * kM + quarter * 32 + lane;
      const bool mine = feature < p.out;
      const float bias =
          p.bias != nullptr && mine
              ? __ldg(p.bias + static_cast<int64_t>(t.group) * p.out + feature)
              : 0.0f;
      const bool ok =
          BarrierWait(SharedAddress(&acc_full_bar), acc_phase, &failed);
      if (!__all_sync(0xffffffffu, ok)) break;
      FenceAfterSync();
      const uint32_t d = tmem + first_column +
                         (static_cast<uint32_t>(quarter * 32) << 16);
      const bool some = first_column < t.rows;
      uint32_t r[C::kPart];
      if (some) {
#pragma unroll
        for (int c = 0; c < C::kPart; c += 16) LoadColumns(d + c, r + c);
        WaitLoads();
      }
      FenceBeforeSync();
      __syncwarp();
      if (lane == 0) BarrierArriveAt(SharedAddress(&acc_empty_bar), 0);
      acc_phase ^= 1;
      if (!some) continue;
      T* y = static_cast<T*>(p.y) + (t.row + first_column) * p.y_stride +
             feature;
      const int rows = t.rows - first_column;
#pragma unroll
      for (int c = 0; c < C::kPart; c += 16) {
        if (c >= rows) break;
        StoreRows(y + c * p.y_stride, p.y_stride, r + c, bias, p.activation,
                  rows - c, mine, p.paired, lane);
      }
    }
    ZeroRowsBehind<T>(p, row_begin);
  }
  // Neither block ends while the other may still arrive at its barriers or
  // read its stages.
  __syncwarp();
  FenceBeforeSync();
  ClusterSync();
  if (warp == 1) {
    FenceAfterSync();
    asm volatile(
        "tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem)
        : "memory");
  }
}

// ------------------------------------------------------------------- launch

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t,
                                 void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

EncodeTiled GetEncodeTiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                         cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

int Encode(CUtensorMap* map, CUtensorMapDataType type, const void* base,
           int rank, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiled encode = GetEncodeTiled();
  if (encode == nullptr) {
    return FailWith(XSE_INTERNAL, "cuTensorMapEncodeTiled is not available");
  }
  const cuuint32_t steps[3] = {1, 1, 1};
  const CUresult r = encode(map, type, rank, const_cast<void*>(base), dims,
                            strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return FailWith(XSE_INTERNAL, "tensor map of a 4-bit matrix: error %d",
                    static_cast<int>(r));
  }
  return XSE_OK;
}

// [groups][rows][row bytes] of codes as boxes of 128 bytes x `box_rows`,
// swizzled; parts of a box outside the matrix read as zero codes.
int EncodeCodes(CUtensorMap* map, const void* codes, int64_t row_bytes,
                int64_t rows, int64_t groups, int rank, int box_rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(row_bytes),
                              static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(groups)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_bytes),
                                 static_cast<cuuint64_t>(row_bytes * rows)};
  const cuuint32_t box[3] = {kStageK / 2, static_cast<cuuint32_t>(box_rows),
                             1};
  return Encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, rank, dims, strides,
                box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scale tiles as rows of 128 words, in boxes of a stage's two.
int EncodeScales(CUtensorMap* map, const void* scales, int64_t tiles) {
  const cuuint64_t dims[2] = {kMxTileBytes / 4,
                              static_cast<cuuint64_t>(tiles)};
  const cuuint64_t strides[1] = {kMxTileBytes};
  const cuuint32_t box[2] = {kMxTileBytes / 4, 2};
  return Encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, 2, dims, strides,
                box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// A launch in clusters of `cluster` blocks that may begin under the end of the
// one before (the kernels wait for that before they touch memory: 64 tokens' 4
// choices of 64 experts 21.2 -> 18.8 us a call).
void SetAttributes(cudaLaunchAttribute* attrs, unsigned cluster,
                   cudaLaunchConfig_t* cfg) {
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = cluster;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attrs;
  cfg->numAttrs = 2;
}

template <int kN, typename T, typename X>
int LaunchGemmAs(GemmParams& p, const void* a_codes, const void* b_codes,
                 int64_t most_items, cudaStream_t s) {
  using C = Config<kN>;
  const int64_t row_bytes = MxRowBytes(p.k);
  int rc = EncodeCodes(&p.a, a_codes, row_bytes, p.out, p.groups, 3, kM);
  if (rc == XSE_OK && std::is_void_v<X>) {
    rc = EncodeCodes(&p.b, b_codes, row_bytes, p.rows, 1, 2, kN);
  }
  if (rc != XSE_OK) return rc;
  size_t shared = C::kStages * C::kStageBytes;
  if constexpr (!std::is_void_v<X>) {
    p.row_stages = (p.k_stages + p.split - 1) / p.split;
    const int rows = p.row_stages * C::kRowStageBytes;
    p.row_buffers = 2 * rows <= kRowBufferBytes ? 2 : 1;
    p.stages = (kSharedBytes - p.row_buffers * rows) / C::kWeightStageBytes;
    if (p.stages > kMostStages) p.stages = kMostStages;
    shared = p.stages * C::kWeightStageBytes + p.row_buffers * rows;
  }
  const size_t smem =
      1024 + shared + (p.offsets != nullptr ? 8 * (p.groups + 1) : 0);
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e =
      AllowShared(MxGemmKernel<kN, T, X>,
                  1024 + kSharedBytes + 8 * (XSE_MAX_EXPERTS + 1), &allowed);
  if (e == cudaSuccess) {
    int64_t blocks = most_items * p.split;
    if (p.split == 1 && blocks > kNumSms) blocks = kNumSms;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(std::is_void_v<X> ? kThreads : kThreadsWithRows);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2] = {};
    SetAttributes(attrs, static_cast<unsigned>(p.split), &cfg);
    e = cudaLaunchKernelEx(&cfg, MxGemmKernel<kN, T, X>, p);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return FailWith(XSE_INTERNAL, "4-bit product launch: %s",
                    cudaGetErrorString(e));
  }
  return XSE_OK;
}

// Many rows, by pairs of blocks.
template <typename T>
int LaunchPairAs(GemmParams& p, const void* a_codes, const void* b_codes,
                 int64_t row_tiles, cudaStream_t s) {
  const int64_t row_bytes = MxRowBytes(p.k);
  int rc = EncodeCodes(&p.a, a_codes, row_bytes, p.out, p.groups, 3, kM);
  if (rc == XSE_OK) {
    rc = EncodeCodes(&p.b, b_codes, row_bytes, p.rows, 1, 2, Pair::kN / 2);
  }
  if (rc == XSE_OK) {
    rc = EncodeScales(&p.a_scale_map, p.a_scales,
                      static_cast<int64_t>(p.groups) * p.m_tiles * p.k_tiles);
  }
  if (rc == XSE_OK) {
    rc = EncodeScales(&p.b_scale_map, p.b_scales, p.b_tiles * p.k_tiles);
  }
  if (rc != XSE_OK) return rc;
  p.m_pairs = (p.m_tiles + 1) / 2;
  constexpr size_t kFixed = 1024 + Pair::kStages * Pair::kStageBytes;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = AllowShared(MxPairKernel<T>,
                              kFixed + 8 * (XSE_MAX_EXPERTS + 1), &allowed);
  if (e == cudaSuccess) {
    const int64_t pairs = row_tiles * p.m_pairs;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(
        2 * (pairs > kNumSms / 2 ? kNumSms / 2 : pairs)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes =
        kFixed + (p.offsets != nullptr ? 8 * (p.groups + 1) : 0);
    cfg.stream = s;
    cudaLaunchAttribute attrs[2] = {};
    SetAttributes(attrs, 2, &cfg);
    e = cudaLaunchKernelEx(&cfg, MxPairKernel<T>, p);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return FailWith(XSE_INTERNAL, "4-bit product launch: %s",
                    cudaGetErrorString(e));
  }
  return XSE_OK;
}

// Rows that come quantised.
template <int kN>
int LaunchGemm(GemmParams& p, int32_t y_dtype, const void* a_codes,
               const void* b_codes, int64_t most_items, cudaStream_t s) {
  return y_dtype == XSE_DT_BF16
             ? LaunchGemmAs<kN, __nv_bfloat16, void>(p, a_codes, b_codes,
                                                     most_items, s)
             : LaunchGemmAs<kN, float, void>(p, a_codes, b_codes, most_items,
                                             s);
}

// Rows that the product quantises.
template <int kN, typename X>
int LaunchGemmOfRows(GemmParams& p, int32_t y_dtype, const void* a_codes,
                     int64_t most_items, cudaStream_t s) {
  return y_dtype == XSE_DT_BF16
             ? LaunchGemmAs<kN, __nv_bfloat16, X>(p, a_codes, nullptr,
                                                  most_items, s)
             : LaunchGemmAs<kN, float, X>(p, a_codes, nullptr, most_items, s);
}

// Rows of a product, quantised (codes, scales in tiles of its n rows) or not
// (x; plan's tokens' rows unless `sorted`).
struct Rows {
  const void* codes;
  const void* scales;
  int64_t scale_tiles;
  const void* x;
  int32_t x_dtype;
  int64_t x_stride;
  bool sorted;
};

// The product of `rows` rows with w in tiles of n rows; plan NULL: one group.
int RunGemm(const Rows& from, int64_t rows, const xse_mx_matrix& w,
            const float* bias, int32_t activation, const xse_expert_plan* plan,
            int n, void* y, int32_t y_dtype, int64_t y_stride,
            cudaStream_t s) {
  GemmParams p{};
  p.a_scales = static_cast<const uint8_t*>(w.scales);
  p.b_scales = static_cast<const uint8_t*>(from.scales);
  p.b_tiles = from.scale_tiles;
  p.x = from.x;
  p.x_stride = from.x_stride;
  p.x_aligned = Aligned16(from.x) &&
                from.x_stride % (from.x_dtype == XSE_DT_BF16 ? 8 : 4) == 0;
  p.bias = bias;
  p.y = y;
  p.offsets = plan != nullptr ? plan->offsets : nullptr;
  p.order = plan != nullptr && !from.sorted ? plan->order : nullptr;
  p.topk = plan != nullptr ? plan->topk : 1;
  p.y_stride = y_stride;
  p.rows = rows;
  p.groups = plan != nullptr ? plan->num_experts : 1;
  p.out = static_cast<int32_t>(w.rows);
  p.k = w.cols;
  p.k_tiles = static_cast<int32_t>(MxKTiles(w.cols));
  p.k_stages = (w.cols + kStageK - 1) / kStageK;
  p.m_tiles = static_cast<int32_t>(MxRowTiles(w.rows));
  p.activation = activation;
  p.paired = y_dtype == XSE_DT_BF16 &&
             (reinterpret_cast<uintptr_t>(y) & 3) == 0 && y_stride % 2 == 0 &&
             w.rows % 2 == 0;
  p.split = 1;
  const int64_t row_tiles =
      plan == nullptr ? (rows + n - 1) / n
                      : rows / n + (p.groups < rows ? p.groups : rows);
  const int64_t items = row_tiles * p.m_tiles;
  // A tile's k is shared where whole tiles would leave SMs idle.
  if (n <= 64) {
    while (p.split < 8 && items * p.split * 2 <= kNumSms &&
           p.split * 2 <= p.k_stages) {
      p.split *= 2;
    }
  }
  if (from.x != nullptr) {
    const bool half = from.x_dtype == XSE_DT_BF16;
    if (n == 16) {
      return half ? LaunchGemmOfRows<16, __nv_bfloat16>(p, y_dtype, w.codes,
                                                        items, s)
                  : LaunchGemmOfRows<16, float>(p, y_dtype, w.codes, items, s);
    }
    return half ? LaunchGemmOfRows<32, __nv_bfloat16>(p, y_dtype, w.codes,
                                                      items, s)
                : LaunchGemmOfRows<32, float>(p, y_dtype, w.codes, items, s);
  }
  switch (n) {
    case 16:
      return LaunchGemm<16>(p, y_dtype, w.codes, from.codes, items, s);
    case 32:
      return LaunchGemm<32>(p, y_dtype, w.codes, from.codes, items, s);
    case 64:
      return LaunchGemm<64>(p, y_dtype, w.codes, from.codes, items, s);
    case 128:
      return LaunchGemm<128>(p, y_dtype, w.codes, from.codes, items, s);
    default:
      return y_dtype == XSE_DT_BF16
                 ? LaunchPairAs<__nv_bfloat16>(p, w.codes, from.codes,
                                               row_tiles, s)
                 : LaunchPairAs<float>(p, w.codes, from.codes, row_tiles, s);
  }
}

int CheckLayer(const xse_mx_matrix* w, int32_t activation, int32_t y_dtype,
               int64_t y_stride) {
  if (int rc = CheckMxMatrix(w, "w"); rc != XSE_OK) return rc;
  if (w->rows < 1) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit matrix w needs at least one output row.");
  }
  if (activation < XSE_ACT_NONE || activation > XSE_ACT_SIGMOID) {
    return FailWith(XSE_INVALID_ARGUMENT, "Unknown activation: %d",
                    activation);
  }
  if (y_dtype != XSE_DT_F32 && y_dtype != XSE_DT_BF16) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layers write float32 or bfloat16, got type %d",
                    y_dtype);
  }
  if (y_stride < w->rows) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer needs an output row stride >= out.");
  }
  return XSE_OK;
}

int CheckRowsIn(const void* x, int32_t x_dtype, int64_t rows, int64_t x_stride,
                int32_t in_dim, const void* workspace, int64_t have,
                int64_t need) {
  if (x_dtype != XSE_DT_F32 && x_dtype != XSE_DT_BF16) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layers read float32 or bfloat16, got type %d",
                    x_dtype);
  }
  if (rows < 0 || rows > INT32_MAX || x_stride < in_dim) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer needs 0 <= rows < 2^31 and an input row "
                    "stride >= in.");
  }
  if (rows > 0 && (x == nullptr || (need > 0 && workspace == nullptr))) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer buffers must be non-null.");
  }
  if (rows > 0 && (have < need || !Aligned16(workspace))) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer needs a 16-byte aligned workspace of %lld "
                    "bytes, got %lld.", static_cast<long long>(need),
                    static_cast<long long>(have));
  }
  return XSE_OK;
}

// A layer over `x_rows` unquantised rows: `rows` products (a sorted row each
// with a plan) in tiles of n rows.
int RunLayer(const void* x, int32_t x_dtype, int64_t x_rows, int64_t x_stride,
             int64_t rows, bool sorted, const xse_expert_plan* plan,
             int64_t scale_tiles, const xse_mx_matrix& w, const float* bias,
             int32_t activation, int n, void* y, int32_t y_dtype,
             int64_t y_stride, void* workspace, cudaStream_t s) {
  Rows from{};
  if (MxQuantizesInProduct(n, w.cols)) {
    from.x = x;
    from.x_dtype = x_dtype;
    from.x_stride = x_stride;
    from.sorted = sorted;
  } else {
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + rows * MxRowBytes(w.cols);
    const int rc = QuantizeRows(x, x_dtype, x_rows, w.cols, x_stride, plan,
                                sorted, n, codes, scales, s);
    if (rc != XSE_OK) return rc;
    from.codes = codes;
    from.scales = scales;
    from.scale_tiles = scale_tiles;
  }
  const int rc = RunGemm(from, rows, w, bias, activation, plan, n, y, y_dtype,
                         y_stride, s);
  if (rc == XSE_OK) SetLastLaunchCount(from.x != nullptr ? 1 : 2);
  return rc;
}

}  // namespace
}  // namespace xse

extern "C" {

int xse_linear_forward_mxfp4_q(const xse_mx_matrix* x, const xse_mx_matrix* w,
                               const float* bias, int32_t activation, void* y,
                               int32_t y_dtype, int64_t y_stride,
                               void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckLayer(w, activation, y_dtype, y_stride); rc != XSE_OK) {
    return rc;
  }
  if (int rc = CheckMxMatrix(x, "x"); rc != XSE_OK) return rc;
  if (x->groups != 1 || w->groups != 1 || x->cols != w->cols) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer needs x and w of one group and of equal "
                    "columns, got %d and %d.", x->cols, w->cols);
  }
  if (x->rows == 0) return XSE_OK;
  if (y == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer buffers must be non-null.");
  }
  const int n = MxTileRowsFor(x->rows, 1, w->cols);
  Rows from{};
  from.codes = x->codes;
  from.scales = x->scales;
  from.scale_tiles = MxRowTiles(x->rows);
  const int rc = RunGemm(from, x->rows, *w, bias, activation, nullptr, n, y,
                         y_dtype, y_stride, static_cast<cudaStream_t>(stream));
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

int64_t xse_linear_mxfp4_workspace(int64_t rows, int32_t in_dim) {
  if (rows < 1 || rows > INT32_MAX || in_dim < 1 ||
      in_dim > xse::kMostColumns) {
    return 0;
  }
  const int n = xse::MxTileRowsFor(rows, 1, in_dim);
  if (xse::MxQuantizesInProduct(n, in_dim)) return 0;
  return rows * xse::MxRowBytes(in_dim) +
         xse::MxRowTiles(rows) * xse::MxKTiles(in_dim) * xse::kMxTileBytes;
}

int xse_linear_forward_mxfp4(const void* x, int32_t x_dtype, int64_t rows,
                             int64_t x_stride, const xse_mx_matrix* w,
                             const float* bias, int32_t activation, void* y,
                             int32_t y_dtype, int64_t y_stride,
                             void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckLayer(w, activation, y_dtype, y_stride); rc != XSE_OK) {
    return rc;
  }
  if (w->groups != 1) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer needs w of one group, got %d.", w->groups);
  }
  if (int rc = CheckRowsIn(x, x_dtype, rows, x_stride, w->cols, workspace,
                           workspace_bytes,
                           xse_linear_mxfp4_workspace(rows, w->cols));
      rc != XSE_OK) {
    return rc;
  }
  if (rows == 0) return XSE_OK;
  if (y == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer buffers must be non-null.");
  }
  const int n = MxTileRowsFor(rows, 1, w->cols);
  return RunLayer(x, x_dtype, rows, x_stride, rows, false, nullptr,
                  MxRowTiles(rows), *w, bias, activation, n, y, y_dtype,
                  y_stride, workspace, static_cast<cudaStream_t>(stream));
}

int64_t xse_expert_linear_workspace(int64_t pairs, int32_t num_experts,
                                    int32_t in_dim) {
  if (pairs < 0 || pairs > INT32_MAX || num_experts < 1 ||
      num_experts > XSE_MAX_EXPERTS || in_dim < 1 ||
      in_dim > xse::kMostColumns) {
    return 0;
  }
  const int n = xse::MxTileRowsFor(pairs, num_experts, in_dim);
  if (xse::MxQuantizesInProduct(n, in_dim)) return 0;
  return pairs * xse::MxRowBytes(in_dim) +
         xse::ExpertScaleTiles(pairs, num_experts, n) *
             xse::MxKTiles(in_dim) * xse::kMxTileBytes;
}

int xse_expert_linear_mxfp4(const void* x, int32_t x_dtype, int64_t x_stride,
                            int32_t sorted, const xse_expert_plan* plan,
                            const xse_mx_matrix* w, const float* bias,
                            int32_t activation, void* y, int32_t y_dtype,
                            int64_t y_stride, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckExpertPlan(plan); rc != XSE_OK) return rc;
  if (int rc = CheckLayer(w, activation, y_dtype, y_stride); rc != XSE_OK) {
    return rc;
  }
  if (w->groups != plan->num_experts) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "Expert layer needs one group of w per expert: %d groups, "
                    "%d experts.", w->groups, plan->num_experts);
  }
  const int64_t pairs = plan->tokens * plan->topk;
  const int64_t rows = sorted ? pairs : plan->tokens;
  if (int rc = CheckRowsIn(x, x_dtype, rows, x_stride, w->cols, workspace,
                           workspace_bytes,
                           xse_expert_linear_workspace(
                               pairs, plan->num_experts, w->cols));
      rc != XSE_OK) {
    return rc;
  }
  if (pairs == 0) return XSE_OK;
  if (y == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit layer buffers must be non-null.");
  }
  const int n = MxTileRowsFor(pairs, plan->num_experts, w->cols);
  return RunLayer(x, x_dtype, rows, x_stride, pairs, sorted != 0, plan,
                  ExpertScaleTiles(pairs, plan->num_experts, n), *w, bias,
                  activation, n, y, y_dtype, y_stride, workspace,
                  static_cast<cudaStream_t>(stream));
}

int xse_mxfp4_check(void* stream) {
  using namespace xse;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int failed = 0;
  cudaError_t e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) {
    e = cudaMemcpyFromSymbol(&failed, g_wait_failed, sizeof(failed));
  }
  if (e == cudaSuccess && failed != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_wait_failed, &zero, sizeof(zero));
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return FailWith(XSE_INTERNAL, "4-bit product check: %s",
                    cudaGetErrorString(e));
  }
  if (failed != 0) {
    return FailWith(XSE_DEADLINE_EXCEEDED,
                    "A wait in a 4-bit product's kernel ran out.");
  }
  return XSE_OK;
}

}  // extern "C"
