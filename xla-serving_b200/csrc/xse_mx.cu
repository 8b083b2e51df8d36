// Quantisation to microscaled 4-bit values and back (include/xse_mx.h).
//
// Both directions are one pass over memory: a block's largest magnitude, its
// power-of-two scale and the rounded codes are computed in registers. All the
// arithmetic is exact (a power of two times a float) except the one rounding
// to E2M1, so results do not depend on the kernel that ran.
//
// Three kernels read rows that differ in what their loads can be:
//   QuantizeVecKernel   16-byte aligned rows: a lane takes 8 elements, four
//                       lanes share a block
//   QuantizeWarpKernel  rows at any alignment: a lane takes one element of
//                       each of four blocks, so that loads stay coalesced, and
//                       the codes are transposed to words with shuffles
//   QuantizeStrideKernel  columns apart (a [in, out] kernel read as [out,
//                       in]): a thread takes one block, neighbouring threads
//                       neighbouring rows

#include <cstdarg>
#include <cstdio>

#include "xse_mx_internal.h"

namespace xse {

int FailWith(int code, const char* fmt, ...) {
  char buf[512];
  va_list args;
  va_start(args, fmt);
  vsnprintf(buf, sizeof(buf), fmt, args);
  va_end(args);
  SetLastErrorMessage(buf);
  return code;
}

int LaunchStatus(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return XSE_OK;
  return FailWith(XSE_INTERNAL, "%s launch: %s", what, cudaGetErrorString(e));
}

int CheckMxMatrix(const xse_mx_matrix* q, const char* what) {
  if (q == nullptr || q->rows < 0 || q->cols < 1 || q->groups < 1 ||
      q->rows > INT32_MAX) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit matrix %s needs 0 <= rows < 2^31, cols >= 1 and "
                    "groups >= 1.", what);
  }
  if (q->rows == 0) return XSE_OK;
  if (q->codes == nullptr || q->scales == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit matrix %s: codes and scales must be non-null.",
                    what);
  }
  if (!Aligned16(q->codes) || !Aligned16(q->scales)) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit matrix %s: codes and scales must be 16-byte "
                    "aligned.", what);
  }
  return XSE_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int kWarpShift = 3;  // warps of a block

// The rows of a kernel whose warps take `chunks` pieces of a row each in turn:
// 2^row_shift warps a row, so that no index needs a division.
int RowShift(int64_t chunks) {
  int shift = 0;
  while (shift < kWarpShift && (1 << shift) < chunks) ++shift;
  return shift;
}

int BlocksForRows(int64_t rows, int row_shift) {
  const int64_t per = 1 << (kWarpShift - row_shift);
  const int64_t b = (rows + per - 1) / per;
  const int64_t most = static_cast<int64_t>(kNumSms) * 8;  // one wave
  return static_cast<int>(b > most ? most : b);
}

struct WarpRow {
  int64_t row, step;  // first row of this warp, rows of a step
  int chunk, chunks;  // first piece of the row, pieces of a step
};

__device__ __forceinline__ WarpRow FirstRow(int row_shift) {
  const int warp = threadIdx.x / 32;
  WarpRow w;
  w.chunks = 1 << row_shift;
  w.chunk = warp & (w.chunks - 1);
  const int per = 1 << (kWarpShift - row_shift);
  w.row = static_cast<int64_t>(blockIdx.x) * per + (warp >> row_shift);
  w.step = static_cast<int64_t>(gridDim.x) * per;
  return w;
}

// Where quantised rows go: row r of group g to code row g * rows + r, or (with
// a plan) token row t to the sorted rows of its choices, or sorted row r to
// itself; see ExpertScaleTiles for the scales' rows.
enum : int { kPlain = 0, kFromTokens = 1, kFromSorted = 2 };

struct QuantParams {
  const void* x;
  int64_t group_stride, row_stride, col_stride;
  int64_t rows;         // of a group
  int64_t total_rows;   // groups * rows
  int32_t groups;
  int32_t row_shift;    // 2^row_shift warps share a row
  int32_t cols;
  int32_t k_tiles;
  int64_t row_bytes;
  int64_t row_tiles;    // scale tiles of a group's rows (of all: with a plan)
  int32_t tile_rows;    // rows of a scale tile
  uint8_t* codes;
  uint8_t* scales;
  const int32_t* offsets;
  const int32_t* slots;
  int32_t topk;
  int32_t num_experts;
  int64_t pairs;
};

template <typename T>
__device__ __forceinline__ float ToFloat(T v) {
  return static_cast<float>(v);
}
template <>
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

// Eight neighbouring elements (16-byte aligned).
__device__ __forceinline__ void Load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void Load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename T>
__device__ __forceinline__ const T* RowOf(const QuantParams& p, int64_t row) {
  const int64_t g = p.groups == 1 ? 0 : row / p.rows;
  return static_cast<const T*>(p.x) + g * p.group_stride +
         (row - g * p.rows) * p.row_stride;
}

// Calls put(code row, scale row) for each place of source row `row`.
template <int kMode, typename Put>
__device__ __forceinline__ void ForPlaces(const QuantParams& p, int64_t row,
                                          int lane, Put put) {
  if constexpr (kMode == kPlain) {
    const int64_t g = p.groups == 1 ? 0 : row / p.rows;
    put(row, g * p.row_tiles * kMxTileRows + (row - g * p.rows));
  } else {
    const int count = kMode == kFromTokens ? p.topk : 1;
    for (int j = 0; j < count; ++j) {
      const int32_t slot = kMode == kFromTokens
                               ? __ldg(p.slots + row * p.topk + j)
                               : static_cast<int32_t>(row);
      if (slot < 0 || slot >= p.pairs) continue;
      const int e = ExpertOfRow(p.offsets, p.num_experts, slot, lane);
      if (e >= p.num_experts) continue;  // behind the last sorted row
      const int32_t begin = __ldg(p.offsets + e);
      if (begin < 0 || begin > slot) continue;
      const int local = slot - begin;
      const int in_tile = local % p.tile_rows;
      const int64_t tile =
          (begin / p.tile_rows + e + local / p.tile_rows) *
              (p.tile_rows > kMxTileRows ? 2 : 1) + in_tile / kMxTileRows;
      if (tile >= p.row_tiles) continue;
      put(static_cast<int64_t>(slot),
          tile * kMxTileRows + in_tile % kMxTileRows);
    }
  }
}

// A warp takes 512 columns of a row, a lane 8 of each half; four lanes share a
// block and agree on its largest magnitude with two shuffles.
template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads)
    QuantizeVecKernel(const __grid_constant__ QuantParams p) {
  const int lane = threadIdx.x & 31;
  const int padded = p.k_tiles * 128, code_cols = (p.cols + 31) / 32 * 32;
  const WarpRow w = FirstRow(p.row_shift);
  for (int64_t row = w.row; row < p.total_rows; row += w.step) {
    const T* x = RowOf<T>(p, row);
    for (int first = w.chunk * 512; first < padded; first += w.chunks * 512) {
      float v[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = first + h * 256 + lane * 8;
        if (col + 8 <= p.cols) {
          Load8(x + col, v[h]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[h][i] = col + i < p.cols ? ToFloat(x[col + i]) : 0.0f;
          }
        }
      }
      uint32_t word[2], scales[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          most = max(most, __float_as_uint(v[h][i]) & 0x7fffffffu);
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const uint32_t s = MxScaleByte(most);
        const float inv = MxInverseScale(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h][i] *= inv;
        word[h] = s == 255u ? 0u : MxCodes8(v[h]);
        // The scale bytes of four blocks (16 lanes) as one word.
        scales[h] = s | __shfl_down_sync(0xffffffffu, s, 4) << 8;
        scales[h] |= __shfl_down_sync(0xffffffffu, scales[h], 8) << 16;
      }
      ForPlaces<kMode>(p, row, lane, [&](int64_t code_row, int64_t scale_row) {
        uint8_t* codes = p.codes + code_row * p.row_bytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = first + h * 256 + lane * 8;
          if (col < code_cols) {
            *reinterpret_cast<uint32_t*>(codes + col / 2) = word[h];
          }
          if ((lane & 15) == 0 && col < padded) {
            *reinterpret_cast<uint32_t*>(
                p.scales + MxScaleAt(scale_row, col / 32, p.k_tiles)) =
                scales[h];
          }
        }
      });
    }
  }
}

// A warp takes 256 columns of a row as two halves of four blocks of 32 lanes.
// Lane l ends with the word of block 2 (l & 1) + (l >> 1 & 1) of each half,
// bytes 4 (l >> 3) on.
template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads)
    QuantizeWarpKernel(const __grid_constant__ QuantParams p) {
  const unsigned all = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1, odd2 = lane & 2;
  const int padded = p.k_tiles * 128, code_cols = (p.cols + 31) / 32 * 32;
  const WarpRow w = FirstRow(p.row_shift);
  for (int64_t row = w.row; row < p.total_rows; row += w.step) {
    const T* x = RowOf<T>(p, row);
    for (int first = w.chunk * 256; first < padded; first += w.chunks * 256) {
      float v[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const int col = first + 32 * b + lane;
        v[b] = col < p.cols ? ToFloat(x[col]) : 0.0f;
      }
      uint32_t word[2], scales[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* u = v + 4 * h;
        scales[h] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t s = MxScaleByte(
              __reduce_max_sync(all, __float_as_uint(u[b]) & 0x7fffffffu));
          scales[h] |= s << (8 * b);
          u[b] = s == 255u ? 0.0f : u[b] * MxInverseScale(s);
        }
        // Even lanes keep blocks 0 and 1, odd lanes 2 and 3, of a pair of
        // elements; then each lane one block of two pairs; then of four.
        const float r0 = __shfl_xor_sync(all, odd ? u[0] : u[2], 1);
        const float r1 = __shfl_xor_sync(all, odd ? u[1] : u[3], 1);
        const uint32_t b0 = odd ? MxCodes2(r0, u[2]) : MxCodes2(u[0], r0);
        const uint32_t b1 = odd ? MxCodes2(r1, u[3]) : MxCodes2(u[1], r1);
        const uint32_t got = __shfl_xor_sync(all, odd2 ? b0 : b1, 2);
        word[h] = odd2 ? (got | b1 << 8) : (b0 | got << 8);
        word[h] |= __shfl_down_sync(all, word[h], 4) << 16;
      }
      const int block = (odd ? 2 : 0) + (odd2 ? 1 : 0);
      ForPlaces<kMode>(p, row, lane, [&](int64_t code_row, int64_t scale_row) {
        uint8_t* codes = p.codes + code_row * p.row_bytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int half = first + 128 * h;
          const int col = half + 32 * block + 8 * (lane >> 3);
          if ((lane & 4) == 0 && col < code_cols) {
            *reinterpret_cast<uint32_t*>(codes + col / 2) = word[h];
          }
          if (lane == 0 && half < padded) {
            *reinterpret_cast<uint32_t*>(
                p.scales + MxScaleAt(scale_row, half / 32, p.k_tiles)) =
                scales[h];
          }
        }
      });
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    QuantizeStrideKernel(const __grid_constant__ QuantParams p) {
  const int blocks = p.k_tiles * 4;
  const int64_t units = p.total_rows * blocks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
       u < units; u += step) {
    // Rows of a group vary fastest.
    const int64_t g = u / (p.rows * blocks);
    const int64_t rest = u - g * p.rows * blocks;
    const int64_t b = rest / p.rows, r = rest - b * p.rows;
    const T* x = static_cast<const T*>(p.x) + g * p.group_stride +
                 r * p.row_stride;
    const int first = static_cast<int>(b) * 32;
    float v[32];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      v[i] = first + i < p.cols ? ToFloat(x[(first + i) * p.col_stride]) : 0.0f;
      most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    const uint32_t s = MxScaleByte(most);
    const float inv = MxInverseScale(s);
    p.scales[MxScaleAt(g * p.row_tiles * kMxTileRows + r, b, p.k_tiles)] =
        static_cast<uint8_t>(s);
    if (first >= p.cols) continue;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = v[8 * i + k] * inv;
      w[i] = s == 255u ? 0u : MxCodes8(t);
    }
    *reinterpret_cast<uint4*>(p.codes + (g * p.rows + r) * p.row_bytes +
                              first / 2) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A warp takes 256 columns of a row: its lanes load a word of eight codes
// each, and every lane takes its element's word by a shuffle, so that the
// stores are coalesced at any alignment.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    DequantizeKernel(const uint8_t* __restrict__ codes,
                     const uint8_t* __restrict__ scales, int64_t rows,
                     int groups, int cols, int64_t row_bytes, int k_tiles,
                     int64_t row_tiles, int row_shift, T* __restrict__ out,
                     int64_t group_stride, int64_t row_stride) {
  const int lane = threadIdx.x & 31;
  const int padded = k_tiles * 128;
  const WarpRow w = FirstRow(row_shift);
  for (int64_t row = w.row; row < rows * groups; row += w.step) {
    const int64_t g = groups == 1 ? 0 : row / rows;
    const int64_t r = row - g * rows;
    T* o = out + g * group_stride + r * row_stride;
    for (int first = w.chunk * 256; first < padded; first += w.chunks * 256) {
      const int at = first / 2 + lane * 4;
      const uint32_t word =
          at < row_bytes
              ? __ldg(reinterpret_cast<const uint32_t*>(codes +
                                                        row * row_bytes + at))
              : 0u;
      uint32_t sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = first + 128 * h < padded
                    ? __ldg(reinterpret_cast<const uint32_t*>(
                          scales + MxScaleAt(g * row_tiles * kMxTileRows + r,
                                             first / 32 + 4 * h, k_tiles)))
                    : 0u;
      }
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint32_t u = __shfl_sync(0xffffffffu, word, 4 * b + (lane >> 3));
        const int col = first + 32 * b + lane;
        const float v = MxCodeValue(u >> (4 * (lane & 7))) *
                        MxScale(sc[b >> 2] >> (8 * (b & 3)) & 0xffu);
        if (col < cols) o[col] = static_cast<T>(v);
      }
    }
  }
}

int BlocksFor(int64_t work, int per_block) {
  const int64_t b = (work + per_block - 1) / per_block;
  const int64_t most = static_cast<int64_t>(kNumSms) * 8;  // one wave
  return static_cast<int>(b < 1 ? 1 : (b > most ? most : b));
}

template <typename T, int kMode>
void LaunchQuantize(QuantParams p, bool vec, cudaStream_t s) {
  p.row_shift = RowShift(vec ? (p.k_tiles + 3) / 4 : (p.k_tiles + 1) / 2);
  const int blocks = BlocksForRows(p.total_rows, p.row_shift);
  if (vec) {
    QuantizeVecKernel<T, kMode><<<blocks, kThreads, 0, s>>>(p);
  } else {
    QuantizeWarpKernel<T, kMode><<<blocks, kThreads, 0, s>>>(p);
  }
}

template <typename T>
void LaunchQuantizeAs(const QuantParams& p, int mode, cudaStream_t s) {
  if (p.col_stride != 1) {
    QuantizeStrideKernel<T>
        <<<BlocksFor(p.total_rows * p.k_tiles * 4, kThreads), kThreads, 0,
           s>>>(p);
    return;
  }
  const int64_t per = 16 / sizeof(T);
  const bool vec = Aligned16(p.x) && p.row_stride % per == 0 &&
                   p.group_stride % per == 0;
  if (mode == kPlain) LaunchQuantize<T, kPlain>(p, vec, s);
  if (mode == kFromTokens) LaunchQuantize<T, kFromTokens>(p, vec, s);
  if (mode == kFromSorted) LaunchQuantize<T, kFromSorted>(p, vec, s);
}

int RunQuantize(const QuantParams& p, int32_t dtype, int mode,
                cudaStream_t s) {
  if (dtype == XSE_DT_F32) LaunchQuantizeAs<float>(p, mode, s);
  if (dtype == XSE_DT_BF16) LaunchQuantizeAs<__nv_bfloat16>(p, mode, s);
  return LaunchStatus("4-bit quantisation");
}

}  // namespace

int QuantizeRows(const void* x, int32_t dtype, int64_t rows, int32_t cols,
                 int64_t row_stride, const xse_expert_plan* plan, bool sorted,
                 void* codes, void* scales, cudaStream_t stream) {
  QuantParams p{};
  p.x = x;
  p.row_stride = row_stride;
  p.col_stride = 1;
  p.rows = p.total_rows = rows;
  p.groups = 1;
  p.cols = cols;
  p.k_tiles = static_cast<int32_t>(MxKTiles(cols));
  p.row_bytes = MxRowBytes(cols);
  p.row_tiles = MxRowTiles(rows);
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  if (plan == nullptr) return RunQuantize(p, dtype, kPlain, stream);
  p.pairs = plan->tokens * plan->topk;
  p.tile_rows = MxTileRowsFor(p.pairs, plan->num_experts);
  p.row_tiles = ExpertScaleTiles(p.pairs, plan->num_experts, p.tile_rows);
  p.offsets = plan->offsets;
  p.slots = plan->slots;
  p.topk = plan->topk;
  p.num_experts = plan->num_experts;
  return RunQuantize(p, dtype, sorted ? kFromSorted : kFromTokens, stream);
}

}  // namespace xse

extern "C" {

int64_t xse_mxfp4_codes_bytes(int64_t rows, int32_t cols, int32_t groups) {
  if (rows < 0 || rows > INT32_MAX || cols < 1 || groups < 1) return 0;
  return groups * rows * xse::MxRowBytes(cols);
}

int64_t xse_mxfp4_scales_bytes(int64_t rows, int32_t cols, int32_t groups) {
  if (rows < 0 || rows > INT32_MAX || cols < 1 || groups < 1) return 0;
  return groups * xse::MxRowTiles(rows) * xse::MxKTiles(cols) *
         xse::kMxTileBytes;
}

int xse_mxfp4_quantize(const void* x, int32_t dtype, int64_t group_stride,
                       int64_t row_stride, int64_t col_stride,
                       const xse_mx_matrix* q, void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckMxMatrix(q, "q"); rc != XSE_OK) return rc;
  if (dtype != XSE_DT_F32 && dtype != XSE_DT_BF16) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit quantisation reads float32 or bfloat16, got type "
                    "%d", dtype);
  }
  if (q->rows == 0) return XSE_OK;
  if (x == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT, "4-bit quantisation: x is null.");
  }
  QuantParams p{};
  p.x = x;
  p.group_stride = q->groups == 1 ? 0 : group_stride;
  p.row_stride = row_stride;
  p.col_stride = q->cols == 1 ? 1 : col_stride;
  p.rows = q->rows;
  p.total_rows = q->rows * q->groups;
  p.groups = q->groups;
  p.cols = q->cols;
  p.k_tiles = static_cast<int32_t>(MxKTiles(q->cols));
  p.row_bytes = MxRowBytes(q->cols);
  p.row_tiles = MxRowTiles(q->rows);
  p.codes = static_cast<uint8_t*>(q->codes);
  p.scales = static_cast<uint8_t*>(q->scales);
  const int rc =
      RunQuantize(p, dtype, kPlain, static_cast<cudaStream_t>(stream));
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

int xse_mxfp4_dequantize(const xse_mx_matrix* q, void* out, int32_t dtype,
                         int64_t group_stride, int64_t row_stride,
                         void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckMxMatrix(q, "q"); rc != XSE_OK) return rc;
  if (dtype != XSE_DT_F32 && dtype != XSE_DT_BF16) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit values are read back as float32 or bfloat16, got "
                    "type %d", dtype);
  }
  if (row_stride < q->cols) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit values need an output row stride >= cols.");
  }
  if (q->rows == 0) return XSE_OK;
  if (out == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT, "4-bit values: out is null.");
  }
  const int k_tiles = static_cast<int>(MxKTiles(q->cols));
  const int row_shift = RowShift((k_tiles + 1) / 2);
  const int blocks = BlocksForRows(q->rows * q->groups, row_shift);
  const uint8_t* codes = static_cast<const uint8_t*>(q->codes);
  const uint8_t* scales = static_cast<const uint8_t*>(q->scales);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == XSE_DT_F32) {
    DequantizeKernel<float><<<blocks, kThreads, 0, s>>>(
        codes, scales, q->rows, q->groups, q->cols, MxRowBytes(q->cols),
        k_tiles, MxRowTiles(q->rows), row_shift, static_cast<float*>(out),
        group_stride, row_stride);
  } else {
    DequantizeKernel<__nv_bfloat16><<<blocks, kThreads, 0, s>>>(
        codes, scales, q->rows, q->groups, q->cols, MxRowBytes(q->cols),
        k_tiles, MxRowTiles(q->rows), row_shift,
        static_cast<__nv_bfloat16*>(out), group_stride, row_stride);
  }
  const int rc = LaunchStatus("4-bit dequantisation");
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

}  // extern "C"
