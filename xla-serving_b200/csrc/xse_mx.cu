// Quantisation to microscaled 4-bit values and back (include/xse_mx.h).
//
// Both directions are one pass over memory: a block's largest magnitude, its
// power-of-two scale and the rounded codes are computed in registers. All the
// arithmetic is exact (a power of two times a float) except the one rounding
// to E2M1, so results do not depend on the kernel that ran.
//
// Two kernels: QuantizeKernel for rows of neighbouring elements (a lane takes
// 64 bytes of a row), QuantizeStrideKernel for elements apart (a [in, out]
// kernel read as [out, in]: a thread takes one block, neighbouring threads
// neighbouring rows).

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
  int64_t codes = 0, scales = 0;
  if (q == nullptr ||
      !MxMatrixBytes(q->rows, q->cols, q->groups, &codes, &scales)) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "4-bit matrix %s needs 0 <= rows < 2^31, 1 <= cols <= "
                    "2^30, groups >= 1 and less than 2^63 bytes.", what);
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

// `per_sm` blocks at most for each SM. The aligned quantisation runs best in one
// wave of the six (to several places: five) that its registers allow (8192 x
// 4096 fp32: 25 us, 28 us with eight); the kernels that turn their elements with eight, whose second wave
// fills the first one's waits (read-back of the same: 29 us, 32 us with six).
int BlocksForRows(int64_t rows, int row_shift, int per_sm) {
  const int64_t per = 1 << (kWarpShift - row_shift);
  const int64_t b = (rows + per - 1) / per;
  const int64_t most = static_cast<int64_t>(kNumSms) * per_sm;
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
  int32_t tile_shift;   // of a product's tile: 2^tile_shift rows
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

// The kBytes of a row that a lane quantises: a block or half of one (two lanes
// then agree on the scale).
template <typename T, int kBytes>
struct Part {
  static constexpr int kElements = kBytes / sizeof(T);
  static constexpr int kLanes = kMxBlock / kElements;  // of a block
  static constexpr int kWords = kElements / 8;         // of codes
  static constexpr int kPieces = kBytes / 16;
  uint4 v[kPieces];

  // The scale byte of the block and this lane's codes.
  __device__ uint32_t Quantize(uint32_t (&codes)[kWords]) const {
    uint32_t most = MxLargest<T, kBytes / 4>(&v[0].x);
    if constexpr (kLanes == 2) {
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    }
    const uint32_t s = MxScaleByte(most);
    MxEncode<T, kWords>(&v[0].x, s, codes);
    return s;
  }
};

template <typename T>
__device__ __forceinline__ const T* RowOf(const QuantParams& p, int64_t row) {
  const int64_t g = p.groups == 1 ? 0 : row / p.rows;
  return static_cast<const T*>(p.x) + g * p.group_stride +
         (row - g * p.rows) * p.row_stride;
}

// Where a source row's quantised row goes: its code row, -1 for nowhere, and its
// row of scales.
struct Place {
  int32_t code_row;
  int64_t scale_row;
};

// The places of choices [first, first + 32) of a row, lane by lane.
template <int kMode>
__device__ __forceinline__ Place PlaceOf(const QuantParams& p, int64_t row,
                                         int choice) {
  Place none{-1, 0};
  int32_t slot = static_cast<int32_t>(row);
  if (kMode == kFromTokens) {
    if (choice >= p.topk) return none;
    slot = __ldg(p.slots + row * p.topk + choice);
  }
  if (slot < 0 || slot >= p.pairs) return none;
  // The experts that end at or before the row.
  int low = 0, high = p.num_experts;
  while (low < high) {
    const int mid = (low + high) / 2;
    if (__ldg(p.offsets + mid + 1) <= slot) {
      low = mid + 1;
    } else {
      high = mid;
    }
  }
  if (low == p.num_experts) return none;  // behind the last sorted row
  const int32_t begin = __ldg(p.offsets + low);
  if (begin < 0 || begin > slot) return none;
  // Tiles have 2^tile_shift rows, those of 256 two scale tiles.
  const int local = slot - begin;
  const int in_tile = local & ((1 << p.tile_shift) - 1);
  const int64_t tile =
      (static_cast<int64_t>(begin >> p.tile_shift) + low +
       (local >> p.tile_shift)) *
          (1 << p.tile_shift > kMxTileRows ? 2 : 1) +
      in_tile / kMxTileRows;
  if (tile >= p.row_tiles) return none;
  return Place{slot, tile * kMxTileRows + in_tile % kMxTileRows};
}

// Calls put(code row, scale row) for each place of source row `row`; all lanes
// of the warp together.
template <int kMode, typename Put>
__device__ __forceinline__ void ForPlaces(const QuantParams& p, int64_t row,
                                          int lane, Put put) {
  if constexpr (kMode == kPlain) {
    const int64_t g = p.groups == 1 ? 0 : row / p.rows;
    put(row, g * p.row_tiles * kMxTileRows + (row - g * p.rows));
  } else if constexpr (kMode == kFromSorted) {
    const Place at = PlaceOf<kMode>(p, row, 0);
    if (at.code_row >= 0) put(at.code_row, at.scale_row);
  } else {
    for (int first = 0; first < p.topk; first += 32) {
      const Place mine = PlaceOf<kMode>(p, row, first + lane);
      const int count = min(p.topk - first, 32);
      for (int j = 0; j < count; ++j) {
        const int64_t code_row = __shfl_sync(0xffffffffu, mine.code_row, j);
        const int64_t scale_row = __shfl_sync(0xffffffffu, mine.scale_row, j);
        if (code_row >= 0) put(code_row, scale_row);
      }
    }
  }
}

// A warp takes 32 parts of a row at a time. kAligned: a lane's 64 bytes are
// loaded as they lie, four 16-byte loads that share cache lines with the
// neighbouring lanes' (with loads contiguous over the warp, four or more lanes
// share a block's scale and its arithmetic is repeated in each: 31 us against
// 16 us for 8192 x 4096 bf16). Otherwise the elements are loaded one by one
// over the warp and turned through shared memory.
template <typename T, bool kAligned>
using PartOf = Part<T, kAligned || sizeof(T) == 4 ? 64 : 32>;

template <typename T, int kMode, bool kAligned>
__global__ void __launch_bounds__(kThreads)
    QuantizeKernel(const __grid_constant__ QuantParams p) {
  using P = PartOf<T, kAligned>;
  constexpr int kSpan = 32 * P::kElements;
  __shared__ uint4 turn[kAligned ? 1 : kThreads / 32]
                       [kAligned ? 1 : 32 * P::kPieces];
  // A product of these rows may be launched; it waits for this kernel's end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int padded = p.k_tiles * 128, code_cols = (p.cols + 31) / 32 * 32;
  const WarpRow w = FirstRow(p.row_shift);
  for (int64_t row = w.row; row < p.total_rows; row += w.step) {
    const T* x = RowOf<T>(p, row);
    for (int first = w.chunk * kSpan; first < padded;
         first += w.chunks * kSpan) {
      const int col = first + lane * P::kElements;
      P part;
      if constexpr (kAligned) {
        const uint4* src = reinterpret_cast<const uint4*>(x + col);
        if (col + P::kElements <= p.cols) {
#pragma unroll
          for (int i = 0; i < P::kPieces; ++i) part.v[i] = __ldg(src + i);
        } else {
          T* e = reinterpret_cast<T*>(part.v);
#pragma unroll
          for (int i = 0; i < P::kElements; ++i) {
            e[i] = col + i < p.cols ? x[col + i] : static_cast<T>(0.0f);
          }
        }
      } else {
        // 16-byte piece c lies where neither the stores nor the lanes' loads
        // meet in a bank.
        T* mine = reinterpret_cast<T*>(turn[threadIdx.x / 32]);
        constexpr int kPiece = 16 / sizeof(T);
        const auto place = [](int c) {
          return P::kPieces == 4 ? c ^ (c >> 3 & 3) : c ^ (c >> 3 & 1);
        };
        T v[P::kElements];
#pragma unroll
        for (int i = 0; i < P::kElements; ++i) {
          const int c = first + 32 * i + lane;
          v[i] = c < p.cols ? x[c] : static_cast<T>(0.0f);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P::kElements; ++i) {
          const int e = 32 * i + lane;
          mine[place(e / kPiece) * kPiece + e % kPiece] = v[i];
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P::kPieces; ++i) {
          part.v[i] = turn[threadIdx.x / 32][place(lane * P::kPieces + i)];
        }
      }
      uint32_t codes[P::kWords];
      uint32_t scales = part.Quantize(codes);
      if (col >= code_cols) scales = 0;  // blocks past the last
      // The scale bytes of four blocks as one word.
      scales |= __shfl_down_sync(0xffffffffu, scales, P::kLanes) << 8;
      scales |= __shfl_down_sync(0xffffffffu, scales, 2 * P::kLanes) << 16;
      ForPlaces<kMode>(p, row, lane, [&](int64_t code_row, int64_t scale_row) {
        if (col < code_cols) {
          uint8_t* dst = p.codes + code_row * p.row_bytes + col / 2;
          if constexpr (P::kWords == 4) {
            *reinterpret_cast<uint4*>(dst) =
                make_uint4(codes[0], codes[1], codes[2], codes[3]);
          } else {
            *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
          }
        }
        if (lane % (4 * P::kLanes) == 0 && col < padded) {
          *reinterpret_cast<uint32_t*>(
              p.scales + MxScaleAt(scale_row, col / 32, p.k_tiles)) = scales;
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

// The values of eight codes as pairs of bfloat16 (exact): two byte tables by
// the low three bits of four codes at a time, then the signs.
__device__ __forceinline__ void DecodeCodes(uint32_t word, uint32_t (&v)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t u = h ? word >> 16 : word;
    const uint32_t pick = u & 0x7777u;
    const uint32_t low = __byte_perm(0xc0800000u, 0xc0804000u, pick);
    const uint32_t high = __byte_perm(0x3f3f3f00u, 0x40404040u, pick);
    v[2 * h] = __byte_perm(low, high, 0x5140) | (u << 12 & 0x8000u) |
               (u << 24 & 0x80000000u);
    v[2 * h + 1] = __byte_perm(low, high, 0x7362) | (u << 4 & 0x8000u) |
                   (u << 16 & 0x80000000u);
  }
}

// Pairs of bfloat16 times a power of two (or NaN), as eight values of T. The
// products are exact in bfloat16, whose multiplication keeps subnormals.
__device__ __forceinline__ void ScaleValues(const uint32_t (&v)[4], uint32_t s,
                                            uint4 (&out)[1], __nv_bfloat16) {
  const uint32_t bits = __float_as_uint(MxScale(s)) >> 16;
  const uint32_t pair = bits << 16 | bits;
  __nv_bfloat162 m;
  __builtin_memcpy(&m, &pair, 4);
  uint32_t* o = &out[0].x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 a;
    __builtin_memcpy(&a, &v[i], 4);
    a = __hmul2(a, m);
    __builtin_memcpy(&o[i], &a, 4);
  }
}
__device__ __forceinline__ void ScaleValues(const uint32_t (&v)[4], uint32_t s,
                                            uint4 (&out)[2], float) {
  const float scale = MxScale(s);
  uint32_t* o = &out[0].x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = __float_as_uint(__uint_as_float(v[i] << 16) * scale);
    o[2 * i + 1] =
        __float_as_uint(__uint_as_float(v[i] & 0xffff0000u) * scale);
  }
}

// A warp takes 512 columns of a row, a lane eight of one block of each half.
// Values go through shared memory, so that the warp stores whole sectors: 16
// bytes a lane where rows are aligned, else single elements (a lane's own 32
// bytes of float32 stored as two halves: 42 us against 29 us for 8192 x 4096).
template <typename T, bool kAligned>
__global__ void __launch_bounds__(kThreads)
    DequantizeKernel(const uint8_t* __restrict__ codes,
                     const uint8_t* __restrict__ scales, int64_t rows,
                     int groups, int cols, int64_t row_bytes, int k_tiles,
                     int64_t row_tiles, int row_shift, T* __restrict__ out,
                     int64_t group_stride, int64_t row_stride) {
  constexpr int kPiece = 16 / sizeof(T), kPieces = 8 / kPiece;
  __shared__ uint4 turn[kThreads / 32][32 * kPieces];
  const int lane = threadIdx.x & 31;
  uint4* mine = turn[threadIdx.x / 32];
  // Piece c lies at c ^ (c / 8 % 2): two pieces of a lane, 32 bytes apart from
  // the next lane's, then meet in no bank.
  const auto place = [](int c) { return kPieces == 2 ? c ^ (c >> 3 & 1) : c; };
  const int padded = k_tiles * 128;
  const WarpRow w = FirstRow(row_shift);
  for (int64_t row = w.row; row < rows * groups; row += w.step) {
    const int64_t g = groups == 1 ? 0 : row / rows;
    const int64_t r = row - g * rows;
    T* o = out + g * group_stride + r * row_stride;
    const uint8_t* row_scales =
        scales + MxScaleAt(g * row_tiles * kMxTileRows + r, 0, k_tiles);
    for (int span = w.chunk * 512; span < padded; span += w.chunks * 512) {
      uint32_t word[2] = {}, s[2] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = span + h * 256 + lane * 8;
        if (col < cols) {
          word[h] = __ldg(reinterpret_cast<const uint32_t*>(
              codes + row * row_bytes + col / 2));
          s[h] = __ldg(row_scales + MxColumnScaleAt(col));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int first = span + h * 256;
        if (first >= cols) break;
        uint32_t v[4];
        uint4 pieces[kPieces];
        DecodeCodes(word[h], v);
        ScaleValues(v, s[h], pieces, T());
        if (kAligned && kPieces == 1 && first + 256 <= cols) {
          reinterpret_cast<uint4*>(o + first)[lane] = pieces[0];
          continue;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          mine[place(lane * kPieces + i)] = pieces[i];
        }
        __syncwarp();
        const T* values = reinterpret_cast<const T*>(mine);
        if (kAligned && first + 256 <= cols) {
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int c = 32 * i + lane;
            reinterpret_cast<uint4*>(o + first)[c] = mine[place(c)];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 32 * i + lane;
            if (first + at < cols) {
              o[first + at] =
                  values[place(at / kPiece) * kPiece + at % kPiece];
            }
          }
        }
      }
    }
  }
}

int BlocksFor(int64_t work, int per_block) {
  const int64_t b = (work + per_block - 1) / per_block;
  const int64_t most = static_cast<int64_t>(kNumSms) * 8;  // one wave
  return static_cast<int>(b < 1 ? 1 : (b > most ? most : b));
}

template <typename T, int kMode, bool kAligned>
void LaunchQuantizeRows(QuantParams p, cudaStream_t s) {
  constexpr int kSpan = 32 * PartOf<T, kAligned>::kElements;
  p.row_shift = RowShift((p.k_tiles * 128 + kSpan - 1) / kSpan);
  QuantizeKernel<T, kMode, kAligned>
      <<<BlocksForRows(p.total_rows, p.row_shift,
                        !kAligned ? 8 : kMode == kFromTokens ? 5 : 6), kThreads,
         0, s>>>(p);
}

template <typename T, int kMode>
void LaunchQuantize(const QuantParams& p, bool aligned, cudaStream_t s) {
  if (aligned) {
    LaunchQuantizeRows<T, kMode, true>(p, s);
  } else {
    LaunchQuantizeRows<T, kMode, false>(p, s);
  }
}

template <typename T>
void LaunchDequantize(const xse_mx_matrix& q, void* out, int64_t group_stride,
                      int64_t row_stride, cudaStream_t s) {
  const int k_tiles = static_cast<int>(MxKTiles(q.cols));
  const int row_shift = RowShift((k_tiles + 3) / 4);
  const int64_t per = 16 / sizeof(T);
  const bool aligned = Aligned16(out) && row_stride % per == 0 &&
                       (q.groups == 1 || group_stride % per == 0);
  const auto kernel =
      aligned ? DequantizeKernel<T, true> : DequantizeKernel<T, false>;
  kernel<<<BlocksForRows(q.rows * q.groups, row_shift, 8), kThreads, 0, s>>>(
      static_cast<const uint8_t*>(q.codes),
      static_cast<const uint8_t*>(q.scales), q.rows, q.groups, q.cols,
      MxRowBytes(q.cols), k_tiles, MxRowTiles(q.rows), row_shift,
      static_cast<T*>(out), group_stride, row_stride);
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
                 int tile_rows, void* codes, void* scales,
                 cudaStream_t stream) {
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
  while ((1 << p.tile_shift) < tile_rows) ++p.tile_shift;
  p.row_tiles = ExpertScaleTiles(p.pairs, plan->num_experts, tile_rows);
  p.offsets = plan->offsets;
  p.slots = plan->slots;
  p.topk = plan->topk;
  p.num_experts = plan->num_experts;
  return RunQuantize(p, dtype, sorted ? kFromSorted : kFromTokens, stream);
}

}  // namespace xse

extern "C" {

int64_t xse_mxfp4_codes_bytes(int64_t rows, int32_t cols, int32_t groups) {
  int64_t codes = 0, scales = 0;
  xse::MxMatrixBytes(rows, cols, groups, &codes, &scales);
  return codes;
}

int64_t xse_mxfp4_scales_bytes(int64_t rows, int32_t cols, int32_t groups) {
  int64_t codes = 0, scales = 0;
  xse::MxMatrixBytes(rows, cols, groups, &codes, &scales);
  return scales;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == XSE_DT_F32) {
    LaunchDequantize<float>(*q, out, group_stride, row_stride, s);
  } else {
    LaunchDequantize<__nv_bfloat16>(*q, out, group_stride, row_stride, s);
  }
  const int rc = LaunchStatus("4-bit dequantisation");
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

}  // extern "C"
