// Shared by the 4-bit and expert kernels: argument checks, the microscaled
// layout (include/xse_mx.h) and its device-side conversions.
#ifndef XSE_MX_INTERNAL_H_
#define XSE_MX_INTERNAL_H_

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/xse_emb.h"
#include "../../include/xse_experts.h"
#include "../../include/xse_mx.h"
#include "xse_internal.h"

namespace xse {

constexpr int kMxBlock = 32;       // elements per scale
constexpr int kMxTileRows = 128;   // rows of a scale tile
constexpr int kMxTileBytes = 512;  // 128 rows x 4 blocks
constexpr int kNumSms = 148;
constexpr int32_t kMostColumns = 1 << 30;  // of a row: offsets into it fit int

// Sets the error text (printf style) and returns `code`.
int FailWith(int code, const char* fmt, ...)
    __attribute__((format(printf, 2, 3)));
// XSE_OK, or XSE_INTERNAL with the pending launch error of `what`.
int LaunchStatus(const char* what);

inline int64_t MxRowBytes(int64_t cols) { return (cols + 31) / 32 * 16; }
inline int64_t MxKTiles(int64_t cols) { return (cols + 127) / 128; }
inline int64_t MxRowTiles(int64_t rows) { return (rows + 127) / 128; }

// Bytes of a matrix's codes and scales, false for sizes that are not served:
// out of range, or with 2^63 bytes or more.
inline bool MxMatrixBytes(int64_t rows, int64_t cols, int64_t groups,
                          int64_t* codes, int64_t* scales) {
  *codes = *scales = 0;
  if (rows < 0 || rows > INT32_MAX || cols < 1 || cols > kMostColumns ||
      groups < 1 || groups > INT32_MAX) {
    return false;
  }
  // Of one group: below 2^60 and 2^56.
  const int64_t group_codes = rows * MxRowBytes(cols);
  const int64_t group_scales =
      MxRowTiles(rows) * MxKTiles(cols) * kMxTileBytes;
  const int64_t most = group_codes > group_scales ? group_codes : group_scales;
  if (most > INT64_MAX / groups) return false;
  *codes = groups * group_codes;
  *scales = groups * group_scales;
  return true;
}

inline bool Aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// Lets `kernel` use `bytes` of shared memory on the current device. `done`, a
// static per kernel, remembers the devices it was set on (the call costs as
// much as a launch).
template <typename Kernel>
cudaError_t AllowShared(Kernel kernel, size_t bytes,
                        std::atomic<uint64_t>* done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
  if ((done->load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(bytes));
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// XSE_OK for a usable matrix of `what`; buffers are checked unless empty.
int CheckMxMatrix(const xse_mx_matrix* q, const char* what);
// XSE_OK for a usable plan (arrays non-null where they have entries).
int CheckExpertPlan(const xse_expert_plan* plan);

// Rows of a product's tile for groups of rows / groups rows on average. The
// scales of an expert product's rows are laid out in 512-byte tiles of that
// many rows each, so that every tile's scales begin a column of tensor memory.
// 256 rows (pairs of SMs) need a k that is long against the end of a tile,
// which nothing overlaps there: 8192 rows to 8192 features in bf16, tiles of 128
// and 256 rows, quantisation included, both sides in turn with pauses (at 1.85 to
// 1.97 GHz, off the power cap): k 1024 62 and 69 us, k 1536 72 and 75 us, k 2048
// 87 and 78 us, k 4096 150 and 111 us; 64 experts of about 512 rows each, k 2048:
// 111 and 102 us. The rule sees the average alone: where one group holds most of
// the rows, its tiles are smaller than its own rows would ask for.
inline int MxTileRowsFor(int64_t rows, int32_t groups, int32_t k) {
  const int64_t mean = (rows + groups - 1) / groups;
  if (mean <= 64) return mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
  return mean <= 128 || k < 1536 ? 128 : 256;
}

// Scale tiles of n rows that hold every expert's rows on tile boundaries:
// expert e's rows start at tile offsets[e] / n + e. With c rows it ends by
// tile offsets[e] / n + e + ceil(c / n) <= (offsets[e] + c) / n + e + 1, the
// next one's start, so no scan of the counts is needed.
inline int64_t ExpertScaleTiles(int64_t pairs, int32_t num_experts, int n) {
  return (pairs / n + num_experts) * (n > kMxTileRows ? 2 : 1);
}

// Whether a product with tiles of n rows quantises its rows itself (then it
// needs no workspace): each of its blocks reads the rows anew, which for few
// rows costs less than a launch and a trip through memory. Their k has to fit
// a buffer of shared memory (n * 128 bytes of codes and 1 KB of scales for
// every 256 elements).
constexpr int kRowBufferBytes = 96 * 1024;
inline bool MxQuantizesInProduct(int n, int32_t k) {
  return n <= 32 &&
         (k + 255) / 256 * static_cast<int64_t>(n * 128 + 1024) <=
             kRowBufferBytes;
}

// Whether expert rows of `cols` elements of `size` bytes may go through the ring
// kernels, which count a row's bytes in 32 bits: the offset after the row's
// last 16-byte pieces, a step of all the threads that share a row further on,
// still has to fit. Wider rows (fp32 within 4 KB of 4 GB, which xse_experts.h
// allows) go element by element.
constexpr int kRingRowThreads = 256;  // that share a row at most
constexpr bool ExpertRowFitsRing(int64_t cols, int64_t size) {
  return cols * size <= UINT32_MAX - kRingRowThreads * 16;
}

// Quantises the rows of x for a product in tiles of `tile_rows`: plan NULL, one
// group as xse_mxfp4_quantize lays it out; else to the sorted rows' places
// (codes by sorted row, scales as ExpertScaleTiles says), from token rows or
// sorted ones.
int QuantizeRows(const void* x, int32_t dtype, int64_t rows, int32_t cols,
                 int64_t row_stride, const xse_expert_plan* plan, bool sorted,
                 int tile_rows, void* codes, void* scales,
                 cudaStream_t stream);

// Byte offset of the scale of column `col` from that of its row's first block.
// 64 bits: a row's scale tiles pass 2^31 bytes from 2^29 columns on.
__host__ __device__ constexpr int64_t MxColumnScaleAt(int32_t col) {
  return static_cast<int64_t>(col / 128) * kMxTileBytes + col / 32 % 4;
}

#ifdef __CUDACC__

// The E8M0 byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t MxScaleByte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  if (e == 255u) return 255u;
  return e > 2u ? e - 2u : 0u;
}

// 2^(127 - s), the factor that brings a block into E2M1's range; 0 for a block
// of NaN. s <= 252 otherwise, so the result is a normal number.
__device__ __forceinline__ float MxInverseScale(uint32_t s) {
  return s == 255u ? 0.0f : __uint_as_float((254u - s) << 23);
}

// 2^(s - 127), NaN for s = 255.
__device__ __forceinline__ float MxScale(uint32_t s) {
  if (s == 0u) return __uint_as_float(0x00400000u);
  return s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s << 23);
}

// Eight E2M1 codes in one word, element 0 lowest: nearest, ties to even,
// saturating at 6.
__device__ __forceinline__ uint32_t MxCodes8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
        "f"(v[6]), "f"(v[7]));
  return r;
}

// The bits of the largest magnitude among kWords words of T (two bfloat16 or
// one float a word). Magnitudes are ordered as integers, infinities and NaN
// last.
template <typename T, int kWords>
__device__ __forceinline__ uint32_t MxLargest(const uint32_t* w) {
  uint32_t most = 0;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      most = __vmaxu2(most, w[i] & 0x7fff7fffu);
    }
    return max(most & 0xffff0000u, most << 16);
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) most = max(most, w[i] & 0x7fffffffu);
    return most;
  }
}

// The codes of 8 * kCodeWords elements of a block with scale byte s.
template <typename T, int kCodeWords>
__device__ __forceinline__ void MxEncode(const uint32_t* w, uint32_t s,
                                         uint32_t* codes) {
  const float inv = MxInverseScale(s);
#pragma unroll
  for (int k = 0; k < kCodeWords; ++k) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t u = w[4 * k + i / 2];
        f[i] = __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16) * inv;
      } else {
        f[i] = __uint_as_float(w[8 * k + i]) * inv;
      }
    }
    codes[k] = s == 255u ? 0u : MxCodes8(f);
  }
}

// Byte offset of the scale of block b of (padded) row r.
__device__ __forceinline__ int64_t MxScaleAt(int64_t r, int64_t b,
                                             int64_t k_tiles) {
  return ((r >> 7) * k_tiles + (b >> 2)) * kMxTileBytes + (r & 31) * 16 +
         ((r >> 5) & 3) * 4 + (b & 3);
}

#endif  // __CUDACC__

}  // namespace xse

#endif  // XSE_MX_INTERNAL_H_
