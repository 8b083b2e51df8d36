// Rows sorted by expert and back (include/xse_experts.h).
//
// Sorting is one launch: a cluster of up to eight blocks counts each warp's
// pairs per expert in shared memory, the blocks read one another's totals over
// distributed shared memory, and every warp then places its pairs in order.
// The row movers work token by token, so that a token's row (or its gradient)
// is read once for all its choices; their traffic is the rows themselves, each
// read and written once, and they are bound by HBM bandwidth.

#include <cooperative_groups.h>

#include "xse_mx_internal.h"

namespace cg = cooperative_groups;

namespace xse {

int CheckExpertPlan(const xse_expert_plan* plan) {
  if (plan == nullptr || plan->tokens < 0 || plan->topk < 1 ||
      plan->num_experts < 1 || plan->num_experts > XSE_MAX_EXPERTS) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "An expert plan needs tokens >= 0, topk >= 1 and 1 to %d "
                    "experts.", XSE_MAX_EXPERTS);
  }
  if (plan->tokens > INT32_MAX / plan->topk) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "An expert plan holds less than 2^31 pairs.");
  }
  if (plan->offsets == nullptr ||
      (plan->tokens > 0 &&
       (plan->order == nullptr || plan->slots == nullptr))) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "An expert plan's arrays must be non-null.");
  }
  return XSE_OK;
}

namespace {

// ------------------------------------------------------------------ sorting

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 8;

template <typename Id>
__device__ __forceinline__ int ExpertId(const Id* ids, int64_t p,
                                        int num_experts) {
  const Id id = ids[p];
  return id >= 0 && id < num_experts ? static_cast<int>(id) : -1;
}

// Warp w of block b takes the pairs [(b * 32 + w) * per_warp, + per_warp).
// Shared: counts[32][experts], then totals[experts] (this block's), then
// starts[experts] (this block's first row of each expert).
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
    SortKernel(const Id* __restrict__ ids, int pairs, int num_experts,
               int64_t per_warp, int32_t* __restrict__ offsets,
               int32_t* __restrict__ order, int32_t* __restrict__ slots) {
  extern __shared__ int shared[];
  __shared__ int warp_sums[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = gridDim.x;  // one cluster
  const int block = blockIdx.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  int* mine = shared + warp * num_experts;
  int* totals = shared + kSortWarps * num_experts;
  int* starts = totals + num_experts;
  for (int i = threadIdx.x; i < kSortWarps * num_experts; i += kSortThreads) {
    shared[i] = 0;
  }
  __syncthreads();
  const int64_t first =
      (static_cast<int64_t>(block) * kSortWarps + warp) * per_warp;
  const int64_t last = min(first + per_warp, static_cast<int64_t>(pairs));
  for (int64_t p = first + lane; p - lane < last; p += 32) {
    const int e = p < last ? ExpertId(ids, p, num_experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // Counts before each warp, within the block.
  for (int e = threadIdx.x; e < num_experts; e += kSortThreads) {
    int sum = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = shared[w * num_experts + e];
      shared[w * num_experts + e] = sum;
      sum += c;
    }
    totals[e] = sum;
  }
  if (blocks > 1) {
    cluster.sync();
  } else {
    __syncthreads();
  }
  // Thread e: all rows of expert e, and those of the blocks before this one;
  // then a scan over the experts (at most one per thread).
  int all = 0, before = 0;
  const int e = threadIdx.x;
  if (e < num_experts) {
    for (int b = 0; b < blocks; ++b) {
      const int c = blocks > 1 ? *cluster.map_shared_rank(totals + e, b)
                               : totals[e];
      if (b < block) before += c;
      all += c;
    }
  }
  int scan = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < warp; ++w) base += warp_sums[w];
  int kept = 0;
  for (int w = 0; w < kSortWarps; ++w) kept += warp_sums[w];
  if (e < num_experts) {
    const int begin = base + scan - all;
    starts[e] = begin + before;
    if (block == 0) {
      offsets[e] = begin;
      if (e == num_experts - 1) offsets[num_experts] = begin + all;
    }
  }
  __syncthreads();
  for (int64_t p = first + lane; p - lane < last; p += 32) {
    const int id = p < last ? ExpertId(ids, p, num_experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (id >= 0) {
      row = starts[id] + mine[id] + rank;
      order[row] = static_cast<int32_t>(p);
    }
    if (p < last) slots[p] = row;
    __syncwarp();
    if (id >= 0 && rank == 0) mine[id] += __popc(same);
    __syncwarp();
  }
  for (int64_t r = static_cast<int64_t>(kept) + block * kSortThreads +
                   threadIdx.x;
       r < pairs; r += blocks * kSortThreads) {
    order[r] = -1;
  }
  // A block's totals stay until the others have read them.
  if (blocks > 1) cluster.sync();
}

template <typename Id>
int LaunchSort(const void* ids, const xse_expert_plan& plan, cudaStream_t s) {
  const int pairs = static_cast<int>(plan.tokens * plan.topk);
  const int blocks = pairs > 4096 ? kSortCluster : 1;
  int64_t per_warp = (pairs + blocks * kSortWarps - 1) / (blocks * kSortWarps);
  per_warp = (per_warp + 31) / 32 * 32;
  const size_t smem = sizeof(int) * (kSortWarps + 2) *
                      static_cast<size_t>(plan.num_experts);
  cudaError_t e = cudaFuncSetAttribute(
      SortKernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
      static_cast<int>(smem));
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, SortKernel<Id>, static_cast<const Id*>(ids),
                           pairs, static_cast<int>(plan.num_experts), per_warp,
                           plan.offsets, plan.order, plan.slots);
  }
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? XSE_OK
                          : FailWith(XSE_INTERNAL, "expert sort launch: %s",
                                     cudaGetErrorString(e));
}

// --------------------------------------------------------------- row movers

constexpr int kThreads = 256;

// A piece of a row as a thread holds it: V elements, loaded and stored whole.
template <typename T, int V>
struct Piece {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Piece<T, V> LoadPiece(const T* p) {
  Piece<T, V> r;
  if constexpr (V == 1) {
    r.v[0] = *p;
  } else {
    static_assert(sizeof(r) == 16, "a piece is 16 bytes");
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    __builtin_memcpy(&r, &u, 16);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void StorePiece(T* p, const Piece<T, V>& r) {
  if constexpr (V == 1) {
    *p = r.v[0];
  } else {
    uint4 u;
    __builtin_memcpy(&u, &r, 16);
    __stcs(reinterpret_cast<uint4*>(p), u);
  }
}

__device__ __forceinline__ float Widen(float v) { return v; }
__device__ __forceinline__ float Widen(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T Narrow(float v);
template <>
__device__ __forceinline__ float Narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 Narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

struct MoveParams {
  const void* src;     // x, y or grad
  const void* y;       // backward only
  void* dst;           // out or grad_y
  float* grad_weights;
  const float* weights;
  const int32_t* offsets;
  const int32_t* slots;
  int64_t src_stride, y_stride, dst_stride;
  int64_t tokens, pairs;
  int32_t topk, num_experts, cols;
};

// Zeros behind the last sorted row of a [pairs, cols] output.
template <typename T>
__device__ void ZeroTail(const MoveParams& p) {
  const int64_t kept = max(0, __ldg(p.offsets + p.num_experts));
  const int64_t total = (p.pairs - kept) * p.cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
       i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / p.cols;
    static_cast<T*>(p.dst)[(kept + r) * p.dst_stride + (i - r * p.cols)] =
        Narrow<T>(0.0f);
  }
}

// One (token, piece) per thread and step.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    GatherKernel(const __grid_constant__ MoveParams p) {
  const int pieces = p.cols / V;
  const int64_t total = p.tokens * pieces;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
       i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t t = i / pieces;
    const int64_t c = (i - t * pieces) * V;
    const Piece<T, V> r = LoadPiece<T, V>(static_cast<const T*>(p.src) +
                                          t * p.src_stride + c);
    for (int j = 0; j < p.topk; ++j) {
      const int32_t slot = __ldg(p.slots + t * p.topk + j);
      if (slot < 0 || slot >= p.pairs) continue;
      StorePiece<T, V>(static_cast<T*>(p.dst) + slot * p.dst_stride + c, r);
    }
  }
  ZeroTail<T>(p);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    CombineKernel(const __grid_constant__ MoveParams p) {
  const int pieces = p.cols / V;
  const int64_t total = p.tokens * pieces;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
       i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t t = i / pieces;
    const int64_t c = (i - t * pieces) * V;
    float sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < p.topk; ++j) {
      const int32_t slot = __ldg(p.slots + t * p.topk + j);
      if (slot < 0 || slot >= p.pairs) continue;
      const float w = p.weights ? __ldg(p.weights + t * p.topk + j) : 1.0f;
      const Piece<T, V> r = LoadPiece<T, V>(static_cast<const T*>(p.src) +
                                            slot * p.src_stride + c);
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = fmaf(w, Widen(r.v[k]), sum[k]);
    }
    Piece<T, V> out;
#pragma unroll
    for (int k = 0; k < V; ++k) out.v[k] = Narrow<T>(sum[k]);
    StorePiece<T, V>(static_cast<T*>(p.dst) + t * p.dst_stride + c, out);
  }
}

// One warp per (token, choice): the gradient row scaled into its sorted row,
// and its dot product with the expert's row.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    CombineBackwardKernel(const __grid_constant__ MoveParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) +
                   threadIdx.x / 32;
       i < p.pairs; i += warps) {
    const int32_t slot = __ldg(p.slots + i);
    float dot = 0.0f;
    if (slot >= 0 && slot < p.pairs) {
      const T* g = static_cast<const T*>(p.src) + i / p.topk * p.src_stride;
      const T* y = static_cast<const T*>(p.y) + slot * p.y_stride;
      T* d = static_cast<T*>(p.dst) + slot * p.dst_stride;
      const float w = p.weights ? __ldg(p.weights + i) : 1.0f;
      for (int c = lane * V; c < p.cols; c += 32 * V) {
        const Piece<T, V> a = LoadPiece<T, V>(g + c);
        if (p.grad_weights != nullptr) {
          const Piece<T, V> b = LoadPiece<T, V>(y + c);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dot = fmaf(Widen(a.v[k]), Widen(b.v[k]), dot);
          }
        }
        if (p.dst != nullptr) {
          Piece<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) o.v[k] = Narrow<T>(w * Widen(a.v[k]));
          StorePiece<T, V>(d + c, o);
        }
      }
    }
    if (p.grad_weights != nullptr) {
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      if (lane == 0) p.grad_weights[i] = dot;
    }
  }
  if (p.dst != nullptr) ZeroTail<T>(p);
}

int BlocksFor(int64_t work) {
  const int64_t b = (work + kThreads - 1) / kThreads;
  const int64_t most = static_cast<int64_t>(kNumSms) * 8;  // one wave
  return static_cast<int>(b < 1 ? 1 : (b > most ? most : b));
}

enum : int { kGather, kCombine, kBackward };

template <typename T, int V>
void LaunchMove(int op, const MoveParams& p, cudaStream_t s) {
  const int64_t pieces = p.tokens * (p.cols / V);
  if (op == kGather) {
    GatherKernel<T, V><<<BlocksFor(pieces), kThreads, 0, s>>>(p);
  } else if (op == kCombine) {
    CombineKernel<T, V><<<BlocksFor(pieces), kThreads, 0, s>>>(p);
  } else {
    CombineBackwardKernel<T, V>
        <<<BlocksFor(p.pairs * 32), kThreads, 0, s>>>(p);
  }
}

template <typename T>
void LaunchMoveAs(int op, const MoveParams& p, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = p.cols % kV == 0 && Aligned16(p.src) && Aligned16(p.y) &&
                   Aligned16(p.dst) && p.src_stride % kV == 0 &&
                   p.y_stride % kV == 0 && p.dst_stride % kV == 0;
  if (vec) {
    LaunchMove<T, kV>(op, p, s);
  } else {
    LaunchMove<T, 1>(op, p, s);
  }
}

int RunMove(int op, int32_t dtype, const MoveParams& p, const char* what,
            cudaStream_t s) {
  if (dtype == XSE_DT_F32) LaunchMoveAs<float>(op, p, s);
  if (dtype == XSE_DT_BF16) LaunchMoveAs<__nv_bfloat16>(op, p, s);
  const int rc = LaunchStatus(what);
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

int CheckRows(const xse_expert_plan* plan, int32_t dtype, int32_t cols) {
  if (int rc = CheckExpertPlan(plan); rc != XSE_OK) return rc;
  if (dtype != XSE_DT_F32 && dtype != XSE_DT_BF16) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "Expert rows are float32 or bfloat16, got type %d", dtype);
  }
  if (cols < 1) {
    return FailWith(XSE_INVALID_ARGUMENT, "Expert rows need cols >= 1.");
  }
  return XSE_OK;
}

MoveParams ParamsOf(const xse_expert_plan& plan, int32_t cols) {
  MoveParams p{};
  p.offsets = plan.offsets;
  p.slots = plan.slots;
  p.tokens = plan.tokens;
  p.pairs = plan.tokens * plan.topk;
  p.topk = plan.topk;
  p.num_experts = plan.num_experts;
  p.cols = cols;
  return p;
}

constexpr char kStrides[] = "Expert rows need row strides >= cols.";
constexpr char kNull[] = "Expert row buffers must be non-null.";

}  // namespace
}  // namespace xse

extern "C" {

int xse_expert_sort(const void* ids, int32_t ids_type,
                    const xse_expert_plan* plan, void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckExpertPlan(plan); rc != XSE_OK) return rc;
  if (ids_type != XSE_INDEX_I32 && ids_type != XSE_INDEX_I64) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "Expert ids must be int32 or int64.");
  }
  if (plan->tokens > 0 && ids == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT, "Expert ids must be non-null.");
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = ids_type == XSE_INDEX_I64 ? LaunchSort<long long>(ids, *plan, s)
                                           : LaunchSort<int>(ids, *plan, s);
  if (rc == XSE_OK) SetLastLaunchCount(1);
  return rc;
}

int xse_expert_gather(const void* x, int32_t dtype, int32_t cols,
                      int64_t x_stride, const xse_expert_plan* plan, void* out,
                      int64_t out_stride, void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckRows(plan, dtype, cols); rc != XSE_OK) return rc;
  if (x_stride < cols || out_stride < cols) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kStrides);
  }
  if (plan->tokens == 0) return XSE_OK;
  if (x == nullptr || out == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kNull);
  }
  MoveParams p = ParamsOf(*plan, cols);
  p.src = x;
  p.src_stride = x_stride;
  p.dst = out;
  p.dst_stride = out_stride;
  return RunMove(kGather, dtype, p, "expert gather",
                 static_cast<cudaStream_t>(stream));
}

int xse_expert_combine(const void* y, int32_t dtype, int32_t cols,
                       int64_t y_stride, const xse_expert_plan* plan,
                       const float* weights, void* out, int64_t out_stride,
                       void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckRows(plan, dtype, cols); rc != XSE_OK) return rc;
  if (y_stride < cols || out_stride < cols) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kStrides);
  }
  if (plan->tokens == 0) return XSE_OK;
  if (y == nullptr || out == nullptr) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kNull);
  }
  MoveParams p = ParamsOf(*plan, cols);
  p.src = y;
  p.src_stride = y_stride;
  p.dst = out;
  p.dst_stride = out_stride;
  p.weights = weights;
  return RunMove(kCombine, dtype, p, "expert combine",
                 static_cast<cudaStream_t>(stream));
}

int xse_expert_combine_backward(const void* grad, const void* y, int32_t dtype,
                                int32_t cols, int64_t grad_stride,
                                int64_t y_stride, const xse_expert_plan* plan,
                                const float* weights, void* grad_y,
                                int64_t grad_y_stride, float* grad_weights,
                                void* stream) {
  using namespace xse;
  SetLastLaunchCount(0);
  if (int rc = CheckRows(plan, dtype, cols); rc != XSE_OK) return rc;
  if (grad_stride < cols || (grad_weights != nullptr && y_stride < cols) ||
      (grad_y != nullptr && grad_y_stride < cols)) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kStrides);
  }
  if (plan->tokens == 0 || (grad_y == nullptr && grad_weights == nullptr)) {
    return XSE_OK;
  }
  if (grad == nullptr || (grad_weights != nullptr && y == nullptr)) {
    return FailWith(XSE_INVALID_ARGUMENT, "%s", kNull);
  }
  MoveParams p = ParamsOf(*plan, cols);
  p.src = grad;
  p.src_stride = grad_stride;
  if (grad_weights != nullptr) {
    p.y = y;
    p.y_stride = y_stride;
  }
  if (grad_y != nullptr) {
    p.dst = grad_y;
    p.dst_stride = grad_y_stride;
  }
  p.grad_weights = grad_weights;
  p.weights = weights;
  return RunMove(kBackward, dtype, p, "expert combine backward",
                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"
