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
constexpr int kChoices = 8;  // a token's choices handled at a time

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
  uint32_t src_bytes, y_bytes, dst_bytes;  // the strides, where they fit
  int32_t topk, num_experts, cols;
  int32_t row_shift;   // 2^row_shift threads share a token's row
  int32_t quads;       // rows of slots and weights are whole 16-byte quads
};

// Zeros behind the last sorted row of a [pairs, cols] output.
template <typename T, int V>
__device__ __forceinline__ void ZeroTail(const MoveParams& p) {
  const int64_t kept = max(0, __ldg(p.offsets + p.num_experts));
  Piece<T, V> zero;
#pragma unroll
  for (int k = 0; k < V; ++k) zero.v[k] = Narrow<T>(0.0f);
  for (int64_t r = kept + blockIdx.x; r < p.pairs; r += gridDim.x) {
    T* row = static_cast<T*>(p.dst) + r * p.dst_stride;
    for (int c = threadIdx.x * V; c < p.cols; c += blockDim.x * V) {
      StorePiece<T, V>(row + c, zero);
    }
  }
}

// The sorted row of choice j of token t, -1 for none.
__device__ __forceinline__ int32_t SlotOf(const MoveParams& p, int64_t t,
                                          int j) {
  if (j >= p.topk) return -1;
  const int32_t slot = __ldg(p.slots + t * p.topk + j);
  return slot < p.pairs ? slot : -1;
}

// The sorted rows of choices [first, first + kChoices) of token t, -1 for none.
__device__ __forceinline__ void LoadSlots(const MoveParams& p, int64_t t,
                                          int first, int32_t (&slot)[kChoices]) {
#pragma unroll
  for (int j = 0; j < kChoices; ++j) {
    slot[j] = SlotOf(p, t, first + j);
  }
}

// 2^row_shift threads per token, a piece each at a time: the row is read once
// and stored for all its choices.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    GatherKernel(const __grid_constant__ MoveParams p) {
  const int per_block = kThreads >> p.row_shift;
  const int mine = threadIdx.x >> p.row_shift;
  const int lane = threadIdx.x & ((1 << p.row_shift) - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block + mine;
       t < p.tokens; t += static_cast<int64_t>(gridDim.x) * per_block) {
    const T* x = static_cast<const T*>(p.src) + t * p.src_stride;
    for (int first = 0; first < p.topk; first += kChoices) {
      int32_t slot[kChoices];
      LoadSlots(p, t, first, slot);
      for (int c = lane * V; c < p.cols; c += V << p.row_shift) {
        const Piece<T, V> r = LoadPiece<T, V>(x + c);
#pragma unroll
        for (int j = 0; j < kChoices; ++j) {
          if (slot[j] < 0) continue;
          StorePiece<T, V>(
              static_cast<T*>(p.dst) + slot[j] * p.dst_stride + c, r);
        }
      }
    }
  }
  ZeroTail<T, V>(p);
}

// Rings. A thread copies its 16 bytes of up to kC choices' rows into slots of
// its own in shared memory with cp.async, several steps ahead of the step it
// adds up: about 190 KB of rows are in flight per SM without holding a
// register, and no thread waits for another.
constexpr int kRingThreads = 512;
constexpr int kRingSlots = 24;  // 16-byte slots per thread
constexpr int kRingBytes = kRingThreads * kRingSlots * 16;

template <int kC>
struct Ring {
  static constexpr int kSteps = kRingSlots / kC < 8 ? kRingSlots / kC : 8;

  // Slots are interleaved by thread: 16-byte accesses of a warp are contiguous.
  __device__ static uint4* Slot(uint4* ring, int step, int j) {
    return ring + (step * kC + j) * kRingThreads + threadIdx.x;
  }
  __device__ static void Copy(uint4* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
  }
  __device__ static void Commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // All but the newest kSteps - 1 groups have landed.
  __device__ static void Wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSteps - 1) : "memory");
  }
};

// Entries [first, first + kC) of token t's row of a [tokens, topk] array, as
// quads where rows allow it; `none` past the last.
template <int kC, typename E>
__device__ __forceinline__ void LoadChoices(const MoveParams& p, const E* a,
                                            int64_t t, int first, E none,
                                            E (&v)[kC]) {
  const E* row = a + t * p.topk + first;
  if constexpr (kC >= 4) {
    if (p.quads) {
#pragma unroll
      for (int j = 0; j < kC; j += 4) {
        uint4 u = make_uint4(0, 0, 0, 0);
        const bool there = first + j < p.topk;
        if (there) u = __ldg(reinterpret_cast<const uint4*>(row + j));
        __builtin_memcpy(&v[j], &u.x, 4);
        __builtin_memcpy(&v[j + 1], &u.y, 4);
        __builtin_memcpy(&v[j + 2], &u.z, 4);
        __builtin_memcpy(&v[j + 3], &u.w, 4);
        if (!there) v[j] = v[j + 1] = v[j + 2] = v[j + 3] = none;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < kC; ++j) {
    v[j] = first + j < p.topk ? __ldg(row + j) : none;
  }
}

__device__ __forceinline__ bool Kept(const MoveParams& p, int32_t slot) {
  return static_cast<uint32_t>(slot) < p.pairs;
}

// acc[k] += w * piece[k] in fp32, two at a time.
__device__ __forceinline__ void Fma2(float2& acc, float2 a, float2 b) {
  uint64_t c = reinterpret_cast<uint64_t&>(acc);
  asm("fma.rn.f32x2 %0, %1, %2, %0;"
      : "+l"(c)
      : "l"(reinterpret_cast<uint64_t&>(a)),
        "l"(reinterpret_cast<uint64_t&>(b)));
  reinterpret_cast<uint64_t&>(acc) = c;
}

// A 16-byte piece widened to pairs of floats.
template <typename T>
struct Pairs {
  static constexpr int kN = 8 / sizeof(T);
  float2 v[kN];
  __device__ explicit Pairs(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = make_float2(__uint_as_float(w[i] << 16),
                           __uint_as_float(w[i] & 0xffff0000u));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[i] = make_float2(__uint_as_float(w[2 * i]),
                           __uint_as_float(w[2 * i + 1]));
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ uint4 NarrowPairs(const float2* v) {
  Piece<T, 16 / sizeof(T)> o;
#pragma unroll
  for (int i = 0; i < Pairs<T>::kN; ++i) {
    o.v[2 * i] = Narrow<T>(v[i].x);
    o.v[2 * i + 1] = Narrow<T>(v[i].y);
  }
  uint4 u;
  __builtin_memcpy(&u, &o, 16);
  return u;
}

// The address of byte `at` of sorted row `slot` (rows closer than 4 GB).
__device__ __forceinline__ const char* SortedRow(const void* base,
                                                 uint32_t row_bytes,
                                                 int32_t slot, uint32_t at) {
  return static_cast<const char*>(base) +
         static_cast<uint64_t>(static_cast<uint32_t>(slot)) * row_bytes + at;
}

// Steps of a thread: tokens, then pieces of the row, then groups of choices.
// The slots of the next step to copy are loaded a step early.
template <typename T, int kC>
__global__ void __launch_bounds__(kRingThreads, 1)
    CombineRingKernel(const __grid_constant__ MoveParams p) {
  using R = Ring<kC>;
  constexpr int kN = Pairs<T>::kN;
  extern __shared__ uint4 ring[];
  const int per_block = kRingThreads >> p.row_shift;
  const uint32_t lane = (threadIdx.x & ((1 << p.row_shift) - 1)) * 16;
  const uint32_t row_end = p.cols * static_cast<uint32_t>(sizeof(T));
  const int64_t step_t = static_cast<int64_t>(gridDim.x) * per_block;
  struct At {
    int64_t t;
    uint32_t byte;
    int first;
  };
  const auto next = [&](At& at) {
    at.first += kC;
    if (at.first < p.topk) return;
    at.first = 0;
    at.byte += 16u << p.row_shift;
    if (at.byte < row_end) return;
    at.byte = lane;
    at.t += step_t;
  };
  At tail{static_cast<int64_t>(blockIdx.x) * per_block +
              (threadIdx.x >> p.row_shift),
          lane, 0};
  if (lane >= row_end) tail.t = p.tokens;
  At head = tail;
  int32_t ahead[kC];
  if (head.t < p.tokens) {
    LoadChoices<kC>(p, p.slots, head.t, head.first, -1, ahead);
  }
  int in = 0;
  const auto issue = [&] {
    if (head.t < p.tokens) {
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        if (Kept(p, ahead[j])) {
          R::Copy(R::Slot(ring, in, j),
                  SortedRow(p.src, p.src_bytes, ahead[j], head.byte));
        }
      }
      next(head);
      if (head.t < p.tokens) {
        LoadChoices<kC>(p, p.slots, head.t, head.first, -1, ahead);
      }
    }
    R::Commit();
    in = in + 1 == R::kSteps ? 0 : in + 1;
  };
  for (int i = 0; i < R::kSteps - 1; ++i) issue();
  float2 sum[kN];
#pragma unroll
  for (int k = 0; k < kN; ++k) sum[k] = make_float2(0.0f, 0.0f);
  for (int out = 0; tail.t < p.tokens;
       out = out + 1 == R::kSteps ? 0 : out + 1) {
    issue();
    int32_t slot[kC];
    float w[kC];
    LoadChoices<kC>(p, p.slots, tail.t, tail.first, -1, slot);
    if (p.weights != nullptr) {
      LoadChoices<kC>(p, p.weights, tail.t, tail.first, 0.0f, w);
    } else {
#pragma unroll
      for (int j = 0; j < kC; ++j) w[j] = 1.0f;
    }
    R::Wait();
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      if (!Kept(p, slot[j])) continue;
      const Pairs<T> r(*R::Slot(ring, out, j));
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        Fma2(sum[k], make_float2(w[j], w[j]), r.v[k]);
      }
    }
    const At at = tail;
    next(tail);
    if (tail.first != 0) continue;
    char* dst = static_cast<char*>(p.dst) +
                at.t * p.dst_stride * static_cast<int64_t>(sizeof(T)) + at.byte;
    __stcs(reinterpret_cast<uint4*>(dst), NarrowPairs<T>(sum));
#pragma unroll
    for (int k = 0; k < kN; ++k) sum[k] = make_float2(0.0f, 0.0f);
  }
}

// Up to 32 threads per token, so that its dot products are added with
// shuffles. Steps of a thread: tokens, then groups of choices, then pieces.
// All threads of a block take the same steps.
template <typename T, int kC>
__global__ void __launch_bounds__(kRingThreads, 1)
    CombineBackwardRingKernel(const __grid_constant__ MoveParams p) {
  using R = Ring<kC>;
  constexpr int kN = Pairs<T>::kN;
  extern __shared__ uint4 ring[];
  const int per_block = kRingThreads >> p.row_shift;
  const uint32_t lane = (threadIdx.x & ((1 << p.row_shift) - 1)) * 16;
  const uint32_t row_end = p.cols * static_cast<uint32_t>(sizeof(T));
  const int64_t step_t = static_cast<int64_t>(gridDim.x) * per_block;
  const int mine = threadIdx.x >> p.row_shift;
  const bool dots = p.grad_weights != nullptr;
  struct At {
    int64_t t;  // of the block's first thread
    int first;
    uint32_t byte;
  };
  const auto next = [&](At& at) {
    at.byte += 16u << p.row_shift;
    if (at.byte < row_end) return;
    at.byte = 0;
    at.first += kC;
    if (at.first < p.topk) return;
    at.first = 0;
    at.t += step_t;
  };
  const auto live = [&](const At& at) {
    return at.t + mine < p.tokens && at.byte + lane < row_end;
  };
  const auto load = [&](const At& at, int32_t(&slot)[kC]) {
    if (live(at)) {
      LoadChoices<kC>(p, p.slots, at.t + mine, at.first, -1, slot);
    } else {
#pragma unroll
      for (int j = 0; j < kC; ++j) slot[j] = -1;
    }
  };
  At tail{static_cast<int64_t>(blockIdx.x) * per_block, 0, 0};
  At head = tail;
  int32_t ahead[kC];
  load(head, ahead);
  int in = 0;
  const auto issue = [&] {
    if (dots && head.t < p.tokens) {
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        if (Kept(p, ahead[j])) {
          R::Copy(R::Slot(ring, in, j),
                  SortedRow(p.y, p.y_bytes, ahead[j], head.byte + lane));
        }
      }
      next(head);
      load(head, ahead);
    }
    R::Commit();
    in = in + 1 == R::kSteps ? 0 : in + 1;
  };
  for (int i = 0; i < R::kSteps - 1; ++i) issue();
  float2 dot[kC];
#pragma unroll
  for (int j = 0; j < kC; ++j) dot[j] = make_float2(0.0f, 0.0f);
  for (int out = 0; tail.t < p.tokens;
       out = out + 1 == R::kSteps ? 0 : out + 1) {
    const int64_t t = tail.t + mine;
    const bool here = live(tail);
    uint4 g = make_uint4(0, 0, 0, 0);
    if (here) {
      g = __ldcs(reinterpret_cast<const uint4*>(
          static_cast<const char*>(p.src) +
          t * p.src_stride * static_cast<int64_t>(sizeof(T)) + tail.byte +
          lane));
    }
    issue();
    int32_t slot[kC];
    load(tail, slot);
    const Pairs<T> a(g);
    if (p.dst != nullptr) {
      float w[kC];
#pragma unroll
      for (int j = 0; j < kC; ++j) w[j] = 1.0f;
      if (here && p.weights != nullptr) {
        LoadChoices<kC>(p, p.weights, t, tail.first, 0.0f, w);
      }
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        if (!Kept(p, slot[j])) continue;
        float2 o[kN];
#pragma unroll
        for (int k = 0; k < kN; ++k) {
          o[k] = make_float2(w[j] * a.v[k].x, w[j] * a.v[k].y);
        }
        __stcs(reinterpret_cast<uint4*>(const_cast<char*>(
                   SortedRow(p.dst, p.dst_bytes, slot[j], tail.byte + lane))),
               NarrowPairs<T>(o));
      }
    }
    R::Wait();
    if (dots) {
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        if (!Kept(p, slot[j])) continue;
        const Pairs<T> b(*R::Slot(ring, out, j));
#pragma unroll
        for (int k = 0; k < kN; ++k) Fma2(dot[j], a.v[k], b.v[k]);
      }
    }
    const At at = tail;
    next(tail);
    if (tail.byte != 0 || !dots) continue;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      float sum = dot[j].x + dot[j].y;
      for (int o = (1 << p.row_shift) >> 1; o >= 1; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      if (lane == 0 && t < p.tokens && at.first + j < p.topk) {
        p.grad_weights[t * p.topk + at.first + j] = sum;
      }
      dot[j] = make_float2(0.0f, 0.0f);
    }
  }
  if (p.dst != nullptr) ZeroTail<T, 16 / sizeof(T)>(p);
}

// Rows at any alignment: one element at a time, several tokens per block.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    CombineKernel(const __grid_constant__ MoveParams p) {
  const int per_block = kThreads >> p.row_shift;
  const int lane = threadIdx.x & ((1 << p.row_shift) - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block +
                   (threadIdx.x >> p.row_shift);
       t < p.tokens; t += static_cast<int64_t>(gridDim.x) * per_block) {
    for (int c = lane; c < p.cols; c += 1 << p.row_shift) {
      float sum = 0.0f;
#pragma unroll 4
      for (int j = 0; j < p.topk; ++j) {
        const int32_t slot = SlotOf(p, t, j);
        if (slot < 0) continue;
        const float w = p.weights ? __ldg(p.weights + t * p.topk + j) : 1.0f;
        sum = fmaf(w, Widen(static_cast<const T*>(p.src)[slot * p.src_stride +
                                                         c]), sum);
      }
      static_cast<T*>(p.dst)[t * p.dst_stride + c] = Narrow<T>(sum);
    }
  }
}

// The same for the gradients: one warp per (token, choice).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    CombineBackwardKernel(const __grid_constant__ MoveParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) +
                   threadIdx.x / 32;
       i < p.pairs; i += warps) {
    const int64_t t = i / p.topk;
    const int32_t slot = SlotOf(p, t, static_cast<int>(i - t * p.topk));
    float dot = 0.0f;
    if (slot >= 0) {
      const T* g = static_cast<const T*>(p.src) + t * p.src_stride;
      const T* y = static_cast<const T*>(p.y) + slot * p.y_stride;
      T* d = static_cast<T*>(p.dst) + slot * p.dst_stride;
      const float w = p.weights ? __ldg(p.weights + i) : 1.0f;
#pragma unroll 4
      for (int c = lane; c < p.cols; c += 32) {
        const float a = Widen(g[c]);
        if (p.grad_weights != nullptr) dot = fmaf(a, Widen(y[c]), dot);
        if (p.dst != nullptr) d[c] = Narrow<T>(w * a);
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
  if (p.dst != nullptr) ZeroTail<T, 1>(p);
}

enum : int { kGather, kCombine, kBackward };

// The smallest 2^n <= `most` threads with a piece each.
int ThreadShift(int pieces, int most) {
  int shift = 0;
  while ((1 << shift) < pieces && (2 << shift) <= most) ++shift;
  return shift;
}

int Blocks(int64_t work, int per_block, int per_sm) {
  const int64_t need = (work + per_block - 1) / per_block;
  const int64_t most = static_cast<int64_t>(kNumSms) * per_sm;  // one wave
  return static_cast<int>(need < 1 ? 1 : need > most ? most : need);
}

template <typename T, int kC>
cudaError_t LaunchRing(int op, MoveParams p, cudaStream_t s) {
  const auto kernel = op == kCombine ? CombineRingKernel<T, kC>
                                     : CombineBackwardRingKernel<T, kC>;
  p.row_shift = ThreadShift(p.cols / (16 / static_cast<int>(sizeof(T))),
                            op == kCombine ? 256 : 32);
  const cudaError_t e = cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (e != cudaSuccess) return e;
  kernel<<<Blocks(p.tokens, kRingThreads >> p.row_shift, 1), kRingThreads,
           kRingBytes, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t LaunchMove(int op, MoveParams p, bool vec, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  if (op == kGather) {
    p.row_shift = ThreadShift(vec ? p.cols / kV : p.cols, kThreads);
    const int blocks = Blocks(p.tokens, kThreads >> p.row_shift, 8);
    if (vec) {
      GatherKernel<T, kV><<<blocks, kThreads, 0, s>>>(p);
    } else {
      GatherKernel<T, 1><<<blocks, kThreads, 0, s>>>(p);
    }
  } else if (vec) {
    return p.topk == 1   ? LaunchRing<T, 1>(op, p, s)
           : p.topk == 2 ? LaunchRing<T, 2>(op, p, s)
           : p.topk <= 4 ? LaunchRing<T, 4>(op, p, s)
                         : LaunchRing<T, 8>(op, p, s);
  } else if (op == kCombine) {
    p.row_shift = ThreadShift(p.cols, kThreads);
    CombineKernel<T><<<Blocks(p.tokens, kThreads >> p.row_shift, 8), kThreads,
                       0, s>>>(p);
  } else {
    CombineBackwardKernel<T>
        <<<Blocks(p.pairs, kThreads / 32, 8), kThreads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t LaunchMoveAs(int op, MoveParams p, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  constexpr int64_t kMost = (int64_t{1} << 32) / sizeof(T);
  const bool vec = p.cols % kV == 0 && Aligned16(p.src) && Aligned16(p.y) &&
                   Aligned16(p.dst) && p.src_stride % kV == 0 &&
                   p.y_stride % kV == 0 && p.dst_stride % kV == 0 &&
                   p.src_stride < kMost && p.y_stride < kMost &&
                   p.dst_stride < kMost;
  p.src_bytes = static_cast<uint32_t>(p.src_stride * sizeof(T));
  p.y_bytes = static_cast<uint32_t>(p.y_stride * sizeof(T));
  p.dst_bytes = static_cast<uint32_t>(p.dst_stride * sizeof(T));
  p.quads = p.topk % 4 == 0 && Aligned16(p.slots) && Aligned16(p.weights);
  return LaunchMove<T>(op, p, vec, s);
}

int RunMove(int op, int32_t dtype, const MoveParams& p, const char* what,
            cudaStream_t s) {
  const cudaError_t e = dtype == XSE_DT_F32
                            ? LaunchMoveAs<float>(op, p, s)
                            : LaunchMoveAs<__nv_bfloat16>(op, p, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return FailWith(XSE_INTERNAL, "%s launch: %s", what,
                    cudaGetErrorString(e));
  }
  SetLastLaunchCount(1);
  return XSE_OK;
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
