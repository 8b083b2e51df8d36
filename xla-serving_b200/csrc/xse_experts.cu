// Rows sorted by expert and back (include/xse_experts.h).
//
// Sorting counts each warp's pairs per expert in shared memory, turns the
// counts into first rows, and lets every warp place its pairs in order; no
// order depends on an atomic's. A block per SM, so that the scattered stores of
// `order` spread over all of them (131072 pairs: 39 us in a cluster of eight
// blocks, 9 us so).
// The row movers work token by token, so that a token's row (or its gradient)
// is read once for all its choices; their traffic is the rows themselves, each
// read and written once, and they are bound by HBM bandwidth.

#include "xse_mx_internal.h"

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
constexpr int kSortLoads = 8;  // ids of a thread in flight

// The expert of pair p, `num_experts` for a dropped one.
template <typename Id>
__device__ __forceinline__ int ExpertId(Id id, int num_experts) {
  return id >= 0 && id < num_experts ? static_cast<int>(id) : num_experts;
}

// A warp's pairs [first, last), 32 a step, the ids of kSortLoads steps in
// registers: up to 256 pairs are loaded once for both passes over them.
template <typename Id>
struct WarpPairs {
  const Id* ids;
  int64_t first, last;
  int num_experts, lane;
  int expert[kSortLoads];

  __device__ void Load(int64_t base) {
#pragma unroll
    for (int i = 0; i < kSortLoads; ++i) {
      const int64_t p = base + 32 * i + lane;
      expert[i] =
          p < last ? ExpertId(__ldg(ids + p), num_experts) : num_experts;
    }
  }
  // Calls step(p, expert) for every pair; all lanes take every step, those
  // past `last` with a dropped pair.
  template <typename Step>
  __device__ void ForEach(bool loaded, Step step) {
    for (int64_t base = first; base < last; base += 32 * kSortLoads) {
      if (!loaded) Load(base);
#pragma unroll
      for (int i = 0; i < kSortLoads; ++i) {
        if (base + 32 * i >= last) break;
        step(base + 32 * i + lane, expert[i]);
      }
    }
  }
  __device__ bool Once() const { return last - first <= 32 * kSortLoads; }
};

// Warp w of block b takes the pairs [(b * warps + w) * per_warp, + per_warp).
// With several blocks, a first launch counts each block's pairs per expert.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
    SortCountKernel(const Id* __restrict__ ids, int pairs, int num_experts,
                    int64_t per_warp, int32_t* __restrict__ counts) {
  extern __shared__ int totals[];
  // The next launch may begin; it waits for the counts where it reads them.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = threadIdx.x; e < num_experts; e += kSortThreads) totals[e] = 0;
  __syncthreads();
  const int64_t first =
      (static_cast<int64_t>(blockIdx.x) * kSortWarps + threadIdx.x / 32) *
      per_warp;
  WarpPairs<Id> mine{ids, first,
                     min(first + per_warp, static_cast<int64_t>(pairs)),
                     num_experts, static_cast<int>(threadIdx.x & 31)};
  mine.ForEach(false, [&](int64_t, int e) {
    if (e < num_experts) atomicAdd(totals + e, 1);
  });
  __syncthreads();
  for (int e = threadIdx.x; e < num_experts; e += kSortThreads) {
    counts[static_cast<int64_t>(blockIdx.x) * num_experts + e] = totals[e];
  }
}

// Each warp counts its pairs per expert, the counts become its first rows, and
// it then places its pairs in order, lanes of one expert by rank. `counts`:
// every block's from the launch before, NULL for one block.
// Shared: counts[warps][experts], all[experts], before[experts] (all pairs of
// an expert, and those of the blocks before this one).
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
    SortKernel(const Id* __restrict__ ids, int pairs, int num_experts,
               int64_t per_warp, const int32_t* counts,
               int32_t* __restrict__ offsets, int32_t* __restrict__ order,
               int32_t* __restrict__ slots) {
  extern __shared__ int shared[];
  __shared__ int warp_sums[kSortWarps];
  const int block = blockIdx.x, blocks = gridDim.x;
  const int threads = blockDim.x, warps = threads / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  int* mine = shared + warp * num_experts;
  int* all = shared + warps * num_experts;
  int* before = all + num_experts;
  const int64_t first =
      (static_cast<int64_t>(block) * warps + warp) * per_warp;
  WarpPairs<Id> part{ids, first,
                     min(first + per_warp, static_cast<int64_t>(pairs)),
                     num_experts, lane};
  const bool once = part.Once();
  if (once) part.Load(first);
  for (int i = threadIdx.x; i < (warps + 2) * num_experts; i += threads) {
    shared[i] = 0;
  }
  __syncthreads();
  part.ForEach(once, [&](int64_t, int e) {
    if (e < num_experts) atomicAdd(mine + e, 1);
  });
  if (counts != nullptr) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Warps share the experts (32 at a time) and, where there are more warps
    // than that, the blocks.
    const int chunks = (num_experts + 31) / 32;
    const int groups = chunks < warps ? warps / chunks : 1;
    for (int chunk = warp / groups; chunk < chunks; chunk += warps / groups) {
      const int e = chunk * 32 + lane;
      if (e >= num_experts) continue;
      int sum = 0, earlier = 0;
#pragma unroll 8
      for (int b = warp % groups; b < blocks; b += groups) {
        const int c = counts[static_cast<int64_t>(b) * num_experts + e];
        sum += c;
        if (b < block) earlier += c;
      }
      if (sum != 0) atomicAdd(all + e, sum);
      if (earlier != 0) atomicAdd(before + e, earlier);
    }
  }
  __syncthreads();
  // Experts in turn: counts before each warp within the block, a scan over
  // the experts, and each warp's first row.
  int carry = 0;
  for (int base = 0; base < num_experts; base += threads) {
    const int e = base + threadIdx.x;
    int total = 0;
    if (e < num_experts) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < warps; ++w) {
        const int c = shared[w * num_experts + e];
        shared[w * num_experts + e] = sum;
        sum += c;
      }
      total = counts != nullptr ? all[e] : sum;
    }
    int scan = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    int sums = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sums, o);
      if (lane >= o) sums += up;
    }
    const int earlier = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
    const int begin = carry + scan - total + (warp > 0 ? earlier : 0);
    carry += __shfl_sync(0xffffffffu, sums, 31);
    if (e < num_experts) {
      if (block == 0) {
        offsets[e] = begin;
        if (e == num_experts - 1) offsets[num_experts] = begin + total;
      }
      before[e] += begin;
    }
    __syncthreads();
  }
  const int bits = 32 - __clz(num_experts);
  part.ForEach(once, [&](int64_t p, int e) {
    // Lanes of the same expert, one vote per bit of its number.
    unsigned same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
      const bool set = e >> b & 1;
      const unsigned votes = __ballot_sync(0xffffffffu, set);
      same &= set ? votes : ~votes;
    }
    const int rank = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e < num_experts) {
      row = before[e] + mine[e] + rank;
      order[row] = static_cast<int32_t>(p);
    }
    if (p < part.last) slots[p] = row;
    __syncwarp();
    if (e < num_experts && rank == 0) mine[e] += __popc(same);
    __syncwarp();
  });
  for (int64_t r = static_cast<int64_t>(carry) + block * threads + threadIdx.x;
       r < pairs; r += blocks * threads) {
    order[r] = -1;
  }
}

// Pairs that one block sorts in one launch; more take a block per SM and two.
// 4096 pairs over 128 experts: 8.3 us in one block, 6.7 us in two launches.
constexpr int kSortOneBlock = 2048;

int SortBlocks(int64_t pairs) {
  if (pairs <= kSortOneBlock) return 1;
  const int64_t blocks = (pairs + kSortThreads - 1) / kSortThreads;
  return static_cast<int>(blocks > kNumSms ? kNumSms : blocks);
}

template <typename Id>
cudaError_t LaunchSort(const Id* ids, const xse_expert_plan& plan,
                       int32_t* counts, cudaStream_t s) {
  const int pairs = static_cast<int>(plan.tokens * plan.topk);
  const int blocks = SortBlocks(pairs);
  const int threads = pairs <= 512 ? 256 : kSortThreads, warps = threads / 32;
  const int64_t all_warps = static_cast<int64_t>(blocks) * warps;
  const int64_t per_warp = (pairs + 32 * all_warps - 1) / (32 * all_warps) * 32;
  const size_t row = sizeof(int) * static_cast<size_t>(plan.num_experts);
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = AllowShared(
      SortKernel<Id>, sizeof(int) * (kSortWarps + 2) * XSE_MAX_EXPERTS,
      &allowed);
  if (e != cudaSuccess) return e;
  if (blocks > 1) {
    SortCountKernel<Id><<<blocks, kSortThreads, row, s>>>(
        ids, pairs, plan.num_experts, per_warp, counts);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (warps + 2) * row;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(
      &cfg, SortKernel<Id>, ids, pairs, static_cast<int>(plan.num_experts),
      per_warp, static_cast<const int32_t*>(blocks > 1 ? counts : nullptr),
      plan.offsets, plan.order, plan.slots);
  return e != cudaSuccess ? e : cudaGetLastError();
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
template <typename T>
__global__ void __launch_bounds__(kThreads)
    GatherKernel(const __grid_constant__ MoveParams p) {
  constexpr int V = 16 / sizeof(T);
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
// adds up, without holding a register, and no thread waits for another. The ring
// holds min(24 / kC, 8) steps of kC choices, kC the next of 1, 2, 4 and 8: 192 KB
// of rows per SM for 4 choices and for 8, 144 KB for 3 (whose fourth slot stays
// empty), 128 KB for 2, 64 KB for 1.
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

// Rows at any alignment, one element at a time: a thread has kWide elements of
// a row (a stride of its group's width apart) and kFew choices in flight, which
// stand in for the wide loads.
constexpr int kWide = 4;
constexpr int kFew = 4;

template <typename T>
__device__ __forceinline__ void LoadWide(const T* row, int c, int step,
                                         int cols, float (&v)[kWide]) {
#pragma unroll
  for (int i = 0; i < kWide; ++i) {
    v[i] = c + i * step < cols ? Widen(row[c + i * step]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void StoreWide(T* row, int c, int step, int cols,
                                          const float (&v)[kWide]) {
#pragma unroll
  for (int i = 0; i < kWide; ++i) {
    if (c + i * step < cols) row[c + i * step] = Narrow<T>(v[i]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    GatherElementsKernel(const __grid_constant__ MoveParams p) {
  const int per_block = kThreads >> p.row_shift, step = 1 << p.row_shift;
  const int lane = threadIdx.x & (step - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block +
                   (threadIdx.x >> p.row_shift);
       t < p.tokens; t += static_cast<int64_t>(gridDim.x) * per_block) {
    const T* x = static_cast<const T*>(p.src) + t * p.src_stride;
    for (int c = lane; c < p.cols; c += kWide * step) {
      float v[kWide];
      LoadWide(x, c, step, p.cols, v);
      for (int first = 0; first < p.topk; first += kFew) {
        int32_t slot[kFew];
        LoadChoices<kFew>(p, p.slots, t, first, -1, slot);
#pragma unroll
        for (int j = 0; j < kFew; ++j) {
          if (!Kept(p, slot[j])) continue;
          StoreWide(static_cast<T*>(p.dst) + slot[j] * p.dst_stride, c, step,
                    p.cols, v);
        }
      }
    }
  }
  ZeroTail<T, 1>(p);
}

// The gather of long rows at any alignment goes through shared memory: a block
// loads a piece of a token's row once and writes it to each of its sorted rows
// in whole 128-byte lines of the destination (ragged at the piece's ends),
// 4 bytes a thread, where single elements that follow the source's lines touch
// two lines a warp and half of each word in 16 bits. Taken for rows of more
// than kWide * kThreads elements, which a block of GatherElementsKernel needs
// several steps for; against it, 16384 tokens x 4: 92 us for 162 at 1501 fp32,
// 129 for 215 at 2047, 90 for 121 at 2047 bf16. Shorter rows leave most of a
// block idle between its barriers: 62 us for 42 at 511 fp32, 65 for 67 at 1001
// bf16.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    GatherPiecesKernel(const __grid_constant__ MoveParams p) {
  constexpr int kPieceElements = 2048, kPer = kPieceElements / kThreads;
  constexpr int kWord = 4 / sizeof(T);  // elements of a word
  __shared__ T piece[kPieceElements];
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(p.src) + t * p.src_stride;
    for (int first = 0; first < p.cols; first += kPieceElements) {
      const int count = min(p.cols - first, kPieceElements);
      T v[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = i * kThreads + threadIdx.x;
        if (c < count) v[i] = x[first + c];
      }
      __syncthreads();  // the last piece has been written
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = i * kThreads + threadIdx.x;
        if (c < count) piece[c] = v[i];
      }
      __syncthreads();
      for (int j = 0; j < p.topk; ++j) {
        const int32_t slot = SlotOf(p, t, j);
        if (!Kept(p, slot)) continue;
        T* dst = static_cast<T*>(p.dst) + slot * p.dst_stride + first;
        // Elements from the last line boundary to the first one of the piece.
        const int ahead = static_cast<int>(
            (reinterpret_cast<uintptr_t>(dst) & 127) / sizeof(T));
        for (int e = static_cast<int>(threadIdx.x) * kWord - ahead; e < count;
             e += kThreads * kWord) {
          if constexpr (kWord == 1) {
            if (e >= 0) dst[e] = piece[e];
          } else if (e >= 0 && e + 1 < count) {
            Piece<T, 2> two;
            two.v[0] = piece[e];
            two.v[1] = piece[e + 1];
            uint32_t w;
            __builtin_memcpy(&w, &two, 4);
            *reinterpret_cast<uint32_t*>(dst + e) = w;
          } else if (e >= 0) {
            dst[e] = piece[e];
          } else if (e + 1 >= 0) {
            dst[e + 1] = piece[e + 1];
          }
        }
      }
    }
  }
  ZeroTail<T, 1>(p);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    CombineElementsKernel(const __grid_constant__ MoveParams p) {
  const int per_block = kThreads >> p.row_shift, step = 1 << p.row_shift;
  const int lane = threadIdx.x & (step - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block +
                   (threadIdx.x >> p.row_shift);
       t < p.tokens; t += static_cast<int64_t>(gridDim.x) * per_block) {
    for (int c = lane; c < p.cols; c += kWide * step) {
      float sum[kWide] = {};
      for (int first = 0; first < p.topk; first += kFew) {
        int32_t slot[kFew];
        float w[kFew], v[kFew][kWide];
        LoadChoices<kFew>(p, p.slots, t, first, -1, slot);
        if (p.weights != nullptr) {
          LoadChoices<kFew>(p, p.weights, t, first, 0.0f, w);
        }
#pragma unroll
        for (int j = 0; j < kFew; ++j) {
          if (!Kept(p, slot[j])) continue;
          LoadWide(static_cast<const T*>(p.src) + slot[j] * p.src_stride, c,
                   step, p.cols, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kFew; ++j) {
          if (!Kept(p, slot[j])) continue;
#pragma unroll
          for (int i = 0; i < kWide; ++i) {
            sum[i] = fmaf(p.weights ? w[j] : 1.0f, v[j][i], sum[i]);
          }
        }
      }
      StoreWide(static_cast<T*>(p.dst) + t * p.dst_stride, c, step, p.cols,
                sum);
    }
  }
}

// 2^row_shift warps of a block per token and kFew of its choices, each with a
// part of the row; their parts of a dot product are added in order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    CombineBackwardElementsKernel(const __grid_constant__ MoveParams p) {
  __shared__ float parts[kThreads / 32][kFew];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int share = 1 << p.row_shift, part = warp & (share - 1);
  const int groups = (p.topk + kFew - 1) / kFew;
  const int64_t units = p.tokens * groups;
  const int per_block = kThreads / 32 >> p.row_shift;
  const bool dots = p.grad_weights != nullptr;
  // All warps of a block take the same steps (they meet at barriers).
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_block;
       base < units; base += static_cast<int64_t>(gridDim.x) * per_block) {
    const int64_t u = base + (warp >> p.row_shift);
    const int64_t t = groups == 1 ? u : u / groups;
    const int first = static_cast<int>(u - t * groups) * kFew;
    int32_t slot[kFew];
    float w[kFew], dot[kFew] = {};
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      slot[j] = -1;
      w[j] = 1.0f;
    }
    if (u < units) {
      LoadChoices<kFew>(p, p.slots, t, first, -1, slot);
      if (p.weights != nullptr) {
        LoadChoices<kFew>(p, p.weights, t, first, 0.0f, w);
      }
      const T* grad = static_cast<const T*>(p.src) + t * p.src_stride;
      for (int c = part * 32 * kWide + lane; c < p.cols;
           c += share * 32 * kWide) {
        float g[kWide], v[kFew][kWide];
        LoadWide(grad, c, 32, p.cols, g);
        if (dots) {
#pragma unroll
          for (int j = 0; j < kFew; ++j) {
            if (!Kept(p, slot[j])) continue;
            LoadWide(static_cast<const T*>(p.y) + slot[j] * p.y_stride, c, 32,
                     p.cols, v[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < kFew; ++j) {
          if (!Kept(p, slot[j])) continue;
          if (dots) {
#pragma unroll
            for (int i = 0; i < kWide; ++i) {
              dot[j] = fmaf(g[i], v[j][i], dot[j]);
            }
          }
          if (p.dst != nullptr) {
            float o[kWide];
#pragma unroll
            for (int i = 0; i < kWide; ++i) o[i] = w[j] * g[i];
            StoreWide(static_cast<T*>(p.dst) + slot[j] * p.dst_stride, c, 32,
                      p.cols, o);
          }
        }
      }
    }
    if (!dots) continue;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      }
      if (lane == 0) parts[warp][j] = dot[j];
    }
    if (share > 1) {
      __syncthreads();
    } else {
      __syncwarp();
    }
    if (part == 0 && u < units && lane < kFew && first + lane < p.topk) {
      float sum = 0.0f;
      for (int k = 0; k < share; ++k) sum += parts[warp + k][lane];
      p.grad_weights[t * p.topk + first + lane] = sum;
    }
    if (share > 1) {
      __syncthreads();
    } else {
      __syncwarp();
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
  static std::atomic<uint64_t> allowed[2] = {};
  const auto kernel = op == kCombine ? CombineRingKernel<T, kC>
                                     : CombineBackwardRingKernel<T, kC>;
  p.row_shift = ThreadShift(p.cols / (16 / static_cast<int>(sizeof(T))),
                            op == kCombine ? kRingRowThreads : 32);
  const cudaError_t e =
      AllowShared(kernel, kRingBytes, &allowed[op == kCombine]);
  if (e != cudaSuccess) return e;
  kernel<<<Blocks(p.tokens, kRingThreads >> p.row_shift, 1), kRingThreads,
           kRingBytes, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t LaunchMove(int op, MoveParams p, bool vec, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  if (vec) {
    if (op != kGather) {
      return p.topk == 1   ? LaunchRing<T, 1>(op, p, s)
             : p.topk == 2 ? LaunchRing<T, 2>(op, p, s)
             : p.topk <= 4 ? LaunchRing<T, 4>(op, p, s)
                           : LaunchRing<T, 8>(op, p, s);
    }
    p.row_shift = ThreadShift(p.cols / kV, kThreads);
    GatherKernel<T><<<Blocks(p.tokens, kThreads >> p.row_shift, 8), kThreads,
                      0, s>>>(p);
  } else if (op == kBackward) {
    p.row_shift =
        ThreadShift((p.cols + 32 * kWide - 1) / (32 * kWide), kThreads / 32);
    CombineBackwardElementsKernel<T>
        <<<Blocks(p.tokens * ((p.topk + kFew - 1) / kFew),
                  kThreads / 32 >> p.row_shift, 8),
           kThreads, 0, s>>>(p);
  } else {
    p.row_shift = ThreadShift((p.cols + kWide - 1) / kWide, kThreads);
    const int blocks = Blocks(p.tokens, kThreads >> p.row_shift, 8);
    if (op == kGather && p.cols > kWide * kThreads) {
      GatherPiecesKernel<T><<<Blocks(p.tokens, 1, 8), kThreads, 0, s>>>(p);
    } else if (op == kGather) {
      GatherElementsKernel<T><<<blocks, kThreads, 0, s>>>(p);
    } else {
      CombineElementsKernel<T><<<blocks, kThreads, 0, s>>>(p);
    }
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
                   p.dst_stride < kMost &&
                   (op == kGather || ExpertRowFitsRing(p.cols, sizeof(T)));
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
  if (cols < 1 || cols > kMostColumns) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "Expert rows need 1 <= cols <= 2^30.");
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

int64_t xse_expert_sort_workspace(int64_t pairs, int32_t num_experts) {
  if (pairs < 0 || pairs > INT32_MAX || num_experts < 1 ||
      num_experts > XSE_MAX_EXPERTS) {
    return 0;
  }
  const int blocks = xse::SortBlocks(pairs);
  return blocks == 1 ? 0 : int64_t{4} * blocks * num_experts;
}

int xse_expert_sort(const void* ids, int32_t ids_type,
                    const xse_expert_plan* plan, void* workspace,
                    int64_t workspace_bytes, void* stream) {
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
  const int64_t need = xse_expert_sort_workspace(plan->tokens * plan->topk,
                                                 plan->num_experts);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)) {
    return FailWith(XSE_INVALID_ARGUMENT,
                    "Expert sort needs a 4-byte aligned workspace of %lld "
                    "bytes, got %lld.", static_cast<long long>(need),
                    static_cast<long long>(workspace_bytes));
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t* counts = static_cast<int32_t*>(workspace);
  const cudaError_t e =
      ids_type == XSE_INDEX_I64
          ? LaunchSort(static_cast<const long long*>(ids), *plan, counts, s)
          : LaunchSort(static_cast<const int*>(ids), *plan, counts, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return FailWith(XSE_INTERNAL, "expert sort launch: %s",
                    cudaGetErrorString(e));
  }
  SetLastLaunchCount(need > 0 ? 2 : 1);
  return XSE_OK;
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
