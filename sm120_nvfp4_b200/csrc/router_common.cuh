// Pieces shared by the forward and the backward kernels of the router's balance loss: rows of logits in
// the registers of a group of threads, reductions over a group, the choice of the group.
#pragma once

#include <cstdint>
#include <mutex>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.hpp"
#include "internal.hpp"
#include "ptx.cuh"

namespace b200 {
namespace router {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = 4096;
constexpr int kMaxSequences = 65536;
constexpr int kMaxTokens = 1 << 30;     // token numbers a few steps past the end fit 32 bits; so do counts of slots
constexpr float kMinSum = 1e-25f;      // below this the sigmoids of a row are e^z to FP32 precision

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_float(float x, __half* p) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

// 1 / x to one ulp (0 for infinite x, infinity for 0).
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// e^x = 2^(x log2 e) by the exponential instruction: off by 2 + 1.173 |x| units of 2^-23 at most, the same bound as
// __expf's. Results below 2^-126 are 0: beside a row's other scores, which add up to kMinSum at least, they do not count;
// rows that have no larger ones are normalised by their maximum. Scores need no more bits than that: the
// probabilities become sums over tokens, and a gradient of a router.
__device__ __forceinline__ float exponential(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// G threads share the row of a token: 8, 16 or 32 lanes of a warp, which then works on 32 / G tokens at
// a time, or a whole block (256). What a token costs beside its elements - ids, votes, exchanges - is
// issued once per warp, so narrow groups with 8 to 20 columns per thread beat one warp per token
// (131072 x 160 BF16: loss 62 us with a warp per token, 46 with groups; gradient 91 and 53).
template <int G>
struct Group {
  static constexpr int kPerWarp = G >= 32 ? 1 : 32 / G;
  static constexpr int kPerBlock = G > 32 ? 1 : kWarps * kPerWarp;
  static __device__ __forceinline__ int lane() { return G > 32 ? threadIdx.x : threadIdx.x & (G - 1); }
  static __device__ __forceinline__ int in_warp() { return G >= 32 ? 0 : (threadIdx.x & 31) / G; }
  static __device__ __forceinline__ int index() { return G > 32 ? 0 : threadIdx.x / G; }

  // sum / maximum over the group; every thread gets the result
  static __device__ __forceinline__ float sum(float x, float* scratch) {
#pragma unroll
    for (int d = (G > 32 ? 32 : G) / 2; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if constexpr (G > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
      __syncthreads();
      x = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) x += scratch[w];
    }
    return x;
  }
  static __device__ __forceinline__ float max(float x, float* scratch) {
#pragma unroll
    for (int d = (G > 32 ? 32 : G) / 2; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    if constexpr (G > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
      __syncthreads();
      x = scratch[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) x = fmaxf(x, scratch[w]);
    }
    return x;
  }
  static __device__ __forceinline__ bool any(bool x) {
    if constexpr (G > 32) return __syncthreads_or(x) != 0;
    const unsigned votes = __ballot_sync(0xffffffffu, x);
    if constexpr (G == 32) return votes != 0;
    return ((votes >> (in_warp() * G)) & ((1u << (G & 31)) - 1u)) != 0;
  }
  // whether any thread that shares the instruction stream needs a path: the answer is uniform
  static __device__ __forceinline__ bool any_here(bool x) {
    if constexpr (G > 32) return __syncthreads_or(x) != 0;
    return __any_sync(0xffffffffu, x);
  }
  static __device__ __forceinline__ void sync() {
    if constexpr (G > 32) __syncthreads();
    else __syncwarp();
  }
};

// Thread `lane` of G holds columns (i * G + lane) * V + j of a row. The rows of the next kDepth - 1 steps are
// on their way into shared memory while one is worked on: every thread copies its own columns and
// reads them back itself, so the queue needs no barrier, only the count of its own outstanding copies.
// (One row ahead in registers left 20 KB in flight per SM, 1.3 TB/s.)
constexpr int kDepth = 4;

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}

template <typename T, int V, int NV, int G, bool kLoose = V == 1 && sizeof(T) == 2>
struct RowQueue {
  using Part = Vec<T, V>;
  static constexpr size_t kBytes = static_cast<size_t>(kDepth) * NV * kThreads * sizeof(Part);   // per block
  static constexpr int kStage = NV * kThreads * static_cast<int>(sizeof(Part));
  uint8_t* mine;                                            // this thread's first part
  __device__ __forceinline__ RowQueue(void* smem, const T*, int, int) : mine(static_cast<uint8_t*>(smem) + threadIdx.x * sizeof(Part)) {}
  __device__ __forceinline__ void push(int stage, const T* row, int experts, int lane) {
    uint8_t* to = mine + stage * kStage;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * G + lane) * V;
      if (col < experts)
        copy_async<static_cast<int>(sizeof(Part))>(static_cast<uint32_t>(__cvta_generic_to_shared(to + i * kThreads * sizeof(Part))), row + col);
    }
  }
  // Columns past the end are -infinity, whose score is zero; no copy ever touches them.
  __device__ __forceinline__ void fill_rest(int experts, int lane) {
    Part rest;
#pragma unroll
    for (int j = 0; j < V; ++j) from_float(__int_as_float(0xff800000), &rest.v[j]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + lane) * V < experts) continue;
      for (int stage = 0; stage < kDepth; ++stage) *reinterpret_cast<Part*>(mine + stage * kStage + i * kThreads * sizeof(Part)) = rest;
    }
  }
  // the row of the step whose copies queue_wait() has waited for
  __device__ __forceinline__ void pop(int stage, const T*, float (&z)[V * NV], int, int) const {
    const uint8_t* from = mine + stage * kStage;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Part w = *reinterpret_cast<const Part*>(from + i * kThreads * sizeof(Part));
#pragma unroll
      for (int j = 0; j < V; ++j) z[i * V + j] = to_float(w.v[j]);
    }
  }
  // one column of that row, whichever thread has copied it (after a Group::sync())
  __device__ __forceinline__ float at(int stage, const T*, int col, int lane) const {
    const int part = col / V;
    const uint8_t* from = mine + stage * kStage + (part / G * kThreads + part % G - lane) * static_cast<int>(sizeof(Part));
    return to_float(reinterpret_cast<const Part*>(from)->v[col % V]);
  }
};

// 16-bit rows that cannot be copied by the column (asynchronous copies have 4 bytes at least): the group
// copies the 16-byte chunks that a row lies in, clipped to the matrix, and its threads pick their columns
// i * G + lane out of them. (FP32 rows do better with copies of 4 bytes: 65536 x 255 33 against 37 us.)
template <typename T, int NV, int G>
struct RowQueue<T, 1, NV, G, true> {
  static constexpr int kRow = (NV * G * static_cast<int>(sizeof(T)) + 15) / 16 * 16 + 16;
  static constexpr size_t kBytes = static_cast<size_t>(kDepth) * Group<G>::kPerBlock * kRow;
  uint8_t* mine;                                            // this group's first row
  const uint8_t *first, *last;                              // ends of the matrix
  __device__ __forceinline__ RowQueue(void* smem, const T* matrix, int tokens, int experts)
      : mine(static_cast<uint8_t*>(smem) + Group<G>::index() * kDepth * kRow),
        first(reinterpret_cast<const uint8_t*>(matrix)),
        last(reinterpret_cast<const uint8_t*>(matrix + static_cast<long long>(tokens) * experts)) {}
  __device__ __forceinline__ void push(int stage, const T* row, int experts, int lane) {
    const uint8_t* begin = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(15));
    const uint8_t* end = reinterpret_cast<const uint8_t*>(row + experts);
    for (int c = lane * 16; begin + c < end; c += G * 16) {
      uint8_t* to = mine + stage * kRow + c;
      if (begin + c >= first) {
        const int bytes = static_cast<int>(min(static_cast<long long>(16), static_cast<long long>(last - (begin + c))));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                     "l"(begin + c), "r"(bytes)
                     : "memory");
      } else {                                              // the chunk that starts before an unaligned matrix
        for (const uint8_t* x = first; x < begin + c + 16 && x < end; x += sizeof(T))
          *reinterpret_cast<T*>(to + (x - (begin + c))) = *reinterpret_cast<const T*>(x);
      }
    }
  }
  __device__ __forceinline__ void fill_rest(int, int) {}
  __device__ __forceinline__ void pop(int stage, const T* row, float (&z)[NV], int experts, int lane) const {
    Group<G>::sync();                                       // the other threads' copies have landed too
    const T* from = reinterpret_cast<const T*>(mine + stage * kRow + (reinterpret_cast<uintptr_t>(row) & 15));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = i * G + lane;
      z[i] = col < experts ? to_float(from[col]) : __int_as_float(0xff800000);
    }
    Group<G>::sync();                                       // before the place is filled again
  }
  __device__ __forceinline__ float at(int stage, const T* row, int col, int) const {
    return to_float(reinterpret_cast<const T*>(mine + stage * kRow + (reinterpret_cast<uintptr_t>(row) & 15))[col]);
  }
};

// A queue of one 4-byte word per thread and step.
template <typename T>
struct WordQueue {
  static constexpr size_t kBytes = static_cast<size_t>(kDepth) * kThreads * 4;
  T* mine;
  __device__ __forceinline__ explicit WordQueue(void* smem) : mine(static_cast<T*>(smem) + threadIdx.x) {}
  __device__ __forceinline__ void push(int stage, const T* src) {
    copy_async<4>(static_cast<uint32_t>(__cvta_generic_to_shared(mine + stage * kThreads)), src);
  }
  __device__ __forceinline__ T pop(int stage) const { return mine[stage * kThreads]; }
};

// Ends a step's copies / waits until those of the oldest of kDepth steps have landed (this thread's own).
__device__ __forceinline__ void queue_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void queue_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory"); }

// z -> e^(z - max); returns one over their sum, 0 for a row of -infinity (it has no probabilities).
template <int N, int G>
__device__ __forceinline__ float exponentials(float (&z)[N], float* scratch) {
  float top = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
  top = Group<G>::max(top, scratch);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    z[i] = z[i] == __int_as_float(0xff800000) ? 0.0f : exponential(z[i] - top);
    sum += z[i];
  }
  sum = Group<G>::sum(sum, scratch);
  return sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
}

// Groups by the number of experts: four columns per load where rows allow it, few idle lanes, at most
// 20 columns per thread; a block per token beyond 512 experts.
template <typename T, template <typename, int, int, int> class Launch, typename... Args>
int dispatch_width(int experts, bool quads, Args... args) {
  if (quads) {
    if (experts <= 32) return Launch<T, 4, 1, 8>::run(args...);
    if (experts <= 64) return Launch<T, 4, 2, 8>::run(args...);
    if (experts <= 128) return Launch<T, 4, 4, 8>::run(args...);
    // 129 to 160: eight lanes of 20 columns instead of sixteen of 12 (131072 x 132 BF16: loss 25.5 us against 29.8, gradient
    // 29.5 against 41.2; x 160 26.0 / 30.3, 30.0 / 41.6). The queues of FP32 rows this wide would not fit twice per SM.
    if constexpr (sizeof(T) == 2) {
      if (experts <= 160) return Launch<T, 4, 5, 8>::run(args...);
    }
    if (experts <= 192) return Launch<T, 4, 3, 16>::run(args...);
    if (experts <= 256) return Launch<T, 4, 4, 16>::run(args...);
    if (experts <= 384) return Launch<T, 4, 3, 32>::run(args...);
    if (experts <= 512) return Launch<T, 4, 4, 32>::run(args...);
    return Launch<T, 4, 4, 256>::run(args...);
  }
  if (experts <= 64) return Launch<T, 1, 8, 8>::run(args...);
  if (experts <= 128) return Launch<T, 1, 16, 8>::run(args...);
  if (experts <= 192) return Launch<T, 1, 12, 16>::run(args...);
  if (experts <= 256) return Launch<T, 1, 16, 16>::run(args...);
  if (experts <= 512) return Launch<T, 1, 16, 32>::run(args...);
  return Launch<T, 1, 16, 256>::run(args...);
}

// More than 48 KB of dynamic shared memory has to be asked for, once per kernel and device.
template <typename Kernel>
int allow_smem(Kernel kernel, std::once_flag (&once)[64], cudaError_t (&status)[64], int device, int bytes) {
  if (device < 0 || device >= 64) return B200_NVFP4_CUDA_ERROR;
  std::call_once(once[device], [&] { status[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  return status[device] == cudaSuccess ? B200_NVFP4_SUCCESS : B200_NVFP4_CUDA_ERROR;
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline size_t element_size(int dtype) { return dtype == 2 ? 4 : 2; }

inline bool valid_router(int tokens, int experts, int topk, int sequences, int dtype) {
  return tokens >= 0 && tokens <= kMaxTokens && static_cast<long long>(tokens) * topk <= 0x7fffffffLL && experts > 0 && experts <= kMaxExperts && topk > 0 && topk <= experts && sequences > 0 &&
         sequences <= kMaxSequences && dtype >= 0 && dtype <= 2;
}

}  // namespace router
}  // namespace b200
