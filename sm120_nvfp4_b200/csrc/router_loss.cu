// Balance loss of the router with per-expert counts, and the router's gradient.
//
// Forward. Token t with logits z: s_e = sigmoid(z_e), p_e = s_e / sum_j s_j (scoring 0), or p =
// softmax(z) (scoring 1). A token counts ("live") when it lies in a sequence and has an id in [0, E).
// Per sequence with T live tokens, of which n_e slots chose expert e:
//   slope_e = alpha * E * n_e / (k * T^2 * S')       (S' = sequences with a live token)
//   loss    = sum over sequences and experts of slope_e * sum_t p_te
// which is the mean over sequences of alpha * sum_e f_e P_e, f_e = n_e E / (k T), P_e = mean_t p_te.
//
// Backward (f is a constant): dz_e = g * p_e (1 - s_e) (slope_e - sum_j slope_j p_j), without the
// (1 - s) for softmax; and for the renormalised weights w_j = s_j / sum of the selected s:
//   dz_j += w_j (1 - s_j) (g_j - sum_i g_i w_i)       for each selected expert j.
// Both terms go out in one pass over the logits.
//
// HBM-bound by design: 4 E bytes of FP32 logits per token forward, 8 E backward. One warp per token
// (a whole block for more than 512 experts) keeps the row in registers; sums over tokens stay in
// registers until a block of tokens is done. Partial sums are written out and added in a fixed
// order, so that results do not depend on scheduling.
#include <cstdint>
#include <mutex>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.hpp"
#include "internal.hpp"

namespace b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = 4096;
constexpr int kMaxSequences = 65536;
constexpr float kMinSum = 1e-25f;      // below this the sigmoids of a row are e^z to FP32 precision

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, float* p) { *p = x; }
__device__ __forceinline__ void from_float(float x, __half* p) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// Sum / maximum over the G threads that share a row; every thread gets the result.
template <int G>
__device__ __forceinline__ float group_sum(float x, float* scratch) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
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

template <int G>
__device__ __forceinline__ float group_max(float x, float* scratch) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
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

template <int G>
__device__ __forceinline__ bool group_any(bool x) {
  if constexpr (G > 32) return __syncthreads_or(x) != 0;
  else return __any_sync(0xffffffffu, x);
}

// Thread `lane` of G holds columns (i * G + lane) * V + j of a row in z[i * V + j]; columns past the
// end hold -infinity, whose score is zero.
template <typename T, int V, int NV, int G>
__device__ __forceinline__ void load_row(const T* row, int experts, int lane, float (&z)[V * NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * G + lane) * V;
    if (col < experts) {
      const Vec<T, V> w = *reinterpret_cast<const Vec<T, V>*>(row + col);
#pragma unroll
      for (int j = 0; j < V; ++j) z[i * V + j] = to_float(w.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) z[i * V + j] = __int_as_float(0xff800000);
    }
  }
}

// z -> p; where kRest, rest = the factor 1 - s of the sigmoid's derivative (1 for softmax).
// The sigmoid is 1 / (1 + e^-z) from __expf and __fdividef: a few ulp, the size of the rounding of
// the logits' own products. Rows whose scores all vanish (every logit below about -57) are
// normalised as e^(z - max), which is what their sigmoids are to FP32 precision; a row of -infinity
// has no scores and gets p = 0.
template <int N, int G, bool kRest>
__device__ __forceinline__ void probabilities(float (&z)[N], float* rest, bool softmax, float* scratch) {
  bool by_max = softmax;
  if (!softmax) {
    float s[N];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kRest) {
        const float e = __expf(-fabsf(z[i]));
        const float r = __fdividef(1.0f, 1.0f + e);
        s[i] = z[i] >= 0.0f ? r : e * r;
        rest[i] = z[i] >= 0.0f ? e * r : r;
      } else {
        s[i] = __fdividef(1.0f, 1.0f + __expf(-z[i]));
      }
      sum += s[i];
    }
    sum = group_sum<G>(sum, scratch);
    by_max = !(sum >= kMinSum);
    if (!by_max) {
      const float inv = __fdividef(1.0f, sum);
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = s[i] * inv;
    }
  }
  if (by_max) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    top = group_max<G>(top, scratch);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      z[i] = z[i] == __int_as_float(0xff800000) ? 0.0f : __expf(z[i] - top);
      sum += z[i];
      if constexpr (kRest) rest[i] = 1.0f;
    }
    sum = group_sum<G>(sum, scratch);
    const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] *= inv;
  }
}

// ------------------------------------------------------------------------------------- forward

struct LossParams {
  const int* ids;
  const int* cu;              // [S + 1] or nullptr: one sequence of all tokens
  int tokens, experts, topk, sequences;
  int chunk, chunks;          // tokens per chunk, number of chunks
  int width;                  // experts rounded up to 4: floats per partial row
  float alpha;
  int softmax;
  float* part_p;              // [chunks + sequences, width]
  int* part_n;                // same
  int2* part_t;               // [chunks + sequences] (sequence, live tokens)
  double* part_loss;          // [sequences, column blocks]
  unsigned* ticket;
  float* loss;
  int* counts;                // [S, E]
  float* slope;               // [S, E]
};

__device__ __forceinline__ int seq_start(const LossParams& p, int s) {
  return p.cu ? min(max(p.cu[s], 0), p.tokens) : (s == 0 ? 0 : p.tokens);
}

// Chunks of tokens cross sequence boundaries, so the work items are the overlaps of a chunk c with a
// sequence s. Walking both lists of ends in merged order visits every overlap, and each step
// advances c or s by one: item i is the pair with c + s = i, found by a binary search for the number
// of sequence ends among the first i merged ends.
__device__ __forceinline__ int item_sequence(const LossParams& p, int i) {
  int lo = max(0, i - p.chunks), hi = min(i, p.sequences);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;                        // is sequence end `mid` among the first i?
    const long long chunk_end = static_cast<long long>(i - mid) * p.chunk;
    if (seq_start(p, mid + 1) < chunk_end) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(kThreads, G == 32 && V * NV <= 8 ? 4 : 2)
balance_partial_kernel(const T* __restrict__ logits, const LossParams p) {
  constexpr int N = V * NV;
  constexpr int kRows = G == 32 ? kWarps : 1;              // tokens a block works on at a time
  extern __shared__ float s_dyn[];                         // kRows x width sums, then width counts
  __shared__ float scratch[kWarps];
  __shared__ int s_live;
  int* s_counts = reinterpret_cast<int*>(s_dyn + kRows * p.width);
  const int item = blockIdx.x;
  const int lane = G == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int group = G == 32 ? threadIdx.x >> 5 : 0;
  if (item == 0 && threadIdx.x == 0) *p.ticket = 0;
  const int s = item_sequence(p, item), c = item - s;
  int lo = 0, hi = 0;
  if (s < p.sequences && c < p.chunks) {
    const long long begin = static_cast<long long>(c) * p.chunk;
    lo = max(static_cast<int>(begin), seq_start(p, s));
    hi = static_cast<int>(min(begin + p.chunk, static_cast<long long>(seq_start(p, s + 1))));
  }
  if (lo >= hi) {
    if (threadIdx.x == 0) p.part_t[item] = make_int2(s, 0);
    return;
  }
  for (int e = threadIdx.x; e < p.width; e += kThreads) s_counts[e] = 0;
  if (threadIdx.x == 0) s_live = 0;
  __syncthreads();
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.0f;
  int live_tokens = 0;
  for (int t = lo + group; t < hi; t += kRows) {
    float z[N];
    load_row<T, V, NV, G>(logits + static_cast<long long>(t) * p.experts, p.experts, lane, z);
    bool mine = false;
    for (int j = lane; j < p.topk; j += G) {
      const int id = p.ids[static_cast<long long>(t) * p.topk + j];
      if (id >= 0 && id < p.experts) {
        mine = true;
        atomicAdd(&s_counts[id], 1);                        // whole numbers: the order does not matter
      }
    }
    if (!group_any<G>(mine)) continue;
    ++live_tokens;
    probabilities<N, G, false>(z, nullptr, p.softmax != 0, scratch);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += z[i];
  }
  if (lane == 0) atomicAdd(&s_live, live_tokens);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (i * G + lane) * V + j;
      if (col < p.width) s_dyn[group * p.width + col] = acc[i * V + j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.width; e += kThreads) {
    float sum = s_dyn[e];
    for (int r = 1; r < kRows; ++r) sum += s_dyn[r * p.width + e];
    p.part_p[static_cast<long long>(item) * p.width + e] = sum;
    p.part_n[static_cast<long long>(item) * p.width + e] = s_counts[e];
  }
  if (threadIdx.x == 0) p.part_t[item] = make_int2(s, s_live);
}

// One block per sequence and 64 columns: adds the sequence's partial rows (in item order within
// sixteen interleaved strands, then the strands), and the last block to finish adds the loss.
__global__ void __launch_bounds__(kThreads)
balance_reduce_kernel(const LossParams p) {
  extern __shared__ unsigned s_filled[];                   // one bit per sequence
  __shared__ float4 s_p[16][16];
  __shared__ int4 s_n[16][16];
  __shared__ int s_tokens, s_count;
  __shared__ double s_loss[kThreads];
  __shared__ bool s_last;
  const int s = blockIdx.x, col_block = blockIdx.y;
  const int items = p.chunks + p.sequences;
  const int words = (p.sequences + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kThreads) s_filled[i] = 0;
  if (threadIdx.x == 0) { s_tokens = 0; s_count = 0; }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int2 t = p.part_t[i];
    if (t.y > 0) {
      atomicOr(&s_filled[t.x >> 5], 1u << (t.x & 31));
      if (t.x == s) atomicAdd(&s_tokens, t.y);
    }
  }
  __syncthreads();
  int filled = 0;
  for (int i = threadIdx.x; i < words; i += kThreads) filled += __popc(s_filled[i]);
  if (filled) atomicAdd(&s_count, filled);
  const int strand = threadIdx.x >> 4, quad = threadIdx.x & 15;
  const int col = col_block * 64 + quad * 4;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  int4 num = make_int4(0, 0, 0, 0);
  const int lo = seq_start(p, s), hi = seq_start(p, s + 1);
  if (hi > lo && col < p.width) {
    const int first = lo / p.chunk + s, last = (hi - 1) / p.chunk + s;
    for (int i = first + strand; i <= last; i += 16) {
      if (p.part_t[i].y == 0) continue;
      const float4 a = *reinterpret_cast<const float4*>(p.part_p + static_cast<long long>(i) * p.width + col);
      const int4 n = *reinterpret_cast<const int4*>(p.part_n + static_cast<long long>(i) * p.width + col);
      sum.x += a.x; sum.y += a.y; sum.z += a.z; sum.w += a.w;
      num.x += n.x; num.y += n.y; num.z += n.z; num.w += n.w;
    }
  }
  s_p[strand][quad] = sum;
  s_n[strand][quad] = num;
  __syncthreads();
  double term = 0.0;
  if (threadIdx.x < 64) {
    const int e = col_block * 64 + threadIdx.x;
    const float* ps = reinterpret_cast<const float*>(&s_p[0][0]) + threadIdx.x;
    const int* ns = reinterpret_cast<const int*>(&s_n[0][0]) + threadIdx.x;
    double total = 0.0;
    int n = 0;
    for (int r = 0; r < 16; ++r) {
      total += static_cast<double>(ps[r * 64]);
      n += ns[r * 64];
    }
    if (e < p.experts) {
      const double t = s_tokens > 0 ? static_cast<double>(s_tokens) : 1.0;
      const double slope = static_cast<double>(p.alpha) * p.experts * n / (static_cast<double>(p.topk) * t * t * max(s_count, 1));
      p.counts[static_cast<long long>(s) * p.experts + e] = n;
      p.slope[static_cast<long long>(s) * p.experts + e] = static_cast<float>(slope);
      term = slope * total;
    }
  }
  s_loss[threadIdx.x] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum64 = 0.0;
    for (int i = 0; i < 64; ++i) sum64 += s_loss[i];
    p.part_loss[static_cast<long long>(s) * gridDim.y + col_block] = sum64;
    __threadfence();
    s_last = atomicAdd(p.ticket, 1u) == gridDim.x * gridDim.y - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const long long terms = static_cast<long long>(p.sequences) * gridDim.y;
  double mine = 0.0;
  for (long long i = threadIdx.x; i < terms; i += kThreads) mine += __ldcg(p.part_loss + i);
  s_loss[threadIdx.x] = mine;
  for (int d = kThreads / 2; d > 0; d >>= 1) {
    __syncthreads();
    if (threadIdx.x < d) s_loss[threadIdx.x] += s_loss[threadIdx.x + d];
  }
  if (threadIdx.x == 0) *p.loss = static_cast<float>(s_loss[0]);
}

// ------------------------------------------------------------------------------------ backward

struct GradParams {
  const int* ids;
  const float* weights;       // [T, k] or nullptr with grad_weights
  const float* grad_weights;  // [T, k] or nullptr: no gradient through the weights
  const float* slope;         // [S, E] or nullptr: no gradient through the loss
  const float* grad_loss;     // scalar on the device
  const int* cu;
  int tokens, experts, topk, sequences;
  int width;
  int chunk;                  // consecutive tokens per group of threads
  int softmax;
};

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(kThreads, G == 32 && V * NV <= 8 ? 4 : 2)
router_grad_kernel(T* __restrict__ grad, const T* __restrict__ logits, const GradParams p) {
  constexpr int N = V * NV;
  extern __shared__ float s_dyn[];                         // per group: the weights' part of one row
  __shared__ float scratch[kWarps];
  const int lane = G == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int group = G == 32 ? threadIdx.x >> 5 : 0;
  float* add = s_dyn + group * p.width;
  for (int e = lane; e < p.width; e += G) add[e] = 0.0f;
  auto sync = [] { if constexpr (G > 32) __syncthreads(); else __syncwarp(); };
  sync();
  const long long first = (static_cast<long long>(blockIdx.x) * (G == 32 ? kWarps : 1) + group) * p.chunk;
  const int begin = static_cast<int>(min(first, static_cast<long long>(p.tokens)));
  const int end = static_cast<int>(min(first + p.chunk, static_cast<long long>(p.tokens)));
  if (begin >= end) return;                                // uniform over the group
  const float g = p.slope ? *p.grad_loss : 0.0f;
  // sequence of the first token: the number of sequence ends at or before it
  int s = 0;
  if (p.cu && p.slope) {
    int hi = p.sequences;
    while (s < hi) {
      const int mid = (s + hi) >> 1;
      if (p.cu[mid + 1] <= begin) s = mid + 1; else hi = mid;
    }
  }
  for (int t = begin; t < end; ++t) {
    const T* row = logits + static_cast<long long>(t) * p.experts;
    const long long slot0 = static_cast<long long>(t) * p.topk;
    float z[N], rest[N];
    load_row<T, V, NV, G>(row, p.experts, lane, z);
    bool inside = p.slope != nullptr;
    if (inside && p.cu) {
      while (s < p.sequences && p.cu[s + 1] <= t) ++s;
      inside = s < p.sequences && p.cu[s] <= t;
    }
    bool mine = false;
    float mean = 0.0f;
    for (int j = lane; j < p.topk; j += G) {
      const int id = p.ids[slot0 + j];
      if (id >= 0 && id < p.experts) {
        mine = true;
        if (p.grad_weights) mean += p.weights[slot0 + j] * p.grad_weights[slot0 + j];
      }
    }
    inside = group_any<G>(mine) && inside;
    if (inside) {
      probabilities<N, G, true>(z, rest, p.softmax != 0, scratch);
      const float* slope = p.slope + static_cast<long long>(p.cu ? s : 0) * p.experts;
      float d[N];
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * G + lane) * V;
        if (col < p.experts) {
          const Vec<float, V> w = *reinterpret_cast<const Vec<float, V>*>(slope + col);
#pragma unroll
          for (int j = 0; j < V; ++j) d[i * V + j] = w.v[j];
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) d[i * V + j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) dot = fmaf(d[i * V + j], z[i * V + j], dot);
      }
      dot = group_sum<G>(dot, scratch);
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = g * z[i] * rest[i] * (d[i] - dot);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = 0.0f;
    }
    if (p.grad_weights) {
      mean = group_sum<G>(mean, scratch);
      // slots of one token that name the same expert add up in slot order
      for (int j0 = 0; j0 < p.topk; j0 += 32) {
        const int j = j0 + lane;
        int id = -1;
        float v = 0.0f;
        if (lane < 32 && j < p.topk) {
          id = p.ids[slot0 + j];
          if (id >= 0 && id < p.experts) {
            const float x = to_float(row[id]);
            const float e = __expf(-fabsf(x));
            const float r = __fdividef(1.0f, 1.0f + e);
            v = p.weights[slot0 + j] * (x >= 0.0f ? e * r : r) * (p.grad_weights[slot0 + j] - mean);
          } else {
            id = -1;
          }
        }
        if (G == 32 || threadIdx.x < 32) {
          const unsigned same = __match_any_sync(0xffffffffu, id);
          const bool alone = id < 0 || (same & (same - 1)) == 0;
          if (__all_sync(0xffffffffu, alone)) {
            if (id >= 0) add[id] += v;
          } else {
            for (int r = 0; r < 32; ++r) {
              if (lane == r && id >= 0) add[id] += v;
              __syncwarp();
            }
          }
          __syncwarp();
        }
      }
      sync();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * G + lane) * V;
        if (col < p.experts) {
#pragma unroll
          for (int j = 0; j < V; ++j) z[i * V + j] += add[col + j];
        }
      }
      sync();
      for (int j = lane; j < p.topk; j += G) {
        const int id = p.ids[slot0 + j];
        if (id >= 0 && id < p.experts) add[id] = 0.0f;
      }
      sync();
    }
    T* out = grad + static_cast<long long>(t) * p.experts;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * G + lane) * V;
      if (col < p.experts) {
        Vec<T, V> w;
#pragma unroll
        for (int j = 0; j < V; ++j) from_float(z[i * V + j], &w.v[j]);
        *reinterpret_cast<Vec<T, V>*>(out + col) = w;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------- host

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int loss_chunk(int tokens, int sms) {
  // about three blocks per SM, at least two rounds of eight tokens each
  const long long target = (static_cast<long long>(tokens) + sms * 3 - 1) / (sms * 3);
  long long chunk = (target + 7) / 8 * 8;
  return static_cast<int>(chunk < 16 ? 16 : chunk);
}

struct LossLayout {
  int chunk, chunks, width, col_blocks;
  size_t p, n, t, loss, ticket, total;
};

LossLayout loss_layout(int tokens, int experts, int sequences) {
  LossLayout l;
  l.chunk = loss_chunk(tokens, 148);      // fixed: the sums' order must not depend on the device
  l.chunks = (tokens + l.chunk - 1) / l.chunk;
  l.width = (experts + 3) / 4 * 4;
  l.col_blocks = (experts + 63) / 64;
  const size_t rows = static_cast<size_t>(l.chunks) + sequences;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.p = 0;
  l.n = up(l.p + rows * l.width * 4);
  l.t = up(l.n + rows * l.width * 4);
  l.loss = up(l.t + rows * 8);
  l.ticket = up(l.loss + static_cast<size_t>(sequences) * l.col_blocks * 8);
  l.total = up(l.ticket + 4);
  return l;
}

// Columns a group of threads covers: four at a time where the rows allow it.
template <typename T, template <typename, int, int, int> class Launch, typename... Args>
int dispatch_width(int experts, bool vec4, Args... args) {
  if (vec4) {
    if (experts <= 128) return Launch<T, 4, 1, 32>::run(args...);
    if (experts <= 256) return Launch<T, 4, 2, 32>::run(args...);
    if (experts <= 512) return Launch<T, 4, 4, 32>::run(args...);
    return Launch<T, 4, 4, 256>::run(args...);
  }
  if (experts <= 128) return Launch<T, 1, 4, 32>::run(args...);
  if (experts <= 256) return Launch<T, 1, 8, 32>::run(args...);
  if (experts <= 512) return Launch<T, 1, 16, 32>::run(args...);
  return Launch<T, 1, 16, 256>::run(args...);
}

template <typename T, int V, int NV, int G>
struct LossLaunch {
  static int run(const void* logits, const LossParams& p, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>((G == 32 ? kWarps : 1) + 1) * p.width * 4;
    balance_partial_kernel<T, V, NV, G><<<p.chunks + p.sequences, kThreads, smem, stream>>>(static_cast<const T*>(logits), p);
    count_launch();
    return launch_status();
  }
};

template <typename T, int V, int NV, int G>
struct GradLaunch {
  static int run(void* grad, const void* logits, GradParams p, int sms, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(G == 32 ? kWarps : 1) * p.width * 4;
    const long long groups = static_cast<long long>(sms) * (G == 32 ? 4 * kWarps : 4);
    p.chunk = static_cast<int>((p.tokens + groups - 1) / groups);
    const long long needed = (static_cast<long long>(p.tokens) + p.chunk - 1) / p.chunk;
    const int blocks = static_cast<int>(G == 32 ? (needed + kWarps - 1) / kWarps : needed);
    router_grad_kernel<T, V, NV, G><<<blocks, kThreads, smem, stream>>>(static_cast<T*>(grad), static_cast<const T*>(logits), p);
    count_launch();
    return launch_status();
  }
};

bool valid_router(int tokens, int experts, int topk, int sequences, int dtype) {
  return tokens >= 0 && experts > 0 && experts <= kMaxExperts && topk > 0 && topk <= experts && sequences > 0 &&
         sequences <= kMaxSequences && dtype >= 0 && dtype <= 2;
}

size_t element_size(int dtype) { return dtype == 2 ? 4 : 2; }

}  // namespace
}  // namespace b200

extern "C" {

size_t b200_nvfp4_moe_balance_loss_workspace_bytes(int num_tokens, int num_experts, int num_sequences) {
  using namespace b200;
  if (!valid_router(num_tokens, num_experts, 1, num_sequences, 0)) return 0;
  return loss_layout(num_tokens, num_experts, num_sequences).total;
}

int b200_nvfp4_moe_balance_loss(void* loss, void* counts, void* slope, const void* logits, const void* topk_ids,
                                const void* cu_seqlens, int num_tokens, int num_experts, int num_topk, int num_sequences,
                                int logits_dtype, int scoring, float alpha, void* workspace, size_t workspace_bytes,
                                b200_stream_t stream) {
  using namespace b200;
  if (!valid_router(num_tokens, num_experts, num_topk, num_sequences, logits_dtype) || loss == nullptr || counts == nullptr ||
      slope == nullptr || (num_tokens > 0 && (logits == nullptr || topk_ids == nullptr)) || scoring < 0 || scoring > 1 ||
      (cu_seqlens == nullptr && num_sequences != 1) || !aligned(logits, element_size(logits_dtype)) || !aligned(workspace, 256))
    return B200_NVFP4_INVALID_ARGUMENT;
  const LossLayout l = loss_layout(num_tokens, num_experts, num_sequences);
  if (workspace == nullptr || workspace_bytes < l.total) return B200_NVFP4_INSUFFICIENT_WORKSPACE;
  const DeviceInfo& dev = current_device_info();
  if (!dev.ok) return B200_NVFP4_CUDA_ERROR;
  if (!device_supported(dev)) return B200_NVFP4_UNSUPPORTED_DEVICE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  LossParams p = {};
  p.ids = static_cast<const int*>(topk_ids);
  p.cu = static_cast<const int*>(cu_seqlens);
  p.tokens = num_tokens;
  p.experts = num_experts;
  p.topk = num_topk;
  p.sequences = num_sequences;
  p.chunk = l.chunk;
  p.chunks = l.chunks;
  p.width = l.width;
  p.alpha = alpha;
  p.softmax = scoring;
  p.part_p = reinterpret_cast<float*>(ws + l.p);
  p.part_n = reinterpret_cast<int*>(ws + l.n);
  p.part_t = reinterpret_cast<int2*>(ws + l.t);
  p.part_loss = reinterpret_cast<double*>(ws + l.loss);
  p.ticket = reinterpret_cast<unsigned*>(ws + l.ticket);
  p.loss = static_cast<float*>(loss);
  p.counts = static_cast<int*>(counts);
  p.slope = static_cast<float*>(slope);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vec4 = num_experts % 4 == 0 && aligned(logits, 4 * element_size(logits_dtype));
  int status;
  switch (logits_dtype) {
    case 0: status = dispatch_width<__half, LossLaunch>(num_experts, vec4, logits, p, s); break;
    case 1: status = dispatch_width<__nv_bfloat16, LossLaunch>(num_experts, vec4, logits, p, s); break;
    default: status = dispatch_width<float, LossLaunch>(num_experts, vec4, logits, p, s); break;
  }
  if (status != B200_NVFP4_SUCCESS) return status;
  balance_reduce_kernel<<<dim3(num_sequences, l.col_blocks), kThreads, static_cast<size_t>((num_sequences + 31) / 32) * 4, s>>>(p);
  count_launch();
  return launch_status();
}

int b200_nvfp4_moe_router_backward(void* grad_logits, const void* logits, const void* topk_ids, const void* topk_weights,
                                   const void* grad_weights, const void* slope, const void* grad_loss, const void* cu_seqlens,
                                   int num_tokens, int num_experts, int num_topk, int num_sequences, int logits_dtype,
                                   int scoring, b200_stream_t stream) {
  using namespace b200;
  if (!valid_router(num_tokens, num_experts, num_topk, num_sequences, logits_dtype) || scoring < 0 || scoring > 1 ||
      (num_tokens > 0 && (grad_logits == nullptr || logits == nullptr || topk_ids == nullptr)) ||
      (grad_weights == nullptr && slope == nullptr) || (grad_weights != nullptr && topk_weights == nullptr) ||
      (slope != nullptr && grad_loss == nullptr) || (cu_seqlens == nullptr && num_sequences != 1) ||
      !aligned(logits, element_size(logits_dtype)) || !aligned(grad_logits, element_size(logits_dtype)))
    return B200_NVFP4_INVALID_ARGUMENT;
  const DeviceInfo& dev = current_device_info();
  if (!dev.ok) return B200_NVFP4_CUDA_ERROR;
  if (!device_supported(dev)) return B200_NVFP4_UNSUPPORTED_DEVICE;
  if (num_tokens == 0) return B200_NVFP4_SUCCESS;
  GradParams p = {};
  p.ids = static_cast<const int*>(topk_ids);
  p.weights = static_cast<const float*>(topk_weights);
  p.grad_weights = static_cast<const float*>(grad_weights);
  p.slope = static_cast<const float*>(slope);
  p.grad_loss = static_cast<const float*>(grad_loss);
  p.cu = static_cast<const int*>(cu_seqlens);
  p.tokens = num_tokens;
  p.experts = num_experts;
  p.topk = num_topk;
  p.sequences = num_sequences;
  p.width = (num_experts + 3) / 4 * 4;
  p.softmax = scoring;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t vec = 4 * element_size(logits_dtype);
  const bool vec4 = num_experts % 4 == 0 && aligned(logits, vec) && aligned(grad_logits, vec) && aligned(slope, 16);
  switch (logits_dtype) {
    case 0: return dispatch_width<__half, GradLaunch>(num_experts, vec4, grad_logits, logits, p, dev.sm_count, s);
    case 1: return dispatch_width<__nv_bfloat16, GradLaunch>(num_experts, vec4, grad_logits, logits, p, dev.sm_count, s);
    default: return dispatch_width<float, GradLaunch>(num_experts, vec4, grad_logits, logits, p, dev.sm_count, s);
  }
}

}  // extern "C"
