// Gradient of the router's logits, through the balance loss and through the renormalised weights, in one
// pass. With the score s = sigmoid(z), the probabilities p and the slope of the balance loss (see the
// forward pass; the counts are constants):
//   loss      dz_e  = g p_e (1 - s_e) (slope_e - sum_j slope_j p_j)       (softmax: without 1 - s)
//   weights   dz_j += w_j (1 - s_j) (g_j - sum_i g_i w_i)                 for each selected expert j,
// the second from w_j = s_j / (sum of the selected s). The threads that hold a token's slots work out what
// the weights add and lay it at the selected columns of a row in shared memory, zero elsewhere; the
// threads that hold the columns add it.
//
// Reads the logits, ids, weights and their gradient once and writes the gradient: 8 E + 12 k bytes per
// token of FP32 logits. 131072 x 160 BF16: 30.4 us where the bytes take 14.2 (through the loss alone 23.3, the weights alone
// 19.0; softmax 28.5); 65536 x 256 FP32: 27.7 us (21). 31 instructions per logit at 61 to 64 % of the issue slots, with 16 warps per SM: three blocks per SM
// instead of two spill (72 us).
#include "router_common.cuh"

namespace b200 {
namespace router {
namespace {

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
__global__ void __launch_bounds__(kThreads, 2)
router_grad_kernel(T* grad, const T* logits, const GradParams p) {
  using Gr = Group<G>;
  constexpr int N = V * NV;
  extern __shared__ __align__(16) uint8_t s_raw[];         // queues; per group the weights' part of a row, and owners
  __shared__ float scratch[kWarps];
  const int lane = Gr::lane();
  using Rows = RowQueue<T, V, NV, G>;
  Rows rows(s_raw, logits, p.tokens, p.experts);
  rows.fill_rest(p.experts, lane);
  WordQueue<int> first_ids(s_raw + Rows::kBytes);
  WordQueue<float> first_w(s_raw + Rows::kBytes + WordQueue<int>::kBytes);
  WordQueue<float> first_g(s_raw + Rows::kBytes + 2 * WordQueue<int>::kBytes);
  float* add = reinterpret_cast<float*>(s_raw + Rows::kBytes + 3 * WordQueue<int>::kBytes) + Gr::index() * 2 * p.width;
  int* owner = reinterpret_cast<int*>(add + p.width);
  for (int e = lane; e < p.width; e += G) add[e] = 0.0f;
  Gr::sync();
  ptx::grid_wait();
  ptx::grid_launch_dependents();
  // a warp (a block for G > 32) takes `chunk` consecutive tokens, its groups neighbouring ones
  const long long worker = G > 32 ? blockIdx.x : static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int begin = static_cast<int>(min(worker * p.chunk, static_cast<long long>(p.tokens)));
  const int end = static_cast<int>(min(worker * p.chunk + p.chunk, static_cast<long long>(p.tokens)));
  if (begin >= end) return;                                // uniform over the worker
  const bool through_weights = p.grad_weights != nullptr, through_loss = p.slope != nullptr;
  const float g = through_loss ? *p.grad_loss : 0.0f;
  int t = begin + Gr::in_warp();
  // sequence of the first token: the number of sequence ends at or before it
  int s = 0, s_begin = 0, s_end = p.tokens;
  auto search = [&](int hi) {
    while (s < hi) {
      const int mid = (s + hi) >> 1;
      if (p.cu[mid + 1] <= t) s = mid + 1; else hi = mid;
    }
  };
  if (p.cu && through_loss) {
    search(p.sequences);
    s_begin = s < p.sequences ? p.cu[s] : p.tokens;
    s_end = s < p.sequences ? p.cu[s + 1] : 0x7fffffff;
  }
  float d[N];
  auto load_slope = [&] {
    const float* slope = p.slope + static_cast<long long>(s) * p.experts;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * G + lane) * V;
      Vec<float, V> x;
#pragma unroll
      for (int j = 0; j < V; ++j) x.v[j] = 0.0f;
      if (through_loss && s < p.sequences && col < p.experts) x = *reinterpret_cast<const Vec<float, V>*>(slope + col);
#pragma unroll
      for (int j = 0; j < V; ++j) d[i * V + j] = x.v[j];
    }
  };
  load_slope();
  const long long row_step = static_cast<long long>(Gr::kPerWarp) * p.experts;
  const int slot_step = Gr::kPerWarp * p.topk;
  long long slots = static_cast<long long>(t) * p.topk, slots_ahead = slots;
  T* out = grad + static_cast<long long>(t) * p.experts;
  const T* row = logits + static_cast<long long>(t) * p.experts;
  const T* row_ahead = row;
  int ahead = t;                                           // the next token to be fetched
  auto fetch = [&](int stage) {
    if (ahead < end) {
      rows.push(stage, row_ahead, p.experts, lane);
      if (lane < p.topk) {
        first_ids.push(stage, p.ids + slots_ahead + lane);
        if (through_weights) {
          first_w.push(stage, p.weights + slots_ahead + lane);
          first_g.push(stage, p.grad_weights + slots_ahead + lane);
        }
      }
    }
    queue_commit();
    ahead += Gr::kPerWarp;
    row_ahead += row_step;
    slots_ahead += slot_step;
  };
  for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  // the slots of a token sit in the first threads of a group: their sum takes as many exchanges as they span
  int span = 1;
  while (span < p.topk && span < G) span *= 2;
  const int steps = (end - begin + Gr::kPerWarp - 1) / Gr::kPerWarp;
  for (int step = 0; step < steps; ++step) {
    const int stage = step & (kDepth - 1);
    fetch((step + kDepth - 1) & (kDepth - 1));
    queue_wait();
    const bool in = t < end;
    float z[N];
    rows.pop(stage, row, z, p.experts, lane);
    int id = -1;
    float w = 0.0f, gw = 0.0f;
    if (in && lane < p.topk) {
      id = first_ids.pop(stage);
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.experts)) id = -1;
      if (through_weights) {
        w = first_w.pop(stage);
        gw = first_g.pop(stage);
      }
    }
    if (t >= s_end && in) {                                // on to the sequence of this token
      // mostly the next one; behind padding of empty sequences, far on
      for (int i = 0; i < 4 && s < p.sequences && p.cu[s + 1] <= t; ++i) ++s;
      if (s < p.sequences && p.cu[s + 1] <= t) search(p.sequences);
      s_begin = s < p.sequences ? p.cu[s] : p.tokens;
      s_end = s < p.sequences ? p.cu[s + 1] : 0x7fffffff;
      load_slope();
    }
    bool mine = id >= 0;
    float mean = mine ? w * gw : 0.0f;
    if (in) {
      for (int j = lane + G; j < p.topk; j += G) {
        const int other = p.ids[slots + j];
        if (static_cast<unsigned>(other) < static_cast<unsigned>(p.experts)) {
          mine = true;
          if (through_weights) mean += p.weights[slots + j] * p.grad_weights[slots + j];
        }
      }
    }
    const bool inside = Gr::any(mine) && in && through_loss && t >= s_begin && t < s_end;
    t += Gr::kPerWarp;

    float out_row[N];                                      // s (1 - s), then the gradient
    if (through_loss) {
      float sum = 0.0f, dot = 0.0f;
      if (!p.softmax) {
        // with w = e^-|z|: the larger of s and 1 - s is r = 1 / (1 + w), the smaller w r
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float w = exponential(-fabsf(z[i]));
          const float r = reciprocal(1.0f + w);
          const float wr = w * r;
          out_row[i] = wr * r;
          const float sc = z[i] < 0.0f ? wr : r;
          sum += sc;
          dot = fmaf(d[i], sc, dot);
        }
        sum = Gr::sum(sum, scratch);
        dot = Gr::sum(dot, scratch);
      }
      const bool by_max = inside && (p.softmax || !(sum >= kMinSum));
      float inv = reciprocal(sum);
      if (Gr::any_here(by_max)) {      // softmax, or scores that all vanish: they are e^z then, and 1 - s is 1
        const float other = exponentials<N, G>(z, scratch);
        float dot2 = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) dot2 = fmaf(d[i], z[i], dot2);
        dot2 = Gr::sum(dot2, scratch);
        inv = by_max ? other : inv;
        dot = by_max ? dot2 : dot;
#pragma unroll
        for (int i = 0; i < N; ++i) out_row[i] = by_max ? z[i] : out_row[i];
      }
      // g p (1 - s) (slope - dot) with the row's constants multiplied out
      const float by = g * inv, minus = -by * (dot * inv);
#pragma unroll
      for (int i = 0; i < N; ++i) out_row[i] *= fmaf(by, d[i], minus);
      if (Gr::any_here(!inside)) {
#pragma unroll
        for (int i = 0; i < N; ++i) out_row[i] = inside ? out_row[i] : 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out_row[i] = 0.0f;
    }
    if (through_weights) {
      if constexpr (G > 32) {
        mean = Gr::sum(mean, scratch);
      } else {
        for (int x = span >> 1; x > 0; x >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, x);
      }
      // Slots of one token that name the same expert add up in slot order. Every thread with a slot
      // signs its column; one that finds another's signature shares the column.
      auto place = [&](int to, float v, int slots_here) {
        if (to >= 0) owner[to] = lane;
        Gr::sync();
        const bool shared = to >= 0 && owner[to] != lane;
        if (!Gr::any_here(shared)) {
          if (to >= 0) add[to] += v;
        } else {
          for (int r = 0; r < slots_here; ++r) {
            if (lane == r && to >= 0) add[to] += v;
            Gr::sync();
          }
        }
        Gr::sync();
      };
      // 1 - s of a selected column
      auto rest = [&](int col) { return reciprocal(1.0f + exponential(rows.at(stage, row, col, lane))); };
      Gr::sync();
      place(id, id >= 0 ? w * (gw - mean) * rest(id) : 0.0f, min(G, p.topk));
      for (int j0 = G; j0 < p.topk; j0 += G) {
        int to = in && j0 + lane < p.topk ? p.ids[slots + j0 + lane] : -1;
        if (static_cast<unsigned>(to) >= static_cast<unsigned>(p.experts)) to = -1;
        place(to, to >= 0 ? p.weights[slots + j0 + lane] * (p.grad_weights[slots + j0 + lane] - mean) * rest(to) : 0.0f, min(G, p.topk - j0));
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * G + lane) * V;
        if (col < p.experts) {
          const Vec<float, V> x = *reinterpret_cast<const Vec<float, V>*>(add + col);
#pragma unroll
          for (int j = 0; j < V; ++j) out_row[i * V + j] += x.v[j];
        }
      }
      Gr::sync();
      if (id >= 0) add[id] = 0.0f;
      if (in) {
        for (int j = lane + G; j < p.topk; j += G) {
          const int other = p.ids[slots + j];
          if (static_cast<unsigned>(other) < static_cast<unsigned>(p.experts)) add[other] = 0.0f;
        }
      }
      Gr::sync();
    }
    if (in) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * G + lane) * V;
        if (col < p.experts) {
          Vec<T, V> x;
#pragma unroll
          for (int j = 0; j < V; ++j) from_float(out_row[i * V + j], &x.v[j]);
          *reinterpret_cast<Vec<T, V>*>(out + col) = x;
        }
      }
    }
    row += row_step;
    out += row_step;
    slots += slot_step;
  }
}

template <typename T, int V, int NV, int G>
struct GradLaunch {
  static int run(void* grad, const void* logits, GradParams p, int sms, int device, cudaStream_t stream) {
    using Gr = Group<G>;
    static std::once_flag once[64];
    static cudaError_t status[64];
    auto kernel = router_grad_kernel<T, V, NV, G>;
    constexpr int kMaxWidth = G > 32 ? kMaxExperts : V * NV * G;
    constexpr size_t kQueues = RowQueue<T, V, NV, G>::kBytes + 3 * WordQueue<int>::kBytes;
    static_assert(kQueues % 16 == 0 && kQueues + Gr::kPerBlock * 2 * kMaxWidth * 4 <= 112 * 1024, "two blocks per SM");
    const int allowed = allow_smem(kernel, once, status, device, static_cast<int>(kQueues + Gr::kPerBlock * 2 * kMaxWidth * 4));
    if (allowed != B200_NVFP4_SUCCESS) return allowed;
    const size_t smem = kQueues + static_cast<size_t>(Gr::kPerBlock) * 2 * p.width * 4;
    // two resident blocks per SM; a worker's tokens are a multiple of what it takes at a time
    const long long workers = static_cast<long long>(sms) * 2 * (G > 32 ? 1 : kWarps);
    const long long chunk = (p.tokens + workers - 1) / workers;
    p.chunk = static_cast<int>((chunk + Gr::kPerWarp - 1) / Gr::kPerWarp * Gr::kPerWarp);
    const long long needed = (static_cast<long long>(p.tokens) + p.chunk - 1) / p.chunk;
    const int blocks = static_cast<int>(G > 32 ? needed : (needed + kWarps - 1) / kWarps);
    return launch_overlapped(kernel, blocks, kThreads, smem, 1, stream, static_cast<T*>(grad), static_cast<const T*>(logits), p);
  }
};

}  // namespace
}  // namespace router
}  // namespace b200

extern "C" {

int b200_nvfp4_moe_router_backward(void* grad_logits, const void* logits, const void* topk_ids, const void* topk_weights,
                                   const void* grad_weights, const void* slope, const void* grad_loss, const void* cu_seqlens,
                                   int num_tokens, int num_experts, int num_topk, int num_sequences, int logits_dtype,
                                   int scoring, b200_stream_t stream) {
  using namespace b200;
  using namespace b200::router;
  if (!valid_router(num_tokens, num_experts, num_topk, num_sequences, logits_dtype) || scoring < 0 || scoring > 1 ||
      (num_tokens > 0 && (grad_logits == nullptr || logits == nullptr || topk_ids == nullptr)) ||
      (grad_weights == nullptr && slope == nullptr) || (grad_weights != nullptr && topk_weights == nullptr) ||
      (slope != nullptr && grad_loss == nullptr) || (cu_seqlens == nullptr && num_sequences != 1) ||
      !aligned(logits, element_size(logits_dtype)) || !aligned(grad_logits, element_size(logits_dtype)) ||
      !aligned(topk_ids, 4) || !aligned(topk_weights, 4) || !aligned(grad_weights, 4) || !aligned(slope, 4) ||
      !aligned(grad_loss, 4) || !aligned(cu_seqlens, 4))
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
  const size_t size = element_size(logits_dtype);
  const bool quads = num_experts % 4 == 0 && aligned(logits, 4 * size) && aligned(grad_logits, 4 * size) && aligned(slope, 16);
  switch (logits_dtype) {
    case 0: return dispatch_width<__half, GradLaunch>(num_experts, quads, grad_logits, logits, p, dev.sm_count, dev.device, s);
    case 1: return dispatch_width<__nv_bfloat16, GradLaunch>(num_experts, quads, grad_logits, logits, p, dev.sm_count, dev.device, s);
    default: return dispatch_width<float, GradLaunch>(num_experts, quads, grad_logits, logits, p, dev.sm_count, dev.device, s);
  }
}

}  // extern "C"
