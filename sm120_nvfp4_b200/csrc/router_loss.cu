// Balance loss of the router with per-expert counts.
//
// Token t with logits z: s_e = sigmoid(z_e), p_e = s_e / sum_j s_j (scoring 0), or p = softmax(z)
// (scoring 1). A token counts ("live") when it lies in a sequence and has an id in [0, E). Per sequence
// with T live tokens, of which n_e slots chose expert e:
//   slope_e = alpha * E * n_e / (k * T^2 * S')       (S' = sequences with a live token)
//   loss    = sum over sequences and experts of slope_e * sum_t p_te
// which is the mean over sequences of alpha * sum_e f_e P_e, f_e = n_e E / (k T), P_e = mean_t p_te.
//
// Reads 4 E bytes of FP32 logits and 4 k of ids per token and writes almost nothing. One pass: a group of
// threads keeps a token's row in registers and the sums over its tokens too; partial sums of a block
// of tokens are written out and added by a second kernel in a fixed order, so that results do not depend
// on scheduling. Counts are whole numbers and may be added in any order.
//
// Probabilities are added in FP32 for kRun tokens at most, then in FP64: equal ones (an indifferent router's) are
// rounded the same way again and again, and one FP32 sum over n of them is off by up to n 2^-25 (2^22 tokens x 520: 1.7e-4,
// 2^26 x 7: 8e-5; now below 3e-7 both). A run is off by 2^-20 at most, whatever the number of tokens. It costs nothing at
// 65536 x 256, 0.5 us at 4096 x 256 (8.5) and 3 % beyond 512 experts.
//
// 65536 x 256 FP32: 24.6 us where the bytes take 10.6 (softmax 23.7); 131072 x 160 BF16: 26.0 us (23.5). In the first kernel no unit is
// full: the special-function unit is busy for 7.4 us (an exponential and a reciprocal per logit, sixteen a
// cycle per SM), 45 % of the issue slots are used; with 16 warps per SM the rest is the latency of dependent
// instructions, and that of the start and the end of blocks with 14 rounds of tokens each. The second
// kernel is a chain of latencies, 7 us on its own, of which its early start hides a part.
#include "router_common.cuh"

namespace b200 {
namespace router {
namespace {

struct LossParams {
  const int* ids;
  const int* cu;              // [S + 1] or nullptr: one sequence of all tokens
  int tokens, experts, topk, sequences;
  int chunk, chunks;          // tokens per chunk, number of chunks
  int width;                  // experts rounded up to 4: values per partial row
  int counts_at;              // place of the counts in shared memory
  float alpha;
  int softmax;
  double* part_p;             // [chunks + sequences, width]
  int* part_n;                // same
  int2* part_t;               // [chunks + sequences] (sequence, live tokens)
  double* part_loss;          // [sequences, column blocks]
  unsigned* ticket;           // blocks of the last kernel that are done; beside it the sequences with a live token, where
  int* live;                  // [sequences] the live tokens are counted first (nullptr: every block counts for itself)
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
  const int lane = threadIdx.x & 31;
  while (lo < hi) {                                        // a warp probes 32 places at a time
    const int stride = (hi - lo + 31) / 32;
    const int mid = lo + lane * stride;
    bool before = false;                                   // is sequence end `mid` among the first i?
    if (mid < hi) before = seq_start(p, mid + 1) < static_cast<long long>(i - mid) * p.chunk;
    const int count = __popc(__ballot_sync(0xffffffffu, before));
    if (count == 0) return lo;
    const int next_hi = min(hi, lo + count * stride);
    lo += (count - 1) * stride + 1;
    hi = next_hi;
  }
  return lo;
}

// value(0) + ... + value(N - 1), as four sums side by side: additions in FP64 that wait for each other take long.
template <int N, typename Value>
__device__ __forceinline__ double sum_rows(Value value) {
  static_assert(N % 4 == 0, "four sums");
  double s[4] = {value(0), value(1), value(2), value(3)};
#pragma unroll
  for (int r = 4; r < N; ++r) s[r & 3] += value(r);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Additions in FP32 before a sum goes into its FP64 one. (Twice as many where these are added to by atomic operations,
// which are slow: 8192 x 4096 57 -> 53 us, 1048576 x 600 4767 -> 4699.)
template <int G>
constexpr int kRun = G > 32 ? 32 : 16;

// Partial sums of one work item, written out. `s_raw`: queues, a row of sums per group, counts. (The one group of a
// wide row adds up in its partial row itself: 32 KB of sums per block would leave room for one block per SM only.)
template <typename T, int V, int NV, int G>
__device__ __forceinline__ void add_item(const T* logits, const LossParams& p, uint8_t* s_raw, int item) {
  using Gr = Group<G>;
  constexpr int N = V * NV;
  __shared__ float scratch[kWarps];
  __shared__ int s_live;
  const int lane = Gr::lane();
  using Rows = RowQueue<T, V, NV, G>;
  Rows rows(s_raw, logits, p.tokens, p.experts);
  rows.fill_rest(p.experts, lane);
  WordQueue<int> first_ids(s_raw + Rows::kBytes);
  double* s_sums = reinterpret_cast<double*>(s_raw + Rows::kBytes + WordQueue<int>::kBytes);
  int* s_counts = reinterpret_cast<int*>(s_raw + p.counts_at);
  ptx::grid_wait();
  ptx::grid_launch_dependents();                           // the second kernel's blocks may take their places
  if (item == 0 && threadIdx.x == 0) p.ticket[0] = p.ticket[1] = 0;
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
  double* part = p.part_p + static_cast<long long>(item) * p.width;
  double* sums = G > 32 ? part : s_sums + Gr::index() * p.width;
  bool begun = false;
  auto flush = [&] {                                       // every thread its own columns: nobody to wait for
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int col = (i * G + lane) * V + j;
        const double run = static_cast<double>(acc[i * V + j]);
        if (col < p.width) {
          if (!begun) sums[col] = run;
          else if constexpr (G > 32) atomicAdd(&sums[col], run);       // (in global memory, and nothing to wait for)
          else sums[col] += run;
        }
        acc[i * V + j] = 0.0f;
      }
    }
    begun = true;
  };
  int live_tokens = 0;
  int t = lo + Gr::index();                                // the next token to be worked on
  int ahead = t;                                           // ... to be fetched
  const T* row = logits + static_cast<long long>(t) * p.experts;
  const T* row_ahead = row;
  const int* slots = p.ids + static_cast<long long>(t) * p.topk;
  const long long row_step = static_cast<long long>(Gr::kPerBlock) * p.experts;
  const int slot_step = Gr::kPerBlock * p.topk;
  const int* slots_ahead = slots;
  auto fetch = [&](int stage) {
    if (ahead < hi) {
      rows.push(stage, row_ahead, p.experts, lane);
      if (lane < p.topk) first_ids.push(stage, slots_ahead + lane);
    }
    queue_commit();
    ahead += Gr::kPerBlock;
    row_ahead += row_step;
    slots_ahead += slot_step;
  };
  auto count = [&](int id) {
    const bool valid = static_cast<unsigned>(id) < static_cast<unsigned>(p.experts);
    if (valid) atomicAdd(&s_counts[id], 1);
    return valid;
  };
  for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  // the threads of a block take the same number of steps; a group without a token left has t >= hi
  const int steps = (hi - lo + Gr::kPerBlock - 1) / Gr::kPerBlock;
  for (int step = 0; step < steps; ++step) {
    const int stage = step & (kDepth - 1);
    if (step != 0 && (step & (kRun<G> - 1)) == 0) flush();
    fetch((step + kDepth - 1) & (kDepth - 1));
    queue_wait();
    float z[N];
    rows.pop(stage, row, z, p.experts, lane);
    const bool in = t < hi;
    bool mine = in && lane < p.topk && count(first_ids.pop(stage));
    if (in)
      for (int j = lane + G; j < p.topk; j += G) mine |= count(slots[j]);
    t += Gr::kPerBlock;
    row += row_step;
    slots += slot_step;
    const bool live = Gr::any(mine);
    if (!Gr::any_here(live)) continue;
    live_tokens += live;
    auto add = [&](const float (&x)[N], float inv) {
      if (live) {
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
      }
    };
    if (!p.softmax) {
      // 1 / (1 + e^-z) from the exponential and the reciprocal instruction: a few ulp
      float sc[N];
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sc[i] = reciprocal(1.0f + exponential(-z[i]));
        sum += sc[i];
      }
      sum = Gr::sum(sum, scratch);
      const bool vanish = live && !(sum >= kMinSum);
      float inv = reciprocal(sum);
      if (Gr::any_here(vanish)) {
        // scores that all vanish (every logit below about -57) are e^z: normalised as e^(z - max)
        const float other = exponentials<N, G>(z, scratch);
        inv = vanish ? other : inv;
#pragma unroll
        for (int i = 0; i < N; ++i) sc[i] = vanish ? z[i] : sc[i];
      }
      add(sc, inv);
    } else {
      add(z, exponentials<N, G>(z, scratch));
    }
  }
  if (lane == 0) atomicAdd(&s_live, live_tokens);
  flush();
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();                                         // every group's sums, and the counts
  for (int e = threadIdx.x; e < p.width; e += kThreads) {
    if constexpr (G <= 32) {
      part[e] = sum_rows<Gr::kPerBlock>([&](int r) { return s_sums[r * p.width + e]; });
    }
    p.part_n[static_cast<long long>(item) * p.width + e] = s_counts[e];
  }
  if (threadIdx.x == 0) p.part_t[item] = make_int2(s, s_live);
}

// Live tokens of every sequence and the number of sequences that have any, a warp per sequence. With few sequences
// the blocks of the next kernel find both among all items themselves, which saves this launch; but that is sequences x
// items in all. 65536 tokens x 256 in 32 / 128 / 256 / 512 / 1024 / 4096 / 16384 sequences, us with the scan: 23 / 31 / 38 / 50 /
// 78 / 388 / 3842; with this kernel: 23 / 32 / 36 / 43 / 58 / 149 / 548. 4096 tokens x 64 in 128 / 256 / 512 / 1024: 8.3 / 9.0 /
// 12.0 / 23 and 9.6 / 10.0 / 12.8 / 21.
__global__ void __launch_bounds__(kThreads)
balance_live_kernel(const LossParams p) {
  const int s = static_cast<int>(blockIdx.x) * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int lo = s < p.sequences ? seq_start(p, s) : 0, hi = s < p.sequences ? seq_start(p, s + 1) : 0;
  ptx::grid_wait();                                        // the items are complete
  ptx::grid_launch_dependents();
  int tokens = 0;
  if (hi > lo) {
    const int first = lo / p.chunk + s, last = (hi - 1) / p.chunk + s;
    for (int i = first + lane; i <= last; i += 32) tokens += p.part_t[i].y;
  }
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  const int filled = __syncthreads_count(tokens > 0) / 32;
  if (s < p.sequences && lane == 0) p.live[s] = tokens;
  if (threadIdx.x == 0 && filled > 0) atomicAdd(&p.ticket[1], static_cast<unsigned>(filled));
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(kThreads, 2)
balance_partial_kernel(const T* logits, const LossParams p) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  add_item<T, V, NV, G>(logits, p, s_raw, blockIdx.x);
}

struct ReduceShared {
  alignas(16) double p[16][64];            // (written two and four columns at a time)
  alignas(16) int n[16][64];
  int tokens, count;
  double loss[kWarps];
};
static_assert(alignof(ReduceShared) == 16, "rows of four");

// Adds a sequence's partial rows for 64 columns (item order within sixteen interleaved strands, then the strands) and
// writes counts and slopes; thread 0 gets their part of the loss. It is a chain of latencies, so everything
// that does not depend on the partial sums happens before `partials_ready` waits for them, and independent
// loads are issued together. `filled_bits`: one per sequence, where the live tokens have not been counted before.
template <typename Ready>
__device__ __forceinline__ double reduce_columns(const LossParams& p, int s, int col_block, unsigned* filled_bits, ReduceShared& sh,
                                                 Ready partials_ready) {
  const int items = p.chunks + p.sequences;
  const int words = (p.sequences + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool scan = p.live == nullptr;
  for (int i = threadIdx.x; scan && i < words; i += kThreads) filled_bits[i] = 0;
  if (threadIdx.x == 0) { sh.tokens = 0; sh.count = 0; }
  const int lo = seq_start(p, s), hi = seq_start(p, s + 1);
  const int strand = threadIdx.x >> 4, quad = threadIdx.x & 15;
  const int col = col_block * 64 + quad * 4;
  __syncthreads();
  partials_ready();
  double2 sum = make_double2(0.0, 0.0), sum2 = sum;       // columns 0 and 1, 2 and 3
  int4 num = make_int4(0, 0, 0, 0);
  if (hi > lo && col < p.width) {
    const int first = lo / p.chunk + s, last = (hi - 1) / p.chunk + s;
#pragma unroll 4
    for (int i = first + strand; i <= last; i += 16) {
      const double2* from = reinterpret_cast<const double2*>(p.part_p + static_cast<long long>(i) * p.width + col);
      const double2 a = from[0], b = from[1];
      const int4 n = *reinterpret_cast<const int4*>(p.part_n + static_cast<long long>(i) * p.width + col);
      sum.x += a.x; sum.y += a.y; sum2.x += b.x; sum2.y += b.y;
      num.x += n.x; num.y += n.y; num.z += n.z; num.w += n.w;
    }
  }
  *reinterpret_cast<double2*>(&sh.p[strand][quad * 4]) = sum;
  *reinterpret_cast<double2*>(&sh.p[strand][quad * 4 + 2]) = sum2;
  *reinterpret_cast<int4*>(&sh.n[strand][quad * 4]) = num;
  if (scan) {
#pragma unroll 2
    for (int i = threadIdx.x; i < items; i += kThreads) {
      const int2 t = p.part_t[i];
      if (t.y > 0) {
        atomicOr(&filled_bits[t.x >> 5], 1u << (t.x & 31));
        if (t.x == s) atomicAdd(&sh.tokens, t.y);
      }
    }
    __syncthreads();
    int filled = 0;
    for (int i = threadIdx.x; i < words; i += kThreads) filled += __popc(filled_bits[i]);
    if (filled) atomicAdd(&sh.count, filled);
  } else if (threadIdx.x == 0) {
    sh.tokens = p.live[s];
    sh.count = static_cast<int>(p.ticket[1]);
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int e = col_block * 64 + threadIdx.x;
    const double total = sum_rows<16>([&](int r) { return sh.p[r][threadIdx.x]; });
    int n = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) n += sh.n[r][threadIdx.x];
    double term = 0.0;
    if (e < p.experts) {
      // alpha E n / (k T^2 S') in FP64, rounded once
      const double t = sh.tokens > 0 ? static_cast<double>(sh.tokens) : 1.0;
      const double slope = static_cast<double>(p.alpha) * p.experts * n / (static_cast<double>(p.topk) * t * t * max(sh.count, 1));
      p.counts[static_cast<long long>(s) * p.experts + e] = n;
      p.slope[static_cast<long long>(s) * p.experts + e] = static_cast<float>(slope);
      term = slope * total;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) term += __shfl_xor_sync(0xffffffffu, term, d);
    if (lane == 0) sh.loss[warp] = term;
  }
  __syncthreads();
  return threadIdx.x == 0 ? sh.loss[0] + sh.loss[1] : 0.0;
}

// The loss from its parts, by one block, in a fixed order.
__device__ __forceinline__ void sum_loss(const LossParams& p, long long terms, ReduceShared& sh) {
  double mine = 0.0;
#pragma unroll 8
  for (long long i = threadIdx.x; i < terms; i += kThreads) mine += __ldcg(p.part_loss + i);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.loss[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < kWarps; ++w) all += sh.loss[w];
    *p.loss = static_cast<float>(all);
  }
}

// One block per sequence and 64 columns; the last one to finish adds up the loss. Whatever ran before the first kernel
// has ended when this one (or the one between) starts: that kernel lets it start only then.
__global__ void __launch_bounds__(kThreads)
balance_reduce_kernel(const LossParams p) {
  extern __shared__ unsigned s_filled[];                   // one bit per sequence
  __shared__ ReduceShared sh;
  __shared__ bool s_last;
  const double part = reduce_columns(p, blockIdx.x, blockIdx.y, s_filled, sh, [] {
    ptx::grid_wait();                                      // the partial sums are complete
    ptx::grid_launch_dependents();
  });
  if (threadIdx.x == 0) {
    p.part_loss[static_cast<long long>(blockIdx.x) * gridDim.y + blockIdx.y] = part;
    __threadfence();
    s_last = atomicAdd(p.ticket, 1u) == gridDim.x * gridDim.y - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  sum_loss(p, static_cast<long long>(p.sequences) * gridDim.y, sh);
}

// Both steps in one launch, for what kOne work items at most hold: a cluster of that many blocks, which meets
// before the sums are added and before the loss is.
constexpr int kOne = 8;

template <typename T, int V, int NV, int G>
__global__ void __cluster_dims__(kOne, 1, 1) __launch_bounds__(kThreads)
balance_one_kernel(const T* logits, const LossParams p) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  __shared__ ReduceShared sh;
  __shared__ unsigned filled;
  if (blockIdx.x < p.chunks + p.sequences) {
    add_item<T, V, NV, G>(logits, p, s_raw, blockIdx.x);
  } else {
    ptx::grid_wait();
    ptx::grid_launch_dependents();
  }
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  const int col_blocks = (p.experts + 63) / 64, parts = p.sequences * col_blocks;
  for (int i = blockIdx.x; i < parts; i += kOne) {
    const double part = reduce_columns(p, i / col_blocks, i % col_blocks, &filled, sh, [] {});
    if (threadIdx.x == 0) p.part_loss[i] = part;
    __syncthreads();
  }
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (blockIdx.x == 0) sum_loss(p, parts, sh);
}

// ---------------------------------------------------------------------------------------- host

// Tokens per work item. Two blocks of the first kernel are resident per SM, and there are about as many
// items as chunks and sequences together: with few sequences the items fill the GPU exactly once (a
// few items more than that cost a second round: 131072 x 160 BF16 46 us with 467 items on 444 places, 40
// with 296), with many sequences there are several rounds anyway. Fixed, so that the order of the sums does
// not depend on the device: 148 SMs.
int loss_chunk(int tokens, int experts, int sequences) {
  constexpr int kResident = 2 * 148;
  const int chunks = sequences <= kResident / 2 ? kResident - sequences : 2 * kResident;
  const long long chunk = (static_cast<long long>(tokens) + chunks - 1) / chunks;
  const int least = experts <= 512 ? 32 : 4;               // (a block goes through 8 to 32 tokens at a time, or one: 400 x 1024 33 -> 12 us)
  return static_cast<int>(chunk < least ? least : chunk);
}

struct LossLayout {
  bool one;
  int chunk, chunks, width, col_blocks;
  size_t p, n, t, loss, ticket, live, total;
};

constexpr int kScanned = 256;  // sequences whose live tokens every block of the last kernel counts for itself


LossLayout loss_layout(int tokens, int experts, int sequences) {
  LossLayout l;
  // A call for a few tokens is launches more than anything: where the kOne blocks of a cluster, less one for each
  // sequence's end, get through the tokens in four steps each, and through the sums in one, one launch does
  // it all (64 x 64: 7.4 -> 6.5 us, 120 x 64 in 3 sequences 6.5 -> 6.2, and 8.4 -> 6.5 on the host; with two rounds of sums
  // 300 x 160, 3 sequences, took 8.6 against 7.5).
  const int most = experts <= 256 ? 64 : 32;
  l.one = sequences < kOne && sequences * ((experts + 63) / 64) <= kOne && tokens <= most * (kOne - sequences);
  l.chunk = l.one ? (tokens <= 32 * (kOne - sequences) ? 32 : 64) : loss_chunk(tokens, experts, sequences);
  l.chunks = (tokens + l.chunk - 1) / l.chunk;
  l.width = (experts + 3) / 4 * 4;
  l.col_blocks = (experts + 63) / 64;
  const size_t rows = static_cast<size_t>(l.chunks) + sequences;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.p = 0;
  l.n = up(l.p + rows * l.width * 8);
  l.t = up(l.n + rows * l.width * 4);
  l.loss = up(l.t + rows * 8);
  l.ticket = up(l.loss + static_cast<size_t>(sequences) * l.col_blocks * 8);
  l.live = up(l.ticket + 8);
  l.total = sequences > kScanned ? up(l.live + static_cast<size_t>(sequences) * 4) : l.live;
  return l;
}

template <typename T, int V, int NV, int G>
struct LossLaunch {
  static int run(const void* logits, LossParams p, bool one, int device, cudaStream_t stream) {
    static std::once_flag once[64], once_one[64];
    static cudaError_t status[64], status_one[64];
    auto kernel = balance_partial_kernel<T, V, NV, G>;
    if constexpr (G <= 32) {                               // (more than 512 experts never go through one launch)
      if (one) kernel = balance_one_kernel<T, V, NV, G>;
    }
    constexpr int kMaxWidth = G > 32 ? kMaxExperts : V * NV * G;
    constexpr size_t kQueues = RowQueue<T, V, NV, G>::kBytes + WordQueue<int>::kBytes;
    auto sums = [](int width) { return G > 32 ? 0 : static_cast<size_t>(Group<G>::kPerBlock) * width * 8; };
    constexpr size_t kMost = kQueues + (G > 32 ? 0 : static_cast<size_t>(Group<G>::kPerBlock) * kMaxWidth * 8) + kMaxWidth * 4;
    static_assert(kQueues % 16 == 0 && kMost <= 112 * 1024, "two blocks per SM");
    const int allowed = allow_smem(kernel, one ? once_one : once, one ? status_one : status, device, static_cast<int>(kMost));
    if (allowed != B200_NVFP4_SUCCESS) return allowed;
    p.counts_at = static_cast<int>(kQueues + sums(p.width));
    return launch_overlapped(kernel, one ? kOne : p.chunks + p.sequences, kThreads, p.counts_at + static_cast<size_t>(p.width) * 4, 1, stream,
                             static_cast<const T*>(logits), p);
  }
};

}  // namespace
}  // namespace router
}  // namespace b200

extern "C" {

size_t b200_nvfp4_moe_balance_loss_workspace_bytes(int num_tokens, int num_experts, int num_sequences) {
  using namespace b200;
  using namespace b200::router;
  if (!valid_router(num_tokens, num_experts, 1, num_sequences, 0)) return 0;
  return loss_layout(num_tokens, num_experts, num_sequences).total;
}

int b200_nvfp4_moe_balance_loss(void* loss, void* counts, void* slope, const void* logits, const void* topk_ids,
                                const void* cu_seqlens, int num_tokens, int num_experts, int num_topk, int num_sequences,
                                int logits_dtype, int scoring, float alpha, void* workspace, size_t workspace_bytes,
                                b200_stream_t stream) {
  using namespace b200;
  using namespace b200::router;
  if (!valid_router(num_tokens, num_experts, num_topk, num_sequences, logits_dtype) || loss == nullptr || counts == nullptr ||
      slope == nullptr || (num_tokens > 0 && (logits == nullptr || topk_ids == nullptr)) || scoring < 0 || scoring > 1 ||
      (cu_seqlens == nullptr && num_sequences != 1) || !aligned(logits, element_size(logits_dtype)) ||
      !aligned(workspace, 256) || !aligned(loss, 4) || !aligned(counts, 4) || !aligned(slope, 4) || !aligned(topk_ids, 4) ||
      !aligned(cu_seqlens, 4))
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
  p.part_p = reinterpret_cast<double*>(ws + l.p);
  p.part_n = reinterpret_cast<int*>(ws + l.n);
  p.part_t = reinterpret_cast<int2*>(ws + l.t);
  p.part_loss = reinterpret_cast<double*>(ws + l.loss);
  p.ticket = reinterpret_cast<unsigned*>(ws + l.ticket);
  p.live = num_sequences > kScanned ? reinterpret_cast<int*>(ws + l.live) : nullptr;
  p.loss = static_cast<float*>(loss);
  p.counts = static_cast<int*>(counts);
  p.slope = static_cast<float*>(slope);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t size = element_size(logits_dtype);
  const bool quads = num_experts % 4 == 0 && aligned(logits, 4 * size);
  int status;
  switch (logits_dtype) {
    case 0: status = dispatch_width<__half, LossLaunch>(num_experts, quads, logits, p, l.one, dev.device, s); break;
    case 1: status = dispatch_width<__nv_bfloat16, LossLaunch>(num_experts, quads, logits, p, l.one, dev.device, s); break;
    default: status = dispatch_width<float, LossLaunch>(num_experts, quads, logits, p, l.one, dev.device, s); break;
  }
  if (status != B200_NVFP4_SUCCESS || l.one) return status;
  // each of the next kernels may start while the one before drains: it waits for its end itself
  if (num_sequences > kScanned) {
    status = launch_overlapped(balance_live_kernel, (num_sequences + kWarps - 1) / kWarps, kThreads, 0, 1, s, p);
    if (status != B200_NVFP4_SUCCESS) return status;
  }
  const size_t bits = num_sequences > kScanned ? 0 : static_cast<size_t>((num_sequences + 31) / 32) * 4;
  return launch_overlapped(balance_reduce_kernel, dim3(num_sequences, l.col_blocks), kThreads, bits, 1, s, p);
}

}  // extern "C"
