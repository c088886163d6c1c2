// Routing: the top-k experts of every sample, and the assignments sorted by
// expert, within an expert by sample.
//
// A score and its expert are one unsigned key, largest score first, of equal
// ones the lower index: 32 bits for 16-bit scores (a 16-bit number as a float
// has 13 zero bits at its end, which hold the index), 64 for fp32.  A lane
// runs down its experts with its K largest keys in order: per score and place
// one maximum and one minimum (32 bits).  With few samples P lanes share one,
// each a part of the experts, and merge their lists.
//
// Places come from one bit per sample and expert of a workgroup's samples: a
// group's count is a population count, a sample's rank in it the count of the bits
// below.  Few samples are one launch; more are three: choices and counts, the
// counts' sums over the workgroups before, places.  Top 4 of 64 experts,
// 1,000,003 bf16 samples: 81 us (chosen) and 96 us (all) where the bytes take 34; bound by
// VALU issue.  8 experts, 96 samples: 5 us, the launch and one pass of dependent steps.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "experts.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr float kLog2eF = 1.4426950408889634f;

template <class S> using Key = std::conditional_t<sizeof(S) == 2, uint32_t, uint64_t>;
constexpr uint32_t kIndexBits = 0x1fff;
static_assert(PONNI_MAX_EXPERTS <= kIndexBits, "an index fits the key");

// 0: the score rules the expert out (-inf or NaN).
template <class S> __device__ inline Key<S> key_of(float s, int expert) {
  uint32_t const b = __builtin_bit_cast(uint32_t, s + 0.0f);  // (-0 and 0 are equal)
  uint32_t const ordered = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
  bool const ok = s > -__builtin_inff();
  if constexpr (sizeof(S) == 2) return ok ? (ordered & ~kIndexBits) | (kIndexBits - expert) : 0u;
  else return ok ? uint64_t(ordered) << 32 | (0xffffffffu - expert) : uint64_t(0);
}
template <class K> __device__ inline int expert_of(K key) {
  if (key == 0) return -1;
  if constexpr (sizeof(K) == 4) return kIndexBits - (key & kIndexBits);
  else return 0xffffffffu - uint32_t(key);
}
template <class K> __device__ inline float score_of(K key) {
  if (key == 0) return -__builtin_inff();
  uint32_t ordered;
  if constexpr (sizeof(K) == 4) ordered = key & ~kIndexBits;
  else ordered = uint32_t(key >> 32);
  uint32_t const b = ordered & 0x80000000u ? ordered ^ 0x80000000u : ~ordered & (sizeof(K) == 4 ? ~kIndexBits : ~0u);
  return __builtin_bit_cast(float, b);
}
template <int K, class T> __device__ inline void insert(T (&list)[K], T key) {
#pragma unroll
  for (int j = 0; j < K; j++) {
    T const above = list[j] > key ? list[j] : key;
    key = list[j] > key ? key : list[j];
    list[j] = above;
  }
}

// Calls f(score, expert) for the experts first .. last - 1 of sample b, eight loads in flight.
template <class S, class F>
__device__ inline void each_score(S const* __restrict__ scores, int64_t ld, int64_t b, int first, int last, F&& f) {
  int e = first;
  for (; e + 8 <= last; e += 8) {
    S s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = scores[int64_t(e + i) * ld + b];
#pragma unroll
    for (int i = 0; i < 8; i++) f(float(s[i]), e + i);
  }
  for (; e < last; e++) f(float(scores[int64_t(e) * ld + b]), e);
}

// exp(s - largest); the same number for equal scores, also infinite ones.
__device__ inline float term(float s, float largest) {
  float const d = (s - largest) * kLog2eF;
  return largest == __builtin_inff() ? (s == largest ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(d);
}

// This workgroup's samples of each expert, one bit each: bits[expert * words + word].
template <int SAMPLES> __device__ inline void mark(unsigned* bits, int expert, int sample) {
  atomicOr(&bits[expert * (SAMPLES / 32) + (sample >> 5)], 1u << (sample & 31));
}
template <int SAMPLES> __device__ inline int count(unsigned const* bits, int expert) {
  int n = 0;
#pragma unroll
  for (int w = 0; w < SAMPLES / 32; w++) n += __popc(bits[expert * (SAMPLES / 32) + w]);
  return n;
}
template <int SAMPLES> __device__ inline int rank(unsigned const* bits, int expert, int sample) {
  unsigned const* b = bits + expert * (SAMPLES / 32);
  int const word = sample >> 5;
  int n = __popc(b[word] & ((1u << (sample & 31)) - 1u));
  for (int w = 0; w < word; w++) n += __popc(b[w]);
  return n;
}

// sums[e] = the first sorted column of expert e's group from counts of n experts
// in sums; returns the total.  All threads of the workgroup; partial holds one per thread.
template <int THREADS> __device__ inline int32_t scan_counts(int32_t* sums, int n, int32_t* partial) {
  int const per = (n + THREADS - 1) / THREADS, at = threadIdx.x * per;
  int32_t own = 0;
  for (int i = at; i < at + per && i < n; i++) own += sums[i];
  partial[threadIdx.x] = own;
  __syncthreads();
  for (int d = 1; d < THREADS; d *= 2) {
    int32_t const t = int(threadIdx.x) >= d ? partial[threadIdx.x - d] : 0;
    __syncthreads();
    partial[threadIdx.x] += t;
    __syncthreads();
  }
  int32_t before = partial[threadIdx.x] - own;
  for (int i = at; i < at + per && i < n; i++) {
    int32_t const c = sums[i];
    sums[i] = before;
    before += c;
  }
  __syncthreads();
  return partial[THREADS - 1];
}

template <class S, int K, int P, int SAMPLES, bool SINGLE>
__global__ __launch_bounds__(SAMPLES * P) void route_choose(S const* __restrict__ scores, int64_t ld, int normalize,
                                                            ponni_routing r, int32_t* __restrict__ counts) {
  extern __shared__ unsigned bits[];
  __shared__ int32_t starts[SINGLE ? PONNI_MAX_EXPERTS : 1], partial[SINGLE ? SAMPLES * P : 1];
  constexpr int THREADS = SAMPLES * P, WAVE_SAMPLES = 64 / P;
  int const E = r.num_experts, k = r.top_k, lane = threadIdx.x & 63;
  int const local = (threadIdx.x >> 6) * WAVE_SAMPLES + lane % WAVE_SAMPLES, part = lane / WAVE_SAMPLES;
  for (int i = threadIdx.x; i < E * (SAMPLES / 32); i += THREADS) bits[i] = 0;
  __syncthreads();
  int64_t const sample = int64_t(blockIdx.x) * SAMPLES + local;
  bool const valid = sample < r.batch;
  int64_t const b = valid ? sample : r.batch - 1;
  int const per = (E + P - 1) / P, first = part * per < E ? part * per : E, last = first + per < E ? first + per : E;
  Key<S> list[K] = {};
  each_score(scores, ld, b, first, last, [&](float s, int e) { insert(list, key_of<S>(s, e)); });
#pragma unroll
  for (int d = WAVE_SAMPLES; d < 64; d *= 2) {
    Key<S> other[K];
#pragma unroll
    for (int j = 0; j < K; j++) other[j] = __shfl_xor(list[j], d);
#pragma unroll
    for (int j = 0; j < K; j++) insert(list, other[j]);
  }
  float const largest = score_of(list[0]);
  float sum = 0.0f;
  if (normalize == PONNI_ROUTE_ALL) {
    // (a score that is NaN counts as -inf)
    each_score(scores, ld, b, first, last, [&](float s, int) { sum += term(fmaxf(s, -__builtin_inff()), largest); });
#pragma unroll
    for (int d = WAVE_SAMPLES; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  }
  float p[K];
#pragma unroll
  for (int j = 0; j < K; j++) {
    float const s = score_of(list[j]);
    p[j] = j >= k || list[j] == 0 ? 0.0f : s == largest ? 1.0f : expf(s - largest);
    if (normalize != PONNI_ROUTE_ALL) sum += p[j];
  }
  int at[K];
#pragma unroll
  for (int j = 0; j < K; j++) {
    at[j] = j < k && valid && part == 0 ? expert_of(list[j]) : -1;
    if (j < k && valid && part == 0) {
      r.experts[j * r.batch + b] = at[j];
      r.weights[j * r.batch + b] = at[j] < 0 ? 0.0f : p[j] / sum;
    }
    if (at[j] >= 0) mark<SAMPLES>(bits, at[j], local);
  }
  __syncthreads();
  if constexpr (SINGLE) {
    for (int e = threadIdx.x; e < E; e += THREADS) starts[e] = count<SAMPLES>(bits, e);
    __syncthreads();
    int32_t const total = scan_counts<THREADS>(starts, E, partial);
    for (int e = threadIdx.x; e < E; e += THREADS) r.offsets[e] = starts[e];
    if (threadIdx.x == 0) r.offsets[E] = total;
    if (valid && part == 0) {
#pragma unroll
      for (int j = 0; j < K; j++) {
        if (j >= k) break;
        int32_t const slot = at[j] < 0 ? -1 : starts[at[j]] + rank<SAMPLES>(bits, at[j], local);
        r.slots[j * r.batch + b] = slot;
        if (slot >= 0) r.source[slot] = static_cast<int32_t>(b);
      }
    }
    for (int64_t i = total + int64_t(threadIdx.x); i < k * r.batch; i += THREADS) r.source[i] = -1;
  } else {
    for (int e = threadIdx.x; e < E; e += THREADS) counts[int64_t(e) * gridDim.x + blockIdx.x] = count<SAMPLES>(bits, e);
  }
}

// One expert: counts[e][block] becomes the number of its samples in the blocks before; totals[e] all of them.
__global__ __launch_bounds__(256) void route_sums(int32_t* __restrict__ counts, int blocks, int32_t* __restrict__ totals) {
  __shared__ int32_t partial[256];
  int32_t* row = counts + int64_t(blockIdx.x) * blocks;
  int32_t before = 0;
  for (int base = 0; base < blocks; base += 1024) {
    // four consecutive blocks a thread
    int32_t n[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      int const at = base + 4 * threadIdx.x + i;
      n[i] = at < blocks ? row[at] : 0;
      own += n[i];
    }
    partial[threadIdx.x] = own;
    __syncthreads();
    for (int d = 1; d < 256; d *= 2) {
      int32_t const t = int(threadIdx.x) >= d ? partial[threadIdx.x - d] : 0;
      __syncthreads();
      partial[threadIdx.x] += t;
      __syncthreads();
    }
    int32_t at = before + partial[threadIdx.x] - own;
    before += partial[255];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (base + 4 * int(threadIdx.x) + i < blocks) row[base + 4 * threadIdx.x + i] = at;
      at += n[i];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

template <int SAMPLES>
__global__ __launch_bounds__(SAMPLES) void route_place(ponni_routing r, int32_t const* __restrict__ counts,
                                                       int32_t const* __restrict__ totals) {
  extern __shared__ unsigned bits[];
  __shared__ int32_t starts[PONNI_MAX_EXPERTS], partial[SAMPLES];
  int const E = r.num_experts, k = r.top_k;
  for (int i = threadIdx.x; i < E * (SAMPLES / 32); i += SAMPLES) bits[i] = 0;
  for (int e = threadIdx.x; e < E; e += SAMPLES) starts[e] = totals[e];
  __syncthreads();
  int32_t const total = scan_counts<SAMPLES>(starts, E, partial);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < E; e += SAMPLES) r.offsets[e] = starts[e];
    if (threadIdx.x == 0) r.offsets[E] = total;
  }
  int64_t const b = int64_t(blockIdx.x) * SAMPLES + threadIdx.x;
  if (b < r.batch)
    for (int j = 0; j < k; j++) {
      int const e = r.experts[j * r.batch + b];
      if (e >= 0) mark<SAMPLES>(bits, e, threadIdx.x);
    }
  __syncthreads();
  if (b >= r.batch) return;
  for (int j = 0; j < k; j++) {
    int const e = r.experts[j * r.batch + b];
    int32_t slot = -1;
    if (e >= 0) {
      slot = starts[e] + counts[int64_t(e) * gridDim.x + blockIdx.x] + rank<SAMPLES>(bits, e, threadIdx.x);
      r.source[slot] = static_cast<int32_t>(b);
    }
    r.slots[j * r.batch + b] = slot;
    if (j * r.batch + b >= total) r.source[j * r.batch + b] = -1;
  }
}

// One launch: up to 64 samples with 16 lanes each, up to 256 with 4 where the experts are few enough for
// one workgroup.  Times in us, one launch / three: 8 experts, top 2, 16 samples 5.2 / 8.8, 256 samples 5.8 / 9.5; 64 experts,
// top 4, 256 samples 9.3 / 11.8; 256 experts, top 8, 64 samples 26 / 32, 256 samples 42 / 34; 1000 experts 59 / 38.
// Three launches: 4 lanes a sample for batches that would leave most of the chip without a wave, each lane's
// loads one after the other.  Top 8 of 512 bf16 scores, 65,000 samples: 59 us with 4 lanes, 85 with one; with
// 16 no fewer (256 fp32 scores, 1,000 samples: 30 with 4, 36 with 16; 64 bf16 scores, top 4, 4096: 11.5 and 12.7).
constexpr int64_t kOneLaunch = 64, kOneLaunchFewExperts = 256, kFewExperts = 128, kSharedBatch = 131072;
bool one_launch(int64_t experts, int64_t batch) {
  return batch <= kOneLaunch || (batch <= kOneLaunchFewExperts && experts <= kFewExperts);
}
int64_t blocks_of(int64_t batch) { return batch <= kSharedBatch ? (batch + 63) / 64 : (batch + 255) / 256; }

template <class S, int K>
void choose(S const* scores, int64_t ld, int normalize, ponni_routing const& r, int32_t* counts, hipStream_t stream) {
  auto launch = [&](auto kernel, int64_t blocks, int threads, int samples) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), size_t(r.num_experts) * samples / 8,
                       stream, scores, ld, normalize, r, counts);
  };
  if (r.batch <= kOneLaunch) launch(route_choose<S, K, 16, 64, true>, 1, 1024, 64);
  else if (one_launch(r.num_experts, r.batch)) launch(route_choose<S, K, 4, 256, true>, 1, 1024, 256);
  else if (r.batch <= kSharedBatch) launch(route_choose<S, K, 4, 64, false>, blocks_of(r.batch), 256, 64);
  else launch(route_choose<S, K, 1, 256, false>, blocks_of(r.batch), 256, 256);
}

}  // namespace

int64_t route_workspace_bytes(int64_t experts, int64_t batch) {
  return one_launch(experts, batch) ? 0 : (blocks_of(batch) + 1) * experts * int64_t(sizeof(int32_t));
}

int64_t route_workspace_bytes_up_to(int64_t experts, int64_t batch) {
  // (larger batches have fewer workgroups at first)
  return std::max(route_workspace_bytes(experts, batch), route_workspace_bytes(experts, std::min(batch, kSharedBatch)));
}

hipError_t launch_route(const void* scores, int64_t ld, int dtype, int normalize, ponni_routing const& r, void* workspace,
                        hipStream_t stream) {
  auto* counts = static_cast<int32_t*>(workspace);
  with_dtype(dtype, [&](auto s) {
    auto const* in = static_cast<decltype(s) const*>(scores);
    using S = decltype(s);
    if (r.top_k == 1) choose<S, 1>(in, ld, normalize, r, counts, stream);
    else if (r.top_k == 2) choose<S, 2>(in, ld, normalize, r, counts, stream);
    else if (r.top_k <= 4) choose<S, 4>(in, ld, normalize, r, counts, stream);
    else if (r.top_k <= 8) choose<S, 8>(in, ld, normalize, r, counts, stream);
    else choose<S, 16>(in, ld, normalize, r, counts, stream);
  });
  if (one_launch(r.num_experts, r.batch)) return hipGetLastError();
  int const blocks = static_cast<int>(blocks_of(r.batch));
  int32_t* totals = counts + int64_t(blocks) * r.num_experts;
  hipLaunchKernelGGL(route_sums, dim3(r.num_experts), dim3(256), 0, stream, counts, blocks, totals);
  int const samples = r.batch <= kSharedBatch ? 64 : 256;
  auto place = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(samples), size_t(r.num_experts) * samples / 8, stream, r, counts, totals);
  };
  if (samples == 64) place(route_place<64>);
  else place(route_place<256>);
  return hipGetLastError();
}

}  // namespace ponni_hip
