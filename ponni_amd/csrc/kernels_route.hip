// Routing: the top-k experts of every sample, and the assignments sorted by
// expert, within an expert by sample.
//
// Three launches: the choices, with one bit per sample and expert; the starts
// of every block of samples within every group; the places.
#include <hip/hip_runtime.h>

#include "experts.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr int kSamples = 256;  // of a workgroup, one lane each
constexpr int kWords = kSamples / 32;

// This block's samples of each expert, one bit each: bits[e * kWords + word].
__device__ inline void mark(unsigned* bits, int expert, int sample) {
  atomicOr(&bits[expert * kWords + (sample >> 5)], 1u << (sample & 31));
}
__device__ inline int count(unsigned const* bits, int expert) {
  int n = 0;
#pragma unroll
  for (int w = 0; w < kWords; w++) n += __popc(bits[expert * kWords + w]);
  return n;
}

template <class S, int K>
__global__ __launch_bounds__(kSamples) void route_choose(S const* __restrict__ scores, int64_t ld, int normalize,
                                                         ponni_routing r, int32_t* __restrict__ counts) {
  extern __shared__ unsigned bits[];
  int const E = r.num_experts, k = r.top_k;
  for (int i = threadIdx.x; i < E * kWords; i += kSamples) bits[i] = 0;
  __syncthreads();
  int64_t const b = int64_t(blockIdx.x) * kSamples + threadIdx.x;
  if (b < r.batch) {
    float v[K];
    int at[K];
#pragma unroll
    for (int j = 0; j < K; j++) {
      v[j] = -__builtin_inff();
      at[j] = -1;
    }
    // The softmax's sum over all experts runs with the largest score so far.
    float largest = -__builtin_inff(), sum = 0.0f;
    for (int e = 0; e < E; e++) {
      float s = float(scores[int64_t(e) * ld + b]);
      if (!(s > -__builtin_inff())) continue;  // ruled out: -inf or NaN
      if (normalize == PONNI_ROUTE_ALL) {
        float const d = s == largest ? 1.0f : expf(-__builtin_fabsf(s - largest));
        sum = s > largest ? fmaf(sum, d, 1.0f) : sum + d;
        largest = fmaxf(largest, s);
      }
      int i = e;
      bool before = false;
#pragma unroll
      for (int j = 0; j < K; j++) {  // (in front of the smaller ones: behind a tie, and all after it move)
        before = before || s > v[j];
        float const t = before ? v[j] : s;
        int const ti = before ? at[j] : i;
        v[j] = before ? s : v[j];
        at[j] = before ? i : at[j];
        s = t;
        i = ti;
      }
    }
    float p[K];
#pragma unroll
    for (int j = 0; j < K; j++) p[j] = at[j] < 0 || j >= k ? 0.0f : v[j] == v[0] ? 1.0f : expf(v[j] - v[0]);
    if (normalize != PONNI_ROUTE_ALL) {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < K; j++) sum += p[j];
    }
#pragma unroll
    for (int j = 0; j < K; j++) {
      if (j >= k) break;
      r.experts[j * r.batch + b] = at[j];
      r.weights[j * r.batch + b] = at[j] < 0 ? 0.0f : p[j] / sum;
      if (at[j] >= 0) mark(bits, at[j], threadIdx.x);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kSamples) counts[int64_t(blockIdx.x) * E + e] = count(bits, e);
}

// offsets, and counts[block][e] becomes the first column of that block's samples in group e.
__global__ __launch_bounds__(1024) void route_offsets(ponni_routing r, int32_t* __restrict__ counts, int64_t blocks) {
  __shared__ int32_t totals[1024];
  int const E = r.num_experts, e = threadIdx.x;
  int32_t total = 0;
  if (e < E)
    for (int64_t i = 0; i < blocks; i++) total += counts[i * E + e];
  totals[e] = total;
  __syncthreads();
  for (int d = 1; d < 1024; d *= 2) {
    int32_t const t = e >= d ? totals[e - d] : 0;
    __syncthreads();
    totals[e] += t;
    __syncthreads();
  }
  if (e < E) {
    int32_t at = totals[e] - total;
    r.offsets[e] = at;
    if (e == E - 1) r.offsets[E] = totals[e];
    for (int64_t i = 0; i < blocks; i++) {
      int32_t const n = counts[i * E + e];
      counts[i * E + e] = at;
      at += n;
    }
  }
}

__global__ __launch_bounds__(kSamples) void route_place(ponni_routing r, int32_t const* __restrict__ starts) {
  extern __shared__ unsigned bits[];
  int const E = r.num_experts, k = r.top_k;
  for (int i = threadIdx.x; i < E * kWords; i += kSamples) bits[i] = 0;
  __syncthreads();
  int64_t const b = int64_t(blockIdx.x) * kSamples + threadIdx.x;
  if (b < r.batch)
    for (int j = 0; j < k; j++) {
      int const e = r.experts[j * r.batch + b];
      if (e >= 0) mark(bits, e, threadIdx.x);
    }
  __syncthreads();
  if (b >= r.batch) return;
  int32_t const total = r.offsets[E];
  for (int j = 0; j < k; j++) {
    int const e = r.experts[j * r.batch + b];
    int32_t slot = -1;
    if (e >= 0) {
      int const word = threadIdx.x >> 5;
      slot = starts[int64_t(blockIdx.x) * E + e] +
             __popc(bits[e * kWords + word] & ((1u << (threadIdx.x & 31)) - 1u));
      for (int w = 0; w < word; w++) slot += __popc(bits[e * kWords + w]);
      r.source[slot] = static_cast<int32_t>(b);
    }
    r.slots[j * r.batch + b] = slot;
    int64_t const tail = j * r.batch + b;
    if (tail >= total) r.source[tail] = -1;
  }
}

template <class S>
void choose(S const* scores, int64_t ld, int normalize, ponni_routing const& r, int32_t* counts, dim3 grid,
            hipStream_t stream) {
  size_t const lds = size_t(r.num_experts) * kWords * 4;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kSamples), lds, stream, scores, ld, normalize, r, counts);
  };
  if (r.top_k == 1) launch(route_choose<S, 1>);
  else if (r.top_k == 2) launch(route_choose<S, 2>);
  else if (r.top_k <= 4) launch(route_choose<S, 4>);
  else if (r.top_k <= 8) launch(route_choose<S, 8>);
  else launch(route_choose<S, 16>);
}

}  // namespace

int64_t route_workspace_bytes(int64_t experts, int64_t batch) {
  return (batch + kSamples - 1) / kSamples * experts * int64_t(sizeof(int32_t));
}

hipError_t launch_route(const void* scores, int64_t ld, int dtype, int normalize, ponni_routing const& r, void* workspace,
                        hipStream_t stream) {
  int64_t const blocks = (r.batch + kSamples - 1) / kSamples;
  dim3 const grid(static_cast<unsigned>(blocks));
  auto* counts = static_cast<int32_t*>(workspace);
  with_dtype(dtype, [&](auto s) { choose(static_cast<decltype(s) const*>(scores), ld, normalize, r, counts, grid, stream); });
  hipLaunchKernelGGL(route_offsets, dim3(1), dim3(1024), 0, stream, r, counts, blocks);
  hipLaunchKernelGGL(route_place, grid, dim3(kSamples), size_t(r.num_experts) * kWords * 4, stream, r, counts);
  return hipGetLastError();
}

}  // namespace ponni_hip
