// Gated blocks over few columns, 32 or less a workgroup (kernels_gated_f32.hip, kernels_gated_f16.hip,
// kernels_gated_bf16.hip): few launches, bound by the weights' way from memory.
//   thin_product   sums of G^T x and U^T x over slices of k
//   thin_product   h = act(sum) * sum of a slice, then sums of D^T h over it
//   thin_join      y
// or with many parts four, h by a launch of its own (thin_hidden).
//
// A wave's step is 32 k x 128 outputs (16 bits; fp32: 16 x 64): a lane loads 16 bytes of 8
// (4) consecutive rows of weights, so its registers hold an 8 x 8 block, which it turns itself
// (v_perm_b32) into eight fragments: output 8 c + j of the block is fragment j's row c.
// Weights thus go from memory to the matrix cores with no LDS between them, at any
// address.  The columns of a slice lie in LDS, k inside.  The waves of a
// workgroup share a slice's steps; their sums meet in LDS, in the order of the waves.
//
// Bound by the weights' way from memory and by the launches' latency.  bf16 1024-4096-1024, one column (25 MB of weights):
// 6.5 + 6.3 + 4.2 us; fp16 2048-4096-2048, 20 columns (50 MB): 15 + 4 + 13 + 5.
#pragma once

#include "activations.h"
#include "column_rows.h"
#include "gated.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr int kThinWaves = 4;

template <class T> struct ThinTile {
  static constexpr int E = 16 / sizeof(T);              // elements of a load, and its rows
  static constexpr int STEP = 4 * E, OUTPUTS = 16 * E;  // of a wave's step
  static constexpr int PITCH_PAD = E;                   // elements behind a column of a slice
};

// Four of h's values of a column from the parts of g and u, zero from feature `end` on.
template <class T> __device__ inline f32x4 hidden_of(ThinArgs const& a, int col, int k, int end) {
  f32x4 v = {0, 0, 0, 0}, u = v;
  float const* p = a.parts_in + int64_t(col) * a.stride_in + k;
  int64_t const problem_stride = int64_t(a.columns) * a.stride_in;
#pragma unroll 4
  for (int s = 0; s < a.slices_in; s++) {
    v += *reinterpret_cast<f32x4 const*>(p + 2 * s * problem_stride);
    u += *reinterpret_cast<f32x4 const*>(p + (2 * s + 1) * problem_stride);
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (k + e >= end) continue;
    if (a.bias[0] != nullptr) v[e] += float(static_cast<T const*>(a.bias[0])[k + e]);
    if (a.bias[1] != nullptr) u[e] += float(static_cast<T const*>(a.bias[1])[k + e]);
  }
  with_activation<sizeof(T) == 4>(a.act, a.slope, [&](auto f) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float h, d;
      f(v[e], h, d);
      v[e] = k + e < end ? h * u[e] : 0.0f;  // (nothing meets the padding's sums)
    }
  });
  return v;
}

// h [columns, stride_in] of the parts.
template <class T> __global__ __launch_bounds__(256) void thin_hidden(ThinArgs a) {
  int const fours = a.stride_in / 4, i = blockIdx.x * 256 + threadIdx.x, col = i / fours, k = i % fours * 4;
  if (col >= a.columns) return;
  f32x4 const v = hidden_of<T>(a, col, k, a.k);
  Pack<T, 4> o;
#pragma unroll
  for (int e = 0; e < 4; e++) o.set(e, v[e]);
  o.store(static_cast<T*>(a.h) + int64_t(col) * a.stride_in + k, 4);
}

template <class T, int NJ, ThinInput INPUT> __global__ __launch_bounds__(64 * kThinWaves) void thin_product(ThinArgs a) {
  using Tile = ThinTile<T>;
  constexpr int E = Tile::E, STEP = Tile::STEP, OUTPUTS = Tile::OUTPUTS, C = 16 * NJ, U = 2;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const xs = reinterpret_cast<T*>(lds);  // [C][pitch]
  float* const sums = reinterpret_cast<float*>(lds);  // [waves][C][OUTPUTS], behind the products
  int const lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const slice = blockIdx.x % a.slices, tile = blockIdx.x / a.slices, problem = blockIdx.y;
  int const first = blockIdx.z * C, columns = a.columns - first;  // (the first of this workgroup's columns)
  int const k0 = slice * a.slice_k, ks = a.k - k0 < a.slice_k ? a.k - k0 : a.slice_k;  // (k's of the slice)
  int const pitch = a.slice_k + Tile::PITCH_PAD;
  int const m = tile * OUTPUTS + E * c, left = a.outputs - m, count = left < 1 ? 0 : left < E ? left : E;
  T const* const w = static_cast<T const*>(a.w[problem]) + m;
  int const steps = (ks + STEP - 1) / STEP;
  typedef Pack<T, E> Row;
  Row rows[U][E];
  auto load = [&](int step, int u) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      int const k = step * STEP + E * g + e;
      rows[u][e].fill(0.0f);
      if (step < steps && k < ks && count > 0) rows[u][e].load(w + int64_t(k0 + k) * a.ld[problem], count, 0.0f);
    }
  };
  // The first steps' weights are under way while the columns are laid out.
#pragma unroll
  for (int u = 0; u < U; u++) load(wave + u * kThinWaves, u);
  if constexpr (INPUT == THIN_PARTS) {
    for (int i = threadIdx.x; i < C * (a.slice_k / 4); i += 64 * kThinWaves) {
      int const col = i / (a.slice_k / 4), k = i % (a.slice_k / 4) * 4;
      f32x4 v = {0, 0, 0, 0};
      if (col < columns && k < ks) v = hidden_of<T>(a, first + col, k0 + k, k0 + ks);
#pragma unroll
      for (int e = 0; e < 4; e++) xs[col * pitch + k + e] = T(v[e]);
    }
  } else if constexpr (INPUT == THIN_ROWS) {
    // (h has rows of whole pieces, zero past the last feature)
    for (int i = threadIdx.x; i < C * (a.slice_k / E); i += 64 * kThinWaves) {
      int const col = i / (a.slice_k / E), k = i % (a.slice_k / E) * E;
      i32x4 v = {0, 0, 0, 0};
      if (col < columns && k < ks)
        v = *reinterpret_cast<i32x4 const*>(static_cast<T const*>(a.h) + int64_t(first + col) * a.stride_in + k0 + k);
      *reinterpret_cast<i32x4*>(xs + col * pitch + k) = v;
    }
  } else {
    // eight (four) columns of a k a thread
    constexpr int GROUPS = C / E;
    T const* const x = static_cast<T const*>(a.x);
#pragma unroll 4
    for (int i = threadIdx.x; i < GROUPS * a.slice_k; i += 64 * kThinWaves) {
      int const k = i / GROUPS, col = i % GROUPS * E, here = columns - col;
      Pack<T, E> v;
      v.fill(0.0f);
      if (here > 0 && k < ks) v.load(x + int64_t(k0 + k) * a.ld_x + first + col, here < E ? here : E, 0.0f);
#pragma unroll
      for (int e = 0; e < E; e++) xs[(col + e) * pitch + k] = v.raw(e);
    }
  }
  __syncthreads();
  f32x4 acc[E][NJ] = {};
  for (int step = wave; step < steps; step += U * kThinWaves) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      int const at = step + u * kThinWaves;
      if (at >= steps) continue;
      i32x4 f[E];
      if constexpr (sizeof(T) == 2) {
        i32x4 r[E];
#pragma unroll
        for (int e = 0; e < E; e++) r[e] = __builtin_bit_cast(i32x4, rows[u][e].v);
#pragma unroll
        for (int j = 0; j < E; j++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            unsigned const lo = r[2 * q][j / 2], hi = r[2 * q + 1][j / 2];
            f[j][q] = int(__builtin_amdgcn_perm(hi, lo, j % 2 ? 0x07060302u : 0x05040100u));
          }
      } else {
#pragma unroll
        for (int j = 0; j < E; j++)
#pragma unroll
          for (int e = 0; e < E; e++) f[j][e] = __float_as_int(rows[u][e][j]);
      }
      load(at + U * kThinWaves, u);
#pragma unroll
      for (int n = 0; n < NJ; n++) {
        i32x4 const b = *reinterpret_cast<i32x4 const*>(xs + (16 * n + c) * pitch + at * STEP + E * g);
#pragma unroll
        for (int e = 0; e < kMfmaParts<T>; e++)
#pragma unroll
          for (int j = 0; j < E; j++) acc[j][n] = mfma_part<T>(f[j], b, acc[j][n], e);
      }
    }
  }
  __syncthreads();
  // Lane (g, c) holds outputs 4 E g + E e + j of column c.
  // (fours of them at places that depend on the column: other banks)
  auto place = [&](int w, int col, int four) { return ((w * C + col) * (OUTPUTS / 4) + (four ^ (col & 7))) * 4; };
#pragma unroll
  for (int n = 0; n < NJ; n++)
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int j = 0; j < E; j += 4)
        *reinterpret_cast<f32x4*>(sums + place(wave, 16 * n + c, (4 * E * g + E * e + j) / 4)) =
            f32x4{acc[j][n][e], acc[j + 1][n][e], acc[j + 2][n][e], acc[j + 3][n][e]};
  __syncthreads();
  float* const out = a.parts + ((int64_t(slice) * gridDim.y + problem) * a.columns + first) * a.stride + tile * OUTPUTS;
  for (int i = threadIdx.x; i < C * (OUTPUTS / 4); i += 64 * kThinWaves) {
    int const col = i / (OUTPUTS / 4), o = i % (OUTPUTS / 4) * 4;
    if (col >= columns) continue;
    f32x4 s = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < kThinWaves; v++) s += *reinterpret_cast<f32x4 const*>(sums + place(v, col, o / 4));
    *reinterpret_cast<f32x4*>(out + int64_t(col) * a.stride + o) = s;
  }
}

// y = the slices' sums in their order, four outputs of a column a thread.
template <class T> __global__ __launch_bounds__(256) void thin_join(ThinArgs a) {
  int const pieces = a.stride / 4, i = blockIdx.x * 256 + threadIdx.x, col = i / pieces, o = i % pieces * 4;
  if (col >= a.columns) return;
  f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
  for (int k = 0; k < a.slices; k++)
    s += *reinterpret_cast<f32x4 const*>(a.parts + (int64_t(k) * a.columns + col) * a.stride + o);
  T* const y = static_cast<T*>(a.y) + col;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (o + e >= a.outputs) continue;
    float const b = a.bias[0] != nullptr ? float(static_cast<T const*>(a.bias[0])[o + e]) : 0.0f;
    y[int64_t(o + e) * a.ld_y] = T(s[e] + b);
  }
}

template <class T, ThinInput INPUT> hipError_t launch_thin_product(ThinArgs const& a, int problems, hipStream_t stream) {
  using Tile = ThinTile<T>;
  int const tiles = (a.outputs + Tile::OUTPUTS - 1) / Tile::OUTPUTS, c = a.columns <= 16 ? 16 : 32;
  size_t const columns = size_t(c) * (a.slice_k + Tile::PITCH_PAD) * sizeof(T),
               sums = size_t(kThinWaves) * c * Tile::OUTPUTS * 4;
  dim3 const grid(unsigned(tiles * a.slices), unsigned(problems), unsigned((a.columns + c - 1) / c)), block(64 * kThinWaves);
  if (c == 16) hipLaunchKernelGGL((thin_product<T, 1, INPUT>), grid, block, columns > sums ? columns : sums, stream, a);
  else hipLaunchKernelGGL((thin_product<T, 2, INPUT>), grid, block, columns > sums ? columns : sums, stream, a);
  return hipGetLastError();
}

// Both products and y.
template <class T> hipError_t launch_thin_as(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream) {
  hipError_t err = launch_thin_product<T, THIN_COLUMNS>(hidden, 2, stream);
  if (err != hipSuccess) return err;
  if (last.h != nullptr) {
    unsigned const groups = unsigned((int64_t(last.columns) * last.stride_in / 4 + 255) / 256);
    hipLaunchKernelGGL(thin_hidden<T>, dim3(groups), dim3(256), 0, stream, last);
    err = hipGetLastError();
    if (err == hipSuccess) err = launch_thin_product<T, THIN_ROWS>(last, 1, stream);
  } else {
    err = launch_thin_product<T, THIN_PARTS>(last, 1, stream);
  }
  if (err != hipSuccess) return err;
  ThinArgs join = last;
  join.bias[0] = last.bias[2];
  hipLaunchKernelGGL(thin_join<T>, dim3(unsigned((int64_t(last.columns) * last.stride / 4 + 255) / 256)), dim3(256), 0, stream, join);
  return hipGetLastError();
}

}  // namespace
}  // namespace ponni_hip
