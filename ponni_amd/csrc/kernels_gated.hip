// Gated feed-forward blocks: y = D^T (act(G^T x + g0) * (U^T x + u0)) + d0 and the
// gradients.  64 x 64 tiles of a product, operands of any strides through LDS as
// floats, 4 x 4 sums a lane.
#include <algorithm>

#include "activations.h"
#include "blocks.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr int kTile = 64, kDepth = 16;

// One operand: element (i, k) at p[i * row + k * step].
struct Operand {
  void const* p;
  int64_t row, step;
};
// Sum over the terms t and k of a[t](m, k) b[t](n, k); with `pair` a second sum of a2 and b[0].
struct Product {
  Operand a[2], b[2], a2;
  int64_t k;
  int terms;
  int64_t rows, columns;
};
enum Output { OUT_PLAIN, OUT_PAIR, OUT_STATES };
struct Outputs {
  void* y;
  int64_t ld;
  void const *bias, *bias2;
  int act;
  float slope;
  void *g, *u;          // states: written by OUT_PAIR (null: not), read by OUT_STATES
  int64_t ld_states;
  void *dg, *du;        // OUT_STATES
  int64_t ld_gradients;
};

// act(v) and act'(v)
__device__ inline void activation(int act, float slope, float v, float& a, float& d) {
  switch (act) {
    case ACT_RELU: a = act_relu(v), d = v > 0.0f ? 1.0f : 0.0f; break;
    case ACT_LEAKY_RELU: a = act_leaky_relu(v, slope), d = v > 0.0f ? 1.0f : slope; break;
    case ACT_TANH: a = tanh_f32(v), d = 1.0f - a * a; break;
    case ACT_SIGMOID: a = sigmoid_f32(v), d = a * sigmoid_f32(-v); break;
    case ACT_SILU: {
      float const p = sigmoid_f32(v);
      a = silu_f32(v), d = p * fmaf(v, sigmoid_f32(-v), 1.0f);
      break;
    }
    case ACT_GELU_TANH: {
      constexpr float c = 0.79788456080286535588f;
      float const p = sigmoid_f32(2.0f * c * v * fmaf(0.044715f * v, v, 1.0f));
      a = gelu_tanh_f32(v);
      d = p * fmaf(2.0f * c * v * fmaf(3.0f * 0.044715f * v, v, 1.0f), 1.0f - p, 1.0f);
      break;
    }
    default: {
      float const p = 0.5f * erfcf(-0.70710678118654752440f * v);
      a = act_gelu_erf(v), d = fmaf(v * 0.39894228040143267794f, exp_f32(-0.5f * v * v), p);
    }
  }
}

template <class T, Output OUT> __global__ __launch_bounds__(256) void product(Product p, Outputs o) {
  constexpr bool PAIR = OUT == OUT_PAIR;
  __shared__ float as[PAIR ? 2 : 1][kDepth][kTile + 4], bs[kDepth][kTile + 4];
  int64_t const m0 = int64_t(blockIdx.y) * kTile, n0 = int64_t(blockIdx.x) * kTile;
  int const ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[PAIR ? 2 : 1][4][4] = {};
  for (int term = 0; term < p.terms; term++) {
    for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
      auto stage = [&](Operand const& from, int64_t first, int64_t end, float (&to)[kDepth][kTile + 4]) {
        for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
          // (neighbouring lanes along the contiguous dimension)
          int const i = from.row == 1 ? e % kTile : e / kDepth, k = from.row == 1 ? e / kTile : e % kDepth;
          bool const in = first + i < end && k0 + k < p.k;
          to[k][i] = in ? float(static_cast<T const*>(from.p)[(first + i) * from.row + (k0 + k) * from.step]) : 0.0f;
        }
      };
      stage(p.a[term], m0, p.rows, as[0]);
      if constexpr (PAIR) stage(p.a2, m0, p.rows, as[1]);
      stage(p.b[term], n0, p.columns, bs);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kDepth; k++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            acc[0][i][j] = fmaf(as[0][k][ty * 4 + i], bs[k][tx * 4 + j], acc[0][i][j]);
            if constexpr (PAIR) acc[1][i][j] = fmaf(as[1][k][ty * 4 + i], bs[k][tx * 4 + j], acc[1][i][j]);
          }
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      int64_t const m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.rows || n >= p.columns) continue;
      float v = acc[0][i][j], a, d;
      if constexpr (OUT != OUT_STATES)
        if (o.bias != nullptr) v += float(static_cast<T const*>(o.bias)[m]);
      if constexpr (OUT == OUT_PAIR) {
        float u = acc[1][i][j];
        if (o.bias2 != nullptr) u += float(static_cast<T const*>(o.bias2)[m]);
        activation(o.act, o.slope, v, a, d);
        if (o.g != nullptr) {
          static_cast<T*>(o.g)[m * o.ld_states + n] = T(v);
          static_cast<T*>(o.u)[m * o.ld_states + n] = T(u);
        }
        v = a * u;
      }
      if constexpr (OUT == OUT_STATES) {
        activation(o.act, o.slope, float(static_cast<T const*>(o.g)[m * o.ld_states + n]), a, d);
        static_cast<T*>(o.dg)[m * o.ld_gradients + n] = T(v * float(static_cast<T const*>(o.u)[m * o.ld_states + n]) * d);
        static_cast<T*>(o.du)[m * o.ld_gradients + n] = T(v * a);
      } else {
        static_cast<T*>(o.y)[m * o.ld + n] = T(v);
      }
    }
}

// y[row] = the sum of a row.
template <class T> __global__ __launch_bounds__(256) void row_sums(T const* x, int64_t ld, int64_t columns, T* y) {
  __shared__ float lds[4];
  T const* row = x + int64_t(blockIdx.x) * ld;
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < columns; c += 256) s += float(row[c]);
  for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) y[blockIdx.x] = T((lds[0] + lds[1]) + (lds[2] + lds[3]));
}

template <class T, Output OUT> hipError_t launch_product(Product const& p, Outputs const& o, hipStream_t stream) {
  int64_t const x = (p.columns + kTile - 1) / kTile, y = (p.rows + kTile - 1) / kTile;
  if (x > int64_t(UINT32_MAX) / 256 / y || y > 65535) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((product<T, OUT>), dim3(unsigned(x), unsigned(y)), dim3(256), 0, stream, p, o);
  return hipGetLastError();
}

int64_t padded(int64_t columns) { return (columns + 63) / 64 * 64; }
int64_t element(ponni_gated const& b) { return b.dtype == PONNI_F32 ? 4 : 2; }

}  // namespace

int64_t gated_workspace_bytes(ponni_gated const& b, int64_t columns, bool backward) {
  return padded(columns) * b.n_hidden * element(b) * (backward ? 2 : 1);
}

hipError_t launch_gated(ponni_gated const& b, int act, void const* x, int64_t ld_x, void* y, int64_t ld_y, void* states,
                        int64_t ld_states, int64_t columns, void* workspace, hipStream_t stream) {
  hipError_t err = hipSuccess;
  with_dtype(b.dtype, [&](auto e) {
    using T = decltype(e);
    T* const s = static_cast<T*>(states);
    int64_t const ld_h = s != nullptr ? ld_states : padded(columns);
    T* const h = s != nullptr ? s + 2 * b.n_hidden * ld_states : static_cast<T*>(workspace);
    Outputs o{};
    o.y = h, o.ld = ld_h, o.bias = b.gate_bias, o.bias2 = b.up_bias, o.act = act, o.slope = float(b.act.attr[0]);
    if (s != nullptr) o.g = s, o.u = s + b.n_hidden * ld_states, o.ld_states = ld_states;
    err = launch_product<T, OUT_PAIR>({{{b.gate, 1, b.ld_gate}}, {{x, 1, ld_x}}, {b.up, 1, b.ld_up}, b.n_in, 1, b.n_hidden,
                                       columns}, o, stream);
    if (err != hipSuccess) return;
    Outputs last{};
    last.y = y, last.ld = ld_y, last.bias = b.down_bias;
    err = launch_product<T, OUT_PLAIN>({{{b.down, 1, b.ld_down}}, {{h, 1, ld_h}}, {}, b.n_hidden, 1, b.n_out, columns}, last,
                                       stream);
  });
  return err;
}

hipError_t launch_gated_backward(ponni_gated const& b, int act, void const* x, int64_t ld_x, void const* states,
                                 int64_t ld_states, void const* dy, int64_t ld_dy, int64_t columns,
                                 ponni_gated_gradients const& d, void* workspace, hipStream_t stream) {
  hipError_t err = hipSuccess;
  with_dtype(b.dtype, [&](auto e) {
    using T = decltype(e);
    T* const s = static_cast<T*>(const_cast<void*>(states));
    int64_t const ld = padded(columns), hidden = b.n_hidden;
    T *const dg = static_cast<T*>(workspace), *const du = dg + hidden * ld;
    auto run = [&](auto out, Product const& p, Outputs const& o) {
      if (err == hipSuccess) err = launch_product<T, decltype(out)::value>(p, o, stream);
    };
    auto plain = [&](void* y, int64_t ld_y, Product const& p) {
      Outputs o{};
      o.y = y, o.ld = ld_y;
      if (y != nullptr) run(std::integral_constant<Output, OUT_PLAIN>{}, p, o);
    };
    auto sums = [&](void* y, T const* from, int64_t rows, int64_t ld_from) {
      if (y == nullptr || err != hipSuccess) return;
      hipLaunchKernelGGL(row_sums<T>, dim3(unsigned(rows)), dim3(256), 0, stream, from, ld_from, columns, static_cast<T*>(y));
      err = hipGetLastError();
    };
    Outputs o{};
    o.act = act, o.slope = float(b.act.attr[0]), o.g = s, o.u = s + hidden * ld_states, o.ld_states = ld_states;
    o.dg = dg, o.du = du, o.ld_gradients = ld;
    run(std::integral_constant<Output, OUT_STATES>{},
        {{{b.down, b.ld_down, 1}}, {{dy, 1, ld_dy}}, {}, b.n_out, 1, hidden, columns}, o);
    plain(d.x, d.ld_x, {{{b.gate, b.ld_gate, 1}, {b.up, b.ld_up, 1}}, {{dg, 1, ld}, {du, 1, ld}}, {}, hidden, 2, b.n_in, columns});
    plain(d.gate, d.ld_gate, {{{x, ld_x, 1}}, {{dg, ld, 1}}, {}, columns, 1, b.n_in, hidden});
    plain(d.up, d.ld_up, {{{x, ld_x, 1}}, {{du, ld, 1}}, {}, columns, 1, b.n_in, hidden});
    plain(d.down, d.ld_down, {{{s + 2 * hidden * ld_states, ld_states, 1}}, {{dy, ld_dy, 1}}, {}, columns, 1, hidden, b.n_out});
    sums(d.gate_bias, dg, hidden, ld);
    sums(d.up_bias, du, hidden, ld);
    sums(d.down_bias, static_cast<T const*>(dy), b.n_out, ld_dy);
  });
  return err;
}

}  // namespace ponni_hip
