// What stands between two blocks: state = residual + scale * gate * after(x) and
// normed = before(state) over columns of n features, and the gradients
// (kernels_norm_f32.hip, kernels_norm_f16.hip, kernels_norm_bf16.hip).
//
// A workgroup holds a tile of columns, all features of them, in registers: a lane 16
// bytes of a row (NC columns) and every R-th row, so that each array goes through
// memory once.  Means and mean squares of deviations are sums over a lane's rows,
// then over the lanes and waves that share a column.  With m1, r1 (m2, r2) the mean and 1 / sqrt of the norm
// after (before), v = (x - m1) r1 w1 + b1:
//   state = residual + scale gate v,  normed = (state - m2) r2 w2 + b2;
//   e2 = d_normed w2,  u2 = (state - m2) r2,
//   D = d_state + r2 (e2 - mean(e2) - u2 mean(e2 u2))        (mean(e2) of a layer norm only)
//   d_residual = D,  d_gate = scale D v,  e1 = scale gate D w1,  u1 = (x - m1) r1,
//   d_x = r1 (e1 - mean(e1) - u1 mean(e1 u1));
// weights' gradients are sums over columns: a workgroup adds those of its tiles in
// registers, a second kernel the workgroups' in their order.
// Columns of more features than the registers hold are read again for each sum.
#pragma once

#include <algorithm>
#include <type_traits>

#include "blocks.h"
#include "column_rows.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;

struct NormArgs {
  ponni_residual_norm r;
  ponni_residual_norm_gradients g;
  int lane_columns;  // log2 of the lanes across a tile's columns
  int chunks;        // of STEPS * (threads down) rows; 1 where a lane holds all of its rows
  int64_t tiles;
  float* parts;      // [workgroups, NORM_SUMS, n]
};

// One float per feature, `otherwise` where there is no array.
__device__ inline float feature(float const* p, int row, float otherwise) { return p != nullptr ? p[row] : otherwise; }

// The workgroup's sums of NC values per lane over the lanes that share columns.
template <int NC> struct Reducer {
  float (*lds)[kWaves][8 * NC];  // [4]: a sum's area is written again four sums later
  int across, tx, next;
  __device__ void sum(float (&v)[NC]) {
    for (int d = across; d < 64; d *= 2)
#pragma unroll
      for (int j = 0; j < NC; j++) v[j] += __shfl_xor(v[j], d);
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto& area = lds[next];
    next = (next + 1) & 3;
    if (lane < across)
#pragma unroll
      for (int j = 0; j < NC; j++) area[wave][tx * NC + j] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NC; j++) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) s += area[w][tx * NC + j];
      v[j] = s;
    }
  }
};

template <class T, int NC, int STEPS, bool HELD, bool GATE>
__global__ __launch_bounds__(kThreads) void residual_norm(NormArgs a) {
  auto const& r = a.r;
  __shared__ float lds[4][kWaves][8 * NC];
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns, n = r.n;
  Reducer<NC> reduce{lds, across, tx, 0};
  int64_t const c0 = (int64_t(blockIdx.x) * across + tx) * NC, left = r.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  float const inv_n = 1.0f / float(n);
  Pack<T, NC> x[STEPS], res[STEPS], gate[GATE ? STEPS : 1];
  auto load = [&](int chunk, bool all) {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      int64_t const row = (chunk * STEPS + s) * down + ty;
      res[s].fill(0.0f);
      if (row >= n || count == 0) continue;
      x[s].load(static_cast<T const*>(r.x) + row * r.ld_x + c0, count, 0.0f);
      if (all && r.residual != nullptr)
        res[s].load(static_cast<T const*>(r.residual) + row * r.ld_residual + c0, count, 0.0f);
      if constexpr (GATE)
        if (all) gate[s].load(static_cast<T const*>(r.gate) + row * r.ld_gate + c0, count, 0.0f);
    }
  };
  // f(step, row) for this lane's rows, whose data is in registers.
  auto each = [&](bool all, auto&& f) {
    for (int chunk = 0; chunk < a.chunks; chunk++) {
      if (!HELD) load(chunk, all);
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int const row = (chunk * STEPS + s) * down + ty;
        x[s].pin();
        res[s].pin();
        if (row < n && count > 0) f(s, row);
      }
    }
  };
  if (HELD) load(0, true);
  float m1[NC], r1[NC], m2[NC], r2[NC];
#pragma unroll
  for (int j = 0; j < NC; j++) m1[j] = m2[j] = 0.0f, r1[j] = r2[j] = 1.0f;
  if (r.after.kind == PONNI_NORM_LAYER) {
    each(false, [&](int s, int) {
#pragma unroll
      for (int j = 0; j < NC; j++) m1[j] += x[s][j];
    });
    reduce.sum(m1);
#pragma unroll
    for (int j = 0; j < NC; j++) m1[j] *= inv_n;
  }
  if (r.after.kind != PONNI_NORM_NONE) {
    float v[NC] = {};
    each(false, [&](int s, int) {
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const d = x[s][j] - m1[j];
        v[j] = fmaf(d, d, v[j]);
      }
    });
    reduce.sum(v);
#pragma unroll
    for (int j = 0; j < NC; j++) r1[j] = 1.0f / sqrtf(fmaf(v[j], inv_n, r.after.eps));
  }
  auto state = [&](int s, int row, float (&v)[NC]) {
    float const w = feature(r.after.weight, row, 1.0f), b = feature(r.after.bias, row, 0.0f);
    float const g = r.scale * feature(r.feature_gate, row, 1.0f);
#pragma unroll
    for (int j = 0; j < NC; j++) {
      float const branch = fmaf((x[s][j] - m1[j]) * r1[j], w, b);
      if constexpr (GATE) v[j] = fmaf(g * gate[s][j], branch, res[s][j]);
      else v[j] = fmaf(g, branch, res[s][j]);
    }
  };
  if (r.before.kind == PONNI_NORM_LAYER) {
    each(true, [&](int s, int row) {
      float v[NC];
      state(s, row, v);
#pragma unroll
      for (int j = 0; j < NC; j++) m2[j] += v[j];
    });
    reduce.sum(m2);
#pragma unroll
    for (int j = 0; j < NC; j++) m2[j] *= inv_n;
  }
  if (r.before.kind != PONNI_NORM_NONE) {
    float q[NC] = {};
    each(true, [&](int s, int row) {
      float v[NC];
      state(s, row, v);
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const d = v[j] - m2[j];
        q[j] = fmaf(d, d, q[j]);
      }
    });
    reduce.sum(q);
#pragma unroll
    for (int j = 0; j < NC; j++) r2[j] = 1.0f / sqrtf(fmaf(q[j], inv_n, r.before.eps));
  }
  each(true, [&](int s, int row) {
    float v[NC];
    state(s, row, v);
    Pack<T, NC> o;
    if (r.state != nullptr) {
#pragma unroll
      for (int j = 0; j < NC; j++) o.set(j, v[j]);
      o.store(static_cast<T*>(r.state) + row * r.ld_state + c0, count);
    }
    if (r.normed != nullptr) {
      float const w = feature(r.before.weight, row, 1.0f), b = feature(r.before.bias, row, 0.0f);
#pragma unroll
      for (int j = 0; j < NC; j++) o.set(j, fmaf((v[j] - m2[j]) * r2[j], w, b));
      o.store(static_cast<T*>(r.normed) + row * r.ld_normed + c0, count);
    }
  });
  if (r.statistics != nullptr && ty == 0)
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < count) {
        float* at = r.statistics + c0 + j;
        at[0] = m1[j], at[r.columns] = r1[j], at[2 * r.columns] = m2[j], at[3 * r.columns] = r2[j];
      }
}

template <class T, int NC, int STEPS, bool HELD, bool GATE>
__global__ __launch_bounds__(kThreads) void residual_norm_backward(NormArgs a) {
  auto const& r = a.r;
  auto const& g = a.g;
  __shared__ float lds[4][kWaves][8 * NC];
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns, n = r.n;
  Reducer<NC> reduce{lds, across, tx, 0};
  float const inv_n = 1.0f / float(n);
  bool const after = r.after.kind != PONNI_NORM_NONE, before = r.before.kind != PONNI_NORM_NONE && g.d_normed != nullptr;
  float sums[STEPS][NORM_SUMS] = {};
  // This workgroup's sums of a chunk's rows, from FROM to TO.
  auto flush = [&](int chunk, int from, int to, bool first) {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      int const row = (chunk * STEPS + s) * down + ty;
#pragma unroll
      for (int q = 0; q < NORM_SUMS; q++) {
        if (q < from || q >= to) continue;
        float v = sums[s][q];
        for (int d = 1; d < across; d *= 2) v += __shfl_xor(v, d);
        if (tx == 0 && row < n) {
          float* at = a.parts + (int64_t(blockIdx.x) * NORM_SUMS + q) * n + row;
          *at = first ? v : *at + v;
        }
        sums[s][q] = 0.0f;
      }
    }
  };
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    bool const first = tile == blockIdx.x;
    int64_t const c0 = (tile * across + tx) * NC, left = r.columns - c0;
    int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
    Pack<T, NC> x[STEPS], res[STEPS], dn[STEPS], gate[GATE ? STEPS : 1];
    auto load = [&](int chunk) {
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int64_t const row = (chunk * STEPS + s) * down + ty;
        dn[s].fill(0.0f);
        res[s].fill(0.0f);
        x[s].fill(0.0f);
        if (row >= n || count == 0) continue;
        x[s].load(static_cast<T const*>(r.x) + row * r.ld_x + c0, count, 0.0f);
        if (before) {
          dn[s].load(static_cast<T const*>(g.d_normed) + row * g.ld_d_normed + c0, count, 0.0f);
          if (r.residual != nullptr)
            res[s].load(static_cast<T const*>(r.residual) + row * r.ld_residual + c0, count, 0.0f);
        }
        if constexpr (GATE) gate[s].load(static_cast<T const*>(r.gate) + row * r.ld_gate + c0, count, 0.0f);
      }
    };
    float m1[NC], r1[NC], m2[NC], r2[NC];
#pragma unroll
    for (int j = 0; j < NC; j++) {
      bool const in = j < count;
      m1[j] = in ? r.statistics[c0 + j] : 0.0f;
      r1[j] = in ? r.statistics[r.columns + c0 + j] : 0.0f;
      m2[j] = in ? r.statistics[2 * r.columns + c0 + j] : 0.0f;
      r2[j] = in ? r.statistics[3 * r.columns + c0 + j] : 0.0f;
    }
    if (HELD) load(0);
    auto unit = [&](int s, int j) { return (x[s][j] - m1[j]) * r1[j]; };
    auto factor = [&](int s, int j, float f) {
      if constexpr (GATE) return f * gate[s][j];
      else return f;
    };
    float e2[NC] = {}, eu2[NC] = {};
    if (before) {
      for (int chunk = 0; chunk < a.chunks; chunk++) {
        if (!HELD) load(chunk);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          int const row = (chunk * STEPS + s) * down + ty;
          if (row >= n || count == 0) continue;
          float const w1 = feature(r.after.weight, row, 1.0f), b1 = feature(r.after.bias, row, 0.0f),
                      w2 = feature(r.before.weight, row, 1.0f), f = r.scale * feature(r.feature_gate, row, 1.0f);
#pragma unroll
          for (int j = 0; j < NC; j++) {
            float const st = fmaf(factor(s, j, f), fmaf(unit(s, j), w1, b1), res[s][j]);
            float const u = (st - m2[j]) * r2[j], d = dn[s][j], e = d * w2;
            e2[j] += e;
            eu2[j] = fmaf(e, u, eu2[j]);
            sums[s][NORM_SUM_W2] = fmaf(d, u, sums[s][NORM_SUM_W2]);
            sums[s][NORM_SUM_B2] += d;
          }
        }
        if (!HELD) flush(chunk, NORM_SUM_W2, NORM_SUMS, first);
      }
      if (r.before.kind == PONNI_NORM_LAYER) reduce.sum(e2);
      reduce.sum(eu2);
#pragma unroll
      for (int j = 0; j < NC; j++) {
        e2[j] = r.before.kind == PONNI_NORM_LAYER ? e2[j] * inv_n : 0.0f;
        eu2[j] *= inv_n;
      }
    } else if (!HELD) {
      for (int chunk = 0; chunk < a.chunks; chunk++) flush(chunk, NORM_SUM_W2, NORM_SUMS, first);
    }
    // D of an element, and v
    auto gradient = [&](int s, int j, float w1, float b1, float w2, float f, float ds, float& v) {
      v = fmaf(unit(s, j), w1, b1);
      if (!before) return ds;
      float const u = (fmaf(factor(s, j, f), v, res[s][j]) - m2[j]) * r2[j];
      return fmaf(r2[j], fmaf(dn[s][j], w2, -e2[j]) - u * eu2[j], ds);
    };
    auto load_state = [&](int64_t row) {
      Pack<T, NC> ds;
      ds.fill(0.0f);
      if (g.d_state != nullptr) ds.load(static_cast<T const*>(g.d_state) + row * g.ld_d_state + c0, count, 0.0f);
      return ds;
    };
    float e1[NC] = {}, eu1[NC] = {};
    for (int chunk = 0; chunk < a.chunks; chunk++) {
      if (!HELD) load(chunk);
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int64_t const row = (chunk * STEPS + s) * down + ty;
        x[s].pin();
        res[s].pin();
        dn[s].pin();
        if (row >= n || count == 0) continue;
        float const w1 = feature(r.after.weight, row, 1.0f), b1 = feature(r.after.bias, row, 0.0f),
                    w2 = feature(r.before.weight, row, 1.0f), f = r.scale * feature(r.feature_gate, row, 1.0f);
        Pack<T, NC> const ds = load_state(row);
        Pack<T, NC> o, og, ox;
#pragma unroll
        for (int j = 0; j < NC; j++) {
          float v;
          float const d = gradient(s, j, w1, b1, w2, f, ds[j], v);
          o.set(j, d);
          float const dv = factor(s, j, f) * d, u = unit(s, j), e = dv * w1;
          og.set(j, r.scale * d * v);
          ox.set(j, dv);
          e1[j] += e;
          eu1[j] = fmaf(e, u, eu1[j]);
          sums[s][NORM_SUM_W1] = fmaf(dv, u, sums[s][NORM_SUM_W1]);
          sums[s][NORM_SUM_B1] += dv;
          sums[s][NORM_SUM_GATE] = fmaf(r.scale * d, v, sums[s][NORM_SUM_GATE]);
        }
        if (g.d_residual != nullptr) o.store(static_cast<T*>(g.d_residual) + row * g.ld_d_residual + c0, count);
        if constexpr (GATE)
          if (g.d_gate != nullptr) og.store(static_cast<T*>(g.d_gate) + row * g.ld_d_gate + c0, count);
        if (!after && g.d_x != nullptr) ox.store(static_cast<T*>(g.d_x) + row * g.ld_d_x + c0, count);
      }
      if (!HELD) flush(chunk, NORM_SUM_W1, NORM_SUM_W2, first);
    }
    if (!after || g.d_x == nullptr) continue;
    if (r.after.kind == PONNI_NORM_LAYER) reduce.sum(e1);
    reduce.sum(eu1);
#pragma unroll
    for (int j = 0; j < NC; j++) {
      e1[j] = r.after.kind == PONNI_NORM_LAYER ? e1[j] * inv_n : 0.0f;
      eu1[j] *= inv_n;
    }
    for (int chunk = 0; chunk < a.chunks; chunk++) {
      if (!HELD) load(chunk);
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int64_t const row = (chunk * STEPS + s) * down + ty;
        x[s].pin();
        res[s].pin();
        dn[s].pin();
        if (row >= n || count == 0) continue;
        float const w1 = feature(r.after.weight, row, 1.0f), b1 = feature(r.after.bias, row, 0.0f),
                    w2 = feature(r.before.weight, row, 1.0f), f = r.scale * feature(r.feature_gate, row, 1.0f);
        Pack<T, NC> const ds = load_state(row);
        Pack<T, NC> o;
#pragma unroll
        for (int j = 0; j < NC; j++) {
          float v;
          float const d = gradient(s, j, w1, b1, w2, f, ds[j], v);
          o.set(j, r1[j] * (factor(s, j, f) * d * w1 - e1[j] - unit(s, j) * eu1[j]));
        }
        o.store(static_cast<T*>(g.d_x) + row * g.ld_d_x + c0, count);
      }
    }
  }
  if (HELD) flush(0, 0, NORM_SUMS, true);
}

// -- launches -----------------------------------------------------------------------------

struct Shape {
  int columns;       // of a lane
  int lane_columns;  // log2 of the lanes across
  int steps;         // rows that a lane holds
  int chunks;
  int64_t tiles;
};

inline Shape shape_of(int32_t n, int64_t columns, int32_t dtype, int max_steps) {
  int const wide = dtype == PONNI_F32 ? 4 : 8;
  Shape s{};
  s.columns = columns < wide ? 1 : wide;
  int64_t const lanes = (columns + s.columns - 1) / s.columns;
  while (s.lane_columns < 3 && (1 << s.lane_columns) < lanes) s.lane_columns++;
  auto steps_at = [&](int l) { return (n + (kThreads >> l) - 1) / (kThreads >> l); };
  auto tiles_at = [&](int l) { return (lanes + (1 << l) - 1) >> l; };
  while (s.lane_columns > 0 && (steps_at(s.lane_columns) > max_steps || tiles_at(s.lane_columns) < 256)) s.lane_columns--;
  int const steps = steps_at(s.lane_columns);
  s.tiles = tiles_at(s.lane_columns);
  s.steps = steps <= 4 ? 4 : 8;
  s.chunks = (steps + s.steps - 1) / s.steps;
  if (steps > max_steps) {
    s.steps = 4;
    s.chunks = (steps + 3) / 4;
  }
  return s;
}

// Rows a lane can hold without spilling.
inline int most_steps(bool backward, bool gate) { return backward && gate ? 4 : 8; }

template <class F> void with_steps(Shape const& s, bool gate, F&& f) {
  auto steps = [&](auto g) {
    if (s.chunks > 1) f(std::integral_constant<int, 4>{}, std::false_type{}, g);
    else if (s.steps == 4) f(std::integral_constant<int, 4>{}, std::true_type{}, g);
    else f(std::integral_constant<int, 8>{}, std::true_type{}, g);
  };
  if (gate) steps(std::true_type{});
  else steps(std::false_type{});
}

template <class T> hipError_t launch_norm(ponni_residual_norm const& r, hipStream_t stream) {
  Shape const s = shape_of(r.n, r.columns, r.dtype, most_steps(false, r.gate != nullptr));
  NormArgs a{};
  a.r = r;
  a.lane_columns = s.lane_columns;
  a.chunks = s.chunks;
  a.tiles = s.tiles;
  if (s.tiles > int64_t(UINT32_MAX) / kThreads) return hipErrorInvalidConfiguration;
  dim3 const grid(static_cast<unsigned>(s.tiles));
  with_steps(s, r.gate != nullptr, [&](auto steps, auto held, auto gate) {
    constexpr int S = decltype(steps)::value, NC = 16 / sizeof(T);
    constexpr bool H = decltype(held)::value, G = decltype(gate)::value;
    if (s.columns == 1) hipLaunchKernelGGL((residual_norm<T, 1, S, H, G>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((residual_norm<T, NC, S, H, G>), grid, dim3(kThreads), 0, stream, a);
  });
  return hipGetLastError();
}

template <class T>
hipError_t launch_norm_backward(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g, void* workspace,
                                int& groups, hipStream_t stream) {
  Shape const s = shape_of(r.n, r.columns, r.dtype, most_steps(true, r.gate != nullptr));
  NormArgs a{};
  a.r = r;
  a.g = g;
  a.lane_columns = s.lane_columns;
  a.chunks = s.chunks;
  a.tiles = s.tiles;
  a.parts = static_cast<float*>(workspace);
  groups = static_cast<int>(std::min<int64_t>(s.tiles, kNormWorkgroups));
  with_steps(s, r.gate != nullptr, [&](auto steps, auto held, auto gate) {
    constexpr int S = decltype(steps)::value, NC = 16 / sizeof(T);
    constexpr bool H = decltype(held)::value, G = decltype(gate)::value;
    if constexpr (!(G && S == 8)) {
      if (s.columns == 1) hipLaunchKernelGGL((residual_norm_backward<T, 1, S, H, G>), dim3(groups), dim3(kThreads), 0, stream, a);
      else hipLaunchKernelGGL((residual_norm_backward<T, NC, S, H, G>), dim3(groups), dim3(kThreads), 0, stream, a);
    }
  });
  return hipGetLastError();
}

}  // namespace
}  // namespace ponni_hip
