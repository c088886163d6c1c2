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
// Columns of more features than the registers hold (shape_of) are read again for each sum, 128 bytes of a row at a time.
//
// Bound by bytes: what a tile reads waits for its sums, which workgroups of the same CU fill up to where registers end.
// By kernel: bf16, 1024 features x 65,536, rms norms after and before, a gate for each feature: 163 us, 3.3 TB/s; its gradients
// 439 + 15.  fp32, 333 x 40,003 (rows at any 4 bytes), all inputs: 89 us, 3.0 TB/s; gradients 168 + 12.  fp16, 4096 x 16,384 (read
// again): 172 us; gradients 284 + 9.  One column of 4096: 6.2 us.
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
  int64_t first;     // tile of a forward launch
  float* parts;      // [workgroups, NORM_SUMS, n]
};

// One float per feature, `otherwise` where there is no array.
__device__ inline float feature(float const* p, int row, float otherwise) { return p != nullptr ? p[row] : otherwise; }

__device__ inline float swap_add32(float a, float b) {  // lanes 0-31: the sum of a over lanes 32 apart, others: of b
  auto const r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float swap_add16(float a, float b) {  // the same of even and odd rows of 16
  auto const r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The workgroup's sums of NC values per lane over the lanes that share columns.  Within a wave each exchange halves
// the columns that a lane holds (8: 15 instructions, where every lane's sum of each would be 24 exchanges through LDS).
template <int NC> struct Reducer {
  float (*lds)[kWaves][8 * NC];  // [4]: a sum's area is written again four sums later
  int across, tx, next;
  __device__ void sum(float (&v)[NC]) {
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float t;
    int column = 0, d = 32;
    if constexpr (NC == 1) {
      t = v[0];
    } else {
      float h[NC / 2];
#pragma unroll
      for (int j = 0; j < NC / 2; j++) h[j] = swap_add32(v[j], v[j + NC / 2]);
      float q[NC / 4];
#pragma unroll
      for (int j = 0; j < NC / 4; j++) q[j] = swap_add16(h[j], h[j + NC / 4]);
      column = (lane >> 5) * (NC / 2) + (lane >> 4 & 1) * (NC / 4);
      t = q[0];
      d = 8;
      if constexpr (NC == 8) {
        bool const upper = lane & 8;
        float const mine = upper ? q[1] : q[0], other = upper ? q[0] : q[1];
        t = mine + __shfl_xor(other, 8);
        column += lane >> 3 & 1;
        d = 4;
      }
    }
    for (; d >= across; d /= 2) t += __shfl_xor(t, d);
    auto& area = lds[next];
    next = (next + 1) & 3;
    constexpr int SHARED = NC == 8 ? 8 : NC == 4 ? 16 : 64;  // lanes from here on hold other columns
    if ((lane & (SHARED - 1)) < across) area[wave][tx * NC + column] = t;
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

// Workgroup b of n: those of an XCD (they go to the eight in turn) are consecutive, since tiles side by side
// share the lines of their rows.
__device__ inline int64_t by_xcd(int64_t b, int64_t n) {
  int64_t const q = n / 8, rest = n % 8, xcd = b % 8;
  return xcd * q + (xcd < rest ? xcd : rest) + b / 8;
}

// A lane's rows of one array: row ty + i * down at at(i).
template <class T> struct Rows {
  T* p;
  int64_t stride;
  __device__ Rows(void const* base, int64_t ld, int ty, int down, int64_t c0)
      : p(static_cast<T*>(const_cast<void*>(base)) + ty * ld + c0), stride(down * ld) {}
  __device__ T* at(int i) const { return p + i * stride; }
};

// LAYER: one of the norms is a layer norm (else the means are zero).
template <class T, int NC, int STEPS, bool HELD, bool GATE, bool LAYER>
__global__ __launch_bounds__(kThreads, (HELD && STEPS > 4) || GATE ? 2 : 4) void residual_norm(NormArgs a) {
  auto const& r = a.r;
  __shared__ float lds[4][kWaves][8 * NC];
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns, n = r.n;
  Reducer<NC> reduce{lds, across, tx, 0};
  int64_t const c0 = ((a.first + by_xcd(blockIdx.x, gridDim.x)) * across + tx) * NC, left = r.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  float const inv_n = 1.0f / float(n);
  Rows<T> const rows_x(r.x, r.ld_x, ty, down, c0), rows_r(r.residual, r.ld_residual, ty, down, c0),
      rows_g(r.gate, r.ld_gate, ty, down, c0);
  Pack<T, NC> x[STEPS], res[STEPS], gate[GATE ? STEPS : 1];
  auto load = [&](int chunk, bool all) {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      int const i = chunk * STEPS + s;
      res[s].fill(0.0f);
      if (i * down + ty >= n || count == 0) continue;
      x[s].load(rows_x.at(i), count, 0.0f);
      if (all && r.residual != nullptr) res[s].load(rows_r.at(i), count, 0.0f);
      if constexpr (GATE)
        if (all) gate[s].load(rows_g.at(i), count, 0.0f);
    }
  };
  // f(step, row's index) for this lane's rows, whose data is in registers.
  auto each = [&](bool all, auto&& f) {
    for (int chunk = 0; chunk < a.chunks; chunk++) {
      if (!HELD) load(chunk, all);
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int const i = chunk * STEPS + s;
        x[s].pin();
        res[s].pin();
        if (i * down + ty < n && count > 0) f(s, i);
      }
    }
  };
  if (HELD) load(0, true);
  // With one column a lane the features' own are under way with the columns, not behind the sums: bf16, one column of 4096,
  // 8.2 us without.
  constexpr bool EARLY = HELD && NC == 1;
  float early[EARLY ? 5 : 1][EARLY ? STEPS : 1];
  float const* const own[5] = {r.after.weight, r.after.bias, r.feature_gate, r.before.weight, r.before.bias};
  if constexpr (EARLY) {
#pragma unroll
    for (int k = 0; k < 5; k++)
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int const row = s * down + ty;
        early[k][s] = feature(own[k], row < n ? row : 0, k == 1 || k == 4 ? 0.0f : 1.0f);
      }
  }
  // Of row s of the lane's, `row` of all: 0, 1 weight and bias after, 2 gate, 3, 4 weight and bias before.
  auto of_feature = [&](int k, int s, int row) {
    if constexpr (EARLY) return early[k][s];
    else return feature(own[k], row, k == 1 || k == 4 ? 0.0f : 1.0f);
  };
  float m1[LAYER ? NC : 1] = {}, m2[LAYER ? NC : 1] = {}, r1[NC], r2[NC];
  auto mean1 = [&](int j) { return LAYER ? m1[j] : 0.0f; };
  auto mean2 = [&](int j) { return LAYER ? m2[j] : 0.0f; };
#pragma unroll
  for (int j = 0; j < NC; j++) r1[j] = r2[j] = 1.0f;
  if constexpr (LAYER) {
    if (r.after.kind == PONNI_NORM_LAYER) {
      each(false, [&](int s, int) {
#pragma unroll
        for (int j = 0; j < NC; j++) m1[j] += x[s][j];
      });
      reduce.sum(m1);
#pragma unroll
      for (int j = 0; j < NC; j++) m1[j] *= inv_n;
    }
  }
  if (r.after.kind != PONNI_NORM_NONE) {
    float v[NC] = {};
    each(false, [&](int s, int) {
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const d = x[s][j] - mean1(j);
        v[j] = fmaf(d, d, v[j]);
      }
    });
    reduce.sum(v);
#pragma unroll
    for (int j = 0; j < NC; j++) r1[j] = 1.0f / sqrtf(fmaf(v[j], inv_n, r.after.eps));
  }
  auto state = [&](int s, int i, float (&v)[NC]) {
    int const row = i * down + ty;
    float const w = of_feature(0, s, row), b = of_feature(1, s, row), g = r.scale * of_feature(2, s, row);
#pragma unroll
    for (int j = 0; j < NC; j++) {
      float const branch = fmaf((x[s][j] - mean1(j)) * r1[j], w, b);
      if constexpr (GATE) v[j] = fmaf(g * gate[s][j], branch, res[s][j]);
      else v[j] = fmaf(g, branch, res[s][j]);
    }
  };
  if constexpr (LAYER) {
    if (r.before.kind == PONNI_NORM_LAYER) {
      each(true, [&](int s, int i) {
        float v[NC];
        state(s, i, v);
#pragma unroll
        for (int j = 0; j < NC; j++) m2[j] += v[j];
      });
      reduce.sum(m2);
#pragma unroll
      for (int j = 0; j < NC; j++) m2[j] *= inv_n;
    }
  }
  if (r.before.kind != PONNI_NORM_NONE) {
    float q[NC] = {};
    each(true, [&](int s, int i) {
      float v[NC];
      state(s, i, v);
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const d = v[j] - mean2(j);
        q[j] = fmaf(d, d, q[j]);
      }
    });
    reduce.sum(q);
#pragma unroll
    for (int j = 0; j < NC; j++) r2[j] = 1.0f / sqrtf(fmaf(q[j], inv_n, r.before.eps));
  }
  Rows<T> const rows_s(r.state, r.ld_state, ty, down, c0), rows_n(r.normed, r.ld_normed, ty, down, c0);
  each(true, [&](int s, int i) {
    float v[NC];
    state(s, i, v);
    Pack<T, NC> o;
    if (r.state != nullptr) {
#pragma unroll
      for (int j = 0; j < NC; j++) o.set(j, v[j]);
      o.store(rows_s.at(i), count);
    }
    if (r.normed != nullptr) {
      int const row = i * down + ty;
      float const w = of_feature(3, s, row), b = of_feature(4, s, row);
#pragma unroll
      for (int j = 0; j < NC; j++) o.set(j, fmaf((v[j] - mean2(j)) * r2[j], w, b));
      o.store(rows_n.at(i), count);
    }
  });
  if (r.statistics != nullptr && ty == 0)
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < count) {
        float* at = r.statistics + c0 + j;
        at[0] = mean1(j), at[r.columns] = r1[j], at[2 * r.columns] = mean2(j), at[3 * r.columns] = r2[j];
      }
}

// AFTER: there is a norm after the block.
template <class T, int NC, int STEPS, bool HELD, bool GATE, bool LAYER, bool AFTER>
__global__ __launch_bounds__(kThreads) void residual_norm_backward(NormArgs a) {
  auto const& r = a.r;
  auto const& g = a.g;
  __shared__ float lds[4][kWaves][8 * NC];
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns, n = r.n;
  Reducer<NC> reduce{lds, across, tx, 0};
  float const inv_n = 1.0f / float(n);
  bool const before = r.before.kind != PONNI_NORM_NONE && g.d_normed != nullptr;
  constexpr int FIRST = AFTER ? 0 : NORM_SUM_GATE;  // of the sums
  float sums[STEPS][NORM_SUMS] = {};
  // This workgroup's sums of a chunk's rows, from FROM to TO.
  auto flush = [&](int chunk, int from, int to, bool first) {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      int const row = (chunk * STEPS + s) * down + ty;
#pragma unroll
      for (int q = FIRST; q < NORM_SUMS; q++) {
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
  int64_t const begin = by_xcd(blockIdx.x, gridDim.x);
  for (int64_t tile = begin; tile < a.tiles; tile += gridDim.x) {
    bool const first = tile == begin;
    int64_t const c0 = (tile * across + tx) * NC, left = r.columns - c0;
    int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
    Rows<T> const rows_x(r.x, r.ld_x, ty, down, c0), rows_r(r.residual, r.ld_residual, ty, down, c0),
        rows_g(r.gate, r.ld_gate, ty, down, c0), rows_n(g.d_normed, g.ld_d_normed, ty, down, c0),
        rows_s(g.d_state, g.ld_d_state, ty, down, c0);
    Pack<T, NC> x[STEPS], res[STEPS], dn[STEPS], gate[GATE ? STEPS : 1];
    auto load = [&](int chunk) {
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        int const i = chunk * STEPS + s;
        dn[s].fill(0.0f);
        res[s].fill(0.0f);
        x[s].fill(0.0f);
        if (i * down + ty >= n || count == 0) continue;
        x[s].load(rows_x.at(i), count, 0.0f);
        if (before) {
          dn[s].load(rows_n.at(i), count, 0.0f);
          if (r.residual != nullptr) res[s].load(rows_r.at(i), count, 0.0f);
        }
        if constexpr (GATE) gate[s].load(rows_g.at(i), count, 0.0f);
      }
    };
    // f(step, row's index, row) for this lane's rows, whose data is in registers; done(chunk) behind each chunk.
    auto each = [&](auto&& f, auto&& done) {
      for (int chunk = 0; chunk < a.chunks; chunk++) {
        if (!HELD) load(chunk);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          int const i = chunk * STEPS + s;
          x[s].pin();
          res[s].pin();
          dn[s].pin();
          if (i * down + ty < n && count > 0) f(s, i, i * down + ty);
        }
        if (!HELD) done(chunk);
      }
    };
    constexpr int MEANS = LAYER ? NC : 1, FIRSTS = AFTER ? NC : 1;
    float m1[LAYER && AFTER ? NC : 1] = {}, m2[MEANS] = {}, r1[FIRSTS], r2[NC];
#pragma unroll
    for (int j = 0; j < NC; j++) {
      bool const in = j < count;
      if constexpr (LAYER && AFTER) m1[j] = in ? r.statistics[c0 + j] : 0.0f;
      if constexpr (AFTER) r1[j] = in ? r.statistics[r.columns + c0 + j] : 0.0f;
      if constexpr (LAYER) m2[j] = in ? r.statistics[2 * r.columns + c0 + j] : 0.0f;
      r2[j] = in ? r.statistics[3 * r.columns + c0 + j] : 0.0f;
    }
    if (HELD) load(0);
    auto unit = [&](int s, int j) {
      if constexpr (AFTER) return (x[s][j] - (LAYER ? m1[j] : 0.0f)) * r1[j];
      else return x[s][j];
    };
    auto factor = [&](int s, int j, float f) {
      if constexpr (GATE) return f * gate[s][j];
      else return f;
    };
    // What a row multiplies with.
    struct Feature {
      float w1, b1, w2, f;
    };
    auto feature_of = [&](int row) {
      return Feature{AFTER ? feature(r.after.weight, row, 1.0f) : 1.0f, AFTER ? feature(r.after.bias, row, 0.0f) : 0.0f,
                     feature(r.before.weight, row, 1.0f), r.scale * feature(r.feature_gate, row, 1.0f)};
    };
    auto branch = [&](int s, int j, Feature const& w) { return AFTER ? fmaf(unit(s, j), w.w1, w.b1) : x[s][j]; };
    auto unit2 = [&](int s, int j, Feature const& w, float v) {
      return (fmaf(factor(s, j, w.f), v, res[s][j]) - (LAYER ? m2[j] : 0.0f)) * r2[j];
    };
    float e2[MEANS] = {}, eu2[NC] = {};
    if (before) {
      each(
          [&](int s, int, int row) {
            Feature const w = feature_of(row);
#pragma unroll
            for (int j = 0; j < NC; j++) {
              float const u = unit2(s, j, w, branch(s, j, w)), d = dn[s][j], e = d * w.w2;
              if constexpr (LAYER) e2[j] += e;
              eu2[j] = fmaf(e, u, eu2[j]);
              sums[s][NORM_SUM_W2] = fmaf(d, u, sums[s][NORM_SUM_W2]);
              sums[s][NORM_SUM_B2] += d;
            }
          },
          [&](int chunk) { flush(chunk, NORM_SUM_W2, NORM_SUMS, first); });
      if constexpr (LAYER) {
        if (r.before.kind == PONNI_NORM_LAYER) reduce.sum(e2);
#pragma unroll
        for (int j = 0; j < NC; j++) e2[j] = r.before.kind == PONNI_NORM_LAYER ? e2[j] * inv_n : 0.0f;
      }
      reduce.sum(eu2);
#pragma unroll
      for (int j = 0; j < NC; j++) eu2[j] *= inv_n;
    } else if (!HELD) {
      for (int chunk = 0; chunk < a.chunks; chunk++) flush(chunk, NORM_SUM_W2, NORM_SUMS, first);
    }
    // D of an element from v.
    auto gradient = [&](int s, int j, Feature const& w, float ds, float v) {
      if (!before) return ds;
      return fmaf(r2[j], fmaf(dn[s][j], w.w2, LAYER ? -e2[j] : 0.0f) - unit2(s, j, w, v) * eu2[j], ds);
    };
    auto load_state = [&](int i) {
      Pack<T, NC> ds;
      ds.fill(0.0f);
      if (g.d_state != nullptr) ds.load(rows_s.at(i), count, 0.0f);
      return ds;
    };
    Rows<T> const out_r(g.d_residual, g.ld_d_residual, ty, down, c0), out_g(g.d_gate, g.ld_d_gate, ty, down, c0),
        out_x(g.d_x, g.ld_d_x, ty, down, c0);
    float e1[LAYER && AFTER ? NC : 1] = {}, eu1[FIRSTS] = {};
    each(
        [&](int s, int i, int row) {
          Feature const w = feature_of(row);
          Pack<T, NC> const ds = load_state(i);
          Pack<T, NC> o, og, ox;
#pragma unroll
          for (int j = 0; j < NC; j++) {
            float const v = branch(s, j, w), d = gradient(s, j, w, ds[j], v), dv = factor(s, j, w.f) * d;
            o.set(j, d);
            if constexpr (GATE) og.set(j, r.scale * d * v);
            else sums[s][NORM_SUM_GATE] = fmaf(r.scale * d, v, sums[s][NORM_SUM_GATE]);
            if constexpr (AFTER) {
              float const u = unit(s, j), e = dv * w.w1;
              if constexpr (LAYER) e1[j] += e;
              eu1[j] = fmaf(e, u, eu1[j]);
              sums[s][NORM_SUM_W1] = fmaf(dv, u, sums[s][NORM_SUM_W1]);
              sums[s][NORM_SUM_B1] += dv;
            } else {
              ox.set(j, dv);
            }
          }
          if (g.d_residual != nullptr) o.store(out_r.at(i), count);
          if constexpr (GATE)
            if (g.d_gate != nullptr) og.store(out_g.at(i), count);
          if constexpr (!AFTER)
            if (g.d_x != nullptr) ox.store(out_x.at(i), count);
        },
        [&](int chunk) { flush(chunk, FIRST, NORM_SUM_W2, first); });
    if constexpr (AFTER) {
      if (g.d_x == nullptr) continue;
      if constexpr (LAYER) {
        if (r.after.kind == PONNI_NORM_LAYER) reduce.sum(e1);
#pragma unroll
        for (int j = 0; j < NC; j++) e1[j] = r.after.kind == PONNI_NORM_LAYER ? e1[j] * inv_n : 0.0f;
      }
      reduce.sum(eu1);
#pragma unroll
      for (int j = 0; j < NC; j++) eu1[j] *= inv_n;
      each(
          [&](int s, int i, int row) {
            Feature const w = feature_of(row);
            Pack<T, NC> const ds = load_state(i);
            Pack<T, NC> o;
#pragma unroll
            for (int j = 0; j < NC; j++) {
              float const v = branch(s, j, w), d = gradient(s, j, w, ds[j], v);
              o.set(j, r1[j] * (fmaf(factor(s, j, w.f) * d, w.w1, LAYER ? -e1[j] : 0.0f) - unit(s, j) * eu1[j]));
            }
            o.store(out_x.at(i), count);
          },
          [](int) {});
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

inline Shape shape_of(int32_t n, int64_t columns, int32_t dtype, int max_steps, int narrowest) {
  int const wide = dtype == PONNI_F32 ? 4 : 8;
  Shape s{};
  s.columns = columns < wide ? 1 : wide;
  int64_t const lanes = (columns + s.columns - 1) / s.columns;
  while (s.lane_columns < 3 && (1 << s.lane_columns) < lanes) s.lane_columns++;
  auto steps_at = [&](int l) { return (n + (kThreads >> l) - 1) / (kThreads >> l); };
  auto tiles_at = [&](int l) { return (lanes + (1 << l) - 1) >> l; };
  while (s.lane_columns > 0 && tiles_at(s.lane_columns) < 256) s.lane_columns--;
  // In registers at 128 bytes of a row or down to `narrowest` (3: 128, 1: 32): the kernel that reads whole lines again reads
  // more, narrower pieces come slower.  us (calls one after the other) in registers / read again, 67 M elements: forward bf16, rms norms, n = 1024
  // (128 bytes) 151 / 170, 2048 (64) 162 / 179, 4096 (32) 285 / 191, with a gate layer norms 2048 (32) 274 / 322;
  // backward fp32 rms norms 1024 (64) 561 / 833, 2048 (32) 771 / 865, a norm before alone 1024 (64) 552 / 542, 2048 (32)
  // 673 / 589; backward bf16 rms norms 2048 (32) 498 / 413, layer norms 700 (64) 588 / 453, a norm before alone 4096 (16
  // bytes) 418 / 230.
  if (steps_at(s.lane_columns) > max_steps && (s.lane_columns < 3 || steps_at(narrowest) <= max_steps))
    while (s.lane_columns > 0 && steps_at(s.lane_columns) > max_steps) s.lane_columns--;
  int const steps = steps_at(s.lane_columns);
  s.tiles = tiles_at(s.lane_columns);
  s.steps = steps <= 4 ? 4 : steps <= 8 ? 8 : 16;
  s.chunks = (steps + s.steps - 1) / s.steps;
  if (steps > max_steps) {
    s.steps = 4;
    s.chunks = (steps + 3) / 4;  // (read again)
  }
  return s;
}

inline bool has_layer(ponni_residual_norm const& r) {
  return r.after.kind == PONNI_NORM_LAYER || r.before.kind == PONNI_NORM_LAYER;
}

// Rows that a lane holds at most.  A few spilled registers cost less than to read again (backward, fp32 rms norms, n = 512
// 455 / 811 us), but not those of two layer norms of 16 bits (bf16, n = 512: 525 / 461).
inline int most_steps(ponni_residual_norm const& r, bool backward) {
  bool const gate = r.gate != nullptr, half = r.dtype != PONNI_F32;
  if (!backward) return gate ? 8 : 16;
  return half && (gate || (has_layer(r) && r.after.kind != PONNI_NORM_NONE)) ? 4 : 8;
}
// log2 of the lanes across, at least.
inline int narrowest(ponni_residual_norm const& r, bool backward) {
  if (!backward) return r.gate != nullptr ? 1 : 2;
  return r.dtype != PONNI_F32 ? 3 : r.after.kind != PONNI_NORM_NONE ? 1 : 2;
}

// f(steps, held, gate, layer) as constants.
template <class F> void with_variant(Shape const& s, bool gate, bool layer, F&& f) {
  auto pick = [&](auto g, auto l) {
    if (s.chunks > 1) f(std::integral_constant<int, 4>{}, std::false_type{}, g, l);
    else if (s.steps == 4) f(std::integral_constant<int, 4>{}, std::true_type{}, g, l);
    else if (s.steps == 8) f(std::integral_constant<int, 8>{}, std::true_type{}, g, l);
    else f(std::integral_constant<int, 16>{}, std::true_type{}, g, l);
  };
  if (gate && layer) pick(std::true_type{}, std::true_type{});
  else if (gate) pick(std::true_type{}, std::false_type{});
  else if (layer) pick(std::false_type{}, std::true_type{});
  else pick(std::false_type{}, std::false_type{});
}

template <class T> hipError_t launch_norm(ponni_residual_norm const& r, hipStream_t stream) {
  Shape const s = shape_of(r.n, r.columns, r.dtype, most_steps(r, false), narrowest(r, false));
  NormArgs a{};
  a.r = r;
  a.lane_columns = s.lane_columns;
  a.chunks = s.chunks;
  a.tiles = s.tiles;
  constexpr int64_t kMost = int64_t(UINT32_MAX) / kThreads;  // workgroups of a launch
  for (; a.first < s.tiles; a.first += kMost) {
    dim3 const grid(static_cast<unsigned>(std::min(s.tiles - a.first, kMost)));
    with_variant(s, r.gate != nullptr, has_layer(r), [&](auto steps, auto held, auto gate, auto layer) {
      constexpr int S = decltype(steps)::value, NC = 16 / sizeof(T);
      constexpr bool H = decltype(held)::value, G = decltype(gate)::value, L = decltype(layer)::value;
      if constexpr (!(G && S == 16)) {  // (most_steps)
        if (s.columns == 1) hipLaunchKernelGGL((residual_norm<T, 1, S, H, G, true>), grid, dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((residual_norm<T, NC, S, H, G, L>), grid, dim3(kThreads), 0, stream, a);
      }
    });
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <class T>
hipError_t launch_norm_backward(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g, void* workspace,
                                int& groups, hipStream_t stream) {
  Shape const s = shape_of(r.n, r.columns, r.dtype, most_steps(r, true), narrowest(r, true));
  NormArgs a{};
  a.r = r;
  a.g = g;
  a.lane_columns = s.lane_columns;
  a.chunks = s.chunks;
  a.tiles = s.tiles;
  a.parts = static_cast<float*>(workspace);
  groups = static_cast<int>(std::min<int64_t>(s.tiles, kNormWorkgroups));
  with_variant(s, r.gate != nullptr, has_layer(r), [&](auto steps, auto held, auto gate, auto layer) {
    constexpr int S = decltype(steps)::value, NC = 16 / sizeof(T);
    constexpr bool H = decltype(held)::value, G = decltype(gate)::value, L = decltype(layer)::value;
    dim3 const grid(groups), block(kThreads);
    if constexpr (!(G && S == 8 && sizeof(T) == 2) && S < 16) {  // (most_steps)
      if (r.after.kind == PONNI_NORM_NONE) {
        if (s.columns == 1) hipLaunchKernelGGL((residual_norm_backward<T, 1, S, H, G, true, false>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((residual_norm_backward<T, NC, S, H, G, L, false>), grid, block, 0, stream, a);
      } else {
        if (s.columns == 1) hipLaunchKernelGGL((residual_norm_backward<T, 1, S, H, G, true, true>), grid, block, 0, stream, a);
        else if constexpr (!(L && H && S == 8 && sizeof(T) == 2))
          hipLaunchKernelGGL((residual_norm_backward<T, NC, S, H, G, L, true>), grid, block, 0, stream, a);
      }
    }
  });
  return hipGetLastError();
}

}  // namespace
}  // namespace ponni_hip
