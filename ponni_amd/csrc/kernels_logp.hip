// Log probabilities, entropies and the largest classes of columns of logits
// x [classes, columns], and their gradient.
//
// One pass over x.  With m the largest x so far and t = (x - m) log2(e) a column keeps
//   z = sum 2^t,  q = sum 2^t t,
// which a larger m' turns into z s, (q + d z) s with d = (m - m') log2(e), s = 2^d, and
//   log_normalizer = m + ln2 log2 z,  entropy = ln2 (log2 z - q / z).
// (x log2(e) by itself, an operation less, has no room for the lowest floats.)
// A lane holds NC consecutive columns (16 bytes of a row) and takes every R-th row;
// lanes, waves and workgroups that share columns join their (m, z, q) in a fixed
// order.  The largest logits are lists in descending order, of equal values by
// class; two lists are joined by a bitonic step.
// Bound by the logits' way from memory; 11 VALU operations an element beside it.
#include <cmath>

#include "activations.h"
#include "blocks.h"
#include "column_rows.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

constexpr int kThreads = 256;
constexpr float kLn2 = 0.693147180559945309f, kInf = __builtin_inff();
constexpr float kFar = -1e30f;  // in the place of -inf, where it is multiplied by zero

struct LogpArgs {
  ponni_log_probs p;
  int lane_columns;       // log2 of the threads across a tile's columns
  int splits;             // workgroups that share a tile's columns
  int64_t rows;           // of one of them
  float* parts;           // [splits, 3, columns]: m, z, q
  float* part_values;     // [splits, K, columns]
  int32_t* part_classes;  // [splits, K, columns]
};

// Sums of one column, and its K largest logits.
template <int K> struct Column {
  float m, z, q;
  float value[K > 0 ? K : 1];
  int32_t index[K > 0 ? K : 1];

  __device__ void clear() {
    m = -kInf;
    z = q = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) value[k] = -kInf, index[k] = INT32_MAX;
  }
  __device__ void move_to(float next) {
    float const d = fmaxf((m - next) * kLog2e, kFar), s = __builtin_amdgcn_exp2f(d);
    q = fmaf(d, z, q) * s;
    z *= s;
    m = next;
  }
  __device__ void join(float m2, float z2, float q2) {
    float const next = fmaxf(m, m2);
    move_to(next);
    float const d = fmaxf((m2 - next) * kLog2e, kFar), s = __builtin_amdgcn_exp2f(d);
    q = fmaf(fmaf(d, z2, q2), s, q);
    z = fmaf(z2, s, z);
  }
  // One more logit, of a higher class than those before.
  __device__ void insert(float v, int32_t i) {
    bool more = false;  // (from its place on, the list moves down)
#pragma unroll
    for (int k = 0; k < K; k++) {
      more = more || v > value[k];
      float const w = value[k];
      int32_t const j = index[k];
      value[k] = more ? v : w;
      index[k] = more ? i : j;
      v = more ? w : v;
      i = more ? j : i;
    }
  }
  static __device__ bool before(float a, int32_t i, float b, int32_t j) { return a > b || (a == b && i < j); }
  // The list joined with another one; other(k, value, index) gives its entries.
  template <class F> __device__ void join_list(F&& other) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      float v;
      int32_t i;
      other(K - 1 - k, v, i);
      bool const mine = before(value[k], index[k], v, i);
      value[k] = mine ? value[k] : v;
      index[k] = mine ? index[k] : i;
    }
#pragma unroll
    for (int d = K / 2; d > 0; d /= 2)
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (k & d) continue;
        bool const order = before(value[k], index[k], value[k + d], index[k + d]);
        float const v = value[k], w = value[k + d];
        int32_t const i = index[k], j = index[k + d];
        value[k] = order ? v : w, value[k + d] = order ? w : v;
        index[k] = order ? i : j, index[k + d] = order ? j : i;
      }
  }
};

template <class T, int K> __device__ void finish(ponni_log_probs const& p, int64_t c, Column<K> const& s) {
  float const lz = __log2f(s.z);
  float const normalizer = fmaf(kLn2, lz, s.m);
  p.log_normalizer[c] = normalizer;
  p.entropy[c] = s.z == 0.0f ? 0.0f : kLn2 * (lz - s.q / s.z);
  if (p.targets != nullptr) {
    int64_t const t = p.targets[c];
    float l = 0.0f;
    if (t >= 0 && t < p.classes) {
      l = static_cast<T const*>(p.logits)[t * p.ld + c];
      if (l != -kInf) l -= normalizer;
    }
    p.log_probs[c] = l;
  }
  if constexpr (K > 0)
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (k >= p.top_k) continue;
      bool const none = s.value[k] == -kInf;
      p.top_classes[k * p.columns + c] = none ? -1 : s.index[k];
      p.top_log_probs[k * p.columns + c] = none ? -kInf : s.value[k] - normalizer;
    }
}

template <class T, int NC, int K> __global__ __launch_bounds__(kThreads) void logp(LogpArgs a) {
  constexpr int U = NC >= 4 ? 4 : 8;  // rows under way
  constexpr int WAVES = kThreads / 64;
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns;
  int const split = blockIdx.x % a.splits;
  int64_t const tile = blockIdx.x / a.splits;
  int64_t const c0 = (tile * across + tx) * NC, left = a.p.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  int64_t const first = split * a.rows, end = first + a.rows < a.p.classes ? first + a.rows : a.p.classes;
  Column<K> s[NC];
#pragma unroll
  for (int j = 0; j < NC; j++) s[j].clear();
  T const* x = static_cast<T const*>(a.p.logits) + c0;
  if (count > 0)
    for (int64_t row = first + ty; row < end; row += int64_t(down) * U) {
      Pack<T, NC> v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (row + u * down < end) v[u].load(x + (row + u * down) * a.p.ld, count, -kInf);
        else v[u].fill(-kInf);
      }
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float top = v[0][j];
#pragma unroll
        for (int u = 1; u < U; u++) top = fmaxf(top, v[u][j]);
        float const m = fmaxf(s[j].m, top);
        s[j].move_to(m);
        float const shift = m == -kInf ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < U; u++) {
          float const t = (v[u][j] - shift) * kLog2e, e = __builtin_amdgcn_exp2f(t);
          s[j].z += e;
          s[j].q = fmaf(e, fmaxf(t, kFar), s[j].q);
        }
        if constexpr (K > 0) {
          if (__any(top > s[j].value[K - 1])) {
#pragma unroll
            for (int u = 0; u < U; u++) s[j].insert(v[u][j], int32_t(row + u * down));
          }
        }
      }
    }
  // Lanes of a wave that share columns, then the waves.
  if (down > 1) {
    for (int d = across; d < 64; d *= 2) {
#pragma unroll
      for (int j = 0; j < NC; j++) {
        s[j].join(__shfl_xor(s[j].m, d), __shfl_xor(s[j].z, d), __shfl_xor(s[j].q, d));
        if constexpr (K > 0) {
          Column<K> o;
#pragma unroll
          for (int k = 0; k < K; k++) o.value[k] = __shfl_xor(s[j].value[k], d), o.index[k] = __shfl_xor(s[j].index[k], d);
          s[j].join_list([&](int k, float& v, int32_t& i) { v = o.value[k], i = o.index[k]; });
        }
      }
    }
    constexpr int WORDS = 3 + 2 * K, COLUMNS = 32 * NC;
    __shared__ float lds[WAVES][WORDS][COLUMNS];
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane < across)
#pragma unroll
      for (int j = 0; j < NC; j++) {
        int const c = tx * NC + j;
        lds[wave][0][c] = s[j].m, lds[wave][1][c] = s[j].z, lds[wave][2][c] = s[j].q;
#pragma unroll
        for (int k = 0; k < K; k++) lds[wave][3 + k][c] = s[j].value[k], lds[wave][3 + K + k][c] = __int_as_float(s[j].index[k]);
      }
    __syncthreads();
    int const c = threadIdx.x;
    int64_t const column = tile * across * NC + c;
    if (c >= across * NC || column >= a.p.columns) return;
    Column<K> r;
    r.clear();
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
      r.join(lds[w][0][c], lds[w][1][c], lds[w][2][c]);
      if constexpr (K > 0)
        r.join_list([&](int k, float& v, int32_t& i) { v = lds[w][3 + k][c], i = __float_as_int(lds[w][3 + K + k][c]); });
    }
    if (a.splits == 1) {
      finish<T, K>(a.p, column, r);
    } else {
      float* part = a.parts + split * 3 * a.p.columns + column;
      part[0] = r.m, part[a.p.columns] = r.z, part[2 * a.p.columns] = r.q;
#pragma unroll
      for (int k = 0; k < K; k++) {
        a.part_values[(split * int64_t(K) + k) * a.p.columns + column] = r.value[k];
        a.part_classes[(split * int64_t(K) + k) * a.p.columns + column] = r.index[k];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < count) finish<T, K>(a.p, c0 + j, s[j]);
  }
}

// The workgroups' parts of a column, by 1 << lane_columns lanes each.
template <class T, int K> __global__ __launch_bounds__(kThreads) void logp_join(LogpArgs a) {
  int const lanes = 1 << a.lane_columns, l = threadIdx.x & (lanes - 1);
  int64_t const column = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> a.lane_columns;
  Column<K> r;
  r.clear();
  if (column < a.p.columns)
    for (int s = l; s < a.splits; s += lanes) {
      float const* part = a.parts + s * 3 * a.p.columns + column;
      r.join(part[0], part[a.p.columns], part[2 * a.p.columns]);
      if constexpr (K > 0)
        r.join_list([&](int k, float& v, int32_t& i) {
          int64_t const at = (s * int64_t(K) + k) * a.p.columns + column;
          v = a.part_values[at], i = a.part_classes[at];
        });
    }
  for (int d = 1; d < lanes; d *= 2) {
    r.join(__shfl_xor(r.m, d), __shfl_xor(r.z, d), __shfl_xor(r.q, d));
    if constexpr (K > 0) {
      Column<K> o;
#pragma unroll
      for (int k = 0; k < K; k++) o.value[k] = __shfl_xor(r.value[k], d), o.index[k] = __shfl_xor(r.index[k], d);
      r.join_list([&](int k, float& v, int32_t& i) { v = o.value[k], i = o.index[k]; });
    }
  }
  if (l == 0 && column < a.p.columns) finish<T, K>(a.p, column, r);
}

struct LogpBackwardArgs {
  ponni_log_probs p;
  float const *d_log_probs, *d_entropy, *d_log_normalizer;
  void* d_logits;
  int64_t ld_d;
  int lane_columns;
  int64_t rows;  // of a workgroup
  int64_t tiles;
};

// p (gz - gl) - gh p (log p + entropy), and gl at the target.
template <class T, int NC> __global__ __launch_bounds__(kThreads) void logp_backward(LogpBackwardArgs a) {
  constexpr int U = NC >= 4 ? 4 : 8;
  constexpr bool EXACT = sizeof(T) == 4;
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns;
  int64_t const tile = blockIdx.x % a.tiles, c0 = (tile * across + tx) * NC, left = a.p.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  if (count == 0) return;
  int64_t const first = blockIdx.x / a.tiles * a.rows, end = first + a.rows < a.p.classes ? first + a.rows : a.p.classes;
  float normalizer[NC], base[NC], entropy_weight[NC], at_target[NC];
  int32_t target[NC];
#pragma unroll
  for (int j = 0; j < NC; j++) {
    int64_t const c = c0 + (j < count ? j : 0);
    float const l = a.p.log_normalizer[c];
    bool const none = l == -kInf;
    normalizer[j] = none ? kInf : l;  // (every p is 0)
    target[j] = a.p.targets != nullptr ? a.p.targets[c] : -1;
    bool const given = !none && target[j] >= 0 && int64_t(target[j]) < a.p.classes && a.d_log_probs != nullptr;
    at_target[j] = given ? a.d_log_probs[c] : 0.0f;
    entropy_weight[j] = a.d_entropy != nullptr ? a.d_entropy[c] : 0.0f;
    base[j] = (a.d_log_normalizer != nullptr ? a.d_log_normalizer[c] : 0.0f) - at_target[j];
    if (a.d_entropy != nullptr) base[j] -= entropy_weight[j] * a.p.entropy[c];
    if (!given) target[j] = -1;
  }
  T const* x = static_cast<T const*>(a.p.logits) + c0;
  T* d = static_cast<T*>(a.d_logits) + c0;
  for (int64_t row = first + ty; row < end; row += int64_t(down) * U) {
    Pack<T, NC> v[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (row + u * down < end) v[u].load(x + (row + u * down) * a.p.ld, count, 0.0f);
#pragma unroll
    for (int u = 0; u < U; u++) {
      int64_t const r = row + u * down;
      if (r >= end) continue;
      Pack<T, NC> o;
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const lp = v[u][j] - normalizer[j], p = EXACT ? exp_f32(lp) : __builtin_amdgcn_exp2f(lp * kLog2e);
        // (below -200 p is 0, and 0 times an infinity is not)
        float const g = p * (base[j] - entropy_weight[j] * (lp < -200.0f ? -200.0f : lp));
        o.set(j, int32_t(r) == target[j] ? g + at_target[j] : g);
      }
      o.store(d + r * a.ld_d, count);
    }
  }
}

// -- launches -----------------------------------------------------------------------------

constexpr int64_t kMostGroups = 1024, kMostParts = kMostGroups * 64;
struct Shape {
  int columns;  // of a lane: 16 bytes of a row, half as many beside lists of 5 to 16
  int lane_columns, splits;
  int64_t tiles, rows;
};

int list_size(int32_t top_k) { return top_k == 0 ? 0 : top_k <= 4 ? 4 : top_k <= 8 ? 8 : 16; }

Shape shape_of(int64_t classes, int64_t columns, int32_t dtype, int32_t top_k) {
  int const wide = dtype == PONNI_F32 ? 4 : 8, k = list_size(top_k);
  Shape s{};
  s.columns = columns < wide ? 1 : k == 0 ? wide : k <= 8 ? 4 : 2;
  int64_t const lanes = (columns + s.columns - 1) / s.columns;
  // Few classes: every lane takes all rows of its columns.  Else at most 8 lanes across.
  if (classes <= 64 && lanes > 64) {
    s.lane_columns = 8;
  } else {
    while (s.lane_columns < 3 && (1 << s.lane_columns) < lanes) s.lane_columns++;
    while (s.lane_columns < 5 && (1 << s.lane_columns) < lanes && (kThreads >> s.lane_columns) > classes) s.lane_columns++;
  }
  int64_t const across = int64_t(s.columns) << s.lane_columns, down = kThreads >> s.lane_columns;
  s.tiles = (columns + across - 1) / across;
  int64_t const turn = down * (s.columns >= 4 ? 4 : 8), turns = (classes + turn - 1) / turn;
  int64_t const want = down == 1 ? 1 : std::max<int64_t>(1, std::min(turns, kMostGroups / s.tiles));
  s.rows = (turns + want - 1) / want * turn;
  s.splits = static_cast<int>((classes + s.rows - 1) / s.rows);
  return s;
}

template <class F> void with_list(int k, F&& f) {
  switch (k) {
    case 0: f(std::integral_constant<int, 0>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    default: f(std::integral_constant<int, 16>{}); break;
  }
}

bool launchable(int64_t workgroups) { return workgroups <= int64_t(UINT32_MAX) / kThreads; }

}  // namespace

int64_t logp_workspace_bytes(int64_t classes, int64_t columns, int32_t dtype, int32_t top_k) {
  Shape const s = shape_of(classes, columns, dtype, top_k);
  return s.splits == 1 ? 0 : int64_t(s.splits) * (3 + 2 * list_size(top_k)) * columns * 4;
}

// A turn is at least 128 rows; more than one workgroup shares a tile of at most 64 columns, 1024 / tiles of them.
int64_t logp_workspace_bytes_up_to(int64_t classes, int64_t columns, int32_t top_k) {
  int64_t const turns = (classes + 127) / 128;
  if (turns == 1) return 0;
  int64_t const parts = columns < kMostParts / turns ? columns * turns : kMostParts;
  return parts * (3 + 2 * list_size(top_k)) * 4;
}

hipError_t launch_logp(ponni_log_probs const& p, void* workspace, hipStream_t stream) {
  Shape const s = shape_of(p.classes, p.columns, p.dtype, p.top_k);
  int const k = list_size(p.top_k);
  LogpArgs a{};
  a.p = p;
  a.lane_columns = s.lane_columns;
  a.splits = s.splits;
  a.rows = s.rows;
  a.parts = static_cast<float*>(workspace);
  a.part_values = a.parts + int64_t(s.splits) * 3 * p.columns;
  a.part_classes = reinterpret_cast<int32_t*>(a.part_values + int64_t(s.splits) * k * p.columns);
  int64_t const groups = s.tiles * s.splits;
  if (!launchable(groups)) return hipErrorInvalidConfiguration;
  with_dtype(p.dtype, [&](auto e) {
    using T = decltype(e);
    with_list(k, [&](auto list) {
      constexpr int K = decltype(list)::value, NC = K == 0 ? 16 / sizeof(T) : K <= 8 ? 4 : 2;
      dim3 const grid(static_cast<unsigned>(groups));
      if (s.columns == 1) hipLaunchKernelGGL((logp<T, 1, K>), grid, dim3(kThreads), 0, stream, a);
      else hipLaunchKernelGGL((logp<T, NC, K>), grid, dim3(kThreads), 0, stream, a);
    });
  });
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || s.splits == 1) return err;
  a.lane_columns = 0;
  while (a.lane_columns < 6 && (1 << a.lane_columns) < s.splits) a.lane_columns++;
  int64_t const joins = ((p.columns << a.lane_columns) + kThreads - 1) / kThreads;
  if (!launchable(joins)) return hipErrorInvalidConfiguration;
  with_dtype(p.dtype, [&](auto e) {
    with_list(k, [&](auto list) {
      hipLaunchKernelGGL((logp_join<decltype(e), decltype(list)::value>), dim3(static_cast<unsigned>(joins)),
                         dim3(kThreads), 0, stream, a);
    });
  });
  return hipGetLastError();
}

hipError_t launch_logp_backward(ponni_log_probs const& p, float const* d_log_probs, float const* d_entropy,
                                float const* d_log_normalizer, void* d_logits, int64_t ld_d_logits, hipStream_t stream) {
  int const wide = p.dtype == PONNI_F32 ? 4 : 8, nc = p.columns < wide ? 1 : wide;
  LogpBackwardArgs a{p, d_log_probs, d_entropy, d_log_normalizer, d_logits, ld_d_logits};
  int64_t const lanes = (p.columns + nc - 1) / nc;
  while (a.lane_columns < 3 && (1 << a.lane_columns) < lanes) a.lane_columns++;
  while (a.lane_columns < 8 && (1 << a.lane_columns) < lanes && (kThreads >> a.lane_columns) > p.classes) a.lane_columns++;
  int64_t const across = int64_t(nc) << a.lane_columns, turn = (kThreads >> a.lane_columns) * (nc >= 4 ? 4 : 8);
  a.tiles = (p.columns + across - 1) / across;
  int64_t const turns = (p.classes + turn - 1) / turn;
  // A workgroup takes a few turns, unless the grid is small.
  int64_t const parts = std::max<int64_t>(1, std::min(turns, std::max<int64_t>(2048 / a.tiles, (turns + 7) / 8)));
  a.rows = (turns + parts - 1) / parts * turn;
  int64_t const groups = a.tiles * ((p.classes + a.rows - 1) / a.rows);
  if (!launchable(groups)) return hipErrorInvalidConfiguration;
  with_dtype(p.dtype, [&](auto e) {
    using T = decltype(e);
    dim3 const grid(static_cast<unsigned>(groups));
    if (nc == 1) hipLaunchKernelGGL((logp_backward<T, 1>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((logp_backward<T, 16 / sizeof(T)>), grid, dim3(kThreads), 0, stream, a);
  });
  return hipGetLastError();
}

}  // namespace ponni_hip
