// Log probabilities, entropies and the largest classes of columns of logits
// x [classes, columns], and their gradient.
//
// One pass over x.  With m the largest x so far and t = (x - m) log2(e) a column keeps
//   z = sum 2^t,  q = sum 2^t t,
// which a larger m' turns into z s, (q + d z) s with d = (m - m') log2(e), s = 2^d, and
//   log_normalizer = m + ln2 log2 z,  entropy = ln2 (log2 z - q / z);
// any m near the largest x serves as well.
// (x log2(e) by itself, an operation less, has no room for the lowest floats.)
// A lane holds NC consecutive columns (16 bytes of a row) and takes every R-th row;
// lanes, waves and workgroups that share columns join their (m, z, q) in a fixed
// order.  The largest logits are lists in descending order, of equal values by
// class; two lists are joined by a bitonic step.
// The hardware's 2^x and log2 in every type, of a reference up to 4 below the largest: fp32 results are off by up to twice what
// a sum of exact powers is (10 classes: 1.1e-7 of their size, where elementary operations are off by 6.4e-8); the gradient in
// fp32 takes exp_f32.
// Bound by the logits' way from memory; 11 VALU operations an element beside it.  By kernel (a trace, with the gradient between
// two calls): bf16 65,536 classes x 4096: 154 + 5 us, 3.5 TB/s, the gradient 205, 5.2 TB/s read and written; fp32 10 x 4,194,304
// with the 3 largest: 95, 3.5 TB/s of logits and results; one bf16 column of 131,072 with the 8 largest: 14 + 8, latency.
// The figures beside the rules below are of calls of one kind one after the other, which leave part of the logits
// in the caches: 135 us for the 154 + 5, and 229 for the gradient's 205.
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
  int64_t first_tile;     // of this launch
  float* parts;           // [splits, 3, columns]: m, z, q
  float* part_values;     // [splits, K, columns]
  int32_t* part_classes;  // [splits, K, columns]
};

// Rows of a turn.
constexpr int rows_under_way(int columns, int k) { return columns == 1 && k == 0 ? 8 : 4; }
// A column's m is its largest logit up to kSlack: few turns have to move it, and no power passes 2^6.
constexpr float kSlack = 4.0f;

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

// The results of `count` of NC columns, whole rows of them at a time.
template <class T, int NC, int K> __device__ void finish(ponni_log_probs const& p, int64_t c, int count, Column<K> const (&s)[NC]) {
  Pack<float, NC> normalizer, entropy, log_prob;
#pragma unroll
  for (int j = 0; j < NC; j++) {
    float const lz = __log2f(s[j].z);
    normalizer.set(j, fmaf(kLn2, lz, s[j].m));
    entropy.set(j, s[j].z == 0.0f ? 0.0f : kLn2 * (lz - s[j].q / s[j].z));
  }
  normalizer.store(p.log_normalizer + c, count);
  entropy.store(p.entropy + c, count);
  if (p.targets != nullptr) {
#pragma unroll
    for (int j = 0; j < NC; j++) {
      int64_t const t = p.targets[c + (j < count ? j : 0)];
      float l = 0.0f;
      if (t >= 0 && t < p.classes) {
        l = static_cast<T const*>(p.logits)[t * p.ld + c + (j < count ? j : 0)];
        if (l != -kInf) l -= normalizer[j];
      }
      log_prob.set(j, l);
    }
    log_prob.store(p.log_probs + c, count);
  }
  if constexpr (K > 0)
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (k >= p.top_k) continue;
      Pack<float, NC> value;
      Pack<int32_t, NC> index;
#pragma unroll
      for (int j = 0; j < NC; j++) {
        bool const none = s[j].value[k] == -kInf;
        index.put(j, none ? -1 : s[j].index[k]);
        value.set(j, none ? -kInf : s[j].value[k] - normalizer[j]);
      }
      index.store(p.top_classes + k * p.columns + c, count);
      value.store(p.top_log_probs + k * p.columns + c, count);
    }
}

// The K largest of a lane's 16-bit logits: a logit's bits in ascending order above the complement of its turn, so
// that a place takes a maximum and a minimum (a value and its class apart take six operations).
template <class T, int K> struct Keys {
  unsigned key[K];
  __device__ void clear() {
#pragma unroll
    for (int k = 0; k < K; k++) key[k] = 0;
  }
  static __device__ unsigned make(T v, unsigned turn) {
    int w;  // (of NaN those of -inf, of -0 those of 0)
    if constexpr (std::is_same_v<T, _Float16>) {
      _Float16 const x = __builtin_fmaxf16(v + _Float16(0.0f), _Float16(-kInf));
      w = int(__builtin_bit_cast(unsigned short, x)) << 16;
    } else {
      w = __float_as_int(fmaxf(float(v) + 0.0f, -kInf));
    }
    return (unsigned(w ^ (w >> 31 | int(0x80000000))) & 0xffff0000u) | (0xffffu - turn);
  }
  __device__ void insert(unsigned x) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      unsigned const more = x > key[k] ? x : key[k], less = x > key[k] ? key[k] : x;
      key[k] = more, x = less;
    }
  }
  // Place k's logit (-inf: none), and its turn.
  __device__ float value(int k, int& turn) const {
    turn = 0xffff - int(key[k] & 0xffffu);
    unsigned const w = key[k] >> 16, bits = w & 0x8000u ? w ^ 0x8000u : w ^ 0xffffu;
    return key[k] == 0 ? -kInf : float(__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
  }
};

template <class T, int NC, int K> __global__ __launch_bounds__(kThreads) void logp(LogpArgs a) {
  constexpr int U = rows_under_way(NC, K);
  constexpr int WAVES = kThreads / 64;
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns;
  int const split = blockIdx.x % a.splits;
  int64_t const tile = a.first_tile + blockIdx.x / a.splits;
  int64_t const c0 = (tile * across + tx) * NC, left = a.p.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  int64_t const first = split * a.rows, end = first + a.rows < a.p.classes ? first + a.rows : a.p.classes;
  constexpr bool KEYS = K > 0 && sizeof(T) == 2;
  Column<K> s[NC];
  Keys<T, KEYS ? K : 1> keys[KEYS ? NC : 1];
#pragma unroll
  for (int j = 0; j < NC; j++) {
    s[j].clear();
    if constexpr (KEYS) keys[j].clear();
  }
  if (count > 0) {
    unsigned at = 0;  // rows of this lane so far
    int64_t const stride = down * a.p.ld;
    T const* x = static_cast<T const*>(a.p.logits) + (first + ty) * a.p.ld + c0;
    for (int64_t row = first + ty; row < end; row += int64_t(down) * U, x += U * stride) {
      Pack<T, NC> v[U];
      if (row + (U - 1) * down < end) {
#pragma unroll
        for (int u = 0; u < U; u++) v[u].load(x + u * stride, count, -kInf);
      } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (row + u * down < end) v[u].load(x + u * stride, count, -kInf);
          else v[u].fill(-kInf);
        }
      }
      float top[NC];
      bool beyond = false;
#pragma unroll
      for (int j = 0; j < NC; j++) {
        top[j] = v[0][j];
#pragma unroll
        for (int u = 1; u < U; u++) top[j] = fmaxf(top[j], v[u][j]);
        beyond = beyond || top[j] > s[j].m + kSlack;
      }
      if (__any(beyond)) {
#pragma unroll
        for (int j = 0; j < NC; j++) s[j].move_to(top[j] > s[j].m + kSlack ? top[j] : s[j].m);
      }
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float const shift = s[j].m == -kInf ? 0.0f : s[j].m;
#pragma unroll
        for (int u = 0; u < U; u++) {
          float const t = (v[u][j] - shift) * kLog2e, e = __builtin_amdgcn_exp2f(t);
          s[j].z += e;
          s[j].q = fmaf(e, fmaxf(t, kFar), s[j].q);
        }
        if constexpr (KEYS) {
          unsigned x[U], most = 0;
#pragma unroll
          for (int u = 0; u < U; u++) x[u] = keys[j].make(v[u].raw(j), at + u), most = x[u] > most ? x[u] : most;
          if (K <= 4 || __any(most > keys[j].key[K - 1])) {
#pragma unroll
            for (int u = 0; u < U; u++) keys[j].insert(x[u]);
          }
        } else if constexpr (K > 0) {
          if (__any(top[j] > s[j].value[K - 1])) {
#pragma unroll
            for (int u = 0; u < U; u++) s[j].insert(v[u][j], int32_t(row + u * down));
          }
        }
      }
      at += U;
    }
  }
  if constexpr (KEYS) {
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
      for (int k = 0; k < K; k++) {
        int turn;
        s[j].value[k] = keys[j].value(k, turn);
        s[j].index[k] = s[j].value[k] == -kInf ? INT32_MAX : int32_t(first + ty + int64_t(turn) * down);
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
#pragma unroll 1  // (code that runs once comes from memory: the shorter the better)
    for (int w = 0; w < WAVES; w++) {
      r.join(lds[w][0][c], lds[w][1][c], lds[w][2][c]);
      if constexpr (K > 0)
        r.join_list([&](int k, float& v, int32_t& i) { v = lds[w][3 + k][c], i = __float_as_int(lds[w][3 + K + k][c]); });
    }
    if (a.splits == 1) {
      Column<K> const one[1] = {r};
      finish<T, 1, K>(a.p, column, 1, one);
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
    if (count > 0) finish<T, NC, K>(a.p, c0, count, s);
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
  if (l == 0 && column < a.p.columns) {
    Column<K> const one[1] = {r};
    finish<T, 1, K>(a.p, column, 1, one);
  }
}

struct LogpBackwardArgs {
  ponni_log_probs p;
  float const *d_log_probs, *d_entropy, *d_log_normalizer;
  void* d_logits;
  int64_t ld_d;
  int lane_columns;
  int64_t rows;        // of a workgroup
  int64_t first_tile;  // of this launch
  int64_t tiles;       // of this launch
};

// p (gz - gl) - gh p (log p + entropy), and gl at the target.
template <class T, int NC> __global__ __launch_bounds__(kThreads) void logp_backward(LogpBackwardArgs a) {
  constexpr int U = NC >= 4 ? 4 : 8;
  constexpr bool EXACT = sizeof(T) == 4;
  int const across = 1 << a.lane_columns, tx = threadIdx.x & (across - 1), ty = threadIdx.x >> a.lane_columns;
  int const down = kThreads >> a.lane_columns;
  int64_t const tile = a.first_tile + blockIdx.x % a.tiles, c0 = (tile * across + tx) * NC, left = a.p.columns - c0;
  int const count = left < 1 ? 0 : left < NC ? int(left) : NC;
  if (count == 0) return;
  int64_t const first = blockIdx.x / a.tiles * a.rows, end = first + a.rows < a.p.classes ? first + a.rows : a.p.classes;
  float normalizer[NC], base[NC], entropy_weight[NC], at_target[NC];
  int32_t target[NC];
  Pack<float, NC> l, h, gp, gh, gn;
  Pack<int32_t, NC> t;
  l.load(a.p.log_normalizer + c0, count, 0.0f);
  gp.fill(0.0f), gh.fill(0.0f), gn.fill(0.0f), h.fill(0.0f);
  if (a.d_log_probs != nullptr) gp.load(a.d_log_probs + c0, count, 0.0f), t.load(a.p.targets + c0, count, -1.0f);
  if (a.d_entropy != nullptr) gh.load(a.d_entropy + c0, count, 0.0f), h.load(a.p.entropy + c0, count, 0.0f);
  if (a.d_log_normalizer != nullptr) gn.load(a.d_log_normalizer + c0, count, 0.0f);
#pragma unroll
  for (int j = 0; j < NC; j++) {
    bool const none = l[j] == -kInf;
    normalizer[j] = none ? kInf : l[j];  // (every p is 0)
    target[j] = a.d_log_probs != nullptr ? t.raw(j) : -1;
    if (none || int64_t(target[j]) >= a.p.classes) target[j] = -1;
    at_target[j] = target[j] >= 0 ? gp[j] : 0.0f;
    entropy_weight[j] = gh[j];
    base[j] = gn[j] - at_target[j];
    if (a.d_entropy != nullptr) base[j] -= gh[j] * h[j];
  }
  int64_t const stride = down * a.p.ld, stride_d = down * a.ld_d;
  T const* x = static_cast<T const*>(a.p.logits) + (first + ty) * a.p.ld + c0;
  T* d = static_cast<T*>(a.d_logits) + (first + ty) * a.ld_d + c0;
  for (int64_t row = first + ty; row < end; row += int64_t(down) * U, x += U * stride, d += U * stride_d) {
    Pack<T, NC> v[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (row + u * down < end) v[u].load(x + u * stride, count, 0.0f);
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
      o.store(d + u * stride_d, count);
    }
  }
}

// -- launches -----------------------------------------------------------------------------

// Workgroups that share columns, at most (1024 / 512 / 256: bf16 65,536 x 4096 135 / 146 / 248 us).
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
  // Few classes: every lane takes all rows of its columns (us with / without: bf16 64 x 1,000,000 43 / 91, fp32 10 x
  // 4,194,304 with the 3 largest 96 / 226, without them 83 / 78).  Else 128 bytes of a row across (128 / 64 / 32 bytes: bf16 65,536 x
  // 4096 135 / 149 / 221, 1000 x 262,144 with the 4 largest 212 / 250 / 388).
  int const line = s.columns == 1 || s.columns == wide ? 3 : s.columns * 2 == wide ? 4 : 5;
  if (classes <= 64 && lanes > 64) {
    s.lane_columns = 8;
  } else {
    while (s.lane_columns < line && (1 << s.lane_columns) < lanes) s.lane_columns++;
    while (s.lane_columns < 5 && (1 << s.lane_columns) < lanes && (kThreads >> s.lane_columns) > classes) s.lane_columns++;
  }
  int64_t const across = int64_t(s.columns) << s.lane_columns, down = kThreads >> s.lane_columns;
  s.tiles = (columns + across - 1) / across;
  int64_t const turn = down * rows_under_way(s.columns, k), turns = (classes + turn - 1) / turn;
  // (lists are worth joining from a few turns on; a lane's rows are counted in 16 bits)
  int64_t const most = k == 0 ? turns : (turns + 3) / 4;
  int64_t const want = down == 1 ? 1 : std::max<int64_t>(1, std::min(most, kMostGroups / s.tiles));
  s.rows = std::min((turns + want - 1) / want * turn, down * int64_t(65536));
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

constexpr int64_t kMostWorkgroups = int64_t(UINT32_MAX) / kThreads;  // of a launch
bool launchable(int64_t workgroups) { return workgroups <= kMostWorkgroups; }
// f(first tile, tiles) for launches of whole tiles, each of `groups` workgroups.
template <class F> hipError_t in_launches(int64_t tiles, int64_t groups, F&& f) {
  if (!launchable(groups)) return hipErrorInvalidConfiguration;
  int64_t const most = kMostWorkgroups / groups;
  for (int64_t first = 0; first < tiles; first += most) {
    f(first, std::min(tiles - first, most));
    hipError_t const err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace

int64_t logp_workspace_bytes(int64_t classes, int64_t columns, int32_t dtype, int32_t top_k) {
  Shape const s = shape_of(classes, columns, dtype, top_k);
  return s.splits == 1 ? 0 : int64_t(s.splits) * (3 + 2 * list_size(top_k)) * columns * 4;
}

// A turn is at least 32 rows; more than one workgroup shares a tile of at most 64 columns, 1024 / tiles of them (or as
// many as count their rows in 16 bits).
int64_t logp_workspace_bytes_up_to(int64_t classes, int64_t columns, int32_t top_k) {
  int64_t const turns = (classes + 31) / 32;
  if (turns == 1) return 0;
  int64_t parts = columns < kMostParts / turns ? columns * turns : kMostParts;
  constexpr int64_t COUNTED = 65536 * (kThreads >> 5);  // rows at least of a workgroup before its lanes' counts end
  if (classes > COUNTED) parts += columns * ((classes + COUNTED - 1) / COUNTED);
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
  hipError_t const err = in_launches(s.tiles, s.splits, [&](int64_t first, int64_t tiles) {
    a.first_tile = first;
    with_dtype(p.dtype, [&](auto e) {
      using T = decltype(e);
      with_list(k, [&](auto list) {
        constexpr int K = decltype(list)::value, NC = K == 0 ? 16 / sizeof(T) : K <= 8 ? 4 : 2;
        dim3 const grid(static_cast<unsigned>(tiles * s.splits));
        if (s.columns == 1) hipLaunchKernelGGL((logp<T, 1, K>), grid, dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL((logp<T, NC, K>), grid, dim3(kThreads), 0, stream, a);
      });
    });
  });
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
  if (p.classes <= 64 && lanes > 64) a.lane_columns = 8;  // (every lane takes all rows of its columns)
  while (a.lane_columns < 3 && (1 << a.lane_columns) < lanes) a.lane_columns++;
  int64_t const across = int64_t(nc) << a.lane_columns, turn = (kThreads >> a.lane_columns) * (nc >= 4 ? 4 : 8);
  int64_t const all_tiles = (p.columns + across - 1) / across;
  int64_t const turns = (p.classes + turn - 1) / turn;
  // A workgroup takes four turns, unless the grid is small (1 / 4 / 8 / 32 turns: bf16 65,536 x 4096 241 / 229 / 235 / 249 us,
  // 1000 x 262,144 255 / 235 / 238 / 238, fp32 30,000 x 4000 165 / 178 / 186 / 186).
  int64_t const parts = std::max<int64_t>(1, std::min(turns, std::max<int64_t>(2048 / all_tiles, (turns + 3) / 4)));
  a.rows = (turns + parts - 1) / parts * turn;
  int64_t const groups = (p.classes + a.rows - 1) / a.rows;
  return in_launches(all_tiles, groups, [&](int64_t first, int64_t tiles) {
    a.first_tile = first, a.tiles = tiles;
    with_dtype(p.dtype, [&](auto e) {
      using T = decltype(e);
      dim3 const grid(static_cast<unsigned>(tiles * groups));
      if (nc == 1) hipLaunchKernelGGL((logp_backward<T, 1>), grid, dim3(kThreads), 0, stream, a);
      else hipLaunchKernelGGL((logp_backward<T, 16 / sizeof(T)>), grid, dim3(kThreads), 0, stream, a);
    });
  });
}

}  // namespace ponni_hip
