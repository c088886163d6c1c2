// Gated feed-forward blocks: their products one after the other (gated_product.h), in
// the caller's arrays and work buffer.
//   forward   h = act(G^T x + g0) * (U^T x + u0) (and g, u), then y = D^T h + d0
//   backward  dg, du from D dy and the states; dx = G dg + U du; dG, dU = x dg^T, x du^T; dD = h dy^T;
//             biases' gradients are sums of rows
// Operands go into LDS by 16-byte pieces from multiples of 4 bytes, so a 16-bit array
// whose rows do not all begin at such is first copied to one whose rows do.
#include <algorithm>

#include "blocks.h"
#include "column_rows.h"
#include "gated.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

// Rows of a strided array at strides of whole pieces.
template <class T> __global__ __launch_bounds__(256) void align_rows(T const* from, int64_t ld, int64_t columns, T* to, int64_t ld_to) {
  constexpr int N = 16 / sizeof(T);
  int64_t const c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * N, row = blockIdx.y;
  if (c >= columns) return;
  Pack<T, N> v;
  v.load(from + row * ld + c, columns - c < N ? int(columns - c) : N, 0.0f);
  v.store(to + row * ld_to + c, N);
}

// y[row] = the sum of a row, of up to three arrays: a launch for all of a block's biases.
struct RowSums {
  void const* x[3];
  int64_t ld[3], rows[3];
  void* y[3];
};
template <class T> __global__ __launch_bounds__(256) void row_sums(RowSums a, int64_t columns) {
  constexpr int N = 16 / sizeof(T);
  __shared__ float lds[4];
  int64_t row = blockIdx.x;
  int const which = row < a.rows[0] ? 0 : row < a.rows[0] + a.rows[1] ? 1 : 2;
  row -= which == 0 ? 0 : which == 1 ? a.rows[0] : a.rows[0] + a.rows[1];
  T const* const x = static_cast<T const*>(a.x[which]) + row * a.ld[which];
  float s[N] = {};
  for (int64_t c = threadIdx.x * N; c < columns; c += 256 * N) {
    Pack<T, N> v;
    v.load(x + c, columns - c < N ? int(columns - c) : N, 0.0f);
#pragma unroll
    for (int e = 0; e < N; e++) s[e] += v[e];
  }
  float t = 0.0f;
#pragma unroll
  for (int e = 0; e < N; e++) t += s[e];
  for (int d = 1; d < 64; d *= 2) t += __shfl_xor(t, d);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = t;
  __syncthreads();
  if (threadIdx.x == 0) static_cast<T*>(a.y[which])[row] = T((lds[0] + lds[1]) + (lds[2] + lds[3]));
}

int64_t round_to(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t element(ponni_gated const& b) { return b.dtype == PONNI_F32 ? 4 : 2; }
// Row strides of the library's own arrays: whole lines of 128 bytes.
int64_t own_stride(int64_t columns, int64_t es) { return round_to(columns, 128 / es); }

// Tiles and parts of k of a product C [rows, columns] x problems over `steps` steps, by the time that each choice
// takes: us for a step of a tile (alone on its CU, or with another) and to begin and end one.  Small
// products lack tiles, so their k is cut; large ones take the tile that reads less.  Forward with states + backward,
// bf16 1024-4096-1024, us:
//                       128 x 128 whole   in 8 parts   256 x 256 whole   in 8 parts   chosen
//   200 columns         53 + 149          32 + 71      105 + 260         54 + 116     34 + 71
//   1000 columns        62 + 174          59 + 116     108 + 295         68 + 161     51 + 119
//   16,000 columns      476 + 1114        462 + 1118   376 + 1183        377 + 835    384 + 839
// and fp32 (128 x 128) 333-1001-77, 5000 columns: whole 159 + 846, chosen 120 + 234.  Gradients of narrow weights over many
// columns are one or two tiles with a long sum: fp32 48-38-131, 274,418 columns, dG and dU in 16 parts 1138 + 6, in 218
// 170 + 14.  Rows of a tile that are not there cost fp32 as much as others, so that narrow blocks take tiles of 64 rows (of a
// pair 32 of each product) x 256 columns.  fp32, calls, tiles of 128 x 128 alone / with those (elementary products):
//   2371-19-18 x 56,961 forward    558 / 176 (216)      64-64-64 x 500,000 forward     308 / 200 (655)
//   2257-17-29 x 13,897 forward    152 / 54 (117)       800-20-600 x 46,000 training   811 / 486 (730)
struct Choice {
  Tile tile;
  int parts;
  bool pair;  // both products of a pair at a time
  double time;
};
constexpr int kMostParts = 256, kLeastSteps = 8;
constexpr int64_t kMostSums = int64_t(256) * 256 * 256 * 4;  // bytes: of as many tiles as run at once

Choice choose(int64_t es, int64_t rows, int64_t columns, int problems, int64_t steps, bool pair, bool may_split) {
  Choice best{TILE_128, 1, pair, 1e300};
  for (Tile tile : {TILE_128, TILE_LARGE, TILE_NARROW}) {
    bool const large = tile == TILE_LARGE, narrow = tile == TILE_NARROW;
    if ((large && es != 2) || (narrow && es != 4)) continue;
    int64_t const bm = narrow ? (pair ? 32 : 64) : (large ? 256 : 128) / (pair && es == 2 ? 2 : 1), bn = tile != TILE_128 ? 256 : 128,
                  at_once = large ? 256 : 512;
    int64_t const tiles = (rows + bm - 1) / bm * ((columns + bn - 1) / bn) * problems;
    for (int parts = 1; parts <= kMostParts; parts += parts < 16 ? 1 : parts / 4) {
      if (parts > 1 && (!(may_split || (pair && narrow)) || steps / parts < kLeastSteps || tiles * parts > at_once)) break;
      int64_t const groups = tiles * parts, rounds = (groups + at_once - 1) / at_once;
      // (a tile of a pair in fp32 is both of them)
      bool const both = pair && es == 4 && !narrow;
      double const alone = es == 4 ? (both ? 2.2 : 1.3) : large ? 1.0 : 0.4, two = es == 4 ? (both ? 3.6 : 2.3) : 0.62;
      double const step = large || groups <= 256 ? alone : two;
      double time = double(rounds) * (double((steps + parts - 1) / parts) * step + (both ? 18.0 : pair && es == 4 ? 10.0 : 5.0));
      if (parts > 1) time += 4.0 + 0.05 * double(parts) + double(parts + 1) * double(rows * columns * problems * (pair ? 2 : 1)) * 4.0 / 3e6;
      if (time < best.time) best = {tile, parts, pair, time};
    }
  }
  return best;
}
// Both first products: one kernel for whole sums, or cut along k one after the other (with states, us whole / cut: fp32
// 4096-1024-4096, 64 columns 498 / 74, 512 528 / 140, 1024-4096-1024, 64 154 / 68).
Choice choose_pair(int64_t es, int64_t rows, int64_t columns, int64_t steps) {
  Choice const whole = choose(es, rows, columns, 1, steps, true, false);
  Choice const cut = choose(es, rows, columns, 1, steps, false, true);
  return cut.parts > 1 && 2 * cut.time < whole.time ? cut : whole;
}

// The caller's work buffer, taken piece by piece (base null: counted only).
struct Taker {
  char* base;
  int64_t used = 0;
  char* take(int64_t bytes) {
    char* const p = base + used;
    used += round_to(bytes, 256);
    return p;
  }
};

struct Matrix {
  void const* p;
  int64_t rows, columns, ld;
};

int64_t aligned_bytes(int64_t rows, int64_t columns, int64_t es) { return rows * own_stride(columns, es) * es; }
// At most, for any number of columns up to the one given.
int64_t sums_bytes(int64_t rows, int64_t columns, int problems, int64_t steps) {
  int64_t const parts = std::min<int64_t>(kMostParts, steps / kLeastSteps);
  return parts < 2 ? 0 : std::min(kMostSums, parts * problems * rows * round_to(columns, 4) * 4);
}

// Whether an array is read where it is: all rows at multiples of 4 bytes.
bool in_place(void const* p, int64_t rows, int64_t ld, int64_t es) {
  return reinterpret_cast<uint64_t>(p) % 4 == 0 && (rows == 1 || ld * es % 4 == 0);
}
// The same of two arrays of one shape, which are read at one stride.
bool pair_in_place(void const* a, int64_t ld_a, void const* b, int64_t ld_b, int64_t rows, int64_t es) {
  return in_place(a, rows, ld_a, es) && in_place(b, rows, ld_b, es) && (rows == 1 || ld_a == ld_b);
}

// One call's products.
template <class T> struct Run {
  Taker work;
  hipStream_t stream;
  hipError_t err = hipSuccess;

  Side side(Matrix const& m) {
    if (!in_place(m.p, m.rows, m.ld, sizeof(T))) return copied(m);
    constexpr int64_t ES = sizeof(T);
    int64_t const ld = m.rows == 1 ? round_to(m.columns, 4 / ES) : m.ld;
    return {static_cast<char const*>(m.p), ld * ES, round_to(((m.rows - 1) * ld + m.columns) * ES, 4), m.rows};
  }
  // Two arrays of one shape, of one stride.
  void sides(Matrix const& a, Matrix const& b, Side (&out)[2]) {
    bool const both = pair_in_place(a.p, a.ld, b.p, b.ld, a.rows, sizeof(T));
    out[0] = both ? side(a) : copied(a), out[1] = both ? side(b) : copied(b);
  }
  Side copied(Matrix const& m) {
    constexpr int64_t ES = sizeof(T);
    int64_t const ld = own_stride(m.columns, ES);
    T* const to = reinterpret_cast<T*>(work.take(m.rows * ld * ES));
    constexpr int64_t ROWS = 65535;
    for (int64_t row = 0; row < m.rows && err == hipSuccess; row += ROWS) {
      dim3 const grid(unsigned((m.columns * ES + 4095) / 4096), unsigned(std::min(ROWS, m.rows - row)));
      hipLaunchKernelGGL(align_rows<T>, grid, dim3(256), 0, stream, static_cast<T const*>(m.p) + row * m.ld, m.ld, m.columns,
                         to + row * ld, ld);
      err = hipGetLastError();
    }
    return {reinterpret_cast<char const*>(to), ld * ES, round_to(((m.rows - 1) * ld + m.columns) * ES, 4), m.rows};
  }
  void product(Form form, ProductArgs p) {
    if (err != hipSuccess) return;
    constexpr int64_t ES = sizeof(T), STEP = 64 / ES;
    if (p.problems == 0) p.problems = 1;
    int64_t const steps = (form == FORM_INPUT ? 2 : 1) * ((p.k + STEP - 1) / STEP);
    Choice const c = form == FORM_PAIR ? choose_pair(ES, p.rows, p.columns, steps)
                                       : choose(ES, p.rows, p.columns, p.problems, steps, false, true);
    p.parts = c.parts, p.pair_parts = c.pair && c.parts > 1;
    Taker const before = work;  // (the sums are read before the next product begins)
    if (c.parts > 1) {
      p.ld_sums = round_to(p.columns, 4);
      p.sums = reinterpret_cast<float*>(
          work.take(c.parts * (form == FORM_PAIR ? 2 : p.problems) * p.rows * p.ld_sums * 4));
    }
    err = (std::is_same_v<T, float>      ? launch_product_f32
           : std::is_same_v<T, _Float16> ? launch_product_f16
                                         : launch_product_bf16)(form, c.tile, p, stream);
    work = before;
  }
  void sums(RowSums const& a, int64_t columns) {
    int64_t const rows = a.rows[0] + a.rows[1] + a.rows[2];
    if (err != hipSuccess || rows == 0) return;
    hipLaunchKernelGGL(row_sums<T>, dim3(unsigned(rows)), dim3(256), 0, stream, a, columns);
    err = hipGetLastError();
  }
};

// Slices of k of a product of few columns: about `groups` workgroups, each with at least a step for each of its four
// waves.
struct Slices {
  int count, k;
};
Slices slices_of(int64_t es, int64_t k, int64_t outputs, int problems, int64_t groups) {
  int64_t const step = 4 * (64 / es), tile = 256 / es, tiles = (outputs + tile - 1) / tile * problems;
  int64_t const want = std::max<int64_t>(1, groups / tiles);
  int64_t const most = std::min((k + step - 1) / step, want), each = round_to((k + most - 1) / most, step);
  // (its columns, and the waves' sums, in 64 KB of LDS)
  int64_t const held = std::min<int64_t>(each, 1024 / es);
  return {int((k + held - 1) / held), int(held)};
}
// Columns that they take at most; in fp32 the fewer the more weights there are.  us so / in tiles: bf16 1024-4096-1024 1
// column 17 / 30, 32 columns 25 / 28; fp16 256-700-256, 8 columns 16 / 20, 32 26 / 24; fp32 1024-4096-1024 (12.6 M weights) 64 columns
// 51 / 67, 128 81 / 75, 4096-1024-4096 (12.6 M) 64 50 / 74, 128 80 / 84, 256 141 / 99; 2048-2000-300 (8.8 M) 128 60 / 69, 256
// 104 / 81; 333-1001-77 (0.7 M) 512 40 / 57; 64-4096-64 (0.8 M) 512 44 / 45.
int64_t most_thin(ponni_gated const& b) {
  constexpr int64_t kThin = 32, kMostThin = 512, kProducts = 1'400'000'000;
  if (element(b) == 2) return kThin;
  return std::clamp(kProducts / ((2 * int64_t(b.n_in) + b.n_out) * b.n_hidden), kThin, kMostThin);
}
struct ThinPlan {
  Slices hidden, last;
  int64_t stride_hidden, stride_last, parts_hidden, parts_last, rows;  // strides in elements, the others in bytes
  int64_t bytes() const { return parts_hidden + parts_last + rows; }
};
ThinPlan thin_plan(ponni_gated const& b, int64_t columns) {
  int64_t const es = element(b), tile = 256 / es, hidden = round_to(b.n_hidden, tile), last = round_to(b.n_out, tile);
  ThinPlan p{slices_of(es, b.n_in, b.n_hidden, 2, columns <= 8 ? 512 : 256), slices_of(es, b.n_hidden, b.n_out, 1, 512), hidden, last, 0, 0, 0};
  p.parts_hidden = round_to(p.hidden.count * 2 * columns * hidden * 4, 256);
  p.parts_last = round_to(p.last.count * columns * last * 4, 256);
  // Every tile of the last product reads all parts of its slice again, unless h is made of them once: us with / without
  // that launch, 2048-4096-2048 fp16, 20 columns: 14 / 16; where few parts are read, as 2 MB at 1024-4096-1024 and one
  // column, it would add its 4.
  if (last / tile * p.parts_hidden > hidden * b.n_out * es) p.rows = round_to(columns * hidden * es, 256);
  return p;
}

int64_t steps_of(int64_t k, int64_t es) { return (k + 64 / es - 1) / (64 / es); }

}  // namespace

int64_t gated_workspace_bytes(ponni_gated const& b, int64_t columns, bool backward, GatedArrays const* arrays) {
  int64_t const es = element(b), i = b.n_in, h = b.n_hidden, o = b.n_out;
  bool const states = arrays != nullptr && arrays->states != nullptr;
  if (!backward && arrays != nullptr && !states && columns <= most_thin(b)) return thin_plan(b, columns).bytes();
  Taker t{nullptr};
  auto copy = [&](bool needed, int64_t rows, int64_t of) {
    if (needed) t.take(aligned_bytes(rows, of, es));
  };
  // Of an array with columns: where it is not known, any of 16 bits may need a copy.
  auto moved = [&](void const* p, int64_t rows, int64_t ld) { return arrays != nullptr ? !in_place(p, rows, ld, es) : es == 2; };
  bool const pair = pair_in_place(b.gate, b.ld_gate, b.up, b.ld_up, i, es);
  GatedArrays const a = arrays != nullptr ? *arrays : GatedArrays{};
  copy(!pair, i, h);
  copy(!pair, i, h);
  copy(!in_place(b.down, h, b.ld_down, es), h, o);
  copy(moved(a.x, i, a.ld_x), i, columns);
  if (!backward) {
    copy(!states || moved(a.states, h, a.ld_states), h, columns);  // h itself, or a copy of the states'
    t.take(std::max(sums_bytes(o, columns, 1, steps_of(h, es)), 2 * sums_bytes(h, columns, 1, steps_of(i, es))));
    if (arrays != nullptr) return t.used;
    // (the slices become fewer past 8 columns)
    return std::max({t.used, thin_plan(b, std::min<int64_t>(columns, 8)).bytes(),
                     thin_plan(b, std::min(columns, most_thin(b))).bytes()});
  }
  copy(moved(a.states, h, a.ld_states), h, columns);
  copy(moved(a.dy, o, a.ld_dy), o, columns);
  t.take(aligned_bytes(2 * h, columns, es));  // dg, du
  t.take(std::max({sums_bytes(i, columns, 1, 2 * steps_of(h, es)), sums_bytes(i, h, 2, steps_of(columns, es)),
                   sums_bytes(h, o, 1, steps_of(columns, es)), sums_bytes(h, columns, 1, steps_of(o, es))}));
  return t.used;
}

hipError_t launch_gated(ponni_gated const& b, int act, void const* x, int64_t ld_x, void* y, int64_t ld_y, void* states,
                        int64_t ld_states, int64_t columns, void* workspace, hipStream_t stream) {
  hipError_t err = hipSuccess;
  with_dtype(b.dtype, [&](auto e) {
    using T = decltype(e);
    Run<T> run{{static_cast<char*>(workspace)}, stream};
    int64_t const hidden = b.n_hidden, es = sizeof(T);
    if (states == nullptr && columns <= most_thin(b)) {
      ThinPlan const plan = thin_plan(b, columns);
      ThinArgs first{}, last{};
      first.w[0] = b.gate, first.w[1] = b.up, first.ld[0] = b.ld_gate, first.ld[1] = b.ld_up;
      first.k = b.n_in, first.outputs = b.n_hidden, first.columns = int(columns);
      first.slices = plan.hidden.count, first.slice_k = plan.hidden.k, first.stride = int(plan.stride_hidden);
      first.x = x, first.ld_x = ld_x;
      first.parts = reinterpret_cast<float*>(run.work.take(plan.parts_hidden));
      last.w[0] = b.down, last.ld[0] = b.ld_down;
      last.k = b.n_hidden, last.outputs = b.n_out, last.columns = int(columns);
      last.slices = plan.last.count, last.slice_k = plan.last.k, last.stride = int(plan.stride_last);
      last.parts = reinterpret_cast<float*>(run.work.take(plan.parts_last));
      if (plan.rows > 0) last.h = run.work.take(plan.rows);
      last.parts_in = first.parts, last.slices_in = first.slices, last.stride_in = first.stride;
      last.act = act, last.slope = float(b.act.attr[0]);
      last.bias[0] = b.gate_bias, last.bias[1] = b.up_bias, last.bias[2] = b.down_bias;
      last.y = y, last.ld_y = ld_y;
      err = (std::is_same_v<T, float>      ? launch_thin_f32
             : std::is_same_v<T, _Float16> ? launch_thin_f16
                                           : launch_thin_bf16)(first, last, stream);
      return;
    }
    T* const s = static_cast<T*>(states);
    int64_t const ld_h = s != nullptr ? ld_states : own_stride(columns, es);
    T* const h = s != nullptr ? s + 2 * hidden * ld_states : reinterpret_cast<T*>(run.work.take(hidden * ld_h * es));
    ProductArgs p{};
    run.sides({b.gate, b.n_in, hidden, b.ld_gate}, {b.up, b.n_in, hidden, b.ld_up}, p.a);
    p.b[0] = run.side({x, b.n_in, columns, ld_x});
    p.k = b.n_in, p.rows = hidden, p.columns = columns;
    p.y[0] = h, p.ld[0] = ld_h, p.bias[0] = b.gate_bias, p.bias[1] = b.up_bias;
    p.act = act, p.slope = float(b.act.attr[0]), p.states = s, p.ld_states = ld_states;
    run.product(FORM_PAIR, p);
    ProductArgs q{};
    q.a[0] = run.side({b.down, hidden, b.n_out, b.ld_down});
    q.b[0] = run.side({h, hidden, columns, ld_h});
    q.k = hidden, q.rows = b.n_out, q.columns = columns, q.y[0] = y, q.ld[0] = ld_y, q.bias[0] = b.down_bias;
    run.product(FORM_FORWARD, q);
    err = run.err;
  });
  return err;
}

hipError_t launch_gated_backward(ponni_gated const& b, int act, void const* x, int64_t ld_x, void const* states,
                                 int64_t ld_states, void const* dy, int64_t ld_dy, int64_t columns,
                                 ponni_gated_gradients const& d, void* workspace, hipStream_t stream) {
  hipError_t err = hipSuccess;
  with_dtype(b.dtype, [&](auto e) {
    using T = decltype(e);
    Run<T> run{{static_cast<char*>(workspace)}, stream};
    int64_t const hidden = b.n_hidden, es = sizeof(T), ld = own_stride(columns, es);
    T const* const s = static_cast<T const*>(states);
    T *const dg = reinterpret_cast<T*>(run.work.take(2 * hidden * ld * es)), *const du = dg + hidden * ld;
    Matrix const m_dy{dy, b.n_out, columns, ld_dy};
    Side const s_dy = run.side(m_dy);
    ProductArgs p{};
    p.a[0] = run.side({b.down, hidden, b.n_out, b.ld_down});
    p.b[0] = s_dy;
    p.k = b.n_out, p.rows = hidden, p.columns = columns, p.y[0] = dg, p.y[1] = du, p.ld[0] = ld;
    p.act = act, p.slope = float(b.act.attr[0]), p.states = const_cast<T*>(s), p.ld_states = ld_states;
    run.product(FORM_STATES, p);
    Side const s_dg = run.side({dg, hidden, columns, ld}), s_du = run.side({du, hidden, columns, ld});
    if (d.x != nullptr) {
      ProductArgs q{};
      run.sides({b.gate, b.n_in, hidden, b.ld_gate}, {b.up, b.n_in, hidden, b.ld_up}, q.a);
      q.b[0] = s_dg, q.b[1] = s_du, q.k = hidden, q.rows = b.n_in, q.columns = columns;
      q.y[0] = d.x, q.ld[0] = d.ld_x;
      run.product(FORM_INPUT, q);
    }
    if (d.gate != nullptr || d.up != nullptr) {
      ProductArgs q{};
      q.a[0] = run.side({x, b.n_in, columns, ld_x});
      q.k = columns, q.rows = b.n_in, q.columns = hidden;
      int n = 0;
      if (d.gate != nullptr) q.b[n] = s_dg, q.y[n] = d.gate, q.ld[n] = d.ld_gate, n++;
      if (d.up != nullptr) q.b[n] = s_du, q.y[n] = d.up, q.ld[n] = d.ld_up, n++;
      q.problems = n;
      run.product(FORM_WEIGHTS, q);
    }
    if (d.down != nullptr) {
      ProductArgs q{};
      q.a[0] = run.side({s + 2 * hidden * ld_states, hidden, columns, ld_states});
      q.b[0] = s_dy;
      q.k = columns, q.rows = hidden, q.columns = b.n_out, q.y[0] = d.down, q.ld[0] = d.ld_down;
      run.product(FORM_WEIGHTS, q);
    }
    run.sums({{dg, du, dy}, {ld, ld, ld_dy},
              {d.gate_bias ? hidden : 0, d.up_bias ? hidden : 0, d.down_bias ? b.n_out : 0},
              {d.gate_bias, d.up_bias, d.down_bias}}, columns);
    err = run.err;
  });
  return err;
}

}  // namespace ponni_hip
