// The products of gated blocks on the matrix cores (kernels_gated_f32.hip,
// kernels_gated_f16.hip, kernels_gated_bf16.hip):
//   C[m, n] = sum over k of A(m, k) B(n, k)
// with operands where the caller has them, in one of two layouts: k outside
// ([k, i]: weights [n_in, n_out] and columns of a forward product) or k inside
// ([i, k]: transposed weights, and both operands of a weight's gradient).
//
// A step is 64 bytes of k of every row: 32 features of a 16-bit type, 16 of fp32.  Its
// tiles go from memory straight into one of four slots of LDS, up to three steps
// ahead (fp32 with k outside: three slots), a request's 64 pieces of 16 bytes in a row; a step's fragments are
// read while the one before is multiplied.  Rows of k outside are
// turned on their way out of LDS (ds_read_b64_tr_b16: four rows of four elements to four
// lanes); pieces lie at places that depend on their row, so that a
// read's lanes fall into different banks.  What lies past an array's end is zero by the
// range check of the buffer request; a row's pieces past its last k are asked
// for out of range, and the part of a piece past it is cleared in registers.
//
// The MFMA's first operand is B's fragment, so that a lane's four sums are
// consecutive columns of one row; 4 x 4 such groups are exchanged between the lanes
// (v_permlane32_swap, v_permlane16_swap) into 16 consecutive columns a lane, 128
// bytes of a row by four lanes.
//
// Bound by the matrix cores where k is long, and by the outputs (three or two arrays, with the states read)
// beside them where it is short: all workgroups come to their outputs together.  bf16 1024-4096-1024, 16,384 columns, us (PFLOP/s):
// g, u and h 306 (0.90), y 110 (1.25), dg and du 275 (0.50), dx 252 (1.09), dG and dU 256 + 12 (1.03),
// dD 147 + 14 (0.85); a library's product of 8192 x 8192 x 8192 1.12.  fp16 2048-8192-2048,
// 32,768: h 1848 (1.19), y 819 (1.34).  fp32 1024-4096-1024, 16,384: 136 to 142 TFLOP/s of 154; 333-1001-77, 5,003: 66 to
// 83, few tiles and short sums; 2371-19, 56,961: 165 us, 3.3 TB/s of x.
#pragma once

#include <algorithm>
#include <type_traits>

#include "activations.h"
#include "blocks.h"
#include "column_rows.h"
#include "gated.h"
#include "lds_requests.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

typedef __attribute__((address_space(3))) void* lds_void;

constexpr int kGroup = 8;  // columns of tiles that workgroups of an XCD share

__device__ inline uint64_t uniform64(uint64_t p) {
  unsigned const lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(p));
  unsigned const hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(p >> 32));
  return uint64_t(hi) << 32 | lo;
}

// each(f), f(v, a, d) giving a = act(v) and d = act'(v): in 16 bits by the hardware's exponential and reciprocal.
template <bool Precise, class Each> __device__ inline void with_activation(int act, float slope, Each&& each) {
  auto const sigmoid = [](float x) { return Precise ? sigmoid_f32(x) : act_sigmoid_fast(x); };
  switch (act) {
    case ACT_RELU: each([](float v, float& a, float& d) { a = act_relu(v), d = v > 0.0f ? 1.0f : 0.0f; }); break;
    case ACT_LEAKY_RELU:
      each([slope](float v, float& a, float& d) { a = act_leaky_relu(v, slope), d = v > 0.0f ? 1.0f : slope; });
      break;
    case ACT_TANH:
      each([](float v, float& a, float& d) { a = Precise ? tanh_f32(v) : tanh_half(v), d = fmaf(-a, a, 1.0f); });
      break;
    case ACT_SIGMOID: each([&](float v, float& a, float& d) { a = sigmoid(v), d = a * sigmoid(-v); }); break;
    case ACT_SILU:
      each([&](float v, float& a, float& d) {
        float const p = sigmoid(v);
        a = Precise ? silu_f32(v) : v * p, d = p * fmaf(v, Precise ? sigmoid(-v) : 1.0f - p, 1.0f);
      });
      break;
    case ACT_GELU_TANH:
      each([&](float v, float& a, float& d) {
        constexpr float c = 2.0f * 0.79788456080286535588f;
        float const p = sigmoid(c * v * fmaf(0.044715f * v, v, 1.0f));
        a = Precise ? gelu_tanh_f32(v) : v * p;
        // (from 16 on p is 0 or 1; a square that overflows must not meet that zero)
        float const w = __builtin_amdgcn_fmed3f(v, -64.0f, 64.0f);
        d = p * fmaf(c * w * fmaf(3.0f * 0.044715f * w, w, 1.0f), 1.0f - p, 1.0f);
      });
      break;
    default:
      each([](float v, float& a, float& d) {
        float const p = 0.5f * erfcf(-0.70710678118654752440f * v);
        a = act_gelu_erf(v), d = fmaf(v * 0.39894228040143267794f, exp_f32(-0.5f * v * v), p);
      });
  }
}

// One 16-byte request per lane into LDS at lds + 16 * lane; offsets past the resource's
// bytes give zeros.  (Wait states: as dma16.)
__device__ inline void dma16_in_range(i32x4 resource, unsigned offset, unsigned lds) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(resource), "{m0}"(lds) : "memory");
}
// A buffer of raw bytes from p on.
__device__ inline i32x4 resource_of(uint64_t p, uint64_t bytes) {
  unsigned high = unsigned(bytes >> 32);
  asm("" : "+s"(high));  // (a comparison of 64 bits would be the vector unit's)
  unsigned const n = high != 0 || unsigned(bytes) > 0xffffffe0u ? 0xffffffe0u : unsigned(bytes);
  // (uniform, which the compiler does not see everywhere)
  return i32x4{__builtin_amdgcn_readfirstlane(int(p)), __builtin_amdgcn_readfirstlane(int((p >> 32) & 0xffff)),
               __builtin_amdgcn_readfirstlane(int(n)), 0x00027000};
}

// A step's product of two fragments, in fp32 of its part e of four (16 bits: of one).
template <class T> constexpr int kMfmaParts = sizeof(T) == 4 ? 4 : 1;
template <class T> __device__ inline f32x4 mfma_part(i32x4 a, i32x4 b, f32x4 c, int e) {
  if constexpr (std::is_same_v<T, float>) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[e], __builtin_bit_cast(f32x4, b)[e], c, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, _Float16>) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  } else {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
}

// 4 x 4 groups of four floats between the 16-lane rows of a wave: group j of row g goes to row j, as its group g.
__device__ inline void exchange(f32x4 (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    // (values of their own: a bit cast of a vector's element is taken of its first one)
    unsigned const u0 = __float_as_uint(v[0][e]), u1 = __float_as_uint(v[1][e]), u2 = __float_as_uint(v[2][e]),
                   u3 = __float_as_uint(v[3][e]);
    auto const a = __builtin_amdgcn_permlane32_swap(u0, u2, false, false);
    auto const b = __builtin_amdgcn_permlane32_swap(u1, u3, false, false);
    auto const c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto const d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    v[0][e] = __uint_as_float(c[0]);
    v[1][e] = __uint_as_float(c[1]);
    v[2][e] = __uint_as_float(d[0]);
    v[3][e] = __uint_as_float(d[1]);
  }
}

// Where a lane's pieces of an operand's tile of SIZE rows come from, and where its fragments
// lie in a slot.  PANELS arrays side by side, each of SIZE / PANELS rows.
template <class T, bool INNER, int SIZE, int PANELS, int W> struct Loader {
  static constexpr int ES = sizeof(T), STEP = 64 / ES, PIECE = 16 / ES;
  static constexpr int BYTES = SIZE * 64, REQUESTS = BYTES / 1024 / W, PANEL = SIZE / PANELS;
  static constexpr int ROW = PANEL * ES;             // bytes of a k's row of a panel
  static constexpr int PLACES = ROW / 16;            // pieces of it
  static constexpr int PER_PANEL = PANEL * 64 / 1024;  // requests
  static constexpr bool APART = PANELS > 1 && PER_PANEL < W;  // a wave's one request is of its panel
  static constexpr int BASES = INNER ? REQUESTS : APART ? 1 : PANELS;
  static_assert(BYTES % (1024 * W) == 0 && 64 % PLACES == 0 && (PANELS == 1 || PER_PANEL % W == 0 || (APART && !INNER && REQUESTS == 1)),
                "whole requests, of one panel each");
  unsigned offset[REQUESTS];  // of the lane's piece from the request's base
  int k[REQUESTS];            // INNER: the first k of the piece, within a step
  // Of the step that is asked for next, uniform: where each base lies, the bytes from there to the array's end, k's left.
  uint64_t at[BASES];
  uint64_t left[BASES];
  int k_left;
  uint64_t stride;

  // A piece's place: pieces of rows that a read's lanes take together lie in different banks.
  static __device__ int twist(int row) {
    return INNER ? (row >> 1) & 3 : ES == 2 ? 2 * ((row & 3) | (PLACES > 8 ? row >> 1 & 4 : 0)) : 0;
  }

  __device__ void init(int wave, int lane, Side const& s, int64_t first) {
#pragma unroll
    for (int r = 0; r < REQUESTS; r++) {
      int const piece = wave + W * r;
      if constexpr (INNER) {
        int64_t const base = base_row(piece, s, first), row = first + piece * 16 + lane / 4;
        k[r] = ((lane % 4) ^ twist(lane / 4)) * PIECE;
        // (rows past the last one repeat it)
        offset[r] = unsigned(((row < s.rows ? row : s.rows - 1) - base) * s.ld) + k[r] * ES;
      } else {
        int const row = piece % PER_PANEL * (64 / PLACES) + lane / PLACES;
        offset[r] = unsigned(row * s.ld) + ((lane % PLACES) ^ twist(row)) * 16;
      }
    }
    stride = INNER ? 64 : uniform64(STEP * s.ld);
  }
  static __device__ int64_t base_row(int piece, Side const& s, int64_t first) {
    int64_t const row = first + piece * 16;
    return row < s.rows ? row : s.rows - 1;
  }
  // The step that begins at k0 of `last` k's is the next one; s: the arrays.
  __device__ void seek(int wave, Side const* s, int64_t first, int64_t k0, int64_t last) {
#pragma unroll
    for (int b = 0; b < BASES; b++) {
      Side const& from = s[INNER ? 0 : APART ? wave / PER_PANEL : b];
      uint64_t const o = INNER ? base_row(wave + W * b, from, first) * from.ld + k0 * ES : k0 * from.ld + first * ES;
      at[b] = uniform64(uint64_t(from.p) + o);
      left[b] = uniform64(from.bytes - o);
    }
    k_left = __builtin_amdgcn_readfirstlane(int(last - k0));
  }
  __device__ void advance() {
#pragma unroll
    for (int b = 0; b < BASES; b++) at[b] = uniform64(at[b] + stride), left[b] = uniform64(left[b] - stride);
    k_left = __builtin_amdgcn_readfirstlane(k_left - STEP);
  }
  // From behind the last step of one array to the first of another `distance` bytes on, of the same shape.
  __device__ void jump(bool now, uint64_t distance, int steps, int64_t last) {
    uint64_t const back = now ? steps * stride : 0, on = now ? distance : 0;
#pragma unroll
    for (int b = 0; b < BASES; b++) at[b] = uniform64(at[b] + on - back), left[b] = uniform64(left[b] + back);
    k_left = __builtin_amdgcn_readfirstlane(now ? int(last) : k_left);
  }
  __device__ void request(int r, int wave, unsigned lds) const {
    int const base = INNER ? r : APART ? 0 : W * r / PER_PANEL;
    unsigned const o = INNER && k[r] >= k_left ? 0xfffffff0u : offset[r];
    dma16_in_range(resource_of(at[base], left[base]), o, lds + (wave + W * r) * 1024);
  }

  // Reads.  The lane's place for fragment 0 of the wave's fragments, which begin at row `first` of a panel.
  static __device__ unsigned read_base(int first, int lane) {
    int const g = lane >> 4, c = lane & 15;
    if constexpr (INNER) return (first + c) * 64 + 16 * (g ^ twist(c));
    else if constexpr (ES == 4 && APART) return c / 8 * (PANEL * 64) + 4 * g * ROW + 16 * (c % 8);  // (panels of 32 rows: a block of 64)
    else if constexpr (ES == 4) return 4 * g * ROW + first * 4 + 16 * c;
    else {
      int const row = 8 * g + c / 4;
      return row * ROW + (((first * 2) ^ (twist(row) * 16)) + c % 4 * 8);
    }
  }
};

// Fragment f of a wave's N, which begin at `base` (Loader::read_base) of a slot: into v.
template <class T, bool INNER, int ROW, int N> __device__ inline void read_fragment(char const* slot, unsigned base, int f, i32x4 (&v)[N], int to) {
  if constexpr (INNER) {
    v[to] = *reinterpret_cast<i32x4 const*>(slot + base + f * 1024);
  } else if constexpr (sizeof(T) == 2) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4* lds_s4;
    char* const p = const_cast<char*>(slot) + (base ^ (f * 32));
    s4 const lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
    s4 const hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * ROW));
    v[to] = __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    // Columns 4 c + j of a block of 64 are fragment j's column c: a read is part f % 4 of four fragments.
    v[to] = *reinterpret_cast<i32x4 const*>(slot + base + f / 4 * 256 + f % 4 * ROW);
  }
}
// Fragment f for mfma_part's part e.
template <class T, bool INNER, int N> __device__ inline i32x4 fragment(i32x4 const (&v)[N], int f, int e) {
  if constexpr (INNER || sizeof(T) == 2) return v[f];
  i32x4 x = v[f];
  x[e] = v[f / 4 * 4 + e][f % 4];
  return x;
}
template <class T, bool INNER> __device__ inline void clear_past(i32x4& v, int lane, int64_t left) {
  // The fragment's k's from `left` on (of the step): zero.
  if constexpr (INNER) {
    constexpr int N = 16 / sizeof(T);
    typedef T Piece __attribute__((ext_vector_type(N)));
    Piece p = __builtin_bit_cast(Piece, v);
#pragma unroll
    for (int e = 0; e < N; e++) p[e] = (lane >> 4) * N + e < left ? p[e] : T(0.0f);
    v = __builtin_bit_cast(i32x4, p);
  }
}

// 16 consecutive elements of a row of `left` from here on.
template <class T> __device__ inline void store16(T* y, int64_t left, float const (&v)[16]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int p = 0; p < 16; p += N) {
    Pack<T, N> o;
#pragma unroll
    for (int e = 0; e < N; e++) o.set(e, v[p + e]);
    if (left > p) o.store(y + p, left - p < N ? int(left - p) : N);
  }
}
template <class T> __device__ inline void load16(T const* x, int64_t left, float (&v)[16]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int p = 0; p < 16; p += N) {
    Pack<T, N> o;
    o.fill(0.0f);
    if (left > p) o.load(x + p, left - p < N ? int(left - p) : N, 0.0f);
#pragma unroll
    for (int e = 0; e < N; e++) v[p + e] = o[e];
  }
}

template <Output OUT> constexpr bool kPair = OUT == OUT_PAIR || OUT == OUT_PAIR_PARTS;

// TWO: a sum of two products, of operands of the same shapes and strides.
template <class T, bool A_INNER, bool B_INNER, Output OUT, bool TWO, int MI, int NJ, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void product(ProductArgs p) {
  constexpr int W = WM * WN, BM = 16 * MI * WM, BN = 16 * NJ * WN, ES = sizeof(T), STEP = 64 / ES;
  constexpr bool PAIR = kPair<OUT>;
  // fp32, 32 features: a block of 64 rows is both products', lanes c < 8 hold the first one's features 4 c + i, others the
  // second one's.
  constexpr bool NARROW = PAIR && ES == 4 && MI == 4;
  using LA = Loader<T, A_INNER, BM, PAIR ? 2 : 1, W>;
  using LB = Loader<T, B_INNER, BN, 1, W>;
  // fp32, k outside: a quarter of k is done with behind its products, so that the next step's takes its registers and two
  // waves of both products fit a SIMD: 1024-4096-1024 x 16,384 2025 us for 2279, 333-1001 x 5,003 101 for 118.
  constexpr bool SINGLE = ES == 4 && !A_INNER && !B_INNER;
  constexpr int kSlots = SINGLE ? 3 : 4, SLOT = LA::BYTES + LB::BYTES, REQ = LA::REQUESTS + LB::REQUESTS;
  static_assert(NJ % 4 == 0 && (ES == 2 || NJ == 4) && MI % (PAIR && ES == 4 && !NARROW ? 8 : 4) == 0 &&
                    !(PAIR && A_INNER) && (!NARROW || WM == 1), "blocks of 64");
  __shared__ __attribute__((aligned(1024))) char lds[kSlots * SLOT];
  int const lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const wm = wave / WN, wn = wave % WN;
  // The tile: each XCD (workgroups go to the eight in turn) takes consecutive ones, of groups of
  // kGroup columns of tiles, column by column within a row of tiles of the group.
  int64_t const total = int64_t(p.m_tiles) * p.n_tiles, all = total * p.parts;
  int64_t const q = all / 8, rest = all % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
  if (at >= q + (xcd < rest ? 1 : 0)) return;
  int64_t const index = xcd * q + (xcd < rest ? xcd : rest) + at;
  int const part = int(index / total);
  int const tile = int(index % total), group = tile / (kGroup * p.m_tiles) * kGroup;
  int const wide = p.n_tiles - group < kGroup ? p.n_tiles - group : kGroup, within = tile - group * p.m_tiles;
  int const mt = within / wide, nt = group + within % wide;
  // The second array of a pair of problems side by side in n.
  int const second = p.split_n > 0 && nt >= p.split_n ? 1 : 0;
  constexpr int FEATURES = PAIR ? BM / 2 : BM;  // rows of C of a tile
  int64_t const m0 = int64_t(mt) * FEATURES, n0 = int64_t(nt - (second ? p.split_n : 0)) * BN;
  int const steps_each = p.steps, all_steps = (TWO ? 2 : 1) * steps_each;
  int const first_step = int(int64_t(all_steps) * part / p.parts), end = int(int64_t(all_steps) * (part + 1) / p.parts);
  unsigned const lds0 = static_cast<unsigned>(reinterpret_cast<uint64_t>((lds_void)lds));

  LA la;
  LB lb;
  la.init(wave, lane, p.a[0], m0);
  lb.init(wave, lane, p.b[second], n0);
  // The next step that is asked for.
  int next = first_step;
  int const term = TWO && next >= steps_each ? 1 : 0;
  int64_t const k0 = int64_t(next - term * steps_each) * STEP;
  la.seek(wave, p.a + term, m0, k0, p.k);
  lb.seek(wave, p.b + (second | term), n0, k0, p.k);
  uint64_t const on_a = TWO ? uniform64(uint64_t(p.a[1].p) - uint64_t(p.a[0].p)) : 0,
                 on_b = TWO ? uniform64(uint64_t(p.b[1].p) - uint64_t(p.b[0].p)) : 0;
  auto request = [&](int r) __attribute__((always_inline)) {
    unsigned const slot = lds0 + unsigned(next - first_step) % kSlots * SLOT;
    if (r < LA::REQUESTS) la.request(r, wave, slot);
    else lb.request(r - LA::REQUESTS, wave, slot + LA::BYTES);
    if (r == REQ - 1) {
      next++;
      la.advance();
      lb.advance();
      if constexpr (TWO) {
        bool const now = next == steps_each;
        la.jump(now, on_a, steps_each, p.k);
        lb.jump(now, on_b, steps_each, p.k);
      }
    }
  };
  constexpr int HALF = PAIR ? MI / 2 : MI;  // fragments of a panel
  unsigned const read_a = LA::read_base(wm * 16 * HALF, lane), read_b = LB::read_base(wn * 16 * NJ, lane);
  f32x4 acc[MI][NJ] = {};
  i32x4 av[SINGLE ? 1 : 2][MI], bv[SINGLE ? 1 : 2][NJ];
  auto read = [&](int step, auto at_set, int r) __attribute__((always_inline)) {
    constexpr int set = SINGLE ? 0 : decltype(at_set)::value;
    char const* slot = lds + unsigned(step - first_step) % kSlots * SLOT;
    if (r < MI) {
      int const panel = NARROW ? 0 : r / HALF;
      read_fragment<T, A_INNER, LA::ROW, MI>(slot + panel * LA::PANEL * 64, read_a, NARROW ? r : r % HALF, av[set], r);
    } else {
      read_fragment<T, B_INNER, LB::ROW, NJ>(slot + LA::BYTES, read_b, r - MI, bv[set], r - MI);
    }
  };
  constexpr int READS = MI + NJ;
  using First = std::integral_constant<int, 0>;
  using Second = std::integral_constant<int, 1>;
  auto multiply = [&](int step, auto at_set, auto whole) __attribute__((always_inline)) {
    constexpr int set = SINGLE ? 0 : decltype(at_set)::value;
    constexpr bool WHOLE = decltype(whole)::value;  // a step kSlots on
    if constexpr (A_INNER || B_INNER) {
      int64_t const left = p.k - int64_t(TWO && step >= steps_each ? step - steps_each : step) * STEP;
      if (left < STEP && left % (16 / ES) != 0) {
#pragma unroll
        for (int i = 0; i < MI; i++) clear_past<T, A_INNER>(av[set][i], lane, left);
#pragma unroll
        for (int j = 0; j < NJ; j++) clear_past<T, B_INNER>(bv[set][j], lane, left);
      }
    }
    // Requests and reads stand between the products of 16 bits; where one side has k inside, before them.  bf16
    // 1024 x 4096 x 16,384: 108 us between, 118 before; with k inside 258 and 253, in fp32 no difference.
    constexpr bool BETWEEN = ES == 2 && !A_INNER;
    // fp32: a sum's four products stand all others apart.
    constexpr int SLOTS = kMfmaParts<T> * MI;
#pragma unroll
    for (int q = 0; q < NJ; q++) {
      int const r0 = q * REQ / NJ, requests = (q + 1) * REQ / NJ - r0;
      int const f0 = q * READS / NJ, events = requests + (SINGLE ? 0 : (q + 1) * READS / NJ - f0);
#pragma unroll
      for (int t = 0; t < SLOTS; t++) {
#pragma unroll
        for (int n = 0; n < events; n++) {
          if ((BETWEEN ? n * SLOTS / events : 0) != t) continue;
          if (n < requests) {
            if (WHOLE || step + kSlots < end) request(r0 + n);
          } else {
            if (WHOLE || step + 1 < end) read(step + 1, std::integral_constant<int, 1 - set>{}, f0 + n - requests);
          }
        }
        int const i = t % MI, j = ES == 4 ? t / MI : q, e = ES == 4 ? q : 0;
        acc[i][j] = mfma_part<T>(fragment<T, B_INNER>(bv[set], j, e), fragment<T, A_INNER>(av[set], i, e), acc[i][j], e);
        if (BETWEEN || t == SLOTS - 1) __builtin_amdgcn_sched_barrier(0);
      }
      if (SINGLE && (WHOLE || step + 1 < end)) {
#pragma unroll
        for (int r = q; r < READS; r += 4) read(step + 1, First{}, r);
      }
    }
  };
  // This step's fragments are in registers and the next step's data has landed, for every wave: this
  // step's slot takes the step kSlots on.
  auto turn = [&](int step, auto set, auto whole) __attribute__((always_inline)) {
    if (decltype(whole)::value || step + kSlots - 1 < end) wait_requests<(kSlots - 2) * REQ>();
    else wait_requests<0>();
    workgroup_barrier();
    multiply(step, set, whole);
  };
#pragma unroll
  for (int s = 0; s < kSlots; s++)
    if (first_step + s < end)
#pragma unroll
      for (int r = 0; r < REQ; r++) request(r);
  if (first_step + kSlots <= end) wait_requests<(kSlots - 1) * REQ>();
  else wait_requests<0>();
  workgroup_barrier();
#pragma unroll
  for (int r = 0; r < READS; r++) read(first_step, First{}, r);
  int step = first_step;
  for (; step + 1 + kSlots < end; step += 2) {
    turn(step, First{}, std::true_type{});
    turn(step + 1, Second{}, std::true_type{});
  }
  for (; step < end; step += 2) {
    turn(step, First{}, std::false_type{});
    if (step + 1 < end) turn(step + 1, Second{}, std::false_type{});
  }

  // Rows: of fragments of k outside in fp32 the four of a block of 64 are dealt one by one.
  auto row_of = [&](int i) {
    if constexpr (NARROW) return m0 + 4 * (c % 8) + c / 8 * HALF + i;
    int const base = wm * 16 * HALF;
    return m0 + base + (ES == 4 && !A_INNER ? i / 4 * 64 + 4 * c + i % 4 : 16 * i + c);
  };
  T* const y = static_cast<T*>(p.y[second]);
#pragma unroll
  for (int i = 0; i < HALF; i++) {
    int64_t const m = row_of(i);
#pragma unroll
    for (int b = 0; b < NJ / 4; b++) {
      auto columns = [&](int row, float (&v)[16]) __attribute__((always_inline)) {
        f32x4 w[4] = {acc[row][4 * b], acc[row][4 * b + 1], acc[row][4 * b + 2], acc[row][4 * b + 3]};
        if constexpr (ES == 4 && !B_INNER) {
#pragma unroll
          for (int e = 0; e < 16; e++) v[e] = w[e % 4][e / 4];
        } else {
          exchange(w);
#pragma unroll
          for (int e = 0; e < 16; e++) v[e] = w[e / 4][e % 4];
        }
      };
      int64_t const n = n0 + (wn * NJ + 4 * b) * 16 + 16 * g, left = p.columns - n;
      float v[16], u[16];
      columns(i, v);
      if constexpr (PAIR) columns(i + HALF, u);
      if constexpr (NARROW) {
        // Lanes c < 8 have features 4 c + i and 4 c + i + 2 of the first product, lanes c + 8 of the second: each takes both
        // of one feature.
        bool const first = c < 8;
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float const other = __shfl_xor(first ? u[e] : v[e], 8);
          u[e] = first ? other : u[e];
          v[e] = first ? v[e] : other;
        }
      }
      if (m >= p.rows || left <= 0) continue;
      if constexpr (OUT == OUT_PAIR_PARTS) {
        float* at = p.sums + (int64_t(part) * p.rows + m) * p.ld_sums + n;
        store16<float>(at, left, v);
        store16<float>(at + int64_t(p.parts) * p.rows * p.ld_sums, left, u);
        continue;
      }
      if constexpr (OUT == OUT_PARTS) {
        float* at = p.sums + ((int64_t(part) * p.problems + second) * p.rows + m) * p.ld_sums + n;
        store16<float>(at, left, v);
        continue;
      }
      if constexpr (OUT == OUT_PLAIN || PAIR) {
        float const bias = p.bias[0] != nullptr ? float(static_cast<T const*>(p.bias[0])[m]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] += bias;
      }
      if constexpr (PAIR) {
        float const bias = p.bias[1] != nullptr ? float(static_cast<T const*>(p.bias[1])[m]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) u[e] += bias;
        if (p.states != nullptr) {
          T* const s = static_cast<T*>(p.states) + m * p.ld_states + n;
          store16<T>(s, left, v);
          store16<T>(s + p.rows * p.ld_states, left, u);
        }
        with_activation<sizeof(T) == 4>(p.act, p.slope, [&](auto f) {
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float a, d;
            f(v[e], a, d);
            v[e] = a * u[e];
          }
        });
      }
      if constexpr (OUT == OUT_STATES) {
        T const* const s = static_cast<T const*>(p.states) + m * p.ld_states + n;
        float gate[16];
        load16<T>(s, left, gate);
        load16<T>(s + p.rows * p.ld_states, left, u);
        with_activation<sizeof(T) == 4>(p.act, p.slope, [&](auto f) {
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float a, d;
            f(gate[e], a, d);
            u[e] *= v[e] * d;
            v[e] *= a;
          }
        });
        store16<T>(y + m * p.ld[0] + n, left, u);
        store16<T>(static_cast<T*>(p.y[1]) + m * p.ld[0] + n, left, v);
      } else {
        store16<T>(y + m * p.ld[second] + n, left, v);
      }
    }
  }
}

// The parts of C in their order.
template <class T> __global__ __launch_bounds__(256) void join_parts(ProductArgs p) {
  int64_t const n = (int64_t(blockIdx.y) * 256 + threadIdx.x) * 4, m = blockIdx.x;
  int const second = blockIdx.z;
  if (n >= p.columns) return;
  f32x4 s = {0, 0, 0, 0};
#pragma unroll 8
  for (int k = 0; k < p.parts; k++)
    s += *reinterpret_cast<f32x4 const*>(p.sums + ((int64_t(k) * p.problems + second) * p.rows + m) * p.ld_sums + n);
  if (p.bias[0] != nullptr) s += float(static_cast<T const*>(p.bias[0])[m]);
  Pack<T, 4> o;
#pragma unroll
  for (int e = 0; e < 4; e++) o.set(e, s[e]);
  o.store(static_cast<T*>(p.y[second]) + m * p.ld[second] + n, p.columns - n < 4 ? int(p.columns - n) : 4);
}

// Four columns of a row of the parts' sum; grid (rows, columns / 1024).
__device__ inline f32x4 sum_of_parts(ProductArgs const& p, float const* sums, int64_t m, int64_t n) {
  f32x4 s = {0, 0, 0, 0};
#pragma unroll 8
  for (int k = 0; k < p.parts; k++) s += *reinterpret_cast<f32x4 const*>(sums + (int64_t(k) * p.rows + m) * p.ld_sums + n);
  return s;
}
// OUT_PAIR's outputs from the parts of the first product, then of the second.
template <class T> __global__ __launch_bounds__(256) void join_pair(ProductArgs p) {
  int64_t const n = (int64_t(blockIdx.y) * 256 + threadIdx.x) * 4, m = blockIdx.x;
  if (n >= p.columns) return;
  int const count = p.columns - n < 4 ? int(p.columns - n) : 4;
  f32x4 v = sum_of_parts(p, p.sums, m, n), u = sum_of_parts(p, p.sums + p.parts * p.rows * p.ld_sums, m, n);
  if (p.bias[0] != nullptr) v += float(static_cast<T const*>(p.bias[0])[m]);
  if (p.bias[1] != nullptr) u += float(static_cast<T const*>(p.bias[1])[m]);
  Pack<T, 4> o;
  auto store = [&](f32x4 const& w, void* to, int64_t ld, int64_t row) {
#pragma unroll
    for (int e = 0; e < 4; e++) o.set(e, w[e]);
    o.store(static_cast<T*>(to) + row * ld + n, count);
  };
  if (p.states != nullptr) {
    store(v, p.states, p.ld_states, m);
    store(u, p.states, p.ld_states, p.rows + m);
  }
  with_activation<sizeof(T) == 4>(p.act, p.slope, [&](auto f) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a, d;
      f(v[e], a, d);
      v[e] = a * u[e];
    }
  });
  store(v, p.y[0], p.ld[0], m);
}
// OUT_STATES' outputs from the parts.
template <class T> __global__ __launch_bounds__(256) void join_states(ProductArgs p) {
  int64_t const n = (int64_t(blockIdx.y) * 256 + threadIdx.x) * 4, m = blockIdx.x;
  if (n >= p.columns) return;
  int const count = p.columns - n < 4 ? int(p.columns - n) : 4;
  f32x4 v = sum_of_parts(p, p.sums, m, n);
  T const* const s = static_cast<T const*>(p.states) + m * p.ld_states + n;
  Pack<T, 4> gate, up, dg, du;
  gate.load(s, count, 0.0f);
  up.load(s + p.rows * p.ld_states, count, 0.0f);
  with_activation<sizeof(T) == 4>(p.act, p.slope, [&](auto f) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a, d;
      f(gate[e], a, d);
      dg.set(e, up[e] * (v[e] * d));
      du.set(e, v[e] * a);
    }
  });
  dg.store(static_cast<T*>(p.y[0]) + m * p.ld[0] + n, count);
  du.store(static_cast<T*>(p.y[1]) + m * p.ld[0] + n, count);
}

template <class T, bool A_INNER, bool B_INNER, Output OUT, bool TWO, int MI, int NJ, int WM, int WN>
hipError_t launch_tiles(ProductArgs p, hipStream_t stream) {
  constexpr int BM = 16 * MI * WM / (kPair<OUT> ? 2 : 1), BN = 16 * NJ * WN, STEP = 64 / sizeof(T);
  int64_t const m_tiles = (p.rows + BM - 1) / BM, n_tiles = (p.columns + BN - 1) / BN * p.problems;
  p.m_tiles = int(m_tiles), p.n_tiles = int(n_tiles);
  p.split_n = p.problems == 2 ? p.n_tiles / 2 : 0;
  p.steps = int((p.k + STEP - 1) / STEP);
  int64_t const groups = (m_tiles * n_tiles * p.parts + 7) / 8 * 8;
  if (groups > int64_t(UINT32_MAX) / (64 * WM * WN)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((product<T, A_INNER, B_INNER, OUT, TWO, MI, NJ, WM, WN>), dim3(unsigned(groups)), dim3(64 * WM * WN), 0, stream, p);
  return hipGetLastError();
}

template <class T, bool A_INNER, bool B_INNER, Output OUT, bool TWO = false> hipError_t launch_sized(Tile tile, ProductArgs const& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 4)
    if (tile == TILE_NARROW) return launch_tiles<T, A_INNER, B_INNER, OUT, TWO, 4, 4, 1, 4>(p, stream);
  if constexpr (sizeof(T) == 2)
    if (tile == TILE_LARGE) return launch_tiles<T, A_INNER, B_INNER, OUT, TWO, 8, 4, 2, 4>(p, stream);
  if constexpr (sizeof(T) == 4 && OUT == OUT_PAIR) return launch_tiles<T, A_INNER, B_INNER, OUT, TWO, 8, 4, 2, 2>(p, stream);
  else return launch_tiles<T, A_INNER, B_INNER, OUT, TWO, 4, 4, 2, 2>(p, stream);
}

template <class T, bool A_INNER, bool B_INNER, bool TWO = false> hipError_t launch_plain(Tile tile, ProductArgs const& p, hipStream_t stream) {
  if (p.parts == 1) return launch_sized<T, A_INNER, B_INNER, OUT_PLAIN, TWO>(tile, p, stream);
  hipError_t const err = launch_sized<T, A_INNER, B_INNER, OUT_PARTS, TWO>(tile, p, stream);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(join_parts<T>, dim3(unsigned(p.rows), unsigned((p.columns + 1023) / 1024), unsigned(p.problems)), dim3(256),
                     0, stream, p);
  return hipGetLastError();
}

// The first products of few tiles, cut along k, of wide tiles one after the other (choose_pair); then the one of D dy.
template <class T> hipError_t launch_pair_in_parts(Tile tile, ProductArgs const& p, hipStream_t stream) {
  hipError_t err = hipSuccess;
  bool const together = sizeof(T) == 4 && p.pair_parts;
  if constexpr (sizeof(T) == 4)
    if (together) err = launch_tiles<T, false, false, OUT_PAIR_PARTS, false, 4, 4, 1, 4>(p, stream);
  for (int q = 0; q < 2 && !together && err == hipSuccess; q++) {
    ProductArgs one = p;
    one.a[0] = p.a[q];
    one.sums = p.sums + q * p.parts * p.rows * p.ld_sums;
    err = launch_sized<T, false, false, OUT_PARTS>(tile, one, stream);
  }
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(join_pair<T>, dim3(unsigned(p.rows), unsigned((p.columns + 1023) / 1024)), dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <class T> hipError_t launch_states_in_parts(Tile tile, ProductArgs const& p, hipStream_t stream) {
  hipError_t const err = launch_sized<T, true, false, OUT_PARTS>(tile, p, stream);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(join_states<T>, dim3(unsigned(p.rows), unsigned((p.columns + 1023) / 1024)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <class T> hipError_t launch_product_as(Form form, Tile tile, ProductArgs const& p, hipStream_t stream) {
  switch (form) {
    case FORM_PAIR:
      if (p.parts > 1) return launch_pair_in_parts<T>(tile, p, stream);
      return launch_sized<T, false, false, OUT_PAIR>(tile, p, stream);
    case FORM_STATES:
      if (p.parts > 1) return launch_states_in_parts<T>(tile, p, stream);
      return launch_sized<T, true, false, OUT_STATES>(tile, p, stream);
    case FORM_FORWARD: return launch_plain<T, false, false>(tile, p, stream);
    case FORM_INPUT: return launch_plain<T, true, false, true>(tile, p, stream);
    default: return launch_plain<T, true, true>(tile, p, stream);
  }
}

}  // namespace
}  // namespace ponni_hip
