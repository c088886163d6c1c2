// Device code that the kernels of expert layers share (kernels_experts.hip,
// kernels_chain_*.hip): MFMAs on fragments, groups and tiles, epilogues.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "activations.h"
#include "experts.h"
#include "operand_types.h"
#include "program.h"

namespace ponni_hip {
namespace {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// acc += A B for one step's fragments of a 16 x 16 tile.  mx4: a_scale holds the
// scales of the 4 tiles of a block (TILE picks its byte), b_scale the column's in its first byte.
template <Operand OP, int TILE>
__device__ inline f32x4 multiply(i32x4 a, i32x4 b, f32x4 acc, int a_scale, int b_scale) {
  if constexpr (OP == OPERAND_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), acc, 0, 0, 0);
  } else if constexpr (OP == OPERAND_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), acc, 0, 0, 0);
  } else if constexpr (OP == OPERAND_MX4) {
    i32x8 const a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, acc, 4, 4, TILE, a_scale, 0, b_scale);
  } else {
    f32x4 const af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], bf[e], acc, 0, 0, 0);
    return acc;
  }
}

// A pointer that every lane of the wave holds, in scalar registers.
__device__ inline char const* uniform(char const* p) {
  uint64_t const v = reinterpret_cast<uint64_t>(p);
  uint64_t const lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v)) & 0xffffffffu;
  uint64_t const hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
  return reinterpret_cast<char const*>(hi << 32 | lo);
}

// Columns of an expert's group, from offsets that a caller's program wrote:
// whatever they hold, a group lies within [0, columns).
struct Group {
  int32_t first, last;
};
__device__ inline Group group_of(int32_t const* offsets, int expert, int32_t columns) {
  auto clamp = [&](int32_t v) { return v < 0 ? 0 : v > columns ? columns : v; };
  if (offsets == nullptr) return {0, columns};
  int32_t const a = clamp(offsets[expert]), b = clamp(offsets[expert + 1]);
  return {a, b < a ? a : b};
}

struct Tile {
  int expert;
  int32_t first, last;  // columns [first, last), at most the tile's width
  int block;            // of output features
  bool none;
};

// This workgroup's tile.  Every group has ceil(columns / width) column tiles; the
// grid holds as many as any offsets can give.  Each XCD (workgroups go to the
// eight in turn) takes a contiguous share of the tiles, which go by GROUP column tiles
// and, within those, by output block: rows are read into one L2 only, an expert's weights by few,
// and the 32 tiles that an XCD has at a time share both (8 x 4 tiles read 12 parts of
// a step where 2 x 16 read 18).
template <int WIDTH, int GROUP = 8>
__device__ inline Tile find_tile(ContractArgs const& a, int out_blocks) {
  int const lane = threadIdx.x & 63;
  int32_t const columns = static_cast<int32_t>(a.columns);
  auto tiles = [&](int base) {
    if (base + lane >= a.experts) return 0;
    Group const g = group_of(a.offsets, base + lane, columns);
    return int((int64_t(g.last) - g.first + WIDTH - 1) / WIDTH);
  };
  auto scan = [&](int n) {  // inclusive, over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      int const t = __shfl_up(n, d);
      n += lane >= d ? t : 0;
    }
    return n;
  };
  int64_t total = 0;
  for (int base = 0; base < a.experts; base += 64) total += __shfl(scan(tiles(base)), 63);
  int64_t const column_tiles = total;
  total *= out_blocks;
  int64_t const q = total / 8, r = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
  Tile t{};
  t.none = true;
  if (at >= q + (xcd < r ? 1 : 0)) return t;
  int64_t const index = xcd * q + (xcd < r ? xcd : r) + at;
  int64_t const group = index / (int64_t(GROUP) * out_blocks) * GROUP, rest = column_tiles - group;
  int const wide = rest < GROUP ? static_cast<int>(rest) : GROUP, within_group = static_cast<int>(index - group * out_blocks);
  int column_tile = static_cast<int>(group) + within_group % wide;
  t.block = __builtin_amdgcn_readfirstlane(within_group / wide);
  for (int base = 0; base < a.experts; base += 64) {
    int const n = tiles(base), end = scan(n);
    int const all = __shfl(end, 63);
    if (column_tile < all) {
      int const l = __builtin_ctzll(__ballot(column_tile < end));
      t.expert = __builtin_amdgcn_readfirstlane(base + l);
      int const within = __builtin_amdgcn_readfirstlane(column_tile - (__shfl(end, l) - __shfl(n, l)));
      Group const g = group_of(a.offsets, t.expert, columns);
      t.first = __builtin_amdgcn_readfirstlane(g.first + within * WIDTH);
      t.last = __builtin_amdgcn_readfirstlane(g.last - t.first < WIDTH ? g.last : t.first + WIDTH);
      t.none = false;
      return t;
    }
    column_tile -= all;
  }
  return t;
}

// CHAIN: without GELU's exact form, the longest.
template <bool Precise, bool CHAIN = false, class Each>
__device__ inline void activate(int act, float slope, Each&& each) {
  switch (act) {
    case ACT_RELU: each([](float v) { return act_relu(v); }); break;
    case ACT_LEAKY_RELU: each([slope](float v) { return act_leaky_relu(v, slope); }); break;
    case ACT_TANH: each([](float v) { return Precise ? tanh_f32(v) : tanh_half(v); }); break;
    case ACT_SIGMOID: each([](float v) { return Precise ? sigmoid_f32(v) : act_sigmoid_fast(v); }); break;
    case ACT_SILU: each([](float v) { return Precise ? silu_f32(v) : act_silu_fast(v); }); break;
    case ACT_GELU_TANH: each([](float v) { return Precise ? gelu_tanh_f32(v) : act_gelu_tanh_fast(v); }); break;
    case ACT_GELU_ERF:
      if constexpr (!CHAIN) each([](float v) { return act_gelu_erf(v); });
      break;
    default: break;
  }
}

// Features past the last one are zero: their weights are, but not those times an
// infinity, nor sigmoid(0).  (16 features from f0 on, of the block of 64 that begins at
// `block`; whole blocks, which the compiler would check feature by feature, need no check.)
__device__ inline void clear_past(f32x4 (&v)[4], int block, int f0, int n_out) {
  if (block + 64 <= n_out) return;
#pragma unroll
  for (int e = 0; e < 16; e++) v[e / 4][e % 4] = f0 + e < n_out ? v[e / 4][e % 4] : 0.0f;
}

// 16 consecutive features from feature f0 on of a row in pieces of 16 bytes (zero past the
// last feature, none past row_features).
template <class S> __device__ inline void write_pieces(char* row, int f0, int row_features, f32x4 (&v)[4]) {
  constexpr int N = 16 / sizeof(S);
  typedef S Piece __attribute__((ext_vector_type(N)));
#pragma unroll
  for (int p = 0; p < 16 / N; p++) {
    Piece o;
#pragma unroll
    for (int e = 0; e < N; e++) o[e] = S(v[(p * N + e) / 4][(p * N + e) % 4]);
    if (f0 + p * N < row_features) *reinterpret_cast<Piece*>(row + (f0 + p * N) * sizeof(S)) = o;
  }
}

// The same of column `col` of the output.
template <OutputKind KIND, class S>
__device__ inline void store_features(ContractArgs const& a, int64_t col, int f0, f32x4 (&v)[4], int n_out) {
  if constexpr (KIND == OUT_FEATURES) {
    S* y = static_cast<S*>(a.y) + int64_t(f0) * a.ldy + col;
    if (f0 + 16 <= n_out) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        *y = S(v[e / 4][e % 4]);
        y += a.ldy;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 15; e++) {
        if (f0 + e < n_out) *y = S(v[e / 4][e % 4]);
        y += a.ldy;
      }
    }
  } else if constexpr (KIND == OUT_FLOATS) {
    int const block = f0 / 64 * 64, groups = float_groups(block, a.row_features);
    float* row = reinterpret_cast<float*>(a.y_rows.data + col * a.y_rows.stride) + block;
    if (f0 < a.row_features)
#pragma unroll
      for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(row + float_place(f0 % 64 / 16, i, groups)) = v[i];
  } else {
    write_pieces<S>(a.y_rows.data + col * a.y_rows.stride, f0, a.row_features, v);
  }
}

// The same as half a block of 32: lanes 16 apart hold its two halves.
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ inline void write_mx4(f32x4 (&v)[4], bool valid, i32x2* codes_at, bool with_scale, unsigned char* scale_at) {
  float amax = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      amax = fmaxf(amax, __builtin_fabsf(v[i][e]));
      finite = finite && v[i][e] == v[i][e];
    }
  if (!finite) amax = __builtin_inff();
  amax = fmaxf(amax, __shfl_xor(amax, 16));
  unsigned const scale = mx4_scale(amax);
  float const scale_value = mx4_scale_value(scale);
  i32x2 codes;
#pragma unroll
  for (int w = 0; w < 2; w++) codes[w] = mx4_word(scale_value, [&](int e) { return v[2 * w + e / 4][e % 4]; });
  if (scale == 255u) codes = {0, 0};
  if (!valid) return;
  *codes_at = codes;
  if (with_scale) *scale_at = static_cast<unsigned char>(scale);
}
__device__ inline void store_mx4(ContractArgs const& a, int64_t col, bool valid, int f0, f32x4 (&v)[4]) {
  write_mx4(v, valid && f0 < a.row_features, reinterpret_cast<i32x2*>(a.y_rows.data + col * a.y_rows.stride + f0 / 2),
            f0 % kMx4Block == 0,
            a.y_rows.scales + col * a.y_rows.scale_stride + f0 / 128 * a.y_rows.scale_step + f0 / kMx4Block % 4);
}

// Fragment `piece` of an input row as the caller holds it ([features, x_rows]), and its scale.
template <Operand OP, class S>
__device__ inline void read_features(ContractArgs const& a, int64_t row, int piece, i32x4& v, int& scale) {
  constexpr int N = OP == OPERAND_F32 ? 4 : OP == OPERAND_MX4 ? 32 : 8;
  S const* x = static_cast<S const*>(a.features) + row;
  S e[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    int const f = piece * N + k;
    e[k] = f < a.n_in ? x[f * a.ldx] : S(0.0f);
  }
  if constexpr (OP == OPERAND_MX4) {
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int k = 0; k < N; k++) {
      amax = fmaxf(amax, __builtin_fabsf(float(e[k])));
      finite = finite && e[k] == e[k];
    }
    scale = finite ? mx4_scale(amax) : 255u;
    float const scale_value = mx4_scale_value(scale);
#pragma unroll
    for (int w = 0; w < 4; w++) v[w] = mx4_word(scale_value, [&](int k) { return e[8 * w + k]; });
    if (scale == 255) v = {0, 0, 0, 0};
  } else {
    typedef S Piece __attribute__((ext_vector_type(N)));
    Piece p;
#pragma unroll
    for (int k = 0; k < N; k++) p[k] = e[k];
    v = __builtin_bit_cast(i32x4, p);
  }
}

// The grid of tiles of `width` columns x `out_blocks` blocks, at least as many as any offsets give.
inline int64_t grid_of(ContractArgs const& a, int64_t width, int64_t out_blocks) {
  // ceil(n / width) summed over the groups: at most one more than n / width for each that has columns
  int64_t const partial = a.experts < a.columns ? a.experts : a.columns;
  // (a share per XCD is rounded up: the grid is whole rounds of the eight)
  return ((a.columns / width + partial) * out_blocks + 7) / 8 * 8;
}
// A launch's threads are counted in 32 bits: a grid of more is cut off, without an error.
inline bool launchable(int64_t workgroups, int threads) { return workgroups <= int64_t(UINT32_MAX) / threads; }

}  // namespace
}  // namespace ponni_hip
