// Rows of samples from [features, columns] arrays, in 16 and 32 bits or
// quantised to 4-bit blocks, and the values of 4-bit rows.
#include <hip/hip_runtime.h>

#include "experts.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

// A workgroup's tile: 128 columns of 128 bytes of their rows (64 bytes, 4 blocks, of
// 4-bit rows).  A lane loads two columns' features, as one word where rows allow
// it (PAIR: columns 2 l and 2 l + 1, else l and l + 64), puts whole pieces of
// 16 bytes together and turns the tile in LDS, so that rows are written in whole lines.
constexpr int kTileColumns = 128;
template <bool PAIR> __device__ inline int column_of(int lane, int i) { return PAIR ? 2 * lane + i : lane + 64 * i; }
// Where a column's piece lies in the tile: 16 consecutive columns' in different banks.
__device__ inline int place(int column, int piece, int pieces) { return column * pieces + (piece ^ (column >> 1) % pieces); }

// Two columns' features f (16 bits: in the low and high half).
template <class S, bool PAIR>
__device__ inline auto load_two(S const* __restrict__ x, int64_t ld, int64_t f, int64_t features, int64_t col0,
                                int64_t columns, int lane) {
  typedef S S2 __attribute__((ext_vector_type(2)));
  S2 v = {S(0.0f), S(0.0f)};
  if (f < features) {
    S const* row = x + f * ld + col0;
    if (PAIR && col0 + 2 * lane + 1 < columns) {
      v = *reinterpret_cast<S2 const*>(row + 2 * lane);
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (col0 + column_of<PAIR>(lane, i) < columns) v[i] = row[column_of<PAIR>(lane, i)];
    }
  }
  return v;
}

// [features, columns] to rows, 128 columns x 128 bytes of features a workgroup: read by
// whole lines, turned in LDS, written by whole lines.  Bound by bytes: 1024 bf16
// features, 65,536 columns: 47-51 us, 5.3 TB/s.
template <class S, bool PAIR>
__global__ __launch_bounds__(256) void to_rows(S const* __restrict__ x, int64_t ld, int64_t features, int64_t columns,
                                               Rows rows) {
  constexpr int N = 16 / sizeof(S);
  typedef S Piece __attribute__((ext_vector_type(N)));
  __shared__ Piece tile[kTileColumns * 8];
  int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t const col0 = int64_t(blockIdx.x) * kTileColumns, piece0 = int64_t(blockIdx.y) * 8;
#pragma unroll
  for (int q = 0; q < 2; q++) {
    int const piece = 2 * wave + q;
    Piece v[2];
#pragma unroll
    for (int e = 0; e < N; e++) {
      auto const two = load_two<S, PAIR>(x, ld, (piece0 + piece) * N + e, features, col0, columns, lane);
      v[0][e] = two[0];
      v[1][e] = two[1];
    }
#pragma unroll
    for (int i = 0; i < 2; i++) tile[place(column_of<PAIR>(lane, i), piece, 8)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; q++) {
    int const p = threadIdx.x + 256 * q, col = p / 8, piece = p % 8;
    int64_t const at = (piece0 + piece) * 16;
    if (col0 + col < columns && at < rows.stride)
      *reinterpret_cast<Piece*>(rows.data + (col0 + col) * rows.stride + at) = tile[place(col, piece, 8)];
  }
}

// One wave per block of 32 features; the largest magnitude of 16-bit numbers is that of their bits.
// Bound by bytes: 1024 bf16 features, 262,144 columns: 183 us, 3.7 TB/s.
template <class S, bool PAIR>
__global__ __launch_bounds__(256) void to_mx4(S const* __restrict__ x, int64_t ld, int64_t features, int64_t columns,
                                              Rows rows) {
  __shared__ i32x4 tile[kTileColumns * 4];
  __shared__ unsigned char scales[kTileColumns][4];
  int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t const col0 = int64_t(blockIdx.x) * kTileColumns, f0 = int64_t(blockIdx.y) * 128 + 32 * wave;
  typedef S S2 __attribute__((ext_vector_type(2)));
  S2 v[kMx4Block];
#pragma unroll
  for (int f = 0; f < kMx4Block; f++) v[f] = load_two<S, PAIR>(x, ld, f0 + f, features, col0, columns, lane);
  unsigned largest[2];
  if constexpr (sizeof(S) == 2) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int f = 0; f < kMx4Block; f++) {
      u16x2 const a = __builtin_bit_cast(u16x2, __builtin_bit_cast(unsigned, v[f]) & 0x7fff7fffu);
      m = __builtin_elementwise_max(m, a);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float const a = float(__builtin_bit_cast(S, static_cast<unsigned short>(m[i])));
      largest[i] = __builtin_bit_cast(unsigned, a);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      largest[i] = 0;
#pragma unroll
      for (int f = 0; f < kMx4Block; f++) {
        float const t = v[f][i];  // (the builtin below takes a vector's first element for any of its elements)
        unsigned const a = __builtin_bit_cast(unsigned, t) & 0x7fffffffu;
        largest[i] = a > largest[i] ? a : largest[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int const col = column_of<PAIR>(lane, i);
    unsigned const scale = mx4_scale(__builtin_bit_cast(float, largest[i]));
    float const scale_value = mx4_scale_value(scale);
    i32x4 codes;
#pragma unroll
    for (int w = 0; w < 4; w++) codes[w] = mx4_word(scale_value, [&](int e) { return S(v[8 * w + e][i]); });
    tile[place(col, wave, 4)] = scale == 255u ? i32x4{0, 0, 0, 0} : codes;
    scales[col][wave] = static_cast<unsigned char>(scale);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; q++) {
    int const p = threadIdx.x + 256 * q, col = p / 4, piece = p % 4;
    if (col0 + col < columns)
      *reinterpret_cast<i32x4*>(rows.data + (col0 + col) * rows.stride + int64_t(blockIdx.y) * 64 + piece * 16) =
          tile[place(col, piece, 4)];
  }
  if (threadIdx.x < kTileColumns && col0 + threadIdx.x < columns)
    *reinterpret_cast<int*>(rows.scales + (col0 + threadIdx.x) * rows.scale_stride + blockIdx.y * rows.scale_step) =
        *reinterpret_cast<int const*>(scales[threadIdx.x]);
}

// The values of 4-bit rows.  Bound by bytes: 1024 bf16 features, 262,144 columns: 163 us, 4.1 TB/s.
template <class S>
__global__ __launch_bounds__(256) void mx4_values(Rows rows, int64_t features, int64_t columns, S* __restrict__ y,
                                                  int64_t ld) {
  int64_t const col = int64_t(blockIdx.x) * 64 + (threadIdx.x & 63);
  int64_t const block = int64_t(blockIdx.y) * 4 + (threadIdx.x >> 6);
  if (col >= columns || block * kMx4Block >= features) return;
  i32x4 const codes = *reinterpret_cast<i32x4 const*>(rows.data + col * rows.stride + block * 16);
  float const scale = mx4_scale_value(rows.scales[col * rows.scale_stride + block / 4 * rows.scale_step + block % 4]);
#pragma unroll
  for (int i = 0; i < kMx4Block; i++) {
    int64_t const f = block * kMx4Block + i;
    if (f < features) y[f * ld + col] = S(mx4_value((unsigned(codes[i / 8]) >> (4 * (i % 8))) & 15u) * scale);
  }
}

}  // namespace

hipError_t launch_to_rows(Operand op, int dtype, const void* x, int64_t ld, int64_t features, int64_t columns,
                          Rows const& rows, hipStream_t stream) {
  int64_t const tile_bytes = op == OPERAND_MX4 ? 64 : 128;
  dim3 const grid(unsigned((columns + kTileColumns - 1) / kTileColumns),
                  unsigned((rows.stride + tile_bytes - 1) / tile_bytes)),
      block(256);
  with_dtype(dtype, [&](auto s) {
    using S = decltype(s);
    auto const* in = static_cast<S const*>(x);
    bool const pair = (reinterpret_cast<uint64_t>(x) | uint64_t(ld) * sizeof(S)) % (2 * sizeof(S)) == 0;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, in, ld, features, columns, rows); };
    if (op == OPERAND_MX4) pair ? launch(to_mx4<S, true>) : launch(to_mx4<S, false>);
    else pair ? launch(to_rows<S, true>) : launch(to_rows<S, false>);
  });
  return hipGetLastError();
}

hipError_t launch_mx4_values(Rows const& rows, int64_t features, int64_t columns, void* y, int64_t ld, int dtype,
                             hipStream_t stream) {
  dim3 const grid(unsigned((columns + 63) / 64), unsigned((features + 127) / 128)), block(256);
  with_dtype(dtype, [&](auto s) {
    using S = decltype(s);
    hipLaunchKernelGGL(mx4_values<S>, grid, block, 0, stream, rows, features, columns, static_cast<S*>(y), ld);
  });
  return hipGetLastError();
}

}  // namespace ponni_hip
