// Rows of samples from [features, columns] arrays, in 16 and 32 bits or
// quantised to 4-bit blocks, and the values of 4-bit rows.
#include <hip/hip_runtime.h>

#include "experts.h"
#include "operand_types.h"

namespace ponni_hip {
namespace {

// One lane per column and 16-byte piece of its row.
template <class S>
__global__ __launch_bounds__(256) void to_rows(S const* __restrict__ x, int64_t ld, int64_t features, int64_t columns,
                                               Rows rows) {
  constexpr int N = 16 / sizeof(S);
  int64_t const col = int64_t(blockIdx.x) * 64 + (threadIdx.x & 63);
  int64_t const piece = int64_t(blockIdx.y) * 4 + (threadIdx.x >> 6);
  if (col >= columns || piece * 16 >= rows.stride) return;
  typedef S Piece __attribute__((ext_vector_type(N)));
  Piece v;
#pragma unroll
  for (int i = 0; i < N; i++) {
    int64_t const f = piece * N + i;
    v[i] = f < features ? x[f * ld + col] : S(0.0f);
  }
  *reinterpret_cast<Piece*>(rows.data + col * rows.stride + piece * 16) = v;
}

// One lane per column and block of 32 features.
template <class S>
__global__ __launch_bounds__(256) void to_mx4(S const* __restrict__ x, int64_t ld, int64_t features, int64_t columns,
                                              Rows rows) {
  int64_t const col = int64_t(blockIdx.x) * 64 + (threadIdx.x & 63);
  int64_t const block = int64_t(blockIdx.y) * 4 + (threadIdx.x >> 6);
  if (col >= columns || block >= rows.scale_stride) return;
  float v[kMx4Block];
  float amax = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < kMx4Block; i++) {
    int64_t const f = block * kMx4Block + i;
    v[i] = f < features ? float(x[f * ld + col]) : 0.0f;
    amax = fmaxf(amax, __builtin_fabsf(v[i]));
    finite = finite && v[i] == v[i];
  }
  unsigned const scale = finite ? mx4_scale(amax) : 255u;
  float const inverse = mx4_inverse(scale);
  i32x4 codes = {0, 0, 0, 0};
  if (scale != 255u) {
#pragma unroll
    for (int i = 0; i < kMx4Block; i++) codes[i / 8] |= mx4_code(v[i] * inverse) << (4 * (i % 8));
  }
  *reinterpret_cast<i32x4*>(rows.data + col * rows.stride + block * 16) = codes;
  rows.scales[col * rows.scale_stride + block] = static_cast<unsigned char>(scale);
}

template <class S>
__global__ __launch_bounds__(256) void mx4_values(Rows rows, int64_t features, int64_t columns, S* __restrict__ y,
                                                  int64_t ld) {
  int64_t const col = int64_t(blockIdx.x) * 64 + (threadIdx.x & 63);
  int64_t const block = int64_t(blockIdx.y) * 4 + (threadIdx.x >> 6);
  if (col >= columns || block * kMx4Block >= features) return;
  i32x4 const codes = *reinterpret_cast<i32x4 const*>(rows.data + col * rows.stride + block * 16);
  float const scale = mx4_scale_value(rows.scales[col * rows.scale_stride + block]);
#pragma unroll
  for (int i = 0; i < kMx4Block; i++) {
    int64_t const f = block * kMx4Block + i;
    if (f < features) y[f * ld + col] = S(mx4_value((unsigned(codes[i / 8]) >> (4 * (i % 8))) & 15u) * scale);
  }
}

}  // namespace

hipError_t launch_to_rows(Operand op, int dtype, const void* x, int64_t ld, int64_t features, int64_t columns,
                          Rows const& rows, hipStream_t stream) {
  dim3 const block(256);
  with_dtype(dtype, [&](auto s) {
    using S = decltype(s);
    auto const* in = static_cast<S const*>(x);
    if (op == OPERAND_MX4) {
      dim3 const grid(unsigned((columns + 63) / 64), unsigned((rows.scale_stride + 3) / 4));
      hipLaunchKernelGGL(to_mx4<S>, grid, block, 0, stream, in, ld, features, columns, rows);
    } else {
      dim3 const grid(unsigned((columns + 63) / 64), unsigned((rows.stride / 16 + 3) / 4));
      hipLaunchKernelGGL(to_rows<S>, grid, block, 0, stream, in, ld, features, columns, rows);
    }
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
