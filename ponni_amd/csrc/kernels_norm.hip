// The norms between blocks (norm.h): kernels by type, and the weights' gradients.
#include <algorithm>

#include "blocks.h"

namespace ponni_hip {

hipError_t launch_norm_f32(ponni_residual_norm const&, hipStream_t);
hipError_t launch_norm_f16(ponni_residual_norm const&, hipStream_t);
hipError_t launch_norm_bf16(ponni_residual_norm const&, hipStream_t);
hipError_t launch_norm_backward_f32(ponni_residual_norm const&, ponni_residual_norm_gradients const&, void*, int&, hipStream_t);
hipError_t launch_norm_backward_f16(ponni_residual_norm const&, ponni_residual_norm_gradients const&, void*, int&, hipStream_t);
hipError_t launch_norm_backward_bf16(ponni_residual_norm const&, ponni_residual_norm_gradients const&, void*, int&, hipStream_t);

namespace {

// The workgroups' sums of a feature, 16 lanes each in the order of the workgroups.
__global__ __launch_bounds__(1024) void join_sums(float const* parts, int groups, int n, NormSums out) {
  __shared__ float lds[16][64];
  float* const y = out.p[blockIdx.y];
  if (y == nullptr) return;
  int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (row < n)
    for (int k = wave; k < groups; k += 16) s += parts[(int64_t(k) * NORM_SUMS + blockIdx.y) * n + row];
  lds[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || row >= n) return;
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; w++) t += lds[w][lane];
  y[row] = t;
}

}  // namespace

hipError_t launch_residual_norm(ponni_residual_norm const& r, hipStream_t stream) {
  return (r.dtype == PONNI_F32 ? launch_norm_f32 : r.dtype == PONNI_F16 ? launch_norm_f16 : launch_norm_bf16)(r, stream);
}

int64_t residual_norm_workspace_bytes(int32_t n, int64_t columns) {
  return std::min<int64_t>(columns, kNormWorkgroups) * NORM_SUMS * n * 4;
}

hipError_t launch_residual_norm_backward(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g,
                                         void* workspace, hipStream_t stream) {
  int groups = 0;
  hipError_t const err = (r.dtype == PONNI_F32   ? launch_norm_backward_f32
                          : r.dtype == PONNI_F16 ? launch_norm_backward_f16
                                                 : launch_norm_backward_bf16)(r, g, workspace, groups, stream);
  if (err != hipSuccess) return err;
  NormSums const out{{g.d_after_weight, g.d_after_bias, g.d_feature_gate, g.d_before_weight, g.d_before_bias}};
  if (std::all_of(out.p, out.p + NORM_SUMS, [](float* p) { return p == nullptr; })) return err;
  hipLaunchKernelGGL(join_sums, dim3((r.n + 63) / 64, NORM_SUMS), dim3(1024), 0, stream, static_cast<float*>(workspace),
                     groups, r.n, out);
  return hipGetLastError();
}

}  // namespace ponni_hip
