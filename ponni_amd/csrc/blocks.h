// Gated blocks, the norms between blocks and log probabilities: what blocks.cpp
// launches (kernels_gated.hip, kernels_norm.hip, kernels_logp.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/ponni_hip.h"

namespace ponni_hip {

// -- log probabilities --------------------------------------------------------------

int64_t logp_workspace_bytes(int64_t classes, int64_t columns, int32_t dtype, int32_t top_k);
int64_t logp_workspace_bytes_up_to(int64_t classes, int64_t columns, int32_t top_k);
hipError_t launch_logp(ponni_log_probs const& p, void* workspace, hipStream_t stream);
hipError_t launch_logp_backward(ponni_log_probs const& p, float const* d_log_probs, float const* d_entropy,
                                float const* d_log_normalizer, void* d_logits, int64_t ld_d_logits, hipStream_t stream);

// -- norms between blocks -------------------------------------------------------------

// Sums over columns that the backward pass leaves: of the weight and bias after, the gate, the weight and bias before.
enum { NORM_SUM_W1, NORM_SUM_B1, NORM_SUM_GATE, NORM_SUM_W2, NORM_SUM_B2, NORM_SUMS };
struct NormSums {
  float* p[NORM_SUMS];
};
constexpr int kNormWorkgroups = 512;  // most of the backward pass, each with sums of its own

hipError_t launch_residual_norm(ponni_residual_norm const& r, hipStream_t stream);
int64_t residual_norm_workspace_bytes(int32_t n, int64_t columns);
hipError_t launch_residual_norm_backward(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g,
                                         void* workspace, hipStream_t stream);

// -- gated blocks -----------------------------------------------------------------------

// The arrays with columns of a call (dy null: forward).
struct GatedArrays {
  void const* x;
  int64_t ld_x;
  void const* states;
  int64_t ld_states;
  void const* dy;
  int64_t ld_dy;
};
// Of a call with those arrays; null: of any call.
int64_t gated_workspace_bytes(ponni_gated const& b, int64_t columns, bool backward, GatedArrays const* arrays = nullptr);
hipError_t launch_gated(ponni_gated const& b, int act, void const* x, int64_t ld_x, void* y, int64_t ld_y, void* states,
                        int64_t ld_states, int64_t columns, void* workspace, hipStream_t stream);
hipError_t launch_gated_backward(ponni_gated const& b, int act, void const* x, int64_t ld_x, void const* states,
                                 int64_t ld_states, void const* dy, int64_t ld_dy, int64_t columns,
                                 ponni_gated_gradients const& g, void* workspace, hipStream_t stream);

}  // namespace ponni_hip
