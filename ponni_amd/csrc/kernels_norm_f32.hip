#include "norm.h"

namespace ponni_hip {
hipError_t launch_norm_f32(ponni_residual_norm const& r, hipStream_t stream) { return launch_norm<float>(r, stream); }
hipError_t launch_norm_backward_f32(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g, void* workspace,
                                    int& groups, hipStream_t stream) {
  return launch_norm_backward<float>(r, g, workspace, groups, stream);
}
}  // namespace ponni_hip
