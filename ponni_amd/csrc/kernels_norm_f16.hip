#include "norm.h"

namespace ponni_hip {
hipError_t launch_norm_f16(ponni_residual_norm const& r, hipStream_t stream) { return launch_norm<_Float16>(r, stream); }
hipError_t launch_norm_backward_f16(ponni_residual_norm const& r, ponni_residual_norm_gradients const& g, void* workspace,
                                    int& groups, hipStream_t stream) {
  return launch_norm_backward<_Float16>(r, g, workspace, groups, stream);
}
}  // namespace ponni_hip
