#include "gated_product.h"

namespace ponni_hip {
hipError_t launch_product_f16(Form form, bool large, ProductArgs const& p, hipStream_t stream) {
  return launch_product_as<_Float16>(form, large, p, stream);
}
}  // namespace ponni_hip
