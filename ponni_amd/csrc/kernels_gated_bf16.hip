#include "gated_product.h"
#include "gated_thin.h"

namespace ponni_hip {
hipError_t launch_product_bf16(Form form, Tile tile, ProductArgs const& p, hipStream_t stream) {
  return launch_product_as<__bf16>(form, tile, p, stream);
}
hipError_t launch_thin_bf16(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream) {
  return launch_thin_as<__bf16>(hidden, last, stream);
}
}  // namespace ponni_hip
