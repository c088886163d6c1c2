#include "gated_product.h"
#include "gated_thin.h"

namespace ponni_hip {
hipError_t launch_product_f16(Form form, Tile tile, ProductArgs const& p, hipStream_t stream) {
  return launch_product_as<_Float16>(form, tile, p, stream);
}
hipError_t launch_thin_f16(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream) {
  return launch_thin_as<_Float16>(hidden, last, stream);
}
}  // namespace ponni_hip
