#include "chain.h"

namespace ponni_hip {
hipError_t launch_chain_mx4_bf16(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream) {
  return launch_chain_as<OPERAND_MX4, __bf16>(kind, columns, a, stream);
}
}  // namespace ponni_hip
