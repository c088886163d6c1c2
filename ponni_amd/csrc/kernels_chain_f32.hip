#include "chain.h"

namespace ponni_hip {
hipError_t launch_chain_f32(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream) {
  return launch_chain_as<OPERAND_F32, float>(kind, columns, a, stream);
}
}  // namespace ponni_hip
