// Argument checks of the operators' C entry points (experts.cpp, blocks.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <new>
#include <stdexcept>
#include <string>

#include "../../include/ponni_hip.h"
#include "program.h"

namespace ponni_hip {

int set_error(int status, std::string const& message);

constexpr int32_t kMaxWidth = 65536;

inline int fail(int status, std::string const& message) { return set_error(status, message); }

// Runs a C entry point's body; nothing is thrown across the ABI.
template <class F> inline int guarded(F&& f) {
  try {
    return f();
  } catch (std::bad_alloc const&) {
    return fail(PONNI_ERR_INVALID_ARGUMENT, "out of host memory");
  } catch (std::exception const& e) {
    return fail(PONNI_ERR_INVALID_ARGUMENT, e.what());
  }
}

inline int device_error(char const* what, hipError_t e) {
  return fail(PONNI_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

inline int64_t element_bytes(int32_t dtype) { return dtype == PONNI_F64 ? 8 : dtype == PONNI_F32 ? 4 : 2; }
inline bool data_type(int32_t dtype) { return dtype == PONNI_F32 || dtype == PONNI_F16 || dtype == PONNI_BF16; }
inline bool aligned(void const* p, uint64_t bytes) { return reinterpret_cast<uint64_t>(p) % bytes == 0; }
inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Range {
  uint64_t begin, end;
};
inline Range array(void const* p, int64_t rows, int64_t ld, int64_t columns, int64_t es) {
  auto const b = reinterpret_cast<uint64_t>(p);
  return {b, b + uint64_t(((rows - 1) * ld + columns) * es)};
}
inline Range bytes(void const* p, int64_t n) {
  auto const b = reinterpret_cast<uint64_t>(p);
  return {b, b + uint64_t(n)};
}
inline bool overlap(Range a, Range b) { return a.begin < b.end && b.begin < a.end; }

inline int check_workspace(void const* workspace, int64_t bytes, int64_t need) {
  if (need > 0 && workspace == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "workspace is null");
  if (!aligned(workspace, 16)) return fail(PONNI_ERR_INVALID_ARGUMENT, "workspace is not at a multiple of 16 bytes");
  if (bytes < need)
    return fail(PONNI_ERR_SHAPE, "workspace holds " + std::to_string(bytes) + " bytes, " + std::to_string(need) +
                                     " are needed");
  return PONNI_OK;
}

// ActCode of an activation layer, -1 for one these operators do not have.
inline int activation_of(ponni_layer_desc const& d) {
  switch (d.kind) {
    case PONNI_LAYER_RELU: return ACT_RELU;
    case PONNI_LAYER_LEAKY_RELU: return ACT_LEAKY_RELU;
    case PONNI_LAYER_GELU: return (d.flags & PONNI_FLAG_GELU_APPROXIMATE) ? ACT_GELU_TANH : ACT_GELU_ERF;
    case PONNI_LAYER_SILU: return ACT_SILU;
    case PONNI_LAYER_SIGMOID: return ACT_SIGMOID;
    case PONNI_LAYER_TANH: return ACT_TANH;
    default: return -1;
  }
}

}  // namespace ponni_hip
