// Expert networks, routing and 4-bit blocks: internal structures
// (experts.cpp, kernels_experts.hip, kernels_route.hip, kernels_mx4.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <vector>

#include "../../include/ponni_hip.h"

namespace ponni_hip {

// Operand types of a contraction.  A fragment is 16 bytes of one row's
// consecutive features per lane, a step four of them: 64 bytes of a row.
enum Operand { OPERAND_F32 = 0, OPERAND_F16 = 1, OPERAND_BF16 = 2, OPERAND_MX4 = 3 };
constexpr int kMx4Block = 32;  // features that share a scale
inline int step_features(Operand o) { return o == OPERAND_F32 ? 16 : o == OPERAND_MX4 ? 128 : 32; }
// Where the four features 16 g + 4 i .. + 3 of a block of 64 lie in an OUT_FLOATS row, `groups` (1 to 4) of 16 features
// in the block: so that what the groups' lanes store together, their pieces i, is consecutive.
__host__ __device__ inline int float_place(int g, int i, int groups) { return 4 * (i * groups + g); }
// Groups of 16 features in the block of 64 that begins at `block`, of a row of row_features.
__host__ __device__ inline int float_groups(int block, int row_features) {
  return row_features - block < 64 ? (row_features - block) / 16 : 4;
}
inline int64_t contraction_steps(Operand o, int64_t features) {
  return (features + step_features(o) - 1) / step_features(o);
}

// Samples as rows: 64 bytes a step, features past the last one zero; mx4 rows
// have 4 scale bytes a step beside them (a caller's row by row; the library's own step by
// step, so that a tile's are consecutive).
struct Rows {
  char* data = nullptr;
  unsigned char* scales = nullptr;  // mx4
  int64_t stride = 0;               // bytes from row to row of `data`
  int64_t scale_stride = 0;         // bytes from a row's 4 scales to the next row's of a step,
  int64_t scale_step = 0;           // and to those of the next step
};

// [features, columns], or rows: a layer's of the operand's type or of 4 bits for the next one; a
// mixture's outputs as fp32, whole groups of 16 features in the order of float_place.
enum OutputKind { OUT_FEATURES = 0, OUT_ROWS = 1, OUT_MX4 = 2, OUT_FLOATS = 3 };

// One layer over columns grouped by expert:
// y[f, c] = act(bias_e[f] + sum_k W_e[k][f] x[k, c]) for offsets[e] <= c < offsets[e + 1].
struct ContractArgs {
  const char* weights;           // [experts][blocks][steps][4 tiles][64 lanes][16 bytes]
  const unsigned char* w_scales; // mx4: [experts][blocks][steps][64 lanes][4 tiles]
  const float* bias;             // [experts][64 blocks], or null
  Rows x;
  const void* features;  // or the input as [features, x_rows] of the model's type, row stride ldx (takes_features)
  int64_t ldx;
  int32_t n_in;
  int64_t x_rows;
  const int32_t* source;   // row of each column (null: the column itself)
  const int32_t* offsets;  // [experts + 1] (null: one group of all columns)
  int64_t columns;
  int32_t experts;
  int32_t steps;
  int32_t blocks;  // of 64 output features
  int32_t n_out;
  int32_t act;  // ActCode, 0: none
  float act_a;
  // OUT_FEATURES: y[f * ldy + c] of `out_type`; else y_rows,
  // `row_features` features each (those past n_out zero).
  void* y;
  int64_t ldy;
  Rows y_rows;
  int32_t row_features;
};

// A whole chain in one kernel, states in LDS (contract_chain).
constexpr int kChainLayers = 8;
struct ChainLayer {
  const char* weights;
  const unsigned char* w_scales;
  const float* bias;
  int32_t steps;
  int32_t blocks;
  int32_t n_out;
  int32_t act;
  float act_a;
};
struct ChainArgs {
  ContractArgs io;  // input, groups and output (weights, steps and the like unused)
  ChainLayer layers[kChainLayers];
  int32_t num_layers;
  int32_t state_bytes;  // of a column's state: its steps * 64, the widest layer's
  int32_t waves;        // of a workgroup: 4, or 8 for layers of more than 4 blocks
};
// A tile's LDS: the states, and their scales.
int64_t chain_lds(Operand op, int state_bytes, int columns);
// Columns of a chain's tile, 0 where the kernel does not take the chain; sets a.waves.
int chain_columns(Operand op, ChainArgs& a);
hipError_t launch_chain_f32(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);
hipError_t launch_chain_f16(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);
hipError_t launch_chain_bf16(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);
hipError_t launch_chain_mx4_f16(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);
hipError_t launch_chain_mx4_bf16(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);
hipError_t launch_chain(Operand op, int out_type, OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream);

// Whether a layer of these sizes reads its input as [features, columns] itself.
bool takes_features(Operand op, int64_t columns, int32_t experts, int32_t blocks);
hipError_t launch_contraction(Operand op, int out_type, OutputKind kind, ContractArgs const& a, hipStream_t stream);

// x [features, columns] of `dtype` as rows of `op`, `row_bytes` a row.
hipError_t launch_to_rows(Operand op, int dtype, const void* x, int64_t ld, int64_t features, int64_t columns,
                          Rows const& rows, hipStream_t stream);
// y[f, b] = sum_j weights[j, b] rows[slots[j, b]][f] (slots outside [0, num_rows) add nothing); rows of floats.
hipError_t launch_combine(int dtype, Rows const& rows, int64_t num_rows, const ponni_routing& r, int64_t features,
                          void* y, int64_t ld, hipStream_t stream);
// W [experts, n_in, n_out] of `dtype` in fragment order (values past n_in or n_out zero).
hipError_t launch_pack_weights(Operand op, int dtype, const void* w, int64_t experts, int64_t n_in, int64_t n_out,
                               int64_t blocks, char* weights, unsigned char* scales, hipStream_t stream);
// b [experts, n] of `dtype` as floats [experts, padded], zero past n.
hipError_t launch_pack_bias(int dtype, const void* b, int64_t experts, int64_t n, int64_t padded, float* bias,
                            hipStream_t stream);
hipError_t launch_mx4_values(Rows const& rows, int64_t features, int64_t columns, void* y, int64_t ld, int dtype,
                             hipStream_t stream);
hipError_t launch_route(const void* scores, int64_t ld, int dtype, int normalize, ponni_routing const& r, void* workspace,
                        hipStream_t stream);
int64_t route_workspace_bytes(int64_t experts, int64_t batch);
int64_t route_workspace_bytes_up_to(int64_t experts, int64_t batch);  // that any smaller batch needs too

int set_error(int status, std::string const& message);

}  // namespace ponni_hip

struct ponni_experts_s {
  struct Layer {
    int32_t n_in = 0, n_out = 0;
    int32_t act = 0;
    float act_a = 0.0f;
    int32_t matvec = -1, bias = -1;  // layers of the descriptor list
    int32_t steps = 0, blocks = 0;
    char* weights = nullptr;
    unsigned char* scales = nullptr;
    float* d_bias = nullptr;
    bool weights_set = false;
  };
  std::vector<ponni_layer_desc> descs;
  std::vector<Layer> layers;
  int32_t num_experts = 0;
  int32_t dtype = PONNI_F32;
  ponni_hip::Operand operand = ponni_hip::OPERAND_F32;
  int device = -1;
};
