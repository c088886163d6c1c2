// A chain of expert layers in one kernel (kernels_chain_*.hip).
#pragma once

#include "contract.h"

namespace ponni_hip {
namespace {

// A whole chain on one tile of C columns: the columns' states stay in LDS, a row of
// whole steps and 16 bytes of padding a column (16 columns' reads of one
// fragment then fall into different banks), and a layer's outputs, complete in the
// accumulators of the W waves, take the place of its inputs between two
// barriers.  Weights come from L2 straight into registers, steps before
// their MFMAs; each serves 16 NJ columns.  The waves are WM x WN, WM the layer's
// blocks of 64 features, so that a narrow layer gives every wave fewer columns.
// FEATURES: the input as the caller holds it.
// fp16 64-256-256-256-64 tanh, 1,000,000 columns of 8 experts: 511 us, 0.64 PFLOP/s: the
// activations' VALU work (78 % of the SIMDs' time) and the MFMAs (31 %) follow one another, where a kernel
// that overlaps them takes 356; LDS bank conflicts a third of its accesses' cycles, 65 + 125 MB
// from and to memory.
template <Operand OP, class S, OutputKind KIND, bool FEATURES, int C, int W>
__global__ __launch_bounds__(64 * W, W == 4 && (OP == OPERAND_F16 || OP == OPERAND_BF16) ? 4 : 2) void contract_chain(ChainArgs chain) {
  constexpr bool MX = OP == OPERAND_MX4;
  constexpr int N = OP == OPERAND_F32 ? 4 : MX ? 32 : 8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  ContractArgs const& a = chain.io;
  int const lane = threadIdx.x & 63;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tile const t = find_tile<C>(a, 1);
  if (t.none) return;
  int const state_stride = chain.state_bytes + 16, state_scale_stride = chain.state_bytes / 16 + 4;
  char* const states = lds;
  unsigned char* const scales = reinterpret_cast<unsigned char*>(lds + C * state_stride);
  {
    // The input's pieces of 16 bytes, one lane per column and piece.
    int const pieces = chain.layers[0].steps * 4;
    for (int p = threadIdx.x; p < C * pieces; p += 64 * W) {
      int const local = p % C, piece = p / C;
      int32_t const col = t.first + local < t.last ? t.first + local : t.last - 1;
      int64_t row = a.source != nullptr ? a.source[col] : col;
      row = row < 0 || row >= a.x_rows ? 0 : row;
      i32x4 v;
      int scale = 0;
      if constexpr (FEATURES) {
        read_features<OP, S>(a, row, piece, v, scale);
      } else {
        v = *reinterpret_cast<i32x4 const*>(a.x.data + row * a.x.stride + piece * 16);
        if constexpr (MX) scale = a.x.scales[row * a.x.scale_stride + piece / 4 * a.x.scale_step + piece % 4];
      }
      *reinterpret_cast<i32x4*>(states + local * state_stride + piece * 16) = v;
      if constexpr (MX) scales[local * state_scale_stride + piece] = static_cast<unsigned char>(scale);
    }
  }
  __syncthreads();
  for (int l = 0; l < chain.num_layers; l++) {
    ChainLayer const& layer = chain.layers[l];
    bool const last = l + 1 == chain.num_layers;
    int const row_features = last ? 0 : chain.layers[l + 1].steps * 4 * N;
    auto pass = [&]<int NJ>(std::integral_constant<int, NJ>, int wn_bits) __attribute__((always_inline)) {
      constexpr int AHEAD = NJ >= 4 ? 1 : 3;  // steps that weights are loaded before their MFMAs; rows one
      int const wm = wave >> wn_bits, wn = wave & ((1 << wn_bits) - 1);
      // (new to the compiler in every layer: it would keep the addresses of every tile of
      // every shape of layer in registers, a hundred more than there are)
      int lane_here = lane, stride = __builtin_amdgcn_readfirstlane(state_stride),
          scale_stride = __builtin_amdgcn_readfirstlane(state_scale_stride);
      asm volatile("" : "+s"(stride));
      asm volatile("" : "+s"(scale_stride));
      asm volatile("" : "+v"(lane_here));
      int const g = lane_here >> 4, c = lane_here & 15;
      bool const busy = wm < layer.blocks && 16 * NJ * wn < C;
      f32x4 acc[4][NJ];
      int const steps = layer.steps;
      if (busy) {
        int64_t const block = int64_t(t.expert) * layer.blocks + wm;
        char const* weights = layer.weights + block * steps * 4096 + 16 * lane;
        int const* w_scales = MX ? reinterpret_cast<int const*>(layer.w_scales + block * steps * 256) + lane : nullptr;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          f32x4 seed = {0, 0, 0, 0};
          if (layer.bias != nullptr) seed = *reinterpret_cast<f32x4 const*>(layer.bias + block * 64 + 16 * g + 4 * i);
#pragma unroll
          for (int j = 0; j < NJ; j++) acc[i][j] = seed;
        }
        char const* rows = states + (16 * NJ * wn + c) * stride + 16 * g;
        unsigned char const* row_scales = scales + (16 * NJ * wn + c) * scale_stride + g;
        i32x4 av[AHEAD + 1][4], bv[2][NJ];
        int as[AHEAD + 1] = {}, bs[2][NJ] = {};
        auto load = [&](int set, int s) {
          s = s < steps ? s : steps - 1;
#pragma unroll
          for (int i = 0; i < 4; i++) av[set][i] = *reinterpret_cast<i32x4 const*>(weights + s * 4096 + i * 1024);
          if constexpr (MX) as[set] = w_scales[s * 64];
        };
        auto read = [&](int set, int s) {
          s = s < steps ? s : steps - 1;
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            bv[set][j] = *reinterpret_cast<i32x4 const*>(rows + 16 * j * stride + s * 64);
            if constexpr (MX) bs[set][j] = row_scales[16 * j * scale_stride + s * 4];
          }
        };
        auto multiply_step = [&](int aset, int bset) {
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            acc[0][j] = multiply<OP, 0>(av[aset][0], bv[bset][j], acc[0][j], as[aset], bs[bset][j]);
            acc[1][j] = multiply<OP, 1>(av[aset][1], bv[bset][j], acc[1][j], as[aset], bs[bset][j]);
            acc[2][j] = multiply<OP, 2>(av[aset][2], bv[bset][j], acc[2][j], as[aset], bs[bset][j]);
            acc[3][j] = multiply<OP, 3>(av[aset][3], bv[bset][j], acc[3][j], as[aset], bs[bset][j]);
          }
        };
#pragma unroll
        for (int u = 0; u < AHEAD; u++) load(u, u);
        read(0, 0);
        // whole turns of the register sets, then the steps left
        constexpr int TURN = AHEAD + 1;
        int s = 0;
        for (; s + TURN <= steps; s += TURN) {
#pragma unroll
          for (int u = 0; u < TURN; u++) {
            load((u + AHEAD) % TURN, s + u + AHEAD);
            read((u + 1) % 2, s + u + 1);
            multiply_step(u, u % 2);
          }
        }
#pragma unroll
        for (int u = 0; u < TURN - 1; u++) {
          if (s + u < steps) {
            if (u > 0) read(u % 2, s + u);
            multiply_step(u, u % 2);
          }
        }
      }
      if (!last) __syncthreads();  // every wave has read the layer's inputs
      if (busy) {
        int const f0 = wm * 64 + 16 * g;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          int const local = 16 * (NJ * wn + j) + c;
          int64_t const col = int64_t(t.first) + local;
          f32x4 v[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
          activate<OP == OPERAND_F32, true>(layer.act, layer.act_a, [&](auto f) {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e / 4][e % 4] = f(v[e / 4][e % 4]);
          });
          clear_past(v, wm * 64, f0, layer.n_out);
          if (last) {
            if (col < t.last) store_features<KIND, S>(a, col, f0, v, layer.n_out);
          } else if constexpr (MX) {
            write_mx4(v, f0 < row_features, reinterpret_cast<i32x2*>(states + local * stride + f0 / 2),
                      f0 % kMx4Block == 0, scales + local * scale_stride + f0 / kMx4Block);
          } else {
            write_pieces<S>(states + local * stride, f0, row_features, v);
          }
          __builtin_amdgcn_sched_barrier(0);  // (one tile's temporaries at a time)
        }
      }
      if (!last) __syncthreads();
    };
    // WM waves along the features, W / WM along the columns
    auto shaped = [&]<int WM>(std::integral_constant<int, WM>) {
      constexpr int NJ = C * WM / (16 * W);
      pass(std::integral_constant<int, NJ < 1 ? 1 : NJ>{}, __builtin_ctz(W / WM));
    };
    if constexpr (W == 8) {
      if (layer.blocks > 4) {
        shaped(std::integral_constant<int, 8>{});
        continue;
      }
    }
    if (layer.blocks > 2) shaped(std::integral_constant<int, 4>{});
    else if (layer.blocks > 1) shaped(std::integral_constant<int, 2>{});
    else shaped(std::integral_constant<int, 1>{});
  }
}

template <Operand OP, class S, OutputKind KIND, bool FEATURES, int C, int W>
hipError_t launch_chain_sized(ChainArgs const& a, hipStream_t stream) {
  int64_t const tiles = grid_of(a.io, C, 1), bytes = chain_lds(OP, a.state_bytes, C);
  if (!launchable(tiles, 64 * W)) return hipErrorInvalidConfiguration;
  auto const kernel = contract_chain<OP, S, KIND, FEATURES, C, W>;
  if (bytes > 65536) {
    hipError_t const e = hipFuncSetAttribute(reinterpret_cast<void const*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(64 * W), static_cast<uint32_t>(bytes), stream, a);
  return hipGetLastError();
}

// The input as [features, columns] where y is (forward), as rows where the outputs are
// (mixture), as 4-bit rows where the caller brings them.
template <Operand OP, class S>
hipError_t launch_chain_as(OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream) {
  auto sized = [&]<OutputKind KIND, bool FEATURES>() {
    if (a.waves == 4) return launch_chain_sized<OP, S, KIND, FEATURES, 64, 4>(a, stream);
    if constexpr (OP == OPERAND_F32) return hipErrorInvalidValue;
    else return columns == 128 ? launch_chain_sized<OP, S, KIND, FEATURES, 128, 8>(a, stream)
                               : launch_chain_sized<OP, S, KIND, FEATURES, 64, 8>(a, stream);
  };
  if (kind == OUT_FLOATS) return sized.template operator()<OUT_FLOATS, false>();
  if (a.io.features != nullptr) return sized.template operator()<OUT_FEATURES, true>();
  if constexpr (OP == OPERAND_MX4) return sized.template operator()<OUT_FEATURES, false>();
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace ponni_hip
