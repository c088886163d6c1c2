// Layers of expert networks over columns grouped by expert:
// y[f, c] = act(bias_e[f] + sum_k W_e[k][f] x[k, c]), e the expert whose group
// holds column c.
//
// Operands are fragments of 16 bytes: 8 features of a 16-bit type, 4 of fp32,
// 32 of 4 bits.  Samples are rows, 64 bytes (4 fragments) a contraction step,
// so that a column taken from anywhere (a mixture gathers its samples by
// expert) is one whole 64-byte piece.  Weights are packed in fragment order.
// Output features are dealt to the MFMA tiles of a block of 64 so that a lane,
// which holds rows 4g .. 4g + 3 of every 16 x 16 tile, holds 16 consecutive
// features 16g + 4i + e of its column: rows are written in whole 16-byte
// pieces from the accumulators, 128 bytes of a row by the four lane groups.
//
// A workgroup computes 16 MI WM features x 16 NJ WN columns of one group; two
// steps' weights and rows, whole 128-byte lines, go from memory straight into
// LDS a turn and a half ahead, fragments into registers a step ahead.  Bound by MFMA:
// bf16 1024-1024, 16 unequal experts, 65,536 columns: 187-200 us, 0.7 PFLOP/s, MFMA busy
// 43 % of the SIMDs' time; 4-bit 4096-4096, 16,384 columns: 175-195 us, 3 PFLOP/s.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "contract.h"
#include "lds_requests.h"

namespace ponni_hip {
namespace {

typedef __attribute__((address_space(3))) void* lds_void;

// Steps a turn of the loop: 128 bytes of a row, one whole line of the L2's.
constexpr int kDepth = 2;

template <Operand OP, class S, OutputKind KIND, int MI, int NJ, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void contract(ContractArgs a) {
  static_assert(MI % 4 == 0, "whole blocks of 64 features");
  constexpr int W = WM * WN, BM = 16 * MI * WM, BN = 16 * NJ * WN, D = kDepth;
  constexpr bool MX = OP == OPERAND_MX4;
  constexpr int A_BYTES = BM * 64 * D, B_BYTES = BN * 64 * D, AS_BYTES = MX ? BM * 4 * D : 0, BS_BYTES = MX ? BN * 4 * D : 0;
  constexpr int SLOT = A_BYTES + B_BYTES + AS_BYTES + BS_BYTES;
  constexpr int A_REQ = A_BYTES / 1024 / W, B_REQ = B_BYTES / 1024 / W, S_REQ = MX ? D * (BM + BN) / 64 / W : 1;
  static_assert(A_BYTES % (1024 * W) == 0 && B_BYTES % (1024 * W) == 0 && (!MX || D * (BM + BN) % (64 * W) == 0), "whole requests");
  __shared__ __attribute__((aligned(16))) char lds[2 * SLOT];
  int const lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const wm = wave / WN, wn = wave % WN;
  Tile const t = find_tile<BN>(a, (a.blocks * 64 + BM - 1) / BM);
  if (t.none) return;
  unsigned const lds0 = static_cast<unsigned>(reinterpret_cast<uint64_t>((lds_void)lds));
  int const steps = a.steps, turns = (steps + D - 1) / D;

  // Columns past the tile's last repeat it.
  auto row_of = [&](int local) {
    int32_t const col = t.first + local < t.last ? t.first + local : t.last - 1;
    int64_t const row = a.source != nullptr ? a.source[col] : col;
    return row < 0 || row >= a.x_rows ? int64_t(0) : row;
  };
  auto block_of = [&](int local) {  // (blocks past the last one are computed and dropped)
    int const b = t.block * (BM / 64) + local;
    return int64_t(t.expert) * a.blocks + (b < a.blocks ? b : a.blocks - 1);
  };
  char const* pa[A_REQ];  // uniform
  char const* pb[B_REQ];
  char const* ps[S_REQ];
  unsigned const lane16 = 16 * lane;
#pragma unroll
  for (int r = 0; r < A_REQ; r++) {
    int const piece = wave + W * r;  // [block][step of the turn][tile]
    pa[r] = uniform(a.weights + block_of(piece / (4 * D)) * steps * 4096 + piece % (4 * D) * 1024);
  }
#pragma unroll
  for (int r = 0; r < B_REQ; r++) {
    int const piece = (wave + W * r) * 64 + lane, col = piece / (4 * D);
    // A row's fragments are kept at places that depend on its column, so that
    // columns' reads of one fragment fall into different banks.
    pb[r] = a.x.data + row_of(col) * a.x.stride + 16 * ((piece ^ col) % (4 * D));
  }
  if constexpr (MX) {
#pragma unroll
    for (int r = 0; r < S_REQ; r++) {
      int const q = (wave + W * r) / D, h = (wave + W * r) % D;  // [block or 64 columns][step of the turn]
      ps[r] = q < BM / 64 ? reinterpret_cast<char const*>(a.w_scales) + (block_of(q) * steps + h) * 256 + 4 * lane
                          : reinterpret_cast<char const*>(a.x.scales) +
                                row_of((q - BM / 64) * 64 + lane) * a.x.scale_stride + h * a.x.scale_step;
    }
  }
  // Request r of a turn: its weights first, then its rows and scales; of a last turn
  // of one step, those of that step.
  constexpr int REQ = A_REQ + B_REQ + (MX ? S_REQ : 0);
  auto request = [&](int turn, int r) {
    unsigned const slot = lds0 + turn % 2 * SLOT;
    bool const whole = D * turn + D <= steps;
    if (r < A_REQ) {
      int const piece = wave + W * r;
      if (whole || piece / 4 % D == 0) dma16(pa[r], lane16, slot + piece * 1024);
      pa[r] += 4096 * D;
    } else if (r < A_REQ + B_REQ) {
      r -= A_REQ;
      int const piece = (wave + W * r) * 64 + lane;
      if (whole || ((piece ^ (piece / (4 * D))) % (4 * D)) < 4) dma16(pb[r], slot + A_BYTES + (wave + W * r) * 1024);
      pb[r] += 64 * D;
    } else if constexpr (MX) {
      r -= A_REQ + B_REQ;
      int const q = wave + W * r;
      if (whole || q % D == 0) dma4(ps[r], slot + A_BYTES + B_BYTES + q * 256);
      ps[r] += q / D < BM / 64 ? int64_t(256 * D) : D * a.x.scale_step;
    }
  };
  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; i++) {
    // bias of features 16 g + 4 i .. + 3 of the block
    f32x4 seed = {0, 0, 0, 0};
    if (a.bias != nullptr)
      seed = *reinterpret_cast<f32x4 const*>(a.bias + block_of((wm * MI + i) / 4) * 64 + 16 * g + 4 * (i % 4));
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[i][j] = seed;
  }
  // The fragments of a step, in one of two sets: read r is a tile's weights, then a tile's rows.
  static_assert(D == 2, "one set a step of the turn");
  constexpr int READS = MI + NJ;
  i32x4 av[D][MI], bv[D][NJ];
  int as[D][MI / 4] = {}, bs[D][NJ] = {};
  auto read = [&](char const* slot, int h, int r) {
    if (r < MI) {
      int const at = (wm * MI + r) / 4 * D + h;
      av[h][r] = reinterpret_cast<i32x4 const*>(slot + (4 * at + r % 4) * 1024)[lane];
      if constexpr (MX)
        if (r % 4 == 0) as[h][r / 4] = reinterpret_cast<int const*>(slot + A_BYTES + B_BYTES + at * 256)[lane];
    } else {
      int const j = r - MI, col = 16 * (wn * NJ + j) + c;
      bv[h][j] = *reinterpret_cast<i32x4 const*>(slot + A_BYTES + 64 * D * col + 16 * (((4 * h + g) ^ col) % (4 * D)));
      if constexpr (MX)
        bs[h][j] = reinterpret_cast<unsigned char const*>(slot)[A_BYTES + B_BYTES + AS_BYTES +
                                                                (col / 64 * D + h) * 256 + 4 * (col % 64) + g];
    }
  };
  // A step's MFMAs, a column tile at a time; `between` makes the reads and requests of that quarter.
  auto multiply_step = [&](int h, auto&& between) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      between(j);
#pragma unroll
      for (int n = 0; n < MI / 4; n++) {
        acc[4 * n][j] = multiply<OP, 0>(av[h][4 * n], bv[h][j], acc[4 * n][j], as[h][n], bs[h][j]);
        acc[4 * n + 1][j] = multiply<OP, 1>(av[h][4 * n + 1], bv[h][j], acc[4 * n + 1][j], as[h][n], bs[h][j]);
        acc[4 * n + 2][j] = multiply<OP, 2>(av[h][4 * n + 2], bv[h][j], acc[4 * n + 2][j], as[h][n], bs[h][j]);
        acc[4 * n + 3][j] = multiply<OP, 3>(av[h][4 * n + 3], bv[h][j], acc[4 * n + 3][j], as[h][n], bs[h][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int r = 0; r < REQ; r++) request(0, r);
  if (turns > 1) {
#pragma unroll
    for (int r = 0; r < REQ; r++) request(1, r);
  }
  if (2 * D <= steps) wait_requests<REQ>();
  else wait_requests<0>();
  workgroup_barrier();
#pragma unroll
  for (int r = 0; r < READS; r++) read(lds, 0, r);
  // One barrier a turn, between its two steps: the next turn's data has landed for every
  // wave, and every wave has this turn's in registers, so its slot takes
  // the turn after the next.  While a step's MFMAs run, the next step's fragments are
  // read (behind the last step: whatever the slot holds, for no use).
  for (int turn = 0; turn < turns; turn++) {
    char const* __restrict__ slot = lds + turn % 2 * SLOT;
    char const* __restrict__ next = lds + (turn + 1) % 2 * SLOT;
    multiply_step(0, [&](int j) {
#pragma unroll
      for (int r = j * READS / NJ; r < (j + 1) * READS / NJ; r++) read(slot, 1, r);
    });
    wait_lds();
    wait_requests<0>();
    workgroup_barrier();
    if (D * turn + 1 >= steps) break;
    multiply_step(1, [&](int j) {
      if (turn + 2 < turns) {
#pragma unroll
        for (int r = j * REQ / NJ; r < (j + 1) * REQ / NJ; r++) request(turn + 2, r);
      }
#pragma unroll
      for (int r = j * READS / NJ; r < (j + 1) * READS / NJ; r++) read(next, 0, r);
    });
  }
#pragma unroll
  for (int n = 0; n < MI / 4; n++) {
    int const f0 = t.block * BM + (wm * MI / 4 + n) * 64 + 16 * g;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      int64_t const col = int64_t(t.first) + 16 * (wn * NJ + j) + c;
      f32x4 v[4] = {acc[4 * n][j], acc[4 * n + 1][j], acc[4 * n + 2][j], acc[4 * n + 3][j]};
      activate<OP == OPERAND_F32>(a.act, a.act_a, [&](auto f) {
#pragma unroll
        for (int e = 0; e < 16; e++) v[e / 4][e % 4] = f(v[e / 4][e % 4]);
      });
      clear_past(v, f0 - 16 * g, f0, a.n_out);
      if constexpr (KIND == OUT_MX4) store_mx4(a, col, col < t.last, f0, v);
      else if (col < t.last) store_features<KIND, S>(a, col, f0, v, a.n_out);
    }
  }
}

// Few columns: 16 MT output features (MT tiles of a block of 64) x 16 NJ columns a
// workgroup, whose W waves share the contraction: what bounds these is the weights' way
// from memory, so each wave has several steps' fragments under way at once,
// straight into registers, and no wave waits for another before the sums meet in LDS
// (in the order of the waves).  FEATURES: the input as the caller holds it, without
// rows made of it first; 4-bit fragments are quantised as they are read.
// bf16 1024-2048 and 2048-1024 of up to 6 of 8 experts, 3 samples: 11.4 and 8.0 us (25 MB
// of weights each at most, 5 us at a copy's rate); 4-bit 2048-2048, 8 columns: 9.0 us,
// the latency of a launch, one load and the sums.
template <Operand OP, class S, OutputKind KIND, bool FEATURES, int MT, int NJ, int W>
__global__ __launch_bounds__(64 * W) void contract_thin(ContractArgs a) {
  static_assert(MT == 4 || (MT == 1 && KIND != OUT_MX4), "a lane's 16 features, or 4 of them");
  constexpr bool MX = OP == OPERAND_MX4;
  constexpr int U = NJ == 1 ? 4 : 2;  // steps under way
  __shared__ f32x4 sums[W][MT * NJ][64];
  int const lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tile const t = find_tile<16 * NJ>(a, a.blocks * (4 / MT));
  if (t.none) return;
  int const steps = a.steps, tile0 = MT == 4 ? 0 : t.block % 4, block_here = MT == 4 ? t.block : t.block / 4;
  int64_t const block = int64_t(t.expert) * a.blocks + block_here;
  char const* const weights = a.weights + block * steps * 4096 + tile0 * 1024 + 16 * lane;
  int64_t row[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    int32_t const col = t.first + 16 * j + c < t.last ? t.first + 16 * j + c : t.last - 1;
    int64_t const r = a.source != nullptr ? a.source[col] : col;
    row[j] = r < 0 || r >= a.x_rows ? int64_t(0) : r;
  }
  // This lane's fragment of step s of column j's row, and its scale.
  auto read_row = [&](int s, int j, i32x4& v, int& scale) {
    if constexpr (FEATURES) {
      read_features<OP, S>(a, row[j], 4 * s + g, v, scale);
    } else {
      v = *reinterpret_cast<i32x4 const*>(a.x.data + row[j] * a.x.stride + s * 64 + 16 * g);
      if constexpr (MX) scale = a.x.scales[row[j] * a.x.scale_stride + s * a.x.scale_step + g];
    }
  };
  f32x4 acc[MT][NJ] = {};
  for (int s0 = wave; s0 < steps; s0 += U * W) {
    i32x4 av[U][MT], bv[U][NJ];
    int as[U] = {}, bs[U][NJ] = {};
#pragma unroll
    for (int u = 0; u < U; u++) {
      int const s = s0 + u * W;
      if (s >= steps) continue;
#pragma unroll
      for (int i = 0; i < MT; i++) av[u][i] = *reinterpret_cast<i32x4 const*>(weights + int64_t(s) * 4096 + i * 1024);
      if constexpr (MX) as[u] = reinterpret_cast<int const*>(a.w_scales + (block * steps + s) * 256)[lane] >> (8 * tile0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s0 + u * W >= steps) continue;
#pragma unroll
      for (int j = 0; j < NJ; j++) read_row(s0 + u * W, j, bv[u][j], bs[u][j]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s0 + u * W >= steps) continue;
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        acc[0][j] = multiply<OP, 0>(av[u][0], bv[u][j], acc[0][j], as[u], bs[u][j]);
        if constexpr (MT == 4) {
          acc[1][j] = multiply<OP, 1>(av[u][1], bv[u][j], acc[1][j], as[u], bs[u][j]);
          acc[2][j] = multiply<OP, 2>(av[u][2], bv[u][j], acc[2][j], as[u], bs[u][j]);
          acc[3][j] = multiply<OP, 3>(av[u][3], bv[u][j], acc[3][j], as[u], bs[u][j]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++) sums[wave][MT * j + i][lane] = acc[i][j];
  __syncthreads();
  if (wave >= NJ) return;
  // Wave j finishes the columns of tile j.
  int const f0 = block_here * 64 + 16 * g + 4 * tile0;
  f32x4 v[4];
#pragma unroll
  for (int i = 0; i < MT; i++) {
    v[i] = a.bias != nullptr ? *reinterpret_cast<f32x4 const*>(a.bias + block * 64 + 16 * g + 4 * (tile0 + i))
                             : f32x4{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; w++) v[i] += sums[w][MT * wave + i][lane];
  }
  activate<OP == OPERAND_F32>(a.act, a.act_a, [&](auto f) {
#pragma unroll
    for (int e = 0; e < 4 * MT; e++) v[e / 4][e % 4] = f(v[e / 4][e % 4]);
  });
  int64_t const col = int64_t(t.first) + 16 * wave + c;
  if constexpr (MT == 4) {
    clear_past(v, block_here * 64, f0, a.n_out);
    if constexpr (KIND == OUT_MX4) store_mx4(a, col, col < t.last, f0, v);
    else if (col < t.last) store_features<KIND, S>(a, col, f0, v, a.n_out);
  } else if (col < t.last) {
    using R = std::conditional_t<KIND == OUT_FLOATS, float, S>;
    int const block0 = block_here * 64;
    int64_t const at = KIND == OUT_FLOATS ? block0 + float_place(g, tile0, float_groups(block0, a.row_features)) : f0;
    R* y = KIND == OUT_FEATURES ? static_cast<R*>(a.y) + at * a.ldy + col
                                : reinterpret_cast<R*>(a.y_rows.data + col * a.y_rows.stride) + at;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (KIND == OUT_FEATURES ? f0 + e < a.n_out : f0 + e < a.row_features)
        y[KIND == OUT_FEATURES ? e * a.ldy : e] = R(f0 + e < a.n_out ? v[0][e] : 0.0f);
    }
  }
}

template <Operand OP, class S, OutputKind KIND, int MI, int NJ, int WM, int WN>
hipError_t launch_tiled(ContractArgs const& a, hipStream_t stream) {
  constexpr int BM = 16 * MI * WM, BN = 16 * NJ * WN;
  int64_t const tiles = grid_of(a, BN, (int64_t(a.blocks) * 64 + BM - 1) / BM);
  if (!launchable(tiles, 64 * WM * WN)) return hipErrorInvalidConfiguration;
  dim3 const grid(static_cast<unsigned>(tiles)), block(64 * WM * WN);
  hipLaunchKernelGGL((contract<OP, S, KIND, MI, NJ, WM, WN>), grid, block, 0, stream, a);
  return hipGetLastError();
}

// Columns of a thin tile, 0 where the other kernels' tiles serve better: with more than 32 columns per expert,
// or more tiles than read their weights, and quantise their input, at the pace of the others' MFMAs.  Times in
// us, thin / 128 x 128 tiles: 16 bits, 2048-2048: 8 experts, 32 columns 17 / 29, 256 columns 22 / 31, 512
// columns 29 / 32; 64 experts, 128 columns 90 / 102, 512 columns 125 / 119; 1024-4096, 16 experts, 256 columns
// 33 / 28. 4 bits, 2048-2048, 8 experts: 32 columns 9.7 / 16, 128 columns 13 to 17 / 16, 256 columns 24 / 16;
// 1024-4096, 16 experts, 64 columns 23 / 16, 512 columns 49 / 17. fp32, whose tiles take as long half empty as
// full, 2048-2048: 64 experts, 128 columns 171 / 482, 2048 columns 378 / 498. (One expert alone is also faster
// in thin tiles above 32 columns: 16 bits 2048-2048, 64 columns 9 / 28, 512 columns 19 / 32, 1024 columns 33 /
// 34; fp32 64 columns 14 / 137.  That is not used.)  Tiles of 16 / 32 columns: 16 bits 2048-2048, one expert, 8
// columns 7.8 / 9.0; 64 experts, 512 columns 126 / 135, 1024 columns 136 / 138, 2048 columns 178 / 159.
inline int thin_columns(Operand op, int64_t columns, int32_t experts, int32_t blocks) {
  int64_t const groups = experts < columns ? experts : columns;
  if (columns > 32 * groups) return 0;
  if (op == OPERAND_MX4 && (columns / 32 + groups) * blocks > 320) return 0;
  if ((op == OPERAND_F16 || op == OPERAND_BF16) && (columns / 128 + groups) * ((blocks + 1) / 2) >= 1024) return 0;
  return columns <= 16 * groups ? 16 : 32;
}

template <Operand OP, class S, OutputKind KIND, bool FEATURES, int NJ>
hipError_t launch_thin(ContractArgs const& a, hipStream_t stream) {
  constexpr int W = 8;
  auto launch = [&]<int MT>(std::integral_constant<int, MT>) {
    int64_t const tiles = grid_of(a, 16 * NJ, int64_t(a.blocks) * (4 / MT));
    if (!launchable(tiles, 64 * W)) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((contract_thin<OP, S, KIND, FEATURES, MT, NJ, W>), dim3(static_cast<unsigned>(tiles)),
                       dim3(64 * W), 0, stream, a);
    return hipGetLastError();
  };
  // Tiles of 16 features where those of 64 leave CUs without one (a 4-bit output's blocks need 64); fewer of
  // them with 16 and 4 bits, where four read the same input as one.  Times in us, 16 / 64 features, 8 columns:
  // 16 bits 2048-2048 7.8 / 9.4 (32 tiles of 64), of 4 experts 10.2 / 9.5 (128), 512-512 of 8, 64 columns 5.3 /
  // 5.8 (96); 4 bits 8.5 / 9.3, 11.6 / 9.3, 5.9 / 6.5; fp32 10.5 / 19.6, 17.7 / 21.0, 8 experts 17.8 / 22.2
  // (256), 32 columns 30.8 / 26.8 (288).
  if constexpr (KIND != OUT_MX4) {
    if (grid_of(a, 16 * NJ, a.blocks) <= (OP == OPERAND_F32 ? 256 : 96)) return launch(std::integral_constant<int, 1>{});
  }
  return launch(std::integral_constant<int, 4>{});
}

template <Operand OP, class S, OutputKind KIND>
hipError_t launch_sized(ContractArgs const& a, hipStream_t stream) {
  bool const features = a.features != nullptr;
  switch (thin_columns(OP, a.columns, a.experts, a.blocks)) {
    case 16: return features ? launch_thin<OP, S, KIND, true, 1>(a, stream) : launch_thin<OP, S, KIND, false, 1>(a, stream);
    case 32: return features ? launch_thin<OP, S, KIND, true, 2>(a, stream) : launch_thin<OP, S, KIND, false, 2>(a, stream);
    default: break;
  }
  if (features) return hipErrorInvalidValue;  // (takes_features)
  // 256 x 256 tiles, which read half as much from L2 per multiply-add, where two rounds of the 256 CUs have one
  // each; else 128 x 128, and always in fp32, whose MFMAs take so long that two workgroups a CU matter more.
  // Times in us, 256 / 128: bf16 1024-1024, 65,536 columns, one expert 207 / 236, 16 226 / 264, 128 253 / 291,
  // 131,072 columns of 512 657 / 715; 16,384 columns (256 tiles) 53 / 56; 4 bits 113 / 123, 128 / 130, 145 /
  // 157, 367 / 434; fp32 1122 / 1110, 1356 / 1173, 1378 / 1235.
  if constexpr (OP != OPERAND_F32) {
    int64_t const large = a.columns / 256 * ((a.blocks + 3) / 4);
    if (a.blocks >= 4 && large >= 512) return launch_tiled<OP, S, KIND, 8, 4, 2, 4>(a, stream);
  }
  return launch_tiled<OP, S, KIND, 4, 4, 2, 2>(a, stream);
}

template <Operand OP, class S>
hipError_t launch_kind(OutputKind kind, ContractArgs const& a, hipStream_t stream) {
  switch (kind) {
    case OUT_FEATURES: return launch_sized<OP, S, OUT_FEATURES>(a, stream);
    case OUT_ROWS:
      if constexpr (OP != OPERAND_MX4) return launch_sized<OP, S, OUT_ROWS>(a, stream);
      return hipErrorInvalidValue;
    case OUT_FLOATS: return launch_sized<OP, S, OUT_FLOATS>(a, stream);
    default:
      if constexpr (OP == OPERAND_MX4) return launch_sized<OP, S, OUT_MX4>(a, stream);
      return hipErrorInvalidValue;
  }
}

// y[f, b] = sum_j weight_j[b] row(slot_j[b])[f], in the order of j.
// 64 samples x 64 features: a lane sums two neighbouring pieces of four features of one
// sample's rows (float_place), the tile turns in LDS.  Bound by bytes: 512 features, top 4,
// 65,536 samples: 130 us for 604 MB, 4.6 TB/s.
template <class S>
__global__ __launch_bounds__(256) void combine(Rows rows, int64_t num_rows, ponni_routing r, int64_t features,
                                               S* __restrict__ y, int64_t ld) {
  __shared__ float tile[64][65];  // [feature][sample]
  int64_t const b0 = int64_t(blockIdx.x) * 64, f0 = int64_t(blockIdx.y) * 64;
  int const groups = float_groups(static_cast<int>(f0), static_cast<int>(rows.stride / 4));
  int const over = groups == 4 ? 8 : groups == 3 ? 11 : groups == 2 ? 16 : 32;  // n / groups is n * over / 32
  for (int p = threadIdx.x; p < 64 * 8; p += 256) {
    int const s = p >> 3, q = 2 * (p & 7);  // pieces q and q + 1 of the block's 4 * groups
    int64_t const b = b0 + s;
    f32x4 sum[2] = {};
    if (q >= 4 * groups) continue;
    if (b < r.batch)
      for (int j = 0; j < r.top_k; j++) {
        int64_t const slot = r.slots[j * r.batch + b];
        if (slot < 0 || slot >= num_rows) continue;
        float const w = r.weights[j * r.batch + b];
        f32x4 const* row = reinterpret_cast<f32x4 const*>(rows.data + slot * rows.stride + f0 * 4) + q;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int e = 0; e < 4; e++) sum[h][e] = fmaf(w, row[h][e], sum[h][e]);
      }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      int const i = (q + h) * over >> 5, g = q + h - i * groups;
#pragma unroll
      for (int e = 0; e < 4; e++) tile[16 * g + 4 * i + e][s] = sum[h][e];
    }
  }
  __syncthreads();
  int const s = threadIdx.x & 63;
  if (b0 + s >= r.batch) return;
  for (int f = threadIdx.x >> 6; f < 64 && f0 + f < features; f += 4) y[(f0 + f) * ld + b0 + s] = S(tile[f][s]);
}

// A parameter on its way to a type of at most 16 bits.  fp64 is rounded to odd (cut off, the last bit set
// where something was lost), so that the rounding that follows sees which side of a middle it lay on.
template <Operand OP, class T> __device__ inline float parameter(T v) {
  float const f = float(v);
  if constexpr (std::is_same_v<T, double> && OP != OPERAND_F32) {
    unsigned const bits = __builtin_bit_cast(unsigned, f);
    if (double(f) != v && !(bits & 1u) && __builtin_fabsf(f) < __builtin_inff())
      return __builtin_bit_cast(float, __builtin_fabs(double(f)) < __builtin_fabs(v) ? bits + 1 : bits - 1);
  }
  return f;
}

// One lane per 16-byte piece of the packed weights; the grid's second dimension is the experts.
template <Operand OP, class T>
__global__ __launch_bounds__(256) void pack_weights(T const* __restrict__ w, int64_t n_in, int64_t n_out,
                                                    int64_t blocks, int64_t steps, char* weights,
                                                    unsigned char* scales) {
  int const lane = threadIdx.x % 64, i = threadIdx.x / 64, g = lane >> 4, row = lane & 15;
  int64_t const step = blockIdx.x % steps, block = blockIdx.x / steps, e = blockIdx.y;
  int64_t const piece = ((e * blocks + block) * steps + step) * 256 + threadIdx.x;
  int64_t const f = block * 64 + 16 * (row >> 2) + 4 * i + (row & 3);
  constexpr int N = OP == OPERAND_F32 ? 4 : OP == OPERAND_MX4 ? 32 : 8;
  int64_t const k0 = step * 4 * N + g * N;
  float v[N];
#pragma unroll
  for (int k = 0; k < N; k++) v[k] = f < n_out && k0 + k < n_in ? parameter<OP>(w[(e * n_in + k0 + k) * n_out + f]) : 0.0f;
  i32x4 out = {0, 0, 0, 0};
  if constexpr (OP == OPERAND_MX4) {
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int k = 0; k < N; k++) {
      amax = fmaxf(amax, __builtin_fabsf(v[k]));
      finite = finite && v[k] == v[k];
    }
    unsigned const scale = finite ? mx4_scale(amax) : 255u;
    float const scale_value = mx4_scale_value(scale);
    if (scale != 255u) {
#pragma unroll
      for (int w = 0; w < 4; w++) out[w] = mx4_word(scale_value, [&](int k) { return v[8 * w + k]; });
    }
    scales[(piece / 256 * 64 + lane) * 4 + i] = static_cast<unsigned char>(scale);
  } else {
    using S = std::conditional_t<OP == OPERAND_F32, float, std::conditional_t<OP == OPERAND_F16, _Float16, __bf16>>;
    typedef S Piece __attribute__((ext_vector_type(N)));
    Piece p;
#pragma unroll
    for (int k = 0; k < N; k++) p[k] = S(v[k]);
    out = __builtin_bit_cast(i32x4, p);
  }
  reinterpret_cast<i32x4*>(weights)[piece] = out;
}

template <class T>
__global__ __launch_bounds__(256) void pack_bias(T const* __restrict__ b, int64_t n, int64_t padded,
                                                 float* __restrict__ bias) {
  int64_t const i = int64_t(blockIdx.x) * 256 + threadIdx.x, e = blockIdx.y;
  if (i < padded) bias[e * padded + i] = i < n ? float(b[e * n + i]) : 0.0f;
}

template <class F> bool with_parameter_dtype(int dtype, F&& f) {
  if (dtype == PONNI_F64) {
    f(double{});
    return true;
  }
  return with_dtype(dtype, f);
}

}  // namespace

int64_t chain_lds(Operand op, int state_bytes, int columns) {
  return int64_t(columns) * (state_bytes + 16) + (op == OPERAND_MX4 ? int64_t(columns) * (state_bytes / 16 + 4) : 0);
}

// One kernel takes the chain where there are more columns than a thin tile's to share an expert's weights,
// layers have at most 8 blocks of 64 outputs (fp32: 4), and states 2 KB a column (512 fp32 or 1024 16-bit
// features; 4 bits 1024 features): its tiles of 64 columns read all weights once each.  Against layer by layer
// (us): fp16 64-256-256-256-64 tanh, 1,000,000 columns 518 / 1117; bf16 512-512-512, 300,000 506 / 613, 5,000
// 25 / 32; 800-500-500, 40,000 105 / 120; 100-200-100, 3,000 13 / 20; 4 bits 256-256, 1,000,000 389 / 411;
// 1024-512-512, 300,000 471 / 550; fp32 300-200-17, 40,000 102 / 123.  Wider inputs: bf16 1200-256-64, 40,000
// 122 / 84, 5,000 33 / 38; 4 bits 2048-256, 5,000 40 / 22 (300,000 483 / 532); 4608-64, 40,000 242 / 127; fp32
// 600-256, 40,000 188 / 159; 200-300-100 (5 blocks), 20,000 99 / 79.  Few columns: bf16 500-500-500, 100 of 8
// experts 21 / 11.
// Layers of more than 4 blocks take tiles of 128 columns where there are 2048 of them: 64 / 128 columns bf16
// 512-512-512, 65,536 133 / 137, 500,000 891 / 797; 64-512-64, 65,536 40 / 48, 500,000 233 / 247; 4 bits
// 512-512-512, 65,536 97 / 109, 500,000 608 / 597; 64-512-64, 65,536 55 / 50, 500,000 322 / 251.
int chain_columns(Operand op, ChainArgs& a) {
  int blocks = 0;
  for (int l = 0; l < a.num_layers; l++) {
    blocks = a.layers[l].blocks > blocks ? a.layers[l].blocks : blocks;
    if (a.layers[l].act == ACT_GELU_ERF) return 0;  // (its code, for every accumulator of every shape of layer)
  }
  if (blocks > (op == OPERAND_F32 ? 4 : 8) || a.state_bytes > (op == OPERAND_MX4 ? 512 : 2048)) return 0;
  if (thin_columns(op, a.io.columns, a.io.experts, blocks) > 0) return 0;
  a.waves = blocks > 4 ? 8 : 4;
  return blocks > 4 && chain_lds(op, a.state_bytes, 128) <= 160 * 1024 && a.io.columns >= 128 * 2048 ? 128 : 64;
}
static_assert(64 * (2048 + 16) <= 160 * 1024, "a tile of 64 columns fits LDS");

hipError_t launch_chain(Operand op, int out_type, OutputKind kind, int columns, ChainArgs const& a, hipStream_t stream) {
  switch (op) {
    case OPERAND_F32: return launch_chain_f32(kind, columns, a, stream);
    case OPERAND_F16: return launch_chain_f16(kind, columns, a, stream);
    case OPERAND_BF16: return launch_chain_bf16(kind, columns, a, stream);
    default:
      return out_type == PONNI_F16 ? launch_chain_mx4_f16(kind, columns, a, stream)
                                   : launch_chain_mx4_bf16(kind, columns, a, stream);
  }
}

bool takes_features(Operand op, int64_t columns, int32_t experts, int32_t blocks) {
  return thin_columns(op, columns, experts, blocks) > 0;
}

hipError_t launch_contraction(Operand op, int out_type, OutputKind kind, ContractArgs const& a, hipStream_t stream) {
  switch (op) {
    case OPERAND_F32: return launch_kind<OPERAND_F32, float>(kind, a, stream);
    case OPERAND_F16: return launch_kind<OPERAND_F16, _Float16>(kind, a, stream);
    case OPERAND_BF16: return launch_kind<OPERAND_BF16, __bf16>(kind, a, stream);
    default:
      return out_type == PONNI_F16 ? launch_kind<OPERAND_MX4, _Float16>(kind, a, stream)
                                   : launch_kind<OPERAND_MX4, __bf16>(kind, a, stream);
  }
}

hipError_t launch_combine(int dtype, Rows const& rows, int64_t num_rows, const ponni_routing& r, int64_t features,
                          void* y, int64_t ld, hipStream_t stream) {
  dim3 const grid(unsigned((r.batch + 63) / 64), unsigned((features + 63) / 64));
  with_dtype(dtype, [&](auto s) {
    using S = decltype(s);
    hipLaunchKernelGGL(combine<S>, grid, dim3(256), 0, stream, rows, num_rows, r, features, static_cast<S*>(y), ld);
  });
  return hipGetLastError();
}

hipError_t launch_pack_weights(Operand op, int dtype, const void* w, int64_t experts, int64_t n_in, int64_t n_out,
                               int64_t blocks, char* weights, unsigned char* scales, hipStream_t stream) {
  int64_t const steps = contraction_steps(op, n_in);
  // (65536 features at most: 2^22 workgroups an expert)
  dim3 const grid(static_cast<unsigned>(blocks * steps), static_cast<unsigned>(experts)), block(256);
  with_parameter_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, block, 0, stream, static_cast<T const*>(w), n_in, n_out, blocks, steps,
                         weights, scales);
    };
    switch (op) {
      case OPERAND_F32: launch(pack_weights<OPERAND_F32, T>); break;
      case OPERAND_F16: launch(pack_weights<OPERAND_F16, T>); break;
      case OPERAND_BF16: launch(pack_weights<OPERAND_BF16, T>); break;
      default: launch(pack_weights<OPERAND_MX4, T>); break;
    }
  });
  return hipGetLastError();
}

hipError_t launch_pack_bias(int dtype, const void* b, int64_t experts, int64_t n, int64_t padded, float* bias,
                            hipStream_t stream) {
  dim3 const grid(static_cast<unsigned>((padded + 255) / 256), static_cast<unsigned>(experts));
  with_parameter_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(pack_bias<T>, grid, dim3(256), 0, stream, static_cast<T const*>(b), n, padded, bias);
  });
  return hipGetLastError();
}

}  // namespace ponni_hip
