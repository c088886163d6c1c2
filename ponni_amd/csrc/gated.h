// Products of gated blocks: what kernels_gated.hip asks of the kernels of gated_product.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ponni_hip {

// An operand: rows `ld` bytes apart, of `rows` rows, `bytes` from the first element to the end of the last row, up to a
// multiple of 4 as p and ld are.
struct Side {
  char const* p;
  int64_t ld, bytes, rows;
};

enum Output {
  OUT_PLAIN,      // y = C (+ bias)
  OUT_PAIR,       // rows of two products: y = act(C) * C2, and both of them as states
  OUT_STATES,     // from C and the states: y[0] = C u act'(g), y[1] = C act(g)
  OUT_PARTS,      // fp32 sums of a part of k
  OUT_PAIR_PARTS  // the same of OUT_PAIR's two products
};
enum Form {
  FORM_PAIR,     // k outside in both; a: two arrays
  FORM_FORWARD,  // k outside in both
  FORM_STATES,   // k inside in a
  FORM_INPUT,    // k inside in a: the sum of a[0] b[0] and a[1] b[1], pairs of one shape and stride
  FORM_WEIGHTS   // k inside in both
};

struct ProductArgs {
  Side a[2], b[2];
  int64_t k, rows, columns;  // C [rows, columns]
  int problems;              // 2: a[0] b[0] and a[0] b[1], into y[0] and y[1]
  int parts;                 // workgroups that share a tile's k
  bool pair_parts;           // a pair's parts of both products at a time (TILE_NARROW), else one product behind the other
  void* y[2];
  int64_t ld[2];
  void const* bias[2];
  int act;
  float slope;
  void* states;  // [2 rows, columns]: OUT_PAIR writes them (null: not), OUT_STATES reads them
  int64_t ld_states;
  float* sums;   // OUT_PARTS: [parts, problems, rows, ld_sums], of FORM_PAIR one product's behind the other's
  int64_t ld_sums;
  // the grid, filled in by the launch
  int m_tiles, n_tiles, split_n, steps;
};

// Rows and columns of a workgroup's tile; of a pair in 16 bits, half the rows of each of two products.
enum Tile {
  TILE_128,    // 128 x 128
  TILE_LARGE,  // 256 x 256, 16 bits
  TILE_NARROW  // 64 x 256, fp32; of a pair, 32 rows of each product
};
hipError_t launch_product_f32(Form form, Tile tile, ProductArgs const& p, hipStream_t stream);
hipError_t launch_product_f16(Form form, Tile tile, ProductArgs const& p, hipStream_t stream);
hipError_t launch_product_bf16(Form form, Tile tile, ProductArgs const& p, hipStream_t stream);

// A product of few columns (gated_thin.h): parts [slices, problems, columns, stride] of fp32.
enum ThinInput { THIN_COLUMNS, THIN_PARTS, THIN_ROWS };
struct ThinArgs {
  void const* w[2];  // [k, outputs]
  int64_t ld[2];
  int k, outputs, columns;
  int slices, slice_k;  // slice_k a multiple of the waves' steps
  float* parts;
  int stride;  // outputs rounded up to whole tiles
  // the columns: x [k, columns], or h of the parts of g and u, or h [columns, stride_in]
  void const* x;
  int64_t ld_x;
  void* h;
  float const* parts_in;
  int slices_in, stride_in, act;
  float slope;
  void const* bias[3];  // of g, u and y
  void* y;
  int64_t ld_y;
};
hipError_t launch_thin_f32(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream);
hipError_t launch_thin_f16(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream);
hipError_t launch_thin_bf16(ThinArgs const& hidden, ThinArgs const& last, hipStream_t stream);

}  // namespace ponni_hip
