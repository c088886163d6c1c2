// C ABI of routing, expert networks and 4-bit rows: argument checks, work
// buffers, launches (kernels_route.hip, kernels_experts.hip, kernels_mx4.hip).
#include "experts.h"

#include <algorithm>
#include <memory>
#include <new>
#include <string>

#include "program.h"

namespace ponni_hip {
namespace {

constexpr int32_t kMaxWidth = 65536;
// (PONNI_MAX_COLUMNS: a launch has fewer than 2^32 threads in a dimension, and where the grid is one of columns alone
// 64 of them have 256 threads at most: 4.0e9.  The layers' tiles, of output features too, are counted when launched.)

int fail(int status, std::string const& message) { return set_error(status, message); }

// Runs a C entry point's body; nothing is thrown across the ABI.
template <class F> int guarded(F&& f) {
  try {
    return f();
  } catch (std::bad_alloc const&) {
    return fail(PONNI_ERR_INVALID_ARGUMENT, "out of host memory");
  } catch (std::exception const& e) {
    return fail(PONNI_ERR_INVALID_ARGUMENT, e.what());
  }
}

int device_error(char const* what, hipError_t e) {
  return fail(PONNI_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

int64_t element_bytes(int32_t dtype) { return dtype == PONNI_F64 ? 8 : dtype == PONNI_F32 ? 4 : 2; }
bool data_type(int32_t dtype) { return dtype == PONNI_F32 || dtype == PONNI_F16 || dtype == PONNI_BF16; }
bool aligned(void const* p, uint64_t bytes) { return reinterpret_cast<uint64_t>(p) % bytes == 0; }
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Range {
  uint64_t begin, end;
};
Range array(void const* p, int64_t rows, int64_t ld, int64_t columns, int64_t es) {
  auto const b = reinterpret_cast<uint64_t>(p);
  return {b, b + uint64_t(((rows - 1) * ld + columns) * es)};
}
Range bytes(void const* p, int64_t n) {
  auto const b = reinterpret_cast<uint64_t>(p);
  return {b, b + uint64_t(n)};
}
bool overlap(Range a, Range b) { return a.begin < b.end && b.begin < a.end; }

// A routing's arrays: weights, slots, source and offsets, which a mixture reads, and experts.
constexpr int kRoutingArrays = 5;
void routing_ranges(ponni_routing const& r, Range (&out)[kRoutingArrays]) {
  int64_t const n = r.top_k * r.batch * 4;
  out[0] = bytes(r.weights, n);
  out[1] = bytes(r.slots, n);
  out[2] = bytes(r.source, n);
  out[3] = bytes(r.offsets, (int64_t(r.num_experts) + 1) * 4);
  out[4] = bytes(r.experts, n);
}

// Work buffers of a call: rows of the input (unless the caller brings them),
// the layers' outputs in two buffers by turns.
struct Workspace {
  int64_t input = 0, input_scales = 0, state[2] = {0, 0}, state_scales[2] = {0, 0}, total = 0;
};

// The chain's layers, and the columns of its tiles where one kernel takes it whole (0: layer by layer).
int chain_of(ponni_experts_s const& e, int64_t columns, ChainArgs& a) {
  a = ChainArgs{};
  if (e.layers.size() > kChainLayers) return 0;
  a.num_layers = static_cast<int32_t>(e.layers.size());
  for (int32_t i = 0; i < a.num_layers; i++) {
    auto const& l = e.layers[i];
    a.layers[i] = {l.weights, l.scales, l.d_bias, l.steps, l.blocks, l.n_out, l.act, l.act_a};
    a.state_bytes = std::max(a.state_bytes, l.steps * 64);
  }
  a.io.columns = columns;
  a.io.experts = e.num_experts;
  return chain_columns(e.operand, a);
}

// A mixture's chains leave their outputs in fp32 for the weighted sum, in batches of every size.
// Rounded to the model's type first, each would add up to half a step of |weight| |output|: more than the
// sum itself where outputs cancel, and infinite where fp16 ends.  That would halve their way
// through memory: fp16 512-1024-512, top 4, 65,536 samples, 537 MB each way, takes 940 us for 810.
int64_t output_row_bytes(ponni_experts_s const& e) { return round_up(e.layers.back().n_out, 16) * 4; }

Workspace workspace_of(ponni_experts_s const& e, int64_t rows, int64_t columns, bool mixture) {
  Workspace w;
  ChainArgs chain;
  bool const whole = chain_of(e, columns, chain) > 0;
  bool const direct = whole ? !mixture : takes_features(e.operand, columns, e.num_experts, e.layers[0].blocks);
  if (direct) rows = 0;
  auto take = [&](int64_t n) {
    int64_t const at = w.total;
    w.total += round_up(n, 256);
    return at;
  };
  bool const mx4 = e.operand == OPERAND_MX4;
  w.input = take(rows * e.layers[0].steps * 64);
  w.input_scales = take(mx4 ? rows * e.layers[0].steps * 4 : 0);
  int64_t data[2] = {0, 0}, scales[2] = {0, 0};
  size_t const last = e.layers.size() - 1;
  for (size_t i = 0; i < last && !whole; i++) {
    data[i % 2] = std::max(data[i % 2], columns * e.layers[i + 1].steps * 64);
    if (mx4) scales[i % 2] = std::max(scales[i % 2], columns * e.layers[i + 1].steps * 4);
  }
  if (mixture) data[last % 2] = std::max(data[last % 2], columns * output_row_bytes(e));
  for (int b = 0; b < 2; b++) {
    w.state[b] = take(data[b]);
    w.state_scales[b] = take(scales[b]);
  }
  return w;
}

// Bytes that any number of columns up to `columns` needs, top_k of them a sample in a mixture (0: none).
// Where the kernels for few columns end, one kernel may take the whole chain and need fewer; on
// either side of that the bytes grow with the columns.
int64_t workspace_bytes_up_to(ponni_experts_s const& e, int32_t top_k, int64_t batch) {
  int64_t const per = std::max(top_k, 1);
  int32_t blocks = 0;
  for (auto const& l : e.layers) blocks = std::max(blocks, l.blocks);
  auto need = [&](int64_t b) { return b < 1 ? 0 : workspace_of(e, b, b * per, top_k > 0).total; };
  int64_t few = 0, more = batch + 1;  // the last batch of few columns, the first of more
  while (few + 1 < more) {
    int64_t const b = few + (more - few) / 2;
    (takes_features(e.operand, b * per, e.num_experts, blocks) ? few : more) = b;
  }
  return std::max(need(batch), need(few));
}

int check_ready(ponni_experts_s const& e) {
  for (size_t i = 0; i < e.layers.size(); i++)
    if (!e.layers[i].weights_set)
      return fail(PONNI_ERR_INVALID_ARGUMENT, "the parameters of layer " + std::to_string(e.layers[i].matvec) +
                                                  " (Matvec) were never set");
  int device = 0;
  hipError_t const err = hipGetDevice(&device);
  if (err != hipSuccess) return device_error("hipGetDevice", err);
  if (device != e.device) return fail(PONNI_ERR_DEVICE, "the expert networks' parameters are on another device");
  return PONNI_OK;
}

int check_workspace(void const* workspace, int64_t bytes, int64_t need) {
  if (need > 0 && workspace == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "workspace is null");
  if (!aligned(workspace, 16)) return fail(PONNI_ERR_INVALID_ARGUMENT, "workspace is not at a multiple of 16 bytes");
  if (bytes < need)
    return fail(PONNI_ERR_SHAPE, "workspace holds " + std::to_string(bytes) + " bytes, " + std::to_string(need) +
                                     " are needed");
  return PONNI_OK;
}

int check_routing_sizes(int32_t experts, int32_t top_k, int64_t batch) {
  if (experts < 1 || experts > PONNI_MAX_EXPERTS)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "num_experts must be 1 to " + std::to_string(PONNI_MAX_EXPERTS));
  if (top_k < 1 || top_k > std::min(PONNI_MAX_TOP_K, experts))
    return fail(PONNI_ERR_INVALID_ARGUMENT,
                "top_k must be 1 to " + std::to_string(std::min(PONNI_MAX_TOP_K, experts)));
  if (batch <= 0) return fail(PONNI_ERR_SHAPE, "routing requires a nonzero batch size");
  if (batch > PONNI_MAX_COLUMNS / top_k)
    return fail(PONNI_ERR_SHAPE, "top_k * batch exceeds " + std::to_string(PONNI_MAX_COLUMNS));
  return PONNI_OK;
}

// The layers over `columns` sorted columns of x [features, input_rows] or of rows made of it (row
// source[c] of them, or c itself): into y [features, columns], or (y null) rows in `result`.
int run_layers(ponni_experts_s const& e, void const* x, int64_t ld_in, Rows input, int64_t input_rows,
               int32_t const* source, int32_t const* offsets, int64_t columns, void* y, int64_t ld_out, char* base,
               Workspace const& w, Rows* result, hipStream_t stream) {
  bool const mx4 = e.operand == OPERAND_MX4;
  size_t const last = e.layers.size() - 1;
  ChainArgs chain;
  int const chain_tile = chain_of(e, columns, chain);
  // (rows are the caller's 4-bit ones, or made here where the first kernel does not read x itself)
  bool const direct = chain_tile > 0 ? y != nullptr : takes_features(e.operand, columns, e.num_experts, e.layers[0].blocks);
  if (x != nullptr && !direct) {
    input.data = base + w.input;
    input.scales = reinterpret_cast<unsigned char*>(base + w.input_scales);
    input.stride = int64_t(e.layers[0].steps) * 64;
    input.scale_stride = 4;
    input.scale_step = input_rows * 4;
    hipError_t const err = launch_to_rows(e.operand, e.dtype, x, ld_in, e.layers[0].n_in, input_rows, input, stream);
    if (err != hipSuccess) return device_error("input rows", err);
    x = nullptr;
  }
  for (size_t i = chain_tile > 0 ? last : 0; i <= last; i++) {
    auto const& l = e.layers[i];
    ContractArgs a{};
    a.weights = l.weights;
    a.w_scales = l.scales;
    a.bias = l.d_bias;
    a.x = input;
    a.features = x;
    a.ldx = ld_in;
    a.n_in = e.layers[chain_tile > 0 ? 0 : i].n_in;
    a.x_rows = input_rows;
    a.source = source;
    a.offsets = offsets;
    a.columns = columns;
    a.experts = e.num_experts;
    a.steps = l.steps;
    a.blocks = l.blocks;
    a.n_out = l.n_out;
    a.act = l.act;
    a.act_a = l.act_a;
    OutputKind kind = OUT_FEATURES;
    if (i == last && y != nullptr) {
      a.y = y;
      a.ldy = ld_out;
    } else {
      kind = i == last ? OUT_FLOATS : mx4 ? OUT_MX4 : OUT_ROWS;
      int const next = i < last ? e.layers[i + 1].steps : 0;
      a.y_rows.data = base + w.state[i % 2];
      a.y_rows.scales = reinterpret_cast<unsigned char*>(base + w.state_scales[i % 2]);
      a.y_rows.stride = i < last ? int64_t(next) * 64 : output_row_bytes(e);
      a.y_rows.scale_stride = 4;
      a.y_rows.scale_step = columns * 4;
      a.row_features = i < last ? next * step_features(e.operand) : static_cast<int32_t>(output_row_bytes(e) / 4);
    }
    hipError_t err;
    if (chain_tile > 0) {
      chain.io = a;
      err = launch_chain(e.operand, e.dtype, kind, chain_tile, chain, stream);
    } else {
      err = launch_contraction(e.operand, e.dtype, kind, a, stream);
    }
    if (err != hipSuccess) return device_error("expert layer", err);
    x = nullptr;
    input = a.y_rows;
    input_rows = columns;
    source = nullptr;
  }
  if (result != nullptr) *result = input;
  return PONNI_OK;
}

int forward_impl(ponni_experts e, const void* x, int64_t ld_in, const void* codes, const void* scales, bool mx4_rows,
                 const int32_t* offsets, void* y, int64_t ld_out, int64_t columns, void* workspace,
                 int64_t workspace_bytes, hipStream_t stream) {
  if (e == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null");
  if (columns <= 0) return fail(PONNI_ERR_SHAPE, "expert networks require a nonzero number of columns");
  if (columns > PONNI_MAX_COLUMNS)
    return fail(PONNI_ERR_SHAPE, "columns exceed " + std::to_string(PONNI_MAX_COLUMNS));
  if (mx4_rows && e->operand != OPERAND_MX4)
    return fail(PONNI_ERR_UNSUPPORTED, "4-bit rows are the input of networks with 4-bit weights");
  if (y == nullptr || (mx4_rows ? codes == nullptr || scales == nullptr : x == nullptr))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "input or output pointer is null");
  if (mx4_rows && !(aligned(codes, 16) && aligned(scales, 16)))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "codes and scales must be at multiples of 16 bytes");
  if (offsets == nullptr && e->num_experts > 1)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "offsets are null with more than one expert");
  if ((!mx4_rows && ld_in < columns) || ld_out < columns)
    return fail(PONNI_ERR_SHAPE, "row strides are smaller than the number of columns");
  Workspace const w = workspace_of(*e, mx4_rows ? 0 : columns, columns, false);
  int st = check_workspace(workspace, workspace_bytes, w.total);
  if (st != PONNI_OK) return st;
  auto const& first = e->layers.front();
  int64_t const es = element_bytes(e->dtype);
  Range const out = array(y, e->layers.back().n_out, ld_out, columns, es), work = bytes(workspace, w.total);
  bool const clash = mx4_rows ? overlap(out, bytes(codes, columns * first.steps * 64)) ||
                                    overlap(work, bytes(codes, columns * first.steps * 64)) ||
                                    overlap(out, bytes(scales, columns * first.steps * 4)) ||
                                    overlap(work, bytes(scales, columns * first.steps * 4))
                              : overlap(out, array(x, first.n_in, ld_in, columns, es)) ||
                                    overlap(work, array(x, first.n_in, ld_in, columns, es));
  Range const groups = bytes(offsets, offsets != nullptr ? (int64_t(e->num_experts) + 1) * 4 : 0);
  if (clash || overlap(out, work) || overlap(out, groups) || overlap(work, groups))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "input, offsets, output and workspace must not overlap");
  if ((st = check_ready(*e)) != PONNI_OK) return st;
  char* base = static_cast<char*>(workspace);
  Rows rows;  // the caller's 4-bit ones
  if (mx4_rows) {
    rows.data = static_cast<char*>(const_cast<void*>(codes));
    rows.scales = static_cast<unsigned char*>(const_cast<void*>(scales));
    rows.stride = int64_t(first.steps) * 64;
    rows.scale_stride = int64_t(first.steps) * 4;
    rows.scale_step = 4;
  }
  return run_layers(*e, mx4_rows ? nullptr : x, ld_in, rows, columns, nullptr, offsets, columns, y, ld_out, base, w,
                    nullptr, stream);
}

int mixture_impl(ponni_experts e, const void* x, int64_t ld_in, const ponni_routing* r, void* y, int64_t ld_out,
                 void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (e == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null");
  if (r == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "routing is null");
  int st = check_routing_sizes(r->num_experts, r->top_k, r->batch);
  if (st != PONNI_OK) return st;
  if (r->num_experts != e->num_experts)
    return fail(PONNI_ERR_SHAPE, "the routing is for " + std::to_string(r->num_experts) + " experts, the networks are " +
                                     std::to_string(e->num_experts));
  if (x == nullptr || y == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "input or output pointer is null");
  if (r->weights == nullptr || r->slots == nullptr || r->source == nullptr || r->offsets == nullptr)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "a routing array is null");
  if (ld_in < r->batch || ld_out < r->batch)
    return fail(PONNI_ERR_SHAPE, "row strides are smaller than the batch");
  int64_t const columns = r->batch * r->top_k, es = element_bytes(e->dtype);
  auto const& first = e->layers.front();
  auto const& last = e->layers.back();
  Workspace const w = workspace_of(*e, r->batch, columns, true);
  if ((st = check_workspace(workspace, workspace_bytes, w.total)) != PONNI_OK) return st;
  Range const in = array(x, first.n_in, ld_in, r->batch, es), out = array(y, last.n_out, ld_out, r->batch, es),
              work = bytes(workspace, w.total);
  bool clash = overlap(in, out) || overlap(in, work) || overlap(out, work);
  Range arrays[kRoutingArrays];
  routing_ranges(*r, arrays);
  for (int i = 0; i < 4; i++) clash = clash || overlap(arrays[i], out) || overlap(arrays[i], work);
  if (clash)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "input, routing arrays, output and workspace must not overlap");
  if ((st = check_ready(*e)) != PONNI_OK) return st;
  char* base = static_cast<char*>(workspace);
  Rows result;
  st = run_layers(*e, x, ld_in, Rows{}, r->batch, r->source, r->offsets, columns, nullptr, 0, base, w, &result, stream);
  if (st != PONNI_OK) return st;
  hipError_t const err = launch_combine(e->dtype, result, columns, *r, last.n_out, y, ld_out, stream);
  return err == hipSuccess ? PONNI_OK : device_error("weighted sum", err);
}

// ActCode of an activation layer, -1 for one the expert kernels do not have.
int activation_of(ponni_layer_desc const& d) {
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

int create_impl(const ponni_layer_desc* descs, int32_t n, int32_t num_experts, int32_t dtype, int32_t weights,
                ponni_experts* out) {
  if (out == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "out_experts is null");
  *out = nullptr;
  if (descs == nullptr || n <= 0) return fail(PONNI_ERR_INVALID_ARGUMENT, "no layers");
  if (num_experts < 1 || num_experts > PONNI_MAX_EXPERTS)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "num_experts must be 1 to " + std::to_string(PONNI_MAX_EXPERTS));
  if (weights != PONNI_WEIGHTS_SAME && weights != PONNI_WEIGHTS_MX4)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "unknown weight format");
  if (!data_type(dtype)) return fail(PONNI_ERR_UNSUPPORTED, "expert networks are F32, F16 or BF16");
  if (weights == PONNI_WEIGHTS_MX4 && dtype == PONNI_F32)
    return fail(PONNI_ERR_UNSUPPORTED, "networks with 4-bit weights are F16 or BF16");
  auto e = std::make_unique<ponni_experts_s>();
  e->descs.assign(descs, descs + n);
  e->num_experts = num_experts;
  e->dtype = dtype;
  e->operand = weights == PONNI_WEIGHTS_MX4 ? OPERAND_MX4
               : dtype == PONNI_F32         ? OPERAND_F32
               : dtype == PONNI_F16         ? OPERAND_F16
                                            : OPERAND_BF16;
  for (int32_t i = 0; i < n; i++) {
    ponni_layer_desc const& d = descs[i];
    std::string const at = "layer " + std::to_string(i);
    if (d.n_in < 1 || d.n_out < 1 || d.n_in > kMaxWidth || d.n_out > kMaxWidth)
      return fail(PONNI_ERR_INVALID_MODEL, at + ": widths must be 1 to " + std::to_string(kMaxWidth));
    if (i > 0 && d.n_in != descs[i - 1].n_out)
      return fail(PONNI_ERR_INVALID_MODEL, at + ": its inputs are not the outputs of the layer before it");
    if (d.kind == PONNI_LAYER_MATVEC) {
      ponni_experts_s::Layer l;
      l.n_in = d.n_in;
      l.n_out = d.n_out;
      l.matvec = i;
      l.steps = static_cast<int32_t>(contraction_steps(e->operand, d.n_in));
      l.blocks = (d.n_out + 63) / 64;
      if (e->operand == OPERAND_MX4) l.blocks += l.blocks % 2;  // a row's padding to 128 features is written too
      e->layers.push_back(l);
      continue;
    }
    if (e->layers.empty()) return fail(PONNI_ERR_INVALID_MODEL, at + ": the chain must begin with a Matvec");
    if (d.n_in != d.n_out) return fail(PONNI_ERR_INVALID_MODEL, at + ": a pointwise layer keeps its width");
    auto& l = e->layers.back();
    if (d.kind == PONNI_LAYER_BIAS) {
      if (l.bias >= 0 || l.act != 0)
        return fail(PONNI_ERR_UNSUPPORTED, at + ": a Bias must follow a Matvec");
      l.bias = i;
      continue;
    }
    int const act = activation_of(d);
    if (act < 0)
      return fail(PONNI_ERR_UNSUPPORTED, at + ": expert networks take Matvec, Bias, Relu, LeakyRelu, Gelu, Silu, "
                                              "Sigmoid and Tanh");
    if (l.act != 0) return fail(PONNI_ERR_UNSUPPORTED, at + ": one activation after a Matvec and its Bias");
    l.act = act;
    l.act_a = static_cast<float>(d.attr[0]);
  }
  *out = e.release();
  return PONNI_OK;
}

int64_t param_count(ponni_experts_s const& e, int32_t layer) {
  ponni_layer_desc const& d = e.descs[layer];
  int64_t const one = d.kind == PONNI_LAYER_MATVEC ? int64_t(d.n_in) * d.n_out : d.kind == PONNI_LAYER_BIAS ? d.n_in : 0;
  return one * e.num_experts;
}

int set_params_impl(ponni_experts e, int32_t layer, const void* values, int32_t dtype, int64_t count, int32_t on_device,
                    hipStream_t stream) {
  if (e == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null");
  if (layer < 0 || layer >= static_cast<int32_t>(e->descs.size()))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "no layer " + std::to_string(layer));
  if (values == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "values is null");
  if (!data_type(dtype) && dtype != PONNI_F64) return fail(PONNI_ERR_INVALID_ARGUMENT, "unknown dtype");
  int64_t const want = param_count(*e, layer);
  if (want == 0) return fail(PONNI_ERR_INVALID_ARGUMENT, "layer " + std::to_string(layer) + " has no parameters");
  if (count != want)
    return fail(PONNI_ERR_SHAPE, "layer " + std::to_string(layer) + " has " + std::to_string(want) + " parameters, got " +
                                     std::to_string(count));
  int device = 0;
  hipError_t err = hipGetDevice(&device);
  if (err != hipSuccess) return device_error("hipGetDevice", err);
  if (e->device >= 0 && device != e->device)
    return fail(PONNI_ERR_DEVICE, "the expert networks' parameters are on another device");
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &capturing) != hipSuccess || capturing != hipStreamCaptureStatusNone)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "parameters cannot be set on a stream that is being captured");
  auto& l = *std::find_if(e->layers.begin(), e->layers.end(),
                          [&](auto const& x) { return x.matvec == layer || x.bias == layer; });
  void* staged = nullptr;
  if (!on_device) {
    int64_t const size = count * element_bytes(dtype);
    if ((err = hipMalloc(&staged, size)) != hipSuccess) return device_error("hipMalloc", err);
    if ((err = hipMemcpyAsync(staged, values, size, hipMemcpyHostToDevice, stream)) != hipSuccess) {
      (void)hipFree(staged);
      return device_error("hipMemcpy", err);
    }
    values = staged;
  }
  // Calls in flight on any stream, and graphs, read the buffers that are there: they are waited
  // for, and written in place.  Until that has ended well the layer counts as not set.
  if (l.weights != nullptr || l.d_bias != nullptr) err = hipDeviceSynchronize();
  bool const weights_set = l.weights_set;
  if (err == hipSuccess) l.weights_set = false;
  auto allocate = [&](auto*& p, int64_t n) {
    if (p != nullptr) return hipSuccess;
    hipError_t const status = hipMalloc(reinterpret_cast<void**>(&p), n);
    if (status == hipSuccess) e->device = device;
    return status;
  };
  if (err == hipSuccess) {
    if (l.matvec == layer) {
      int64_t const fragments = int64_t(e->num_experts) * l.blocks * l.steps;
      err = allocate(l.weights, fragments * 4096);
      if (err == hipSuccess && e->operand == OPERAND_MX4) err = allocate(l.scales, fragments * 256);
      if (err == hipSuccess)
        err = launch_pack_weights(e->operand, dtype, values, e->num_experts, l.n_in, l.n_out, l.blocks, l.weights,
                                  l.scales, stream);
    } else {
      int64_t const padded = int64_t(l.blocks) * 64;
      err = allocate(l.d_bias, e->num_experts * padded * 4);
      if (err == hipSuccess) err = launch_pack_bias(dtype, values, e->num_experts, l.n_out, padded, l.d_bias, stream);
    }
  }
  hipError_t const done = hipStreamSynchronize(stream);
  if (staged != nullptr) (void)hipFree(staged);
  if (err == hipSuccess) err = done;
  if (err != hipSuccess) return device_error("setting parameters", err);
  l.weights_set = weights_set || l.matvec == layer;
  return PONNI_OK;
}

int check_mx4(const void* codes, const void* scales, const void* values, int64_t ld, int32_t dtype, int64_t features,
              int64_t columns) {
  if (features < 1 || features > kMaxWidth)
    return fail(PONNI_ERR_SHAPE, "features must be 1 to " + std::to_string(kMaxWidth));
  if (columns < 1 || columns > PONNI_MAX_COLUMNS)
    return fail(PONNI_ERR_SHAPE, "columns must be 1 to " + std::to_string(PONNI_MAX_COLUMNS));
  if (codes == nullptr || scales == nullptr || values == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "null array");
  if (!aligned(codes, 16) || !aligned(scales, 16))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "codes and scales must be at multiples of 16 bytes");
  if (!data_type(dtype)) return fail(PONNI_ERR_UNSUPPORTED, "values are F32, F16 or BF16");
  if (ld < columns) return fail(PONNI_ERR_SHAPE, "row stride is smaller than the number of columns");
  Range const a = array(values, features, ld, columns, element_bytes(dtype)),
              b = bytes(codes, columns * contraction_steps(OPERAND_MX4, features) * 64),
              c = bytes(scales, columns * contraction_steps(OPERAND_MX4, features) * 4);
  if (overlap(a, b) || overlap(a, c) || overlap(b, c))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "values, codes and scales must not overlap");
  return PONNI_OK;
}

Rows mx4_rows(const void* codes, const void* scales, int64_t features) {
  Rows r;
  r.data = static_cast<char*>(const_cast<void*>(codes));
  r.scales = static_cast<unsigned char*>(const_cast<void*>(scales));
  r.stride = contraction_steps(OPERAND_MX4, features) * 64;
  r.scale_stride = contraction_steps(OPERAND_MX4, features) * 4;
  r.scale_step = 4;
  return r;
}

}  // namespace
}  // namespace ponni_hip

using namespace ponni_hip;

extern "C" {

int64_t ponni_route_workspace_bytes(int32_t num_experts, int32_t top_k, int64_t batch) {
  int64_t n = -1;
  (void)guarded([&] {
    int const st = check_routing_sizes(num_experts, top_k, batch);
    if (st == PONNI_OK) n = route_workspace_bytes_up_to(num_experts, batch);
    return st;
  });
  return n;
}

int ponni_route(const void* scores, int64_t ld, int32_t dtype, int32_t normalize, const ponni_routing* r, void* workspace,
                int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] {
    if (r == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "routing is null");
    int st = check_routing_sizes(r->num_experts, r->top_k, r->batch);
    if (st != PONNI_OK) return st;
    if (scores == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "scores is null");
    if (!data_type(dtype)) return fail(PONNI_ERR_UNSUPPORTED, "scores are F32, F16 or BF16");
    if (normalize != PONNI_ROUTE_CHOSEN && normalize != PONNI_ROUTE_ALL)
      return fail(PONNI_ERR_INVALID_ARGUMENT, "unknown normalization");
    if (!r->experts || !r->weights || !r->slots || !r->source || !r->offsets)
      return fail(PONNI_ERR_INVALID_ARGUMENT, "a routing array is null");
    if (ld < r->batch) return fail(PONNI_ERR_SHAPE, "row stride is smaller than the batch");
    st = check_workspace(workspace, workspace_bytes, route_workspace_bytes(r->num_experts, r->batch));
    if (st != PONNI_OK) return st;
    Range arrays[kRoutingArrays];
    routing_ranges(*r, arrays);
    Range const in = array(scores, r->num_experts, ld, r->batch, element_bytes(dtype)),
                work = bytes(workspace, route_workspace_bytes(r->num_experts, r->batch));
    bool clash = overlap(in, work);
    for (int i = 0; i < kRoutingArrays; i++) {
      clash = clash || overlap(arrays[i], in) || overlap(arrays[i], work);
      for (int j = 0; j < i; j++) clash = clash || overlap(arrays[i], arrays[j]);
    }
    if (clash)
      return fail(PONNI_ERR_INVALID_ARGUMENT, "scores, routing arrays and workspace must not overlap");
    hipError_t const err = launch_route(scores, ld, dtype, normalize, *r, workspace, stream);
    return err == hipSuccess ? int(PONNI_OK) : device_error("routing", err);
  });
}

int64_t ponni_mx4_code_bytes(int64_t features) { return features < 1 ? -1 : contraction_steps(OPERAND_MX4, features) * 64; }
int64_t ponni_mx4_scale_bytes(int64_t features) { return features < 1 ? -1 : contraction_steps(OPERAND_MX4, features) * 4; }

int ponni_mx4_quantize(const void* x, int64_t ld, int32_t dtype, int64_t features, int64_t columns, void* codes,
                       void* scales, hipStream_t stream) {
  return guarded([&] {
    int const st = check_mx4(codes, scales, x, ld, dtype, features, columns);
    if (st != PONNI_OK) return st;
    hipError_t const err =
        launch_to_rows(OPERAND_MX4, dtype, x, ld, features, columns, mx4_rows(codes, scales, features), stream);
    return err == hipSuccess ? int(PONNI_OK) : device_error("quantisation", err);
  });
}

int ponni_mx4_dequantize(const void* codes, const void* scales, int64_t features, int64_t columns, void* y, int64_t ld,
                         int32_t dtype, hipStream_t stream) {
  return guarded([&] {
    int const st = check_mx4(codes, scales, y, ld, dtype, features, columns);
    if (st != PONNI_OK) return st;
    hipError_t const err = launch_mx4_values(mx4_rows(codes, scales, features), features, columns, y, ld, dtype, stream);
    return err == hipSuccess ? int(PONNI_OK) : device_error("dequantisation", err);
  });
}

int ponni_experts_create(const ponni_layer_desc* layers, int32_t num_layers, int32_t num_experts, int32_t dtype,
                         int32_t weights, ponni_experts* out_experts) {
  return guarded([&] { return create_impl(layers, num_layers, num_experts, dtype, weights, out_experts); });
}

void ponni_experts_destroy(ponni_experts e) {
  if (e == nullptr) return;
  for (auto& l : e->layers) {
    (void)hipFree(l.weights);
    (void)hipFree(l.scales);
    (void)hipFree(l.d_bias);
  }
  delete e;
}

int64_t ponni_experts_layer_param_count(ponni_experts e, int32_t layer) {
  if (e == nullptr || layer < 0 || layer >= static_cast<int32_t>(e->descs.size())) {
    (void)guarded([&] { return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null or has no such layer"); });
    return -1;
  }
  return param_count(*e, layer);
}

int ponni_experts_set_layer_params(ponni_experts e, int32_t layer, const void* values, int32_t dtype, int64_t count,
                                   int32_t on_device, hipStream_t stream) {
  return guarded([&] { return set_params_impl(e, layer, values, dtype, count, on_device, stream); });
}

int ponni_experts_forward(ponni_experts e, const void* x, int64_t ld_in, const int32_t* offsets, void* y, int64_t ld_out,
                          int64_t columns, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] {
    return forward_impl(e, x, ld_in, nullptr, nullptr, false, offsets, y, ld_out, columns, workspace, workspace_bytes,
                        stream);
  });
}

int ponni_experts_forward_mx4(ponni_experts e, const void* codes, const void* scales, const int32_t* offsets, void* y,
                              int64_t ld_out, int64_t columns, void* workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  return guarded([&] {
    return forward_impl(e, nullptr, 0, codes, scales, true, offsets, y, ld_out, columns, workspace, workspace_bytes,
                        stream);
  });
}

int64_t ponni_experts_workspace_bytes(ponni_experts e, int64_t columns) {
  int64_t n = -1;
  (void)guarded([&] {
    if (e == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null");
    if (columns <= 0 || columns > PONNI_MAX_COLUMNS)
      return fail(PONNI_ERR_SHAPE, "columns must be 1 to " + std::to_string(PONNI_MAX_COLUMNS));
    n = workspace_bytes_up_to(*e, 0, columns);
    return int(PONNI_OK);
  });
  return n;
}

int ponni_experts_forward_mixture(ponni_experts e, const void* x, int64_t ld_in, const ponni_routing* routing, void* y,
                                  int64_t ld_out, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] { return mixture_impl(e, x, ld_in, routing, y, ld_out, workspace, workspace_bytes, stream); });
}

int64_t ponni_experts_mixture_workspace_bytes(ponni_experts e, int32_t top_k, int64_t batch) {
  int64_t n = -1;
  (void)guarded([&] {
    if (e == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "experts is null");
    int const st = check_routing_sizes(e->num_experts, top_k, batch);
    if (st == PONNI_OK) n = workspace_bytes_up_to(*e, top_k, batch);
    return st;
  });
  return n;
}

}  // extern "C"
