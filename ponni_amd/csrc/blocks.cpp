// C ABI of gated blocks, the norms between blocks and log probabilities: argument checks and launches
// (kernels_gated.hip, norm.h, kernels_logp.hip).
#include "blocks.h"

#include <cmath>
#include <initializer_list>
#include <string>

#include "abi_checks.h"

namespace ponni_hip {
namespace {

// An array of a call: rows of `columns` elements, `ld` apart.
struct Array {
  char const* what;
  void const* p;
  int64_t rows, columns, ld, es;
};
// Whether two arrays share an element (arrays of equal row strides may be column ranges of one).
bool share(Array const& a, Array const& b) {
  if (a.p == nullptr || b.p == nullptr || a.rows * a.columns == 0 || b.rows * b.columns == 0) return false;
  if (!overlap(array(a.p, a.rows, a.ld, a.columns, a.es), array(b.p, b.rows, b.ld, b.columns, b.es))) return false;
  int64_t const pitch = a.ld * a.es;
  if (a.rows == 1 || b.rows == 1 || pitch != b.ld * b.es) return true;
  int64_t const distance = int64_t(reinterpret_cast<uint64_t>(b.p) - reinterpret_cast<uint64_t>(a.p)) % pitch;
  int64_t const at = distance < 0 ? distance + pitch : distance;
  return at < a.columns * a.es || at + b.columns * b.es > pitch;
}

int check_arrays(std::initializer_list<Array> read, std::initializer_list<Array> written) {
  for (auto const* list : {&read, &written})
    for (Array const& a : *list)
      if (a.p != nullptr && a.rows > 1 && a.ld < a.columns)
        return fail(PONNI_ERR_SHAPE, std::string("the row stride of ") + a.what + " is smaller than its number of columns");
  for (auto w = written.begin(); w != written.end(); w++) {
    for (Array const& r : read)
      if (share(*w, r)) return fail(PONNI_ERR_INVALID_ARGUMENT, std::string(w->what) + " overlaps " + r.what);
    for (auto v = written.begin(); v != w; v++)
      if (share(*w, *v)) return fail(PONNI_ERR_INVALID_ARGUMENT, std::string(w->what) + " overlaps " + v->what);
  }
  return PONNI_OK;
}
Array whole(char const* what, void const* p, int64_t n, int64_t es) { return {what, p, 1, n, n, es}; }

int launched(char const* what, hipError_t err) { return err == hipSuccess ? int(PONNI_OK) : device_error(what, err); }

// -- gated blocks -----------------------------------------------------------------------

int check_gated_sizes(ponni_gated const* b, int64_t columns) {
  if (b == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "block is null");
  for (int32_t n : {b->n_in, b->n_hidden, b->n_out})
    if (n < 1 || n > kMaxWidth)
      return fail(PONNI_ERR_INVALID_MODEL, "widths must be 1 to " + std::to_string(kMaxWidth));
  if (!data_type(b->dtype)) return fail(PONNI_ERR_UNSUPPORTED, "gated blocks are F32, F16 or BF16");
  if (activation_of(b->act) < 0)
    return fail(PONNI_ERR_UNSUPPORTED, "the activation of a gated block is Relu, LeakyRelu, Gelu, Silu, Sigmoid or Tanh");
  if (b->act.n_in != b->n_hidden || b->act.n_out != b->n_hidden)
    return fail(PONNI_ERR_INVALID_MODEL, "the activation's width is not the block's n_hidden");
  if (columns <= 0) return fail(PONNI_ERR_SHAPE, "gated blocks require a nonzero number of columns");
  if (columns > PONNI_GATED_MAX_COLUMNS)
    return fail(PONNI_ERR_SHAPE, "columns exceed " + std::to_string(PONNI_GATED_MAX_COLUMNS));
  return PONNI_OK;
}

int check_strides(std::initializer_list<int64_t> strides) {
  for (int64_t ld : strides)
    if (ld > PONNI_GATED_MAX_COLUMNS)
      return fail(PONNI_ERR_SHAPE, "a row stride exceeds " + std::to_string(PONNI_GATED_MAX_COLUMNS));
  return PONNI_OK;
}

int gated_impl(ponni_gated const* b, void const* x, int64_t ld_x, void* y, int64_t ld_y, void* states, int64_t ld_states,
               int64_t columns, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  int st = check_gated_sizes(b, columns);
  if (st != PONNI_OK) return st;
  if (!b->gate || !b->up || !b->down) return fail(PONNI_ERR_INVALID_ARGUMENT, "a weight array is null");
  if (x == nullptr || y == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "input or output pointer is null");
  GatedArrays const arrays{x, ld_x, states, ld_states, nullptr, 0};
  int64_t const need = gated_workspace_bytes(*b, columns, false, &arrays), es = element_bytes(b->dtype);
  if ((st = check_workspace(workspace, workspace_bytes, need)) != PONNI_OK) return st;
  if ((st = check_strides({ld_x, ld_y, states ? ld_states : 0, b->ld_gate, b->ld_up, b->ld_down})) != PONNI_OK) return st;
  st = check_arrays({{"x", x, b->n_in, columns, ld_x, es},
                     {"the gate weights", b->gate, b->n_in, b->n_hidden, b->ld_gate, es},
                     {"the up weights", b->up, b->n_in, b->n_hidden, b->ld_up, es},
                     {"the down weights", b->down, b->n_hidden, b->n_out, b->ld_down, es},
                     whole("the gate bias", b->gate_bias, b->n_hidden, es),
                     whole("the up bias", b->up_bias, b->n_hidden, es),
                     whole("the down bias", b->down_bias, b->n_out, es)},
                    {{"y", y, b->n_out, columns, ld_y, es},
                     {"states", states, 3 * int64_t(b->n_hidden), columns, ld_states, es},
                     whole("workspace", workspace, need, 1)});
  if (st != PONNI_OK) return st;
  return launched("gated block", launch_gated(*b, activation_of(b->act), x, ld_x, y, ld_y, states, ld_states, columns,
                                              workspace, stream));
}

int gated_backward_impl(ponni_gated const* b, void const* x, int64_t ld_x, void const* states, int64_t ld_states,
                        void const* dy, int64_t ld_dy, int64_t columns, ponni_gated_gradients const* d, void* workspace,
                        int64_t workspace_bytes, hipStream_t stream) {
  int st = check_gated_sizes(b, columns);
  if (st != PONNI_OK) return st;
  if (d == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "gradients is null");
  if (!b->gate || !b->up || !b->down) return fail(PONNI_ERR_INVALID_ARGUMENT, "a weight array is null");
  if (!x || !states || !dy) return fail(PONNI_ERR_INVALID_ARGUMENT, "x, states or dy is null");
  GatedArrays const arrays{x, ld_x, states, ld_states, dy, ld_dy};
  int64_t const need = gated_workspace_bytes(*b, columns, true, &arrays), es = element_bytes(b->dtype);
  if ((st = check_workspace(workspace, workspace_bytes, need)) != PONNI_OK) return st;
  st = check_strides({ld_x, ld_states, ld_dy, b->ld_gate, b->ld_up, b->ld_down, d->x ? d->ld_x : 0, d->gate ? d->ld_gate : 0,
                      d->up ? d->ld_up : 0, d->down ? d->ld_down : 0});
  if (st != PONNI_OK) return st;
  st = check_arrays({{"x", x, b->n_in, columns, ld_x, es},
                     {"states", states, 3 * int64_t(b->n_hidden), columns, ld_states, es},
                     {"dy", dy, b->n_out, columns, ld_dy, es},
                     {"the gate weights", b->gate, b->n_in, b->n_hidden, b->ld_gate, es},
                     {"the up weights", b->up, b->n_in, b->n_hidden, b->ld_up, es},
                     {"the down weights", b->down, b->n_hidden, b->n_out, b->ld_down, es}},
                    {{"the gradient of x", d->x, b->n_in, columns, d->ld_x, es},
                     {"the gradient of the gate weights", d->gate, b->n_in, b->n_hidden, d->ld_gate, es},
                     {"the gradient of the up weights", d->up, b->n_in, b->n_hidden, d->ld_up, es},
                     {"the gradient of the down weights", d->down, b->n_hidden, b->n_out, d->ld_down, es},
                     whole("the gradient of the gate bias", d->gate_bias, b->n_hidden, es),
                     whole("the gradient of the up bias", d->up_bias, b->n_hidden, es),
                     whole("the gradient of the down bias", d->down_bias, b->n_out, es),
                     whole("workspace", workspace, need, 1)});
  if (st != PONNI_OK) return st;
  return launched("gradients of a gated block",
                  launch_gated_backward(*b, activation_of(b->act), x, ld_x, states, ld_states, dy, ld_dy, columns, *d,
                                        workspace, stream));
}

// -- norms between blocks -------------------------------------------------------------

int check_norm_sizes(int64_t n, int32_t dtype, int64_t columns) {
  if (n < 1 || n > kMaxWidth) return fail(PONNI_ERR_SHAPE, "n must be 1 to " + std::to_string(kMaxWidth));
  if (!data_type(dtype)) return fail(PONNI_ERR_UNSUPPORTED, "norms between blocks are F32, F16 or BF16");
  if (columns <= 0) return fail(PONNI_ERR_SHAPE, "norms require a nonzero number of columns");
  if (columns > PONNI_MAX_COLUMNS) return fail(PONNI_ERR_SHAPE, "columns exceed " + std::to_string(PONNI_MAX_COLUMNS));
  return PONNI_OK;
}

int check_norms(ponni_residual_norm const* r) {
  if (r == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "residual norm is null");
  int const st = check_norm_sizes(r->n, r->dtype, r->columns);
  if (st != PONNI_OK) return st;
  for (ponni_norm const* n : {&r->after, &r->before}) {
    if (n->kind != PONNI_NORM_NONE && n->kind != PONNI_NORM_RMS && n->kind != PONNI_NORM_LAYER)
      return fail(PONNI_ERR_INVALID_ARGUMENT, "unknown kind of norm");
    if (n->kind == PONNI_NORM_NONE && (n->weight != nullptr || n->bias != nullptr))
      return fail(PONNI_ERR_INVALID_ARGUMENT, "weights of no norm");
    if (n->kind != PONNI_NORM_NONE && !(n->eps >= 0.0f))
      return fail(PONNI_ERR_INVALID_ARGUMENT, "a norm's eps must not be negative");
  }
  if (r->x == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "x is null");
  if (r->gate != nullptr && r->feature_gate != nullptr)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "a gate has one value per feature, or one per feature and column");
  return PONNI_OK;
}

int residual_norm_impl(ponni_residual_norm const* r, hipStream_t stream) {
  int st = check_norms(r);
  if (st != PONNI_OK) return st;
  if (r->normed != nullptr && r->before.kind == PONNI_NORM_NONE)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "normed without a norm before the next block");
  if (r->state == nullptr && r->normed == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "state and normed are null");
  int64_t const es = element_bytes(r->dtype), n = r->n, c = r->columns;
  st = check_arrays({{"x", r->x, n, c, r->ld_x, es},
                     {"residual", r->residual, n, c, r->ld_residual, es},
                     {"gate", r->gate, n, c, r->ld_gate, es},
                     whole("feature_gate", r->feature_gate, n, 4),
                     whole("the weight after", r->after.weight, n, 4),
                     whole("the bias after", r->after.bias, n, 4),
                     whole("the weight before", r->before.weight, n, 4),
                     whole("the bias before", r->before.bias, n, 4)},
                    {{"state", r->state, n, c, r->ld_state, es},
                     {"normed", r->normed, n, c, r->ld_normed, es},
                     whole("statistics", r->statistics, 4 * c, 4)});
  if (st != PONNI_OK) return st;
  return launched("norms", launch_residual_norm(*r, stream));
}

int residual_norm_backward_impl(ponni_residual_norm const* r, ponni_residual_norm_gradients const* g, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  int st = check_norms(r);
  if (st != PONNI_OK) return st;
  if (g == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "gradients is null");
  if (r->statistics == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "statistics is null");
  if (g->d_normed != nullptr && r->before.kind == PONNI_NORM_NONE)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "d_normed without a norm before the next block");
  if ((g->d_gate != nullptr) && r->gate == nullptr)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "d_gate without a gate of every feature and column");
  if (g->d_feature_gate != nullptr && r->gate != nullptr)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "d_feature_gate beside a gate of every feature and column");
  // (a norm without a weight or bias has their gradients all the same, at ones and zeros)
  struct Parameter {
    char const* what;
    float const* gradient;
    int32_t kind;
  };
  for (Parameter const& p : {Parameter{"d_after_weight", g->d_after_weight, r->after.kind},
                             Parameter{"d_after_bias", g->d_after_bias, r->after.kind},
                             Parameter{"d_before_weight", g->d_before_weight, r->before.kind},
                             Parameter{"d_before_bias", g->d_before_bias, r->before.kind}})
    if (p.gradient != nullptr && p.kind == PONNI_NORM_NONE)
      return fail(PONNI_ERR_INVALID_ARGUMENT, std::string(p.what) + " without such a norm");
  int64_t const es = element_bytes(r->dtype), n = r->n, c = r->columns, need = residual_norm_workspace_bytes(r->n, c);
  if ((st = check_workspace(workspace, workspace_bytes, need)) != PONNI_OK) return st;
  st = check_arrays({{"x", r->x, n, c, r->ld_x, es},
                     {"residual", r->residual, n, c, r->ld_residual, es},
                     {"gate", r->gate, n, c, r->ld_gate, es},
                     {"d_state", g->d_state, n, c, g->ld_d_state, es},
                     {"d_normed", g->d_normed, n, c, g->ld_d_normed, es},
                     whole("feature_gate", r->feature_gate, n, 4),
                     whole("the weight after", r->after.weight, n, 4),
                     whole("the bias after", r->after.bias, n, 4),
                     whole("the weight before", r->before.weight, n, 4),
                     whole("the bias before", r->before.bias, n, 4),
                     whole("statistics", r->statistics, 4 * c, 4)},
                    {{"d_x", g->d_x, n, c, g->ld_d_x, es},
                     {"d_residual", g->d_residual, n, c, g->ld_d_residual, es},
                     {"d_gate", g->d_gate, n, c, g->ld_d_gate, es},
                     whole("d_feature_gate", g->d_feature_gate, n, 4),
                     whole("d_after_weight", g->d_after_weight, n, 4),
                     whole("d_after_bias", g->d_after_bias, n, 4),
                     whole("d_before_weight", g->d_before_weight, n, 4),
                     whole("d_before_bias", g->d_before_bias, n, 4),
                     whole("workspace", workspace, need, 1)});
  if (st != PONNI_OK) return st;
  return launched("gradients of norms", launch_residual_norm_backward(*r, *g, workspace, stream));
}

// -- log probabilities --------------------------------------------------------------

int check_logp_sizes(int64_t classes, int64_t columns, int64_t top_k) {
  if (classes < 1 || classes > PONNI_MAX_COLUMNS)
    return fail(PONNI_ERR_SHAPE, "classes must be 1 to " + std::to_string(PONNI_MAX_COLUMNS));
  if (columns <= 0) return fail(PONNI_ERR_SHAPE, "log probabilities require a nonzero number of columns");
  if (columns > PONNI_MAX_COLUMNS) return fail(PONNI_ERR_SHAPE, "columns exceed " + std::to_string(PONNI_MAX_COLUMNS));
  int64_t const most = classes < PONNI_MAX_TOP_K ? classes : PONNI_MAX_TOP_K;
  if (top_k < 0 || top_k > most)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "top_k must be 0 to " + std::to_string(most));
  return PONNI_OK;
}

int check_logp(ponni_log_probs const* p) {
  if (p == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "log_probs is null");
  int const st = check_logp_sizes(p->classes, p->columns, p->top_k);
  if (st != PONNI_OK) return st;
  if (!data_type(p->dtype)) return fail(PONNI_ERR_UNSUPPORTED, "logits are F32, F16 or BF16");
  if (!p->logits || !p->entropy || !p->log_normalizer)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "logits, entropy or log_normalizer is null");
  return PONNI_OK;
}

int log_probs_impl(ponni_log_probs const* p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  int st = check_logp(p);
  if (st != PONNI_OK) return st;
  if ((p->targets == nullptr) != (p->log_probs == nullptr))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "targets and log_probs go together");
  if (p->top_k > 0 && (!p->top_classes || !p->top_log_probs))
    return fail(PONNI_ERR_INVALID_ARGUMENT, "an array of the top classes is null");
  int64_t const need = logp_workspace_bytes(p->classes, p->columns, p->dtype, p->top_k), c = p->columns;
  if ((st = check_workspace(workspace, workspace_bytes, need)) != PONNI_OK) return st;
  st = check_arrays({{"logits", p->logits, p->classes, c, p->ld, element_bytes(p->dtype)},
                     whole("targets", p->targets, c, 4)},
                    {whole("log_probs", p->log_probs, c, 4),
                     whole("entropy", p->entropy, c, 4),
                     whole("log_normalizer", p->log_normalizer, c, 4),
                     whole("top_classes", p->top_k > 0 ? p->top_classes : nullptr, p->top_k * c, 4),
                     whole("top_log_probs", p->top_k > 0 ? p->top_log_probs : nullptr, p->top_k * c, 4),
                     whole("workspace", workspace, need, 1)});
  if (st != PONNI_OK) return st;
  return launched("log probabilities", launch_logp(*p, workspace, stream));
}

int log_probs_backward_impl(ponni_log_probs const* p, float const* d_log_probs, float const* d_entropy,
                            float const* d_log_normalizer, void* d_logits, int64_t ld_d_logits, hipStream_t stream) {
  int st = check_logp(p);
  if (st != PONNI_OK) return st;
  if (d_log_probs != nullptr && p->targets == nullptr)
    return fail(PONNI_ERR_INVALID_ARGUMENT, "d_log_probs without targets");
  if (d_logits == nullptr) return fail(PONNI_ERR_INVALID_ARGUMENT, "d_logits is null");
  int64_t const c = p->columns, es = element_bytes(p->dtype);
  bool const in_place = d_logits == p->logits && (p->classes == 1 || ld_d_logits == p->ld);
  st = check_arrays({{"logits", in_place ? nullptr : p->logits, p->classes, c, p->ld, es},
                     whole("targets", p->targets, c, 4), whole("entropy", p->entropy, c, 4),
                     whole("log_normalizer", p->log_normalizer, c, 4), whole("d_log_probs", d_log_probs, c, 4),
                     whole("d_entropy", d_entropy, c, 4), whole("d_log_normalizer", d_log_normalizer, c, 4)},
                    {{"d_logits", d_logits, p->classes, c, ld_d_logits, es}});
  if (st != PONNI_OK) return st;
  return launched("gradient of log probabilities",
                  launch_logp_backward(*p, d_log_probs, d_entropy, d_log_normalizer, d_logits, ld_d_logits, stream));
}

// A size, or -1 where `check` refuses it.
template <class Check, class Size> int64_t size_or_refusal(Check&& check, Size&& size) {
  int64_t n = -1;
  (void)guarded([&] {
    int const st = check();
    if (st == PONNI_OK) n = size();
    return st;
  });
  return n;
}

}  // namespace
}  // namespace ponni_hip

using namespace ponni_hip;

extern "C" {

int ponni_gated_forward(const ponni_gated* block, const void* x, int64_t ld_x, void* y, int64_t ld_y, void* states,
                        int64_t ld_states, int64_t columns, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream) {
  return guarded([&] {
    return gated_impl(block, x, ld_x, y, ld_y, states, ld_states, columns, workspace, workspace_bytes, stream);
  });
}

int64_t ponni_gated_workspace_bytes(const ponni_gated* block, int64_t columns) {
  return size_or_refusal([&] { return check_gated_sizes(block, columns); },
                         [&] { return gated_workspace_bytes(*block, columns, false); });
}

int ponni_gated_backward(const ponni_gated* block, const void* x, int64_t ld_x, const void* states, int64_t ld_states,
                         const void* dy, int64_t ld_dy, int64_t columns, const ponni_gated_gradients* gradients,
                         void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] {
    return gated_backward_impl(block, x, ld_x, states, ld_states, dy, ld_dy, columns, gradients, workspace,
                               workspace_bytes, stream);
  });
}

int64_t ponni_gated_backward_workspace_bytes(const ponni_gated* block, int64_t columns) {
  return size_or_refusal([&] { return check_gated_sizes(block, columns); },
                         [&] { return gated_workspace_bytes(*block, columns, true); });
}

int64_t ponni_gated_call_workspace_bytes(const ponni_gated* block, const void* x, int64_t ld_x, const void* states,
                                         int64_t ld_states, const void* dy, int64_t ld_dy, int64_t columns) {
  GatedArrays const arrays{x, ld_x, states, ld_states, dy, ld_dy};
  return size_or_refusal([&] { return check_gated_sizes(block, columns); },
                         [&] { return gated_workspace_bytes(*block, columns, dy != nullptr, &arrays); });
}

int ponni_residual_norm_forward(const ponni_residual_norm* r, hipStream_t stream) {
  return guarded([&] { return residual_norm_impl(r, stream); });
}

int ponni_residual_norm_backward(const ponni_residual_norm* r, const ponni_residual_norm_gradients* gradients,
                                 void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] { return residual_norm_backward_impl(r, gradients, workspace, workspace_bytes, stream); });
}

int64_t ponni_residual_norm_workspace_bytes(int32_t n, int32_t dtype, int64_t columns) {
  return size_or_refusal([&] { return check_norm_sizes(n, dtype, columns); },
                         [&] { return residual_norm_workspace_bytes(n, columns); });
}

int ponni_log_probs_forward(const ponni_log_probs* p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return guarded([&] { return log_probs_impl(p, workspace, workspace_bytes, stream); });
}

int64_t ponni_log_probs_workspace_bytes(int64_t classes, int64_t columns, int32_t top_k) {
  return size_or_refusal([&] { return check_logp_sizes(classes, columns, top_k); },
                         [&] { return logp_workspace_bytes_up_to(classes, columns, top_k); });
}

int ponni_log_probs_backward(const ponni_log_probs* p, const float* d_log_probs, const float* d_entropy,
                             const float* d_log_normalizer, void* d_logits, int64_t ld_d_logits, hipStream_t stream) {
  return guarded([&] {
    return log_probs_backward_impl(p, d_log_probs, d_entropy, d_log_normalizer, d_logits, ld_d_logits, stream);
  });
}

}  // extern "C"
