// fastmoe_amd._block: the host side of the router, the norms around a block and the 4-bit weights (not part of the C
// ABI): as in fastmoe_amd._rows, a call allocates its results and calls the C entry point in one go, and a backward
// runs in the engine's thread without the interpreter.
//
// Each function but bind checks its arguments and returns NotImplemented where something is not as it
// takes it, and under tracing; the caller then goes through the checks one by one and says what is wrong.
//
//   bind({name: address}) once, with the library's entry points
//   route(logits, bias | None, top_k, score, groups, top_groups, group score, renormalize, scale, dtype code of
//         the weights, recorded) -> (weights, ids): records its backward if `recorded`
//   sandwich(x, post, residual, pre | None, gate | None, scale, eps, recorded) -> (y | None, stream)
//   quantize_fp4(x) -> (data, scales)
//   restore_fp4(data, scales, features, dtype code) -> values
//   fp4_linear(x, weights' data, scales, features, offsets | None, rows | None, bias | None, activation,
//              dtype code) -> out
constexpr const char* kModuleName = "fastmoe_amd._block";
#include "host_tensors.h"

#include <vector>

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

namespace {

#define FMOE_ENTRIES(X)                          \
  X(fmoe_last_error)                             \
  X(fmoe_route)                                  \
  X(fmoe_route_backward)                         \
  X(fmoe_sandwich_norm)                          \
  X(fmoe_sandwich_norm_backward)                 \
  X(fmoe_sandwich_norm_backward_workspace_bytes) \
  X(fmoe_quantize_fp4)                           \
  X(fmoe_restore_fp4)                            \
  X(fmoe_fp4_linear)

struct Api {
#define FMOE_DECLARE(name) decltype(&::name) name = nullptr;
  FMOE_ENTRIES(FMOE_DECLARE)
#undef FMOE_DECLARE
} api;

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void refuse_capture(const char* what) {
  if (capturing())
    throw std::runtime_error(
        std::string("fastmoe_amd: ") + what +
        " under HIP graph capture is not supported (a captured autograd step once crashed the host in "
        "CUDAGraph.capture_end).  Run the autograd step eagerly.");
}

// A backward under create_graph: gradients that would need one of their own are refused, and results that
// depend on `inputs` say so to whoever differentiates them.
void refuse_second(const variable_list& grads, const char* message) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& g : grads)
    if (g.defined() && g.requires_grad()) throw std::runtime_error(message);
}
void refuse_history(Tensor& t, torch::autograd::edge_list to, const char* message) {
  torch::autograd::set_history(t, std::shared_ptr<torch::autograd::Node>(
                                      new torch::autograd::Error(message, std::move(to)), torch::autograd::deleteNode));
}
void mark_second(std::initializer_list<Tensor*> results, const variable_list& inputs, const char* message) {
  if (!at::GradMode::is_enabled()) return;
  bool any = false;
  for (const Tensor& t : inputs) any |= t.defined() && t.requires_grad();
  if (!any) return;
  for (Tensor* g : results)
    if (g->defined()) refuse_history(*g, torch::autograd::collect_next_edges(inputs), message);
}

// ---- the router -----------------------------------------------------------------------------------

struct Routing {
  Tensor bias;
  int64_t k, groups, top_groups;
  int score, group_score, renormalize, w_dtype;
  float scale;
};

struct Routed {
  Tensor weights, ids, share, rest, norm;
};

Routed run_route(const Tensor& logits, const Routing& o, bool keep) {
  Place place(logits);
  const int64_t T = logits.size(0), E = logits.size(1);
  Routed r;
  r.weights = empty({T, o.k}, logits, type_of(o.w_dtype));
  r.ids = empty({T, o.k}, logits, at::kLong);
  if (keep) {
    r.share = empty({T, o.k}, logits, at::kFloat);
    if (o.score == FMOE_SCORE_SIGMOID) r.rest = empty({T, o.k}, logits, at::kFloat);
    else if (!o.renormalize) r.norm = empty({T, 2}, logits, at::kFloat);
  }
  check(api.fmoe_route(data(logits), pitch(logits), T, E, code(logits.scalar_type()),
                       static_cast<const float*>(data(o.bias)), o.k, o.score, o.groups, o.top_groups,
                       o.group_score, o.renormalize, o.scale, data(r.weights), o.w_dtype,
                       static_cast<int64_t*>(data(r.ids)), static_cast<float*>(data(r.share)),
                       static_cast<float*>(data(r.rest)), static_cast<float*>(data(r.norm)), place.stream),
        "fmoe_route");
  return r;
}

constexpr const char* kNoSecondRoute = "fastmoe_amd: the router's gradient has no gradient of its own";

class Route : public torch::autograd::Function<Route> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor logits, Routing o) {
    Routed r = run_route(logits, o, true);
    // the logits are kept where the gradient reads them
    ctx->save_for_backward({r.norm.defined() ? logits : Tensor(), r.ids, r.share, r.rest, r.norm});
    ctx->saved_data["experts"] = logits.size(1);
    ctx->saved_data["dtype"] = (int64_t)logits.scalar_type();
    ctx->saved_data["renormalize"] = (int64_t)o.renormalize;
    ctx->saved_data["scale"] = (double)o.scale;
    ctx->mark_non_differentiable({r.ids});
    ctx->set_materialize_grads(false);
    return {r.weights, r.ids};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &ids = saved[1], &share = saved[2], &rest = saved[3], &norm = saved[4];
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    refuse_second(grads, kNoSecondRoute);
    Place place(share);
    refuse_capture("the router's backward");
    const Tensor g = by_rows(grads[0]).contiguous();
    const int64_t T = ids.size(0), E = ctx->saved_data["experts"].toInt();
    const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    Tensor out = empty({T, E}, share, dtype);
    check(api.fmoe_route_backward(data(g), code(g.scalar_type()), static_cast<const int64_t*>(data(ids)),
                                  static_cast<const float*>(data(share)), static_cast<const float*>(data(rest)),
                                  static_cast<const float*>(data(norm)), data(logits),
                                  logits.defined() ? pitch(logits) : E, T, E, ids.size(1), code(dtype),
                                  (int)ctx->saved_data["renormalize"].toInt(),
                                  (float)ctx->saved_data["scale"].toDouble(), data(out), place.stream),
          "fmoe_route_backward");
    // the result depends on the logits, whether they are kept or not: what this node's gradient goes to
    if (at::GradMode::is_enabled()) {
      const auto node = torch::autograd::get_current_node();
      if (!node) throw std::runtime_error(kNoSecondRoute);
      refuse_history(out, node->next_edges(), kNoSecondRoute);
    }
    return {out, Tensor()};
  }
};

PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<11>(n, [&] {
    if (!tensors({a[0], a[1]})) return not_taken();
    const Tensor logits = tensor(a[0]);
    Routing o;
    o.bias = tensor(a[1]);
    o.k = integer(a[2]);
    o.score = (int)integer(a[3]);
    o.groups = integer(a[4]);
    o.top_groups = integer(a[5]);
    o.group_score = (int)integer(a[6]);
    o.renormalize = a[7] == Py_True;
    o.scale = (float)real(a[8]);
    o.w_dtype = (int)integer(a[9]);
    const bool records = a[10] == Py_True;
    if (!good_matrix(logits) || (recorded(logits) && !records) || o.k < 1 || o.k > logits.size(1) ||
        (o.bias.defined() &&
         (!plain(o.bias) || o.bias.device() != logits.device() || o.bias.scalar_type() != at::kFloat ||
          o.bias.dim() != 1 || o.bias.size(0) != logits.size(1) || !o.bias.is_contiguous() || recorded(o.bias))))
      return not_taken();
    if (records) {
      const auto r = Route::apply(logits, o);
      return tuple(r[0], r[1]);
    }
    const Routed r = run_route(logits, o, false);
    return tuple(r.weights, r.ids);
  });
}

// ---- the norms around a block -------------------------------------------------------------------------

struct Sandwich {
  Tensor x, post, residual, pre, gate;  // pre, gate: or undefined
  double scale, eps;
  int64_t gate_rows() const { return !gate.defined() ? 0 : gate.dim() == 1 ? 1 : gate.size(0); }
};

bool good_param(const Tensor& t, const Tensor& x, bool matrix) {
  return plain(t) && t.is_contiguous() && t.device() == x.device() &&
         (t.dim() == 1 || (matrix && t.dim() == 2)) && t.size(-1) == x.size(1) &&
         (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat);
}

bool good_sandwich(const Sandwich& s) {
  return good_matrix(s.x) && good_matrix(s.residual) && s.residual.sizes() == s.x.sizes() &&
         s.residual.scalar_type() == s.x.scalar_type() && s.residual.device() == s.x.device() &&
         s.post.defined() && good_param(s.post, s.x, false) &&
         (!s.pre.defined() || (good_param(s.pre, s.x, false) && s.pre.scalar_type() == s.post.scalar_type())) &&
         (!s.gate.defined() ||
          (good_param(s.gate, s.x, true) &&
           (s.gate_rows() ? s.x.size(0) % s.gate_rows() == 0 : s.x.size(0) == 0))) &&
         std::isfinite(s.scale) && s.eps >= 0 && s.eps < HUGE_VAL;
}

struct Sandwiched {
  Tensor y, h, rstd;
};

Sandwiched run_sandwich(const Sandwich& s, bool keep) {
  Place place(s.x);
  const int64_t T = s.x.size(0), D = s.x.size(1);
  Sandwiched r;
  r.h = empty({T, D}, s.x);
  if (s.pre.defined()) r.y = empty({T, D}, s.x);
  if (keep) r.rstd = empty({T, 2}, s.x, at::kFloat);
  if (T)
    check(api.fmoe_sandwich_norm(data(s.x), pitch(s.x), data(s.residual), pitch(s.residual), data(s.post),
                                 data(s.pre), code(s.post.scalar_type()), data(s.gate),
                                 s.gate.defined() ? code(s.gate.scalar_type()) : FMOE_F32, s.gate_rows(), T, D,
                                 code(s.x.scalar_type()), (float)s.scale, (float)s.eps, data(r.h), data(r.y),
                                 static_cast<float*>(data(r.rstd)), place.stream),
          "fmoe_sandwich_norm");
  return r;
}

constexpr const char* kNoSecondSandwich =
    "fastmoe_amd: the gradient of the norms around a block has no gradient of its own";

class SandwichNorm : public torch::autograd::Function<SandwichNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor post, Tensor residual,
                               std::optional<Tensor> pre, std::optional<Tensor> gate, double scale, double eps) {
    const Sandwich s{x, post, residual, pre.value_or(Tensor()), gate.value_or(Tensor()), scale, eps};
    const Sandwiched r = run_sandwich(s, true);
    ctx->save_for_backward({x, r.h, post, s.pre, s.gate, r.rstd});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    if (!s.pre.defined()) return {r.h};
    return {r.h, r.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &h = saved[1], &post = saved[2], &pre = saved[3], &gate = saved[4],
                 &rstd = saved[5];
    Tensor gh = grads[0], gy = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(7);
    if (!gh.defined() && !gy.defined()) return out;
    refuse_second(grads, kNoSecondSandwich);
    Place place(h);
    refuse_capture("the backward of the norms around a block");
    if (gh.defined()) gh = by_rows(gh);
    if (gy.defined()) gy = by_rows(gy);
    // inputs that were not given are not counted
    const bool has_pre = pre.defined(), has_gate = gate.defined();
    const bool need_pre = has_pre && ctx->needs_input_grad(3),
               need_gate = has_gate && ctx->needs_input_grad(has_pre ? 4 : 3);
    const int64_t T = h.size(0), D = h.size(1),
                  runs = !has_gate ? 0 : gate.dim() == 1 ? 1 : gate.size(0);
    if (ctx->needs_input_grad(0)) out[0] = empty({T, D}, h);
    if (ctx->needs_input_grad(1)) out[1] = empty({D}, post);
    if (ctx->needs_input_grad(2)) out[2] = empty({T, D}, h);
    if (need_pre) out[3] = gy.defined() ? empty({D}, pre) : at::zeros_like(pre);
    if (need_gate) out[4] = T ? empty(gate.sizes(), gate) : at::zeros_like(gate);
    const int64_t bytes = api.fmoe_sandwich_norm_backward_workspace_bytes(T, D, runs);
    const Tensor ws = empty({bytes}, h, at::kByte);
    check(api.fmoe_sandwich_norm_backward(
              data(gy), gy.defined() ? pitch(gy) : 0, data(gh), gh.defined() ? pitch(gh) : 0, data(x), pitch(x),
              data(h), data(post), data(pre), code(post.scalar_type()),
              runs ? data(gate) : nullptr, has_gate ? code(gate.scalar_type()) : FMOE_F32, runs,
              static_cast<const float*>(data(rstd)), T, D,
              code(h.scalar_type()), (float)ctx->saved_data["scale"].toDouble(), data(out[0]), data(out[2]),
              data(out[1]), gy.defined() ? data(out[3]) : nullptr, T ? data(out[4]) : nullptr, data(ws), bytes,
              place.stream),
          "fmoe_sandwich_norm_backward");
    mark_second({&out[0], &out[1], &out[2], &out[3], &out[4]}, {x, post, h, pre, gate}, kNoSecondSandwich);
    return out;
  }
};

PyObject* sandwich(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<8>(n, [&] {
    if (!tensors({a[0], a[1], a[2], a[3], a[4]})) return not_taken();
    const Sandwich s{tensor(a[0]), tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4]), real(a[5]), real(a[6])};
    const bool records = a[7] == Py_True;
    if (!good_sandwich(s)) return not_taken();
    if (records) {
      auto maybe = [](const Tensor& t) { return t.defined() ? std::make_optional(t) : std::nullopt; };
      const auto r = SandwichNorm::apply(s.x, s.post, s.residual, maybe(s.pre), maybe(s.gate), s.scale, s.eps);
      return tuple(r.size() > 1 ? r[1] : Tensor(), r[0]);
    }
    for (const Tensor* t : {&s.x, &s.post, &s.residual, &s.pre, &s.gate})
      if (recorded(*t)) return not_taken();
    const Sandwiched r = run_sandwich(s, false);
    return tuple(r.y, r.h);
  });
}

// ---- weights in 4 bits --------------------------------------------------------------------------------

int64_t whole_pieces(int64_t n) { return (n + 127) / 128 * 128; }

// [..., N, bytes of codes] and [..., N, bytes of scales] of `features` columns.
bool good_fp4(const Tensor& q, const Tensor& s, int64_t features) {
  return q.defined() && s.defined() && plain(q) && plain(s) && q.scalar_type() == at::kByte &&
         s.scalar_type() == at::kByte && s.device() == q.device() && q.is_contiguous() && s.is_contiguous() &&
         q.dim() >= 2 && q.dim() <= 3 && s.dim() == q.dim() && q.sizes().slice(0, q.dim() - 1) ==
         s.sizes().slice(0, q.dim() - 1) && features >= 1 && features <= (int64_t(1) << 40) &&
         q.size(-1) == whole_pieces(features) / 2 && s.size(-1) == whole_pieces(features) / 32 &&
         (q.numel() == 0 || (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 &&
                             reinterpret_cast<uintptr_t>(s.data_ptr()) % 4 == 0));
}

PyObject* quantize_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<1>(n, [&] {
    if (!tensors({a[0]})) return not_taken();
    const Tensor x = tensor(a[0]);
    if (!good_matrix(x) || recorded(x)) return not_taken();
    const int64_t R = x.size(0), pad = whole_pieces(x.size(1));
    Place place(x);
    const Tensor q = empty({R, pad / 2}, x, at::kByte), s = empty({R, pad / 32}, x, at::kByte);
    if (R)
      check(api.fmoe_quantize_fp4(data(x), pitch(x), R, x.size(1), code(x.scalar_type()), data(q), data(s),
                                  place.stream),
            "fmoe_quantize_fp4");
    return tuple(q, s);
  });
}

PyObject* restore_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<4>(n, [&] {
    if (!tensors({a[0], a[1]})) return not_taken();
    const Tensor q = tensor(a[0]), s = tensor(a[1]);
    const int64_t K = integer(a[2]);
    const int dtype = (int)integer(a[3]);
    if (!good_fp4(q, s, K)) return not_taken();
    Place place(q);
    std::vector<int64_t> sizes(q.sizes().begin(), q.sizes().end());
    sizes.back() = K;
    const Tensor out = empty(sizes, q, type_of(dtype));
    if (q.numel())
      check(api.fmoe_restore_fp4(data(q), data(s), q.numel() / q.size(-1), K, data(out), dtype, place.stream),
            "fmoe_restore_fp4");
    return wrap(out);
  });
}

PyObject* fp4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<9>(n, [&] {
    if (!tensors({a[0], a[1], a[2], a[4], a[5], a[6]})) return not_taken();
    const Tensor x = tensor(a[0]), w = tensor(a[1]), s = tensor(a[2]), off = tensor(a[4]), rows = tensor(a[5]),
                 bias = tensor(a[6]);
    const int64_t K = integer(a[3]);
    if (!good_matrix(x) || x.scalar_type() == at::kFloat || recorded(x) || x.size(1) != K || !good_fp4(w, s, K) ||
        w.device() != x.device())
      return not_taken();
    const int64_t E = w.dim() == 3 ? w.size(0) : 1, N = w.size(-2);
    auto here = [&](const Tensor& t) { return plain(t) && t.device() == x.device() && t.is_contiguous(); };
    if (E < 1 || N < 1 ||
        (off.defined() ? !here(off) || off.scalar_type() != at::kLong || off.dim() != 1 || off.size(0) != E + 1
                       : E != 1) ||
        (rows.defined() && (!here(rows) || rows.dim() != 1 ||
                            (rows.scalar_type() != at::kLong && rows.scalar_type() != at::kInt) ||
                            (rows.size(0) > 0 && x.size(0) == 0))) ||
        (bias.defined() && (!here(bias) || !is_float(bias) || recorded(bias) ||
                            !((bias.dim() == 2 && bias.size(0) == E && bias.size(1) == N) ||
                              (E == 1 && bias.dim() == 1 && bias.size(0) == N)))))
      return not_taken();
    const int64_t R = rows.defined() ? rows.size(0) : x.size(0);
    const int act = (int)integer(a[7]), dtype = (int)integer(a[8]);
    Place place(x);
    const Tensor out = empty({R, N}, x, type_of(dtype));
    if (R)
      check(api.fmoe_fp4_linear(data(x), pitch(x), x.size(0), code(x.scalar_type()), data(rows),
                                rows.defined() ? code(rows.scalar_type()) : FMOE_I64, data(w), data(s), data(bias),
                                bias.defined() ? code(bias.scalar_type()) : FMOE_F32, act,
                                static_cast<const int64_t*>(data(off)), E, N, K, R, data(out), N, dtype,
                                place.stream),
            "fmoe_fp4_linear");
    return wrap(out);
  });
}

PyObject* bind(PyObject*, PyObject* dict) {
  Api found;
#define FMOE_FIND(name)                                                                         \
  {                                                                                             \
    PyObject* v = PyDict_Check(dict) ? PyDict_GetItemString(dict, #name) : nullptr;             \
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;                                                \
    if (!p) {                                                                                   \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "fastmoe_amd._block: no " #name); \
      return nullptr;                                                                           \
    }                                                                                           \
    std::memcpy(&found.name, &p, sizeof(p));                                                    \
  }
  FMOE_ENTRIES(FMOE_FIND)
#undef FMOE_FIND
  api = found;
  last_error = found.fmoe_last_error;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_O, "bind({name: address}): the library's entry points"},
    {"route", FMOE_FAST(route),
     "route(logits, bias, top_k, score, groups, top_groups, group_score, renormalize, scale, dtype, recorded)"},
    {"sandwich", FMOE_FAST(sandwich), "sandwich(x, post, residual, pre, gate, scale, eps, recorded)"},
    {"quantize_fp4", FMOE_FAST(quantize_fp4), "quantize_fp4(x)"},
    {"restore_fp4", FMOE_FAST(restore_fp4), "restore_fp4(data, scales, features, dtype)"},
    {"fp4_linear", FMOE_FAST(fp4_linear),
     "fp4_linear(x, data, scales, features, offsets, rows, bias, activation, dtype)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_block",
                       "Host side of fastmoe_amd's router, norms around a block and 4-bit weights", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__block(void) { return PyModule_Create(&kModule); }
