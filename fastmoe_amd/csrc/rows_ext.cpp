// fastmoe_amd._rows: the host side of the 8-bit operators and the norm (not part of the C ABI).
//
// A call of these operators on a decoding step's rows takes the GPU 3 to 6 us; through ctypes and
// torch's Python allocations its host side took 8 to 14 us, and the norm's training step 130 us, 48 of
// them the engine's.  Here a call allocates its results and calls the C entry point in one go, and the
// norm's backward runs in the engine's thread without the interpreter.
//
// Each function but bind checks its arguments and returns NotImplemented where something is not as it
// takes it, and under tracing; the caller (quantize.py) then goes through the checks one by one and says
// what is wrong.
//
//   bind({name: address}) once, with the library's entry points
//   norm(x, weight, residual | None, eps, want_y, want_rows8) -> (stream, y | None, data | None, scales | None)
//   norm_recorded(x, weight, residual | None, eps) -> (y, stream): records its backward
//   quantize(x, activation) -> (data, scales)
//   compress(x, gelu, hold) -> (gelu(x) | None, data | None, scales | None)
//   restore(data, scales, a scale for every 128 columns, features, dtype code) -> values
//   gelu_backward(data, scales, features, grad, again) -> (gelu | None, grad)
//   linear(x data, x scales, features, weights, their scales, offsets | None, rows | None, bias | None,
//          dtype code) -> out
constexpr const char* kModuleName = "fastmoe_amd._rows";
#include "host_tensors.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

namespace {

#define FMOE_ENTRIES(X)                                                                       \
  X(fmoe_last_error)                                                                          \
  X(fmoe_add_rms_norm)                                                                        \
  X(fmoe_add_rms_norm_backward)                                                               \
  X(fmoe_add_rms_norm_backward_workspace_bytes)                                               \
  X(fmoe_quantize_rows)                                                                       \
  X(fmoe_compress_rows)                                                                       \
  X(fmoe_restore_rows)                                                                        \
  X(fmoe_gelu_compressed_backward)                                                            \
  X(fmoe_int8_linear)

struct Api {
#define FMOE_DECLARE(name) decltype(&::name) name = nullptr;
  FMOE_ENTRIES(FMOE_DECLARE)
#undef FMOE_DECLARE
} api;

int64_t padded(int64_t n) { return (n + 127) / 128 * 128; }

struct Normed {
  Tensor h, y, rstd, q, scales;
};

Normed run_norm(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, bool y,
                bool rstd, bool rows8) {
  Place place(x);
  const int64_t T = x.size(0), D = x.size(1), pad = padded(D);
  Normed n;
  n.h = residual.defined() ? empty({T, D}, x) : x;
  if (y) n.y = empty({T, D}, x);
  if (rstd) n.rstd = empty({T}, x, at::kFloat);
  if (rows8) {
    n.q = empty({T, pad}, x, at::kChar);
    n.scales = empty({T}, x, at::kFloat);
  }
  if (T)
    check(api.fmoe_add_rms_norm(data(x), pitch(x), data(residual),
                                residual.defined() ? pitch(residual) : 0, data(weight),
                                code(weight.scalar_type()), T, D, code(x.scalar_type()), (float)eps,
                                residual.defined() ? data(n.h) : nullptr, data(n.y),
                                static_cast<float*>(data(n.rstd)), data(n.q), rows8 ? pad : 0,
                                static_cast<float*>(data(n.scales)), place.stream),
          "fmoe_add_rms_norm");
  return n;
}

// ---- what the functions take ----------------------------------------------------------------------
bool good_norm(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
  return good_matrix(x) && weight.defined() && plain(weight) && weight.dim() == 1 &&
         weight.size(0) == x.size(1) && weight.is_contiguous() && weight.device() == x.device() &&
         (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat) &&
         (!residual.defined() ||
          (good_matrix(residual) && residual.sizes() == x.sizes() &&
           residual.scalar_type() == x.scalar_type() && residual.device() == x.device())) &&
         eps >= 0 && eps < HUGE_VAL;
}
bool good_int8(const Tensor& q, const Tensor& s, int64_t features, int64_t dims) {
  return q.defined() && s.defined() && plain(q) && plain(s) && q.scalar_type() == at::kChar &&
         q.dim() == dims && s.scalar_type() == at::kFloat && s.device() == q.device() && !recorded(s) &&
         s.is_contiguous() && features >= 1 && features <= INT64_MAX - 127 &&
         q.size(dims - 1) == padded(features) &&
         (q.numel() == 0 ||
          (q.stride(dims - 1) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0));
}
// Rows in 8 bits with `per_row` scales each (1: one dimension).
bool good_rows8(const Tensor& q, const Tensor& s, int64_t features, int64_t per_row, bool packed) {
  return good_int8(q, s, features, 2) && s.numel() == q.size(0) * per_row && s.size(0) == q.size(0) &&
         s.dim() == (packed ? 2 : 1) &&
         (q.size(0) <= 1 || (packed ? q.is_contiguous()
                                    : q.stride(0) >= q.size(1) && q.stride(0) % 16 == 0));
}

constexpr const char* kNoSecond = "fastmoe_amd: the norm's gradient has no gradient of its own";

class AddRmsNorm : public torch::autograd::Function<AddRmsNorm> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor x,
                                                Tensor weight, std::optional<Tensor> maybe,
                                                double eps) {
    const Tensor residual = maybe.value_or(Tensor());
    Normed n = run_norm(x, weight, residual, eps, true, true, false);
    ctx->save_for_backward({n.h, weight, n.rstd});
    ctx->set_materialize_grads(false);
    if (!residual.defined()) return {n.y};
    return {n.y, n.h};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &weight = saved[1], &rstd = saved[2];
    Tensor gy = grads[0], gh = grads.size() > 1 ? grads[1] : Tensor();
    if (at::GradMode::is_enabled() && ((gy.defined() && gy.requires_grad()) ||
                                       (gh.defined() && gh.requires_grad())))
      throw std::runtime_error(kNoSecond);
    // the third input is counted only where there was a residual, which has an output of its own
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
               need_r = grads.size() > 1 && ctx->needs_input_grad(2);
    Place place(h);
    if (capturing())
      throw std::runtime_error(
          "fastmoe_amd: the norm's backward under HIP graph capture is not supported (a captured "
          "autograd step once crashed the host in CUDAGraph.capture_end).  Run the autograd step "
          "eagerly.");
    Tensor gx, gw;
    if (!gy.defined()) {  // only the stream was used
      gx = gh;
      if (need_w) gw = at::zeros_like(weight);
    } else {
      gy = by_rows(gy);
      if (gh.defined()) gh = by_rows(gh);
      const int64_t T = h.size(0), D = h.size(1);
      gx = empty({T, D}, h);
      Tensor ws;
      int64_t bytes = 0;
      if (need_w) {
        gw = empty({D}, weight);
        bytes = api.fmoe_add_rms_norm_backward_workspace_bytes(T, D);
        ws = empty({bytes}, h, at::kByte);
      }
      check(api.fmoe_add_rms_norm_backward(
                data(gy), pitch(gy), data(gh), gh.defined() ? pitch(gh) : 0, data(h), pitch(h),
                data(weight), code(weight.scalar_type()), static_cast<const float*>(data(rstd)), T,
                D, code(h.scalar_type()), data(gx), data(gw), data(ws), bytes, place.stream),
            "fmoe_add_rms_norm_backward");
      // Under create_graph the results depend on h and the weight too: who differentiates them is told, and
      // does not get a part of the derivative.
      if (at::GradMode::is_enabled() && (h.requires_grad() || weight.requires_grad()))
        for (Tensor* g : {&gx, &gw})
          if (g->defined())
            torch::autograd::set_history(
                *g, std::shared_ptr<torch::autograd::Node>(
                        new torch::autograd::Error(kNoSecond, torch::autograd::collect_next_edges(h, weight)),
                        torch::autograd::deleteNode));
    }
    return {need_x ? gx : Tensor(), need_w ? gw : Tensor(), need_r ? gx : Tensor(), Tensor()};
  }
};

// ---- Python's side ------------------------------------------------------------------------------

PyObject* bind(PyObject*, PyObject* dict) {
  Api found;
#define FMOE_FIND(name)                                                                        \
  {                                                                                            \
    PyObject* v = PyDict_Check(dict) ? PyDict_GetItemString(dict, #name) : nullptr;            \
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;                                               \
    if (!p) {                                                                                  \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "fastmoe_amd._rows: no " #name); \
      return nullptr;                                                                          \
    }                                                                                          \
    std::memcpy(&found.name, &p, sizeof(p));                                                   \
  }
  FMOE_ENTRIES(FMOE_FIND)
#undef FMOE_FIND
  api = found;
  last_error = found.fmoe_last_error;
  Py_RETURN_NONE;
}

PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<6>(n, [&] {
    if (!tensors({a[0], a[1], a[2]})) return not_taken();
    const Tensor x = tensor(a[0]), weight = tensor(a[1]), residual = tensor(a[2]);
    const double eps = real(a[3]);
    if (!good_norm(x, weight, residual, eps) || recorded(x) || recorded(weight) || recorded(residual))
      return not_taken();
    const Normed r = run_norm(x, weight, residual, eps, a[4] == Py_True, false, a[5] == Py_True);
    return tuple(r.h, r.y, r.q, r.scales);
  });
}

PyObject* norm_recorded(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<4>(n, [&] {
    if (!tensors({a[0], a[1], a[2]})) return not_taken();
    const Tensor x = tensor(a[0]), weight = tensor(a[1]), residual = tensor(a[2]);
    const double eps = real(a[3]);
    if (!good_norm(x, weight, residual, eps)) return not_taken();
    const auto r = AddRmsNorm::apply(
        x, weight, residual.defined() ? std::make_optional(residual) : std::nullopt,
        eps);
    return tuple(r[0], residual.defined() ? r[1] : x);
  });
}

PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<2>(n, [&] {
    if (!tensors({a[0]})) return not_taken();
    const Tensor x = tensor(a[0]);
    if (!good_matrix(x) || recorded(x)) return not_taken();
    const int64_t act = integer(a[1]), pad = padded(x.size(1)), R = x.size(0);
    Place place(x);
    const Tensor q = empty({R, pad}, x, at::kChar), s = empty({R}, x, at::kFloat);
    if (R)
      check(api.fmoe_quantize_rows(data(x), pitch(x), R, x.size(1), code(x.scalar_type()), (int)act,
                                   data(q), pad, static_cast<float*>(data(s)), place.stream),
            "fmoe_quantize_rows");
    return tuple(q, s);
  });
}

PyObject* compress(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<3>(n, [&] {
    if (!tensors({a[0]})) return not_taken();
    const Tensor x = tensor(a[0]);
    if (!good_matrix(x) || recorded(x)) return not_taken();
    const int64_t pad = padded(x.size(1)), R = x.size(0), C = x.size(1);
    Place place(x);
    Tensor g, q, s;
    if (a[2] == Py_True) {
      q = empty({R, pad}, x, at::kChar);
      s = empty({R, pad / 128}, x, at::kFloat);
    }
    if (a[1] == Py_True) g = empty({R, C}, x);
    if (R)
      check(api.fmoe_compress_rows(data(x), pitch(x), R, C, code(x.scalar_type()), data(q), pad,
                                   static_cast<float*>(data(s)), data(g), place.stream),
            "fmoe_compress_rows");
    return tuple(g, q, s);
  });
}

PyObject* restore(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<5>(n, [&] {
    if (!tensors({a[0], a[1]})) return not_taken();
    const Tensor q = tensor(a[0]), s = tensor(a[1]);
    const int64_t C = integer(a[3]);
    const bool blocks = a[2] == Py_True;
    const int64_t per_row = blocks ? (C + 127) / 128 : 1;
    if (!good_rows8(q, s, C, per_row, blocks)) return not_taken();
    const int64_t R = q.size(0);
    const int dtype = (int)integer(a[4]);
    Place place(q);
    const Tensor out = empty({R, C}, q, type_of(dtype));
    if (R)
      check(api.fmoe_restore_rows(data(q), pitch(q), static_cast<const float*>(data(s)), per_row, R,
                                  C, data(out), dtype, place.stream),
            "fmoe_restore_rows");
    return wrap(out);
  });
}

PyObject* gelu_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<5>(n, [&] {
    if (!tensors({a[0], a[1], a[3]})) return not_taken();
    const Tensor q = tensor(a[0]), s = tensor(a[1]), grad = tensor(a[3]);
    const int64_t C = integer(a[2]);
    if (!good_rows8(q, s, C, (C + 127) / 128, true) || !good_matrix(grad) || recorded(grad) ||
        grad.size(0) != q.size(0) || grad.size(1) != C || grad.device() != q.device())
      return not_taken();
    const int64_t R = q.size(0);
    Place place(q);
    const Tensor out = empty({R, C}, grad);
    Tensor again;
    if (a[4] == Py_True) again = empty({R, C}, grad);
    if (R)
      check(api.fmoe_gelu_compressed_backward(data(q), pitch(q), static_cast<const float*>(data(s)),
                                              data(grad), pitch(grad), R, C,
                                              code(grad.scalar_type()), data(again), data(out),
                                              place.stream),
            "fmoe_gelu_compressed_backward");
    return tuple(again, out);
  });
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded<9>(n, [&] {
    if (!tensors({a[0], a[1], a[3], a[4], a[5], a[6], a[7]})) return not_taken();
    const Tensor q = tensor(a[0]), s = tensor(a[1]), off = tensor(a[5]), rows = tensor(a[6]),
                 bias = tensor(a[7]);
    Tensor w = tensor(a[3]), sw = tensor(a[4]);
    const int64_t K = integer(a[2]);
    if (w.defined() && w.dim() == 2) {
      w = w.unsqueeze(0);
      if (sw.defined()) sw = sw.unsqueeze(0);
    }
    if (!good_rows8(q, s, K, 1, false) || !good_int8(w, sw, K, 3) || !w.is_contiguous() ||
        w.size(0) < 1 || w.size(1) < 1 || sw.dim() != 2 || sw.size(0) != w.size(0) ||
        sw.size(1) != w.size(1))
      return not_taken();
    const int64_t E = w.size(0), N = w.size(1);
    auto here = [&](const Tensor& t) { return plain(t) && t.device() == q.device() && t.is_contiguous(); };
    if (w.device() != q.device() ||
        (off.defined() ? !here(off) || off.scalar_type() != at::kLong || off.dim() != 1 ||
                             off.size(0) != E + 1
                       : E != 1) ||
        (rows.defined() && (!here(rows) || rows.dim() != 1 ||
                            (rows.scalar_type() != at::kLong && rows.scalar_type() != at::kInt) ||
                            (rows.size(0) > 0 && q.size(0) == 0))) ||
        (bias.defined() && (!here(bias) || !is_float(bias) || recorded(bias) ||
                            !((bias.dim() == 2 && bias.size(0) == E && bias.size(1) == N) ||
                              (E == 1 && bias.dim() == 1 && bias.size(0) == N)))))
      return not_taken();
    const int64_t R = rows.defined() ? rows.size(0) : q.size(0);
    const int dtype = (int)integer(a[8]);
    Place place(q);
    const Tensor out = empty({R, N}, q, type_of(dtype));
    if (R)
      check(api.fmoe_int8_linear(data(q), pitch(q), q.size(0), static_cast<const float*>(data(s)),
                                 data(rows), rows.defined() ? code(rows.scalar_type()) : FMOE_I64,
                                 data(w), static_cast<const float*>(data(sw)), data(bias),
                                 bias.defined() ? code(bias.scalar_type()) : FMOE_F32,
                                 static_cast<const int64_t*>(data(off)), E, N, K, R, data(out), N,
                                 dtype, place.stream),
            "fmoe_int8_linear");
    return wrap(out);
  });
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_O, "bind({name: address}): the library's entry points"},
    {"norm", FMOE_FAST(norm), "norm(x, weight, residual, eps, want_y, want_rows8)"},
    {"norm_recorded", FMOE_FAST(norm_recorded), "norm_recorded(x, weight, residual, eps)"},
    {"quantize", FMOE_FAST(quantize), "quantize(x, activation)"},
    {"compress", FMOE_FAST(compress), "compress(x, gelu, hold)"},
    {"restore", FMOE_FAST(restore), "restore(data, scales, blocks, features, dtype)"},
    {"gelu_backward", FMOE_FAST(gelu_backward), "gelu_backward(data, scales, features, grad, again)"},
    {"linear", FMOE_FAST(linear),
     "linear(data, scales, features, weights, their scales, offsets, rows, bias, dtype)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_rows",
                       "Host side of fastmoe_amd's 8-bit operators and norm", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__rows(void) { return PyModule_Create(&kModule); }
