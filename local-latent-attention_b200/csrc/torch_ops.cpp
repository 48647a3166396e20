// The eager path of lm_ops.py's operators: torch tensors in, libllattn calls, autograd nodes in
// C++. What Python costs a call (an autograd.Function 40 us, a list of 400 gradients 200) is
// more than the kernels of small calls take. Every function returns None for what it does not
// handle (other types, devices, shapes or wrapped tensors): lm_ops.py then goes its own way, which
// checks the arguments and says what is wrong with them.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "llattn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// what the library takes
constexpr int64_t kMostTokens = 1 << 26, kMostIds = 1 << 30, kMostWords = 1 << 24, kMostColumns = 1 << 20;

constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize});

// (without a tangent: nothing here carries forward-mode derivatives on)
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(kWrapped) && !t._fw_grad(0).defined();
}
int dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? LLATTN_F32 : t.scalar_type() == at::kBFloat16 ? LLATTN_BF16 : -1;
}
bool like(const Tensor& t, const Tensor& o) { return plain(t) && t.scalar_type() == o.scalar_type() && t.device() == o.device(); }
// a view whose sign is still to be applied (imag of a conjugate) with it applied: the kernels read the memory
Tensor signs(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// contiguous columns and rows that do not overlap
Tensor rows(const Tensor& u) {
  const Tensor t = signs(u);
  return t.stride(1) == 1 && (t.size(0) == 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t stride_of(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }
Tensor bytes(size_t n, const Tensor& like) { return at::detail::empty_cuda({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }
void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (status ", rc, "): ", llattn_last_error()); }
void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Gradients of gradients are not supported: under create_graph the results hang on a node that says so.
struct Once : torch::autograd::Function<Once> {
  static Tensor forward(AutogradContext*, const Tensor& g, const Tensor&) { return g.view_as(g); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "llattn: trying to differentiate twice an operator whose gradients are not differentiable");
  }
};
// (calls with dual inputs have gone to lm_ops.py, which refuses them; here it is the upstream gradient that may be one)
void no_tangent(const Tensor& g, const char* what) {
  TORCH_CHECK(!g._fw_grad(0).defined(), "llattn: ", what, "'s backward has no forward-mode derivatives (the upstream gradient is a dual tensor)");
}
variable_list once(variable_list grads, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto leaf = std::find_if(from.begin(), from.end(), [](const Tensor& t) { return t.defined() && t.requires_grad(); });
  if (leaf == from.end()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = Once::apply(g, *leaf);
  return grads;
}

// ---- gated feed-forward block ------------------------------------------------------

llattn_gated_args gated_args(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int act) {
  llattn_gated_args a = {};
  a.tokens = (int32_t)x.size(0);
  a.d = (int32_t)x.size(1);
  a.ff = (int32_t)wg.size(0);
  a.d_out = (int32_t)wd.size(0);
  a.dtype = dtype_of(x);
  a.activation = act;
  a.x = x.data_ptr();
  a.ldx = stride_of(x);
  a.w_gate = wg.data_ptr();
  a.ldg = stride_of(wg);
  a.w_up = wu.data_ptr();
  a.ldu = stride_of(wu);
  a.w_down = wd.data_ptr();
  a.ldd = stride_of(wd);
  return a;
}

Tensor gated_forward(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& wd_, int act, Tensor* kept) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows(x_), wg = rows(wg_), wu = rows(wu_), wd = rows(wd_);
  llattn_gated_args a = gated_args(x, wg, wu, wd, act);
  Tensor y = at::empty({x.size(0), wd.size(0)}, x.options().requires_grad(false));
  if (kept) {
    *kept = bytes(llattn_gated_kept_bytes(&a), x);
    a.kept = kept->data_ptr();
  }
  a.y = y.data_ptr();
  a.workspace_bytes = llattn_gated_workspace_bytes(&a, 0);
  const Tensor ws = bytes(a.workspace_bytes, x);
  a.workspace = ws.data_ptr();
  check(llattn_gated_fwd(&a, stream(x)), "llattn_gated_fwd");
  return y;
}

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
    Tensor kept;
    Tensor y = gated_forward(x, wg, wu, wd, (int)act, &kept);
    ctx->save_for_backward({x, wg, wu, wd, kept});
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(5);
    if (!grads[0].defined()) return out;
    no_tangent(grads[0], "gated_mlp");
    {
      at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard guard(saved[0].device());
      const Tensor x = rows(saved[0]), wg = rows(saved[1]), wu = rows(saved[2]), wd = rows(saved[3]), dy = rows(grads[0]);
      llattn_gated_args a = gated_args(x, wg, wu, wd, (int)ctx->saved_data["act"].toInt());
      for (int i = 0; i < 4; ++i)
        if (ctx->needs_input_grad(i))
          out[i] = at::empty(saved[i].sizes(), x.options().requires_grad(false));
      a.kept = saved[4].data_ptr();
      a.dy = dy.data_ptr();
      a.lddy = stride_of(dy);
      a.dx = data(out[0]);
      a.dw_gate = data(out[1]);
      a.dw_up = data(out[2]);
      a.dw_down = data(out[3]);
      a.workspace_bytes = llattn_gated_workspace_bytes(&a, 1);
      const Tensor ws = bytes(a.workspace_bytes, x);
      a.workspace = ws.data_ptr();
      check(llattn_gated_bwd(&a, stream(x)), "llattn_gated_bwd");
    }
    return once(out, {grads[0], saved[0], saved[1], saved[2], saved[3]});
  }
};

// gated(x, w_gate, w_up, w_down, act)
PyObject* py_gated(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &wg = THPVariable_Unpack(args[1]), &wu = THPVariable_Unpack(args[2]),
               &wd = THPVariable_Unpack(args[3]);
  if (!plain(x) || dtype_of(x) < 0 || !like(wg, x) || !like(wu, x) || !like(wd, x) || x.dim() < 1 || x.numel() == 0 || wg.dim() != 2 ||
      wd.dim() != 2 || wg.sizes() != wu.sizes() || x.size(-1) != wg.size(1) || wd.size(1) != wg.size(0) || wg.numel() == 0 ||
      wd.numel() == 0 || x.numel() / x.size(-1) > kMostTokens || wg.size(0) > kMostColumns || wg.size(1) > kMostColumns ||
      wd.size(0) > kMostColumns)
    Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(args[4]);
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const Tensor flat = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    if (at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
      y = Gated::apply(flat, wg, wu, wd, act);
    else
      y = gated_forward(flat, wg, wu, wd, act, nullptr);
    if (x.dim() != 2) {
      auto sizes = x.sizes().vec();
      sizes.back() = wd.size(0);
      y = y.view(sizes);
    }
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- token embedding ----------------------------------------------------------------

llattn_embed_args embed_args(const Tensor& ids, int64_t vocab, int64_t d, int dtype, int64_t position_rows, double scale,
                             int64_t padding) {
  llattn_embed_args a = {};
  a.batch = (int32_t)ids.size(0);
  a.length = (int32_t)ids.size(1);
  a.d = (int32_t)d;
  a.dtype = dtype;
  a.ids_wide = ids.scalar_type() == at::kLong;
  a.position_rows = (int32_t)position_rows;
  a.vocab = vocab;
  a.padding = padding;
  a.scale = (float)scale;
  a.ids = ids.data_ptr();
  return a;
}

Tensor embed_forward(const Tensor& ids_, const Tensor& w_, const Tensor& pos_, double scale) {
  const c10::cuda::CUDAGuard guard(w_.device());
  const Tensor ids = ids_.contiguous(), w = rows(w_), pos = pos_.defined() ? rows(pos_) : pos_;
  llattn_embed_args a = embed_args(ids, w.size(0), w.size(1), dtype_of(w), pos.defined() ? pos.size(0) : 0, scale, -1);
  Tensor out = at::detail::empty_cuda({ids.size(0), ids.size(1), w.size(1)}, w.options().requires_grad(false));
  a.w = w.data_ptr();
  a.ldw = stride_of(w);
  a.out = out.data_ptr();
  if (pos.defined()) {
    a.positions = pos.data_ptr();
    a.ldp = stride_of(pos);
  }
  check(llattn_embed_fwd(&a, stream(w)), "llattn_embed_fwd");
  return out;
}

// (A node of its own: a Function's context and boxed attributes cost a small call 5 us of its 55.)
struct EmbedBackward : torch::autograd::Node {
  torch::autograd::SavedVariable ids_;
  int64_t vocab, position_rows, padding;
  double scale;

  std::string name() const override { return "TokenEmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids_.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(2);
    const bool need_w = task_should_compute_output(0), need_p = position_rows && task_should_compute_output(1);
    if (!grads[0].defined() || !(need_w || need_p)) return out;
    no_tangent(grads[0], "token_embedding");
    {
      at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard guard(grads[0].device());
      const Tensor ids = ids_.unpack().contiguous(), dout = signs(grads[0]).contiguous();
      const int64_t d = dout.size(2);
      llattn_embed_args a = embed_args(ids, vocab, d, dtype_of(dout), position_rows, scale, padding);
      const auto opts = dout.options().requires_grad(false);
      if (need_w) out[0] = at::detail::empty_cuda({vocab, d}, opts);
      if (need_p) out[1] = at::detail::empty_cuda({position_rows, d}, opts);
      a.dout = dout.data_ptr();
      a.dw = data(out[0]);
      a.dpositions = data(out[1]);
      a.workspace_bytes = llattn_embed_workspace_bytes(&a);
      const Tensor ws = bytes(a.workspace_bytes, dout);
      a.workspace = ws.data_ptr();
      check(llattn_embed_bwd(&a, ::stream(dout)), "llattn_embed_bwd");
    }
    return once(out, grads);
  }
};

// embed(ids, weight, positions or None, scale, padding)
PyObject* py_embed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) ||
      (args[2] != Py_None && !THPVariable_CheckExact(args[2])))
    Py_RETURN_NONE;
  const Tensor &ids = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  std::optional<Tensor> pos;
  if (args[2] != Py_None) pos = THPVariable_Unpack(args[2]);
  if (!plain(ids) || !plain(w) || dtype_of(w) < 0 || ids.device() != w.device() || w.dim() != 2 || w.numel() == 0 ||
      (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || ids.numel() == 0 || ids.numel() > kMostIds ||
      w.size(0) > kMostWords || w.size(1) > kMostColumns)
    Py_RETURN_NONE;
  if (pos && (!like(*pos, w) || ids.dim() < 1 || pos->dim() != 2 || pos->size(0) < ids.size(-1) || pos->size(1) != w.size(1) ||
              pos->size(0) > INT32_MAX))
    Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(args[3]);
  const int64_t padding = PyLong_AsLongLong(args[4]);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const Tensor flat = ids.dim() == 2 ? ids : ids.reshape({-1, ids.dim() ? ids.size(-1) : 1});
    if (at::GradMode::is_enabled() && (w.requires_grad() || (pos && pos->requires_grad()))) {
      std::shared_ptr<EmbedBackward> node(new EmbedBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(w, pos ? *pos : Tensor()));
      node->ids_ = torch::autograd::SavedVariable(flat, false);
      node->vocab = w.size(0);
      node->position_rows = pos ? pos->size(0) : 0;
      node->padding = padding;
      node->scale = scale;
      {
        at::NoGradGuard no_grad;
        out = embed_forward(flat, w, pos ? *pos : Tensor(), scale);
      }
      torch::autograd::set_history(out, node);
    } else {
      out = embed_forward(flat, w, pos ? *pos : Tensor(), scale);
    }
    if (ids.dim() != 2) {
      auto sizes = ids.sizes().vec();
      sizes.push_back(w.size(1));
      out = out.view(sizes);
    }
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- norm and clipping --------------------------------------------------------------

// clip(list, grads, norm_type, max_norm, scale): the norm of a list's tensors, or of their gradients
// where they have some (grads), scaled with scale. None too where two share memory.
PyObject* py_clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !PyList_Check(args[0])) Py_RETURN_NONE;
  const bool grads = PyObject_IsTrue(args[1]) == 1, scale = PyObject_IsTrue(args[4]) == 1;
  const Py_ssize_t count = PyList_GET_SIZE(args[0]);
  std::vector<void*> pointers;
  std::vector<int64_t> sizes;
  std::vector<int32_t> dtypes;
  pointers.reserve(count);
  sizes.reserve(count);
  dtypes.reserve(count);
  std::vector<const Tensor*> used;
  used.reserve(count);
  const Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_CheckExact(o)) Py_RETURN_NONE;
    const Tensor& p = THPVariable_Unpack(o);
    if (p.key_set().has_any(kWrapped)) Py_RETURN_NONE;
    const Tensor& t = grads ? p.grad() : p;
    if (!t.defined()) continue;
    const int dtype = dtype_of(t);
    if (!plain(t) || dtype < 0 || (first && t.device() != first->device()) || !t.is_non_overlapping_and_dense()) Py_RETURN_NONE;
    if (!first) first = &t;
    used.push_back(&t);
    pointers.push_back(t.data_ptr());
    sizes.push_back(t.numel());
    dtypes.push_back(dtype);
  }
  if (!first || pointers.size() > INT32_MAX) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(first->device());
  llattn_clip_args a = {};
  a.count = (int32_t)pointers.size();
  a.norm_type = (int32_t)PyLong_AsLong(args[2]);
  a.scale = scale;
  a.tensors = pointers.data();
  a.sizes = sizes.data();
  a.dtypes = dtypes.data();
  a.max_norm = PyFloat_AsDouble(args[3]);
  at::NoGradGuard no_grad;
  Tensor norm = at::empty({}, first->options().dtype(at::kFloat).requires_grad(false));
  a.norm = norm.data_ptr<float>();
  a.workspace_bytes = llattn_clip_workspace_bytes(&a);
  const Tensor ws = bytes(a.workspace_bytes, norm);
  a.workspace = ws.data_ptr();
  const int rc = llattn_clip(&a, stream(norm));
  if (rc == LLATTN_ERR_ARG) Py_RETURN_NONE;
  check(rc, "llattn_clip");
  if (scale)  // autograd has to see that they changed
    for (const Tensor* t : used)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"gated", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_gated)), METH_FASTCALL, nullptr},
    {"embed", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_embed)), METH_FASTCALL, nullptr},
    {"clip", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_clip)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&module); }
