// The layer operators as differentiable torch functions: tensors in, C entry points of libbnpvi called, gradients as
// autograd nodes in C++.  bnp_vae_amd/layers.py checks the arguments and calls what is here; a Python autograd function
// would cost a training pass of a small batch more than its kernels do (500 rows sorted, sent and brought back with
// gradients: 152 us with nodes in Python).
#include <dlfcn.h>

#include <mutex>
#include <unordered_map>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/bnpvi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// The entry points of the library that Python has loaded (the same instance, so the same contexts).
struct Library {
  decltype(&bnpvi_last_error) last_error;
  decltype(&bnpvi_top_leaves) top_leaves;
  decltype(&bnpvi_top_leaves_backward) top_leaves_backward;
  decltype(&bnpvi_leaf_sort_workspace) leaf_sort_workspace;
  decltype(&bnpvi_leaf_sort) leaf_sort;
  decltype(&bnpvi_rows_to_leaves) rows_to_leaves;
  decltype(&bnpvi_rows_from_leaves) rows_from_leaves;
  decltype(&bnpvi_rows_from_leaves_backward) rows_from_leaves_backward;
  decltype(&bnpvi_dense_workspace_for) dense_workspace;
  decltype(&bnpvi_dense) dense;
  decltype(&bnpvi_dense_backward_act) dense_backward;
} lib;

template <typename F>
void find(void* handle, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(handle, name));
  if (f == nullptr) throw Failure(std::string("libbnpvi does not export ") + name);
}

void bind(const std::string& path) {
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_NOLOAD);
  if (h == nullptr) throw Failure("libbnpvi is not loaded: " + path);
  find(h, "bnpvi_last_error", lib.last_error);
  find(h, "bnpvi_top_leaves", lib.top_leaves);
  find(h, "bnpvi_top_leaves_backward", lib.top_leaves_backward);
  find(h, "bnpvi_leaf_sort_workspace", lib.leaf_sort_workspace);
  find(h, "bnpvi_leaf_sort", lib.leaf_sort);
  find(h, "bnpvi_rows_to_leaves", lib.rows_to_leaves);
  find(h, "bnpvi_rows_from_leaves", lib.rows_from_leaves);
  find(h, "bnpvi_rows_from_leaves_backward", lib.rows_from_leaves_backward);
  find(h, "bnpvi_dense_workspace_for", lib.dense_workspace);
  find(h, "bnpvi_dense", lib.dense);
  find(h, "bnpvi_dense_backward_act", lib.dense_backward);
}

void check(int rc, const char* what) {
  if (rc != BNPVI_OK) {
    const char* msg = lib.last_error();
    throw Failure(std::string(what) + " failed (code " + std::to_string(rc) + "): " + (msg ? msg : "?"));
  }
}

bnpvi_ctx* ctx_of(int64_t ctx) { return reinterpret_cast<bnpvi_ctx*>(ctx); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(ptr(t));
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return BNPVI_F32;
    case at::kBFloat16:
      return BNPVI_BF16;
    default:
      return BNPVI_F16;
  }
}

// A gradient whose memory holds its values (views of complex conjugates hold the negated ones).
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A 2-D tensor with contiguous rows at a pitch the kernels take: itself where it is so already.
constexpr int64_t kMaxPitchBytes = int64_t(1) << 22;
Tensor rows(const Tensor& t) {
  const int64_t n = t.size(0), w = t.size(1);
  if (n == 0 || w == 0) return t;
  if ((w == 1 || t.stride(1) == 1) && (n == 1 || (t.stride(0) >= w && t.stride(0) * t.element_size() <= kMaxPitchBytes))) return t;
  return t.contiguous();
}
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

// A backward pass gives values without a history of their own.  Where one is asked for, every gradient hangs on all that
// it was computed from through a node that refuses to be differentiated: an error instead of a silent zero.
variable_list once(variable_list grads, const variable_list& given, const variable_list& saved) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list all = grads;
  for (const variable_list* list : {&given, &saved})
    for (const Tensor& t : *list)
      if (t.defined() && t.requires_grad()) all.push_back(t);
  if (all.size() == grads.size()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>("the layer operators can be differentiated once, not twice",
                                                              static_cast<int64_t>(all.size()));
  all = (*node)(std::move(all));
  all.resize(grads.size());
  return all;
}

// A tangent of forward-mode differentiation would be dropped without a word: the results here carry none.
void no_tangents(std::initializer_list<const Tensor*> list) {
  for (const Tensor* t : list)
    if (t->defined() && t->_fw_grad(0).defined())
      throw Failure("the layer operators have no forward-mode derivative (an input is a dual tensor)");
}

// Recorders of torch calls (torch.jit.trace, make_fx) see the allocation of a result and not the kernel that fills it: the
// recorded program would give unwritten memory.
void not_recorded() {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    throw Failure("the layer operators cannot be traced: a recorder of torch calls does not see their kernels");
}

bool needs(const Tensor& t) { return t.defined() && t.requires_grad(); }
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ---- top leaves -------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> top_forward(const Tensor& phi, int64_t L, int64_t k, bool renorm, int64_t ctx, bool want_total) {
  const Tensor p = rows(phi);
  const int64_t N = p.size(0);
  Tensor leaf = at::empty({N, k}, p.options().dtype(at::kInt)), weight = at::empty({N, k}, p.options()), total;
  if (want_total) total = at::empty({N}, p.options());
  check(lib.top_leaves(ctx_of(ctx), ptr<float>(p), std::max(pitch(p), L), N, L, k, renorm, ptr<int32_t>(leaf), ptr<float>(weight),
                       ptr<float>(total), stream_of(p)),
        "bnpvi_top_leaves");
  return {leaf, weight, total};
}

struct TopLeaves : Function<TopLeaves> {
  static variable_list forward(AutogradContext* c, const Tensor& phi, int64_t L, int64_t k, bool renorm, int64_t ctx) {
    auto [leaf, weight, total] = top_forward(phi, L, k, renorm, ctx, renorm);
    c->mark_non_differentiable({leaf});
    c->save_for_backward({leaf, weight, total});
    c->saved_data["s"] = std::vector<int64_t>{phi.size(0), phi.size(1), L, k, renorm, ctx};
    return {leaf, weight};
  }
  static variable_list backward(AutogradContext* c, variable_list given) {
    const auto saved = c->get_saved_variables();
    const auto s = c->saved_data["s"].toIntVector();
    const Tensor &leaf = saved[0], &weight = saved[1], &total = saved[2];
    Tensor dphi;
    if (given[1].defined()) {
      const Tensor d = plain(given[1]).contiguous();
      dphi = at::empty({s[0], s[1]}, weight.options());
      check(lib.top_leaves_backward(ctx_of(s[5]), ptr<int32_t>(leaf), ptr<float>(weight), ptr<float>(total), ptr<float>(d), s[0], s[2], s[3],
                                    s[4], ptr<float>(dphi), s[1], s[1], stream_of(leaf)),
            "bnpvi_top_leaves_backward");
    }
    return once({dphi, Tensor(), Tensor(), Tensor(), Tensor()}, given, saved);
  }
};

std::tuple<Tensor, Tensor> top_leaves(const Tensor& phi, int64_t L, int64_t k, bool renorm, int64_t ctx) {
  not_recorded();
  no_tangents({&phi});
  if (at::GradMode::is_enabled() && phi.requires_grad()) {
    auto out = TopLeaves::apply(phi, L, k, renorm, ctx);
    return {out[0], out[1]};
  }
  auto [leaf, weight, total] = top_forward(phi, L, k, renorm, ctx, false);
  return {leaf, weight};
}

// ---- sort, dispatch, combine ----------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> sort_by_leaf(const Tensor& leaf_in, int64_t L, int64_t ctx) {
  not_recorded();
  const Tensor leaf = leaf_in.contiguous();
  const int64_t N = leaf.size(0), k = leaf.size(1), M = N * k;
  Tensor place = at::empty({N, k}, leaf.options()), order = at::empty({M}, leaf.options()), offsets = at::empty({L + 1}, leaf.options()), work;
  const int64_t need = lib.leaf_sort_workspace(M, L);
  if (need > 0) work = at::empty({need}, leaf.options().dtype(at::kByte));
  check(lib.leaf_sort(ctx_of(ctx), ptr<int32_t>(leaf), M, L, ptr<int32_t>(place), ptr<int32_t>(order), ptr<int32_t>(offsets), ptr(work), need,
                      stream_of(leaf)),
        "bnpvi_leaf_sort");
  return {place, order, offsets};
}

Tensor to_leaves(const Tensor& x_in, const Tensor& place, const Tensor& offsets, int64_t ctx) {
  const Tensor x = rows(x_in);
  const int64_t N = place.size(0), k = place.size(1), D = x.size(1);
  Tensor xs = at::empty({N * k, D}, x.options());
  if (D)
    check(lib.rows_to_leaves(ctx_of(ctx), type_of(x), ptr(x), pitch(x), N, k, D, ptr<int32_t>(place), ptr<int32_t>(offsets), offsets.size(0) - 1,
                             ptr(xs), D, stream_of(x)),
          "bnpvi_rows_to_leaves");
  return xs;
}

Tensor from_leaves(const Tensor& ys_in, const Tensor& place, const Tensor& offsets, const Tensor& weight, int64_t ctx) {
  const Tensor ys = rows(ys_in);
  const int64_t N = place.size(0), k = place.size(1), D = ys.size(1);
  Tensor y = at::empty({N, D}, ys.options());
  if (D)
    check(lib.rows_from_leaves(ctx_of(ctx), type_of(ys), ptr(ys), pitch(ys), ptr<int32_t>(place), ptr<float>(weight), ptr<int32_t>(offsets),
                               offsets.size(0) - 1, N, k, D, ptr(y), D, stream_of(ys)),
          "bnpvi_rows_from_leaves");
  return y;
}

struct Dispatch : Function<Dispatch> {
  static Tensor forward(AutogradContext* c, const Tensor& x, const Tensor& place, const Tensor& offsets, int64_t ctx) {
    c->save_for_backward({place, offsets});
    c->saved_data["ctx"] = ctx;
    return to_leaves(x, place, offsets, ctx);
  }
  static variable_list backward(AutogradContext* c, variable_list given) {
    const auto saved = c->get_saved_variables();
    return once({from_leaves(plain(given[0]), saved[0], saved[1], Tensor(), c->saved_data["ctx"].toInt()), Tensor(), Tensor(), Tensor()}, given, saved);
  }
};

struct Combine : Function<Combine> {
  static Tensor forward(AutogradContext* c, const Tensor& ys, const std::optional<Tensor>& given, const Tensor& place, const Tensor& offsets,
                        int64_t ctx) {
    const Tensor weight = given.value_or(Tensor());
    c->save_for_backward({weight.defined() ? ys : Tensor(), weight, place, offsets});
    c->saved_data["ctx"] = ctx;
    return from_leaves(ys, place, offsets, weight, ctx);
  }
  static variable_list backward(AutogradContext* c, variable_list given) {
    const auto saved = c->get_saved_variables();
    const Tensor &weight = saved[1], &place = saved[2], &offsets = saved[3];
    const int64_t ctx = c->saved_data["ctx"].toInt();
    Tensor dys, dweight;
    if (!weight.defined()) {
      dys = to_leaves(plain(given[0]), place, offsets, ctx);
    } else {
      const Tensor dy = rows(plain(given[0])), ys = rows(saved[0]);
      const int64_t N = place.size(0), k = place.size(1), D = ys.size(1);
      if (c->needs_input_grad(0)) dys = at::empty({N * k, D}, ys.options());
      if (c->needs_input_grad(1)) dweight = D ? at::empty({N, k}, weight.options()) : at::zeros({N, k}, weight.options());
      if (D)
        check(lib.rows_from_leaves_backward(ctx_of(ctx), type_of(ys), ptr(dy), pitch(dy), ptr(ys), pitch(ys), ptr<int32_t>(place),
                                            ptr<float>(weight), ptr<int32_t>(offsets), offsets.size(0) - 1, N, k, D, ptr(dys), D,
                                            ptr<float>(dweight), stream_of(ys)),
              "bnpvi_rows_from_leaves_backward");
    }
    return once({dys, dweight, Tensor(), Tensor(), Tensor()}, given, saved);
  }
};

Tensor dispatch(const Tensor& x, const Tensor& place, const Tensor& offsets, int64_t ctx) {
  not_recorded();
  no_tangents({&x});
  if (at::GradMode::is_enabled() && x.requires_grad()) return Dispatch::apply(x, place, offsets, ctx);
  return to_leaves(x, place, offsets, ctx);
}

Tensor combine(const Tensor& ys, const Tensor& place, const Tensor& offsets, const std::optional<Tensor>& weight, int64_t ctx) {
  not_recorded();
  const Tensor w = weight ? weight->contiguous() : Tensor();
  no_tangents({&ys, &w});
  if (at::GradMode::is_enabled() && (ys.requires_grad() || needs(w)))
    return Combine::apply(ys, maybe(w), place, offsets, ctx);
  return from_leaves(ys, place, offsets, w, ctx);
}

// ---- dense -----------------------------------------------------------------------------------------------------------
// The workspace of a call goes by its sizes and the bits of `call`; a program has few of them.
int64_t dense_workspace(int type, int64_t M, int64_t K, int64_t n, int64_t G, int call) {
  struct Key {
    int64_t v[6];
    bool operator==(const Key& o) const { return std::equal(v, v + 6, o.v); }
  };
  struct Hash {
    size_t operator()(const Key& k) const {
      size_t h = 0;
      for (int64_t x : k.v) h = h * 1000003u ^ std::hash<int64_t>()(x);
      return h;
    }
  };
  static std::mutex mutex;
  static std::unordered_map<Key, int64_t, Hash> known;
  const Key key{{type, M, K, n, G, call}};
  std::lock_guard<std::mutex> hold(mutex);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  if (known.size() >= 4096) known.clear();
  return known[key] = lib.dense_workspace(type, M, K, n, static_cast<int>(G), call);
}

// A weight (n, K) or (G, n, K) with contiguous rows, and its pitches.
struct Weights {
  Tensor t;
  int64_t row, group;
};
Weights weights(const Tensor& w) {
  const int64_t n = w.size(-2), K = w.size(-1);
  const bool fits = (K == 1 || w.stride(-1) == 1) && (n == 1 || (w.stride(-2) >= K && w.stride(-2) * w.element_size() <= kMaxPitchBytes));
  const Tensor t = fits ? w : w.contiguous();
  return {t, n > 1 ? t.stride(-2) : K, t.dim() == 3 && t.size(0) > 1 ? t.stride(0) : 0};
}

// `bit` where the operand is off 16 bytes.
int off16(const Tensor& t, int64_t pitch, int64_t group, int64_t width, int bit) {
  const uint64_t all = reinterpret_cast<uint64_t>(ptr(t)) | static_cast<uint64_t>((pitch | group | width) * t.element_size());
  return all & 15 ? bit : 0;
}

std::tuple<Tensor, Tensor> dense_forward(const Tensor& x_in, const Tensor& w_in, const Tensor& bias_in, const Tensor& res_in,
                                         const Tensor& offsets, int64_t act, int64_t ctx, bool want_dact) {
  const Tensor x = rows(x_in), bias = bias_in.defined() ? bias_in.contiguous() : bias_in, res = res_in.defined() ? rows(res_in) : res_in;
  const Weights w = weights(w_in);
  const int64_t M = x.size(0), K = x.size(1), n = w.t.size(-2), G = w.t.dim() == 3 ? w.t.size(0) : 0;
  const int type = type_of(x);
  Tensor y = at::empty({M, n}, x.options()), dact, work;
  if (want_dact && act != BNPVI_ACT_NONE) dact = at::empty({M, n}, x.options().dtype(at::kFloat));
  const int64_t need = dense_workspace(type, M, K, n, G, off16(x, pitch(x), 0, K, BNPVI_DENSE_X_OFF) |
                                                             off16(w.t, w.row, w.group, K, BNPVI_DENSE_W_OFF));
  if (need > 0) work = at::empty({need}, x.options().dtype(at::kByte));
  check(lib.dense(ctx_of(ctx), type, ptr(x), pitch(x), ptr(w.t), w.row, w.group, ptr(bias), G > 1 ? n : 0, act, ptr(res),
                  res.defined() ? pitch(res) : 0, ptr<int32_t>(offsets), G, M, K, n, ptr(y), n, ptr(dact), n, ptr(work), need, stream_of(x)),
        "bnpvi_dense");
  return {y, dact};
}

struct Dense : Function<Dense> {
  static Tensor forward(AutogradContext* c, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                        const std::optional<Tensor>& res, const std::optional<Tensor>& bounds, int64_t act, int64_t ctx, bool want_dact) {
    const Tensor offsets = bounds.value_or(Tensor());
    auto [y, dact] = dense_forward(x, w, bias.value_or(Tensor()), res.value_or(Tensor()), offsets, act, ctx, want_dact);
    c->save_for_backward({x, w, offsets, dact});
    c->saved_data["ctx"] = ctx;
    c->saved_data["act"] = act;
    c->saved_data["given"] = (bias ? 1 : 0) + (res ? 2 : 0);          // only tensors that are there count as inputs
    return y;
  }
  static variable_list backward(AutogradContext* c, variable_list given) {
    const auto saved = c->get_saved_variables();
    const Tensor &x0 = saved[0], &w0 = saved[1], &offsets = saved[2], &dact = saved[3];
    const int64_t ctx = c->saved_data["ctx"].toInt(), M = x0.size(0), K = x0.size(1), n = w0.size(-2), G = w0.dim() == 3 ? w0.size(0) : 0;
    const int type = type_of(x0);
    Tensor dx, dw, db, dres, work;
    const Tensor dy = rows(plain(given[0])), x = rows(x0);
    const Weights w = weights(w0);
    if (c->needs_input_grad(0)) dx = at::empty({M, K}, x.options());
    if (c->needs_input_grad(1)) dw = at::empty(w0.sizes(), x.options());
    const int64_t has = c->saved_data["given"].toInt(), act = c->saved_data["act"].toInt();
    if ((has & 1) && c->needs_input_grad(2)) db = at::empty(w0.sizes().slice(0, w0.dim() - 1), x.options());
    const bool need_res = (has & 2) && c->needs_input_grad(2 + (has & 1));
    if (need_res && G) dres = at::empty({M, n}, x.options());
    if (dx.defined() || dw.defined() || db.defined() || dres.defined()) {
      const int call = BNPVI_DENSE_BACKWARD | off16(x, pitch(x), 0, K, BNPVI_DENSE_X_OFF) | off16(w.t, w.row, w.group, K, BNPVI_DENSE_W_OFF) |
                       off16(dy, pitch(dy), 0, n, BNPVI_DENSE_DY_OFF) | (ptr(dact) ? BNPVI_DENSE_DACT : 0) |
                       (ptr(dact) && act == BNPVI_ACT_RELU ? BNPVI_DENSE_STEP : 0) | (ptr(dx) ? BNPVI_DENSE_DX : 0) |
                       (dw.defined() ? BNPVI_DENSE_DW : 0) | (db.defined() ? BNPVI_DENSE_DB : 0) | (ptr(dres) ? BNPVI_DENSE_DRES : 0);
      const int64_t need = dense_workspace(type, M, K, n, G, call);
      if (need > 0) work = at::empty({need}, x.options().dtype(at::kByte));
      check(lib.dense_backward(ctx_of(ctx), type, static_cast<int>(act), ptr(dy), pitch(dy), ptr(dact), n, ptr(x), pitch(x), ptr(w.t), w.row, w.group,
                               ptr<int32_t>(offsets), G, M, K, n, ptr(dx), K, ptr(dw), ptr(db), ptr(dres), n, ptr(work), need, stream_of(x)),
            "bnpvi_dense_backward");
    }
    if (need_res && !G) dres = given[0];
    return once({dx, dw, db, dres, Tensor(), Tensor(), Tensor(), Tensor()}, given, saved);
  }
};

Tensor dense(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const std::optional<Tensor>& res,
             const std::optional<Tensor>& offsets, int64_t act, int64_t ctx) {
  not_recorded();
  const Tensor b = bias.value_or(Tensor()), r = res.value_or(Tensor()), o = offsets ? offsets->contiguous() : Tensor();
  no_tangents({&x, &w, &b, &r});
  if (at::GradMode::is_enabled()) {
    const bool inner = x.requires_grad() || w.requires_grad() || needs(b);
    if (inner || needs(r)) return Dense::apply(x, w, maybe(b), maybe(r), maybe(o), act, ctx, inner);
  }
  return std::get<0>(dense_forward(x, w, b, r, o, act, ctx, false));
}

}  // namespace

PYBIND11_MODULE(_torch_layers, m) {
  m.def("bind", &bind);
  m.def("top_leaves", &top_leaves, py::call_guard<py::gil_scoped_release>());
  m.def("sort_by_leaf", &sort_by_leaf, py::call_guard<py::gil_scoped_release>());
  m.def("dispatch", &dispatch, py::call_guard<py::gil_scoped_release>());
  m.def("combine", &combine, py::call_guard<py::gil_scoped_release>());
  m.def("dense", &dense, py::call_guard<py::gil_scoped_release>());
  static PyObject* error = py::object(py::module_::import("bnp_vae_amd._lib").attr("BnpviError")).release().ptr();
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      PyErr_SetString(error, e.what());
    }
  });
}
