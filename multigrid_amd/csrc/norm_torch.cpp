// The torch side of include/mgrid_norm.h: argument checks, autograd and memory of layer_norm, grad_norm and clip_grads, with
// the plain torch expression of the same formulas for tensors that are not on a GPU.  multigrid_amd/norm_ops.py documents and
// re-exports them.  In C++ because the smallest calls are bound by their host time: the autograd graph's nodes, the
// allocations and a list of gradients cost several times as much from Python (a small layer norm's forward call 9.4 us
// against 4.2 here, forward and backward 98 against 61, clipping a list of 36 gradients 48 against 14).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "mgrid_norm.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

// the kernels' number of an element type; -1: none
int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MGNN_F32;
    case at::kBFloat16: return MGNN_BF16;
    case at::kHalf: return MGNN_F16;
    default: return -1;
  }
}
bool takes(const Tensor& t) { return type_of(t) >= 0 && t.layout() == at::kStrided; }

void check(int rc, const char* what) {
  TORCH_CHECK(rc != MGNN_ERR_LAUNCH, what, ": the kernel launch failed");
  TORCH_CHECK_VALUE(rc != MGNN_ERR_OVERLAP, what, ": a gradient that is written overlaps another one of the call");
  TORCH_CHECK_VALUE(rc == MGNN_OK, what, ": refused with MGNN error ", rc);
}

// The kernels carry no forward-mode tangent, and would lose that of an input without a word
void check_no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative on a GPU");
}

// A trace (torch.jit.trace, make_fx) records the allocation of a kernel's results but not the kernel: its replay would return
// memory that nothing has written
void check_no_trace(const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                              what, "'s kernels cannot be recorded in a trace");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor bytes_on(const Tensor& t, int64_t size) { return size > 0 ? at::empty({size}, t.options().dtype(at::kByte)) : Tensor(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- layer norm ----

// x by rows (x itself, a view of it, or a copy) with the elements of a row contiguous, and the distance of its rows
std::pair<Tensor, int64_t> rows_of(const Tensor& x, int64_t cols) {
  if (x.is_contiguous()) return {x, cols};
  Tensor r = x.reshape({-1, cols});
  if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < cols)) return {r.contiguous(), cols};
  return {r, r.size(0) > 1 ? r.stride(0) : cols};
}

struct Sizes {
  int64_t groups, rows, cols;
  int type, wtype;
};

Tensor forward_kernel(const Tensor& x, int64_t ld, at::IntArrayRef shape, const Tensor& w, const Tensor& b, const Tensor& stats, double eps,
                      const Sizes& s) {
  Tensor y = at::empty(shape, x.options());
  check(mgnn_layer_norm(x.data_ptr(), ld, data(w), data(b), y.data_ptr(), stats.defined() ? stats.data_ptr<float>() : nullptr, s.groups, s.rows,
                        (int)s.cols, eps, s.type, s.wtype, stream_of(x)),
        "layer_norm");
  return y;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                        const Sizes& s) {
    const auto [rows, ld] = rows_of(x, s.cols);
    const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
    const Tensor stats = at::empty({s.groups * s.rows, 2}, x.options().dtype(at::kFloat));
    Tensor y = forward_kernel(rows, ld, x.sizes(), w, b, stats, eps, s);
    ctx->save_for_backward({rows, stats, w});
    ctx->saved_data["sizes"] = std::vector<int64_t>{s.groups, s.rows, s.cols, s.type, s.wtype};
    ctx->saved_data["affine"] = std::vector<int64_t>{weight.has_value(), bias.has_value(), weight ? weight->dim() : bias ? bias->dim() : 0};
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm is differentiable once: its gradients have no graph (create_graph)");
    check_no_tangent(grads[0], "layer_norm's backward pass");
    check_no_trace("layer_norm's backward pass");
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["sizes"].toIntVector(), affine = ctx->saved_data["affine"].toIntVector();
    const Sizes s{n[0], n[1], n[2], (int)n[3], (int)n[4]};
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor dy = grads[0].contiguous();
    // hooks on saved tensors may give them back in other memory, with other strides
    const auto as_saved = [&](const Tensor& t, int type, int64_t count) {
      return t.device() == dy.device() && t.layout() == at::kStrided && type_of(t) == type && t.numel() == count;
    };
    TORCH_CHECK(as_saved(saved[0], s.type, s.groups * s.rows * s.cols) && as_saved(saved[1], MGNN_F32, s.groups * s.rows * 2) &&
                    (!affine[0] || as_saved(saved[2], s.wtype, s.groups * s.cols)),
                "layer_norm's saved tensors came back on another device, or of another type or size");
    const auto [x, ld] = rows_of(saved[0], s.cols);
    const Tensor stats = saved[1].contiguous(), w = affine[0] ? saved[2].contiguous() : Tensor();
    // the node's edges are those of the tensors that were given
    const bool want_w = affine[0] && ctx->needs_input_grad(1), want_b = affine[1] && ctx->needs_input_grad(affine[0] ? 2 : 1);
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = at::empty_like(dy);
    const auto row_shape = affine[2] == 2 ? std::vector<int64_t>{s.groups, s.cols} : std::vector<int64_t>{s.cols};
    const auto row_options = x.options().dtype(s.wtype == MGNN_F32 ? at::kFloat : x.scalar_type());
    if (want_w) dw = at::empty(row_shape, row_options);
    if (want_b) db = at::empty(row_shape, row_options);
    const int64_t size = want_w || want_b ? mgnn_layer_norm_workspace(s.groups, s.rows, (int)s.cols, s.type) : 0;
    const Tensor room = bytes_on(x, size);
    check(mgnn_layer_norm_backward(x.data_ptr(), ld, dy.data_ptr(), data(w), stats.data_ptr<float>(), data(dx), data(dw), data(db), data(room),
                                   size, s.groups, s.rows, (int)s.cols, s.type, s.wtype, stream_of(x)),
          "layer_norm's backward pass");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

Tensor plain_layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
  const auto row = [&](const Tensor& t) {      // a stacked weight against x
    if (t.dim() == 1) return t.to(at::kFloat);
    std::vector<int64_t> shape(x.dim(), 1);
    shape.front() = x.size(0);
    shape.back() = x.size(-1);
    return t.to(at::kFloat).reshape(shape);
  };
  Tensor h = at::layer_norm(x.to(at::kFloat), {x.size(-1)}, {}, {}, eps);
  if (weight) h = h * row(*weight);
  if (bias) h = h + row(*bias);
  return h.to(x.scalar_type());
}

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
  TORCH_CHECK_TYPE(takes(x), "layer_norm takes dense float32, bfloat16 or float16 tensors, not ", x.scalar_type(), ", ", x.layout());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= MGNN_LN_MAX_C, "layer_norm takes rows of 1 to ", MGNN_LN_MAX_C,
                    " elements, not a tensor of shape ", x.sizes());
  TORCH_CHECK_VALUE(eps >= 0 && !std::isinf(eps), "layer_norm takes a finite eps >= 0, not ", eps);
  Sizes s{1, 0, x.size(-1), type_of(x), type_of(x)};
  for (const MaybeTensor* p : {&weight, &bias}) {
    if (!*p) continue;
    const Tensor& t = **p;
    TORCH_CHECK_TYPE(takes(t) && (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat),
                     "layer_norm's weight and bias are dense, of x's type (", x.scalar_type(), ") or float32, not ", t.scalar_type());
    TORCH_CHECK_VALUE(t.device() == x.device(), "layer_norm's weight and bias are on ", t.device(), ", x on ", x.device());
    const bool stacked = t.dim() == 2 && x.dim() >= 2 && t.size(0) == x.size(0);
    TORCH_CHECK_VALUE((t.dim() == 1 || stacked) && t.size(-1) == s.cols, "layer_norm's weight or bias of shape ", t.sizes(),
                      " does not fit x of shape ", x.sizes(), ": [cols] or [x.shape[0], cols] is wanted");
    if (stacked) s.groups = t.size(0);
    s.wtype = type_of(t);
  }
  TORCH_CHECK_VALUE(!weight || !bias || (weight->sizes() == bias->sizes() && weight->scalar_type() == bias->scalar_type()),
                    "layer_norm's weight and bias differ in shape or type");
  TORCH_CHECK_VALUE(s.groups <= MGNN_MAX_GROUPS, "layer_norm takes at most ", MGNN_MAX_GROUPS, " weight rows, not ", s.groups);
  if (!x.is_cuda()) return plain_layer_norm(x, weight, bias, eps);
  check_no_trace("layer_norm");
  check_no_tangent(x, "layer_norm");
  if (weight) check_no_tangent(*weight, "layer_norm");
  if (bias) check_no_tangent(*bias, "layer_norm");
  s.rows = s.groups ? x.numel() / s.cols / s.groups : 0;
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
    return LayerNorm::apply(x, weight, bias, eps, s);
  const auto [rows, ld] = rows_of(x, s.cols);
  return forward_kernel(rows, ld, x.sizes(), weight ? weight->contiguous() : Tensor(), bias ? bias->contiguous() : Tensor(), Tensor(), eps, s);
}

// ---- the global gradient norm ----

using Tensors = std::vector<Tensor>;

// Whether t's elements fill one stretch of memory, in whatever order (stacked: agent by agent)
bool dense(const Tensor& t, bool stacked) {
  return t.is_contiguous() || (t.is_non_overlapping_and_dense() && (!stacked || t.size(0) == 1 || t.stride(0) == t.numel() / t.size(0)));
}

void check_grads(const Tensors& grads, int64_t stacked) {
  TORCH_CHECK_VALUE(stacked >= 0 && stacked <= MGNN_MAX_GROUPS, "stacked is the length of the leading agent axis, 0 (none) to ", MGNN_MAX_GROUPS,
                    ", not ", stacked);
  for (const Tensor& g : grads) {
    TORCH_CHECK_TYPE(takes(g), "gradients are dense float32, bfloat16 or float16 tensors, not ", g.scalar_type(), ", ", g.layout());
    TORCH_CHECK_VALUE(g.device() == grads[0].device(), "gradients are on ", grads[0].device(), " and ", g.device(), ": one device is wanted");
    TORCH_CHECK_VALUE(!stacked || (g.dim() >= 1 && g.size(0) == stacked), "a gradient of shape ", g.sizes(), " has no leading agent axis of ",
                      stacked);
  }
}

// Whether a sum of step * i over all terms, with 0 <= i <= most for each, can be `total`: exactly, by the terms from the largest
// step down.  Steps that nest, as those of a slice do, leave two or three choices each, and a rest whose terms reach every
// value needs none; other steps may leave many, of which 2^20 are tried before the answer is yes.
class Sums {
 public:
  void add(int64_t step, int64_t most) {
    if (step > 0 && most > 0) terms_.push_back({step, most, 0, false});
  }
  bool reach(int64_t total) {
    std::sort(terms_.begin(), terms_.end(), [](const Term& a, const Term& b) { return a.step < b.step; });
    int64_t below = 0;
    bool every = true;
    size_t n = 0;
    for (const Term& t : terms_) {
      if (n && terms_[n - 1].step == t.step) terms_[n - 1].most += t.most;
      else terms_[n++] = t;
    }
    terms_.resize(n);
    for (Term& t : terms_) {
      t.below = below;
      t.every = every;
      every = every && t.step <= below + 1;
      below += t.step * t.most;
    }
    tries_ = 1 << 20;
    return search(n, total, below, every);
  }

 private:
  struct Term {
    int64_t step, most;
    int64_t below;      // what the smaller ones reach together
    bool every;         // whether they reach all values up to that
  };
  bool search(size_t n, int64_t total, int64_t limit, bool every) {
    if (total < 0 || total > limit) return false;
    if (every) return true;
    const Term& t = terms_[n - 1];
    const int64_t high = std::min(t.most, total / t.step), low = std::max<int64_t>(0, (total - t.below + t.step - 1) / t.step);
    for (int64_t i = high; i >= low; --i)
      if (--tries_ < 0 || search(n - 1, total - i * t.step, t.below, t.every)) return true;
    return false;
  }
  c10::SmallVector<Term, 8> terms_;
  int64_t tries_ = 0;
};

// Whether two of t's elements lie at one address: with k the axis of largest number along which their places differ by at least 1, the
// other differences, counted from the least possible one, have to make up for it
bool overlaps_itself(const Tensor& t) {
  if (t.numel() <= 1 || t.is_non_overlapping_and_dense()) return false;
  for (int64_t k = 0; k < t.dim(); ++k) {
    if (t.size(k) <= 1) continue;
    Sums sums;
    int64_t total = -t.stride(k);
    for (int64_t d = 0; d < t.dim(); ++d) {
      sums.add(t.stride(d), d == k ? t.size(d) - 2 : 2 * (t.size(d) - 1));
      if (d != k) total += t.stride(d) * (t.size(d) - 1);
    }
    if (sums.reach(total)) return true;
  }
  return false;
}

// A tensor's elements in memory
struct Place {
  const Tensor* t;
  uintptr_t from, to;      // its first byte, and the one behind its last
  size_t index;
  bool written;
};
Place place_of(const Tensor& t, size_t index, bool written) {
  uintptr_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += t.stride(d) * (t.size(d) - 1);
  const uintptr_t from = reinterpret_cast<uintptr_t>(written ? t.mutable_data_ptr() : t.const_data_ptr());
  return {&t, from, from + (last + 1) * t.element_size(), index, written};
}
bool overlap(const Place& a, const Place& b) {      // a.from <= b.from
  if (b.from >= a.to) return false;
  Sums sums;
  int64_t total = b.to - 1 - a.from;      // a's bytes counted from its first, b's from its last backwards
  for (const Place* p : {&a, &b}) {
    sums.add(1, p->t->element_size() - 1);
    for (int64_t d = 0; d < p->t->dim(); ++d) sums.add(p->t->stride(d) * p->t->element_size(), p->t->size(d) - 1);
  }
  return sums.reach(total);
}

// Refuses results whose memory holds another result, another tensor's gradient or two elements of their own.  (A result may
// lie over its own gradient: that is read whole before the result is written, or is the very same tensor.)
void check_memory(const Tensors& grads, const Tensors& out) {
  std::vector<Place> places;
  for (size_t i = 0; i < out.size(); ++i) {
    const Tensor &o = out[i], &g = grads[i];
    // without memory of their own: tensors of the meta device, and those that Python classes stand for (fake tensors)
    const auto none = [](const Tensor& t) { return t.is_meta() || t.key_set().has(c10::DispatchKey::Python); };
    if (o.numel() == 0 || none(o) || none(g)) continue;
    TORCH_CHECK_VALUE(!overlaps_itself(o), "a gradient that is written has several elements at one address (it overlaps itself)");
    places.push_back(place_of(o, i, true));
    if (!g.is_same(o)) places.push_back(place_of(g, i, false));
  }
  std::sort(places.begin(), places.end(), [](const Place& a, const Place& b) { return a.from < b.from; });
  std::vector<const Place*> open;      // those that may reach the next one
  for (const Place& p : places) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Place* q) { return q->to <= p.from; }), open.end());
    for (const Place* q : open)
      TORCH_CHECK_VALUE(q->index == p.index || !(q->written || p.written) || !overlap(*q, p),
                        "clip_grads: a gradient that is written overlaps another one of the call");
    open.push_back(&p);
  }
}

// What these return has no graph: an input's would end there without a word
void check_no_graph(const Tensors& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& g : grads)
    TORCH_CHECK(!g.requires_grad(), what, " has no derivative, and one of the gradients requires grad: detach them or call it under torch.no_grad()");
}

std::vector<int64_t> norm_shape(int64_t stacked) { return stacked ? std::vector<int64_t>{stacked} : std::vector<int64_t>{}; }

Tensor plain_norms(const Tensors& grads, int64_t stacked) {      // float64
  Tensor sum = grads.empty() ? at::zeros(norm_shape(stacked), at::kDouble) : at::zeros(norm_shape(stacked), grads[0].options().dtype(at::kDouble));
  for (const Tensor& g : grads) {
    const Tensor sq = g.to(at::kDouble).square();
    sum = sum + (stacked ? sq.reshape({stacked, -1}).sum(1) : sq.sum());
  }
  return sum.sqrt();
}

// The kernels on dense tensors; dst NULL: the norms alone
Tensor launch(const Tensors& src, const Tensors* dst, double max_norm, int64_t stacked) {
  const int64_t groups = std::max<int64_t>(stacked, 1), count = (int64_t)src.size();
  std::vector<const void*> from(count);
  std::vector<void*> to(count);
  std::vector<int64_t> n(count);
  std::vector<int32_t> type(count);
  for (int64_t i = 0; i < count; ++i) {
    from[i] = src[i].data_ptr();
    if (dst) to[i] = (*dst)[i].data_ptr();
    n[i] = src[i].numel() / groups;
    type[i] = type_of(src[i]);
  }
  const c10::DeviceGuard guard(src[0].device());
  Tensor norms = at::empty(norm_shape(stacked), src[0].options().dtype(at::kFloat));
  const int64_t size = mgnn_grad_norm_workspace(n.data(), type.data(), count, groups);
  const Tensor room = bytes_on(src[0], size);
  void* const stream = stream_of(src[0]);
  check(dst ? mgnn_clip_grads(from.data(), to.data(), n.data(), type.data(), count, groups, max_norm, norms.data_ptr<float>(), data(room), size,
                              stream)
            : mgnn_grad_norm(from.data(), n.data(), type.data(), count, groups, norms.data_ptr<float>(), data(room), size, stream),
        dst ? "clip_grads" : "grad_norm");
  return norms;
}

Tensor grad_norm(const Tensors& grads, int64_t stacked) {
  check_grads(grads, stacked);
  check_no_graph(grads, "grad_norm");
  const at::NoGradGuard no_grad;
  if (grads.empty() || !grads[0].is_cuda()) return plain_norms(grads, stacked).to(at::kFloat);
  check_no_trace("grad_norm");
  for (const Tensor& g : grads) check_no_tangent(g, "grad_norm");
  Tensors src;
  for (const Tensor& g : grads) src.push_back(dense(g, stacked) ? g : g.contiguous());
  return launch(src, nullptr, 0.0, stacked);
}

std::tuple<Tensors, Tensor> clip_grads(const Tensors& grads, double max_norm, int64_t stacked, const std::optional<Tensors>& given) {
  check_grads(grads, stacked);
  TORCH_CHECK_VALUE(max_norm >= 0, "max_norm is a number >= 0, not ", max_norm);
  if (!given) check_no_graph(grads, "clip_grads without out");
  const at::NoGradGuard no_grad;
  const size_t count = grads.size();
  Tensors out;
  if (given) {
    TORCH_CHECK_VALUE(given->size() == count, given->size(), " tensors in out for ", count, " gradients");
    out = *given;
    for (size_t i = 0; i < count; ++i) {
      const Tensor &o = out[i], &g = grads[i];
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && o.scalar_type() == g.scalar_type() && o.device() == g.device() && o.layout() == at::kStrided,
                        "out does not match the gradients in shape, type or device");
    }
  } else {
    for (const Tensor& g : grads) out.push_back(at::empty_like(g));
  }
  if (count == 0 || !grads[0].is_cuda()) {
    if (given) check_memory(grads, out);
    const Tensor norms = plain_norms(grads, stacked), factor = (max_norm / (norms + 1e-6)).clamp_max(1.0).to(at::kFloat);
    for (size_t i = 0; i < count; ++i) {
      std::vector<int64_t> wide(grads[i].dim(), 1);
      if (stacked) wide[0] = stacked;
      out[i].copy_(grads[i].to(at::kFloat) * (stacked ? factor.reshape(wide) : factor));
    }
    return {out, norms.to(at::kFloat)};
  }
  check_no_trace("clip_grads");
  for (const Tensor& g : grads) check_no_tangent(g, "clip_grads");
  // tensors without a common dense order go through contiguous copies; the kernels' entry point, which sees those instead of the
  // caller's memory, checks the lists that need none
  Tensors src(grads), dst(out);
  bool copies = false;
  for (size_t i = 0; i < count; ++i) {
    if ((src[i].is_contiguous() && dst[i].is_contiguous()) || (src[i].strides() == dst[i].strides() && dense(src[i], stacked))) continue;
    if (given && !copies) check_memory(grads, out);
    copies = true;
    src[i] = src[i].contiguous();
    dst[i] = at::empty(out[i].sizes(), out[i].options());
  }
  const Tensor norms = launch(src, &dst, max_norm, stacked);
  for (size_t i = 0; i < count; ++i) {
    if (!dst[i].is_same(out[i])) out[i].copy_(dst[i]);
    else if (!out[i].is_inference()) out[i].unsafeGetTensorImpl()->bump_version();      // a graph that saved it will say so
  }
  return {out, norms};
}

}  // namespace

PYBIND11_MODULE(_norm_ops, m) {
  namespace py = pybind11;
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight") = py::none(), py::arg("bias") = py::none(), py::arg("eps") = 1e-5);
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("stacked") = 0);
  m.def("clip_grads", &clip_grads, py::arg("grads"), py::arg("max_norm"), py::arg("stacked") = 0, py::arg("out") = py::none());
}
