// The Python module fedsim_amd._fedtrain: libfedtrain's entries on torch tensors.
//
// Arguments are checked here (TypeError for types, ValueError for shapes,
// devices and strides), outputs and workspaces come from torch's allocator on
// the tensors' device, launches go to its current stream.  The differentiable
// operators live on this side too: a step of a small model is bound by the
// host, and a Python backward costs three times its kernels there.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/fedtrain.h"

namespace {

using at::Tensor;
using std::optional;

constexpr int64_t kMax = 2147483647;  // of one dimension
constexpr int64_t kStateBlock = 256;

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed (", status, "): ", fedtrain_strerror(status));
}

// A tracer sees torch's own operators alone: of a call here the allocation of its
// results, which a replay would return as they come.
void not_traced() {
  using Mode = c10::impl::TorchDispatchModeKey;
  bool traced = torch::jit::tracer::isTracing() ||
                c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  if (c10::impl::TorchDispatchModeTLS::any_modes_set())
    for (const Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
      traced |= c10::impl::TorchDispatchModeTLS::get_mode(m).has_value();
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "the training operators cannot be traced (torch.jit.trace, "
                                       "make_fx, torch.export): a graph would hold their "
                                       "results' allocation alone");
}

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return FEDTRAIN_F32;
    case at::kBFloat16: return FEDTRAIN_BF16;
    case at::kHalf: return FEDTRAIN_F16;
    default:
      TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, got ",
                       t.scalar_type());
  }
}

void require(const Tensor& t, const char* name) {
  dtype_of(t, name);
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must live on a HIP device, got ", t.device());
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, name, " must be a strided tensor");
}

void require(const Tensor& t, const char* name, const Tensor& like) {
  require(t, name);
  TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), name, " must be ", like.scalar_type(),
                   " like x, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must live on ", like.device(), ", got ",
                    t.device());
}

// The last dimension's elements next to each other, as they are in memory.
Tensor rows(const Tensor& t) {
  if (t.is_neg()) return t.resolve_neg().contiguous();
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// Elements from one row (dim -2) or matrix (-3) to the next; where there is one,
// what a packed tensor has.
int64_t step(const Tensor& t, int64_t dim = -2) {
  if (t.size(dim) > 1) return t.stride(dim);
  return dim == -2 ? t.size(-1) : t.size(-1) * t.size(-2);
}

void fits(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= kMax, name, " = ", n, " is over the largest size, ", kMax);
}

int activation_of(const std::string& name) {
  if (name == "none") return FEDTRAIN_ACT_NONE;
  if (name == "relu") return FEDTRAIN_ACT_RELU;
  if (name == "gelu") return FEDTRAIN_ACT_GELU;
  if (name == "silu") return FEDTRAIN_ACT_SILU;
  TORCH_CHECK_VALUE(false, "activation must be one of none, relu, gelu, silu, got ", name);
}

// A device made current for a launch (a stream handle of 0 is the current
// device's default stream), and its current stream.
struct On {
  explicit On(const at::Device& d)
      : guard(d), stream(c10::hip::getCurrentHIPStream(d.index()).stream()) {}
  c10::DeviceGuard guard;
  void* stream;
};

template <class Args>
int groups_of(int64_t groups, const Tensor& offsets, const at::Device& d, Args* a) {
  TORCH_CHECK_TYPE(offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong,
                   "offsets must be int32 or int64, got ", offsets.scalar_type());
  TORCH_CHECK_VALUE(offsets.device() == d, "offsets must live on ", d, ", got ",
                    offsets.device());
  if (groups < 0) groups = offsets.numel() - 1;
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() == groups + 1 && groups >= 1,
                    "offsets must hold one more value than there are groups (", groups,
                    "), got shape ", offsets.sizes());
  TORCH_CHECK_VALUE(offsets.is_contiguous(), "offsets must be contiguous");
  fits(groups + 2, "groups");
  a->groups = static_cast<int32_t>(groups);
  a->offsets = offsets.const_data_ptr();
  a->offsets64 = offsets.scalar_type() == at::kLong;
  return a->groups;
}

void launch(fedtrain_product_args& a, const Tensor& on) {
  const On at(on.device());
  Tensor work;
  const int64_t need = fedtrain_product_workspace(&a);
  TORCH_CHECK(need >= 0, "fedtrain_product_workspace failed (", need,
              "): ", fedtrain_strerror(static_cast<int>(need)));
  if (need > 0) {
    work = at::empty({need}, on.options().dtype(at::kByte).requires_grad(false));
    a.workspace = work.mutable_data_ptr();
    a.workspace_bytes = need;
  }
  check(fedtrain_product(&a, at.stream), "fedtrain_product");
}

Tensor make(at::IntArrayRef sizes, const Tensor& like) {
  return at::empty(sizes, like.options().requires_grad(false));
}

std::tuple<Tensor, Tensor> forward_of(const Tensor& x_, const Tensor& w_,
                                      const optional<Tensor>& b_, const optional<Tensor>& r_,
                                      int act, const optional<Tensor>& offsets, bool want_z) {
  not_traced();
  require(x_, "x");
  require(w_, "weight", x_);
  const bool grouped = offsets.has_value();
  TORCH_CHECK_VALUE(x_.dim() == 2 && w_.dim() == (grouped ? 3 : 2) && w_.size(-1) == x_.size(1),
                    "x ", x_.sizes(), " and weight ", w_.sizes(), " do not fit [N, in] and ",
                    grouped ? "[G, out, in]" : "[out, in]");
  const int64_t N = x_.size(0), K = x_.size(1), M = w_.size(-2);
  fits(N, "rows");
  fits(K, "inputs");
  fits(M, "outputs");
  fedtrain_product_args a = {};
  a.dtype = dtype_of(x_, "x");
  a.form = FEDTRAIN_FORWARD;
  a.act = act;
  if (grouped) groups_of(w_.size(0), *offsets, x_.device(), &a);
  Tensor b, r;
  if (b_) {
    require(*b_, "bias", x_);
    TORCH_CHECK_VALUE(b_->sizes() == w_.sizes().slice(0, w_.dim() - 1), "bias must have shape ",
                      w_.sizes().slice(0, w_.dim() - 1), ", got ", b_->sizes());
    b = rows(*b_);
    a.bias = b.const_data_ptr();
    a.bias_group = grouped ? step(b) : 0;
  }
  if (r_) {
    require(*r_, "residual", x_);
    TORCH_CHECK_VALUE(r_->dim() == 2 && r_->size(0) == N && r_->size(1) == M,
                      "residual must have shape [", N, ", ", M, "], got ", r_->sizes());
    r = rows(*r_);
    a.res = r.const_data_ptr();
    a.ldr = step(r);
  }
  const Tensor x = rows(x_), w = rows(w_);
  Tensor y = make({N, M}, x), z;
  if (want_z) {
    z = make({N, M}, x);
    a.z = z.mutable_data_ptr();
    a.ldz = M;
  }
  a.m = N;
  a.n = M;
  a.k = K;
  a.a = x.const_data_ptr();
  a.lda = step(x);
  a.b = w.const_data_ptr();
  a.ldb = step(w);
  a.b_group = grouped ? step(w, -3) : 0;
  a.c = y.mutable_data_ptr();
  a.ldc = M;
  launch(a, x);
  return {y, z};
}

Tensor grad_input_of(const Tensor& dz_, const Tensor& w_, const optional<Tensor>& offsets) {
  not_traced();
  require(dz_, "dz");
  require(w_, "weight", dz_);
  const bool grouped = offsets.has_value();
  TORCH_CHECK_VALUE(dz_.dim() == 2 && w_.dim() == (grouped ? 3 : 2) &&
                        w_.size(-2) == dz_.size(1),
                    "dz ", dz_.sizes(), " does not fit weight ", w_.sizes());
  const int64_t N = dz_.size(0), M = dz_.size(1), K = w_.size(-1);
  fits(N, "rows");
  fits(K, "inputs");
  fits(M, "outputs");
  fedtrain_product_args a = {};
  a.dtype = dtype_of(dz_, "dz");
  a.form = FEDTRAIN_GRAD_INPUT;
  if (grouped) groups_of(w_.size(0), *offsets, dz_.device(), &a);
  const Tensor dz = rows(dz_), w = rows(w_);
  Tensor dx = make({N, K}, dz);
  a.m = N;
  a.n = K;
  a.k = M;
  a.a = dz.const_data_ptr();
  a.lda = step(dz);
  a.b = w.const_data_ptr();
  a.ldb = step(w);
  a.b_group = grouped ? step(w, -3) : 0;
  a.c = dx.mutable_data_ptr();
  a.ldc = K;
  launch(a, dz);
  return dx;
}

std::tuple<Tensor, Tensor> grad_weight_of(const Tensor& dz_, const Tensor& x_,
                                          const optional<Tensor>& offsets, bool want_weight,
                                          bool want_bias) {
  not_traced();
  require(x_, "x");
  require(dz_, "dz", x_);
  TORCH_CHECK_VALUE(dz_.dim() == 2 && x_.dim() == 2 && dz_.size(0) == x_.size(0), "dz ",
                    dz_.sizes(), " and x ", x_.sizes(), " do not fit");
  const int64_t N = dz_.size(0), M = dz_.size(1), K = x_.size(1);
  fits(N, "rows");
  fits(K, "inputs");
  fits(M, "outputs");
  fedtrain_product_args a = {};
  a.dtype = dtype_of(x_, "x");
  a.form = FEDTRAIN_GRAD_WEIGHT;
  const int64_t G = offsets ? groups_of(-1, *offsets, x_.device(), &a) : 0;
  Tensor dw, db;
  if (want_weight) dw = G ? make({G, M, K}, x_) : make({M, K}, x_);
  if (want_bias) db = G ? make({G, M}, x_) : make({M}, x_);
  if (!want_weight && !want_bias) return {dw, db};
  const Tensor dz = rows(dz_), x = rows(x_);
  a.m = M;
  a.n = want_weight ? K : 0;
  a.k = N;
  a.a = dz.const_data_ptr();
  a.lda = step(dz);
  a.b = x.const_data_ptr();
  a.ldb = step(x);
  if (want_weight) {
    a.c = dw.mutable_data_ptr();
    a.ldc = K;
    a.c_group = M * K;
  }
  if (want_bias) {
    a.colsum = db.mutable_data_ptr();
    a.colsum_group = M;
  }
  launch(a, x);
  return {dw, db};
}

Tensor act_backward_of(const Tensor& dy_, const Tensor& z_, int act) {
  not_traced();
  require(dy_, "dy");
  require(z_, "z", dy_);
  TORCH_CHECK_VALUE(dy_.dim() == 2 && dy_.sizes() == z_.sizes(), "dy ", dy_.sizes(), " and z ",
                    z_.sizes(), " must be one [N, out]");
  fits(dy_.size(0), "rows");
  fits(dy_.size(1), "outputs");
  const Tensor dy = rows(dy_), z = rows(z_);
  Tensor dz = make(dy.sizes(), dy);
  const On at(dy.device());
  check(fedtrain_act_backward(dtype_of(dy, "dy"), act, dy.size(0), dy.size(1),
                              dy.const_data_ptr(), step(dy), z.const_data_ptr(), step(z),
                              dz.mutable_data_ptr(), dz.size(1), at.stream),
        "fedtrain_act_backward");
  return dz;
}

// (dz, db) of a 16-bit dy: db from the terms before they are rounded.
std::tuple<Tensor, Tensor> act_backward_sums_of(const Tensor& dy_, const Tensor& z_, int act,
                                                const optional<Tensor>& offsets) {
  not_traced();
  require(dy_, "dy");
  require(z_, "z", dy_);
  TORCH_CHECK_VALUE(dy_.dim() == 2 && dy_.sizes() == z_.sizes(), "dy ", dy_.sizes(), " and z ",
                    z_.sizes(), " must be one [N, out]");
  fits(dy_.size(0), "rows");
  fits(dy_.size(1), "outputs");
  const Tensor dy = rows(dy_), z = rows(z_);
  fedtrain_act_args a = {};
  a.dtype = dtype_of(dy, "dy");
  a.act = act;
  if (offsets) groups_of(-1, *offsets, dy.device(), &a);
  const int64_t M = dy.size(1);
  Tensor dz = make(dy.sizes(), dy);
  Tensor db = offsets ? make({a.groups, M}, dy) : make({M}, dy);
  a.rows = dy.size(0);
  a.cols = M;
  a.dy = dy.const_data_ptr();
  a.lddy = step(dy);
  a.z = z.const_data_ptr();
  a.ldz = step(z);
  a.dz = dz.mutable_data_ptr();
  a.lddz = M;
  a.colsum = db.mutable_data_ptr();
  a.colsum_group = M;
  const On at(dy.device());
  Tensor work;
  const int64_t need = fedtrain_act_backward_sums_workspace(&a);
  TORCH_CHECK(need >= 0, "fedtrain_act_backward_sums_workspace failed (", need,
              "): ", fedtrain_strerror(static_cast<int>(need)));
  if (need > 0) {
    work = at::empty({need}, dy.options().dtype(at::kByte).requires_grad(false));
    a.workspace = work.mutable_data_ptr();
    a.workspace_bytes = need;
  }
  check(fedtrain_act_backward_sums(&a, at.stream), "fedtrain_act_backward_sums");
  return {dz, db};
}

// ---------------------------------------------------------------------------
// the differentiable product
// ---------------------------------------------------------------------------
optional<Tensor> given(const Tensor& t) {
  return t.defined() ? optional<Tensor>(t) : optional<Tensor>();
}

bool wants(const optional<Tensor>& t) { return t && t->requires_grad(); }

struct Product : torch::autograd::Function<Product> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const optional<Tensor>& b, const optional<Tensor>& r,
                        const optional<Tensor>& offsets, int64_t act) {
    const bool nx = x.requires_grad(), nw = w.requires_grad();
    const bool inner = nx || nw || wants(b);
    // relu's gradient can be told from its output; the others need z
    const bool keep_z = inner && act != FEDTRAIN_ACT_NONE && (act != FEDTRAIN_ACT_RELU || r);
    auto [y, z] = forward_of(x, w, b, r, static_cast<int>(act), offsets, keep_z);
    Tensor kept;
    if (inner && act != FEDTRAIN_ACT_NONE) kept = keep_z ? z : y;
    ctx->save_for_backward({nw ? x : Tensor(), nx ? w : Tensor(),
                            offsets ? *offsets : Tensor(), kept});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["residual"] = r.has_value();
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const Tensor dy = grads[0];
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &kept = saved[3];
    const optional<Tensor> offsets = given(saved[2]);
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    // numbered over the tensors that were given
    const bool has_b = ctx->saved_data["bias"].toBool();
    const bool has_r = ctx->saved_data["residual"].toBool();
    const bool nb = has_b && ctx->needs_input_grad(2);
    const bool nr = has_r && ctx->needs_input_grad(2 + has_b);
    Tensor dx, dw, db;
    const bool again = at::GradMode::is_enabled();
    {
      const at::NoGradGuard no_grad;
      if (dy.defined() && (nx || nw || nb)) {
        const int act = static_cast<int>(ctx->saved_data["act"].toInt());
        Tensor dz = dy;
        if (kept.defined()) {
          if (nb && dy.scalar_type() != at::kFloat)
            std::tie(dz, db) = act_backward_sums_of(dy, kept, act, offsets);
          else
            dz = act_backward_of(dy, kept, act);
        }
        if (nx) dx = grad_input_of(dz, w, offsets);
        const bool sum = nb && !db.defined();
        if (nw || sum) {
          auto [weight, bias] = grad_weight_of(dz, nw ? x : dz, offsets, nw, sum);
          dw = weight;
          if (sum) db = bias;
        }
      }
    }
    torch::autograd::variable_list out = {dx, dw, db, nr ? dy : Tensor(), Tensor(), Tensor()};
    if (again) {
      // asked for with create_graph: a second derivative raises when it is taken
      torch::autograd::variable_list first(out.begin(), out.begin() + 3);
      for (auto& t : first)
        if (t.defined()) t.requires_grad_(true);
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "linear_act and grouped_linear can be differentiated once", 3);
      first = (*error)(std::move(first));
      for (int i = 0; i < 3; ++i) out[i] = first[i];
    }
    return out;
  }
};

Tensor product(const Tensor& x, const Tensor& w, const optional<Tensor>& b,
               const optional<Tensor>& r, const optional<Tensor>& offsets, int act) {
  auto dual = [](const Tensor& t) { return t._fw_grad(0).defined(); };
  TORCH_CHECK_NOT_IMPLEMENTED(!dual(x) && !dual(w) && !(b && dual(*b)) && !(r && dual(*r)),
                              "linear_act and grouped_linear have no forward-mode derivative");
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || w.requires_grad() || wants(b) || wants(r)))
    return Product::apply(x, w, b, r, offsets, act);
  return std::get<0>(forward_of(x, w, b, r, act, offsets, false));
}

Tensor linear_act(const Tensor& x, const Tensor& w, const optional<Tensor>& b,
                  const optional<Tensor>& r, const std::string& activation) {
  not_traced();
  const int act = activation_of(activation);
  require(x, "x");
  require(w, "weight", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1), "x ", x.sizes(),
                    " and weight ", w.sizes(), " do not fit [..., in] and [out, in]");
  if (x.dim() == 2) return product(x, w, b, r, {}, act);
  std::vector<int64_t> out(x.sizes().begin(), x.sizes().end() - 1);
  int64_t n = 1;
  for (int64_t d : out) n *= d;
  out.push_back(w.size(0));
  optional<Tensor> r2;
  if (r) {
    require(*r, "residual", x);
    TORCH_CHECK_VALUE(r->sizes() == at::IntArrayRef(out), "residual must have shape ",
                      at::IntArrayRef(out), ", got ", r->sizes());
    r2 = r->reshape({n, w.size(0)});
  }
  return product(x.reshape({n, x.size(-1)}), w, b, r2, {}, act).view(out);
}

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& offsets,
                      const optional<Tensor>& b, const optional<Tensor>& r,
                      const std::string& activation) {
  return product(x, w, b, r, offsets, activation_of(activation));
}

// ---------------------------------------------------------------------------
// the AdamW step
// ---------------------------------------------------------------------------
using Tensors = std::vector<Tensor>;

void same(const Tensors& ts, const char* name, at::ScalarType type, const at::Device& d,
          const std::vector<int64_t>& sizes) {
  TORCH_CHECK_VALUE(ts.size() == sizes.size(), name, ": ", ts.size(), " tensors for ",
                    sizes.size(), " parameters");
  for (size_t i = 0; i < ts.size(); ++i) {
    const Tensor& t = ts[i];
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == d && t.numel() == sizes[i] &&
                          t.is_contiguous() && !t.is_neg(),
                      name, "[", i, "] must be a contiguous ", type, " tensor of ", sizes[i],
                      " elements on ", d, ", got ", t.scalar_type(), " ", t.sizes(), " on ",
                      t.device());
  }
}

struct Listed {
  const Tensors& tensors;
  const char* name;
  bool written;
};

// What is written shares memory with nothing else: two workgroups would write the
// same elements, or one read what another has already changed.
void apart(std::initializer_list<Listed> lists) {
  struct Range {
    uintptr_t begin, end;
    const Listed* of;
  };
  std::vector<Range> at;
  at.reserve(lists.size() * lists.begin()->tensors.size());
  for (const Listed& list : lists)
    for (const Tensor& t : list.tensors) {
      const auto p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
      if (t.numel()) at.push_back({p, p + t.nbytes(), &list});
    }
  std::sort(at.begin(), at.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  // the ranges that reach furthest so far: of those written, and of the others
  const Range none = {0, 0, nullptr};
  Range written = none, read = none;
  for (const Range& r : at) {
    for (const Range* other : {&written, &read})
      TORCH_CHECK_VALUE(r.begin >= other->end || !(r.of->written || other->of->written),
                        other->of->name, " and ", r.of->name,
                        " share memory: a tensor is given once");
    Range& far = r.of->written ? written : read;
    if (r.end > far.end) far = r;
  }
}

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& ms,
                const Tensors& vs, const optional<Tensors>& m_scales,
                const optional<Tensors>& v_scales, int64_t step,
                const optional<Tensor>& device_step, const optional<Tensors>& device_steps,
                double lr, double b1, double b2, double eps,
                double weight_decay, bool maximize, int64_t seed,
                const optional<std::vector<int64_t>>& first_blocks) {
  not_traced();
  TORCH_CHECK_VALUE(lr >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0 &&
                        weight_decay >= 0,
                    "lr ", lr, ", betas (", b1, ", ", b2, "), eps ", eps, ", weight_decay ",
                    weight_decay, ": betas lie in [0, 1), the others are not negative");
  if (params.empty()) return;
  const int dtype = dtype_of(params[0], "params[0]");
  require(params[0], "params[0]");
  const at::Device d = params[0].device();
  const size_t n = params.size();
  std::vector<int64_t> sizes(n), blocks(n);
  for (size_t i = 0; i < n; ++i) {
    sizes[i] = params[i].numel();
    blocks[i] = (sizes[i] + kStateBlock - 1) / kStateBlock;
  }
  const bool eight = m_scales.has_value();
  TORCH_CHECK_VALUE(eight == v_scales.has_value(),
                    "exp_avg_scales and exp_avg_sq_scales are given together");
  same(params, "params", params[0].scalar_type(), d, sizes);
  same(grads, "grads", params[0].scalar_type(), d, sizes);
  same(ms, "exp_avgs", eight ? at::kFloat8_e4m3fn : at::kFloat, d, sizes);
  same(vs, "exp_avg_sqs", eight ? at::kFloat8_e5m2 : at::kFloat, d, sizes);
  if (eight) {
    same(*m_scales, "exp_avg_scales", at::kFloat, d, blocks);
    same(*v_scales, "exp_avg_sq_scales", at::kFloat, d, blocks);
  }
  const Tensors no_scales;
  apart({{params, "params", true},
         {grads, "grads", false},
         {ms, "exp_avgs", true},
         {vs, "exp_avg_sqs", true},
         {eight ? *m_scales : no_scales, "exp_avg_scales", true},
         {eight ? *v_scales : no_scales, "exp_avg_sq_scales", true}});
  TORCH_CHECK_VALUE(!first_blocks || first_blocks->size() == n, "first_blocks: one for each of ",
                    n, " parameters");
  std::vector<fedtrain_adamw_tensor> table(n);
  int64_t block = 0;
  for (size_t i = 0; i < n; ++i) {
    fedtrain_adamw_tensor& t = table[i];
    t.p = params[i].mutable_data_ptr();
    t.g = grads[i].const_data_ptr();
    t.m = ms[i].mutable_data_ptr();
    t.v = vs[i].mutable_data_ptr();
    t.m_scale = eight ? static_cast<float*>((*m_scales)[i].mutable_data_ptr()) : nullptr;
    t.v_scale = eight ? static_cast<float*>((*v_scales)[i].mutable_data_ptr()) : nullptr;
    t.n = sizes[i];
    t.block0 = first_blocks ? (*first_blocks)[i] : block;
    block += blocks[i];
  }
  fedtrain_adamw_scalars s = {};
  s.lr = lr;
  s.beta1 = b1;
  s.beta2 = b2;
  s.eps = eps;
  s.weight_decay = weight_decay;
  s.seed = static_cast<uint32_t>(seed);
  s.maximize = maximize;
  const On at(d);
  Tensor work;
  std::vector<const int64_t*> counts;
  auto count_of = [&](const Tensor& t) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kLong && t.device() == d && t.numel() == 1,
                      "a step on the device must be one int64 on ", d);
    return static_cast<const int64_t*>(t.const_data_ptr());
  };
  auto scratch = [&](size_t tensors) {
    work = at::empty({static_cast<int64_t>(4 * tensors)},
                     at::TensorOptions().dtype(at::kFloat).device(d));
    s.workspace = work.mutable_data_ptr();
  };
  if (device_steps) {
    TORCH_CHECK_VALUE(device_steps->size() == n, "steps: ", device_steps->size(),
                      " counts for ", n, " parameters");
    for (const Tensor& t : *device_steps) counts.push_back(count_of(t));
    s.device_steps = counts.data();
    scratch(n);
  } else if (device_step) {
    s.device_step = count_of(*device_step);
    scratch(1);
  } else {
    TORCH_CHECK_VALUE(step >= 1, "steps are counted from 1, got ", step);
    s.step = step;
  }
  check(fedtrain_adamw(dtype, eight ? 8 : 32, static_cast<int64_t>(n), table.data(), &s,
                       at.stream),
        "fedtrain_adamw");
  // autograd sees that they changed
  for (const Tensors* ts : {&params, &ms, &vs})
    for (const Tensor& t : *ts)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("linear_act", &linear_act);
  m.def("grouped_linear", &grouped_linear);
  m.def("product_forward", [](const Tensor& x, const Tensor& w, const optional<Tensor>& b,
                              const optional<Tensor>& r, const std::string& act,
                              const optional<Tensor>& offsets, bool want_z) {
    auto [y, z] = forward_of(x, w, b, r, activation_of(act), offsets, want_z);
    return std::make_tuple(y, given(z));
  });
  m.def("product_grad_input", &grad_input_of);
  m.def("product_grad_weight", [](const Tensor& dz, const Tensor& x,
                                  const optional<Tensor>& offsets, bool want_weight,
                                  bool want_bias) {
    auto [dw, db] = grad_weight_of(dz, x, offsets, want_weight, want_bias);
    return std::make_tuple(given(dw), given(db));
  });
  m.def("act_backward", [](const Tensor& dy, const Tensor& z, const std::string& act) {
    return act_backward_of(dy, z, activation_of(act));
  });
  m.def("adamw_step", &adamw_step);
  m.def("abi_version", &fedtrain_abi_version);
}
