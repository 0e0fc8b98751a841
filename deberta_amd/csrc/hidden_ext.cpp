// hidden_ext.cpp — the operators on hidden states for PyTorch tensors: the
// argument checks, the results' memory, the calls of libdsa.so's entry points
// (include/dsa_block.h) on the current stream, and their autograd nodes.
//
// It is host code of its own because a call's host time is what bounds these
// operators on all but large batches.  A forward and backward of 256 x 128
// values takes 10 us on the GPU; through a ctypes call inside a Python
// autograd function it took 114 us of host time, through these nodes 58 (the
// engine's own hand-over between threads is 35 of them), and a forward that
// autograd does not record 4.6 instead of 11.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/dsa.h"
#include "../../include/dsa_block.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

constexpr int64_t kMaxRmsWidth = 16384;

bool has(const Maybe& t) { return t.has_value() && t->defined(); }

int type_of(const Tensor& t, const char* what, const char* name) {
  const ScalarType s = t.scalar_type();
  TORCH_CHECK_TYPE(s == at::kFloat || s == at::kBFloat16, what, " ", name, ": dtype must be float32 or bfloat16, got ", s);
  return s == at::kBFloat16 ? DSA_BF16 : DSA_F32;
}

void check_device(const char* what, const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " is on ", t.device(), ", x is on ", x.device());
}

// t with its values in memory as they count.  A tensor may have elements and no
// memory behind them (a wrapper subclass, a parameter whose storage was freed);
// its null pointer would read as "not given" further down.  And its sign may be
// pending: the imaginary part of a conjugated tensor is a view of the values
// before their negation, which is made here.
Tensor held(const char* what, const char* name, const Tensor& t) {
  if (t.numel() == 0) return t;
  const size_t need = t.is_contiguous()
                          ? (size_t)(t.storage_offset() + t.numel()) * t.element_size()
                          : at::detail::computeStorageNbytes(t.sizes(), t.strides(), t.element_size(), t.storage_offset());
  const c10::Storage& s = t.storage();
  TORCH_CHECK_VALUE(s.data() != nullptr && s.nbytes() >= need, what, ": ", name,
                    " has elements but no memory for them (a wrapper tensor, or its storage was freed)");
  return t.is_neg() ? t.resolve_neg() : t;
}

// x's width, x on the GPU
int64_t width_of(const char* what, const Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda(), what, ": x must be on the GPU, it is on ", x.device());
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, what, ": x needs a last dimension of at least one column, got shape ",
                    x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) <= INT32_MAX, what, ": rows of at most 2^31 - 1 columns, got ", x.size(-1));
  return x.size(-1);
}

// A parameter vector of C values, contiguous.
Tensor vector_of(const char* what, const char* name, const Tensor& t, int64_t C, const Tensor& x) {
  check_device(what, name, t, x);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == C, what, " ", name, " must have shape (", C, ",), got ", t.sizes());
  return held(what, name, t).contiguous();
}

// A tensor as rows of its last dimension with unit stride (a copy only where
// the leading dimensions have no one stride).
struct Rows {
  Tensor t;
  int64_t stride;
  Rows(const char* what, const char* name, const Tensor& given) {
    const int64_t C = given.size(-1);
    const Tensor v = held(what, name, given);
    t = v.is_contiguous() || v.dim() == 2 ? v : v.reshape({-1, C});
    if (t.stride(-1) != 1 && C > 1) t = t.contiguous();
    stride = t.is_contiguous() ? C : t.stride(0);
  }
};

// A residual of x's shape; one that is broadcast along the second of three
// dimensions is read in place.
struct Residual {
  Tensor t;
  int64_t strides[2] = {0, 0}, per_group = 1;
  Residual(const char* what, const Tensor& given, const Tensor& x) {
    check_device(what, "res", given, x);
    TORCH_CHECK_VALUE(given.sizes() == x.sizes(), what, ": res must have x's shape ", x.sizes(), ", got ", given.sizes());
    const Tensor res = held(what, "res", given);
    if (res.dim() == 3 && !res.is_contiguous() && (res.stride(2) == 1 || res.size(2) == 1)) {
      t = res;
      strides[0] = res.stride(0), strides[1] = res.stride(1), per_group = res.size(1);
    } else {
      const Rows r(what, "res", res);
      t = r.t;
      strides[1] = r.stride, per_group = std::max<int64_t>(1, res.numel() / res.size(-1));
    }
  }
};

ScalarType stream_type(const Tensor& x, const Maybe& res) {
  return has(res) ? at::promote_types(x.scalar_type(), res->scalar_type()) : x.scalar_type();
}

Tensor empty(const Tensor& like, ScalarType t) { return at::empty(like.sizes(), like.options().dtype(t)); }
Tensor bytes(const Tensor& on, size_t n) { return at::empty({(int64_t)n}, on.options().dtype(at::kByte)); }

// Calls an entry point on the current stream of t's device.
template <typename A>
void launch(int (*entry)(const A*, void*), const char* name, const A& a, const Tensor& t) {
  const c10::DeviceGuard guard(t.device());
  const int rc = entry(&a, c10::hip::getCurrentHIPStream(t.get_device()).stream());
  TORCH_CHECK(rc == 0, name, " failed: ", dsa_last_error());
}

uint64_t seed_of(const char* what, const Maybe& seed, int64_t t) {
  TORCH_CHECK_VALUE(t >= 0 && t <= 65536, what, ": dropout threshold must be in [0, 65536], got ", t);
  if (t == 0) return 0;
  TORCH_CHECK_VALUE(has(seed) && seed->is_cpu() && seed->numel() == 1 && seed->scalar_type() == at::kLong, what,
                    ": dropout needs its seed, an int64 CPU tensor of one element");
  return (uint64_t)*held(what, "the seed", *seed).const_data_ptr<int64_t>();
}

// Whether autograd has to see the call (a node refuses forward-mode tangents).
bool needs_grad(std::initializer_list<const Tensor*> ts) {
  const bool backward = at::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t && t->defined() && ((backward && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}
const Tensor* at_or_null(const Maybe& t) { return has(t) ? &*t : nullptr; }

// Whether the call may be made here.  torch.jit.trace records the results that
// are allocated and not the launches, so a traced call is the registered op's; a
// subclass with a dispatch of its own may hold its values elsewhere, and has to
// see the op.
bool here(std::initializer_list<const Tensor*> ts) {
  if (torch::jit::tracer::isTracing()) return false;
  for (const Tensor* t : ts)
    if (t && t->defined() && t->key_set().has(c10::DispatchKey::Python)) return false;
  return true;
}

// The gradients of a backward whose own graph is asked for: they raise when
// that is walked.
variable_list once(variable_list g, bool graph) {
  if (!graph) return g;
  for (Tensor& t : g)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "the operators on hidden states are not twice differentiable", (int64_t)g.size());
  return (*error)(std::move(g));
}

// ---------------------------------------------------------------------------
// dropout

Tensor dropout_fwd(const Tensor& x, const Maybe& bias, const Maybe& res, int64_t t, const Maybe& seed) {
  const char* what = "hidden_dropout";
  const int64_t C = width_of(what, x);
  dsa_dropout_args a{};
  a.x_dtype = type_of(x, what, "x");
  a.seed = seed_of(what, seed, t), a.threshold = (uint32_t)t;
  a.N = x.numel() / C, a.C = (int32_t)C;
  Tensor b;
  std::optional<Residual> r;
  if (has(bias)) {
    b = vector_of(what, "bias", *bias, C, x);
    a.bias = b.const_data_ptr(), a.bias_dtype = type_of(b, what, "bias");
  }
  if (has(res)) {
    r.emplace(what, *res, x);
    a.res = r->t.const_data_ptr(), a.res_dtype = type_of(*res, what, "res");
    a.res_strides[0] = r->strides[0], a.res_strides[1] = r->strides[1], a.rows_per_group = r->per_group;
  }
  const Tensor y = empty(x, stream_type(x, res));
  if (a.N == 0) return y;
  const Rows xr(what, "x", x);
  a.x = xr.t.const_data_ptr(), a.x_stride = xr.stride;
  a.y = y.data_ptr(), a.y_stride = C, a.y_dtype = type_of(y, what, "y");
  launch(dsa_dropout_fwd, "dsa_dropout_fwd", a, x);
  return y;
}

// (dx in type x_t, dbias in type *bias_t, empty without)
std::tuple<Tensor, Tensor> dropout_bwd(const Tensor& dy, ScalarType x_t, std::optional<ScalarType> bias_t, int64_t t,
                                       const Maybe& seed) {
  const char* what = "hidden_dropout_bwd";
  const int64_t C = width_of(what, dy);
  dsa_dropout_args a{};
  a.dy_dtype = type_of(dy, what, "dy");
  a.seed = seed_of(what, seed, t), a.threshold = (uint32_t)t;
  a.N = dy.numel() / C, a.C = (int32_t)C;
  const Tensor dx = empty(dy, x_t);
  Tensor dbias = at::empty({bias_t ? C : 0}, dy.options().dtype(bias_t.value_or(x_t))), ws;
  a.dx = dx.data_ptr(), a.dx_stride = C, a.dx_dtype = type_of(dx, what, "dx");
  if (a.N == 0) return {dx, dbias.zero_()};
  const Rows dyr(what, "dy", dy);
  a.dy = dyr.t.const_data_ptr(), a.dy_stride = dyr.stride;
  if (bias_t) {
    a.dbias = dbias.data_ptr(), a.bias_dtype = type_of(dbias, what, "bias");
    if (const size_t n = dsa_block_workspace_bytes(DSA_BLOCK_DROPOUT, a.N, a.C)) {
      ws = bytes(dy, n);
      a.workspace = ws.data_ptr(), a.workspace_bytes = n;
    }
  }
  launch(dsa_dropout_bwd, "dsa_dropout_bwd", a, dy);
  return {dx, dbias};
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& bias, const Maybe& res, int64_t t, const Maybe& seed) {
    ctx->save_for_backward({has(seed) ? *seed : Tensor()});
    ctx->saved_data["t"] = t;
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["bias"] = has(bias) ? (int64_t)bias->scalar_type() : -1;
    ctx->saved_data["res"] = has(res) ? (int64_t)res->scalar_type() : -1;
    return dropout_fwd(x, bias, res, t, seed);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const Tensor& dy = grads[0];
    const Tensor seed = ctx->get_saved_variables()[0];
    const int64_t bias = ctx->saved_data["bias"].toInt(), res = ctx->saved_data["res"].toInt();
    // edges: x, then the bias and the residual that are there, then the seed
    size_t edge = 0;
    const bool for_x = ctx->needs_input_grad(edge++);
    const bool for_bias = bias >= 0 && ctx->needs_input_grad(edge++);
    const bool for_res = res >= 0 && ctx->needs_input_grad(edge++);
    Tensor dx, dbias, dres;
    if (for_x || for_bias) {
      std::tie(dx, dbias) = dropout_bwd(dy, (ScalarType)ctx->saved_data["x"].toInt(),
                                        for_bias ? std::optional<ScalarType>((ScalarType)bias) : std::nullopt,
                                        ctx->saved_data["t"].toInt(), seed.defined() ? Maybe(seed) : std::nullopt);
      if (!for_bias) dbias = Tensor();
    }
    if (for_res) dres = dy.to((ScalarType)res);
    return once({dx, dbias, dres, Tensor(), Tensor()}, graph);
  }
};

Maybe dropout(const Tensor& x, const Maybe& bias, const Maybe& res, int64_t t, const Maybe& seed) {
  if (!here({&x, at_or_null(bias), at_or_null(res), at_or_null(seed)})) return std::nullopt;
  if (!needs_grad({&x, at_or_null(bias), at_or_null(res)})) return dropout_fwd(x, bias, res, t, seed);
  return Dropout::apply(x, bias, res, t, seed);
}

// ---------------------------------------------------------------------------
// residual + RMS norm

// What every form shares, and the tensors that it points into.
struct Rms {
  dsa_rms_args a{};
  Tensor bias, weight;
  std::optional<Residual> res;
  std::optional<Rows> x;
  Rms(const char* what, const Tensor& xt, const Maybe& b, const Maybe& r, const Tensor& w, int64_t t, const Maybe& seed) {
    const int64_t C = width_of(what, xt);
    TORCH_CHECK_VALUE(C <= kMaxRmsWidth, what, ": rows of at most ", kMaxRmsWidth, " columns, got ", C);
    a.x_dtype = type_of(xt, what, "x");
    a.seed = seed_of(what, seed, t), a.threshold = (uint32_t)t;
    a.N = xt.numel() / C, a.C = (int32_t)C;
    weight = vector_of(what, "weight", w, C, xt);
    a.weight = weight.const_data_ptr(), a.weight_dtype = type_of(weight, what, "weight");
    if (has(b)) {
      bias = vector_of(what, "bias", *b, C, xt);
      a.bias = bias.const_data_ptr(), a.bias_dtype = type_of(bias, what, "bias");
    }
    if (has(r)) {
      res.emplace(what, *r, xt);
      a.res = res->t.const_data_ptr(), a.res_dtype = type_of(*r, what, "res");
      a.res_strides[0] = res->strides[0], a.res_strides[1] = res->strides[1], a.rows_per_group = res->per_group;
    }
    if (a.N) {
      x.emplace(what, "x", xt);
      a.x = x->t.const_data_ptr(), a.x_stride = x->stride;
    }
  }
};

// z is x itself
bool plain(const Maybe& bias, const Maybe& res, int64_t t) { return !has(bias) && !has(res) && t == 0; }

// (y, z, 1 / rms per row); z is undefined where it is x itself, the statistics
// where they are not asked for
std::tuple<Tensor, Tensor, Tensor> rms_run(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight, double eps,
                                           ScalarType out, int64_t t, const Maybe& seed, bool stats) {
  Rms m("add_rms_norm", x, bias, res, weight, t, seed);
  const Tensor y = empty(x, out);
  Tensor z, rstd;
  m.a.y = y.data_ptr(), m.a.y_stride = m.a.C, m.a.y_dtype = type_of(y, "add_rms_norm", "y"), m.a.eps = (float)eps;
  if (!plain(bias, res, t)) {
    z = empty(x, stream_type(x, res));
    m.a.z = z.data_ptr(), m.a.z_stride = m.a.C;
  }
  if (stats) {
    rstd = at::empty({m.a.N}, x.options().dtype(at::kFloat));
    m.a.rstd = rstd.data_ptr<float>();
  }
  if (m.a.N) launch(dsa_add_rms_fwd, "dsa_add_rms_fwd", m.a, x);
  return {y, z, rstd};
}

// the same for the registered op: z empty where it is x itself
std::tuple<Tensor, Tensor, Tensor> rms_fwd(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight, double eps,
                                           ScalarType out, int64_t t, const Maybe& seed) {
  auto [y, z, rstd] = rms_run(x, bias, res, weight, eps, out, t, seed, true);
  if (!z.defined()) z = at::empty({0}, x.options());
  return {y, z, rstd};
}

// (dx, dres, dweight, dbias).  dres is empty without a residual and where it
// equals dx (no dropout, one type); dbias is empty without a bias.
std::tuple<Tensor, Tensor, Tensor, Tensor> rms_bwd(const Tensor& dy, const Maybe& dz, const Tensor& x, const Maybe& bias,
                                                   const Maybe& res, const Tensor& weight, const Tensor& rstd, int64_t t,
                                                   const Maybe& seed) {
  const char* what = "add_rms_norm_bwd";
  Rms m(what, x, bias, res, weight, t, seed);
  check_device(what, "dy", dy, x);
  check_device(what, "rstd", rstd, x);
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), what, ": dy must have x's shape ", x.sizes(), ", got ", dy.sizes());
  TORCH_CHECK_VALUE(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == m.a.N, what, ": bad rstd");
  const Tensor stats = held(what, "rstd", rstd);
  const Tensor dx = empty(x, x.scalar_type());
  const bool apart = has(res) && (t != 0 || res->scalar_type() != x.scalar_type());
  const Tensor dres = apart ? empty(x, res->scalar_type()) : at::empty({0}, x.options());
  Tensor dweight = at::empty_like(m.weight);
  Tensor dbias = has(bias) ? at::empty_like(m.bias) : at::empty({0}, weight.options());
  if (m.a.N == 0) return {dx, dres, dweight.zero_(), dbias.zero_()};
  const Rows dyr(what, "dy", dy);
  std::optional<Rows> dzr;
  m.a.dy = dyr.t.const_data_ptr(), m.a.dy_stride = dyr.stride, m.a.dy_dtype = type_of(dy, what, "dy");
  m.a.rstd = stats.data_ptr<float>();
  if (has(dz)) {
    check_device(what, "dz", *dz, x);
    TORCH_CHECK_VALUE(dz->sizes() == x.sizes(), what, ": dz must have x's shape ", x.sizes(), ", got ", dz->sizes());
    dzr.emplace(what, "dz", dz->to(stream_type(x, res)));
    m.a.dzu = dzr->t.const_data_ptr(), m.a.dzu_stride = dzr->stride;
  }
  m.a.dx = dx.data_ptr(), m.a.dx_stride = m.a.C;
  if (apart) m.a.dres = dres.data_ptr(), m.a.dres_stride = m.a.C;
  m.a.dweight = dweight.data_ptr();
  if (has(bias)) m.a.dbias = dbias.data_ptr();
  const size_t n = dsa_block_workspace_bytes(DSA_BLOCK_RMS, m.a.N, m.a.C);
  const Tensor ws = bytes(x, n);
  m.a.workspace = ws.data_ptr(), m.a.workspace_bytes = n;
  launch(dsa_add_rms_bwd, "dsa_add_rms_bwd", m.a, x);
  return {dx, dres, dweight, dbias};
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight,
                               double eps, ScalarType out, int64_t t, const Maybe& seed) {
    auto [y, z, rstd] = rms_run(x, bias, res, weight, eps, out, t, seed, true);
    ctx->save_for_backward({x, has(bias) ? *bias : Tensor(), has(res) ? *res : Tensor(), weight, rstd, has(seed) ? *seed : Tensor()});
    ctx->saved_data["t"] = t;
    ctx->saved_data["out"] = (int64_t)out;
    ctx->set_materialize_grads(false);
    if (!z.defined()) return {y};
    return {y, z};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    Tensor dy = grads[0];
    const Tensor dz = grads.size() > 1 ? grads[1] : Tensor();
    variable_list g(8);
    if (!dy.defined() && !dz.defined()) return g;
    const variable_list v = ctx->get_saved_variables();
    const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; };
    const int64_t t = ctx->saved_data["t"].toInt();
    // where only z was used
    if (!dy.defined()) dy = at::zeros(v[0].sizes(), v[0].options().dtype((ScalarType)ctx->saved_data["out"].toInt()));
    auto [dx, dres, dweight, dbias] = rms_bwd(dy, maybe(dz), v[0], maybe(v[1]), maybe(v[2]), v[3], v[4], t, maybe(v[5]));
    g[0] = dx;
    if (v[1].defined()) g[1] = dbias;
    if (v[2].defined()) g[2] = t != 0 || v[2].scalar_type() != v[0].scalar_type() ? dres : dx;
    g[3] = dweight;
    return once(std::move(g), graph);
  }
};

// (y, z); z is x where there is nothing to add or drop
std::optional<std::tuple<Tensor, Tensor>> rms(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight, double eps,
                                              ScalarType out, int64_t t, const Maybe& seed) {
  if (!here({&x, at_or_null(bias), at_or_null(res), &weight, at_or_null(seed)})) return std::nullopt;
  if (!needs_grad({&x, at_or_null(bias), at_or_null(res), &weight})) {
    auto [y, z, rstd] = rms_run(x, bias, res, weight, eps, out, t, seed, false);
    return std::make_tuple(y, z.defined() ? z : x);
  }
  const variable_list o = AddRmsNorm::apply(x, bias, res, weight, eps, out, t, seed);
  return std::make_tuple(o[0], o.size() > 1 ? o[1] : x);
}

// (y as float8_e4m3fn, its scales, z); z is undefined where it is x itself.
// group 0: one scale a row.
std::tuple<Tensor, Tensor, Tensor> quant_run(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight, double eps,
                                             int64_t group) {
  const char* what = "add_rms_norm_quant";
  Rms m(what, x, bias, res, weight, 0, std::nullopt);
  const int64_t C = m.a.C;
  TORCH_CHECK_VALUE(group == 0 || (group >= 32 && group <= 512 && (group & (group - 1)) == 0 && C % group == 0),
                    "group_size must be 32, 64, 128, 256 or 512 and divide the width ", C, ", got ", group);
  const Tensor q = empty(x, at::kFloat8_e4m3fn);
  auto shape = x.sizes().vec();
  shape.back() = group ? C / group : 1;
  const Tensor scales = at::empty(shape, x.options().dtype(at::kFloat));
  Tensor z;
  m.a.y = q.data_ptr(), m.a.y_stride = C, m.a.scales = scales.data_ptr<float>(), m.a.group_size = (int32_t)group;
  m.a.eps = (float)eps;
  if (!plain(bias, res, 0)) {
    z = empty(x, stream_type(x, res));
    m.a.z = z.data_ptr(), m.a.z_stride = C;
  }
  if (m.a.N) launch(dsa_add_rms_quant, "dsa_add_rms_quant", m.a, x);
  return {q, scales, z};
}

std::tuple<Tensor, Tensor, Tensor> quant_fwd(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight, double eps,
                                             int64_t group) {
  auto [q, scales, z] = quant_run(x, bias, res, weight, eps, group);
  if (!z.defined()) z = at::empty({0}, x.options());
  return {q, scales, z};
}

std::optional<std::tuple<Tensor, Tensor, Tensor>> quant(const Tensor& x, const Maybe& bias, const Maybe& res, const Tensor& weight,
                                                        double eps, int64_t group) {
  if (!here({&x, at_or_null(bias), at_or_null(res), &weight})) return std::nullopt;
  auto [q, scales, z] = quant_run(x, bias, res, weight, eps, group);
  return std::make_tuple(q, scales, z.defined() ? z : x);
}

// ---------------------------------------------------------------------------
// embedding

Tensor ids_of(const char* what, const Tensor& ids, const Tensor& x) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "embed: ids must be int64 or int32, got ",
                   ids.scalar_type());
  TORCH_CHECK_VALUE(ids.device() == x.device(), what, ": ids are on ", ids.device(), ", the weight or its gradient on ", x.device());
  return held(what, "ids", ids).contiguous();
}

Tensor embed_fwd(const Tensor& ids, const Tensor& weight, int64_t padding, double scale, ScalarType out) {
  const char* what = "embed";
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) > 0, what, ": weight must be (V, C) with V >= 1, got shape ", weight.sizes());
  const int64_t C = width_of(what, weight);
  const Tensor idr = ids_of(what, ids, weight);
  const Rows w(what, "weight", weight);
  auto shape = ids.sizes().vec();
  shape.push_back(C);
  const Tensor y = at::empty(shape, weight.options().dtype(out));
  dsa_embed_args a{};
  a.ids = idr.const_data_ptr(), a.ids_bytes = (int32_t)idr.element_size();
  a.weight = w.t.const_data_ptr(), a.weight_stride = w.stride, a.weight_dtype = type_of(weight, what, "weight");
  a.y = y.data_ptr(), a.y_stride = C, a.y_dtype = type_of(y, what, "y");
  a.N = ids.numel(), a.V = weight.size(0), a.C = (int32_t)C, a.padding = padding, a.scale = (float)scale;
  if (a.N) launch(dsa_embed_fwd, "dsa_embed_fwd", a, weight);
  return y;
}

// the gradient of the whole table
Tensor embed_bwd(const Tensor& dy, const Tensor& ids, int64_t V, ScalarType weight_t, int64_t padding, double scale) {
  const char* what = "embed_bwd";
  const int64_t C = width_of(what, dy);
  TORCH_CHECK_VALUE(V > 0, what, ": the table needs at least one row, got ", V);
  TORCH_CHECK_VALUE(dy.dim() == ids.dim() + 1 && dy.sizes().slice(0, ids.dim()) == ids.sizes(), what, ": dy must have ids' shape ",
                    ids.sizes(), " and columns, got ", dy.sizes());
  const Tensor idr = ids_of(what, ids, dy);
  Tensor dw = at::empty({V, C}, dy.options().dtype(weight_t));
  dsa_embed_args a{};
  a.dweight = dw.data_ptr(), a.weight_dtype = type_of(dw, what, "weight");
  a.dy_dtype = type_of(dy, what, "dy");
  a.N = ids.numel(), a.V = V, a.C = (int32_t)C, a.padding = padding, a.scale = (float)scale;
  if (a.N == 0) return dw.zero_();
  const Rows dyr(what, "dy", dy);
  a.ids = idr.const_data_ptr(), a.ids_bytes = (int32_t)idr.element_size();
  a.dy = dyr.t.const_data_ptr(), a.dy_stride = dyr.stride;
  const size_t n = dsa_embed_workspace_bytes(a.N, a.C, V);
  const Tensor ws = bytes(dy, n);
  a.workspace = ws.data_ptr(), a.workspace_bytes = n;
  launch(dsa_embed_bwd, "dsa_embed_bwd", a, dy);
  return dw;
}

struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, int64_t padding, double scale, ScalarType out) {
    ctx->save_for_backward({ids});
    ctx->saved_data["V"] = weight.size(0);
    ctx->saved_data["weight"] = (int64_t)weight.scalar_type();
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["scale"] = scale;
    return embed_fwd(ids, weight, padding, scale, out);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const Tensor dw = embed_bwd(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["V"].toInt(),
                                (ScalarType)ctx->saved_data["weight"].toInt(), ctx->saved_data["padding"].toInt(),
                                ctx->saved_data["scale"].toDouble());
    return once({Tensor(), dw, Tensor(), Tensor(), Tensor()}, graph);
  }
};

Maybe embed(const Tensor& ids, const Tensor& weight, int64_t padding, double scale, ScalarType out) {
  if (!here({&ids, &weight})) return std::nullopt;
  if (!needs_grad({&weight})) return embed_fwd(ids, weight, padding, scale, out);
  return Embed::apply(ids, weight, padding, scale, out);
}

}  // namespace

// The functions named like an operator record autograd, and give None for a call
// that the registered op has to see; _fwd and _bwd are what the ops call.
PYBIND11_MODULE(_hidden_ext, m) {
  m.attr("abi_version") = DSA_VERSION;      // whose structs it passes
  m.attr("torch_version") = TORCH_VERSION;  // whose classes it was compiled with
  m.def("dropout", torch::wrap_pybind_function_no_gil(dropout));
  m.def("dropout_fwd", torch::wrap_pybind_function_no_gil(dropout_fwd));
  m.def("dropout_bwd", torch::wrap_pybind_function_no_gil(dropout_bwd));
  m.def("rms", torch::wrap_pybind_function_no_gil(rms));
  m.def("rms_fwd", torch::wrap_pybind_function_no_gil(rms_fwd));
  m.def("rms_bwd", torch::wrap_pybind_function_no_gil(rms_bwd));
  m.def("quant", torch::wrap_pybind_function_no_gil(quant));
  m.def("quant_fwd", torch::wrap_pybind_function_no_gil(quant_fwd));
  m.def("embed", torch::wrap_pybind_function_no_gil(embed));
  m.def("embed_fwd", torch::wrap_pybind_function_no_gil(embed_fwd));
  m.def("embed_bwd", torch::wrap_pybind_function_no_gil(embed_bwd));
}
