// vocab_ext.h — the operators on a vocabulary's logits for PyTorch tensors: the
// part of hidden_ext.cpp's extension over include/dsa_vocab.h, with its helpers
// (included there, in its namespace).
#pragma once

// Logits of (..., V) as rows.
struct Logits {
  Rows rows;
  int64_t N, V;
  int dt;
  Logits(const char* what, const Tensor& t) : rows((check(what, t), what), "logits", t), N(t.numel() / t.size(-1)), V(t.size(-1)), dt(type_of(t, what, "logits")) {}
  static void check(const char* what, const Tensor& t) {
    TORCH_CHECK_VALUE(t.is_cuda(), what, ": logits must be on the GPU, they are on ", t.device());
    TORCH_CHECK_VALUE(t.dim() > 0 && t.size(-1) > 0, what, ": logits need a last dimension of at least one column, got shape ", t.sizes());
    TORCH_CHECK_VALUE(t.size(-1) <= INT32_MAX - 127, what, ": rows of at most 2^31 - 128 columns, got ", t.size(-1));
  }
};

c10::IntArrayRef row_shape(const Tensor& logits) { return logits.sizes().slice(0, logits.dim() - 1); }
// Results, allocated without the dispatcher's two calls for at::empty (a call on one
// row makes five of them).
Tensor fresh(const Tensor& on, c10::IntArrayRef shape, ScalarType t) { return at::detail::empty_cuda(shape, t, on.device(), std::nullopt); }
Tensor floats(const Tensor& on, c10::IntArrayRef shape) { return fresh(on, shape, at::kFloat); }
Tensor with_columns(const Tensor& logits, int64_t k, ScalarType t) {
  auto shape = row_shape(logits).vec();
  shape.push_back(k);
  return fresh(logits, shape, t);
}
Tensor row_stats(const Tensor& logits, int64_t N) { return floats(logits, {N, 4}); }

void check_with(const char* what, const char* name, const Tensor& t, const Tensor& logits) {
  TORCH_CHECK_VALUE(t.device() == logits.device(), what, ": ", name, " are on ", t.device(), ", the logits on ", logits.device());
}

// Whole numbers of `shape`, contiguous.
Tensor whole(const char* what, const char* name, const Tensor& t, c10::IntArrayRef shape, const Tensor& logits) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, ": ", name, " must be int64 or int32, got ", t.scalar_type());
  check_with(what, name, t, logits);
  TORCH_CHECK_VALUE(t.sizes() == shape, what, ": ", name, " must have shape ", shape, ", got ", t.sizes());
  return held(what, name, t).contiguous();
}

// A gradient of one float32 a row: its values, or the one that all rows read
// (the gradient of a sum is a broadcast number; no copy of it is made).
struct PerRow {
  Tensor t;
  const float* data = nullptr;
  int64_t stride = 0;
  PerRow(const char* what, const char* name, const Tensor& g, const Tensor& logits) {
    if (!g.defined()) return;
    check_with(what, name, g, logits);
    TORCH_CHECK_VALUE(g.sizes() == row_shape(logits), what, ": ", name, " must have shape ", row_shape(logits), ", got ", g.sizes());
    TORCH_CHECK_TYPE(g.scalar_type() == at::kFloat, what, ": ", name, " must be float32, got ", g.scalar_type());
    t = held(what, name, g);
    bool one = true;
    for (int64_t i = 0; i < t.dim(); ++i) one = one && (t.stride(i) == 0 || t.size(i) == 1);
    if (!one) t = t.contiguous(), stride = 1;
    data = t.const_data_ptr<float>();
  }
};

Tensor stats_of(const char* what, const Tensor& stats, int64_t N, const Tensor& logits) {
  check_with(what, "stats", stats, logits);
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.dim() == 2 && stats.size(0) == N && stats.size(1) == 4, what,
                    ": bad stats");
  return held(what, "stats", stats);
}

template <typename A>
Tensor vocab_workspace(A& a, int32_t top, const Tensor& on) {
  const size_t n = dsa_vocab_workspace_bytes(a.N, a.V, a.dtype, top);
  if (n == 0) return Tensor();
  const Tensor ws = fresh(on, {(int64_t)n}, at::kByte);
  a.workspace = ws.data_ptr(), a.workspace_bytes = n;
  return ws;
}

// ---------------------------------------------------------------------------
// log probabilities

void check_scale(const char* what, double temperature) {
  TORCH_CHECK_VALUE(temperature >= 0x1p-100 && temperature <= 0x1p100, what, ": temperature must be positive and finite (2^-100 to 2^100), got ", temperature);
}

struct Logprobs {
  Tensor logprobs, entropy, lse, top_logprobs, top_ids, stats;
};

Logprobs logprobs_run(const Tensor& logits, const Maybe& ids, int64_t top_k, double temperature, int64_t ignore, bool stats) {
  const char* what = "token_logprobs";
  const Logits l(what, logits);
  check_scale(what, temperature);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= std::min<int64_t>(l.V, DSA_VOCAB_MAX_ENTRIES), what, ": top_k must be in [0, min(V, ",
                    (int)DSA_VOCAB_MAX_ENTRIES, ")], got ", top_k, " for ", l.V, " columns");
  TORCH_CHECK_VALUE(top_k == 0 || l.V <= DSA_VOCAB_MAX_TOP_V, what, ": top_k needs a vocabulary of at most ", (int)DSA_VOCAB_MAX_TOP_V, ", got ", l.V);
  dsa_logprobs_args a{};
  a.N = l.N, a.V = l.V, a.dtype = l.dt, a.top_k = (int32_t)top_k, a.inv_temperature = (float)(1.0 / temperature), a.ignore_index = ignore;
  Tensor idr;
  Logprobs o;
  const auto shape = row_shape(logits);
  if (has(ids)) {
    idr = whole(what, "ids", *ids, shape, logits);
    o.logprobs = floats(logits, shape);
    a.ids_bytes = (int32_t)idr.element_size();
  }
  o.entropy = floats(logits, shape), o.lse = floats(logits, shape);
  if (top_k) o.top_logprobs = with_columns(logits, top_k, at::kFloat), o.top_ids = with_columns(logits, top_k, at::kLong);
  if (stats) o.stats = row_stats(logits, l.N);
  if (l.N == 0) return o;
  a.logits = l.rows.t.const_data_ptr(), a.logits_stride = l.rows.stride;
  if (has(ids)) a.ids = idr.const_data_ptr(), a.logprobs = o.logprobs.data_ptr<float>();
  a.entropy = o.entropy.data_ptr<float>(), a.lse = o.lse.data_ptr<float>();
  if (top_k) a.top_logprobs = o.top_logprobs.data_ptr<float>(), a.top_ids = o.top_ids.data_ptr<int64_t>();
  if (stats) a.stats = o.stats.data_ptr<float>();
  const Tensor ws = vocab_workspace(a, a.top_k, logits);
  launch(dsa_logprobs_fwd, "dsa_logprobs_fwd", a, logits);
  return o;
}

// dlogits; each gradient may be undefined, not all of them
Tensor logprobs_grad(const Tensor& dlogprobs, const Tensor& dentropy, const Tensor& dlse, const Tensor& dtop, const Tensor& logits,
                     const Tensor& ids, const Tensor& top_ids, const Tensor& stats, double temperature, int64_t ignore) {
  const char* what = "token_logprobs_bwd";
  const Logits l(what, logits);
  check_scale(what, temperature);
  dsa_logprobs_args a{};
  a.N = l.N, a.V = l.V, a.dtype = l.dt, a.inv_temperature = (float)(1.0 / temperature), a.ignore_index = ignore;
  const Tensor dx = empty(logits, logits.scalar_type());
  const Tensor st = stats_of(what, stats, l.N, logits);
  a.stats = const_cast<float*>(st.const_data_ptr<float>());
  const PerRow gl(what, "dlogprobs", dlogprobs, logits), ge(what, "dentropy", dentropy, logits), gs(what, "dlse", dlse, logits);
  Tensor idr, tops, gt;
  if (ids.defined()) idr = whole(what, "ids", ids, row_shape(logits), logits), a.ids_bytes = (int32_t)idr.element_size();
  TORCH_CHECK_VALUE(!gl.t.defined() || ids.defined(), what, ": dlogprobs need ids");
  if (dtop.defined()) {
    TORCH_CHECK_VALUE(top_ids.defined() && top_ids.dim() == logits.dim() && top_ids.size(-1) <= std::min<int64_t>(l.V, DSA_VOCAB_MAX_ENTRIES), what, ": dtop needs top_ids");
    auto shape = row_shape(logits).vec();
    shape.push_back(top_ids.size(-1));
    tops = whole(what, "top_ids", held(what, "top_ids", top_ids).to(at::kLong), shape, logits);
    check_with(what, "dtop", dtop, logits);
    TORCH_CHECK_VALUE(dtop.sizes() == tops.sizes() && dtop.scalar_type() == at::kFloat, what, ": dtop must be float32 of shape ", tops.sizes());
    gt = held(what, "dtop", dtop).contiguous();
  }
  if (l.N == 0) return dx;
  a.logits = l.rows.t.const_data_ptr(), a.logits_stride = l.rows.stride;
  if (ids.defined()) a.ids = idr.const_data_ptr();
  a.dlogprobs = gl.data, a.dlogprobs_stride = gl.stride, a.dentropy = ge.data, a.dentropy_stride = ge.stride;
  a.dlse = gs.data, a.dlse_stride = gs.stride;
  if (dtop.defined()) a.top_k = (int32_t)tops.size(-1), a.top_ids = const_cast<int64_t*>(tops.const_data_ptr<int64_t>()), a.dtop = gt.const_data_ptr<float>();
  a.dlogits = dx.data_ptr(), a.dlogits_stride = l.V;
  launch(dsa_logprobs_bwd, "dsa_logprobs_bwd", a, logits);
  return dx;
}

const Tensor& or_undefined(const Maybe& t) {
  static const Tensor none;
  return has(t) ? *t : none;
}
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

// for the registered op: what is not there is empty
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> logprobs_fwd(const Tensor& logits, const Maybe& ids, int64_t top_k,
                                                                        double temperature, int64_t ignore) {
  Logprobs o = logprobs_run(logits, ids, top_k, temperature, ignore, true);
  if (!o.logprobs.defined()) o.logprobs = floats(logits, {0});
  if (!top_k) o.top_logprobs = with_columns(logits, 0, at::kFloat), o.top_ids = with_columns(logits, 0, at::kLong);
  return {o.logprobs, o.entropy, o.lse, o.top_logprobs, o.top_ids, o.stats};
}

Tensor logprobs_bwd(const Maybe& dlogprobs, const Maybe& dentropy, const Maybe& dlse, const Maybe& dtop, const Tensor& logits, const Maybe& ids,
                    const Maybe& top_ids, const Tensor& stats, double temperature, int64_t ignore) {
  TORCH_CHECK_VALUE(has(dlogprobs) || has(dentropy) || has(dlse) || has(dtop), "token_logprobs_bwd: a gradient is required");
  return logprobs_grad(or_undefined(dlogprobs), or_undefined(dentropy), or_undefined(dlse), or_undefined(dtop), logits, or_undefined(ids),
                       or_undefined(top_ids), stats, temperature, ignore);
}

constexpr const char* kOnLogits = "the operators on logits are not twice differentiable";

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  // entropy and lse, then the log probabilities with ids, then the largest and
  // their ids with top_k
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Maybe& ids, int64_t top_k, double temperature, int64_t ignore) {
    const Logprobs o = logprobs_run(logits, ids, top_k, temperature, ignore, true);
    ctx->save_for_backward({logits, has(ids) ? *ids : Tensor(), o.top_ids, o.stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    variable_list out{o.entropy, o.lse};
    if (has(ids)) out.push_back(o.logprobs);
    if (top_k) {
      out.push_back(o.top_logprobs), out.push_back(o.top_ids);
      ctx->mark_non_differentiable({o.top_ids});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const variable_list v = ctx->get_saved_variables();
    const bool ids = v[1].defined();
    const Tensor dlogprobs = ids ? grads[2] : Tensor(), dtop = v[2].defined() ? grads[ids ? 3 : 2] : Tensor();
    variable_list g(5);
    if (!grads[0].defined() && !grads[1].defined() && !dlogprobs.defined() && !dtop.defined()) return g;
    g[0] = logprobs_grad(dlogprobs, grads[0], grads[1], dtop, v[0], v[1], v[2], v[3], ctx->saved_data["temperature"].toDouble(),
                         ctx->saved_data["ignore"].toInt());
    return once(std::move(g), graph, kOnLogits);
  }
};

// (logprobs or None, entropy, lse, the largest or None, their ids or None)
typedef std::tuple<Maybe, Tensor, Tensor, Maybe, Maybe> LogprobsTuple;
std::optional<LogprobsTuple> logprobs(const Tensor& logits, const Maybe& ids, int64_t top_k, double temperature, int64_t ignore) {
  if (!here({&logits, at_or_null(ids)})) return std::nullopt;
  if (!needs_grad({&logits})) {
    const Logprobs o = logprobs_run(logits, ids, top_k, temperature, ignore, false);
    return LogprobsTuple(maybe(o.logprobs), o.entropy, o.lse, maybe(o.top_logprobs), maybe(o.top_ids));
  }
  const variable_list o = TokenLogprobs::apply(logits, ids, top_k, temperature, ignore);
  const size_t top = has(ids) ? 3 : 2;
  return LogprobsTuple(has(ids) ? Maybe(o[2]) : std::nullopt, o[0], o[1], top_k ? Maybe(o[top]) : std::nullopt,
                       top_k ? Maybe(o[top + 1]) : std::nullopt);
}

// ---------------------------------------------------------------------------
// distillation

// What both directions share, and the tensors that it points into.
struct Distill {
  dsa_distill_args a{};
  Logits l;
  Tensor ids, teacher, lse;
  Distill(const char* what, const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse, double temperature)
      : l(what, logits) {
    check_scale(what, temperature);
    TORCH_CHECK_VALUE(teacher_ids.dim() == logits.dim() && teacher_ids.size(-1) >= 1 && teacher_ids.size(-1) <= DSA_VOCAB_MAX_ENTRIES, what,
                      ": teacher_ids must be (..., K) with the logits' rows and K in [1, ", (int)DSA_VOCAB_MAX_ENTRIES, "], got shape ", teacher_ids.sizes());
    auto shape = row_shape(logits).vec();
    shape.push_back(teacher_ids.size(-1));
    ids = whole(what, "teacher_ids", teacher_ids, shape, logits);
    check_with(what, "teacher_logits", teacher_logits, logits);
    TORCH_CHECK_VALUE(teacher_logits.sizes() == c10::IntArrayRef(shape), what, ": teacher_logits must have teacher_ids' shape ", shape, ", got ", teacher_logits.sizes());
    a.teacher_dtype = type_of(teacher_logits, what, "teacher_logits");
    teacher = held(what, "teacher_logits", teacher_logits).contiguous();
    if (has(teacher_lse)) {
      check_with(what, "teacher_lse", *teacher_lse, logits);
      TORCH_CHECK_VALUE(teacher_lse->sizes() == row_shape(logits), what, ": teacher_lse must have shape ", row_shape(logits), ", got ", teacher_lse->sizes());
      TORCH_CHECK_TYPE(teacher_lse->scalar_type() == at::kFloat, what, ": teacher_lse must be float32, got ", teacher_lse->scalar_type());
      lse = held(what, "teacher_lse", *teacher_lse).contiguous();
      a.teacher_lse = lse.const_data_ptr<float>();
    }
    a.N = l.N, a.V = l.V, a.dtype = l.dt, a.K = (int32_t)shape.back(), a.ids_bytes = (int32_t)ids.element_size(), a.temperature = (float)temperature;
    a.teacher_ids = ids.const_data_ptr(), a.teacher = teacher.const_data_ptr();
    a.logits = l.rows.t.const_data_ptr(), a.logits_stride = l.rows.stride;
  }
};

std::tuple<Tensor, Tensor> distill_run(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse,
                                       double temperature, bool stats) {
  Distill d("distill_loss", logits, teacher_ids, teacher_logits, teacher_lse, temperature);
  const Tensor loss = floats(logits, row_shape(logits));
  Tensor st;
  if (stats) st = row_stats(logits, d.l.N);
  if (d.l.N == 0) return {loss, st};
  d.a.loss = loss.data_ptr<float>();
  if (stats) d.a.stats = st.data_ptr<float>();
  const Tensor ws = vocab_workspace(d.a, 0, logits);
  launch(dsa_distill_fwd, "dsa_distill_fwd", d.a, logits);
  return {loss, st};
}

std::tuple<Tensor, Tensor> distill_fwd(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse,
                                       double temperature) {
  return distill_run(logits, teacher_ids, teacher_logits, teacher_lse, temperature, true);
}

Tensor distill_bwd(const Tensor& dloss, const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse,
                   const Tensor& stats, double temperature) {
  const char* what = "distill_loss_bwd";
  Distill d(what, logits, teacher_ids, teacher_logits, teacher_lse, temperature);
  const PerRow g(what, "dloss", dloss, logits);
  const Tensor st = stats_of(what, stats, d.l.N, logits);
  d.a.stats = const_cast<float*>(st.const_data_ptr<float>());
  const Tensor dx = empty(logits, logits.scalar_type());
  if (d.l.N == 0) return dx;
  d.a.dloss = g.data, d.a.dloss_stride = g.stride;
  d.a.dlogits = dx.data_ptr(), d.a.dlogits_stride = d.l.V;
  launch(dsa_distill_bwd, "dsa_distill_bwd", d.a, logits);
  return dx;
}

struct DistillLoss : torch::autograd::Function<DistillLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse,
                        double temperature) {
    const auto [loss, stats] = distill_run(logits, teacher_ids, teacher_logits, teacher_lse, temperature, true);
    ctx->save_for_backward({logits, teacher_ids, teacher_logits, has(teacher_lse) ? *teacher_lse : Tensor(), stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const variable_list v = ctx->get_saved_variables();
    variable_list g(5);
    g[0] = distill_bwd(grads[0], v[0], v[1], v[2], maybe(v[3]), v[4], ctx->saved_data["temperature"].toDouble());
    return once(std::move(g), graph, kOnLogits);
  }
};

Maybe distill(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, const Maybe& teacher_lse, double temperature) {
  if (!here({&logits, &teacher_ids, &teacher_logits, at_or_null(teacher_lse)})) return std::nullopt;
  // a teacher's tangent is refused by the node, its gradient before this call
  if (!needs_grad({&logits, &teacher_logits, at_or_null(teacher_lse)})) return std::get<0>(distill_run(logits, teacher_ids, teacher_logits, teacher_lse, temperature, false));
  return DistillLoss::apply(logits, teacher_ids, teacher_logits, teacher_lse, temperature);
}
