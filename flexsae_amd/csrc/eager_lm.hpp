// The calls of the operators around a dictionary in a model, as part of the extension module (eager.cpp): layer norm, the lookup of
// rows by token, distillation, each with its autograd node.  A backward that is not plain goes to the op of its gradient, through
// torch's dispatcher, which every tracer, mode and transform sees.
// (Included by eager.cpp within its namespace.)
#pragma once

// Rows along the last dimension at one distance (in elements) from each other: the tensor itself, or a contiguous copy.
struct RowsOf {
  Tensor t;
  int64_t stride;
};
RowsOf rows_of(const Tensor &t) {
  const int64_t dims = t.dim(), cols = t.size(-1);
  if (t.numel() > 0 && (cols == 1 || t.stride(-1) == 1)) {
    int64_t rows = 1, stride = cols, d = dims - 2;
    for (; d >= 0; --d) {
      if (t.size(d) == 1) continue;
      if (rows == 1) stride = t.stride(d);
      else if (t.stride(d) != stride * rows) break;
      rows *= t.size(d);
    }
    if (d < 0) return {t, stride};
  }
  return {t.contiguous(), cols};
}

at::IntArrayRef leading(const Tensor &t) { return t.sizes().slice(0, static_cast<size_t>(t.dim()) - 1); }

const void *or_null(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *or_null_out(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
int dtype_or_f32(const Tensor &t) { return t.defined() ? dtype_of(t.scalar_type()) : FLEXSAE_F32; }
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool known_device(const Tensor &t) {
  const int device = t.device().index();
  return device >= 0 && device < kMaxDevices && status_flags[device].defined();
}
bool plain_beside(const Tensor &t, const Tensor &other) { return plain_tensor(t) && t.device() == other.device(); }
Tensor given_or_none(const Tensor &t, bool wanted) { return wanted ? t : Tensor(); }

// A tensor argument, or None: an undefined tensor.  False: neither.
bool take_optional(PyObject *o, Tensor &out) {
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  out = THPVariable_Unpack(o);
  return true;
}

// ---- layer norm ----------------------------------------------------------------------------
bool usable_norm(const Tensor &x, const Tensor &weight, const Tensor &bias) {
  if (!plain_tensor(x) || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) >= (int64_t{1} << 27) || dtype_of(x.scalar_type()) < 0) return false;
  for (const Tensor *t : {&weight, &bias})
    if (t->defined() && (!plain_beside(*t, x) || t->dim() != 1 || t->size(0) != x.size(-1) || dtype_of(t->scalar_type()) < 0)) return false;
  return true;
}

flexsae_norm norm_of(const Tensor &x, int64_t x_stride, int64_t dy_stride, const Tensor &weight, const Tensor &bias, double eps) {
  return {x.numel() / x.size(-1), x.size(-1), x_stride, dy_stride, static_cast<float>(eps), dtype_of(x.scalar_type()),
          dtype_or_f32(weight), dtype_or_f32(bias)};
}

// (y, mean, rstd); mean and rstd only where asked for
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor &given, const Tensor &given_weight, const Tensor &given_bias, double eps,
                                                bool stats) {
  const c10::DeviceGuard guard(given.device());
  const RowsOf x = rows_of(given);
  const Tensor weight = given_weight.defined() ? given_weight.contiguous() : Tensor();
  const Tensor bias = given_bias.defined() ? given_bias.contiguous() : Tensor();
  const Tensor y = make(given, given.sizes(), given.scalar_type());
  Tensor mean, rstd;
  if (stats) {
    mean = make(given, leading(given), c10::ScalarType::Float);
    rstd = make(given, leading(given), c10::ScalarType::Float);
  }
  const flexsae_norm n = norm_of(given, x.stride, 0, weight, bias, eps);
  check(lib.layer_norm_fwd(&n, x.t.const_data_ptr(), or_null(weight), or_null(bias), y.data_ptr(), stats ? f32(mean) : nullptr,
                           stats ? f32(rstd) : nullptr, stream_of(given)),
        "flexsae_layer_norm_fwd");
  return {y, mean, rstd};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext *ctx, const Variable &x, const std::optional<Tensor> &weight,
                               const std::optional<Tensor> &bias, double eps) {
    auto [y, mean, rstd] = norm_forward(x, weight.value_or(Tensor()), bias.value_or(Tensor()), eps, true);
    ctx->save_for_backward({x, weight.value_or(Tensor()), bias.value_or(Tensor()), mean, rstd});
    ctx->mark_non_differentiable({mean, rstd});
    ctx->set_materialize_grads(false);
    return {y, mean, rstd};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor &given = grads[0];
    if (!given.defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &given_weight = saved[1], &given_bias = saved[2], &mean = saved[3], &rstd = saved[4];
    // (the edges are those of the tensors that there are)
    const bool need_x = ctx->needs_input_grad(0), need_weight = given_weight.defined() && ctx->needs_input_grad(1),
               need_bias = given_bias.defined() && ctx->needs_input_grad(given_weight.defined() ? 2 : 1);
    const bool plain = plain_backward(given) && usable_norm(x, given_weight, given_bias) && plain_beside(given, x) &&
                       given.scalar_type() == x.scalar_type() && given.sizes() == x.sizes() && usable_fp32(mean, x, leading(x)) &&
                       usable_fp32(rstd, x, leading(x));
    if (!plain) {
      static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("flexsae_amd::layer_norm_bwd", "").typed<
          std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const std::optional<Tensor> &,
                                             const std::optional<Tensor> &, const Tensor &, const Tensor &, bool, bool, bool)>();
      const auto [dx, dw, db] = op.call(given, x, maybe(given_weight), maybe(given_bias), mean, rstd, need_x, need_weight, need_bias);
      return {given_or_none(dx, need_x), given_or_none(dw, need_weight), given_or_none(db, need_bias), Tensor()};
    }
    const c10::DeviceGuard guard(x.device());
    const RowsOf in = rows_of(x), dy = rows_of(given);
    const Tensor weight = given_weight.defined() ? given_weight.contiguous() : Tensor();
    const Tensor m = mean.contiguous(), r = rstd.contiguous();
    Tensor dx, dw, db;
    if (need_x) dx = make(x, x.sizes(), x.scalar_type());
    if (need_weight) dw = make(x, {x.size(-1)}, given_weight.scalar_type());
    if (need_bias) db = make(x, {x.size(-1)}, given_bias.scalar_type());
    const flexsae_norm n = norm_of(x, in.stride, dy.stride, given_weight, given_bias, 0.);
    const size_t bytes = need_weight || need_bias ? lib.layer_norm_bwd_workspace_bytes(&n) : 0;
    const Tensor workspace = make_workspace(x, bytes);
    check(lib.layer_norm_bwd(&n, in.t.const_data_ptr(), dy.t.const_data_ptr(), or_null(weight), f32(m), f32(r), or_null_out(dx),
                             or_null_out(dw), or_null_out(db), workspace.data_ptr(), bytes, stream_of(x)),
          "flexsae_layer_norm_bwd");
    return {dx, dw, db, Tensor()};
  }
};

// layer_norm(x, weight, bias, eps, stats) -> y, or with stats (y, mean, rstd)
PyObject *py_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 5)) return nullptr;
  Tensor x, weight, bias;
  if (!PyFloat_Check(args[3]) || !THPVariable_CheckExact(args[0]) || !take_optional(args[1], weight) || !take_optional(args[2], bias))
    Py_RETURN_NONE;
  x = THPVariable_Unpack(args[0]);
  const double eps = real(args[3]);
  const bool stats = number(args[4]) != 0;
  if (!plain_surroundings() || !usable_norm(x, weight, bias) || !(eps >= 0.) || !(eps < 3e38)) Py_RETURN_NONE;
  Tensor y, mean, rstd;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = c10::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) ||
                                                      (bias.defined() && bias.requires_grad()));
    if (grad) {
      const auto out = LayerNorm::apply(x, maybe(weight), maybe(bias), eps);
      y = out[0], mean = out[1], rstd = out[2];
    } else {
      std::tie(y, mean, rstd) = norm_forward(x, weight, bias, eps, stats);
    }
  }
  if (!stats) return THPVariable_Wrap(y);
  return Py_BuildValue("NNN", THPVariable_Wrap(y), THPVariable_Wrap(mean), THPVariable_Wrap(rstd));
  END_HANDLE_TH_ERRORS
}

// ---- lookup --------------------------------------------------------------------------------
bool usable_lookup(const Tensor &tokens, const Tensor &weight, const Tensor &scale) {
  if (!plain_tensor(weight) || weight.dim() != 2 || weight.numel() == 0 || dtype_of(weight.scalar_type()) < 0 || !known_device(weight) ||
      weight.size(0) >= (int64_t{1} << 31) || weight.size(1) >= (int64_t{1} << 29))
    return false;
  if (!plain_beside(tokens, weight) || tokens.scalar_type() != c10::ScalarType::Long || tokens.numel() >= (int64_t{1} << 32)) return false;
  return !scale.defined() || (plain_beside(scale, weight) && scale.sizes() == tokens.sizes() && dtype_of(scale.scalar_type()) >= 0);
}

flexsae_lookup lookup_of(const Tensor &tokens, const Tensor &weight, const Tensor &scale, int64_t weight_stride, int64_t dout_stride,
                         double factor) {
  return {tokens.numel(), weight.size(0), weight.size(1), weight_stride, dout_stride, static_cast<float>(factor),
          dtype_of(weight.scalar_type()), dtype_or_f32(scale)};
}

c10::SmallVector<int64_t, 6> looked_up(const Tensor &tokens, const Tensor &weight) {
  c10::SmallVector<int64_t, 6> sizes(tokens.sizes().begin(), tokens.sizes().end());
  sizes.push_back(weight.size(1));
  return sizes;
}

Tensor lookup_forward(const Tensor &given_tokens, const Tensor &weight, const Tensor &given_scale, double factor) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor tokens = given_tokens.contiguous(), scale = given_scale.defined() ? given_scale.contiguous() : Tensor();
  const RowsOf w = rows_of(weight);
  const Tensor out = make(weight, looked_up(tokens, weight), weight.scalar_type());
  const flexsae_lookup l = lookup_of(tokens, weight, scale, w.stride, 0, factor);
  check(lib.lookup_fwd(&l, index_ptr(tokens), w.t.const_data_ptr(), or_null(scale), out.data_ptr(), flag_of(weight), stream_of(weight)),
        "flexsae_lookup_fwd");
  return out;
}

struct Lookup : torch::autograd::Function<Lookup> {
  static Variable forward(AutogradContext *ctx, const Variable &tokens, const Variable &weight, const std::optional<Tensor> &scale,
                          double factor) {
    ctx->save_for_backward({tokens, weight, scale.value_or(Tensor())});
    ctx->set_materialize_grads(false);
    ctx->saved_data["factor"] = factor;
    return lookup_forward(tokens, weight, scale.value_or(Tensor()), factor);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor &given = grads[0];
    if (!given.defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    const Tensor &weight = saved[1], &given_scale = saved[2];
    const double factor = ctx->saved_data["factor"].toDouble();
    const bool need_weight = ctx->needs_input_grad(1), need_scale = given_scale.defined() && ctx->needs_input_grad(2);
    if (!plain_backward(given) || !usable_lookup(saved[0], weight, given_scale) || !plain_beside(given, weight) ||
        given.scalar_type() != weight.scalar_type() || given.sizes() != at::IntArrayRef(looked_up(saved[0], weight))) {
      static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("flexsae_amd::lookup_bwd", "").typed<
          std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const std::optional<Tensor> &, double, bool, bool)>();
      const auto [dw, ds] = op.call(given, saved[0], weight, maybe(given_scale), factor, need_weight, need_scale);
      return {Tensor(), given_or_none(dw, need_weight), given_or_none(ds, need_scale), Tensor()};
    }
    const c10::DeviceGuard guard(weight.device());
    const Tensor tokens = saved[0].contiguous(), scale = given_scale.defined() ? given_scale.contiguous() : Tensor();
    const RowsOf w = rows_of(weight), dout = rows_of(given);
    Tensor dw, ds;
    if (need_weight) dw = make(weight, weight.sizes(), weight.scalar_type());
    if (need_scale) ds = make(weight, tokens.sizes(), scale.scalar_type());
    const flexsae_lookup l = lookup_of(tokens, weight, scale, w.stride, dout.stride, factor);
    const size_t bytes = lib.lookup_bwd_workspace_bytes(&l);
    const Tensor workspace = make_workspace(weight, bytes);
    check(lib.lookup_bwd(&l, index_ptr(tokens), w.t.const_data_ptr(), or_null(scale), dout.t.const_data_ptr(), or_null_out(dw),
                         or_null_out(ds), workspace.data_ptr(), bytes, stream_of(weight)),
          "flexsae_lookup_bwd");
    return {Tensor(), dw, ds, Tensor()};
  }
};

// embedding_lookup(tokens, weight, scale, factor) -> out
PyObject *py_embedding_lookup(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 4)) return nullptr;
  Tensor tokens, weight, scale;
  if (!THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) || !take_optional(args[2], scale)) Py_RETURN_NONE;
  tokens = THPVariable_Unpack(args[0]);
  weight = THPVariable_Unpack(args[1]);
  const double factor = real(args[3]);
  if (!plain_surroundings() || !usable_lookup(tokens, weight, scale) || !(std::abs(factor) < 3e38)) Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = c10::GradMode::is_enabled() && (weight.requires_grad() || (scale.defined() && scale.requires_grad()));
    out = grad ? Lookup::apply(tokens, weight, maybe(scale), factor) : lookup_forward(tokens, weight, scale, factor);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- distillation --------------------------------------------------------------------------
struct Teacher {
  Tensor top, index, row_weights;
};

bool usable_distill(const Tensor &logits, const Teacher &t) {
  if (!plain_tensor(logits) || logits.dim() < 1 || logits.numel() == 0 || dtype_of(logits.scalar_type()) < 0 || !known_device(logits) ||
      logits.size(-1) >= (int64_t{1} << 31) || logits.numel() / logits.size(-1) >= (int64_t{1} << 31))
    return false;
  if (!plain_beside(t.top, logits) || !plain_beside(t.index, logits) || t.index.scalar_type() != c10::ScalarType::Long ||
      dtype_of(t.top.scalar_type()) < 0 || t.top.dim() != logits.dim() || t.top.sizes() != t.index.sizes() || t.top.size(-1) < 1 ||
      leading(t.top) != leading(logits))
    return false;
  return !t.row_weights.defined() || usable_fp32(t.row_weights, logits, leading(logits));
}

flexsae_distill distill_of(const Tensor &logits, int64_t stride, const Tensor &top, double temperature, bool by_row) {
  return {logits.numel() / logits.size(-1), logits.size(-1), top.size(-1), stride, static_cast<float>(temperature),
          dtype_of(logits.scalar_type()), dtype_of(top.scalar_type()), by_row ? FLEXSAE_DISTILL_BY_ROW : 0};
}

Teacher contiguous(const Teacher &t) {
  return {t.top.contiguous(), t.index.contiguous(), t.row_weights.defined() ? t.row_weights.contiguous() : Tensor()};
}
const float *weights_ptr(const Teacher &t) { return t.row_weights.defined() ? t.row_weights.const_data_ptr<float>() : nullptr; }

// (loss, stats, the gradient for an upstream gradient of one where asked for)
std::tuple<Tensor, Tensor, Tensor> distill_forward(const Tensor &logits, const Teacher &given, double temperature, bool by_row, bool early) {
  const c10::DeviceGuard guard(logits.device());
  const RowsOf z = rows_of(logits);
  const Teacher t = contiguous(given);
  const flexsae_distill d = distill_of(logits, z.stride, t.top, temperature, by_row);
  const Tensor loss = make(logits, by_row ? leading(logits) : at::IntArrayRef{}, c10::ScalarType::Float);
  const Tensor stats = make(logits, {d.rows + 1, 4}, c10::ScalarType::Float);
  const Tensor dlogits = early ? make(logits, logits.sizes(), logits.scalar_type()) : Tensor();
  const size_t bytes = lib.distill_workspace_bytes(&d);
  const Tensor workspace = make_workspace(logits, bytes);
  check(lib.distill_fwd(&d, z.t.const_data_ptr(), t.top.const_data_ptr(), index_ptr(t.index), weights_ptr(t), f32(loss), f32(stats),
                        or_null_out(dlogits), workspace.data_ptr(), bytes, flag_of(logits), stream_of(logits)),
        "flexsae_distill_fwd");
  return {loss, stats, dlogits};
}

struct Distill : torch::autograd::Function<Distill> {
  static Variable forward(AutogradContext *ctx, const Variable &logits, const Teacher &t, double temperature, bool by_row) {
    // (gradients of fp16 logits carry a loss scale, without which they vanish in that type)
    const bool early = !by_row && logits.scalar_type() != c10::ScalarType::Half;
    auto [loss, stats, dlogits] = distill_forward(logits, t, temperature, by_row, early);
    ctx->save_for_backward({logits, t.top, t.index, t.row_weights, stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["t"] = temperature;
    ctx->saved_data["by_row"] = by_row;
    // no saved tensor: the backward completes it in place and hands the very buffer on
    if (early) {
      ctx->saved_data["dlogits"] = dlogits;
      ctx->saved_data["capture"] = capture_of(logits);
    }
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor &given = grads[0];
    if (!given.defined()) return variable_list(4);
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0];
    const Teacher teacher = {saved[1], saved[2], saved[3]};
    const double temperature = ctx->saved_data["t"].toDouble();
    const bool by_row = ctx->saved_data["by_row"].toBool();
    const int64_t rows = logits.numel() / (logits.dim() > 0 && logits.size(-1) > 0 ? logits.size(-1) : 1);
    if (!plain_backward(given) || !usable_distill(logits, teacher) || !plain_beside(given, logits) ||
        given.sizes() != (by_row ? leading(logits) : at::IntArrayRef{}) || !usable_fp32(saved[4], logits, {rows + 1, 4})) {
      static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("flexsae_amd::distill_bwd", "").typed<
          Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const std::optional<Tensor> &, const Tensor &, double, bool)>();
      return {op.call(given, logits, teacher.top, teacher.index, maybe(teacher.row_weights), saved[4], temperature, by_row), Tensor(),
              Tensor(), Tensor()};
    }
    const c10::DeviceGuard guard(logits.device());
    const Tensor grad = given.to(c10::ScalarType::Float).contiguous(), stats = prepared(saved[4]);
    const RowsOf z = rows_of(logits);
    const Teacher t = contiguous(teacher);
    Tensor dlogits;
    const auto at = ctx->saved_data.find("dlogits");
    if (at != ctx->saved_data.end()) {
      dlogits = at->second.toTensor();
      ctx->saved_data.erase("dlogits");  // the buffer now belongs to whoever receives the gradient
    }
    // (not one of another graph, or of none: what a replay writes there would be another's, or what it finds there no gradient for
    // an upstream gradient of one any more)
    const bool early = dlogits.defined() && dlogits.device() == logits.device() && dlogits.sizes() == logits.sizes() &&
                       dlogits.scalar_type() == logits.scalar_type() && ctx->saved_data["capture"].toInt() == capture_of(logits);
    if (!early) dlogits = make(logits, logits.sizes(), logits.scalar_type());
    const flexsae_distill d = distill_of(logits, z.stride, t.top, temperature, by_row);
    check(lib.distill_bwd(&d, z.t.const_data_ptr(), t.top.const_data_ptr(), index_ptr(t.index), weights_ptr(t), f32(stats), f32(grad),
                          early, dlogits.data_ptr(), stream_of(logits)),
          "flexsae_distill_bwd");
    return {dlogits, Tensor(), Tensor(), Tensor()};
  }
};

// distillation_loss(logits, top_logits, top_indices, row_weights, temperature, by_row) -> loss
PyObject *py_distillation_loss(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 6)) return nullptr;
  Teacher t;
  if (!THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) || !THPVariable_CheckExact(args[2]) ||
      !take_optional(args[3], t.row_weights) || !(PyFloat_Check(args[4]) || PyLong_Check(args[4])))
    Py_RETURN_NONE;
  const Tensor logits = THPVariable_Unpack(args[0]);
  t.top = THPVariable_Unpack(args[1]);
  t.index = THPVariable_Unpack(args[2]);
  const double temperature = real(args[4]);
  const bool by_row = number(args[5]) != 0;
  if (!plain_surroundings() || !usable_distill(logits, t) || !(temperature > 1e-18) || !(temperature < 1e18)) Py_RETURN_NONE;
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    t.top = t.top.detach();
    loss = c10::GradMode::is_enabled() && logits.requires_grad() ? Distill::apply(logits, t, temperature, by_row)
                                                                 : std::get<0>(distill_forward(logits, t, temperature, by_row, false));
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}
