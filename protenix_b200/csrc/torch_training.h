// The host path of the training operators: dropout-add from a counter-based generator, relative position encoding, windowed attention,
// cross entropy of a linear head, rotary positions, orthogonalised matrices.
// Part of torch_ext.cpp (inside its unnamed namespace).  Each is an autograd function whose two directions are launches of the
// C ABI.  Gradients are computed in kernels, so the ones that are not linear in what they differentiate have no second derivative: a
// backward pass that is asked to build a graph is refused.
#pragma once

void first_derivative_only(const char* name) {
  if (at::GradMode::is_enabled()) fail(std::string(name) + " has no second derivative: call it without create_graph");
}
std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t d : t.sizes()) s += (s.size() == 1 ? "" : ", ") + std::to_string(d);
  return s + "]";
}
// The data of t where the kernels can take it: 16-byte aligned and contiguous.
Tensor aligned(const Tensor& t) {
  const Tensor c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15) == 0 ? c : c.clone();
}

// ---- residual + dropout from a counter-based generator ---------------------------------------------------------------
struct Drop {
  double p;
  int64_t seed, offset, dim;      // dim: the shared axis, -1 where there is none
};

// residual + dropped x (residual undefined: the product alone).  state: (seed, offset) on the device, or undefined; used: receives them.
Tensor dropout_launch(const Tensor& residual, const Tensor& x_, const Drop& d, const Tensor& state, const Tensor& used) {
  c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.contiguous(), r = residual.defined() ? residual.contiguous() : residual;
  const Tensor out = at::empty_like(x);
  int64_t outer = 1, shared = 1, inner = 1;
  for (int64_t i = 0; i < x.dim(); ++i) (d.dim < 0 || i > d.dim ? inner : i == d.dim ? shared : outer) *= x.size(i);
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_dropout_add", st, [&] {
    return abi.px_dropout_add(r.defined() ? r.data_ptr() : nullptr, x.data_ptr(), out.data_ptr(), outer, shared, inner, d.p, d.seed, d.offset,
                              state.defined() ? (const int64_t*)state.data_ptr() : nullptr,
                              used.defined() ? (int64_t*)used.data_ptr() : nullptr, dtype_code(x, "x"), st);
  });
  return out;
}

Tensor dropout_apply(const OptTensor& residual, const Tensor& x, const Drop& d, const Tensor& state);

struct CounterDropoutFunction : torch::autograd::Function<CounterDropoutFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const OptTensor& residual, const Tensor& x, const OptTensor& state, double p,
                        int64_t seed, int64_t offset, int64_t dim) {
    // what a device-side state held at this call: the backward pass drops the same elements, however it has moved on since
    const Tensor used = has(state) ? at::empty({2}, state->options()) : Tensor();
    const Tensor out = dropout_launch(has(residual) ? *residual : Tensor(), x, Drop{p, seed, offset, dim}, has(state) ? *state : Tensor(), used);
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["dim"] = dim;
    ctx->saved_data["f"] = (int64_t)(has(residual) && residual->requires_grad()) | (int64_t)x.requires_grad() << 1;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const int64_t f = ctx->saved_data["f"].toInt();
    const Drop d = {ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(),
                    ctx->saved_data["dim"].toInt()};
    Tensor dx;      // the op again, on the gradient: differentiable like it
    if (f & 2) dx = dropout_apply(c10::nullopt, grads[0], d, ctx->get_saved_variables()[0]);
    return {f & 1 ? grads[0] : Tensor(), dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout_apply(const OptTensor& residual, const Tensor& x, const Drop& d, const Tensor& state) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || (has(residual) && residual->requires_grad())))
    return CounterDropoutFunction::apply(residual, x, state.defined() ? OptTensor(state) : OptTensor(), d.p, d.seed, d.offset, d.dim);
  return dropout_launch(has(residual) ? *residual : Tensor(), x, d, state, Tensor());
}

Tensor counter_dropout_add(const OptTensor& residual, const Tensor& x, double p, int64_t seed, int64_t offset, const OptTensor& state,
                           const c10::optional<int64_t>& shared_dim, bool training) {
  need_cuda(x, "x");
  dtype_code(x, "x");
  if (!(p >= 0.0 && p <= 1.0)) fail("the dropout probability must lie in [0, 1]");
  if (has(residual)) {
    need_on(*residual, x.device(), "residual");
    if (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()) fail("residual must match x");
  }
  if (has(state)) {
    need_on(*state, x.device(), "seed");
    if (state->scalar_type() != at::kLong || state->numel() != 2 || !state->is_contiguous())
      fail("seed as a tensor must hold two contiguous int64 values, the seed and the offset");
  }
  int64_t dim = -1;
  if (shared_dim.has_value()) {
    dim = *shared_dim < 0 ? *shared_dim + x.dim() : *shared_dim;
    if (dim < 0 || dim >= x.dim()) fail("shared_dim " + std::to_string(*shared_dim) + " is out of range for x of shape " + shape_of(x));
  }
  if (!training) return has(residual) ? *residual + x : x.clone();
  no_tangent(x, "x");
  if (has(residual)) no_tangent(*residual, "residual");
  return dropout_apply(residual, x, Drop{p, seed, offset, dim}, has(state) ? *state : Tensor());
}

// ---- relative position encoding --------------------------------------------------------------------------------------
struct RelposSizes {
  int64_t batch, n, c, r, s, type;      // type: of z
};

typedef std::vector<Tensor> Features;      // asym, residue, entity, token, copy numbers: int64, contiguous

// codes: receives the buckets of the pairs, for the backward pass (NULL: not wanted)
Tensor relpos_forward(const Tensor& weight, const Features& f, const RelposSizes& z, Tensor* codes) {
  const Tensor w = aligned(weight.scalar_type() == at::kFloat ? weight : weight.to(at::kFloat));
  const Tensor out = at::empty({z.batch, z.n, z.n, z.c}, w.options().dtype((at::ScalarType)z.type));
  if (codes) *codes = bytes_like(w, abi.px_relpos_codes_bytes(z.batch, z.n));
  const int64_t* id[5];
  for (int i = 0; i < 5; ++i) id[i] = (const int64_t*)f[i].data_ptr();
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_relpos_fwd", st, [&] {
    return abi.px_relpos_fwd(id[0], id[1], id[2], id[3], id[4], (const float*)w.data_ptr(), out.data_ptr(),
                             codes ? (uint32_t*)codes->data_ptr() : nullptr, z.batch, z.n, z.c, (int32_t)z.r, (int32_t)z.s,
                             dtype_code(out, "dtype"), st);
  });
  return out;
}

struct RelposFunction : torch::autograd::Function<RelposFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& weight, const Features& f, int64_t batch, int64_t n, int64_t r,
                        int64_t s, int64_t type) {
    Tensor codes;
    const Tensor z = relpos_forward(weight, f, {batch, n, weight.size(0), r, s, type}, &codes);
    ctx->save_for_backward({codes});
    ctx->saved_data["sizes"] = c10::List<int64_t>({batch, n, weight.size(0), r, s, (int64_t)weight.scalar_type()});
    return z;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    first_derivative_only("relative_position_encoding");
    const Tensor codes = ctx->get_saved_variables()[0];
    const auto v = ctx->saved_data["sizes"].toIntVector();
    c10::cuda::CUDAGuard guard(codes.device());
    const Tensor dz = aligned(grads[0]);
    const int64_t batch = v[0], n = v[1], c = v[2];
    const int32_t r = (int32_t)v[3], s = (int32_t)v[4];
    const Tensor dw = at::empty({c, 4 * r + 2 * s + 7}, dz.options().dtype(at::kFloat));
    const int64_t bytes = abi.px_relpos_workspace_bytes(batch, n, c, r, s);
    const Tensor ws = bytes_like(dz, bytes);
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    launch("px_relpos_bwd", st, [&] {
      return abi.px_relpos_bwd((const uint32_t*)codes.data_ptr(), dz.data_ptr(), (float*)dw.data_ptr(), ws.data_ptr(), bytes, batch, n, c, r, s,
                               dtype_code(dz, "the gradient"), st);
    });
    return {dw.to((at::ScalarType)v[5]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor relative_position_encoding(const Tensor& weight, const std::vector<Tensor>& features, int64_t r, int64_t s,
                                  const c10::optional<at::ScalarType>& z_type) {
  static const char* const names[] = {"asym_id", "residue_index", "entity_id", "token_index", "sym_id"};
  need_cuda(weight, "weight");
  dtype_code(weight, "weight");
  no_tangent(weight, "weight");
  if (r < 0 || s < 0 || r > (1 << 20) || s > (1 << 20)) fail("r_max and s_max must not be negative");
  if (weight.dim() != 2 || weight.size(1) != 4 * r + 2 * s + 7)
    fail("weight must be [c, " + std::to_string(4 * r + 2 * s + 7) + "] for these r_max and s_max, got " + shape_of(weight));
  if (weight.size(0) == 0 || weight.size(0) % 8 != 0 || 4 * r + 2 * s + 5 > 380)
    fail("the kernels handle a multiple of 8 channels and 4 r_max + 2 s_max of up to 375");
  c10::cuda::CUDAGuard guard(weight.device());
  Features rows;
  for (int i = 0; i < 5; ++i) {
    const Tensor& f = features[i];
    need_on(f, weight.device(), names[i]);
    if (!at::isIntegralType(f.scalar_type(), false)) fail(std::string(names[i]) + " must be an integer tensor");
    if (f.dim() < 1 || f.sizes() != features[0].sizes()) fail("the features must have one shape [..., N]");
    rows.push_back(f.to(at::kLong).contiguous());
  }
  const int64_t n = features[0].size(-1), batch = n ? features[0].numel() / n : 0;
  auto shape = features[0].sizes().vec();
  shape.push_back(n);
  shape.push_back(weight.size(0));
  const int64_t type = (int64_t)(z_type.has_value() ? *z_type : weight.scalar_type());
  if (type != (int64_t)at::kFloat && type != (int64_t)at::kBFloat16 && type != (int64_t)at::kHalf) fail("dtype must be float32, bfloat16 or float16");
  const Tensor z = at::GradMode::is_enabled() && weight.requires_grad() ? RelposFunction::apply(weight, rows, batch, n, r, s, type)
                                                                        : relpos_forward(weight, rows, {batch, n, weight.size(0), r, s, type}, nullptr);
  return z.view(shape);
}

// ---- attention with a sliding window ---------------------------------------------------------------------------------
struct WindowCall {
  int64_t left, right, sinks;
  double scale;
};

// [B, H, N, D] as the kernels address it: rows of neighbouring elements, 16-byte aligned, that do not overlap, strides that are multiples of 16 bytes.
Tensor rows_fitted(const Tensor& t) {
  bool fits = t.size(3) <= 1 || t.stride(3) == 1;
  for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) >= t.size(3) && t.stride(i) % 8 == 0));
  if (fits && ((uintptr_t)t.data_ptr() & 15) == 0) return t;
  const Tensor c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15) == 0 ? c : c.clone();
}
px_rows rows_of(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
// A tensor of t's shape whose heads lie inside the rows where t's do, so that what follows (a projection of all heads) needs no copy.
Tensor rows_like(const Tensor& t) {
  const int64_t b = t.size(0), h = t.size(1), n = t.size(2), d = t.size(3);
  const bool inside = h > 1 && n > 1 && t.stride(1) < t.stride(2);
  return inside ? at::empty_strided({b, h, n, d}, {n * h * d, d, h * d, 1}, t.options()) : at::empty(t.sizes(), t.options());
}
px_window window_of(const Tensor& q, const Tensor& k, const Tensor& bias, const Tensor& mask, const WindowCall& c) {
  px_window w = {};
  w.batch = q.size(0), w.heads = q.size(1), w.kv_heads = k.size(1), w.n = q.size(2), w.d = q.size(3);
  w.left = c.left, w.right = c.right, w.sinks = c.sinks;
  w.r_max = bias.defined() ? (bias.size(1) - 1) / 2 : -1;
  w.bias = bias.defined() ? bias.data_ptr() : nullptr;
  w.bias_dtype = bias.defined() ? dtype_code(bias, "rel_bias") : PX_F32;
  w.mask = mask.defined() ? (const uint8_t*)mask.data_ptr() : nullptr;
  w.scale = (float)c.scale;
  w.dtype = dtype_code(q, "q");
  return w;
}
Tensor window_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias, const Tensor& mask, const WindowCall& c, Tensor* lse, Tensor* rest) {
  const Tensor o = rows_like(q);
  const px_window w = window_of(q, k, bias, mask, c);
  if (lse) *lse = at::empty({abi.px_window_lse_floats(w.batch, w.heads, w.n)}, q.options().dtype(at::kFloat));
  if (rest) *rest = rows_like(q);
  const px_rows rq = rows_of(q), rk = rows_of(k), rv = rows_of(v), ro = rows_of(o), rr = rest ? rows_of(*rest) : px_rows{};
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_window_fwd", st, [&] { return abi.px_window_fwd(&w, &rq, &rk, &rv, &ro, rest ? &rr : nullptr, lse ? (float*)lse->data_ptr() : nullptr, st); });
  return o;
}

struct WindowFunction : torch::autograd::Function<WindowFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& bias_,
                        const OptTensor& mask_, int64_t left, int64_t right, int64_t sinks, double scale) {
    c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = rows_fitted(q_), k = rows_fitted(k_), v = rows_fitted(v_);
    const Tensor bias = has(bias_) ? bias_->contiguous() : Tensor(), mask = has(mask_) ? *mask_ : Tensor();
    Tensor lse, rest;
    const Tensor o = window_forward(q, k, v, bias, mask, {left, right, sinks, scale}, &lse, &rest);
    ctx->save_for_backward({q, k, v, o, lse, bias, mask, rest});
    ctx->saved_data["window"] = c10::List<int64_t>({left, right, sinks});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["f"] = (int64_t)q_.requires_grad() | (int64_t)k_.requires_grad() << 1 | (int64_t)v_.requires_grad() << 2 |
                           (int64_t)(has(bias_) && bias_->requires_grad()) << 3;
    return o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    first_derivative_only("window_attention");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4], &bias = saved[5], &mask = saved[6];
    c10::cuda::CUDAGuard guard(q.device());
    const auto at3 = ctx->saved_data["window"].toIntVector();
    const int64_t f = ctx->saved_data["f"].toInt();
    const px_window w = window_of(q, k, bias, mask, {at3[0], at3[1], at3[2], ctx->saved_data["scale"].toDouble()});
    const Tensor dout = rows_fitted(grads[0]);
    Tensor dq, dk, dv, dbias;
    if (f & 1) dq = rows_like(q);
    if (f & 2) dk = rows_like(k);
    if (f & 4) dv = rows_like(v);
    if (f & 8) dbias = at::empty_like(bias);
    const int64_t bytes = abi.px_window_workspace_bytes(&w, f >> 3 & 1);
    const Tensor ws = bytes_like(q, bytes);
    const auto opt = [](const Tensor& t) { return t.defined() ? rows_of(t) : px_rows{}; };
    const px_rows rq = rows_of(q), rk = rows_of(k), rv = rows_of(v), ro = rows_of(o), rr = rows_of(saved[7]), rg = rows_of(dout), gq = opt(dq), gk = opt(dk), gv = opt(dv);
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    launch("px_window_bwd", st, [&] {
      return abi.px_window_bwd(&w, &rq, &rk, &rv, &ro, &rr, &rg, (const float*)lse.data_ptr(), dq.defined() ? &gq : nullptr,
                               dk.defined() ? &gk : nullptr, dv.defined() ? &gv : nullptr, dbias.defined() ? dbias.data_ptr() : nullptr,
                               ws.data_ptr(), bytes, st);
    });
    return {dq, dk, dv, dbias, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t left, int64_t right, int64_t sinks, const OptTensor& bias,
                        const OptTensor& mask, const c10::optional<double>& scale_) {
  need_cuda(q, "q");
  if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) fail("q, k and v must be bfloat16 or float16");
  if (q.dim() < 3) fail("q must be [..., H, N, D], got " + shape_of(q));
  const int64_t h = q.size(-3), n = q.size(-2), d = q.size(-1);
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(k, "k"), std::pair<const Tensor&, const char*>(v, "v")}) {
    need_on(t, q.device(), name);
    if (t.scalar_type() != q.scalar_type()) fail(std::string(name) + " must have the type of q");
    if (t.dim() != q.dim() || t.sizes() != k.sizes() || t.size(-2) != n || t.size(-1) != d || t.size(-3) < 1 || h % t.size(-3) != 0 ||
        !t.sizes().slice(0, t.dim() - 3).equals(q.sizes().slice(0, q.dim() - 3)))
      fail("k and v must be [..., H_kv, N, D] with the batch axes, N and D of q and H_kv a divisor of H; got " + shape_of(q) + ", " +
           shape_of(k) + " and " + shape_of(v));
  }
  if (h < 1 || d < 8 || d > 128 || d % 8 != 0) fail("the kernels handle head sizes of 8 to 128 in steps of 8, got " + shape_of(q));
  if (n > (1 << 24)) fail("at most 2^24 rows");
  if (left < 0 || right < 0 || sinks < 0) fail("window and sinks must not be negative");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)d);
  if (!(scale > 0.0) || !((float)scale > 0.f) || !((float)scale <= 2.35e38f)) fail("scale must be positive and finite, also times log2(e)");
  int64_t batch = 1;
  for (int64_t i = 0; i < q.dim() - 3; ++i) batch *= q.size(i);
  if (batch > 65535 || h > 65535) fail("at most 65535 samples and heads");
  if (has(bias)) {
    need_on(*bias, q.device(), "rel_bias");
    if (bias->dim() != 2 || bias->size(0) != h || bias->size(1) % 2 != 1 || bias->size(1) > 513)
      fail("rel_bias must be [H, 2 r + 1] with r at most 256, got " + shape_of(*bias));
    if (bias->scalar_type() != at::kFloat && bias->scalar_type() != q.scalar_type()) fail("rel_bias must be float32 or of the type of q");
  }
  no_tangent(q, "q");
  no_tangent(k, "k");
  no_tangent(v, "v");
  if (has(bias)) no_tangent(*bias, "rel_bias");
  c10::cuda::CUDAGuard guard(q.device());
  OptTensor m;
  if (has(mask)) {
    need_on(*mask, q.device(), "mask");
    auto want = q.sizes().slice(0, q.dim() - 3).vec();
    want.push_back(n);
    if (mask->dim() < 1 || !at::is_expandable_to(mask->sizes(), want)) fail("mask must be [..., N] over the batch axes of q, got " + shape_of(*mask));
    const Tensor truth = mask->scalar_type() == at::kBool ? mask->detach() : mask->detach().ne(0);
    m = truth.dim() == 2 && truth.size(0) == batch && truth.size(1) == n ? truth.contiguous() : truth.expand(want).reshape({batch, n}).contiguous();
  }
  const auto four = [&](const Tensor& t) { return t.dim() == 4 ? t : t.reshape({batch, t.size(-3), n, d}); };
  const Tensor q4 = four(q), k4 = four(k), v4 = four(v);
  const auto wants = [](const Tensor& t) { return t.requires_grad(); };
  Tensor o;
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || (has(bias) && wants(*bias)))) {
    o = WindowFunction::apply(q4, k4, v4, bias, m, left, right, sinks, scale);
  } else {
    const Tensor b = has(bias) ? bias->contiguous() : Tensor();
    o = window_forward(rows_fitted(q4), rows_fitted(k4), rows_fitted(v4), b, m.has_value() ? *m : Tensor(), {left, right, sinks, scale}, nullptr, nullptr);
  }
  return q.dim() == 4 ? o : o.reshape(q.sizes());
}

// ---- cross entropy of a linear head ----------------------------------------------------------------------------------
struct HeadCall {
  int64_t ignore;
  double smoothing;
  int64_t reduction;      // 0: a loss for each row, 1: mean, 2: sum
};

// [rows, C] as the kernels address it: rows of neighbouring elements that do not overlap, 16-byte aligned.
Tensor matrix_fitted(const Tensor& t) {
  const bool fits = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0));
  return fits && ((uintptr_t)t.data_ptr() & 15) == 0 ? t : aligned(t);
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
px_head head_of(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& target, const HeadCall& c) {
  px_head h = {};
  h.x = x.data_ptr(), h.w = w.data_ptr(), h.target = (const int64_t*)target.data_ptr();
  h.bias = bias.defined() ? bias.data_ptr() : nullptr, h.bias_dtype = bias.defined() ? dtype_code(bias, "bias") : PX_F32;
  h.rows = x.size(0), h.c = x.size(1), h.classes = w.size(0);
  h.x_stride = row_stride(x), h.w_stride = row_stride(w);
  h.ignore = c.ignore, h.smoothing = (float)c.smoothing, h.dtype = dtype_code(x, "x");
  return h;
}
// The loss; norm and inverse receive what the backward pass reads.
Tensor head_loss_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& target, const HeadCall& c, Tensor& norm, Tensor& inverse) {
  const px_head h = head_of(x, w, bias, target, c);
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor loss = c.reduction ? at::empty({}, f32) : at::empty({h.rows}, f32);
  norm = at::empty({h.rows + 1, 2}, f32);
  if (c.reduction) inverse = at::empty({}, f32);
  const int64_t bytes = abi.px_head_loss_workspace_bytes(h.rows, h.classes);
  const Tensor ws = bytes_like(x, bytes);
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_head_loss_fwd", st, [&] {
    return abi.px_head_loss_fwd(&h, (float*)norm.data_ptr(), c.reduction ? nullptr : (float*)loss.data_ptr(), c.reduction ? (float*)loss.data_ptr() : nullptr,
                                c.reduction ? (float*)inverse.data_ptr() : nullptr, c.reduction == 1, ws.data_ptr(), bytes, st);
  });
  return loss;
}

struct HeadLossFunction : torch::autograd::Function<HeadLossFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, const Tensor& target,
                        int64_t ignore, double smoothing, int64_t reduction) {
    c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = matrix_fitted(x_), w = matrix_fitted(w_), bias = has(bias_) ? aligned(*bias_) : Tensor();
    Tensor norm, inverse;
    const Tensor loss = head_loss_forward(x, w, bias, target, {ignore, smoothing, reduction}, norm, inverse);
    ctx->save_for_backward({x, w, bias, target, norm, inverse});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["smoothing"] = smoothing;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    first_derivative_only("linear_cross_entropy");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &bias = saved[2], &target = saved[3], &norm = saved[4], &inverse = saved[5];
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t reduction = ctx->saved_data["reduction"].toInt();
    // of the tensors in their order; without a bias the third is the target, which never does
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = ctx->needs_input_grad(2);
    const px_head h = head_of(x, w, bias, target, {ctx->saved_data["ignore"].toInt(), ctx->saved_data["smoothing"].toDouble(), reduction});
    const Tensor g = grads[0].to(at::kFloat).contiguous();
    Tensor dx, dw, db;
    if (want_x) dx = at::empty({h.rows, h.c}, x.options());
    if (want_w) dw = at::empty({h.classes, h.c}, w.options());
    if (want_b) db = at::empty({h.classes}, bias.options());
    const int64_t bytes = abi.px_head_loss_bwd_workspace_bytes(&h, want_x, want_w, want_b);
    const Tensor ws = bytes_like(x, bytes);
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    launch("px_head_loss_bwd", st, [&] {
      return abi.px_head_loss_bwd(&h, (const float*)norm.data_ptr(), (const float*)g.data_ptr(), reduction == 0, reduction ? (const float*)inverse.data_ptr() : nullptr,
                                  dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr, db.defined() ? db.data_ptr() : nullptr,
                                  ws.data_ptr(), bytes, st);
    });
    return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& target, const OptTensor& bias, int64_t ignore, double smoothing,
                            const std::string& reduction) {
  need_cuda(x, "x");
  if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf) fail("x and weight must be bfloat16 or float16");
  need_on(weight, x.device(), "weight");
  need_on(target, x.device(), "target");
  if (weight.scalar_type() != x.scalar_type()) fail("weight must have the type of x");
  if (x.dim() < 1 || weight.dim() != 2 || weight.size(1) != x.size(-1)) fail("x must be [..., C] and weight [V, C], got " + shape_of(x) + " and " + shape_of(weight));
  const int64_t c = x.size(-1), classes = weight.size(0);
  if (classes < 1 || classes > (1 << 24) || c < 8 || c % 8 != 0 || c > (1 << 20))
    fail("the kernels handle 1 to 2^24 classes and a multiple of 8 channels up to 2^20, got a weight of " + shape_of(weight));
  if (!at::isIntegralType(target.scalar_type(), false)) fail("target must be an integer tensor");
  if (!target.sizes().equals(x.sizes().slice(0, x.dim() - 1))) fail("target must be [...] for x [..., C], got " + shape_of(target) + " and " + shape_of(x));
  if (!(smoothing >= 0.0 && smoothing <= 1.0)) fail("label_smoothing must lie in [0, 1]");
  const int64_t how = reduction == "none" ? 0 : reduction == "mean" ? 1 : reduction == "sum" ? 2 : -1;
  if (how < 0) fail("reduction must be 'none', 'mean' or 'sum', got '" + reduction + "'");
  if (has(bias)) {
    need_on(*bias, x.device(), "bias");
    if (bias->dim() != 1 || bias->size(0) != classes) fail("bias must be [V], got " + shape_of(*bias));
    if (bias->scalar_type() != at::kFloat && bias->scalar_type() != x.scalar_type()) fail("bias must be float32 or of the type of x");
  }
  const int64_t rows = target.numel();
  if (rows > (1 << 26) || (rows + 127) / 128 * ((classes + 63) / 64) > (1ll << 30)) fail("at most 2^26 rows, and 2^43 logits");
  no_tangent(x, "x");
  no_tangent(weight, "weight");
  if (has(bias)) no_tangent(*bias, "bias");
  c10::cuda::CUDAGuard guard(x.device());
  const auto wants = [](const Tensor& t) { return t.requires_grad(); };
  const bool train = at::GradMode::is_enabled() && (wants(x) || wants(weight) || (has(bias) && wants(*bias)));
  if (rows == 0) {      // nothing to launch: what the formula gives, with gradients of zero
    Tensor rest = weight.slice(0, 0, 0).to(at::kFloat).sum();
    if (has(bias)) rest = rest + bias->slice(0, 0, 0).to(at::kFloat).sum();
    const Tensor each = x.to(at::kFloat).sum(-1) + rest;
    return how == 0 ? each : how == 1 ? each.sum() / 0.0 : each.sum();
  }
  const Tensor x2 = x.dim() == 2 ? x : x.reshape({rows, c});      // a view would be a node of the graph
  Tensor t = target.to(at::kLong);
  t = (t.dim() == 1 ? t : t.reshape({rows})).contiguous();
  Tensor loss;
  if (train) {
    loss = HeadLossFunction::apply(x2, weight, bias, t, ignore, smoothing, how);
  } else {
    Tensor norm, inverse;
    loss = head_loss_forward(matrix_fitted(x2), matrix_fitted(weight), has(bias) ? aligned(*bias) : Tensor(), t, {ignore, smoothing, how}, norm, inverse);
  }
  return how == 0 && target.dim() != 1 ? loss.reshape(target.sizes()) : loss;
}

// ---- rotary positions ------------------------------------------------------------------------------------------------
struct RotaryCall {
  std::vector<int64_t> sections;
  double base;
  bool interleaved, per_axis, inverse;
  int64_t batch, row, axis;      // strides of the positions
};
typedef std::pair<Tensor, Tensor> TwoTensors;

Tensor channels_fitted(const Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }
// q and k [B, H, N, D] turned (k undefined: q alone); positions int64, by the strides of the call.
TwoTensors rotary_launch(const Tensor& q_, const Tensor& k_, const Tensor& positions, const RotaryCall& c) {
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = channels_fitted(q_), k = k_.defined() ? channels_fitted(k_) : k_;
  const Tensor qo = rows_like(q), ko = k.defined() ? rows_like(k) : k;
  const std::vector<int32_t> sections(c.sections.begin(), c.sections.end());
  px_rotary r = {};
  r.positions = (const int64_t*)positions.data_ptr();
  r.position_batch = c.batch, r.position_row = c.row, r.position_axis = c.axis;
  r.batch = q.size(0), r.heads = q.size(1), r.kv_heads = k.defined() ? k.size(1) : 0, r.n = q.size(2), r.d = q.size(3);
  r.sections = sections.data(), r.axes = (int32_t)sections.size(), r.base = c.base;
  r.interleaved = c.interleaved, r.per_axis = c.per_axis, r.dtype = dtype_code(q, "q");
  const px_rows iq = rows_of(q), oq = rows_of(qo), ik = k.defined() ? rows_of(k) : px_rows{}, ok = k.defined() ? rows_of(ko) : px_rows{};
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_rotary_turn", st, [&] { return abi.px_rotary_turn(&r, &iq, &oq, k.defined() ? &ik : nullptr, k.defined() ? &ok : nullptr, c.inverse, st); });
  return {qo, ko};
}

TwoTensors rotary_apply(const Tensor& q, const Tensor& k, const Tensor& positions, const RotaryCall& c);

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                                                std::vector<int64_t> sections, double base, bool interleaved, bool per_axis, bool inverse,
                                                std::vector<int64_t> strides) {
    ctx->set_materialize_grads(false);
    const auto out = rotary_launch(q, has(k) ? *k : Tensor(), positions, {sections, base, interleaved, per_axis, inverse, strides[0], strides[1], strides[2]});
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = c10::List<int64_t>(c10::ArrayRef<int64_t>(sections));
    ctx->saved_data["strides"] = c10::List<int64_t>(c10::ArrayRef<int64_t>(strides));
    ctx->saved_data["base"] = base;
    ctx->saved_data["how"] = (int64_t)interleaved | (int64_t)per_axis << 1 | (int64_t)inverse << 2;
    if (!out.second.defined()) return {out.first};
    // what does not depend on a leaf asks for no gradient
    if (!q.requires_grad()) ctx->mark_non_differentiable({out.first});
    if (!k->requires_grad()) ctx->mark_non_differentiable({out.second});
    return {out.first, out.second};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const int64_t how = ctx->saved_data["how"].toInt();
    const Tensor positions = ctx->get_saved_variables()[0];
    const auto st = ctx->saved_data["strides"].toIntVector();
    const RotaryCall c = {ctx->saved_data["sections"].toIntVector(), ctx->saved_data["base"].toDouble(), (how & 1) != 0, (how & 2) != 0, (how & 4) == 0, st[0], st[1], st[2]};
    const Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    Tensor dq, dk;      // the operator again, by the negated angles: differentiable like it
    if (gq.defined() && gk.defined())
      std::tie(dq, dk) = rotary_apply(gq, gk, positions, c);
    else if (gq.defined())
      dq = rotary_apply(gq, Tensor(), positions, c).first;
    else if (gk.defined())
      dk = rotary_apply(gk, Tensor(), positions, c).first;
    return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

TwoTensors rotary_apply(const Tensor& q, const Tensor& k, const Tensor& positions, const RotaryCall& c) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
    const auto out = RotaryFunction::apply(q, k.defined() ? OptTensor(k) : OptTensor(), positions, c.sections, c.base, c.interleaved, c.per_axis, c.inverse,
                                           std::vector<int64_t>{c.batch, c.row, c.axis});
    return {out[0], k.defined() ? out[1] : Tensor()};
  }
  return rotary_launch(q, k, positions, c);
}

py::object rotary_embedding(const Tensor& q, const OptTensor& k, const Tensor& positions, const std::vector<int64_t>& sections, double base,
                            bool interleaved, bool per_axis) {
  need_cuda(q, "q");
  dtype_code(q, "q");
  if (q.dim() < 3) fail("q must be [..., H, N, D], got " + shape_of(q));
  const int64_t n = q.size(-2), d = q.size(-1), axes = (int64_t)sections.size();
  const auto batch_axes = q.sizes().slice(0, q.dim() - 3);
  if (q.size(-3) < 1 || d < 2 || d > 65536) fail("q must have at least one head and 2 to 65536 channels, got " + shape_of(q));
  if (has(k)) {
    need_on(*k, q.device(), "k");
    if (k->scalar_type() != q.scalar_type()) fail("k must have the type of q");
    if (k->dim() != q.dim() || k->size(-1) != d || k->size(-2) != n || k->size(-3) < 1 || !k->sizes().slice(0, k->dim() - 3).equals(batch_axes))
      fail("k must be [..., H_kv, N, D] with the batch axes, N and D of q; got " + shape_of(q) + " and " + shape_of(*k));
  }
  need_on(positions, q.device(), "positions");
  if (!at::isIntegralType(positions.scalar_type(), false)) fail("positions must be an integer tensor");
  int64_t pairs = 0;
  for (int64_t s : sections) {
    if (s < 0 || s > d / 2) fail("sections must be numbers of pairs, from 0 to D / 2");
    pairs += s;
  }
  if (axes < 1 || axes > 255 || pairs < 1 || pairs > 256 || 2 * pairs > d) fail("sections must hold 1 to D / 2 pairs, 256 at most, on up to 255 axes");
  if (!(base >= 1.0 && base <= 1e30)) fail("base must lie in [1, 1e30]");
  auto want = batch_axes.vec();
  want.push_back(n);
  want.push_back(axes);
  if (positions.dim() < 2 || positions.size(-1) != axes || !at::is_expandable_to(positions.sizes(), want))
    fail("positions must be [..., N, A] over the batch axes of q, one axis for each section, got " + shape_of(positions));
  no_tangent(q, "q");
  if (has(k)) no_tangent(*k, "k");
  int64_t batch = 1;
  for (int64_t b : batch_axes) batch *= b;
  const int64_t heads = q.size(-3) + (has(k) ? k->size(-3) : 0);
  if (batch > 65535 || heads > 65536 || n > (1 << 30)) fail("at most 65535 samples, 65536 heads and 2^30 rows");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor p = positions.scalar_type() == at::kLong ? positions : positions.to(at::kLong);
  RotaryCall call = {sections, base, interleaved, per_axis, false, 0, p.stride(-2), p.stride(-1)};
  if (p.size(-2) != n) call.row = 0;      // one place for all rows
  if (p.dim() == 3 && q.dim() == 4 && p.size(0) == batch) {
    call.batch = p.stride(0);
  } else if (p.numel() != p.size(-2) * axes) {      // samples of their own, over several axes or broadcast along some
    p = p.expand(want).reshape({batch, n, axes});
    call.batch = p.stride(0), call.row = p.stride(1), call.axis = p.stride(2);
  }
  const auto four = [&](const Tensor& t) { return t.dim() == 4 ? t : t.reshape({batch, t.size(-3), n, d}); };
  const auto out = rotary_apply(four(q), has(k) ? four(*k) : Tensor(), p, call);
  const auto back = [&](const Tensor& t, const Tensor& like) { return like.dim() == 4 ? t : t.reshape(like.sizes()); };
  const py::object first = py::cast(back(out.first, q));
  return has(k) ? py::object(py::make_tuple(first, back(out.second, *k))) : first;
}

// ---- orthogonalised matrices -----------------------------------------------------------------------------------------
Tensor orthogonalize(const Tensor& g_, const std::vector<double>& coefficients, double eps) {
  need_cuda(g_, "g");
  const int type = dtype_code(g_, "g");
  if (g_.dim() < 2) fail("g must be [..., M, N], got " + shape_of(g_));
  const int64_t m = g_.size(-2), n = g_.size(-1), batch = m && n ? g_.numel() / (m * n) : 0;
  const int64_t steps = (int64_t)coefficients.size() / 3;
  if (coefficients.size() % 3 != 0 || steps < 1 || steps > 1000) fail("coefficients must be 1 to 1000 triples (a, b, c)");
  for (double c : coefficients)
    if (!std::isfinite((float)c)) fail("coefficients must be finite");
  if (!(eps >= 0.0) || !std::isfinite(eps)) fail("eps must not be negative");
  if (batch > 65535 || m > (1 << 20) || n > (1 << 20)) fail("at most 65535 matrices of 2^20 rows and columns, got " + shape_of(g_));
  no_tangent(g_, "g");
  if (at::GradMode::is_enabled() && g_.requires_grad()) fail("orthogonalize is not differentiable: call it on a detached tensor or under no_grad");
  c10::cuda::CUDAGuard guard(g_.device());
  const Tensor g = g_.contiguous(), out = at::empty(g.sizes(), g.options());
  if (batch == 0) return out;
  const std::vector<float> c(coefficients.begin(), coefficients.end());
  const int64_t bytes = abi.px_orthogonalize_steps_workspace_bytes(batch, m, n, (int32_t)steps);
  const Tensor ws = bytes_like(g, bytes);
  const cudaStream_t st = at::cuda::getCurrentCUDAStream();
  launch("px_orthogonalize", st, [&] {
    return abi.px_orthogonalize(g.data_ptr(), out.data_ptr(), batch, m, n, c.data(), (int32_t)steps, eps, type, ws.data_ptr(), bytes, st);
  });
  return out;
}
