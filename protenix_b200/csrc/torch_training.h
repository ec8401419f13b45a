// The host path of the training operators: dropout-add from a counter-based generator, relative position encoding.
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
                           const c10::optional<int64_t>& shared_dim) {
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
  return dropout_apply(residual, x, Drop{p, seed, offset, dim}, has(state) ? *state : Tensor());
}

// ---- relative position encoding --------------------------------------------------------------------------------------
struct RelposSizes {
  int64_t batch, n, c, r, s, type;      // type: of z
};

struct RelposFunction : torch::autograd::Function<RelposFunction> {
  // ids: [5][batch][n], in the order of the C ABI
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& weight, const Tensor& ids, int64_t batch, int64_t n, int64_t r,
                        int64_t s, int64_t type) {
    ctx->save_for_backward({ids});
    ctx->saved_data["sizes"] = c10::List<int64_t>({batch, n, weight.size(0), r, s, type, (int64_t)weight.scalar_type()});
    return run(weight, ids, {batch, n, weight.size(0), r, s, type});
  }
  static Tensor run(const Tensor& weight, const Tensor& ids, const RelposSizes& z) {
    c10::cuda::CUDAGuard guard(ids.device());
    const Tensor w = weight.detach().to(at::kFloat).contiguous();
    const Tensor out = at::empty({z.batch, z.n, z.n, z.c}, w.options().dtype((at::ScalarType)z.type));
    const int64_t *id = (const int64_t*)ids.data_ptr(), per = z.batch * z.n;
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    launch("px_relpos_fwd", st, [&] {
      return abi.px_relpos_fwd(id, id + per, id + 2 * per, id + 3 * per, id + 4 * per, (const float*)w.data_ptr(), out.data_ptr(), z.batch, z.n,
                               z.c, (int32_t)z.r, (int32_t)z.s, dtype_code(out, "dtype"), st);
    });
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    first_derivative_only("relative_position_encoding");
    const Tensor ids = ctx->get_saved_variables()[0];
    const auto v = ctx->saved_data["sizes"].toIntVector();
    c10::cuda::CUDAGuard guard(ids.device());
    const Tensor dz = aligned(grads[0]);
    const int64_t batch = v[0], n = v[1], c = v[2];
    const int32_t r = (int32_t)v[3], s = (int32_t)v[4];
    const Tensor dw = at::empty({c, 4 * r + 2 * s + 7}, ids.options().dtype(at::kFloat));
    const int64_t bytes = abi.px_relpos_workspace_bytes(batch, n, c, r, s);
    const Tensor ws = bytes_like(ids, bytes);
    const int64_t *id = (const int64_t*)ids.data_ptr(), per = batch * n;
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    launch("px_relpos_bwd", st, [&] {
      return abi.px_relpos_bwd(id, id + per, id + 2 * per, id + 3 * per, id + 4 * per, dz.data_ptr(), (float*)dw.data_ptr(), ws.data_ptr(), bytes,
                               batch, n, c, r, s, dtype_code(dz, "the gradient"), st);
    });
    return {dw.to((at::ScalarType)v[6]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor relative_position_encoding(const Tensor& weight, const std::vector<Tensor>& features, int64_t r, int64_t s,
                                  const c10::optional<at::ScalarType>& z_type) {
  static const char* const names[] = {"asym_id", "residue_index", "entity_id", "token_index", "sym_id"};
  need_cuda(weight, "weight");
  dtype_code(weight, "weight");
  if (r < 0 || s < 0 || r > (1 << 20) || s > (1 << 20)) fail("r_max and s_max must not be negative");
  if (weight.dim() != 2 || weight.size(1) != 4 * r + 2 * s + 7)
    fail("weight must be [c, " + std::to_string(4 * r + 2 * s + 7) + "] for these r_max and s_max, got " + shape_of(weight));
  if (weight.size(0) == 0 || weight.size(0) % 8 != 0 || 4 * r + 2 * s + 5 > 380)
    fail("the kernels handle a multiple of 8 channels and 4 r_max + 2 s_max of up to 375");
  std::vector<Tensor> rows;
  for (int i = 0; i < 5; ++i) {
    const Tensor& f = features[i];
    need_on(f, weight.device(), names[i]);
    if (!at::isIntegralType(f.scalar_type(), false)) fail(std::string(names[i]) + " must be an integer tensor");
    if (f.dim() < 1 || f.sizes() != features[0].sizes()) fail("the features must have one shape [..., N]");
    rows.push_back(f.to(at::kLong));
  }
  const int64_t n = features[0].size(-1), batch = n ? features[0].numel() / n : 0;
  auto shape = features[0].sizes().vec();
  shape.push_back(n);
  shape.push_back(weight.size(0));
  c10::cuda::CUDAGuard guard(weight.device());
  Tensor ids;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    ids = at::stack(rows).reshape({5, batch, n});      // one piece, and a snapshot: the backward pass reads it again
  }
  const int64_t type = (int64_t)(z_type.has_value() ? *z_type : weight.scalar_type());
  if (type != (int64_t)at::kFloat && type != (int64_t)at::kBFloat16 && type != (int64_t)at::kHalf) fail("dtype must be float32, bfloat16 or float16");
  const Tensor z = at::GradMode::is_enabled() && weight.requires_grad() ? RelposFunction::apply(weight, ids, batch, n, r, s, type)
                                                                        : RelposFunction::run(weight, ids, {batch, n, weight.size(0), r, s, type});
  return z.view(shape);
}
