// Host side of the operators around a language model's layers: token lookup, layer norm and the head's cross entropy, each
// with its autograd node.  Part of host.cpp (inside its namespace, behind what it shares with the other operators).
//
// What the kernels take by address is checked here: device, type and shape; tensors whose last dimension is not contiguous, or
// whose negation is still to be done, are copied first.  Operators and nodes compute in the type of their rows, under autocast too.

// (..., dim) as rows that are `stride` elements apart.  A contiguous tensor is taken as it is: views made by the dispatcher cost as much as
// a launch's half, and a token's norm or lookup is little more than its launch.
struct Rows {
  Tensor keep;
  void* data;
  int64_t count, dim, stride;
};
Rows as_rows(const Tensor& t, int64_t rows, int64_t dim) {
  if (!t.is_neg() && t.is_contiguous()) return {t, t.data_ptr(), rows, dim, dim};
  Tensor r = t.resolve_neg().reshape({rows, dim});
  if (dim > 1 && r.stride(1) != 1) r = r.contiguous();
  void* data = r.data_ptr();
  const int64_t stride = rows > 1 ? r.stride(0) : dim;
  return {std::move(r), data, rows, dim, stride};
}
Tensor as_plain(const Tensor& t) { return !t.defined() || (!t.is_neg() && t.is_contiguous()) ? t : t.resolve_neg().contiguous(); }
Tensor as_long(const Tensor& t) { return t.scalar_type() == at::kLong && t.is_contiguous() ? t : t.to(at::kLong).contiguous(); }

// A tensor of its own memory: no wrapper of a batched gradient, of a transform or of a class with a dispatch of its own.
bool own_memory(const Tensor& t) {
  return t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.key_set().has(c10::DispatchKey::Batched) &&
         !t.key_set().has(c10::DispatchKey::FuncTorchBatched) && !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper) &&
         !t.key_set().has(c10::DispatchKey::Functionalize);
}
void need_plain(const Tensor& t, const char* who) {
  if (!t.is_cuda()) throw std::runtime_error(std::string(who) + ": expected CUDA tensors; this package has no CPU path");
  if (!own_memory(t)) throw std::runtime_error(std::string(who) + ": plain strided tensors expected (no tensor class of its own, no vmap or functional transform)");
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), who, ": forward-mode differentiation is not implemented");
}
void need_type(const Tensor& t, const char* who) {
  if (dtype_code(t.scalar_type()) < 0) throw std::runtime_error(std::string(who) + ": bf16, fp16 or fp32 expected");
}
void need_dim(int64_t dim, const char* who) {   // the C ABI takes a row's length as 32 bits
  if (dim > std::numeric_limits<int32_t>::max()) throw std::runtime_error(std::string(who) + ": rows of " + std::to_string(dim) + " elements are not supported");
}
void need_gradient(const Tensor& g, at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev, const char* who) {
  if (g.sizes() != sizes || g.scalar_type() != type || g.device() != dev || !own_memory(g))
    throw std::runtime_error(std::string(who) + ": the gradient's shape, type or device is not the output's");
}
// Under autocast a layer gives rows of its type beside parameters of theirs: these are cast to the rows' type, as autocast casts a projection's
// weight (their gradients come back in their own type).  Elsewhere other types are refused.
Tensor in_type_of(const Tensor& x, const Tensor& t) {
  return t.defined() && t.scalar_type() != x.scalar_type() && t.is_cuda() && own_memory(t) && dtype_code(t.scalar_type()) >= 0 && dtype_code(x.scalar_type()) >= 0 &&
                 at::autocast::is_autocast_enabled(at::kCUDA)
             ? t.to(x.scalar_type())
             : t;
}
Rows restored_rows(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev, int64_t rows, int64_t dim, const char* who) {
  return as_rows(restored(t, sizes, type, dev, who), rows, dim);
}

// ------------------------------------------------------------------------------------------------ token lookup
struct EmbeddingBackward : public Node {
  SavedVariable tokens;
  std::vector<int64_t> token_sizes;
  at::ScalarType token_type = at::kLong, dtype = at::kFloat;
  int64_t vocab = 0, dim = 0, padding = -1;
  double scale = 1;

  std::string name() const override { return "CastleEmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const char* who = "castle_embedding";
    if (grads.empty() || !grads[0].defined()) return {Tensor()};
    const Tensor saved = tokens.unpack();
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
    const Tensor t = restored(saved, token_sizes, token_type, dev, who).contiguous();
    const int64_t n = t.numel();
    std::vector<int64_t> out_sizes = token_sizes;
    out_sizes.push_back(dim);
    need_gradient(grads[0], out_sizes, dtype, dev, who);
    const auto options = at::TensorOptions().dtype(dtype).device(dev);
    if (n == 0) return {at::zeros({vocab, dim}, options)};
    const Rows g = as_rows(grads[0], n, dim);
    const Tensor dw = at::empty({vocab, dim}, options), status = status_word(dev.index());
    StreamUse use(stream);
    const Tensor ws = use.scratch(api.embedding_bwd_workspace_bytes(n, vocab, (int32_t)dim));
    check(api.embedding_bwd(dtype_code(dtype), (int32_t)t.element_size(), n, vocab, (int32_t)dim, t.data_ptr(), padding, g.data, g.stride,
                            (float)scale, dw.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), stream.stream()),
          "castle_embedding_bwd");
    variable_list result{dw};
    refuse_second(result, who, grads[0], *this, 0);   // (it does not depend on the table)
    return result;
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  const char* who = "castle_embedding";
  need_plain(weight, who);
  need_plain(tokens, who);
  need_type(weight, who);
  need(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "castle_embedding: tokens must be int64 or int32");
  need(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "castle_embedding: a (vocabulary, dim) weight expected");
  need(weight.device() == tokens.device(), "castle_embedding: tokens and weight must be on one device");
  const int64_t n = tokens.numel(), vocab = weight.size(0), dim = weight.size(1);
  need_dim(dim, who);
  std::vector<int64_t> sizes = tokens.sizes().vec();
  sizes.push_back(dim);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = weight.device();
    const c10::cuda::CUDAGuard guard(dev);
    y = at::empty(sizes, weight.options().requires_grad(false));
    if (n > 0) {
      const Tensor t = tokens.contiguous(), status = status_word(dev.index());
      const Rows w = as_rows(weight, vocab, dim);
      check(api.embedding_fwd(dtype_code(weight.scalar_type()), (int32_t)t.element_size(), n, vocab, (int32_t)dim, t.data_ptr(), w.data,
                              w.stride, (float)scale, y.data_ptr(), status.data_ptr<int32_t>(),
                              c10::cuda::getCurrentCUDAStream(dev.index()).stream()), "castle_embedding_fwd");
    }
  }
  if (!(at::GradMode::is_enabled() && weight.requires_grad())) return y;
  auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(weight));
  torch::autograd::set_history(y, node);
  node->tokens = SavedVariable(tokens, false);
  node->token_sizes = tokens.sizes().vec();
  node->token_type = tokens.scalar_type();
  node->dtype = weight.scalar_type();
  node->vocab = vocab; node->dim = dim; node->padding = padding; node->scale = scale;
  return y;
}

// ------------------------------------------------------------------------------------------------ layer norm
// Launches on rows; y, dx contiguous.  Weight, bias and the results may be undefined.
void launch_layernorm(const Rows& x, at::ScalarType type, const Tensor& weight, const Tensor& bias, double eps, const Tensor& y, const Tensor& stats,
                      const c10::cuda::CUDAStream& stream) {
  check(api.layernorm_fwd(dtype_code(type), x.count, (int32_t)x.dim, x.data, x.stride, weight.defined() ? weight.data_ptr() : nullptr,
                          bias.defined() ? bias.data_ptr() : nullptr, (float)eps, y.data_ptr(), stats.defined() ? stats.data_ptr<float>() : nullptr,
                          stream.stream()), "castle_layernorm_fwd");
}
void launch_layernorm_bwd(const Rows& dy, const Rows& x, at::ScalarType type, const Tensor& weight, const Tensor& stats, const Tensor& dx, const Tensor& dw,
                          const Tensor& db, const c10::cuda::CUDAStream& stream) {
  StreamUse use(stream);
  const Tensor ws = use.scratch(api.layernorm_bwd_workspace_bytes(x.count, (int32_t)x.dim));
  auto address = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check(api.layernorm_bwd(dtype_code(type), x.count, (int32_t)x.dim, dy.data, dy.stride, x.data, x.stride, address(weight), stats.data_ptr<float>(),
                          address(dx), address(dw), address(db), ws.data_ptr(), ws.numel(), stream.stream()), "castle_layernorm_bwd");
}

struct LayerNormBackward : public Node {   // of x, weight, bias
  SavedVariable x, weight, stats;
  std::vector<int64_t> sizes;
  at::ScalarType dtype = at::kFloat;
  bool has_weight = false;

  std::string name() const override { return "CastleLayerNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(); weight.reset_data(); stats.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const char* who = "castle_layer_norm";
    variable_list result(3);
    if (grads.empty() || !grads[0].defined()) return result;
    const Tensor xs = x.unpack(), ws = has_weight ? weight.unpack() : Tensor(), ss = stats.unpack();
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t dim = sizes.back();
    need_gradient(grads[0], sizes, dtype, dev, who);
    const int64_t rows = grads[0].numel() / dim;
    const auto options = at::TensorOptions().dtype(dtype).device(dev);
    for (int i = 0; i < 3; ++i)
      if (task_should_compute_output(i)) result[i] = rows == 0 ? (i == 0 ? at::empty(sizes, options) : at::zeros({dim}, options))
                                                              : i == 0 ? at::empty(sizes, options) : at::empty({dim}, options);
    if (rows == 0 || !(result[0].defined() || result[1].defined() || result[2].defined())) return result;
    const Tensor w = has_weight ? as_plain(restored(ws, {dim}, dtype, dev, who)) : Tensor();
    launch_layernorm_bwd(as_rows(grads[0], rows, dim), restored_rows(xs, sizes, dtype, dev, rows, dim, who), dtype, w,
                         restored_contiguous(ss, {rows, 2}, at::kFloat, dev, who), result[0], result[1], result[2], c10::cuda::getCurrentCUDAStream(dev.index()));
    refuse_second(result, who, grads[0], *this, 2);
    return result;
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& own_weight, const Tensor& own_bias, double eps) {
  const char* who = "castle_layer_norm";
  const Tensor weight = in_type_of(x, own_weight), bias = in_type_of(x, own_bias);
  need_plain(x, who);
  need_type(x, who);
  need(x.dim() >= 1 && x.size(-1) > 0, "castle_layer_norm: (..., dim) rows expected");
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  need_dim(dim, who);
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    need_plain(*t, who);
    need(t->dim() == 1 && t->size(0) == dim && t->scalar_type() == x.scalar_type() && t->device() == x.device(),
         "castle_layer_norm: weight and bias must be (dim) tensors of the input's type and device");
  }
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()));
  Tensor y, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto options = x.options().requires_grad(false);
    y = at::empty(x.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    if (grad) stats = at::empty({rows, 2}, options.dtype(at::kFloat));
    if (rows > 0)
      launch_layernorm(as_rows(x, rows, dim), x.scalar_type(), as_plain(weight), as_plain(bias), eps, y, stats, c10::cuda::getCurrentCUDAStream(dev.index()));
  }
  if (!grad) return y;
  auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
  torch::autograd::set_history(y, node);
  node->x = SavedVariable(x, false);
  node->has_weight = weight.defined();
  if (node->has_weight) node->weight = SavedVariable(weight, false);
  node->stats = SavedVariable(stats, false);
  node->sizes = x.sizes().vec();
  node->dtype = x.scalar_type();
  return y;
}

// ------------------------------------------------------------------------------------------------ cross entropy of a linear head
struct LinearCrossEntropyBackward : public Node {   // of x, weight
  SavedVariable x, weight, targets, lse;
  std::vector<int64_t> x_sizes, target_sizes;
  at::ScalarType dtype = at::kFloat, target_type = at::kLong;
  int64_t vocab = 0, ignore = -100;
  int reduction = CASTLE_REDUCE_MEAN;

  std::string name() const override { return "CastleLinearCrossEntropyBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &weight, &targets, &lse}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const char* who = "castle_linear_cross_entropy";
    variable_list result(2);
    if (grads.empty() || !grads[0].defined()) return result;
    const Tensor xs = x.unpack(), ws = weight.unpack(), ts = targets.unpack(), ls = lse.unpack();
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
    const int64_t dim = x_sizes.back();
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < x_sizes.size(); ++i) rows *= x_sizes[i];
    const bool each = reduction == CASTLE_REDUCE_NONE;
    need_gradient(grads[0], each ? at::IntArrayRef(target_sizes) : at::IntArrayRef(), at::kFloat, dev, who);
    const auto options = at::TensorOptions().dtype(dtype).device(dev);
    if (rows == 0) {
      if (task_should_compute_output(0)) result[0] = at::empty(x_sizes, options);
      if (task_should_compute_output(1)) result[1] = at::zeros({vocab, dim}, options);
      return result;
    }
    if (task_should_compute_output(0)) result[0] = at::empty(x_sizes, options);
    if (task_should_compute_output(1)) result[1] = at::empty({vocab, dim}, options);
    const Rows xr = restored_rows(xs, x_sizes, dtype, dev, rows, dim, who), w = restored_rows(ws, {vocab, dim}, dtype, dev, vocab, dim, who);
    const Tensor t = as_long(restored(ts, target_sizes, target_type, dev, who)), l = restored_contiguous(ls, {rows}, at::kFloat, dev, who), g = as_plain(grads[0]),
                 status = status_word(dev.index());
    StreamUse use(stream);
    const Tensor scratch = use.scratch(api.linear_ce_workspace_bytes(dtype_code(dtype), rows, (int32_t)dim, vocab, 1));
    check(api.linear_ce_bwd(dtype_code(dtype), rows, (int32_t)dim, vocab, xr.data, xr.stride, w.data, w.stride, t.data_ptr<int64_t>(), ignore,
                            reduction, l.data_ptr<float>(), g.data_ptr<float>(), result[0].defined() ? result[0].data_ptr() : nullptr,
                            result[1].defined() ? result[1].data_ptr() : nullptr, scratch.data_ptr(), scratch.numel(), status.data_ptr<int32_t>(), stream.stream()),
          "castle_linear_ce_bwd");
    refuse_second(result, who, grads[0], *this, 2);
    return result;
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& own_weight, const Tensor& targets, int64_t ignore, int reduction) {
  const char* who = "castle_linear_cross_entropy";
  const Tensor weight = in_type_of(x, own_weight);
  for (const Tensor* t : {&x, &weight, &targets}) need_plain(*t, who);
  need_type(x, who);
  need(x.dim() >= 1 && x.size(-1) > 0 && weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) == x.size(-1),
       "castle_linear_cross_entropy: (..., dim) inputs and a (vocabulary, dim) weight expected");
  need(weight.scalar_type() == x.scalar_type() && weight.device() == x.device() && targets.device() == x.device(),
       "castle_linear_cross_entropy: input and weight must have one type, and all tensors one device");
  need(targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt, "castle_linear_cross_entropy: targets must be int64 or int32");
  need(targets.sizes() == x.sizes().slice(0, x.dim() - 1), "castle_linear_cross_entropy: a target for each row of the input expected");
  const int64_t dim = x.size(-1), rows = targets.numel(), vocab = weight.size(0);
  need_dim(dim, who);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad()), each = reduction == CASTLE_REDUCE_NONE;
  Tensor loss, lse;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
    const auto options = at::TensorOptions().dtype(at::kFloat).device(dev);
    if (rows == 0 && !each) loss = at::full({}, reduction == CASTLE_REDUCE_MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, options);
    else loss = each ? at::empty(targets.sizes(), options) : at::empty({}, options);
    lse = at::empty({rows}, options);
    if (rows > 0) {
      const Rows xr = as_rows(x, rows, dim), w = as_rows(weight, vocab, dim);
      const Tensor t = as_long(targets), status = status_word(dev.index());
      StreamUse use(stream);
      const Tensor scratch = use.scratch(api.linear_ce_workspace_bytes(dtype_code(x.scalar_type()), rows, (int32_t)dim, vocab, 0));
      check(api.linear_ce_fwd(dtype_code(x.scalar_type()), rows, (int32_t)dim, vocab, xr.data, xr.stride, w.data, w.stride,
                              t.data_ptr<int64_t>(), ignore, reduction, loss.data_ptr<float>(), lse.data_ptr<float>(), scratch.data_ptr(), scratch.numel(),
                              status.data_ptr<int32_t>(), stream.stream()), "castle_linear_ce_fwd");
    }
  }
  if (!grad) return loss;
  auto node = std::shared_ptr<LinearCrossEntropyBackward>(new LinearCrossEntropyBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, weight));
  torch::autograd::set_history(loss, node);
  node->x = SavedVariable(x, false);
  node->weight = SavedVariable(weight, false);
  node->targets = SavedVariable(targets, false);
  node->lse = SavedVariable(lse, false);
  node->x_sizes = x.sizes().vec();
  node->target_sizes = targets.sizes().vec();
  node->dtype = x.scalar_type();
  node->target_type = targets.scalar_type();
  node->vocab = vocab;
  node->ignore = ignore;
  node->reduction = reduction;
  return loss;
}
