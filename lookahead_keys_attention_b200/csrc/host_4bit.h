// Host side of the products with weights of 4 bits.  Part of host.cpp (inside its namespace, behind `product`).

struct Codes {   // a weight's, as the kernels take them
  Tensor codes, scales, zeros;
  int64_t N = 0, K = 0, group = 0;
};
Codes check_codes(const Tensor& codes, const Tensor& scales, const Tensor& zeros, int64_t K, int64_t group, at::ScalarType dtype, const at::Device& dev) {
  const char* who = "castle_linear_4bit";
  need_plain(codes, who);
  need(scales.defined() && scales.dim() == 2 && scales.size(0) > 0, "castle_linear_4bit: (out, groups) scales expected");
  need(codes.dim() == 2 && codes.scalar_type() == at::kInt && codes.size(0) == (scales.size(0) + 15) / 16 && codes.size(1) == (K + 255) / 256 * 512,
       "castle_linear_4bit: codes of castle_pack_4bit for weights of the rows' length and as many as the scales' expected");
  need(group >= 32 && group <= (1 << 24) && (group & (group - 1)) == 0, "castle_linear_4bit: the group size must be a power of two from 32 up");
  Codes c;
  c.N = scales.size(0); c.K = K; c.group = group;
  const std::array<int64_t, 2> sizes{c.N, (K + group - 1) / group};
  for (const Tensor* t : {&scales, &zeros}) {
    if (!t->defined()) continue;
    need_plain(*t, who);
    need(t->sizes() == at::IntArrayRef(sizes) && t->scalar_type() == dtype && t->device() == dev,
         "castle_linear_4bit: scales and zero points must be (out, groups) tensors of the rows' type and device");
    need(!(t->requires_grad() && at::GradMode::is_enabled()), "castle_linear_4bit: scales and zero points have no gradient");
  }
  need(codes.device() == dev, "castle_linear_4bit: codes and rows must be on one device");
  c.codes = aligned_contiguous(codes); c.scales = as_plain(scales); c.zeros = as_plain(zeros);
  return c;
}

// The weights at full width.
Tensor expand_4bit(const Codes& c, at::ScalarType dtype, const at::Device& dev) {
  const int64_t unit = 16 / (int64_t)c10::elementSize(dtype), ld = (c.K + unit - 1) / unit * unit;
  const Tensor w = at::empty({c.N, ld}, at::TensorOptions().dtype(dtype).device(dev));
  check(api.expand_4bit(dtype_code(dtype), (int32_t)c.K, c.N, (int32_t)c.group, c.codes.data_ptr(), c.scales.data_ptr(), c.zeros.defined() ? c.zeros.data_ptr() : nullptr,
                        w.data_ptr(), ld, c10::cuda::getCurrentCUDAStream(dev.index()).stream()), "castle_expand_4bit");
  return w.narrow(1, 0, c.K);
}

struct Linear4bitBackward : public Node {   // of x: the weights are frozen
  SavedVariable codes, scales, zeros;
  std::vector<int64_t> x_sizes;
  at::ScalarType dtype = at::kFloat;
  int64_t out_features = 0, group = 0;
  bool has_zeros = false;

  std::string name() const override { return "CastleLinear4bitBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&codes, &scales, &zeros}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const char* who = "castle_linear_4bit";
    variable_list result(1);
    if (grads.empty() || !grads[0].defined()) return result;
    const Tensor cs = codes.unpack(), ss = scales.unpack(), zs = has_zeros ? zeros.unpack() : Tensor();
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);   // the products keep the rows' type
    const at::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    std::vector<int64_t> y_sizes = x_sizes;
    y_sizes.back() = out_features;
    need_gradient(grads[0], y_sizes, dtype, dev, who);
    const int64_t K = x_sizes.back(), rows = grads[0].numel() / out_features;
    if (rows == 0) {
      result[0] = at::empty(x_sizes, grads[0].options());
      return result;
    }
    const Codes c = check_codes(restored(cs, {(out_features + 15) / 16, (K + 255) / 256 * 512}, at::kInt, dev, who), ss, zs, K, group, dtype, dev);
    result[0] = product(1, as_plain(grads[0]).view({rows, out_features}), expand_4bit(c, dtype, dev), rows).view(x_sizes);
    refuse_second(result, who, grads[0], *this, 0);   // (it does not depend on x)
    return result;
  }
};

// Whether 9 to 32 rows of 16 bits go through the codes rather than through tiles, by what either takes: the one by the number of weights (us, bf16: 16 x 4096 ->
// 16384 22.6, 32 x 4096 -> 16384 46.7, 16 x 4096 -> 4096 10.8, 32 x 4096 -> 4096 17.6, 32 x 512 -> 2048 5.9) and, where the rows are wide, what their share of a CTA's
// shared memory costs (12 x 16384 -> 1024 20.0, by tiles 12), the other by its plan.
bool few_rows(int64_t rows, int64_t K, int64_t N) {
  const double weights = 1e-6 * (double)K * (double)N, wide = 7e-4 * (double)std::max<int64_t>(0, K - 4096);
  const double codes = (rows <= 16 ? 3.3 + 0.29 * weights : 5.0 + 0.64 * weights) + wide;
  return codes <= castle::linear_4bit_tile_plan(rows, K, N).us;
}

// Rows of 32 bits go through the codes ten at a time, or five where ten are wider than two CTAs' shared memory (us: 10 x 4096 -> 4096 18.9, 5 14.1, 10 x 8136 -> 5307
// 111, 5 31.3), or through the weights at full width, whose making and products take some 12 + 5.5 for each million of them up to 64 rows (in turns / at full width:
// 45 x 4096 -> 4096 88 / 121, 64 x 1000 -> 50021 167 / 251, 30 x 8136 -> 5307 180 / 277, 45 x 1024 -> 4096 44 / 29).  The latter is a line through few shapes: 45 x 4096 -> 1024
// take 63 where it says 35, 45 x 8136 -> 5307 309 where it says 250, a little less than nine turns.
constexpr int64_t kWholeF32 = 4096;
bool few_rows_f32(int64_t rows, int64_t turns, int64_t K, int64_t N) {
  const double weights = 1e-6 * (double)K * (double)N;
  const double turn = K <= kWholeF32 ? 5.5 + 0.0021 * (double)K + 0.38 * weights : 4.0 + 0.0018 * (double)K + 0.23 * weights;
  return rows <= 10 || (double)turns * turn <= 12.0 + 5.5 * weights;
}

Tensor linear_4bit(const Tensor& x, const Tensor& codes, const Tensor& own_scales, const Tensor& own_zeros, int64_t group) {
  const char* who = "castle_linear_4bit";
  need_plain(x, who);
  need_type(x, who);
  need(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) <= (1 << 24), "castle_linear_4bit: (..., in) rows expected");
  const int64_t K = x.size(-1), rows = x.numel() / K;
  const Tensor scales = in_type_of(x, own_scales), zeros = in_type_of(x, own_zeros);
  const at::Device dev = x.device();
  const auto dtype = x.scalar_type();
  std::vector<int64_t> sizes = x.sizes().vec();
  Tensor y;
  Codes c;
  {
    const c10::cuda::CUDAGuard guard(dev);
    c = check_codes(codes, scales, zeros, K, group, dtype, dev);
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
    const at::NoGradGuard no_grad;
    sizes.back() = c.N;
    // The rows of a few tokens go through the codes, fp32 ones as many at a time as the kernel takes; more rows of 16 bits through tiles of weights that
    // are unpacked on their way to the tensor cores, and of 32 through the weights at full width (their products are FMA).
    const int64_t most = dtype != at::kFloat ? 32 : K <= kWholeF32 ? 10 : 5, turns = (rows + most - 1) / most, each = turns > 0 ? (rows + turns - 1) / turns : 0;
    const bool few = dtype == at::kFloat ? few_rows_f32(rows, turns, K, c.N) : rows <= 8 || (turns == 1 && few_rows(rows, K, c.N));
    if (rows == 0) {
      y = at::empty(sizes, x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    } else if (few && api.linear_4bit_fits(dtype_code(dtype), (int32_t)each, (int32_t)K)) {
      y = at::empty(sizes, x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
      const Rows r = as_rows(x, rows, K);
      const int64_t es = x.element_size();
      const Tensor status = status_word(dev.index());
      for (int64_t i = 0; i < rows; i += each)
        check(api.linear_4bit(dtype_code(dtype), (int32_t)std::min(each, rows - i), (int32_t)K, c.N, (int32_t)group, static_cast<char*>(r.data) + i * r.stride * es, r.stride,
                              c.codes.data_ptr(), c.scales.data_ptr(), c.zeros.defined() ? c.zeros.data_ptr() : nullptr, static_cast<char*>(y.data_ptr()) + i * c.N * es, status.data_ptr<int32_t>(),
                              c10::cuda::getCurrentCUDAStream(dev.index()).stream()), who);
    } else if (dtype != at::kFloat) {
      y = at::empty(sizes, x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
      Rows r = as_rows(x, rows, K);
      if (reinterpret_cast<uintptr_t>(r.data) % 16 != 0 || r.stride % 8 != 0 || (r.stride < K && rows > 1)) {   // rows at 16-byte boundaries, one behind the other
        const int64_t ld = (K + 7) / 8 * 8;
        const Tensor t = at::empty({rows, ld}, x.options().requires_grad(false).memory_format(c10::nullopt));
        t.narrow(1, 0, K).copy_(r.keep.reshape({rows, K}));
        r = {t, t.data_ptr(), rows, K, ld};
      }
      const Tensor status = status_word(dev.index());
      check(api.linear_4bit_tile(dtype_code(dtype), rows, (int32_t)K, c.N, (int32_t)group, r.data, r.stride, c.codes.data_ptr(), c.scales.data_ptr(),
                                 c.zeros.defined() ? c.zeros.data_ptr() : nullptr, y.data_ptr(), status.data_ptr<int32_t>(),
                                 c10::cuda::getCurrentCUDAStream(dev.index()).stream()), who);
    } else {
      y = product(0, as_plain(x).view({rows, K}), expand_4bit(c, dtype, dev), rows).view(sizes);
    }
  }
  if (!(at::GradMode::is_enabled() && x.requires_grad())) return y;
  auto node = std::shared_ptr<Linear4bitBackward>(new Linear4bitBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(y, node);
  node->codes = SavedVariable(codes, false);
  node->scales = SavedVariable(scales, false);
  node->has_zeros = zeros.defined();
  if (node->has_zeros) node->zeros = SavedVariable(zeros, false);
  node->x_sizes = x.sizes().vec();
  node->dtype = dtype;
  node->out_features = c.N;
  node->group = group;
  return y;
}
