// Host side of serving from a paged cache: the cached step of sequences of different lengths, and the pages' copies.  Part of
// host.cpp (inside its namespace, behind host_lm.h).
//
// Lengths and tables stay on the device: nothing here waits for it, so a step can be captured and replayed while they change.

struct Pages {   // U, qu, kc, vc
  castle_pages_t t[4];
  int64_t u_pages = 0, pages = 0, heads = 0, page_size = 0, d = 0;
};
Pages check_pages(const Tensor* pools, at::ScalarType dtype, const at::Device& dev, const char* who) {
  Pages p;
  for (int i = 0; i < 4; ++i) {
    const Tensor& t = pools[i];
    need_plain(t, who);
    if (t.dim() != 4 || t.scalar_type() != dtype || t.device() != dev)
      throw std::runtime_error(std::string(who) + ": four (pages, heads, page size, dim_head) pools of the rows' type and device expected");
    if (i == 0) { p.u_pages = t.size(0); p.heads = t.size(1); p.page_size = t.size(2); p.d = t.size(3); }
    if (i == 1) p.pages = t.size(0);
    if (t.size(1) != p.heads || t.size(2) != p.page_size || t.size(3) != p.d || (i > 1 && t.size(0) != p.pages))
      throw std::runtime_error(std::string(who) + ": the pools must have pages of one shape, and those of qu, kc and vc as many of them");
    const bool apart = (t.size(0) <= 1 || t.stride(0) > 0) && (p.heads <= 1 || t.stride(1) > 0);
    if (t.is_neg() || t.requires_grad() || (p.d > 1 && t.stride(3) != 1) || (p.page_size > 1 && t.stride(2) != p.d) || !apart)
      throw std::runtime_error(std::string(who) + ": a pool is written in place: no gradient, a head's rows of a page adjacent, no repeated dimension");
    p.t[i] = {t.data_ptr(), t.stride(0), t.stride(1)};
  }
  if (p.u_pages > std::numeric_limits<int32_t>::max() || p.pages > std::numeric_limits<int32_t>::max() || p.heads > std::numeric_limits<int32_t>::max())
    throw std::runtime_error(std::string(who) + ": at most 2^31 - 1 pages and heads");
  return p;
}

struct Places {   // the tables and lengths of a batch
  Tensor u_table, table, lengths;
  int64_t width = 0;
};
Places check_places(const Tensor& u_table, const Tensor& table, const Tensor& lengths, int64_t batch, const at::Device& dev, const char* who) {
  for (const Tensor* t : {&u_table, &table, &lengths}) {
    need_plain(*t, who);
    if (t->scalar_type() != at::kInt || t->device() != dev) throw std::runtime_error(std::string(who) + ": tables and lengths must be int32 on the pools' device");
  }
  if (u_table.dim() != 2 || table.dim() != 2 || lengths.dim() != 1 || u_table.size(0) != batch || table.size(0) != batch || lengths.size(0) != batch ||
      u_table.size(1) == 0 || table.size(1) == 0)
    throw std::runtime_error(std::string(who) + ": (sequences, pages) tables and a length for each sequence expected");
  Places p;
  auto rows = [](const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); };
  p.u_table = rows(u_table);
  p.table = rows(table);
  p.lengths = lengths.contiguous();
  p.width = std::min(u_table.size(1), table.size(1));
  if (p.width > std::numeric_limits<int32_t>::max()) throw std::runtime_error(std::string(who) + ": the tables are too wide");
  return p;
}

void written(const Tensor* pools, int count) {   // in place, as autograd's check of saved tensors has to know
  for (int i = 0; i < count; ++i)
    if (!pools[i].is_inference()) pools[i].unsafeGetTensorImpl()->bump_version();
}

Tensor paged_core(const castle_tensor_t* news, const Tensor* pools, const Tensor& u_table, const Tensor& table, const Tensor& lengths, int64_t B, int64_t H, int64_t d,
                  at::ScalarType dtype, double scale, Rotary rotary, const at::Device& dev) {
  const char* who = "castle_paged_decode_step";
  const c10::cuda::CUDAGuard guard(dev);
  rotary.fit(dev, d);
  const auto stream = c10::cuda::getCurrentCUDAStream(dev.index());
  const Pages pages = check_pages(pools, dtype, dev, who);
  const Places places = check_places(u_table, table, lengths, B, dev, who);
  need(pages.heads == H && pages.d == d, "castle_paged_decode_step: the pools' heads and dim_head are not the new rows'");
  Tensor out = at::empty({B, H, 1, d}, at::TensorOptions().dtype(dtype).device(dev));
  if (B == 0) return out;
  const castle_problem_t cp{(int32_t)std::min<int64_t>(B, std::numeric_limits<int32_t>::max()), (int32_t)H, 1, (int32_t)d, dtype_code(dtype), (float)scale};
  const castle_tensor_t od = desc(out);
  castle_rotary_t rot{};
  if (rotary.on()) rot = rotary.desc(false);
  const int32_t page_size = (int32_t)std::min<int64_t>(pages.page_size, 1 << 20);
  StreamUse use(stream);
  const Tensor status = status_word(dev.index()), words = use.zero_words(B * H),
               ws = use.scratch(api.paged_decode_workspace_bytes(&cp, page_size, (int32_t)places.width));
  check(api.paged_decode_step(&cp, page_size, (int32_t)pages.u_pages, (int32_t)pages.pages, &news[0], &news[1], &news[2], &news[3], &news[4], &news[5], &pages.t[0],
                              &pages.t[1], &pages.t[2], &pages.t[3], places.u_table.data_ptr<int32_t>(), places.u_table.stride(0), places.table.data_ptr<int32_t>(),
                              places.table.stride(0), (int32_t)places.width, places.lengths.data_ptr<int32_t>(), &od, rotary.on() ? &rot : nullptr,
                              reinterpret_cast<uint32_t*>(words.data_ptr()) + kAmaxWords, ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), stream.stream()), who);
  written(pools, 4);
  return out;
}

// `news` in the operator's order qc, kc, vc, qu, ku, vu; no gradient flows through the cached step.
Tensor paged_decode_step(const Tensor* news, const Tensor* pools, const Tensor& u_table, const Tensor& table, const Tensor& lengths, double scale) {
  const char* who = "castle_paged_decode_step";
  for (int i = 0; i < 6; ++i) need_plain(news[i], who);
  need_type(news[0], who);
  need(news[0].dim() == 4 && news[0].size(2) == 1, "castle_paged_decode_step: (B, H, 1, d) rows expected");
  at::NoGradGuard no_grad;
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(news[0].device());
  Tensor keep[6];
  castle_tensor_t nd[6];
  for (int i = 0; i < 6; ++i) {
    need(news[i].scalar_type() == news[0].scalar_type() && news[i].sizes() == news[0].sizes() && news[i].device() == news[0].device(),
         "castle_paged_decode_step: the new rows must have one shape, type and device");
    keep[i] = aligned_view(news[i]);
    nd[i] = desc(keep[i]);
  }
  return paged_core(nd, pools, u_table, table, lengths, news[0].size(0), news[0].size(1), news[0].size(3), news[0].scalar_type(), scale, Rotary{}, news[0].device());
}

// From the packed projection (B, 1, 6, H, d): (B, 1, H * d).
Tensor paged_decode_packed(const Tensor& packed, const Tensor* pools, const Tensor& u_table, const Tensor& table, const Tensor& lengths, double scale, const Rotary& rotary) {
  const char* who = "castle_paged_decode_step";
  need_plain(packed, who);
  need_type(packed, who);
  need(packed.dim() == 5 && packed.size(1) == 1 && packed.size(2) == 6, "castle_paged_decode_step: a (B, 1, 6, H, d) projection expected");
  at::NoGradGuard no_grad;
  at::AutoDispatchBelowADInplaceOrView below;
  const int64_t B = packed.size(0), H = packed.size(3), d = packed.size(4);
  const c10::cuda::CUDAGuard guard(packed.device());
  const Tensor t = aligned_view(packed);
  castle_tensor_t nd[6];
  for (int i = 0; i < 6; ++i) nd[i] = packed_desc(t, kPackedOrder[i]);
  return paged_core(nd, pools, u_table, table, lengths, B, H, d, packed.scalar_type(), scale, rotary, packed.device()).view({B, 1, H * d});
}

void write_pages(const Tensor* caches, const Tensor* pools, const Tensor& u_table, const Tensor& table, const Tensor& lengths) {
  const char* who = "castle_write_pages";
  for (int i = 0; i < 4; ++i) need_plain(caches[i], who);
  need_type(caches[0], who);
  need(caches[0].dim() == 4, "castle_write_pages: four (B, H, N, d) caches expected");
  const at::Device dev = caches[0].device();
  at::NoGradGuard no_grad;
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t B = caches[0].size(0), H = caches[0].size(1), N = caches[0].size(2), d = caches[0].size(3);
  const Pages pages = check_pages(pools, caches[0].scalar_type(), dev, who);
  const Places places = check_places(u_table, table, lengths, B, dev, who);
  need(pages.heads == H && pages.d == d, "castle_write_pages: the pools' heads and dim_head are not the caches'");
  need(N <= std::numeric_limits<int32_t>::max() && B <= std::numeric_limits<int32_t>::max(), "castle_write_pages: the caches are too large");
  Tensor keep[4];
  castle_tensor_t src[4];
  for (int i = 0; i < 4; ++i) {
    need(caches[i].sizes() == caches[0].sizes() && caches[i].scalar_type() == caches[0].scalar_type() && caches[i].device() == dev,
         "castle_write_pages: the caches must have one shape, type and device");
    if (B == 0 || N == 0) continue;
    keep[i] = aligned_view(caches[i]);
    src[i] = desc(keep[i]);
  }
  if (B == 0 || N == 0) return;
  const castle_problem_t cp{(int32_t)B, (int32_t)H, (int32_t)N, (int32_t)d, dtype_code(caches[0].scalar_type()), 1.f};
  const Tensor status = status_word(dev.index());
  check(api.write_pages(&cp, (int32_t)std::min<int64_t>(pages.page_size, 1 << 20), (int32_t)pages.u_pages, (int32_t)pages.pages, &src[0], &src[1], &src[2], &src[3],
                        &pages.t[0], &pages.t[1], &pages.t[2], &pages.t[3], places.u_table.data_ptr<int32_t>(), places.u_table.stride(0),
                        places.table.data_ptr<int32_t>(), places.table.stride(0), (int32_t)places.width, places.lengths.data_ptr<int32_t>(),
                        status.data_ptr<int32_t>(), c10::cuda::getCurrentCUDAStream(dev.index()).stream()), who);
  written(pools, 4);
}

std::vector<int32_t> page_list(const Tensor& t, int64_t pages, const char* what) {
  if (t.device() != at::kCPU || t.dim() != 1 || (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt))
    throw std::runtime_error(std::string("castle_copy_pages: ") + what + " must be a list of page numbers, on the host");
  const Tensor c = t.to(at::kLong).contiguous();
  const int64_t* v = c.data_ptr<int64_t>();
  std::vector<int32_t> r(c.numel());
  for (size_t i = 0; i < r.size(); ++i) {
    if (v[i] < 0 || v[i] >= pages) throw std::runtime_error(std::string("castle_copy_pages: ") + what + " " + std::to_string(v[i]) + " is not one of " + std::to_string(pages) + " pages");
    r[i] = (int32_t)v[i];
  }
  return r;
}

void copy_pages(const std::vector<Tensor>& pools, const Tensor& source, const Tensor& target) {
  const char* who = "castle_copy_pages";
  need(!pools.empty(), "castle_copy_pages: a pool, or a list of pools, expected");
  const Tensor& first = pools[0];
  std::vector<void*> ptr;
  std::vector<int64_t> stride_page, stride_block;
  need(first.dim() >= 2, "castle_copy_pages: (pages, ...) pools expected");
  const int64_t pages = first.size(0), es = first.element_size();
  need(pages <= std::numeric_limits<int32_t>::max(), "castle_copy_pages: at most 2^31 - 1 pages");
  int64_t page = 1;
  for (int64_t i = 1; i < first.dim(); ++i) page *= first.size(i);
  bool by_head = false;   // pages that are not contiguous as a whole are copied head by head
  auto adjacent = [](const Tensor& t, int64_t from) {
    int64_t want = 1;
    for (int64_t i = t.dim() - 1; i >= from; --i) {
      if (t.size(i) != 1 && t.stride(i) != want) return false;
      want *= t.size(i);
    }
    return true;
  };
  for (const Tensor& t : pools) {
    need_plain(t, who);
    need(t.sizes() == first.sizes() && t.scalar_type() == first.scalar_type() && t.device() == first.device(), "castle_copy_pages: the pools must have one shape, type and device");
    need(!t.is_neg() && !t.requires_grad() && !t.is_complex(), "castle_copy_pages: a pool is written in place: plain real tensors without a gradient expected");
    need((pages <= 1 || t.stride(0) > 0) && (t.size(1) <= 1 || t.stride(1) > 0), "castle_copy_pages: a pool must not repeat its pages or heads");
    if (page > 0 && !adjacent(t, 1)) {
      by_head = true;
      need(adjacent(t, 2), "castle_copy_pages: the rows of a page's heads must be adjacent");
    }
  }
  const std::vector<int32_t> from = page_list(source, pages, "source"), to = page_list(target, pages, "target");
  need(from.size() == to.size(), "castle_copy_pages: a target for each source expected");
  if (from.empty() || page == 0) return;
  const int64_t blocks = by_head ? first.size(1) : 1, block = page / blocks * es;
  for (const Tensor& t : pools) {
    ptr.push_back(t.data_ptr());
    stride_page.push_back(pages > 1 ? t.stride(0) * es : 0);
    stride_block.push_back(by_head ? t.stride(1) * es : 0);
  }
  const c10::cuda::CUDAGuard guard(first.device());
  check(api.copy_pages((int32_t)pools.size(), ptr.data(), stride_page.data(), stride_block.data(), blocks, block, pages, from.data(), to.data(), (int64_t)from.size(),
                       c10::cuda::getCurrentCUDAStream(first.device().index()).stream()), who);
  written(pools.data(), (int)pools.size());
}
