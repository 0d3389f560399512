// PyTorch operators of the serving path (norm and rotation, paged append, plan, paged attention) on top of the C ABI.
// Included by torch_op.cpp, whose helpers it uses.
#pragma once

using OptAxes = std::optional<std::vector<int64_t>>;

// Dense outputs keep the layout of their input, others are contiguous.
Tensor empty_dense_as(const Tensor& t) {
  return t.is_non_overlapping_and_dense() ? empty_as(t) : empty_on(t.sizes(), t.scalar_type(), t);
}

bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

void check_16bit_cuda(const Tensor& t) {
  FB_ASSERT(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "Only support fp16 and bf16");
  FB_ASSERT(t.is_cuda(), "tensors lie in device memory");
}
void check_beside(const Tensor& t, const Tensor& like) { FB_ASSERT(t.device() == like.device(), "all tensors lie on one device"); }

// ---- norm and rotation ------------------------------------------------------------------------------------------
struct RopeArgs {
  Tensor positions, inv_freq, q_weight, k_weight;  // undefined where absent
  OptAxes axes;
  bool interleaved;
  double eps;
};

// The parameter block without tensors q and k.  rows of (B, S): the tokens.
void fill_rope(fb_rope_params& p, const RopeArgs& a, const Tensor& like, int64_t B, int64_t S, int64_t D) {
  FB_ASSERT(D >= 1 && D <= 128, "norm_rope supports head dimensions up to 128");
  FB_ASSERT(B <= 0x7fff0000 && S <= 0x7fff0000 && (S == 0 || B <= 0x7fff0000 / S), "too many tokens");
  p.B = (int32_t)B;
  p.S = (int32_t)S;
  p.D = (int32_t)D;
  p.dtype = dtype_code(like.scalar_type());
  p.eps = (float)a.eps;
  p.interleaved = a.interleaved ? 1 : 0;
  p.naxes = 1;
  p.position_bits = 32;
  p.status = status_ptr();
  FB_ASSERT(a.positions.defined() == a.inv_freq.defined(), "positions and inv_freq must be given together");
  if (a.inv_freq.defined()) {
    const Tensor &f = a.inv_freq, &pos = a.positions;
    check_beside(f, like);
    check_beside(pos, like);
    FB_ASSERT(f.dim() == 1 && (f.scalar_type() == at::kFloat || f.scalar_type() == at::kDouble) && f.is_contiguous(),
              "inv_freq holds fp32 or fp64 frequencies, one per rotated pair");
    FB_ASSERT(2 * f.numel() <= D, "inv_freq has more frequencies than the head has pairs");
    FB_ASSERT(is_index(pos), "positions are int32 or int64");
    p.rot = (int32_t)(2 * f.numel());
    p.inv_freq = f.data_ptr();
    p.freq_dtype = f.scalar_type() == at::kDouble ? FB_DTYPE_F64 : FB_DTYPE_F32;
    p.position_bits = pos.scalar_type() == at::kLong ? 64 : 32;
    const int64_t lead = a.axes ? 1 : 0;  // dimensions in front of ([batch,] row)
    FB_ASSERT(pos.dim() == lead + 1 || pos.dim() == lead + 2, "positions are (S), (B | 1, S), or with axes (A, S), (A, B | 1, S)");
    FB_ASSERT(pos.size(-1) == S && (pos.dim() == lead + 1 || pos.size(-2) == 1 || pos.size(-2) == B), "positions do not fit the tokens");
    p.position_stride[2] = pos.stride(-1);
    p.position_stride[1] = pos.dim() == lead + 2 && pos.size(-2) > 1 ? pos.stride(-2) : 0;
    if (a.axes) {
      FB_ASSERT(pos.size(0) >= 1 && pos.size(0) <= 4, "one to four position axes");
      FB_ASSERT((int64_t)a.axes->size() == f.numel(), "axes names the axis of every rotated pair");
      p.naxes = (int32_t)pos.size(0);
      p.position_stride[0] = pos.stride(0);
      for (size_t i = 0; i < a.axes->size(); ++i) {
        const int64_t x = (*a.axes)[i];
        FB_ASSERT(x >= 0 && x < p.naxes, "axes names an axis that positions does not have");
        p.pair_axis[i] = (uint8_t)x;
      }
    }
    p.positions = p.rot ? pos.data_ptr() : nullptr;
  } else {
    FB_ASSERT(!a.axes, "axes without positions");
  }
  FB_ASSERT(a.eps >= 0.0 && std::isfinite(a.eps), "eps is a finite number that is not negative");
  for (const Tensor* w : {&a.q_weight, &a.k_weight}) {
    if (!w->defined()) continue;
    check_beside(*w, like);
    FB_ASSERT(w->dim() == 1 && w->numel() == D && w->is_contiguous(), "norm weights hold one value per column of a head");
    FB_ASSERT(w->scalar_type() == at::kHalf || w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat,
              "norm weights are fp16, bf16 or fp32");
    p.weight_dtype = dtype_code(w->scalar_type());
  }
  FB_ASSERT(!a.q_weight.defined() || !a.k_weight.defined() || a.q_weight.scalar_type() == a.k_weight.scalar_type(),
            "both norm weights have the same type");
  p.q_weight = a.q_weight.defined() ? a.q_weight.data_ptr() : nullptr;
  p.k_weight = a.k_weight.defined() ? a.k_weight.data_ptr() : nullptr;
}

constexpr int64_t kMaxRopeHeads = 65536;
void check_rope_qk(const Tensor& q, const Tensor& k) {
  FB_ASSERT(q.dim() == 4 && (!k.defined() || k.dim() == 4), "q and k are (batch, seqlen, nheads, headdim)");
  check_16bit_cuda(q);
  if (k.defined()) {
    check_beside(k, q);
    FB_ASSERT(k.scalar_type() == q.scalar_type(), "All tensors must have the same type");
    FB_ASSERT(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3), "q and k differ in more than their heads");
  }
  FB_ASSERT(q.size(2) <= kMaxRopeHeads && (!k.defined() || q.size(2) + k.size(2) <= kMaxRopeHeads), "too many heads");
}

// (q_out, k_out); k may be undefined
std::tuple<Tensor, Tensor> rope_forward(const Tensor& q, const Tensor& k, const RopeArgs& a) {
  check_device_status();
  check_rope_qk(q, k);
  c10::cuda::CUDAGuard guard(q.device());
  fb_rope_params p{};
  fill_rope(p, a, q, q.size(0), q.size(1), q.size(3));
  Tensor qo = empty_dense_as(q), ko = k.defined() ? empty_dense_as(k) : Tensor();
  p.Hq = (int32_t)q.size(2);
  p.q = q.data_ptr();
  strides_bhs(q, p.q_stride);
  p.q_out = qo.data_ptr();
  strides_bhs(qo, p.q_out_stride);
  if (k.defined()) {
    p.Hk = (int32_t)k.size(2);
    p.k = k.data_ptr();
    strides_bhs(k, p.k_stride);
    p.k_out = ko.data_ptr();
    strides_bhs(ko, p.k_out_stride);
  }
  if ((int64_t)p.B * p.S * (p.Hq + p.Hk) > 0) check_rc(fb_norm_rope(&p, at::cuda::getCurrentCUDAStream().stream()), "fb_norm_rope");
  return {qo, ko};
}

// A tensor whose gradient is taken: itself where the backward reads it (norm weights), else its layout alone.
struct RopeSource {
  Tensor x;  // undefined where it is not read
  std::vector<int64_t> sizes, strides;  // empty without the tensor; strides empty where its gradient is contiguous
};
RopeSource rope_source(const Tensor& x, bool read) {
  if (!x.defined()) return {};
  return {read ? x : Tensor(), x.sizes().vec(), x.is_non_overlapping_and_dense() ? x.strides().vec() : std::vector<int64_t>()};
}
Tensor empty_dense_as(const RopeSource& s, const Tensor& like) {
  if (s.strides.empty()) return empty_on(s.sizes, like.scalar_type(), like);
  if (c10::impl::dispatch_mode_enabled()) return at::empty_strided(s.sizes, s.strides, like.options());
  return Tensor(at::detail::empty_strided_cuda(s.sizes, s.strides, like.scalar_type(), like.device()));
}

// Gradients of (q, k, q_weight, k_weight); dq_out or dk_out may be undefined: that tensor is left out.
std::tuple<Tensor, Tensor, Tensor, Tensor> rope_backward(Tensor dqo, Tensor dko, const RopeSource& q, const RopeSource& k, at::ScalarType type,
                                                         const RopeArgs& a, bool want_qw, bool want_kw) {
  check_device_status();
  Tensor dq, dk, dqw, dkw;
  if (!dqo.defined() && !dko.defined()) return {dq, dk, dqw, dkw};
  const Tensor& like = dqo.defined() ? dqo : dko;
  c10::cuda::CUDAGuard guard(like.device());
  fb_rope_params p{};
  FB_ASSERT(like.scalar_type() == type, "");
  fill_rope(p, a, like, q.sizes[0], q.sizes[1], q.sizes[3]);
  auto take = [&](Tensor& g, const RopeSource& s, const Tensor& w, bool want_w, int32_t& H, const void*& xp, int64_t(&xs)[3], const void*& gp,
                  int64_t(&gs)[3], Tensor& dx, void*& dxp, int64_t(&dxs)[3], Tensor& dw, void*& dwp) {
    if (!g.defined() || s.sizes.empty()) return;
    FB_ASSERT(g.sizes() == s.sizes && g.scalar_type() == type && g.device() == like.device(), "");
    if (g.stride(-1) != 1) g = g.contiguous();
    H = (int32_t)s.sizes[2];
    if (s.x.defined()) {
      FB_ASSERT(s.x.device() == g.device(), "");
      xp = s.x.data_ptr();
      strides_bhs(s.x, xs);
    }
    gp = g.data_ptr();
    strides_bhs(g, gs);
    dx = empty_dense_as(s, g);
    dxp = dx.data_ptr();
    strides_bhs(dx, dxs);
    if (want_w && w.defined()) {
      dw = empty_on(w.sizes(), w.scalar_type(), w);
      dwp = dw.data_ptr();
    }
  };
  take(dqo, q, a.q_weight, want_qw, p.Hq, p.q, p.q_stride, p.dq_out, p.dq_out_stride, dq, p.dq, p.dq_stride, dqw, p.dq_weight);
  take(dko, k, a.k_weight, want_kw, p.Hk, p.k, p.k_stride, p.dk_out, p.dk_out_stride, dk, p.dk, p.dk_stride, dkw, p.dk_weight);
  if ((int64_t)p.B * p.S * (p.Hq + p.Hk) == 0) {
    for (Tensor* t : {&dqw, &dkw})
      if (t->defined()) t->zero_();
    return {dq, dk, dqw, dkw};
  }
  Tensor ws;
  if (const size_t need = fb_norm_rope_bwd_workspace_bytes(&p)) {
    ws = workspace(need, like);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
  }
  check_rc(fb_norm_rope_bwd(&p, at::cuda::getCurrentCUDAStream().stream()), "fb_norm_rope_bwd");
  return {dq, dk, dqw, dkw};
}

Tensor or_undefined(const OptTensor& t) { return t ? *t : Tensor(); }
Tensor unit_rows_or_undefined(const OptTensor& t) { return t ? unit_rows(*t) : Tensor(); }
Tensor contiguous_or_undefined(const OptTensor& t) { return t ? t->contiguous() : Tensor(); }

struct NormRopeNode : torch::autograd::Function<NormRopeNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q_, const OptTensor& k_,
                                                const OptTensor& positions, const OptTensor& inv_freq, const OptTensor& q_weight,
                                                const OptTensor& k_weight, const std::vector<int64_t>& axes, bool has_axes,
                                                bool interleaved, double eps) {
    const Tensor q = unit_rows(q_), k = unit_rows_or_undefined(k_);
    const RopeArgs a = {or_undefined(positions), contiguous_or_undefined(inv_freq), contiguous_or_undefined(q_weight),
                        contiguous_or_undefined(k_weight), has_axes ? OptAxes(axes) : std::nullopt, interleaved, eps};
    auto [qo, ko] = rope_forward(q, k, a);
    ctx->set_materialize_grads(false);
    // (a tensor without a weight is not read again: kept, it would hold on to the projection it is a slice of)
    const RopeSource qs = rope_source(q, a.q_weight.defined()), ks = rope_source(k, a.k_weight.defined());
    ctx->save_for_backward({qs.x, ks.x, a.positions, a.inv_freq, a.q_weight, a.k_weight});
    ctx->saved_data["q_sizes"] = qs.sizes;
    ctx->saved_data["q_strides"] = qs.strides;
    ctx->saved_data["k_sizes"] = ks.sizes;
    ctx->saved_data["k_strides"] = ks.strides;
    ctx->saved_data["type"] = (int64_t)q.scalar_type();
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["has_axes"] = has_axes;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    if (!k.defined()) return {qo};
    return {qo, ko};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const bool again = at::GradMode::is_enabled();  // (create_graph)
    at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const RopeArgs a = {s[2], s[3], s[4], s[5],
                        ctx->saved_data["has_axes"].toBool() ? OptAxes(ctx->saved_data["axes"].toIntVector()) : std::nullopt,
                        ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble()};
    const RopeSource q = {s[0], ctx->saved_data["q_sizes"].toIntVector(), ctx->saved_data["q_strides"].toIntVector()};
    const RopeSource k = {s[1], ctx->saved_data["k_sizes"].toIntVector(), ctx->saved_data["k_strides"].toIntVector()};
    // (edges are counted over the tensors that were given)
    const int w0 = 1 + (k.sizes.empty() ? 0 : 1) + (s[2].defined() ? 1 : 0) + (s[3].defined() ? 1 : 0);
    const bool want_qw = s[4].defined() && ctx->needs_input_grad(w0);
    const bool want_kw = s[5].defined() && ctx->needs_input_grad(w0 + (s[4].defined() ? 1 : 0));
    auto [dq, dk, dqw, dkw] =
        rope_backward(grads[0], grads.size() > 1 ? grads[1] : Tensor(), q, k, (at::ScalarType)ctx->saved_data["type"].toInt(), a, want_qw, want_kw);
    if (again) {  // there is no second derivative: to ask for it is an error, not a zero
      // (with the edges of this node, so that a search for the inputs passes it)
      auto edges = torch::autograd::get_current_node()->next_edges();
      const auto stop = std::make_shared<torch::autograd::Error>("norm_rope_func cannot be differentiated twice", std::move(edges));
      for (Tensor* t : {&dq, &dk, &dqw, &dkw})
        if (t->defined()) torch::autograd::create_gradient_edge(*t, stop);
    }
    return {dq, dk, Tensor(), Tensor(), dqw, dkw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, OptTensor> norm_rope(const Tensor& q, const OptTensor& k, const OptTensor& positions, const OptTensor& inv_freq,
                                        const OptTensor& q_weight, const OptTensor& k_weight, const OptAxes& axes, bool interleaved,
                                        double eps) {
  refuse_tangents(q, k, q_weight, k_weight, inv_freq);
  FB_ASSERT(!wants_grad(inv_freq), "inv_freq is a constant: it gets no gradient");
  if (at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k) || wants_grad(q_weight) || wants_grad(k_weight))) {
    auto out = NormRopeNode::apply(q, k, positions, inv_freq, q_weight, k_weight, axes ? *axes : std::vector<int64_t>(),
                                   axes.has_value(), interleaved, eps);
    return {out[0], out.size() > 1 ? OptTensor(out[1]) : std::nullopt};
  }
  const RopeArgs a = {or_undefined(positions), contiguous_or_undefined(inv_freq), contiguous_or_undefined(q_weight),
                      contiguous_or_undefined(k_weight), axes, interleaved, eps};
  auto [qo, ko] = rope_forward(unit_rows(q), unit_rows_or_undefined(k), a);
  return {qo, defined_or_none(ko)};
}

// ---- paged cache ------------------------------------------------------------------------------------------------
template <typename... Ts>
void refuse_grads(const Ts&... t) {
  auto needs = [](const OptTensor& x) { return wants_grad(x); };
  FB_ASSERT(!at::GradMode::is_enabled() || !(needs(t) || ...), "the paged operators are for inference: no input may require a gradient");
}

// a cache of (num_pages, page_size, heads, columns), addressed where it lies
void check_cache(const Tensor& c, const Tensor& like, int64_t pages, int64_t page_size, int64_t heads, int64_t cols) {
  check_beside(c, like);
  FB_ASSERT(c.scalar_type() == like.scalar_type(), "All tensors must have the same type");
  FB_ASSERT(c.dim() == 4 && c.size(0) == pages && c.size(1) == page_size && c.size(2) == heads && c.size(3) == cols,
            "caches are (pages, page size, heads, columns)");
  FB_ASSERT(c.stride(3) == 1 || cols == 1, "the columns of a cache are contiguous");
}
// the same of one that is written
void check_written(const Tensor& c) {
  FB_ASSERT(at::has_internal_overlap(c) != at::MemOverlap::Yes, "a cache that is written may not be an expanded view");
}
void cache_strides(const Tensor& c, int64_t (&out)[3]) {
  for (int i = 0; i < 3; ++i) out[i] = c.stride(i);
}
// the same beside what is read: rows that lie in a cache may be those that another token overwrites
void check_apart(const Tensor& cache, const Tensor& read) {
  if (!read.defined() || !cache.is_alias_of(read)) return;
  auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  FB_ASSERT(read.numel() == 0 || end(read) <= cache.data_ptr() || end(cache) <= read.data_ptr(), "what is appended may not lie in a cache itself: copy it first");
}
// Caches of one call that certainly share elements (views that interleave, like keys beside values in one pool, do not).
void check_distinct(const Tensor& a, const Tensor& b) {
  const at::MemOverlapStatus o = at::get_overlap_status(a, b);
  FB_ASSERT(o != at::MemOverlapStatus::Full && o != at::MemOverlapStatus::Partial && (a.numel() == 0 || b.numel() == 0 || a.data_ptr() != b.data_ptr()),
            "the caches of a call may not share memory");
}
// a tensor that a kernel has written behind autograd's back
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

OptTensor paged_append(const OptTensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& key_cache, const Tensor& value_cache,
                       const Tensor& slots, const OptTensor& positions, const OptTensor& inv_freq, const OptTensor& q_weight,
                       const OptTensor& k_weight, const OptAxes& axes, bool interleaved, double eps, const OptTensor& k_bias_,
                       const OptTensor& bias_cache) {
  refuse_tangents(q_, k_, v_, q_weight, k_weight, k_bias_);
  refuse_grads(q_, k_, v_, q_weight, k_weight, inv_freq, k_bias_, OptTensor(key_cache), OptTensor(value_cache), bias_cache);
  check_device_status();
  FB_ASSERT(k_.dim() == 3 && v_.dim() == 3 && (!q_ || q_->dim() == 3), "q, k and v are (tokens, nheads, headdim)");
  check_16bit_cuda(k_);
  FB_ASSERT(v_.sizes() == k_.sizes(), "k and v have the same shape");
  const int64_t N = k_.size(0), Hk = k_.size(1), D = k_.size(2);
  FB_ASSERT(Hk > 0, "no key heads");
  check_beside(v_, k_);
  FB_ASSERT(v_.scalar_type() == k_.scalar_type(), "All tensors must have the same type");
  if (q_) {
    check_beside(*q_, k_);
    FB_ASSERT(q_->scalar_type() == k_.scalar_type(), "All tensors must have the same type");
    FB_ASSERT(q_->size(0) == N && q_->size(2) == D, "q and k differ in more than their heads");
  }
  FB_ASSERT(Hk <= kMaxRopeHeads && (!q_ || q_->size(1) + Hk <= kMaxRopeHeads), "too many heads");
  FB_ASSERT(key_cache.dim() == 4 && key_cache.size(0) > 0 && key_cache.size(1) > 0 && key_cache.size(1) <= 0x7fffffff,
            "caches are (pages, page size, heads, columns)");
  const int64_t pages = key_cache.size(0), page_size = key_cache.size(1);
  check_cache(key_cache, k_, pages, page_size, Hk, D);
  check_cache(value_cache, k_, pages, page_size, Hk, D);
  check_written(key_cache);
  check_written(value_cache);
  check_distinct(key_cache, value_cache);
  check_beside(slots, k_);
  FB_ASSERT(slots.dim() == 1 && slots.size(0) == N && is_index(slots), "slots holds one int32 or int64 per token");
  FB_ASSERT(k_bias_.has_value() == bias_cache.has_value(), "k_bias and bias_cache must be given together");
  const Tensor k = unit_rows(k_), v = unit_rows(v_), q = unit_rows_or_undefined(q_), kb = unit_rows_or_undefined(k_bias_);
  for (const Tensor* c : {&key_cache, &value_cache})
    for (const Tensor* t : {&q, &k, &v, &kb}) check_apart(*c, *t);
  if (bias_cache)
    for (const Tensor* t : {&q, &k, &v, &kb}) check_apart(*bias_cache, *t);
  c10::cuda::CUDAGuard guard(k.device());
  const RopeArgs a = {or_undefined(positions), contiguous_or_undefined(inv_freq), contiguous_or_undefined(q_weight),
                      contiguous_or_undefined(k_weight), axes, interleaved, eps};
  fb_rope_params p{};
  fill_rope(p, a, k, 1, N, D);
  auto strides_nh = [](const Tensor& t, int64_t(&out)[3]) {
    out[0] = 0;
    out[1] = t.stride(1);
    out[2] = t.stride(0);
  };
  Tensor qo;
  if (q.defined()) {
    qo = empty_dense_as(q);
    p.Hq = (int32_t)q.size(1);
    p.q = q.data_ptr();
    strides_nh(q, p.q_stride);
    p.q_out = qo.data_ptr();
    strides_nh(qo, p.q_out_stride);
  }
  p.Hk = (int32_t)Hk;
  p.k = k.data_ptr();
  strides_nh(k, p.k_stride);
  p.v = v.data_ptr();
  strides_nh(v, p.v_stride);
  p.key_cache = key_cache.data_ptr();
  p.value_cache = value_cache.data_ptr();
  cache_strides(key_cache, p.key_cache_stride);
  cache_strides(value_cache, p.value_cache_stride);
  p.num_pages = pages;
  p.page_size = (int32_t)page_size;
  p.slots = slots.data_ptr();
  p.slot_stride = slots.stride(0);
  p.slot_bits = slots.scalar_type() == at::kLong ? 64 : 32;
  if (kb.defined()) {
    FB_ASSERT(kb.dim() == 3 && kb.size(0) == N && (kb.size(1) == 1 || kb.size(1) == Hk) && kb.size(2) >= 1 && kb.size(2) <= 256,
              "k_bias is (tokens, 1 | nheads, rank)");
    check_beside(kb, k);
    FB_ASSERT(kb.scalar_type() == k.scalar_type(), "All tensors must have the same type");
    check_cache(*bias_cache, k, pages, page_size, kb.size(1), kb.size(2));
    check_written(*bias_cache);
    check_distinct(key_cache, *bias_cache);
    check_distinct(value_cache, *bias_cache);
    p.R = (int32_t)kb.size(2);
    p.bias_heads = (int32_t)kb.size(1);
    p.k_bias = kb.data_ptr();
    strides_nh(kb, p.k_bias_stride);
    p.bias_cache = bias_cache->data_ptr();
    cache_strides(*bias_cache, p.bias_cache_stride);
  }
  if (N > 0) {
    check_rc(fb_paged_append(&p, at::cuda::getCurrentCUDAStream().stream()), "fb_paged_append");
    written(key_cache);
    written(value_cache);
    if (bias_cache) written(*bias_cache);
  }
  return defined_or_none(qo);
}

void check_ints(const Tensor& t, const Tensor& like, int64_t n) {
  check_beside(t, like);
  FB_ASSERT(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), "lengths, counts and offsets are contiguous int32 vectors");
}

// (slots, positions, cu_tokens, lens, tree_mask)
std::tuple<Tensor, Tensor, Tensor, Tensor, OptTensor> paged_plan(const Tensor& block_table, const Tensor& pages_held,
                                                                 const Tensor& free_pages, const Tensor& free_count, const Tensor& lens,
                                                                 const Tensor& new_lens, int64_t page_size, int64_t num_tokens,
                                                                 const OptTensor& parents, int64_t max_tree) {
  check_device_status();
  FB_ASSERT(block_table.is_cuda(), "tensors lie in device memory");
  FB_ASSERT(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) > 0 && block_table.size(1) > 0 &&
                block_table.stride(1) == 1 && (block_table.size(0) == 1 || block_table.stride(0) >= block_table.size(1)),
            "the block table is (requests, pages) of int32 with contiguous rows");
  const int64_t B = block_table.size(0), M = block_table.size(1);
  FB_ASSERT(B <= 0x7fff0000 && page_size > 0 && M <= 0x7fffffff && page_size <= 0x7fffffff && M * page_size <= 0x7fffffff,
            "a row of the block table holds at most 2^31 - 1 tokens");
  FB_ASSERT(num_tokens >= 0 && num_tokens <= 0x7fff0000, "num_tokens out of range");
  check_ints(pages_held, block_table, B);
  check_ints(lens, block_table, B);
  check_ints(new_lens, block_table, B);
  check_ints(free_count, block_table, 1);
  FB_ASSERT(free_pages.dim() == 1 && free_pages.size(0) < 0x7fffffff, "free_pages is a vector");
  check_ints(free_pages, block_table, free_pages.size(0));
  c10::cuda::CUDAGuard guard(block_table.device());
  const Tensor slots = empty_on({num_tokens}, at::kLong, block_table), positions = empty_on({num_tokens}, at::kInt, block_table),
               cu = empty_on({B + 1}, at::kInt, block_table), lens_out = empty_on({B}, at::kInt, block_table);
  OptTensor mask;
  fb_plan_params p{};
  if (parents) {
    FB_ASSERT(max_tree >= 1 && max_tree <= 4096, "max_tree is 1 to 4096 drafted tokens");
    check_ints(*parents, block_table, num_tokens);
    p.mask_words = (int32_t)((max_tree + 63) / 64);
    mask = empty_on({num_tokens, p.mask_words}, at::kLong, block_table);
    p.parents = num_tokens ? parents->data_ptr<int32_t>() : nullptr;
    p.tree_mask = mask->data_ptr<int64_t>();
  }
  p.B = (int32_t)B;
  p.num_tokens = (int32_t)num_tokens;
  p.page_size = (int32_t)page_size;
  p.table_width = (int32_t)M;
  p.stack_size = (int32_t)free_pages.size(0);
  p.block_table = block_table.data_ptr<int32_t>();
  p.table_stride = B == 1 ? M : block_table.stride(0);
  p.pages_held = pages_held.data_ptr<int32_t>();
  p.free_pages = free_pages.data_ptr<int32_t>();
  p.free_count = free_count.data_ptr<int32_t>();
  p.lens = lens.data_ptr<int32_t>();
  p.new_lens = new_lens.data_ptr<int32_t>();
  p.cu_tokens = cu.data_ptr<int32_t>();
  p.lens_out = lens_out.data_ptr<int32_t>();
  p.positions = positions.data_ptr<int32_t>();
  p.slots = slots.data_ptr<int64_t>();
  p.status = status_ptr();
  check_rc(fb_paged_plan(&p, at::cuda::getCurrentCUDAStream().stream()), "fb_paged_plan");
  for (const Tensor& t : {block_table, pages_held, free_pages, free_count}) written(t);
  return {slots, positions, cu, lens_out, mask};
}

// (o, lse)
std::tuple<Tensor, OptTensor> paged_forward(const Tensor& q_, const Tensor& key_cache, const Tensor& value_cache,
                                            const Tensor& block_table, const Tensor& lens, const Tensor& cu_tokens,
                                            const OptTensor& tree_mask_, const OptTensor& positions, const OptTensor& slopes_,
                                            const OptTensor& q_bias_, const OptTensor& bias_cache, std::optional<double> softmax_scale,
                                            bool want_lse, int64_t flags) {
  refuse_tangents(q_, key_cache, value_cache, slopes_, q_bias_, bias_cache);
  refuse_grads(q_, key_cache, value_cache, slopes_, q_bias_, bias_cache);
  check_device_status();
  FB_ASSERT(q_.dim() == 3, "q is (tokens, nheads, headdim)");
  check_16bit_cuda(q_);
  const int64_t N = q_.size(0), Hq = q_.size(1), D = q_.size(2);
  FB_ASSERT(D >= 1 && D <= 128, "FlashAttention only support head dimensions up to 128");
  FB_ASSERT(N <= 0x7fff0000 && Hq <= 65536, "too many tokens or heads");
  FB_ASSERT(key_cache.dim() == 4 && key_cache.size(0) > 0 && key_cache.size(1) > 0 && key_cache.size(2) > 0,
            "caches are (pages, page size, heads, columns)");
  const int64_t pages = key_cache.size(0), page_size = key_cache.size(1), Hk = key_cache.size(2);
  FB_ASSERT(Hq > 0 && Hq % Hk == 0, "the heads of q are a multiple of the heads of the cache");
  check_cache(key_cache, q_, pages, page_size, Hk, D);
  check_cache(value_cache, q_, pages, page_size, Hk, D);
  check_beside(block_table, q_);
  FB_ASSERT(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) > 0 && block_table.size(1) > 0 &&
                (block_table.stride(1) == 1 || block_table.size(1) == 1),
            "the block table is (requests, pages) of int32 with contiguous rows");
  const int64_t B = block_table.size(0), M = block_table.size(1);
  FB_ASSERT(B <= 0x7fff0000, "too many requests");
  FB_ASSERT(page_size <= 0x7fffffff && M <= 0x7fffffff && M * page_size <= 0x7fff0000, "a row of the block table holds at most 2^31 - 2^16 tokens");
  check_ints(lens, q_, B);
  check_ints(cu_tokens, q_, B + 1);
  const Tensor q = unit_rows(q_), qb = unit_rows_or_undefined(q_bias_);
  c10::cuda::CUDAGuard guard(q.device());
  fb_paged_params p{};
  p.N = (int32_t)N;
  p.B = (int32_t)B;
  p.Hq = (int32_t)Hq;
  p.Hk = (int32_t)Hk;
  p.D = (int32_t)D;
  p.dtype = dtype_code(q.scalar_type());
  p.page_size = (int32_t)page_size;
  p.table_width = (int32_t)M;
  p.num_pages = pages;
  p.flags = (int32_t)flags;
  p.softmax_scale = (float)scale_or_default(softmax_scale, D);
  Tensor mask, slopes;
  if (tree_mask_) {
    mask = tree_mask_->dim() == 1 ? tree_mask_->unsqueeze(1) : *tree_mask_;
    check_beside(mask, q);
    FB_ASSERT(mask.dim() == 2 && mask.size(0) == N && mask.size(1) >= 1 && mask.scalar_type() == at::kLong, "tree_mask is (tokens, words) of int64");
    if (mask.size(1) > 1 && mask.stride(1) != 1) mask = mask.contiguous();
    p.tree_mask = mask.data_ptr<int64_t>();
    p.mask_words = (int32_t)mask.size(1);
    p.mask_stride = mask.stride(0);
  }
  if (positions) {
    check_ints(*positions, q, N);
    p.positions = positions->data_ptr<int32_t>();
  }
  if (slopes_) {
    FB_ASSERT(!q_bias_, "slopes and factors exclude each other");
    // (as it is in the common case: the conversions, which do nothing then, cost three trips through the dispatcher)
    slopes = slopes_->scalar_type() == at::kFloat && slopes_->device() == q.device() && slopes_->is_contiguous()
                 ? *slopes_
                 : slopes_->detach().to(q.device(), at::kFloat).reshape({-1}).contiguous();
    FB_ASSERT(slopes.numel() == Hq, "one slope per head");
    p.slopes = slopes.data_ptr<float>();
  }
  if (q_bias_.has_value() != bias_cache.has_value()) throw std::runtime_error("q_bias and bias_cache must be given together");
  if (qb.defined()) {
    check_beside(qb, q);
    FB_ASSERT(qb.scalar_type() == q.scalar_type(), "All tensors must have the same type");
    FB_ASSERT(qb.dim() == 3 && qb.size(0) == N && (qb.size(1) == 1 || qb.size(1) == Hq) && qb.size(2) >= 1 && qb.size(2) <= 256,
              "q_bias is (tokens, 1 | nheads, rank)");
    FB_ASSERT(bias_cache->dim() == 4 && (bias_cache->size(2) == 1 || bias_cache->size(2) == Hk), "bias_cache has one head or those of the keys");
    check_cache(*bias_cache, q, pages, page_size, bias_cache->size(2), qb.size(2));
    p.R = (int32_t)qb.size(2);
    p.bias_heads = (int32_t)bias_cache->size(2);
    p.q_bias = qb.data_ptr();
    p.q_bias_stride[0] = qb.stride(0);
    p.q_bias_stride[1] = qb.size(1) == 1 ? 0 : qb.stride(1);
    p.bias_cache = bias_cache->data_ptr();
    cache_strides(*bias_cache, p.bias_cache_stride);
  }
  p.q = q.data_ptr();
  p.q_stride[0] = q.stride(0);
  p.q_stride[1] = q.stride(1);
  p.key_cache = key_cache.data_ptr();
  p.value_cache = value_cache.data_ptr();
  cache_strides(key_cache, p.key_cache_stride);
  cache_strides(value_cache, p.value_cache_stride);
  p.block_table = block_table.data_ptr<int32_t>();
  p.table_stride = block_table.stride(0);
  p.lens = lens.data_ptr<int32_t>();
  p.cu_tokens = cu_tokens.data_ptr<int32_t>();
  p.status = status_ptr();
  Tensor o = empty_on({N, Hq, D}, q.scalar_type(), q);
  p.o = o.data_ptr();
  p.o_stride[0] = o.stride(0);
  p.o_stride[1] = o.stride(1);
  OptTensor lse;
  if (want_lse) {
    lse = empty_on({N, Hq}, at::kFloat, q);
    p.lse = lse->data_ptr<float>();
  }
  if (N == 0) return {o, lse};
  Tensor ws;
  if (const size_t need = fb_paged_workspace_bytes(&p)) {
    ws = workspace(need, q);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
  }
  check_rc(fb_paged_fwd(&p, at::cuda::getCurrentCUDAStream().stream()), "fb_paged_fwd");
  return {o, lse};
}
