// Autograd nodes of the operators without handles (part of autograd_node.cpp): attention with a relative position bias
// (relative_bias.py), attention to keys of another length (attention_cross.py), the root-mean-square norm and the layer norm (norm.py).
// They do what the Python functions there do, checks of arguments included, with the node, the saved tensors and the allocations on
// the C++ side: a training step of 16 heads of 1024 and one of a few rows are bound by the host.
#pragma once

// A tensor as it was saved, which hooks may have brought back as something else: the kernels take types and sizes as they
// were.
void save_as_is(AutogradContext* ctx, const variable_list& tensors) {
    std::vector<int64_t> numbers;
    for (const Tensor& t : tensors) {
        numbers.push_back(t.defined() ? t.dim() : -1);
        if (!t.defined()) continue;
        numbers.push_back(static_cast<int64_t>(t.scalar_type()));
        numbers.push_back(t.device().index());
        for (int64_t n : t.sizes()) numbers.push_back(n);
    }
    ctx->saved_data["as_saved"] = numbers;
    ctx->save_for_backward(tensors);
}
variable_list saved_as_is(AutogradContext* ctx) {
    const std::vector<int64_t> n = ctx->saved_data["as_saved"].toIntVector();
    const variable_list saved = ctx->get_saved_variables();
    size_t at = 0;
    for (const Tensor& t : saved) {
        const int64_t dim = n.at(at++);
        bool same = t.defined() == (dim >= 0);
        if (dim >= 0) {
            same = same && t.is_cuda() && t.dim() == dim && static_cast<int64_t>(t.scalar_type()) == n.at(at) &&
                   t.device().index() == n.at(at + 1);
            at += 2;
            for (int64_t i = 0; i < dim; ++i) same = same && t.size(i) == n.at(at + i);
            at += dim;
        }
        TORCH_CHECK_TYPE(same, "saved tensors of the device, type and size they were saved with expected");
    }
    return saved;
}

// A call of the library by its status: its message is this thread's, whatever other calls have left behind.
void check_call(bool ok, const char* where) {
    if (ok) return;
    const std::string text = spion_take_call_error();
    throw std::runtime_error(std::string(where) + (text.empty() ? " failed" : ": " + text));
}

// Gradients that a second derivative would have to go through: it is refused, not left out.
void once_differentiable(variable_list& grads, size_t used) {
    if (!torch::GradMode::is_enabled()) return;
    variable_list given;
    std::vector<size_t> at;
    for (size_t i = 0; i < used; ++i)
        if (grads[i].defined()) {
            given.push_back(grads[i].detach().requires_grad_(true));
            at.push_back(i);
        }
    auto refuse = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with "
                                                                  "@once_differentiable", static_cast<int64_t>(given.size()));
    const variable_list out = refuse->apply(std::move(given));
    for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = out[i];
}

void on_one_gpu(const Tensor& t, const Tensor& as) {
    TORCH_CHECK(!t.defined() || (t.is_cuda() && t.device() == as.device()), "tensors on one GPU expected");
}
void fp32_or_bf16(const Tensor& t, const char* what) {
    TORCH_CHECK_TYPE(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, "fp32 or bf16 ", what,
                     " expected, got ", t.scalar_type());
}

// ---- attention with a relative position bias ------------------------------------------------------------------------
// Heads as the kernels read them: themselves, or a copy where their strides or address are not theirs.
Tensor readable_heads(const Tensor& t) {
    spion_head_layout lay{};
    const auto fits = [&](const Tensor& x) { return head_layout(x, lay) && x.stride(2) * x.element_size() <= 1 << 24; };
    if (fits(t)) return t;
    const Tensor c = t.contiguous();
    return fits(c) ? c : t.clone(at::MemoryFormat::Contiguous);
}
// In the memory order of t, [B, L, H, d] where the heads of a row lie next to each other and the kernels take that.
Tensor empty_like_heads(const Tensor& t) {
    const int64_t row = t.size(1) * t.size(3);
    const bool interleaved = t.stride(1) < t.stride(2) && row * t.element_size() <= 1 << 24 && t.size(2) * row < int64_t(1) << 29;
    return empty_heads(t.sizes(), interleaved, t.options());
}
spion_heads heads_of(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

spion_bias_attention bias_call(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& w, const Tensor& buckets,
                               const Tensor& mask, const Tensor& mat, const Tensor& lse, int64_t block, int64_t offset) {
    spion_bias_attention c{};
    c.Q = heads_of(q);
    c.K = heads_of(k);
    c.V = heads_of(v);
    c.Out = heads_of(out);
    c.weight = w.data_ptr();
    c.buckets = ip(buckets);
    if (mask.defined()) {
        c.key_mask = mask.data_ptr();
        c.mask_bytes = (int)mask.element_size();
    }
    c.mat = fp(mat);
    c.Lse = static_cast<float*>(lse.data_ptr());
    c.batch = (int)q.size(0);
    c.heads = (int)q.size(1);
    c.q_len = (int)q.size(2);
    c.k_len = (int)k.size(2);
    c.head_dim = (int)q.size(3);
    c.bf16 = q.scalar_type() == torch::kBFloat16;
    c.num_buckets = (int)w.size(0);
    c.max_distance = (int)(buckets.size(0) / 2);
    c.offset = (int)offset;
    c.block_size = (int)block;
    return c;
}
Tensor bias_workspace(spion_bias_attention& c, bool backward, const Tensor& q) {
    const int64_t n = spion_bias_workspace(&c, backward);
    check_call(n >= 0, "spion_bias_workspace");
    if (n == 0) return Tensor();
    Tensor ws = torch::empty({n}, q.options().dtype(torch::kFloat32));
    c.workspace = fpm(ws);
    c.workspace_floats = n;
    return ws;
}

struct BiasForward {
    Tensor q, k, v, w, buckets, out, lse, mean;
};
BiasForward bias_forward(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& weight, const Tensor& buckets,
                         const Tensor& mask, const Tensor& mat, int64_t block, int64_t offset, bool score_map) {
    BiasForward r;
    r.q = readable_heads(query);
    r.k = readable_heads(key);
    r.v = readable_heads(value);
    r.w = weight.contiguous();
    r.buckets = buckets.contiguous();
    r.out = empty_like_heads(query);
    const auto fp32 = query.options().dtype(torch::kFloat32);
    r.lse = torch::empty({query.size(0) * query.size(1), query.size(2)}, fp32);
    if (score_map) r.mean = torch::empty({query.size(2), key.size(2)}, fp32);
    spion_bias_attention c = bias_call(r.q, r.k, r.v, r.out, r.w, r.buckets, mask, mat, r.lse, block, offset);
    if (score_map) c.Mean = fpm(r.mean);
    const Tensor ws = bias_workspace(c, false, query);
    void* const stream = reinterpret_cast<void*>(current_stream(query.device().index()));
    check_call(spion_bias_attention_forward(&c, stream) == 0, "spion_bias_attention_forward");
    return r;
}

struct BiasNode : public torch::autograd::Function<BiasNode> {
    static Tensor forward(AutogradContext* ctx, Tensor query, Tensor key, Tensor value, Tensor weight, Tensor buckets,
                          c10::optional<Tensor> mask, c10::optional<Tensor> mat, int64_t block, int64_t offset, bool score_map,
                          Tensor* mean) {
        const Tensor m = mask.value_or(Tensor()), p = mat.value_or(Tensor());
        const BiasForward r = bias_forward(query, key, value, weight, buckets, m, p, block, offset, score_map);
        *mean = r.mean;
        ctx->saved_data["block"] = block;
        ctx->saved_data["offset"] = offset;
        save_as_is(ctx, {r.q, r.k, r.v, r.w, r.out, r.lse, r.buckets, m, p});
        return r.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = saved_as_is(ctx);
        const c10::DeviceGuard on(s[0].device());
        const Tensor q = readable_heads(s[0]), k = readable_heads(s[1]), v = readable_heads(s[2]), out = readable_heads(s[4]);
        const Tensor w = s[3].contiguous(), lse = s[5].contiguous(), buckets = s[6].contiguous();
        const auto rest = [&](size_t i) { return s[i].defined() ? s[i].contiguous() : Tensor(); };
        const Tensor mask = rest(7), mat = rest(8);
        const Tensor go = readable_heads(grads[0].to(q.scalar_type()));
        variable_list g(11);
        if (q.scalar_type() == torch::kFloat32 && q.sizes() == k.sizes() && adjacent_head_views(q, k, v)) {
            // slices of one fused projection: the gradients likewise
            const Tensor buf = torch::empty({q.size(0), q.size(2), 3, q.size(1), q.size(3)}, q.options());
            for (int i = 0; i < 3; ++i) g[i] = buf.select(2, i).transpose(1, 2);
        } else {
            g[0] = empty_like_heads(q);
            g[1] = empty_like_heads(k);
            g[2] = empty_like_heads(v);
        }
        g[3] = torch::empty_like(w);
        spion_bias_attention c = bias_call(q, k, v, out, w, buckets, mask, mat, lse, ctx->saved_data["block"].toInt(),
                                           ctx->saved_data["offset"].toInt());
        c.dO = heads_of(go);
        c.dQ = heads_of(g[0]);
        c.dK = heads_of(g[1]);
        c.dV = heads_of(g[2]);
        c.dweight = g[3].data_ptr();
        const Tensor ws = bias_workspace(c, true, q);
        void* const stream = reinterpret_cast<void*>(current_stream(q.device().index()));
        check_call(spion_bias_attention_backward(&c, stream) == 0, "spion_bias_attention_backward");
        once_differentiable(g, 4);
        return g;
    }
};

std::vector<Tensor> relative_bias_attention(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& weight,
                                            const Tensor& buckets, const c10::optional<Tensor>& key_mask,
                                            const c10::optional<Tensor>& pattern, int64_t block, int64_t offset, bool score_map) {
    constexpr int64_t far = int64_t(1) << 29;
    TORCH_CHECK_VALUE(query.dim() == 4 && key.dim() == 4, "heads [B, H, L, d] expected");
    const int64_t B = query.size(0), H = query.size(1), Lq = query.size(2), d = query.size(3), Lk = key.size(2);
    for (const Tensor* t : {&key, &value})
        TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == B && t->size(1) == H && t->size(2) == Lk && t->size(3) == d,
                          t == &key ? "key" : "value", " shape ", t->sizes(), " does not match the query's ", query.sizes());
    fp32_or_bf16(query, "heads");
    TORCH_CHECK_VALUE(d == 32 || d == 64, "head dimension ", d, ": 32 or 64 expected");
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == H && weight.size(0) >= 1, "weight shape ", weight.sizes(),
                      ": [num_buckets, ", H, "] expected");
    TORCH_CHECK_VALUE(buckets.dim() == 1 && buckets.size(0) % 2 == 1 && buckets.size(0) >= 3 &&
                          buckets.size(0) <= 2 * SPION_BIAS_MAX_DISTANCE + 1,
                      "buckets: [2 R + 1] with R from 1 to ", SPION_BIAS_MAX_DISTANCE, " expected, got ", buckets.sizes());
    TORCH_CHECK_TYPE(buckets.scalar_type() == torch::kInt32, "buckets: int32 expected");
    TORCH_CHECK_VALUE(offset >= -far && offset <= far, "offset out of range");
    Tensor mask = key_mask.value_or(Tensor()), mat = pattern.value_or(Tensor());
    TORCH_CHECK_VALUE(!mask.defined() || (mask.dim() == 2 && mask.size(0) == B && mask.size(1) == Lk), "key mask shape ",
                      mask.defined() ? mask.sizes() : c10::IntArrayRef(), ": [", B, ", ", Lk, "] expected");
    if (mat.defined()) {
        TORCH_CHECK_VALUE(block >= 32 && block % 32 == 0 && block <= far, "block_size ", block, ": a multiple of 32 expected with a pattern");
        const int64_t nb = (Lk + block - 1) / block;
        TORCH_CHECK_VALUE(mat.dim() == 2 && mat.size(0) == nb && mat.size(1) == nb, "pattern shape ", mat.sizes(), ": [", nb, ", ", nb,
                          "] expected");
        TORCH_CHECK_VALUE(Lq == Lk && offset == 0, "a pattern has as many queries as keys and no offset");
        TORCH_CHECK_VALUE(!score_map, "the mean map is of the dense phase, without a pattern");
    } else {
        block = 0;
    }
    TORCH_CHECK_VALUE(B <= INT_MAX && H <= INT_MAX && Lq <= far && Lk <= far && weight.size(0) <= INT_MAX, "sizes out of range");
    for (const Tensor* t : {&query, &key, &value, &weight, &buckets, static_cast<const Tensor*>(&mask), static_cast<const Tensor*>(&mat)})
        on_one_gpu(*t, query);
    TORCH_CHECK_TYPE(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type() &&
                         weight.scalar_type() == query.scalar_type(),
                     "heads and weight of one type expected");
    const c10::DeviceGuard on(query.device());
    if (mask.defined()) {
        const auto type = mask.scalar_type();
        if (type != torch::kFloat32 && type != torch::kBool && type != torch::kUInt8) mask = mask.ne(0);
        mask = mask.detach().contiguous();
    }
    if (mat.defined()) mat = mat.detach().to(torch::kFloat32).contiguous();
    if (query.numel() == 0 || key.numel() == 0) {  // nothing to attend to, or nobody to
        const Tensor every = torch::ones({}, query.options().dtype(torch::kBool));
        const auto nothing = [&](const Tensor& t) { return t.masked_fill(every, 0.0); };
        const Tensor out = nothing(query) + nothing(key).sum() + nothing(value).sum() + nothing(weight).sum();
        if (!score_map) return {out};
        return {out, torch::zeros({Lq, Lk}, query.options().dtype(torch::kFloat32))};
    }
    if (without_node({&query, &key, &value, &weight})) {
        const BiasForward r = bias_forward(query, key, value, weight, buckets, mask, mat, block, offset, score_map);
        return score_map ? std::vector<Tensor>{r.out, r.mean} : std::vector<Tensor>{r.out};
    }
    const auto given = [](const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; };
    Tensor mean;
    const Tensor out = BiasNode::apply(query, key, value, weight, buckets, given(mask), given(mat), block, offset, score_map, &mean);
    return score_map ? std::vector<Tensor>{out, mean} : std::vector<Tensor>{out};
}

// ---- the root-mean-square norm ----------------------------------------------------------------------------------------
// [rows, width] with the elements of a row next to each other: a view where the strides allow one.
Tensor rows_of(const Tensor& t) {
    const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return (r.stride(1) == 1 || r.size(1) == 1) && r.stride(0) >= 0 ? r : r.contiguous();
}
spion_rms_norm norm_call(const Tensor& rows, const Tensor& w, double eps) {
    spion_rms_norm c{};
    c.x = rows.data_ptr();
    c.weight = w.data_ptr();
    c.rows = rows.size(0);
    c.width = (int)rows.size(1);
    c.bf16 = rows.scalar_type() == torch::kBFloat16;
    c.x_stride = rows.stride(0);
    c.eps = (float)eps;
    return c;
}
// {y or codes, h or nothing, scales or nothing}
variable_list norm_forward(const Tensor& x, const Tensor& weight, const Tensor& res, double eps, bool fp8) {
    variable_list r(3);
    r[0] = torch::empty(x.sizes(), fp8 ? x.options().dtype(torch::kFloat8_e4m3fn) : x.options());
    if (res.defined()) r[1] = torch::empty(x.sizes(), x.options());
    if (fp8) r[2] = torch::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(torch::kFloat32));
    if (x.numel() == 0) {
        if (fp8) r[2].fill_(0x1p-126);  // rows without elements
        return r;
    }
    const Tensor xr = rows_of(x), w = weight.contiguous(), rr = res.defined() ? rows_of(res) : Tensor();
    spion_rms_norm c = norm_call(xr, w, eps);
    if (res.defined()) {
        c.residual = rr.data_ptr();
        c.residual_stride = rr.stride(0);
        c.h = r[1].data_ptr();
    }
    if (fp8) {
        c.codes = static_cast<unsigned char*>(r[0].data_ptr());
        c.scales = fpm(r[2]);
    } else {
        c.y = r[0].data_ptr();
    }
    void* const stream = reinterpret_cast<void*>(current_stream(x.device().index()));
    check_call(spion_rms_norm_forward(&c, stream) == 0, "spion_rms_norm_forward");
    return r;
}

struct NormNode : public torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, c10::optional<Tensor> res, double eps) {
        variable_list r = norm_forward(x, weight, res.value_or(Tensor()), eps, false);
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        save_as_is(ctx, {r[1].defined() ? r[1] : x, weight});
        r.resize(r[1].defined() ? 2 : 1);
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = saved_as_is(ctx);
        const Tensor &h = s[0], &dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        variable_list g(4);
        if (!dy.defined() && !dh.defined()) return g;
        const bool residual = grads.size() > 1;
        const c10::DeviceGuard on(h.device());
        if (!dy.defined() || h.numel() == 0) {  // only the stream was used
            g[0] = dh.defined() ? dh : torch::zeros_like(h);
            g[1] = torch::zeros_like(s[1]);
            if (residual) g[2] = g[0];
            return g;
        }
        const Tensor hr = rows_of(h), w = s[1].contiguous(), dyr = rows_of(dy.to(h.scalar_type()));
        const Tensor dhr = dh.defined() ? rows_of(dh.to(h.scalar_type())) : Tensor();
        g[0] = torch::empty(h.sizes(), h.options());
        g[1] = torch::empty(w.sizes(), w.options());
        spion_rms_norm c = norm_call(hr, w, ctx->saved_data["eps"].toDouble());
        c.dy = dyr.data_ptr();
        c.dy_stride = dyr.stride(0);
        if (dhr.defined()) {
            c.dh = dhr.data_ptr();
            c.dh_stride = dhr.stride(0);
        }
        c.dx = g[0].data_ptr();
        c.dweight = g[1].data_ptr();
        c.workspace_floats = spion_rms_norm_workspace(&c);
        check_call(c.workspace_floats >= 0, "spion_rms_norm_workspace");
        Tensor ws = torch::empty({(int64_t)c.workspace_floats}, h.options().dtype(torch::kFloat32));
        c.workspace = fpm(ws);
        void* const stream = reinterpret_cast<void*>(current_stream(h.device().index()));
        check_call(spion_rms_norm_backward(&c, stream) == 0, "spion_rms_norm_backward");
        once_differentiable(g, 2);
        if (residual) g[2] = g[0];
        return g;
    }
};

void check_norm(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& res, double eps) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1), "weight shape ", weight.sizes(),
                      " does not match rows of ", x.sizes());
    TORCH_CHECK_VALUE(!res.has_value() || res->sizes() == x.sizes(), "residual shape ", res.has_value() ? res->sizes() : x.sizes(),
                      " does not match ", x.sizes());
    fp32_or_bf16(x, "rows");
    TORCH_CHECK_VALUE(x.size(-1) <= int64_t(1) << 29, "width out of range");
    TORCH_CHECK_VALUE(eps >= 0, "eps is not negative");
    on_one_gpu(x, x);
    on_one_gpu(weight, x);
    if (res.has_value()) on_one_gpu(*res, x);
    TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() && (!res.has_value() || res->scalar_type() == x.scalar_type()),
                     "rows and weight of one type expected");
}
std::vector<Tensor> rms_norm(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& res, double eps) {
    check_norm(x, weight, res, eps);
    const c10::DeviceGuard on(x.device());
    const Tensor r = res.value_or(Tensor());
    if (without_node({&x, &weight, &r})) {
        variable_list out = norm_forward(x, weight, r, eps, false);
        out.resize(r.defined() ? 2 : 1);
        return out;
    }
    return NormNode::apply(x, weight, res, eps);
}
std::vector<Tensor> rms_norm_fp8(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& res, double eps) {
    check_norm(x, weight, res, eps);
    TORCH_CHECK(!torch::GradMode::is_enabled() ||
                    !(x.requires_grad() || weight.requires_grad() || (res.has_value() && res->requires_grad())),
                "rms_norm_fp8 has no gradient: call it under torch.no_grad()");
    const c10::DeviceGuard on(x.device());
    variable_list r = norm_forward(x, weight, res.value_or(Tensor()), eps, true);
    if (!r[1].defined()) return {r[0], r[2]};
    return {r[0], r[2], r[1]};
}

// ---- the layer norm ---------------------------------------------------------------------------------------------------
spion_layer_norm layer_norm_call(const Tensor& rows, const Tensor& w, double eps) {
    spion_layer_norm c{};
    c.x = rows.data_ptr();
    c.weight = w.data_ptr();
    c.rows = rows.size(0);
    c.width = (int)rows.size(1);
    c.bf16 = rows.scalar_type() == torch::kBFloat16;
    c.x_stride = rows.stride(0);
    c.eps = (float)eps;
    return c;
}
// {y, h or nothing}
variable_list layer_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& res, double eps) {
    variable_list r{torch::empty(x.sizes(), x.options())};
    if (res.defined()) r.push_back(torch::empty(x.sizes(), x.options()));
    if (x.numel() == 0) return r;
    const Tensor xr = rows_of(x), w = weight.contiguous(), b = bias.defined() ? bias.contiguous() : Tensor(), rr = res.defined() ? rows_of(res) : Tensor();
    spion_layer_norm c = layer_norm_call(xr, w, eps);
    if (b.defined()) c.bias = b.data_ptr();
    if (res.defined()) {
        c.residual = rr.data_ptr();
        c.residual_stride = rr.stride(0);
        c.h = r[1].data_ptr();
    }
    c.y = r[0].data_ptr();
    void* const stream = reinterpret_cast<void*>(current_stream(x.device().index()));
    check_call(spion_layer_norm_forward(&c, stream) == 0, "spion_layer_norm_forward");
    return r;
}

struct LayerNormNode : public torch::autograd::Function<LayerNormNode> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, c10::optional<Tensor> bias, c10::optional<Tensor> res, double eps) {
        variable_list r = layer_norm_forward(x, weight, bias.value_or(Tensor()), res.value_or(Tensor()), eps);
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->set_materialize_grads(false);
        save_as_is(ctx, {r.size() > 1 ? r[1] : x, weight});
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = saved_as_is(ctx);
        const Tensor &h = s[0], &dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        variable_list g(5);
        if (!dy.defined() && !dh.defined()) return g;
        const bool residual = grads.size() > 1, bias = ctx->saved_data["bias"].toBool();
        const c10::DeviceGuard on(h.device());
        if (!dy.defined() || h.numel() == 0) {  // only the stream was used
            g[0] = dh.defined() ? dh : torch::zeros_like(h);
            g[1] = torch::zeros_like(s[1]);
            if (bias) g[2] = torch::zeros_like(s[1]);
            if (residual) g[3] = g[0];
            return g;
        }
        const Tensor hr = rows_of(h), w = s[1].contiguous(), dyr = rows_of(dy.to(h.scalar_type()));
        const Tensor dhr = dh.defined() ? rows_of(dh.to(h.scalar_type())) : Tensor();
        g[0] = torch::empty(h.sizes(), h.options());
        g[1] = torch::empty(w.sizes(), w.options());
        if (bias) g[2] = torch::empty(w.sizes(), w.options());
        spion_layer_norm c = layer_norm_call(hr, w, ctx->saved_data["eps"].toDouble());
        c.dy = dyr.data_ptr();
        c.dy_stride = dyr.stride(0);
        if (dhr.defined()) {
            c.dh = dhr.data_ptr();
            c.dh_stride = dhr.stride(0);
        }
        c.dx = g[0].data_ptr();
        c.dweight = g[1].data_ptr();
        if (bias) c.dbias = g[2].data_ptr();
        c.workspace_floats = spion_layer_norm_workspace(&c);
        check_call(c.workspace_floats >= 0, "spion_layer_norm_workspace");
        Tensor ws = torch::empty({(int64_t)c.workspace_floats}, h.options().dtype(torch::kFloat32));
        c.workspace = fpm(ws);
        void* const stream = reinterpret_cast<void*>(current_stream(h.device().index()));
        check_call(spion_layer_norm_backward(&c, stream) == 0, "spion_layer_norm_backward");
        once_differentiable(g, 3);
        if (residual) g[3] = g[0];
        return g;
    }
};

std::vector<Tensor> layer_norm(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, const c10::optional<Tensor>& res, double eps) {
    TORCH_CHECK_VALUE(!bias.has_value() || bias->sizes() == weight.sizes(), "bias shape ", bias.has_value() ? bias->sizes() : weight.sizes(),
                      " does not match the weight's ", weight.sizes());
    check_norm(x, weight, res, eps);
    if (bias.has_value()) {
        on_one_gpu(*bias, x);
        TORCH_CHECK_TYPE(bias->scalar_type() == x.scalar_type(), "rows, weight and bias of one type expected");
    }
    const c10::DeviceGuard on(x.device());
    const Tensor b = bias.value_or(Tensor()), r = res.value_or(Tensor());
    if (without_node({&x, &weight, &b, &r})) return layer_norm_forward(x, weight, b, r, eps);
    return LayerNormNode::apply(x, weight, bias, res, eps);
}

// ---- attention to keys of another length ------------------------------------------------------------------------------
// Heads as the kernels read them: themselves, or a copy where their strides or address are not theirs (multiples of 16 bytes, rows up to
// 2^24 bytes apart).  `together` heads, within 2^31 bytes, are reached from one address.
Tensor readable_group(const Tensor& t, int64_t together) {
    const auto fits = [&](const Tensor& x) {
        const int64_t sb = x.stride(0), sh = x.stride(1), sl = x.stride(2), d = x.size(3), e = x.element_size();
        if (x.stride(3) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || sb < 0 || sh < 0 || sb * e % 16 || sh * e % 16 || sl * e % 16 ||
            sl < d || sl * e > 1 << 24)
            return false;
        return ((together - 1) * sh + (x.size(2) - 1) * sl + d) * e < int64_t(1) << 31;
    };
    if (fits(t)) return t;
    const Tensor c = t.contiguous();
    return fits(c) ? c : t.clone(at::MemoryFormat::Contiguous);
}
// k, v are the two slices of one [B, L, 2, G, d] buffer, in this order
bool paired_views(const Tensor& k, const Tensor& v) {
    const int64_t G = k.size(1), L = k.size(2), d = k.size(3);
    const int64_t want[4] = {L * 2 * G * d, d, 2 * G * d, 1};
    for (int i = 0; i < 4; ++i)
        if (k.stride(i) != want[i] || v.stride(i) != want[i]) return false;
    return (const char*)v.data_ptr() - (const char*)k.data_ptr() == G * d * (int64_t)k.element_size();
}
spion_cross_attention cross_call(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, const Tensor& mask) {
    spion_cross_attention c{};
    c.Q = heads_of(q);
    c.K = heads_of(k);
    c.V = heads_of(v);
    c.Out = heads_of(out);
    if (mask.defined()) {
        c.key_mask = mask.data_ptr();
        c.mask_bytes = (int)mask.element_size();
    }
    c.Lse = static_cast<float*>(lse.data_ptr());
    c.batch = (int)q.size(0);
    c.heads = (int)q.size(1);
    c.key_heads = (int)k.size(1);
    c.q_len = (int)q.size(2);
    c.k_len = (int)k.size(2);
    c.head_dim = (int)q.size(3);
    c.bf16 = q.scalar_type() == torch::kBFloat16;
    return c;
}
Tensor cross_workspace(spion_cross_attention& c, bool backward, const Tensor& q) {
    const int64_t n = spion_cross_workspace(&c, backward);
    check_call(n >= 0, "spion_cross_workspace");
    if (n == 0) return Tensor();
    Tensor ws = torch::empty({n}, q.options().dtype(torch::kFloat32));
    c.workspace = fpm(ws);
    c.workspace_floats = n;
    return ws;
}
struct CrossForward {
    Tensor q, k, v, out, lse;
};
CrossForward cross_forward(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& mask) {
    CrossForward r;
    r.q = readable_group(query, query.size(1) / key.size(1));
    r.k = readable_group(key, 1);
    r.v = readable_group(value, 1);
    r.out = empty_like_heads(query);
    r.lse = torch::empty({query.size(0) * query.size(1), query.size(2)}, query.options().dtype(torch::kFloat32));
    spion_cross_attention c = cross_call(r.q, r.k, r.v, r.out, r.lse, mask);
    const Tensor ws = cross_workspace(c, false, query);
    void* const stream = reinterpret_cast<void*>(current_stream(query.device().index()));
    check_call(spion_cross_attention_forward(&c, stream) == 0, "spion_cross_attention_forward");
    return r;
}

struct CrossNode : public torch::autograd::Function<CrossNode> {
    static Tensor forward(AutogradContext* ctx, Tensor query, Tensor key, Tensor value, c10::optional<Tensor> mask) {
        const Tensor m = mask.value_or(Tensor());
        const CrossForward r = cross_forward(query, key, value, m);
        save_as_is(ctx, {r.q, r.k, r.v, r.out, r.lse, m});
        return r.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = saved_as_is(ctx);
        const c10::DeviceGuard on(s[0].device());
        const int64_t each = s[0].size(1) / s[1].size(1);
        const Tensor q = readable_group(s[0], each), k = readable_group(s[1], 1), v = readable_group(s[2], 1), out = readable_group(s[3], each);
        const Tensor lse = s[4].contiguous(), mask = s[5].defined() ? s[5].contiguous() : Tensor();
        const Tensor go = readable_group(grads[0].to(q.scalar_type()), each);
        variable_list g(4);
        g[0] = empty_like_heads(q);
        if (paired_views(k, v)) {  // slices of one projection: the gradients likewise
            const Tensor both = torch::empty({k.size(0), k.size(2), 2, k.size(1), k.size(3)}, k.options());
            for (int i = 0; i < 2; ++i) g[1 + i] = both.select(2, i).transpose(1, 2);
        } else {
            g[1] = empty_like_heads(k);
            g[2] = empty_like_heads(v);
        }
        spion_cross_attention c = cross_call(q, k, v, out, lse, mask);
        c.dO = heads_of(go);
        c.dQ = heads_of(g[0]);
        c.dK = heads_of(g[1]);
        c.dV = heads_of(g[2]);
        const Tensor ws = cross_workspace(c, true, q);
        void* const stream = reinterpret_cast<void*>(current_stream(q.device().index()));
        check_call(spion_cross_attention_backward(&c, stream) == 0, "spion_cross_attention_backward");
        once_differentiable(g, 3);
        return g;
    }
};

Tensor cross_attention(const Tensor& query, const Tensor& key, const Tensor& value, const c10::optional<Tensor>& key_mask) {
    constexpr int64_t far = int64_t(1) << 29;
    TORCH_CHECK_VALUE(query.dim() == 4 && key.dim() == 4, "heads [B, H, L, d] expected");
    const int64_t B = query.size(0), H = query.size(1), Lq = query.size(2), d = query.size(3), G = key.size(1), Lk = key.size(2);
    TORCH_CHECK_VALUE(key.size(0) == B && key.size(3) == d, "key shape ", key.sizes(), " does not match the query's ", query.sizes());
    TORCH_CHECK_VALUE(value.sizes() == key.sizes(), "value shape ", value.sizes(), " does not match the key's ", key.sizes());
    TORCH_CHECK_VALUE((G == 0) == (H == 0) && (G == 0 || H % G == 0), H, " heads over ", G, " heads of keys: a multiple expected");
    fp32_or_bf16(query, "heads");
    TORCH_CHECK_VALUE(d == 32 || d == 64 || d == 128, "head dimension ", d, ": 32, 64 or 128 expected");
    Tensor mask = key_mask.value_or(Tensor());
    TORCH_CHECK_VALUE(!mask.defined() || (mask.dim() == 2 && mask.size(0) == B && mask.size(1) == Lk), "key mask shape ",
                      mask.defined() ? mask.sizes() : c10::IntArrayRef(), ": [", B, ", ", Lk, "] expected");
    TORCH_CHECK_VALUE(B <= INT_MAX && H <= INT_MAX && Lk <= far && Lq <= far && (G == 0 || H / G * Lq <= far), "sizes out of range");
    for (const Tensor* t : {&query, &key, &value, static_cast<const Tensor*>(&mask)}) on_one_gpu(*t, query);
    TORCH_CHECK_TYPE(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type(), "heads of one type expected");
    const c10::DeviceGuard on(query.device());
    if (mask.defined()) {
        const auto type = mask.scalar_type();
        if (type != torch::kFloat32 && type != torch::kBool && type != torch::kUInt8) mask = mask.ne(0);
        mask = mask.detach().contiguous();
    }
    if (query.numel() == 0 || key.numel() == 0) {  // nothing to attend to, or nobody to
        const Tensor every = torch::ones({}, query.options().dtype(torch::kBool));
        const auto nothing = [&](const Tensor& t) { return t.masked_fill(every, 0.0); };
        return nothing(query) + nothing(key).sum() + nothing(value).sum();
    }
    if (without_node({&query, &key, &value})) return cross_forward(query, key, value, mask).out;
    return CrossNode::apply(query, key, value, mask.defined() ? c10::optional<Tensor>(mask) : c10::nullopt);
}
