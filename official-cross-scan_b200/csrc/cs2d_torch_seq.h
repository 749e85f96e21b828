// Native host path of the operators over tokens (cs2d/seq.py, cs2d/norm.py): included by cs2d_torch.cpp, whose helpers it uses.

// A backward pass that is recorded into a CUDA graph synchronises with the stream of every leaf's accumulation node.  A node that an
// eager graph on the default stream made, and still holds, would pull that stream into the capture, which ends the process; it is
// refused here, where the forward of the recorded step meets the leaf.
void no_stale_leaves(std::initializer_list<const Tensor *> inputs) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    for (const Tensor *t : inputs) {
        if (!given(*t) || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto s = node->stream();
        CS2D_CHECK(!s || s->device_type() != c10::DeviceType::CUDA || c10::cuda::CUDAStream(*s).stream() != nullptr,
                   "a graph that was built on the default stream still holds a leaf of this recorded step: drop its outputs before the capture");
    }
}
void once_differentiable(const char *what) {
    CS2D_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative: call the backward without create_graph");
}
// Forward-mode differentiation: a tangent would be lost without a word where nothing wants a gradient.
void no_tangents(std::initializer_list<const Tensor *> inputs, const char *what) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : inputs) CS2D_CHECK(!given(*t) || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}
int64_t step_of(const Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
Tensor rows_of(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }
void same_place(const Tensor &t, const Tensor &like, const char *name) {
    CS2D_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the device of the first argument");
}

// ---- gated scan --------------------------------------------------------------------------------------------
struct GatedArgs {
    Tensor u, gate, h0, offsets;
    int64_t form;
    bool weighted;
    int64_t states() const { return given(offsets) ? offsets.size(0) - 1 : u.size(0); }
    int64_t dim() const { return u.size(-1); }
    bool empty() const { return u.numel() == 0; }
};

GatedArgs gated_args(const Tensor &u, const Tensor &gate, const OptT &h0, const OptT &offsets, int64_t form, bool weighted) {
    GatedArgs a{u, gate, opt(h0), opt(offsets), form, weighted};
    CS2D_CHECK(u.is_cuda(), "u must be a CUDA tensor");
    CS2D_CHECK(dtype_code(u.scalar_type()) >= 0, "gated_scan_1d not implemented for input type '", u.scalar_type(), "'");
    same_place(gate, u, "gate");
    CS2D_CHECK(gate.scalar_type() == u.scalar_type(), "gate must have the dtype of u");
    if (given(a.offsets)) {
        same_place(a.offsets, u, "offsets");
        CS2D_CHECK(u.dim() == 2, "with offsets u must have shape (total, dim)");
        CS2D_CHECK(a.offsets.dim() == 1 && a.offsets.size(0) >= 1 && (a.offsets.scalar_type() == at::kInt || a.offsets.scalar_type() == at::kLong),
                   "offsets must be int32 or int64 of shape (sequences + 1)");
        CS2D_CHECK(a.offsets.size(0) - 1 <= INT32_MAX, "too many sequences");
        a.offsets = a.offsets.contiguous();
    } else {
        CS2D_CHECK(u.dim() == 3, "u must have shape (batch, length, dim)");
    }
    CS2D_CHECK(gate.sizes() == u.sizes(), "gate must have the shape of u");
    CS2D_CHECK(u.size(0) <= INT32_MAX && u.size(-1) <= INT32_MAX, "u is too large");
    if (given(a.h0)) {
        same_place(a.h0, u, "h0");
        CS2D_CHECK(a.h0.scalar_type() == at::kFloat, "h0 must be float32");
        CS2D_CHECK(a.h0.sizes() == at::IntArrayRef({a.states(), a.dim()}), "h0 must have shape (", a.states(), ", ", a.dim(), ")");
        a.h0 = rows_of(a.h0);
    }
    a.u = rows_of(u);
    a.gate = rows_of(gate);
    return a;
}

cs2d_gscan gated_problem(const GatedArgs &a) {
    cs2d_gscan p{};
    const bool packed = given(a.offsets);
    const int64_t ld = packed ? 0 : 1;
    p.batch = packed ? 1 : (int32_t)a.u.size(0); p.length = a.u.size(ld); p.dim = (int32_t)a.dim();
    p.io_dtype = dtype_code(a.u.scalar_type()); p.form = (int32_t)a.form; p.weighted = a.weighted;
    p.u = a.u.const_data_ptr(); p.u_bs = packed ? 0 : step_of(a.u, 0); p.u_ls = step_of(a.u, ld);
    p.gate = a.gate.const_data_ptr(); p.gate_bs = packed ? 0 : step_of(a.gate, 0); p.gate_ls = step_of(a.gate, ld);
    if (given(a.h0)) { p.h0 = a.h0.const_data_ptr<float>(); p.h0_bs = step_of(a.h0, 0); }
    if (packed) {
        p.offsets = a.offsets.const_data_ptr();
        p.n_seq = (int32_t)a.states();
        p.offsets64 = a.offsets.scalar_type() == at::kLong;
    }
    return p;
}

Tensor states_f32(const GatedArgs &a, const Tensor &from) {   // the states of rows without tokens: what comes in goes out
    Tensor t = at::empty({a.states(), a.dim()}, a.u.options().dtype(at::kFloat));
    if (given(from)) t.copy_(from); else t.zero_();
    return t;
}

// y, the last states, what a backward reads (undefined for an empty call)
std::tuple<Tensor, Tensor, Tensor> gated_forward(const GatedArgs &a, bool keep) {
    const c10::cuda::CUDAGuard guard(a.u.device());
    Tensor y = at::empty(a.u.sizes(), a.u.options());
    if (a.empty()) return {y, states_f32(a, a.h0), Tensor()};
    const cs2d_gscan p = gated_problem(a);
    const size_t nbytes = cs2d_gscan_saved_bytes(&p, keep);
    CS2D_CHECK(nbytes != 0, "cs2d gated scan: ", cs2d_last_error());
    Tensor last = at::empty({a.states(), a.dim()}, a.u.options().dtype(at::kFloat)), saved = f32(a.u, (int64_t)(nbytes / 4));
    raise_on(cs2d_gscan_fwd(&p, y.data_ptr(), p.length * p.dim, p.dim, last.data_ptr<float>(), saved.data_ptr(), keep, stream_of(a.u)), "gated scan");
    return {y, last, saved};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &gate, const OptT &h0, const OptT &offsets, int64_t form,
                                 bool weighted) {
        at::AutoDispatchBelowADInplaceOrView below;
        const GatedArgs a = gated_args(u, gate, h0, offsets, form, weighted);
        auto [y, last, saved] = gated_forward(a, true);
        ctx->saved_data["form"] = form;
        ctx->saved_data["weighted"] = weighted;
        ctx->save_for_backward({u, gate, opt(h0), opt(offsets), saved});
        ctx->set_materialize_grads(false);
        return {y, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        once_differentiable("gated_scan_1d");
        const auto s = ctx->get_saved_variables();
        variable_list none(6);
        if (!go[0].defined() && !go[1].defined()) return none;
        const OptT h0 = given(s[2]) ? OptT(s[2]) : OptT(), offsets = given(s[3]) ? OptT(s[3]) : OptT();
        const GatedArgs a = gated_args(s[0], s[1], h0, offsets, ctx->saved_data["form"].toInt(), ctx->saved_data["weighted"].toBool());
        const c10::cuda::CUDAGuard guard(a.u.device());
        Tensor du = at::empty(a.u.sizes(), a.u.options()), dgate = at::empty(a.u.sizes(), a.u.options()), dh0;
        Tensor dlast = go[1].defined() ? rows_of(go[1]) : Tensor();
        if (a.empty()) return {du, dgate, given(a.h0) ? states_f32(a, dlast) : Tensor(), Tensor(), Tensor(), Tensor()};
        const Tensor dy = go[0].defined() ? rows_of(go[0]) : at::zeros(a.u.sizes(), a.u.options());
        if (given(a.h0)) dh0 = at::empty({a.states(), a.dim()}, a.u.options().dtype(at::kFloat));
        const cs2d_gscan p = gated_problem(a);
        const bool packed = given(a.offsets);
        raise_on(cs2d_gscan_bwd(&p, dy.const_data_ptr(), packed ? 0 : step_of(dy, 0), step_of(dy, packed ? 0 : 1),
                                given(dlast) ? dlast.const_data_ptr<float>() : nullptr, given(dlast) ? step_of(dlast, 0) : 0, s[4].const_data_ptr(),
                                du.data_ptr(), dgate.data_ptr(), given(dh0) ? dh0.data_ptr<float>() : nullptr, stream_of(a.u)), "gated scan backward");
        return {du, dgate, dh0, Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> py_gated_scan(const Tensor &u, const Tensor &gate, const OptT &h0, const OptT &offsets, int64_t form, bool weighted) {
    const Tensor h = opt(h0);
    no_tangents({&u, &gate, &h}, "gated_scan_1d");
    if (at::GradMode::is_enabled() && (wants_grad(u) || wants_grad(gate) || wants_grad(h))) {
        no_stale_leaves({&u, &gate, &h});
        const variable_list r = GatedScan::apply(u, gate, h0, offsets, form, weighted);
        return {r[0], r[1]};
    }
    at::NoGradGuard no_grad;
    auto [y, last, saved] = gated_forward(gated_args(u, gate, h0, offsets, form, weighted), false);
    return {y, last};
}

Tensor py_gated_step(const Tensor &u, const Tensor &gate, const Tensor &h, int64_t form, bool weighted) {
    CS2D_CHECK(!(at::GradMode::is_enabled() && (wants_grad(u) || wants_grad(gate) || wants_grad(h))),
               "gated_scan_step has no gradient: call it under torch.no_grad(), or gated_scan_1d on one token");
    no_tangents({&u, &gate, &h}, "gated_scan_step");
    at::NoGradGuard no_grad;
    CS2D_CHECK(u.is_cuda(), "u must be a CUDA tensor");
    CS2D_CHECK(dtype_code(u.scalar_type()) >= 0, "gated_scan_step not implemented for input type '", u.scalar_type(), "'");
    same_place(gate, u, "gate");
    same_place(h, u, "h");
    CS2D_CHECK(u.dim() == 2, "u must have shape (batch, dim)");
    CS2D_CHECK(gate.scalar_type() == u.scalar_type() && gate.sizes() == u.sizes(), "gate must have the dtype and the shape of u");
    CS2D_CHECK(h.scalar_type() == at::kFloat && h.sizes() == u.sizes(), "h must be float32 with the shape of u");
    CS2D_CHECK((h.stride(1) == 1 || h.size(1) <= 1) && (h.size(0) <= 1 || h.stride(0) >= h.size(1)),
               "h is updated in place: its rows must be contiguous and must not overlap");
    CS2D_CHECK(!h.is_inference() || c10::InferenceMode::is_enabled(), "h is an inference tensor: outside inference mode it cannot be updated in place");
    CS2D_CHECK(u.size(0) <= INT32_MAX && u.size(1) <= INT32_MAX, "u is too large");
    const c10::cuda::CUDAGuard guard(u.device());
    const Tensor ur = rows_of(u), gr = rows_of(gate);
    Tensor y = at::empty(u.sizes(), u.options());
    if (u.numel() == 0) return y;
    cs2d_gscan p{};
    p.batch = (int32_t)u.size(0); p.dim = (int32_t)u.size(1);
    p.io_dtype = dtype_code(u.scalar_type()); p.form = (int32_t)form; p.weighted = weighted;
    p.u = ur.const_data_ptr(); p.u_bs = step_of(ur, 0);
    p.gate = gr.const_data_ptr(); p.gate_bs = step_of(gr, 0);
    raise_on(cs2d_gscan_step(&p, y.data_ptr(), p.dim, h.data_ptr<float>(), step_of(h, 0), stream_of(u)), "gated scan step");
    h.unsafeGetTensorImpl()->bump_version();
    return y;
}

// ---- layer norm ----------------------------------------------------------------------------------------------
// Rows of a tensor (..., dim) as (outer, inner): outer is the first dimension of three or more, inner all between it and the channels.
struct Rows { int64_t os, is, cs; };
bool as_rows(const Tensor &t, Rows &r) {
    const int64_t n = t.dim();
    r = Rows{n >= 3 ? step_of(t, 0) : 0, 0, t.size(-1) > 1 ? t.stride(-1) : 1};
    int64_t need = 0;   // stride that the next dimension outwards must have; 0: free
    for (int64_t d = n - 2; d >= (n >= 3 ? 1 : 0); --d) {
        if (t.size(d) <= 1) continue;
        if (need == 0) r.is = t.stride(d);
        else if (t.stride(d) != need) return false;
        need = t.stride(d) * t.size(d);
        if (need == 0) return false;   // an expanded dimension
    }
    return true;
}
struct NormArgs { Tensor x, weight, bias, gate; double eps; };

NormArgs norm_args(const Tensor &x, const OptT &weight, const OptT &bias, const OptT &gate, double eps) {
    NormArgs a{x, opt(weight), opt(bias), opt(gate), eps};
    CS2D_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    CS2D_CHECK(dtype_code(x.scalar_type()) >= 0, "layer_norm not implemented for input type '", x.scalar_type(), "'");
    CS2D_CHECK(x.dim() >= 1, "x must have shape (..., dim)");
    CS2D_CHECK(x.size(-1) >= 1 && x.size(-1) <= INT32_MAX, "layer_norm needs at least one channel");
    CS2D_CHECK(eps >= 0, "eps must not be negative");
    for (const auto &m : {std::make_pair("weight", &a.weight), std::make_pair("bias", &a.bias)}) {
        Tensor &t = *m.second;
        if (!given(t)) continue;
        same_place(t, x, m.first);
        CS2D_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), m.first, " must have shape (", x.size(-1), ")");
        CS2D_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), m.first, " must be float32 or have the dtype of x");
        t = t.contiguous();
    }
    if (given(a.weight) && given(a.bias)) CS2D_CHECK(a.weight.scalar_type() == a.bias.scalar_type(), "weight and bias must have one dtype");
    Rows r;
    if (!as_rows(a.x, r) || (r.cs != 1 && r.is != 1)) a.x = a.x.contiguous();
    if (given(a.gate)) {
        same_place(a.gate, x, "gate");
        CS2D_CHECK(a.gate.scalar_type() == x.scalar_type(), "gate must have the dtype of x");
        CS2D_CHECK(a.gate.sizes() == x.sizes(), "gate must have the shape of x");
        if (!as_rows(a.gate, r) || r.cs != 1) a.gate = a.gate.contiguous();
    }
    return a;
}
cs2d_norm norm_problem(const NormArgs &a) {
    cs2d_norm p{};
    const int64_t n = a.x.dim();
    p.dim = (int32_t)a.x.size(-1); p.io_dtype = dtype_code(a.x.scalar_type()); p.eps = (float)a.eps;
    p.param_dtype = given(a.weight) ? dtype_code(a.weight.scalar_type()) : given(a.bias) ? dtype_code(a.bias.scalar_type()) : CS2D_F32;
    p.outer = n >= 3 ? a.x.size(0) : 1;
    p.inner = a.x.numel() / p.dim / p.outer;
    Rows r;
    as_rows(a.x, r);
    p.x = a.x.const_data_ptr(); p.x_os = r.os; p.x_is = r.is; p.x_cs = r.cs;
    if (given(a.gate)) {
        as_rows(a.gate, r);
        p.gate = a.gate.const_data_ptr(); p.g_os = r.os; p.g_is = r.is;
    }
    if (given(a.weight)) p.weight = a.weight.const_data_ptr();
    if (given(a.bias)) p.bias = a.bias.const_data_ptr();
    return p;
}
std::pair<Tensor, Tensor> norm_forward(const NormArgs &a, bool keep) {
    const c10::cuda::CUDAGuard guard(a.x.device());
    Tensor y = at::empty(a.x.sizes(), a.x.options()), stats;
    if (a.x.numel() == 0) return {y, stats};
    const cs2d_norm p = norm_problem(a);
    if (keep) stats = f32(a.x, p.outer * p.inner * 2);
    raise_on(cs2d_norm_fwd(&p, y.data_ptr(), fp(stats), stream_of(a.x)), "layer norm");
    return {y, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptT &weight, const OptT &bias, const OptT &gate, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        const NormArgs a = norm_args(x, weight, bias, gate, eps);
        auto r = norm_forward(a, true);
        ctx->saved_data["eps"] = eps;
        ctx->save_for_backward({x, opt(weight), opt(bias), opt(gate), r.second});
        return r.first;
    }
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        once_differentiable("layer_norm");
        if (!go[0].defined()) return variable_list(5);
        const auto s = ctx->get_saved_variables();
        const auto o = [&](int i) { return given(s[i]) ? OptT(s[i]) : OptT(); };
        const NormArgs a = norm_args(s[0], o(1), o(2), o(3), ctx->saved_data["eps"].toDouble());
        const c10::cuda::CUDAGuard guard(a.x.device());
        Tensor dw, db, dz, scratch;
        const auto parameters = [&]() {
            if (given(a.weight)) dw = at::empty(a.weight.sizes(), a.weight.options());
            if (given(a.bias)) db = at::empty(a.bias.sizes(), a.bias.options());
        };
        if (given(a.gate)) dz = at::empty(a.gate.sizes(), a.gate.options());
        if (a.x.numel() == 0) {
            parameters();
            if (given(dw)) dw.zero_();
            if (given(db)) db.zero_();
            return {at::empty(a.x.sizes(), a.x.options()), dw, db, dz, Tensor()};
        }
        const cs2d_norm p = norm_problem(a);
        Rows r;
        Tensor dy = go[0];
        if (!as_rows(dy, r) || r.cs != 1) { dy = dy.contiguous(); as_rows(dy, r); }
        Tensor dx;
        int64_t os = p.inner * p.dim, is = p.dim, cs = 1;
        if (p.x_cs == 1) {
            dx = at::empty(a.x.sizes(), a.x.options());
        } else {   // a channel-major image: its gradient is one too
            const int64_t n = a.x.dim();
            c10::SmallVector<int64_t, 6> strides(n);
            strides[n - 1] = p.inner;
            int64_t run = 1;
            for (int64_t d = n - 2; d >= (n >= 3 ? 1 : 0); --d) { strides[d] = run; run *= a.x.size(d); }
            if (n >= 3) strides[0] = p.inner * p.dim;
            dx = at::empty_strided(a.x.sizes(), strides, a.x.options());
            is = 1; cs = p.inner;
        }
        const size_t nbytes = cs2d_norm_bwd_scratch_bytes(&p);
        CS2D_CHECK(nbytes != 0, "cs2d layer norm: ", cs2d_last_error());
        const int64_t ns = (int64_t)(nbytes / 4), d4 = (p.dim + 3) / 4 * 4;
        if (p.param_dtype == CS2D_F32 && ns + 2 * d4 <= (1 << 16)) {   // small problems: one allocation (what a caller keeps keeps no more than 256 KB alive)
            scratch = f32(a.x, ns + 2 * d4);
            if (given(a.weight)) dw = part_of(scratch, ns, {p.dim});
            if (given(a.bias)) db = part_of(scratch, ns + d4, {p.dim});
        } else {
            parameters();
            scratch = f32(a.x, ns);
        }
        raise_on(cs2d_norm_bwd(&p, dy.const_data_ptr(), r.os, r.is, s[4].const_data_ptr<float>(), scratch.data_ptr(), dx.data_ptr(), os, is, cs,
                               given(dz) ? dz.data_ptr() : nullptr, given(dw) ? dw.data_ptr() : nullptr, given(db) ? db.data_ptr() : nullptr,
                               stream_of(a.x)), "layer norm backward");
        return {dx, dw, db, dz, Tensor()};
    }
};

Tensor py_layer_norm(const Tensor &x, const OptT &weight, const OptT &bias, const OptT &gate, double eps) {
    const Tensor w = opt(weight), b = opt(bias), z = opt(gate);
    no_tangents({&x, &w, &b, &z}, "layer_norm");
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b) || wants_grad(z))) {
        no_stale_leaves({&x, &w, &b, &z});
        return LayerNorm::apply(x, weight, bias, gate, eps);
    }
    at::NoGradGuard no_grad;
    return norm_forward(norm_args(x, weight, bias, gate, eps), false).first;
}
