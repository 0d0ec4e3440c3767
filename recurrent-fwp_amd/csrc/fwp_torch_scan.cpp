// The selective state space block as C++ autograd functions over the C ABI: the short causal convolution, the selective
// scan, and the norms around a block with its gate, scale and residual addition.  Host code only.
//
// Arguments are checked against one another before the device is, and a rejected call has changed nothing.  States are updated in place and get no
// gradient, as in the fast-weight operators; gradients cannot be differentiated again, and there is no forward-mode derivative.
#include "fwp_torch_rows.hpp"

namespace {

// ------------------------------------------------------------------ short causal convolution

struct ConvFn : torch::autograd::Function<ConvFn> {
    static fwp_conv_args args(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, const at::Tensor &lengths, bool silu) {
        fwp_conv_args a{};
        a.x = view(x);
        a.weight = floats(w);
        a.bias = floats(b);
        a.lengths = whole_numbers(lengths);
        a.type = type_of(x, "X");
        a.silu = silu;
        a.N = (int)x.size(0), a.H = (int)x.size(1), a.L = (int)x.size(2), a.D = (int)x.size(3), a.K = (int)w.size(2);
        return a;
    }
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x_in, const at::Tensor &w_in, const Optional &b_in, const Optional &state_in,
                              const Optional &lengths_in, bool silu) {
        const at::Tensor state = given(state_in);
        if (x_in.dim() != 4) fail("expected a 4-D [N,H,L,D] tensor, got " + std::to_string(x_in.dim()) + "-D");
        const int64_t N = x_in.size(0), H = x_in.size(1), L = x_in.size(2), D = x_in.size(3);
        require_sizes({N, H, L, D});
        type_of(x_in, "X");
        if (w_in.dim() != 3) misfit("weight", w_in, "[H,D,K]");
        const int64_t K = w_in.size(2);
        if (K < 1 || K > 8) fail("a filter has 1 to 8 taps, got " + std::to_string(K));
        const at::Tensor w = parameter(w_in, {H, D, K}, "weight", "[H,D,K]"), b = parameter(given(b_in), {H, D}, "bias", "[H,D]"),
                         lengths = lengths_of(given(lengths_in), N);
        if (state.defined()) {
            if (!same_shape(state, {N, H, K - 1, D})) misfit("state", state, "[N,H,K-1,D]");
            same_type(state, x_in, "state");
            if (!state.is_contiguous() || state.is_neg()) fail("state must be contiguous");
        }
        require_device(x_in);
        same_device(x_in, {w, b, state, lengths});
        const at::Tensor x = rows_of(x_in), y = empty_rows(x);
        if (ctx) may_be_kept({x, w, b, lengths});
        at::Tensor before;
        if (ctx && state.defined()) before = state.detach().clone();
        {
            LaunchGuard guard(x);
            const fwp_conv_args a = args(x, w, b, lengths, silu);
            check(fwp_conv_fwd(&a, state.defined() && K > 1 ? state.data_ptr() : nullptr, out_view(y), stream_of(x)), "fwp_conv_fwd");
        }
        overwritten(state);
        if (ctx) {
            ctx->save_for_backward({x, w, b, before, lengths});
            ctx->saved_data["silu"] = silu;
            ctx->saved_data["params"] = w_in.requires_grad() || (b.defined() && given(b_in).requires_grad());
            ctx->set_materialize_grads(false);
        }
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(6);
        if (!grads[0].defined()) return res;
        once_only();
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &b = saved[2], &before = saved[3], &lengths = saved[4], g = rows_of(grads[0]);
        const fwp_conv_args a = args(x, w, b, lengths, ctx->saved_data["silu"].toBool());
        LaunchGuard guard(x);
        const at::Tensor gx = empty_rows(x), work = scratch(fwp_conv_workspace(a.N, a.H, a.L, a.D, a.K), x);
        at::Tensor gw, gb;
        if (ctx->saved_data["params"].toBool()) gw = room_like(w), gb = at::empty({a.H, a.D}, w.options());
        check(fwp_conv_bwd(&a, before.defined() && a.K > 1 ? before.const_data_ptr() : nullptr, view(g), out_view(gx), floats_out(gw),
                           floats_out(gb), work.data_ptr<float>(), stream_of(x)),
              "fwp_conv_bwd");
        res[0] = gx, res[1] = gw;
        if (b.defined()) res[2] = gb;
        return res;
    }
};

at::Tensor causal_conv(const at::Tensor &x, const at::Tensor &w, const Optional &b, const Optional &state, bool silu, const Optional &lengths) {
    const at::Tensor bias = given(b), state_ = given(state);
    no_tangents({&x, &w, &bias, &state_});
    if (records({&x, &w, &bias})) return ConvFn::apply(x, w, b, state, lengths, silu);
    at::AutoDispatchBelowADInplaceOrView below;
    return ConvFn::forward(nullptr, x, w, b, state, lengths, silu);
}

// ------------------------------------------------------------------ selective scan

struct ScanFn : torch::autograd::Function<ScanFn> {
    static fwp_scan_args args(const at::Tensor &v, const at::Tensor &delta, const at::Tensor &z, const at::Tensor &A, const at::Tensor &D,
                              const at::Tensor &bias, const at::Tensor &lengths, bool softplus) {
        fwp_scan_args a{};
        a.v = view(v), a.delta = view(delta), a.z = view(z);
        a.A = floats(A), a.D = floats(D), a.delta_bias = floats(bias);
        a.lengths = whole_numbers(lengths);
        a.type = type_of(v, "V");
        a.softplus = softplus;
        a.N = (int)v.size(0), a.H = (int)v.size(1), a.L = (int)v.size(2), a.E = (int)A.size(1), a.M = (int)v.size(3);
        return a;
    }
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &v_in,
                              const at::Tensor &delta_in, const at::Tensor &A_in, const Optional &D_in, const Optional &z_in,
                              const Optional &bias_in, const Optional &W_in, const Optional &lengths_in, bool softplus) {
        const at::Tensor z_ = given(z_in), W = given(W_in);
        if (q_in.dim() != 4 || v_in.dim() != 4) fail("expected 4-D [N,H,L,E] queries and [N,H,L,M] values");
        const int64_t N = q_in.size(0), H = q_in.size(1), L = q_in.size(2), E = q_in.size(3), M = v_in.size(3);
        require_sizes({N, H, L, E, M});
        if (E > 64) fail("states of at most 64 keys, got " + std::to_string(E));
        type_of(q_in, "Q");
        for (const auto &[t, name] : {std::pair(&k_in, "K"), std::pair(&v_in, "V"), std::pair(&delta_in, "delta"), std::pair(&z_, "Z")})
            same_type(*t, q_in, name);
        if (!same_shape(k_in, {N, H, L, E})) misfit("K", k_in, "[N,H,L,E] as Q is");
        if (!same_shape(v_in, {N, H, L, M})) misfit("V", v_in, "[N,H,L,M]");
        if (!same_shape(delta_in, {N, H, L, M})) misfit("delta", delta_in, "[N,H,L,M] as V is");
        if (z_.defined() && !same_shape(z_, {N, H, L, M})) misfit("Z", z_, "[N,H,L,M] as V is");
        const at::Tensor A = parameter(A_in, {H, E, M}, "A", "[H,E,M]"), D = parameter(given(D_in), {H, M}, "D", "[H,M]"),
                         bias = parameter(given(bias_in), {H, M}, "delta_bias", "[H,M]"), lengths = lengths_of(given(lengths_in), N);
        if (W.defined() && (!same_shape(W, {N, H, E, M}) || !W.is_contiguous() || W.is_neg() || W.scalar_type() != at::kFloat))
            fail("W must be a contiguous fp32 [N,H,E,M] tensor");
        require_device(q_in);
        same_device(q_in, {k_in, v_in, delta_in, A, D, z_, bias, W, lengths});
        const at::Tensor q = rows_of(q_in, kMaxStep), k = rows_of(k_in, kMaxStep), v = rows_of(v_in, kMaxStep), delta = rows_of(delta_in, kMaxStep),
                         z = rows_of(z_, kMaxStep), out = empty_rows(v);
        fwp_scan_args a = args(v, delta, z, A, D, bias, lengths, softplus);
        a.q = view(q), a.k = view(k);
        if (ctx) may_be_kept({v, delta, z, A, D, bias, lengths, q, k});
        LaunchGuard guard(q);
        at::Tensor saved;
        if (ctx) saved = scratch(fwp_scan_saved_floats(a.N, a.H, a.L, a.E, a.M), v);
        at::Tensor work;
        if (const int64_t n = a.L == 1 ? 0 : fwp_scan_workspace(a.N, a.H, a.L, a.E, a.M, 0)) work = scratch(n, v);
        check(fwp_scan_fwd(&a, floats_out(W), out_view(out), floats_out(saved), floats_out(work), stream_of(q)), "fwp_scan_fwd");
        overwritten(W);
        if (ctx) {
            ctx->save_for_backward({v, delta, z, A, D, bias, lengths, saved, q, k});
            ctx->saved_data["softplus"] = softplus;
            ctx->set_materialize_grads(false);
        }
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(11);
        if (!grads[0].defined()) return res;
        once_only();
        const auto s = ctx->get_saved_variables();
        const at::Tensor &v = s[0], &delta = s[1], &z = s[2], &A = s[3], &D = s[4], &bias = s[5], &lengths = s[6], &saved = s[7];
        const at::Tensor g = rows_of(grads[0], kMaxStep);
        fwp_scan_args a = args(v, delta, z, A, D, bias, lengths, ctx->saved_data["softplus"].toBool());
        a.q = view(s[8]), a.k = view(s[9]);
        LaunchGuard guard(v);
        const at::Tensor gq = empty_rows(s[8]), gk = empty_rows(s[9]), gv = empty_rows(v), gdelta = empty_rows(delta),
                         gz = z.defined() ? empty_rows(z) : at::Tensor(), work = scratch(fwp_scan_workspace(a.N, a.H, a.L, a.E, a.M, 1), v);
        const at::Tensor gA = room_like(A), gD = at::empty({a.H, a.M}, A.options()), gbias = at::empty({a.H, a.M}, A.options());
        check(fwp_scan_bwd(&a, floats(saved), view(g), out_view(gq), out_view(gk), out_view(gv), out_view(gdelta), out_view(gz), floats_out(gA),
                           floats_out(gD), floats_out(gbias), work.data_ptr<float>(), stream_of(v)),
              "fwp_scan_bwd");
        res[0] = gq, res[1] = gk, res[2] = gv, res[3] = gdelta, res[4] = gA;
        if (D.defined()) res[5] = gD;
        res[6] = gz;
        if (bias.defined()) res[7] = gbias;
        return res;
    }
};

at::Tensor selective_scan(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &delta, const at::Tensor &A,
                          const Optional &W, const Optional &D, const Optional &z, const Optional &bias, bool softplus, const Optional &lengths) {
    const at::Tensor D_ = given(D), z_ = given(z), bias_ = given(bias), W_ = given(W);
    no_tangents({&q, &k, &v, &delta, &A, &W_, &D_, &z_, &bias_});
    if (records({&q, &k, &v, &delta, &A, &D_, &z_, &bias_})) return ScanFn::apply(q, k, v, delta, A, D, z, bias, W, lengths, softplus);
    at::AutoDispatchBelowADInplaceOrView below;
    return ScanFn::forward(nullptr, q, k, v, delta, A, D, z, bias, W, lengths, softplus);
}

// ------------------------------------------------------------------ norms around a block

struct ResidualNormFn : torch::autograd::Function<ResidualNormFn> {
    static fwp_norm_args args(const at::Tensor &y, const at::Tensor &x, const at::Tensor &gate, const at::Tensor &scale, const at::Tensor &aw,
                              const at::Tensor &ab, const at::Tensor &bw, const at::Tensor &bb, double eps, bool rms, int64_t act) {
        fwp_norm_args a{};
        a.y = y.const_data_ptr();
        a.x = x.const_data_ptr();
        a.gate = gate.defined() ? gate.const_data_ptr() : nullptr;
        a.scale = floats(scale);
        a.after_weight = floats(aw), a.after_bias = floats(ab), a.before_weight = floats(bw), a.before_bias = floats(bb);
        a.eps = (float)eps;
        a.type = type_of(y, "y");
        a.stream_type = type_of(x, "x");
        a.rms = rms;
        a.act = (int)act;
        a.gate_rows = gate.defined() && gate.size(-1) == 1 && y.size(-1) != 1;
        a.cols = (int)y.size(-1);
        a.rows = (int)(y.numel() / y.size(-1));
        return a;
    }
    static variable_list forward(AutogradContext *ctx, const at::Tensor &y_in, const at::Tensor &x_in, const Optional &gate_in,
                                 const Optional &scale_in, const Optional &aw_in, const Optional &ab_in, const Optional &bw_in,
                                 const Optional &bb_in, double eps, bool rms, int64_t act) {
        const at::Tensor g = given(gate_in);
        if (y_in.dim() < 1 || x_in.sizes() != y_in.sizes()) misfit("x", x_in, "the shape of y");
        const int64_t cols = y_in.size(-1);
        require_sizes({cols});
        require_sizes({y_in.numel() / cols});      // rows; their elements may be more
        if (cols > 8192) fail("rows of at most 8192 columns, got " + std::to_string(cols));
        type_of(y_in, "y");
        if (x_in.scalar_type() != y_in.scalar_type() && x_in.scalar_type() != at::kFloat) fail("x must be fp32 or have the type of y");
        if (g.defined()) {
            std::vector<int64_t> one = y_in.sizes().vec();
            one.back() = 1;
            if (g.sizes() != y_in.sizes() && g.sizes() != at::IntArrayRef(one)) misfit("gate", g, "the shape of y, or one column");
            same_type(g, y_in, "gate");
        }
        const at::Tensor scale = parameter(given(scale_in), {cols}, "scale", "[cols]"), aw = parameter(given(aw_in), {cols}, "after", "[cols]"),
                         ab = parameter(given(ab_in), {cols}, "after's bias", "[cols]"), bw = parameter(given(bw_in), {cols}, "before", "[cols]"),
                         bb = parameter(given(bb_in), {cols}, "before's bias", "[cols]");
        if ((ab.defined() && !aw.defined()) || (bb.defined() && !bw.defined())) fail("a norm's bias without its weight");
        require_device(y_in);
        same_device(y_in, {x_in, g, scale, aw, ab, bw, bb});
        const at::Tensor y = plain(y_in), x = plain(x_in), gate = plain(g), r = at::empty(x.sizes(), x.options());
        at::Tensor n, stats;
        if (bw.defined()) n = at::empty(y.sizes(), y.options());
        const fwp_norm_args a = args(y, x, gate, scale, aw, ab, bw, bb, eps, rms, act);
        LaunchGuard guard(y);
        if (ctx) stats = at::empty({a.rows, 4}, fp32(y));
        check(fwp_residual_norm_fwd(&a, r.data_ptr(), n.defined() ? n.data_ptr() : nullptr, floats_out(stats), stream_of(y)), "fwp_residual_norm_fwd");
        if (ctx) {
            ctx->save_for_backward({y, x, gate, scale, aw, ab, bw, bb, stats});
            ctx->saved_data["eps"] = eps;
            ctx->saved_data["rms"] = rms;
            ctx->saved_data["act"] = act;
            ctx->saved_data["gate"] = g.defined() && g.requires_grad();
            ctx->set_materialize_grads(false);
        }
        return n.defined() ? variable_list{r, n} : variable_list{r};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(11);
        const at::Tensor gr_in = grads[0], gn_in = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!gr_in.defined() && !gn_in.defined()) return res;
        once_only();
        const auto s = ctx->get_saved_variables();
        const at::Tensor &y = s[0], &x = s[1], &gate = s[2], &scale = s[3], &aw = s[4], &ab = s[5], &bw = s[6], &bb = s[7], &stats = s[8];
        const at::Tensor gr = plain(gr_in), gn = plain(gn_in);
        const fwp_norm_args a =
            args(y, x, gate, scale, aw, ab, bw, bb, ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool(), ctx->saved_data["act"].toInt());
        LaunchGuard guard(y);
        res[0] = room_like(y), res[1] = room_like(x);
        if (ctx->saved_data["gate"].toBool()) res[2] = room_like(gate);
        res[3] = room_like(scale), res[4] = room_like(aw), res[5] = room_like(ab), res[6] = room_like(bw), res[7] = room_like(bb);
        const at::Tensor work = scratch(fwp_residual_norm_workspace(a.rows, a.cols), y);
        fwp_norm_grads g{};
        g.gy = res[0].data_ptr();
        g.gx = res[1].data_ptr();
        g.ggate = res[2].defined() ? res[2].data_ptr() : nullptr;
        g.gscale = floats_out(res[3]);
        g.gafter_weight = floats_out(res[4]), g.gafter_bias = floats_out(res[5]);
        g.gbefore_weight = floats_out(res[6]), g.gbefore_bias = floats_out(res[7]);
        check(fwp_residual_norm_bwd(&a, floats(stats), gr.defined() ? gr.const_data_ptr() : nullptr, gn.defined() ? gn.const_data_ptr() : nullptr, &g,
                                    work.data_ptr<float>(), stream_of(y)),
              "fwp_residual_norm_bwd");
        return res;
    }
};

std::pair<at::Tensor, Optional> residual_norm(const at::Tensor &y, const at::Tensor &x, const Optional &gate, const Optional &scale,
                                              const Optional &aw, const Optional &ab, const Optional &bw, const Optional &bb, double eps, bool rms,
                                              int64_t act) {
    const at::Tensor g = given(gate), sc = given(scale), t0 = given(aw), t1 = given(ab), t2 = given(bw), t3 = given(bb);
    variable_list out;
    no_tangents({&y, &x, &g, &sc, &t0, &t1, &t2, &t3});
    if (records({&y, &x, &g, &sc, &t0, &t1, &t2, &t3})) {
        out = ResidualNormFn::apply(y, x, gate, scale, aw, ab, bw, bb, eps, rms, act);
    } else {
        at::AutoDispatchBelowADInplaceOrView below;
        out = ResidualNormFn::forward(nullptr, y, x, gate, scale, aw, ab, bw, bb, eps, rms, act);
    }
    return {out[0], out.size() > 1 ? Optional(out[1]) : std::nullopt};
}

}  // namespace

void bind_scan(py::module_ &m) {
    m.def("causal_conv", &causal_conv, py::arg("X"), py::arg("weight"), py::arg("bias") = py::none(), py::arg("state") = py::none(),
          py::arg("silu") = false, py::arg("lengths") = py::none(), "short causal convolution of every channel; state is updated in place");
    m.def("selective_scan", &selective_scan, py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("delta"), py::arg("A"), py::arg("W") = py::none(),
          py::arg("D") = py::none(), py::arg("Z") = py::none(), py::arg("delta_bias") = py::none(), py::arg("softplus") = false,
          py::arg("lengths") = py::none(), "selective scan; W is updated in place");
    m.def("residual_norm", &residual_norm, "the norms around a block with its gate, scale and residual addition -> (r, n or None)");
}
