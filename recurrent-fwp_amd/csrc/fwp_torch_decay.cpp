// The block of a decayed sum rule as C++ autograd functions over the C ABI: the sum rule with a decay for each head, rotary positions, and the norm of groups
// of channels with its gate.  Host code only; checks, states and gradients as in the selective state space block.
#include "fwp_torch_rows.hpp"

namespace {

// ------------------------------------------------------------------ decayed sum rule

constexpr int64_t kMost = FWP_DSUM_MAX_STEP;

struct DecayedSumFn : torch::autograd::Function<DecayedSumFn> {
    static fwp_dsum_args args(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &decay, const at::Tensor &lengths,
                              double scale) {
        fwp_dsum_args a{};
        a.q = view(q), a.k = view(k), a.v = view(v);
        a.per_head = decay.dim() == 1;
        a.decay = floats(decay);
        if (a.per_head) a.dH = decay.stride(0);
        else a.dN = decay.stride(0), a.dH = decay.stride(1), a.dL = decay.stride(2);
        a.lengths = whole_numbers(lengths);
        a.scale = (float)scale;
        a.type = type_of(q, "Q");
        a.N = (int)q.size(0), a.H = (int)decay.size(a.per_head ? 0 : 1), a.L = (int)q.size(2), a.E = (int)q.size(3), a.M = (int)v.size(3);
        a.HQ = (int)q.size(1), a.HK = (int)k.size(1), a.HV = (int)v.size(1);
        return a;
    }
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &v_in, const at::Tensor &decay_in,
                              const Optional &W_in, const Optional &lengths_in, double scale) {
        const at::Tensor W = given(W_in);
        if (q_in.dim() != 4 || k_in.dim() != 4 || v_in.dim() != 4) fail("expected 4-D [N,H,L,E] queries and keys and [N,H,L,M] values");
        if (decay_in.dim() != 1 && decay_in.dim() != 3) misfit("log_decay", decay_in, "[H] or [N,H,L]");
        const int64_t N = q_in.size(0), H = decay_in.size(decay_in.dim() == 1 ? 0 : 1), L = q_in.size(2), E = q_in.size(3), M = v_in.size(3);
        require_sizes({N, H, L, E, M, q_in.size(1), k_in.size(1), v_in.size(1)});
        if (E > 128) fail("states of at most 128 keys, got " + std::to_string(E));
        if (M > 65536) fail("at most 65536 values a head, got " + std::to_string(M));
        type_of(q_in, "Q");
        same_type(k_in, q_in, "K");
        same_type(v_in, q_in, "V");
        if (!same_shape(k_in, {N, k_in.size(1), L, E})) misfit("K", k_in, "[N,.,L,E] as Q is");
        if (!same_shape(v_in, {N, v_in.size(1), L, M})) misfit("V", v_in, "[N,.,L,M]");
        if (decay_in.scalar_type() != at::kFloat) fail("log_decay must be fp32");
        if (decay_in.dim() == 3 && !same_shape(decay_in, {N, H, L})) misfit("log_decay", decay_in, "[H] or [N,H,L]");
        for (const auto &[t, name] : {std::pair(&q_in, "Q"), std::pair(&k_in, "K"), std::pair(&v_in, "V")})
            if (H % t->size(1)) fail(std::string("the heads of ") + name + " must divide those of log_decay: " + std::to_string(t->size(1)) + " beside " + std::to_string(H));
        const at::Tensor lengths = lengths_of(given(lengths_in), N);
        if (W.defined() && (!same_shape(W, {N, H, E, M}) || !W.is_contiguous() || W.is_neg() || W.scalar_type() != at::kFloat))
            fail("W must be a contiguous fp32 [N,H,E,M] tensor");
        require_device(q_in);
        same_device(q_in, {k_in, v_in, decay_in, W, lengths});
        const at::Tensor q = rows_of(q_in, kMost), k = rows_of(k_in, kMost), v = rows_of(v_in, kMost), decay = decay_in.is_neg() ? plain(decay_in) : decay_in,
                         out = empty_rows(v, H, kMost);
        const fwp_dsum_args a = args(q, k, v, decay, lengths, scale);
        if (ctx) may_be_kept({q, k, v, decay, lengths});
        LaunchGuard guard(q);
        at::Tensor saved, work;
        if (ctx) saved = scratch(fwp_decayed_sum_saved_floats(a.type, a.N, a.H, a.L, a.E, a.M), q);
        if (const int64_t n = a.L == 1 ? 0 : fwp_decayed_sum_workspace(&a, 0)) work = scratch(n, q);
        check(fwp_decayed_sum_fwd(&a, floats_out(W), out_view(out), floats_out(saved), floats_out(work), stream_of(q)), "fwp_decayed_sum_fwd");
        overwritten(W);
        if (ctx) {
            ctx->save_for_backward({q, k, v, decay, lengths, saved});
            ctx->saved_data["scale"] = scale;
            ctx->set_materialize_grads(false);
        }
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(7);
        if (!grads[0].defined()) return res;
        once_only();
        const auto s = ctx->get_saved_variables();
        const at::Tensor &q = s[0], &k = s[1], &v = s[2], &decay = s[3], &lengths = s[4], &saved = s[5], g = rows_of(grads[0], kMost);
        const fwp_dsum_args a = args(q, k, v, decay, lengths, ctx->saved_data["scale"].toDouble());
        LaunchGuard guard(q);
        const at::Tensor work = scratch(fwp_decayed_sum_workspace(&a, 1), q);
        res[0] = empty_rows(q, 0, kMost), res[1] = empty_rows(k, 0, kMost), res[2] = empty_rows(v, 0, kMost), res[3] = at::empty(decay.sizes(), decay.options());
        check(fwp_decayed_sum_bwd(&a, floats(saved), view(g), out_view(res[0]), out_view(res[1]), out_view(res[2]), floats_out(res[3]),
                                  work.data_ptr<float>(), stream_of(q)),
              "fwp_decayed_sum_bwd");
        return res;
    }
};

at::Tensor decayed_sum(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &decay, const Optional &W, double scale,
                       const Optional &lengths) {
    const at::Tensor W_ = given(W);
    no_tangents({&q, &k, &v, &decay, &W_});
    if (records({&q, &k, &v, &decay})) return DecayedSumFn::apply(q, k, v, decay, W, lengths, scale);
    at::AutoDispatchBelowADInplaceOrView below;
    return DecayedSumFn::forward(nullptr, q, k, v, decay, W, lengths, scale);
}

// ------------------------------------------------------------------ rotary positions

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    // q and, where there is one, k, turned
    static variable_list turned(const at::Tensor &q_in, const at::Tensor &k_in, const at::Tensor &frequencies, const at::Tensor &positions,
                                const at::Tensor &lengths, bool interleaved, double scale, bool inverse) {
        const at::Tensor q = rows_of(q_in), k = rows_of(k_in);
        variable_list out{empty_rows(q)};
        if (k.defined()) out.push_back(empty_rows(k));
        fwp_rotary_args a{};
        a.q = view(q), a.k = view(k);
        a.frequencies = frequencies.const_data_ptr<double>();
        a.positions = whole_numbers(positions), a.lengths = whole_numbers(lengths);
        a.scale = (float)scale;
        a.type = type_of(q, "Q");
        a.interleaved = interleaved, a.inverse = inverse, a.each_step = positions.defined() && positions.dim() == 2;
        a.N = (int)q.size(0), a.HQ = (int)q.size(1), a.HK = k.defined() ? (int)k.size(1) : 0, a.L = (int)q.size(2), a.D = (int)q.size(3);
        a.pairs = (int)frequencies.size(0);
        LaunchGuard guard(q);
        check(fwp_rotary(&a, out_view(out[0]), out_view(k.defined() ? out[1] : at::Tensor()), stream_of(q)), "fwp_rotary");
        return out;
    }
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const Optional &k_in, const at::Tensor &frequencies_in,
                                 const Optional &positions_in, const Optional &lengths_in, bool interleaved, double scale) {
        const at::Tensor k = given(k_in), p = given(positions_in);
        if (q.dim() != 4 || (k.defined() && k.dim() != 4)) fail("expected 4-D [N,H,L,D] queries and keys");
        const int64_t N = q.size(0), L = q.size(2), D = q.size(3);
        require_sizes({N, q.size(1), L, D});
        type_of(q, "Q");
        if (k.defined()) {
            require_sizes({k.size(1)});
            same_type(k, q, "K");
            if (!same_shape(k, {N, k.size(1), L, D})) misfit("K", k, "[N,.,L,D] as Q is");
        }
        if (D > 65536) fail("at most 65536 channels a head, got " + std::to_string(D));
        if (frequencies_in.dim() != 1 || frequencies_in.scalar_type() != at::kDouble) fail("frequencies must be an fp64 tensor [pairs]");
        const int64_t pairs = frequencies_in.size(0);
        if (pairs < 1 || 2 * pairs > D) fail("1 to D / 2 frequencies, got " + std::to_string(pairs) + " for " + std::to_string(D) + " channels");
        if (frequencies_in.requires_grad()) fail("there is no gradient of the frequencies: detach them");
        if (p.defined() && (p.scalar_type() != at::kLong || (!same_shape(p, {N}) && !same_shape(p, {N, L})))) fail("positions must be an int64 tensor [N] or [N,L]");
        const at::Tensor lengths = lengths_of(given(lengths_in), N), frequencies = plain(frequencies_in), positions = plain(p);
        require_device(q);
        same_device(q, {k, frequencies, positions, lengths});
        if (ctx) may_be_kept({frequencies, positions, lengths});
        const variable_list out = turned(q, k, frequencies, positions, lengths, interleaved, scale, false);
        if (ctx) {
            ctx->save_for_backward({frequencies, positions, lengths});
            ctx->saved_data["interleaved"] = interleaved;
            ctx->saved_data["scale"] = scale;
            ctx->set_materialize_grads(false);
        }
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(7);
        const at::Tensor gq = grads[0], gk = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!gq.defined() && !gk.defined()) return res;
        once_only();
        const auto s = ctx->get_saved_variables();
        const variable_list out = turned(gq.defined() ? gq : gk, gq.defined() ? gk : at::Tensor(), s[0], s[1], s[2], ctx->saved_data["interleaved"].toBool(),
                                         ctx->saved_data["scale"].toDouble(), true);
        if (gq.defined()) res[0] = out[0];
        if (gk.defined()) res[1] = out.back();
        return res;
    }
};

std::pair<at::Tensor, Optional> rotary(const at::Tensor &q, const Optional &k, const at::Tensor &frequencies, const Optional &positions, bool interleaved,
                                       double scale, const Optional &lengths) {
    const at::Tensor k_ = given(k);
    no_tangents({&q, &k_, &frequencies});
    variable_list out;
    if (records({&q, &k_})) {
        out = RotaryFn::apply(q, k, frequencies, positions, lengths, interleaved, scale);
    } else {
        at::AutoDispatchBelowADInplaceOrView below;
        out = RotaryFn::forward(nullptr, q, k, frequencies, positions, lengths, interleaved, scale);
    }
    return {out[0], out.size() > 1 ? Optional(out[1]) : std::nullopt};
}

// ------------------------------------------------------------------ norm of groups of channels

struct GroupNormFn : torch::autograd::Function<GroupNormFn> {
    // [..., channels] whose rows lie one step apart in memory, from the first to the last; a copy where they do not
    static at::Tensor even_rows(const at::Tensor &t) {
        if (!t.defined()) return t;
        bool even = !t.is_neg() && (t.size(-1) == 1 || t.stride(-1) == 1);
        int64_t inner = -1;      // the next axis inwards that has more than one row
        for (int64_t i = t.dim() - 2; even && i >= 0; i--) {
            if (t.size(i) == 1) continue;
            if (inner >= 0) even = t.stride(i) == t.size(inner) * t.stride(inner);
            inner = i;
        }
        return even ? t : t.resolve_neg().clone(at::MemoryFormat::Contiguous);
    }
    static int64_t step_of(const at::Tensor &t) {
        for (int64_t i = t.dim() - 2; i >= 0; i--)
            if (t.size(i) > 1) return t.stride(i);
        return t.size(-1);
    }
    static fwp_group_norm_args args(const at::Tensor &x, const at::Tensor &gate, const at::Tensor &w, const at::Tensor &b, int64_t groups, double eps, bool rms,
                                    int64_t act) {
        fwp_group_norm_args a{};
        a.x = x.const_data_ptr();
        a.x_step = step_of(x);
        if (gate.defined()) a.gate = gate.const_data_ptr(), a.gate_step = step_of(gate);
        a.weight = floats(w), a.bias = floats(b);
        a.eps = (float)eps;
        a.type = type_of(x, "X");
        a.rms = rms, a.act = (int)act;
        a.groups = (int)groups, a.size = (int)(x.size(-1) / groups), a.rows = (int)(x.numel() / x.size(-1));
        return a;
    }
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x_in, const Optional &gate_in, const Optional &w_in, const Optional &b_in, int64_t groups,
                              double eps, bool rms, int64_t act) {
        const at::Tensor g = given(gate_in);
        if (x_in.dim() < 1) fail("expected [..., channels]");
        const int64_t C = x_in.size(-1);
        require_sizes({C});
        require_sizes({x_in.numel() / C});
        type_of(x_in, "X");
        if (groups < 1 || C % groups) fail("the channels must be a multiple of the groups: " + std::to_string(C) + " in " + std::to_string(groups));
        if (C / groups > 1024 || C > 65536) fail("groups of at most 1024 channels, 65536 in all, got " + std::to_string(groups) + " of " + std::to_string(C / groups));
        if (g.defined() && g.sizes() != x_in.sizes()) misfit("gate", g, "the shape of X");
        same_type(g, x_in, "gate");
        const at::Tensor w = parameter(given(w_in), {C}, "weight", "[channels]"), b = parameter(given(b_in), {C}, "bias", "[channels]");
        require_device(x_in);
        same_device(x_in, {g, w, b});
        const at::Tensor x = even_rows(x_in), gate = even_rows(g), y = at::empty(x.sizes(), x.options());
        if (ctx) may_be_kept({x, gate, w, b});
        LaunchGuard guard(x);
        const fwp_group_norm_args a = args(x, gate, w, b, groups, eps, rms, act);
        check(fwp_group_norm_fwd(&a, y.data_ptr(), stream_of(x)), "fwp_group_norm_fwd");
        if (ctx) {
            ctx->save_for_backward({x, gate, w, b});
            ctx->saved_data["groups"] = groups;
            ctx->saved_data["eps"] = eps;
            ctx->saved_data["rms"] = rms;
            ctx->saved_data["act"] = act;
            ctx->set_materialize_grads(false);
        }
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list res(8);
        if (!grads[0].defined()) return res;
        once_only();
        const auto s = ctx->get_saved_variables();
        const at::Tensor &x = s[0], &gate = s[1], &w = s[2], &b = s[3], gy = plain(grads[0]);
        const fwp_group_norm_args a = args(x, gate, w, b, ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool(),
                                           ctx->saved_data["act"].toInt());
        LaunchGuard guard(x);
        res[0] = room_like(x), res[1] = room_like(gate), res[2] = room_like(w), res[3] = room_like(b);
        at::Tensor work;
        if (w.defined() || b.defined()) work = scratch(fwp_group_norm_workspace(a.type, a.rows, a.groups, a.size), x);
        check(fwp_group_norm_bwd(&a, gy.const_data_ptr(), res[0].data_ptr(), gate.defined() ? res[1].data_ptr() : nullptr, floats_out(res[2]),
                                 floats_out(res[3]), floats_out(work), stream_of(x)),
              "fwp_group_norm_bwd");
        return res;
    }
};

at::Tensor group_norm(const at::Tensor &x, int64_t groups, const Optional &w, const Optional &b, const Optional &gate, double eps, bool rms, int64_t act) {
    const at::Tensor w_ = given(w), b_ = given(b), gate_ = given(gate);
    no_tangents({&x, &w_, &b_, &gate_});
    if (records({&x, &w_, &b_, &gate_})) return GroupNormFn::apply(x, gate, w, b, groups, eps, rms, act);
    at::AutoDispatchBelowADInplaceOrView below;
    return GroupNormFn::forward(nullptr, x, gate, w, b, groups, eps, rms, act);
}

}  // namespace

void bind_decay(py::module_ &m) {
    m.def("decayed_sum", &decayed_sum, py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("log_decay"), py::arg("W") = py::none(), py::arg("scale") = 1.0,
          py::arg("lengths") = py::none(), "the sum rule with a decay for each head; W is updated in place");
    m.def("rotary", &rotary, py::arg("Q"), py::arg("K"), py::arg("frequencies"), py::arg("positions") = py::none(), py::arg("interleaved") = false,
          py::arg("scale") = 1.0, py::arg("lengths") = py::none(), "rotary positions -> (q, k or None)");
    m.def("group_norm", &group_norm, py::arg("X"), py::arg("groups"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
          py::arg("gate") = py::none(), py::arg("eps") = 1e-5, py::arg("rms") = false, py::arg("act") = 0, "norm of groups of channels with a gate or an activation");
}
