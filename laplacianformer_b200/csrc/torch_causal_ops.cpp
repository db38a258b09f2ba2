// PyTorch-tensor front end of the causal operators: decayed linear attention,
// rotary positions and the sandwich norm (checks, outputs and workspaces on
// the current stream, then the C ABI), and their autograd nodes.
#include "CausalOperators.h"
#include "torch_checks.h"

namespace laplace {
namespace {

at::Tensor last_dense(const at::Tensor& t) {
    return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
// [b, h, n, d] in memory [b, n, h, d]: the heads of a token side by side, as projections read and write them.
at::Tensor fresh_heads(const at::Tensor& like, int64_t d) {
    return fresh({like.size(0), like.size(2), like.size(1), d}, like).transpose(1, 2);
}
void set_strides(int64_t* s, const at::Tensor& t) { s[0] = t.stride(0), s[1] = t.stride(1), s[2] = t.stride(2); }

void check_decay(const at::Tensor& q, const at::Tensor& log_decay, double scale) {
    need_cuda(log_decay, "log_decay");
    TORCH_CHECK(log_decay.device() == q.device(), "log_decay must be on the input's device");
    TORCH_CHECK(log_decay.scalar_type() == at::kFloat && log_decay.dim() == 1 && log_decay.size(0) == q.size(1),
                "log_decay must be float32 with one value per head");
    TORCH_CHECK(scale > 0, "scale must be positive");
}

void check_state(const at::Tensor& s, const at::Tensor& q, int64_t dk, int64_t dv, const char* name) {
    need_cuda(s, name);
    TORCH_CHECK(s.device() == q.device(), std::string(name) + " must be on the input's device");
    TORCH_CHECK(s.scalar_type() == at::kFloat, std::string(name) + " must be float32");
    TORCH_CHECK(s.sizes() == at::IntArrayRef({q.size(0), q.size(1), dk, dv}), std::string(name) + " must be [batch, heads, key size, value size]");
}

struct DecayCall {
    lf_decay_attention_t a{};
    at::Tensor q, k, v, log_decay, state, lengths;
};
DecayCall decay_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay, const at::Tensor& state,
                     const at::Tensor& lengths, double scale) {
    need_cuda(q, "q");
    TORCH_CHECK(q.dim() == 4, "q must be [batch, heads, tokens, size]");
    check_operand(k, q, "k");
    check_shape(k, q.sizes(), "k");
    check_operand(v, q, "v");
    TORCH_CHECK(v.dim() == 4, "v must be [batch, heads, tokens, size]");
    check_shape(v, with_last(q, v.size(3)), "v");
    check_decay(q, log_decay, scale);
    DecayCall c;
    c.a.b = q.size(0), c.a.h = q.size(1), c.a.t = q.size(2), c.a.key_size = q.size(3), c.a.value_size = v.size(3);
    if (state.defined()) check_state(state, q, c.a.key_size, c.a.value_size, "state");
    if (lengths.defined()) {
        need_cuda(lengths, "lengths");
        TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kLong && lengths.dim() == 1 && lengths.size(0) == c.a.b,
                    "lengths must be int64 on the input's device, one per sequence");
    }
    c.q = last_dense(q), c.k = last_dense(k), c.v = last_dense(v);
    c.log_decay = dense(log_decay), c.state = dense(state), c.lengths = dense(lengths);
    c.a.q = ptr(c.q), c.a.k = ptr(c.k), c.a.v = ptr(c.v);
    c.a.log_decay = (const float*)ptr(c.log_decay), c.a.state = (const float*)ptr(c.state), c.a.lengths = (const int64_t*)ptr(c.lengths);
    set_strides(c.a.q_strides, c.q), set_strides(c.a.k_strides, c.k), set_strides(c.a.v_strides, c.v);
    c.a.scale = scale, c.a.dtype = dtype_code(q);
    return c;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> DecayAttention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                          const at::Tensor& log_decay, const at::Tensor& state, const at::Tensor& lengths,
                                                          double scale, bool want_state, at::Tensor* sums) {
    need_cuda(q, "q");
    c10::cuda::CUDAGuard guard(q.device());
    DecayCall c = decay_call(q, k, v, log_decay, state, lengths, scale);
    if (sums) {
        *sums = workspace(lf_decay_attention_sums_size(&c.a), q);
        c.a.sums = (float*)mut(*sums);
    }
    at::Tensor o = fresh_heads(q, c.a.value_size), out;
    if (want_state) out = fresh({c.a.b, c.a.h, c.a.key_size, c.a.value_size}, at::kFloat, q);
    c.a.o = mut(o), c.a.state_out = (float*)mut(out);
    const size_t need = lf_decay_attention_fwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, q);
    raise_on(lf_decay_attention_fwd(&c.a, mut(ws), need, stream_of(q)), "DecayAttention_forward");
    return {o, out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> DecayAttention_backward(
    const at::Tensor& d_o_, const at::Tensor& d_state_, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& log_decay, const at::Tensor& state, const at::Tensor& lengths, double scale, bool need_q, bool need_k, bool need_v,
    bool need_state, const at::Tensor& sums) {
    need_cuda(q, "q");
    c10::cuda::CUDAGuard guard(q.device());
    DecayCall c = decay_call(q, k, v, log_decay, state, lengths, scale);
    if (sums.defined()) c.a.sums = (float*)sums.data_ptr();
    check_operand(d_o_, q, "d_o");
    check_shape(d_o_, v.sizes(), "d_o");
    if (d_state_.defined()) check_state(d_state_, q, c.a.key_size, c.a.value_size, "d_state");
    const at::Tensor d_o = last_dense(d_o_), d_state = dense(d_state_);
    at::Tensor dq, dk, dv, ds;
    if (need_q) dq = fresh_heads(q, c.a.key_size);
    if (need_k) dk = fresh_heads(q, c.a.key_size);
    if (need_v || need_state) dv = fresh_heads(q, c.a.value_size);
    if (need_state) ds = fresh({c.a.b, c.a.h, c.a.key_size, c.a.value_size}, at::kFloat, q);
    c.a.d_o = ptr(d_o), c.a.d_state_out = (const float*)ptr(d_state);
    set_strides(c.a.do_strides, d_o);
    c.a.dq = mut(dq), c.a.dk = mut(dk), c.a.dv = mut(dv), c.a.d_state = (float*)mut(ds);
    const size_t need = lf_decay_attention_bwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, q);
    raise_on(lf_decay_attention_bwd(&c.a, mut(ws), need, stream_of(q)), "DecayAttention_backward");
    return {dq, dk, need_v ? dv : at::Tensor(), ds};
}

at::Tensor DecayAttention_step(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& log_decay_,
                               const at::Tensor& state, double scale) {
    need_cuda(q_, "q");
    TORCH_CHECK(q_.dim() == 3, "q must be [batch, heads, size]");
    check_operand(k_, q_, "k");
    check_shape(k_, q_.sizes(), "k");
    check_operand(v_, q_, "v");
    TORCH_CHECK(v_.dim() == 3, "v must be [batch, heads, size]");
    check_shape(v_, with_last(q_, v_.size(2)), "v");
    check_decay(q_, log_decay_, scale);
    check_state(state, q_, q_.size(2), v_.size(2), "state");
    TORCH_CHECK(state.is_contiguous(), "state must be contiguous: it is updated in place");
    for (const at::Tensor* t : {&q_, &k_, &v_, &log_decay_, &state}) {
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), "decay_attention_step has no forward-mode derivative");
        TORCH_CHECK(!t->requires_grad() || !at::GradMode::is_enabled(), "decay_attention_step has no gradient: call it under torch.no_grad()");
    }
    c10::cuda::CUDAGuard guard(q_.device());
    const at::Tensor q = last_dense(q_), k = last_dense(k_), v = last_dense(v_), log_decay = dense(log_decay_);
    at::Tensor o = fresh(v.sizes(), v);
    lf_decay_step_t a{};
    a.q = ptr(q), a.k = ptr(k), a.v = ptr(v), a.log_decay = (const float*)ptr(log_decay), a.state = (float*)state.data_ptr(), a.o = mut(o);
    a.q_strides[0] = q.stride(0), a.q_strides[1] = q.stride(1), a.k_strides[0] = k.stride(0), a.k_strides[1] = k.stride(1);
    a.v_strides[0] = v.stride(0), a.v_strides[1] = v.stride(1);
    a.b = q.size(0), a.h = q.size(1), a.key_size = q.size(2), a.value_size = v.size(2), a.scale = scale, a.dtype = dtype_code(q);
    raise_on(lf_decay_attention_step(&a, stream_of(q)), "DecayAttention_step");
    // The state was written behind autograd's back: a backward pass that saved it is refused.
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return o;
}

namespace {

struct DecayAttentionNode : torch::autograd::Function<DecayAttentionNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const at::Tensor& log_decay, const c10::optional<at::Tensor>& state,
                                 const c10::optional<at::Tensor>& lengths, double scale, bool want_state) {
        at::AutoDispatchBelowADInplaceOrView below;
        at::Tensor sums;  // (a few matrices per head, where sequences are long and heads few)
        auto [o, out] = DecayAttention_forward(q, k, v, log_decay, opt(state), opt(lengths), scale, want_state, q.requires_grad() ? &sums : nullptr);
        ctx->save_for_backward({q, k, v, log_decay, opt(state), opt(lengths), sums});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        if (want_state) return {o, out};
        return {o};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("decay_attention");
        const auto s = ctx->get_saved_variables();
        const bool st = s[4].defined();
        const bool nq = ctx->needs_input_grad(0), nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2);
        const bool ns = st && ctx->needs_input_grad(4);
        const at::Tensor d_state = g.size() > 1 ? g[1] : at::Tensor();
        at::Tensor dq, dk, dv, ds;
        if (g[0].defined() || d_state.defined()) {
            const at::Tensor d_o = g[0].defined() ? g[0] : at::zeros_like(s[2]);  // only the state was used
            std::tie(dq, dk, dv, ds) = DecayAttention_backward(d_o, d_state, s[0], s[1], s[2], s[3], s[4], s[5],
                                                               ctx->saved_data["scale"].toDouble(), nq, nk, nv, ns, s[6]);
        }
        return {dq, dk, dv, at::Tensor(), ds, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> DecayAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                  const at::Tensor& state, const at::Tensor& lengths, double scale, bool want_state) {
    if (tracked("decay_attention", {&q, &k, &v, &log_decay, &state})) {
        TORCH_CHECK(!log_decay.requires_grad(), "decay_attention has no gradient for log_decay: detach it");
        variable_list out = DecayAttentionNode::apply(q, k, v, log_decay, as_opt(state), as_opt(lengths), scale, want_state);
        return {out[0], out.size() > 1 ? out[1] : at::Tensor()};
    }
    return DecayAttention_forward(q, k, v, log_decay, state, lengths, scale, want_state);
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> Rotary_forward(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& frequencies_,
                                                  const at::Tensor& positions_, int64_t offset, bool interleaved, double magnitude, bool inverse) {
    need_cuda(q_, "q");
    TORCH_CHECK(q_.dim() == 4, "q must be [batch, heads, tokens, size]");
    if (k_.defined()) {
        check_operand(k_, q_, "k");
        TORCH_CHECK(k_.dim() == 4 && k_.size(0) == q_.size(0) && k_.size(2) == q_.size(2) && k_.size(3) == q_.size(3),
                    "k must have q's batch, tokens and size");
    }
    TORCH_CHECK(frequencies_.is_cpu() && frequencies_.scalar_type() == at::kDouble && frequencies_.dim() == 1,
                "frequencies must be a float64 vector on the host (ops.rotary_frequencies)");
    TORCH_CHECK(2 * frequencies_.size(0) <= q_.size(3), "frequencies has more pairs than a head has");
    c10::cuda::CUDAGuard guard(q_.device());
    const at::Tensor q = last_dense(q_), k = last_dense(k_), frequencies = frequencies_.contiguous();
    at::Tensor positions;
    lf_rotary_t a{};
    if (positions_.defined()) {
        need_cuda(positions_, "positions");
        TORCH_CHECK(positions_.device() == q.device() && positions_.scalar_type() == at::kLong, "positions must be int64 on the input's device");
        const bool each = positions_.dim() == 2;
        TORCH_CHECK((positions_.dim() == 1 || (each && positions_.size(0) == q.size(0))) && positions_.size(-1) == q.size(2),
                    "positions must be [tokens] or [batch, tokens]");
        positions = positions_.contiguous();
        a.positions = (const int64_t*)positions.data_ptr();
        a.position_stride = each ? q.size(2) : 0;
    }
    at::Tensor yq = fresh_heads(q, q.size(3)), yk;
    if (k.defined()) yk = fresh_heads(k, k.size(3));
    a.x[0] = ptr(q), a.y[0] = mut(yq), a.heads[0] = q.size(1), set_strides(a.strides[0], q);
    if (k.defined()) a.x[1] = ptr(k), a.y[1] = mut(yk), a.heads[1] = k.size(1), set_strides(a.strides[1], k);
    a.offset = offset, a.frequencies = (const double*)frequencies.data_ptr();
    a.b = q.size(0), a.t = q.size(2), a.size = q.size(3), a.pairs = frequencies.size(0);
    a.magnitude = magnitude, a.interleaved = interleaved, a.inverse = inverse, a.dtype = dtype_code(q);
    raise_on(lf_rotary(&a, stream_of(q)), "Rotary_forward");
    return {yq, yk};
}

namespace {

struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& frequencies,
                                 const c10::optional<at::Tensor>& positions, int64_t offset, bool interleaved, double magnitude) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, z] = Rotary_forward(q, opt(k), frequencies, opt(positions), offset, interleaved, magnitude, false);
        ctx->save_for_backward({opt(positions), frequencies});
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["magnitude"] = magnitude;
        ctx->saved_data["k"] = k.has_value();
        ctx->set_materialize_grads(false);
        if (z.defined()) return {y, z};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("rotary");
        const auto s = ctx->get_saved_variables();
        const bool k = ctx->saved_data["k"].toBool();
        at::Tensor dq = ctx->needs_input_grad(0) ? g[0] : at::Tensor(), dk = k && ctx->needs_input_grad(1) ? g[1] : at::Tensor();
        const bool nq = dq.defined(), nk = dk.defined();
        if (nq || nk) {
            auto [a, b] = Rotary_forward(nq ? dq : dk, nq ? dk : at::Tensor(), s[1], s[0],
                                         ctx->saved_data["offset"].toInt(), ctx->saved_data["interleaved"].toBool(),
                                         ctx->saved_data["magnitude"].toDouble(), true);
            if (nq) dq = a, dk = b;
            else dk = a;
        }
        return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> Rotary(const at::Tensor& q, const at::Tensor& k, const at::Tensor& frequencies, const at::Tensor& positions,
                                          int64_t offset, bool interleaved, double magnitude) {
    if (tracked("rotary", {&q, &k, &frequencies})) {
        TORCH_CHECK(!frequencies.requires_grad(), "rotary has no gradient for frequencies: detach them");
        variable_list out = RotaryNode::apply(q, as_opt(k), frequencies, as_opt(positions), offset, interleaved, magnitude);
        return {out[0], out.size() > 1 ? out[1] : at::Tensor()};
    }
    return Rotary_forward(q, k, frequencies, positions, offset, interleaved, magnitude, false);
}

// ---------------------------------------------------------------------------
// Sandwich norm
// ---------------------------------------------------------------------------
namespace {

struct SandwichCall {
    lf_sandwich_norm_t a{};
    at::Tensor x, weight, residual, gate, next;
};
SandwichCall sandwich_call(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, const at::Tensor& gate,
                           const at::Tensor& next, int64_t activation, double scale, double eps) {
    need_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    check_vector(weight, x, x.size(-1), "weight");
    if (next.defined()) check_vector(next, x, x.size(-1), "next_weight");
    check_operand(residual, x, "residual");
    check_shape(residual, x.sizes(), "residual");
    SandwichCall c;
    c.a.rows = rows_of(x), c.a.cols = x.size(-1);
    if (gate.defined()) {
        // x's leading dimensions, then ones: each gate row serves the rows of the dimensions that are one.
        check_operand(gate, x, "gate");
        bool ok = gate.dim() >= 1 && gate.dim() <= x.dim() && gate.size(-1) == x.size(-1);
        int64_t shared = 1;
        bool all = true;  // so far (from the last dimension on) the gate's dimensions are one
        for (int64_t i = x.dim() - 2, j = gate.dim() - 2; ok && i >= 0; --i, --j) {
            const int64_t n = x.size(i), m = j >= 0 ? gate.size(j) : 1;
            if (all && m == 1) shared *= n;
            else ok = m == n, all = all && n == 1;
        }
        TORCH_CHECK(ok, "gate must have x's shape, with ones in the place of its last dimensions before the channels (or of all of them)");
        c.a.rows_per_gate = shared;
    }
    c.x = dense(x), c.weight = dense(weight), c.residual = dense(residual), c.gate = dense(gate), c.next = dense(next);
    c.a.x = ptr(c.x), c.a.weight = ptr(c.weight), c.a.residual = ptr(c.residual), c.a.gate = ptr(c.gate), c.a.next_weight = ptr(c.next);
    c.a.scale = scale, c.a.eps = eps, c.a.activation = (int32_t)activation, c.a.dtype = dtype_code(x);
    return c;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> SandwichNorm_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual,
                                                                    const at::Tensor& gate, const at::Tensor& next, int64_t activation,
                                                                    double scale, double eps, bool keep) {
    need_cuda(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    SandwichCall c = sandwich_call(x, weight, residual, gate, next, activation, scale, eps);
    at::Tensor s = fresh(x.sizes(), x), y, rstd;
    if (next.defined()) y = fresh(x.sizes(), x);
    if (keep) rstd = fresh({2, c.a.rows}, at::kFloat, x);
    c.a.s = mut(s), c.a.y = mut(y), c.a.rstd = (float*)mut(rstd);
    raise_on(lf_sandwich_norm_fwd(&c.a, stream_of(x)), "SandwichNorm_forward");
    return {s, y, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> SandwichNorm_backward(
    const at::Tensor& ds_, const at::Tensor& dy_, const at::Tensor& x, const at::Tensor& s_, const at::Tensor& rstd, const at::Tensor& weight,
    const at::Tensor& gate, const at::Tensor& next, int64_t activation, double scale, double eps, bool need_x, bool need_w, bool need_r,
    bool need_g, bool need_n) {
    need_cuda(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    SandwichCall c = sandwich_call(x, weight, s_, gate, next, activation, scale, eps);
    TORCH_CHECK(rstd.is_cuda() && rstd.device() == x.device() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == 2 * c.a.rows,
                "rstd must be float32 with two values per row");
    TORCH_CHECK(ds_.defined() || dy_.defined(), "ds or dy is required");
    for (const auto* t : {&ds_, &dy_})
        if (t->defined()) {
            check_operand(*t, x, "a gradient");
            check_shape(*t, x.sizes(), "a gradient");
        }
    TORCH_CHECK(!dy_.defined() || next.defined(), "dy needs next_weight");
    const at::Tensor ds = dense(ds_), dy = dense(dy_);
    at::Tensor dx = maybe(need_x, x.sizes(), x), dr = maybe(need_r, x.sizes(), x), dw = maybe(need_w, weight.sizes(), x), dg, dn;
    if (need_g && gate.defined()) dg = fresh(gate.sizes(), x);
    if (need_n && next.defined()) dn = fresh(next.sizes(), x);
    if (dn.defined() && !dy.defined()) dn.zero_();
    if (dg.defined() && c.a.rows == 0) dg.zero_();
    c.a.residual = nullptr;
    c.a.s = const_cast<void*>(ptr(c.residual)), c.a.rstd = (float*)rstd.data_ptr();
    c.a.ds = ptr(ds), c.a.dy = ptr(dy), c.a.dx = mut(dx), c.a.d_residual = mut(dr), c.a.d_weight = mut(dw), c.a.d_gate = mut(dg);
    c.a.d_next_weight = dy.defined() ? mut(dn) : nullptr;
    const size_t need = lf_sandwich_norm_bwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, x);
    raise_on(lf_sandwich_norm_bwd(&c.a, mut(ws), need, stream_of(x)), "SandwichNorm_backward");
    return {dx, dw, dr, dg, dn};
}

namespace {

struct SandwichNormNode : torch::autograd::Function<SandwichNormNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual,
                                 const c10::optional<at::Tensor>& gate, const c10::optional<at::Tensor>& next, int64_t act, double scale, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [s, y, rstd] = SandwichNorm_forward(x, weight, residual, opt(gate), opt(next), act, scale, eps, true);
        ctx->save_for_backward({x, s, rstd, weight, opt(gate), opt(next)});
        ctx->saved_data["act"] = act;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        if (y.defined()) return {s, y};
        return {s};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("sandwich_norm");
        const auto t = ctx->get_saved_variables();
        const bool gate = t[4].defined(), next = t[5].defined();
        // Inputs of the node: x, weight, residual and, where given, gate and next weight.
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nr = ctx->needs_input_grad(2);
        const bool ng = gate && ctx->needs_input_grad(3), nn = next && ctx->needs_input_grad(3 + gate);
        const at::Tensor dy = next ? g[1] : at::Tensor();
        at::Tensor dx, dw, dr, dg, dn;
        if (g[0].defined() || dy.defined())
            std::tie(dx, dw, dr, dg, dn) = SandwichNorm_backward(g[0], dy, t[0], t[1], t[2], t[3], t[4], t[5], ctx->saved_data["act"].toInt(),
                                                                 ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), nx, nw, nr, ng, nn);
        return {dx, dw, dr, dg, dn, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> SandwichNorm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, const at::Tensor& gate,
                                                const at::Tensor& next, int64_t activation, double scale, double eps) {
    if (tracked("sandwich_norm", {&x, &weight, &residual, &gate, &next})) {
        variable_list out = SandwichNormNode::apply(x, weight, residual, as_opt(gate), as_opt(next), activation, scale, eps);
        return {out[0], out.size() > 1 ? out[1] : at::Tensor()};
    }
    auto [s, y, rstd] = SandwichNorm_forward(x, weight, residual, gate, next, activation, scale, eps, false);
    return {s, y};
}

}  // namespace laplace
