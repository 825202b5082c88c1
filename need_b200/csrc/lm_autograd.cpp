// lm_autograd.cpp -- the operators of need_b200.lm over the C ABI of libneed_scan.so
// (module need_b200._lib._lm): the checks of their arguments, allocations and launches,
// and the autograd node of token_log_probs.  need_b200/lm.py documents them.
//
// Nothing is kept between calls: outputs and scratch come from torch's allocator on the
// current stream, so a call can be captured into a graph and run on any stream.
#include "torch_common.h"

using namespace need_torch;
using torch::autograd::AutogradContext;

namespace {

void no_tangent(const char* name, std::initializer_list<const Tensor*> ts) {
    if (has_tangent(ts)) throw std::runtime_error(c10::str(name, " has no forward-mode derivative"));
}

Tensor features(const Tensor& t) {
    return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ------------------------------------------------------------------ linear attention
// [..., heads, features] as the kernels take it; `lead` dims before the heads (1 or 2).
need_heads heads_of(const Tensor& t, int64_t lead) {
    const int64_t h = lead;
    return need_heads{t.const_data_ptr(), t.stride(0), lead == 2 ? t.stride(1) : 0, t.stride(h), t.size(h)};
}
// q, k and v over the same leading dims, and H a multiple of their heads.
void check_heads(const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, int64_t lead, const char* what) {
    bool ok = q.dim() == lead + 2 && k.dim() == lead + 2 && v.dim() == lead + 2 && q.size(-1) == k.size(-1);
    for (int64_t d = 0; ok && d < lead; ++d) ok = q.size(d) == k.size(d) && q.size(d) == v.size(d);
    check_value(ok, "q and k must be ", what, ", heads, dk] and v ", what, ", heads, dv]; got ", q.sizes(), ", ", k.sizes(), ", ",
                v.sizes());
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        throw py::type_error("q, k and v must have one dtype");
    for (const Tensor* t : {&q, &k, &v})
        check_value(t->size(lead) > 0 ? H % t->size(lead) == 0 : H == 0, "the heads of q, k and v must divide the decay's H = ", H,
                    "; got ", q.size(lead), ", ", k.size(lead), ", ", v.size(lead));
}

std::pair<Tensor, OptTensor> linear_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay, double scale,
                                              const OptTensor& seg_, const OptTensor& state_, bool want_final) {
    Tensor seg = or_none(seg_), state = or_none(state_);
    check_tensors("linear_attention", q_, {&k_, &v_, &decay, &seg, &state});
    no_tangent("linear_attention", {&q_, &k_, &v_, &decay, &state});
    check_value(decay.dim() == 1 || decay.dim() == 3, "log_decay must be [H] or [B, T, H]; got ", decay.sizes());
    const int64_t H = decay.size(-1);
    check_heads(q_, k_, v_, H, 2, "[B, T");
    const int64_t B = q_.size(0), T = q_.size(1), dk = q_.size(3), dv = v_.size(3);
    check_value(decay.dim() == 1 || (decay.size(0) == B && decay.size(1) == T), "log_decay must be [H] or [B, T, H] = [", B, ", ", T,
                ", ", H, "]; got ", decay.sizes());
    if (state.defined()) {
        check_value(state.dim() == 4 && state.size(0) == B && state.size(1) == H && state.size(2) == dk && state.size(3) == dv,
                    "state must be [B, H, dk, dv] = [", B, ", ", H, ", ", dk, ", ", dv, "]; got ", state.sizes());
        state = state.to(at::kFloat).contiguous();
    }
    seg = mask_of(seg, B, T);
    On on(q_);
    at::NoGradGuard no_grad;
    const auto ty = q_.scalar_type();
    Tensor final;
    if (B * T * H * dk * dv == 0) {
        if (want_final) final = state.defined() ? state.clone() : at::zeros({B, H, dk, dv}, q_.options().dtype(at::kFloat));
        return {at::zeros({B, T, H, dv}, q_.options()), opt(final)};
    }
    const Tensor q = features(q_), k = features(k_), v = features(v_), ld = decay.to(at::kFloat);
    Tensor out = empty(q, {B, T, H, dv}, ty);
    if (want_final) final = floats(q, {B, H, dk, dv});
    need_linear_attention_args a{};
    a.dtype = dtype_of(ty), a.scale = static_cast<float>(scale);
    a.nb = B, a.T = T, a.H = H, a.dk = dk, a.dv = dv;
    a.q = heads_of(q, 2), a.k = heads_of(k, 2), a.v = heads_of(v, 2);
    a.log_decay = ptr<float>(ld), a.ld_stride_h = ld.stride(-1);
    if (ld.dim() == 3) a.ld_stride_b = ld.stride(0), a.ld_stride_t = ld.stride(1);
    if (seg.defined()) a.seg_start = ptr<uint8_t>(seg), a.seg_stride_b = seg.stride(0), a.seg_stride_t = seg.stride(1);
    a.state = ptr<float>(state), a.final_state = ptr<float>(final);
    a.out = out.data_ptr(), a.out_stride_b = out.stride(0), a.out_stride_t = out.stride(1), a.out_stride_h = out.stride(2);
    const size_t bytes = need_linear_attention_workspace_size(a.dtype, B, T, H, dk, dv);
    Tensor ws;
    if (bytes > 16) ws = scratch(q, bytes), a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    check("need_linear_attention", need_linear_attention(&a, on.stream));
    return {out, opt(final)};
}

Tensor linear_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay, const Tensor& state,
                             double scale, const OptTensor& slot_) {
    Tensor slot = or_none(slot_);
    check_tensors("linear_attention_step", q_, {&k_, &v_, &decay, &state, &slot});
    no_tangent("linear_attention_step", {&q_, &k_, &v_, &decay, &state});
    check_value(decay.dim() == 1 || decay.dim() == 2, "log_decay must be [H] or [N, H]; got ", decay.sizes());
    const int64_t H = decay.size(-1);
    check_heads(q_, k_, v_, H, 1, "[N");
    const int64_t N = q_.size(0), dk = q_.size(2), dv = v_.size(2);
    check_value(decay.dim() == 1 || decay.size(0) == N, "log_decay must be [H] or [N, H] = [", N, ", ", H, "]; got ", decay.sizes());
    check_value(state.dim() == 4 && state.size(1) == H && state.size(2) == dk && state.size(3) == dv,
                "state must be [S, H, dk, dv] = [S, ", H, ", ", dk, ", ", dv, "]; got ", state.sizes());
    if (state.scalar_type() != at::kFloat) throw py::type_error("state must be fp32: it is updated in place");
    const int64_t S = state.size(0);
    check_value((dv <= 1 || state.stride(3) == 1) && (dk <= 1 || state.stride(2) == dv) && (H <= 1 || state.stride(1) == dk * dv) &&
                    (S <= 1 || state.stride(0) >= H * dk * dv),
                "a state's [H, dk, dv] must be contiguous: it is updated in place; got strides ", state.strides());
    if (slot.defined()) {
        if (slot.scalar_type() != at::kInt) throw py::type_error("slot must be int32");
        check_value(slot.dim() == 1 && slot.size(0) == N, "slot must be [N] = [", N, "]; got ", slot.sizes());
        slot = slot.contiguous();
    } else {
        check_value(S >= N, "state holds ", S, " sequences for ", N, " tokens");
    }
    On on(q_);
    at::NoGradGuard no_grad;
    if (N * H * dk * dv == 0) return at::zeros({N, H, dv}, q_.options());
    const Tensor q = features(q_), k = features(k_), v = features(v_), ld = decay.to(at::kFloat);
    Tensor out = empty(q, {N, H, dv}, q.scalar_type());
    need_linear_attention_step_args a{};
    a.dtype = dtype_of(q), a.scale = static_cast<float>(scale);
    a.n = N, a.H = H, a.dk = dk, a.dv = dv;
    a.q = heads_of(q, 1), a.k = heads_of(k, 1), a.v = heads_of(v, 1);
    a.log_decay = ptr<float>(ld), a.ld_stride_h = ld.stride(-1), a.ld_stride_n = ld.dim() == 2 ? ld.stride(0) : 0;
    a.state = ptr<float>(state), a.state_stride = state.stride(0), a.slots = S, a.slot = ptr<int32_t>(slot);
    a.out = out.data_ptr(), a.out_stride_n = out.stride(0), a.out_stride_h = out.stride(1);
    state.unsafeGetTensorImpl()->bump_version();  // or raises: an inference tensor outside its mode
    check("need_linear_attention_step", need_linear_attention_step(&a, on.stream));
    return out;
}

// ------------------------------------------------------------------ residual + norm
// (stream, out, scales or None); group < 0: out in x's dtype, 0: one scale a row.
std::tuple<Tensor, Tensor, OptTensor> residual_norm(const Tensor& x_, const Tensor& y_, const Tensor& weight, double eps,
                                                    double scale, int64_t group) {
    check_tensors("residual_rms_norm", x_, {&y_, &weight});
    no_tangent("residual_rms_norm", {&x_, &y_, &weight});
    check_value(x_.dim() >= 1 && y_.sizes() == x_.sizes(), "x and y must have one shape; got ", x_.sizes(), ", ", y_.sizes());
    if (y_.scalar_type() != x_.scalar_type()) throw py::type_error("x and y must have one dtype");
    const int64_t C = x_.size(-1);
    check_value(weight.numel() == C, "weight must have as many elements as x's last dim; got ", weight.sizes(), " for ", x_.sizes());
    check_value(eps >= 0.0, "eps must be >= 0; got ", eps);
    const bool out8 = group >= 0;
    if (group == 0) group = C;
    On on(x_);
    at::NoGradGuard no_grad;
    const auto ty = x_.scalar_type();
    Tensor stream = empty(x_, x_.sizes(), ty), out = empty(x_, x_.sizes(), out8 ? at::kFloat8_e4m3fn : ty), scales;
    if (out8) {
        auto shape = x_.sizes().vec();
        shape.back() = C == 0 ? 0 : (C + group - 1) / group;
        scales = floats(x_, shape);
    }
    if (x_.numel() == 0) return {stream, out, opt(scales)};
    const Tensor x = even_rows(x_), y = even_rows(y_), w = weight.to(at::kFloat).contiguous();
    need_residual_norm_args a{};
    a.dtype = dtype_of(ty), a.out8 = out8 ? 1 : 0, a.rows = x.numel() / C, a.C = C, a.group = group;
    a.x = x.const_data_ptr(), a.x_stride = row_stride(x), a.y = y.const_data_ptr(), a.y_stride = row_stride(y);
    a.weight = ptr<float>(w), a.eps = eps, a.scale = scale;
    a.stream = stream.data_ptr(), a.stream_stride = C, a.out = out.data_ptr(), a.out_stride = C, a.scales = ptr<float>(scales);
    check("need_residual_rms_norm", need_residual_rms_norm(&a, on.stream));
    return {stream, out, opt(scales)};
}

// ------------------------------------------------------------------ log probabilities
need_token_log_probs_args logp_args(const Tensor& logits, const Tensor& tokens, double temperature) {
    need_token_log_probs_args a{};
    a.dtype = dtype_of(logits), a.V = logits.size(-1), a.rows = logits.numel() / a.V;
    a.logits = logits.const_data_ptr(), a.stride = row_stride(logits);
    a.tokens = static_cast<const int64_t*>(tokens.const_data_ptr()), a.temperature = temperature;
    return a;
}

struct LogProbs {
    Tensor log_prob, entropy, top_log_probs, top_tokens, stats;
};
// logits with even rows, tokens contiguous
LogProbs logp_forward(const Tensor& logits, const Tensor& tokens, double temperature, int64_t top, bool keep) {
    On on(logits);
    LogProbs r;
    need_token_log_probs_args a = logp_args(logits, tokens, temperature);
    r.log_prob = floats(logits, tokens.sizes()), r.entropy = floats(logits, tokens.sizes());
    a.log_prob = ptr<float>(r.log_prob), a.entropy = ptr<float>(r.entropy);
    a.top = static_cast<int32_t>(top);
    if (top > 0) {
        auto shape = tokens.sizes().vec();
        shape.push_back(top);
        r.top_log_probs = floats(logits, shape), r.top_tokens = empty(logits, shape, at::kLong);
        a.top_log_probs = ptr<float>(r.top_log_probs), a.top_tokens = ptr<int64_t>(r.top_tokens);
    }
    if (keep) r.stats = floats(logits, {a.rows, 2}), a.stats = ptr<float>(r.stats);
    const size_t bytes = need_token_log_probs_workspace_size(a.dtype, a.rows, a.V, a.top);
    Tensor ws;
    if (bytes > 16) ws = scratch(logits, bytes), a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
    check("need_token_log_probs", need_token_log_probs(&a, on.stream));
    return r;
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits_, const Tensor& tokens, double temperature, int64_t top) {
        const Tensor logits = even_rows(logits_);
        LogProbs r = logp_forward(logits, tokens, temperature, top, true);
        ctx->save_for_backward({logits, tokens, r.stats, r.entropy});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        if (top == 0) return {r.log_prob, r.entropy};
        ctx->mark_non_differentiable({r.top_log_probs, r.top_tokens});
        return {r.log_prob, r.entropy, r.top_log_probs, r.top_tokens};
    }
    static variable_list backward(AutogradContext* ctx, variable_list go) {
        variable_list s = ctx->get_saved_variables();
        const Tensor& logits = s[0];
        On on(logits);
        need_token_log_probs_args a = logp_args(logits, s[1], ctx->saved_data["temperature"].toDouble());
        const Tensor g = go[0].defined() ? go[0].contiguous() : Tensor(), gh = go[1].defined() ? go[1].contiguous() : Tensor();
        a.stats = ptr<float>(s[2]), a.entropy = ptr<float>(s[3]);
        a.g_log_prob = ptr<float>(g), a.g_entropy = ptr<float>(gh);
        Tensor grad = empty(logits, logits.sizes(), logits.scalar_type());
        a.grad = grad.data_ptr(), a.grad_stride = a.V;
        check("need_token_log_probs_backward", need_token_log_probs_backward(&a, on.stream));
        return once({grad, Tensor(), Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor, OptTensor, OptTensor> token_log_probs(const Tensor& logits, const Tensor& tokens_, double temperature,
                                                                 int64_t top) {
    check_tensors("token_log_probs", logits, {&tokens_});
    check_value(logits.dim() >= 1 && logits.size(-1) > 0 && tokens_.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                "logits must be [..., V] and tokens [...]; got ", logits.sizes(), ", ", tokens_.sizes());
    if (tokens_.scalar_type() != at::kLong && tokens_.scalar_type() != at::kInt) throw py::type_error("tokens must be int64 or int32");
    check_value(temperature >= 1e-30 && temperature <= 1e30, "temperature must lie in [1e-30, 1e30]; got ", temperature);
    check_value(top >= 0 && top <= logits.size(-1), "top must lie in [0, V = ", logits.size(-1), "]; got ", top);
    const Tensor tokens = tokens_.to(at::kLong).contiguous();
    if (logits.numel() == 0) {
        auto shape = tokens.sizes().vec();
        shape.push_back(top);
        const Tensor none = logits.to(at::kFloat).sum(-1);  // no rows; of logits' graph
        if (top == 0) return {none, none, std::nullopt, std::nullopt};
        return {none, none.clone(), floats(logits, shape), empty(logits, shape, at::kLong)};
    }
    if (!wants_grad({&logits}) && !has_tangent({&logits})) {  // nothing to keep
        at::NoGradGuard no_grad;
        LogProbs r = logp_forward(even_rows(logits), tokens, temperature, top, false);
        return {r.log_prob, r.entropy, opt(r.top_log_probs), opt(r.top_tokens)};
    }
    variable_list r = TokenLogProbs::apply(logits, tokens, temperature, top);
    if (top == 0) return {r[0], r[1], std::nullopt, std::nullopt};
    return {r[0], r[1], r[2], r[3]};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("linear_attention", &linear_attention, nogil);
    m.def("linear_attention_step", &linear_attention_step, nogil);
    m.def("residual_norm", &residual_norm, nogil);
    m.def("token_log_probs", &token_log_probs, nogil);
}
