// train_autograd.cpp -- the autograd nodes of need_b200.train, over the C ABI
// of libneed_scan.so (module need_b200._lib._train).
//
// A training pass of a small call is bound by the host, not the GPU: as Python
// autograd functions over ctypes these operators took 160 to 390 us a pass
// where their kernels took 20 to 60.  The nodes, the checks of their arguments,
// the argument structs and the allocations are therefore here (70 to 130 us, of
// which torch's engine is 30 to 40); need_b200/train.py documents the operators.
//
// Nothing is kept between calls: outputs, saved tensors and scratch come from
// torch's allocator on the current stream, so a call can be captured into a
// graph and run on any stream.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "need_scan.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int64_t kSpan = 64, kGroup = 64;  // need_scan_train_chunk_len(), need_scan_train_group()

template <class... Args>
void check_value(bool ok, const Args&... args) {
    if (!ok) throw py::value_error(c10::str(args...));
}
void check(const char* fn, int rc) {
    if (rc != NEED_OK)
        throw std::runtime_error(c10::str(fn, " failed (status ", rc, "): ", need_last_error()));
}

int32_t dtype_of(at::ScalarType t) {
    return t == at::kFloat ? NEED_F32 : t == at::kBFloat16 ? NEED_BF16 : NEED_F16;
}
int32_t dtype_of(const Tensor& t) { return dtype_of(t.scalar_type()); }

using OptTensor = std::optional<Tensor>;
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// CUDA tensors of one device, x of a dtype the kernels take.
void check_tensors(const char* name, const Tensor& x, std::initializer_list<const Tensor*> others) {
    if (!x.is_cuda())
        throw std::runtime_error(c10::str(name, " takes CUDA tensors only (no CPU fallback); got ", x.sizes(), " on ", x.device()));
    for (const Tensor* t : others)
        if (t->defined() && t->device() != x.device())
            throw std::runtime_error("all tensors must be on the same CUDA device (no CPU fallback)");
    const auto ty = x.scalar_type();
    if (ty != at::kFloat && ty != at::kBFloat16 && ty != at::kHalf)
        throw py::type_error(c10::str(name, " takes fp32, bf16 or f16 data; got ", c10::toString(ty)));
}
// The reset mask as the kernels read it.
Tensor mask_of(const Tensor& seg, int64_t B, int64_t T) {
    if (!seg.defined()) return seg;
    check_value(seg.dim() == 2 && seg.size(0) == B && seg.size(1) == T, "seg_start must be [B, T] = [", B, ", ", T,
                "]; got ", seg.sizes());
    return seg.scalar_type() == at::kByte ? seg : seg.ne(0).to(at::kByte);
}

Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

// `t` with channel stride 1; a copy if its channels are apart.
Tensor channels(const Tensor& t) {
    return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.clone(at::MemoryFormat::Contiguous);
}
// A new [B, T, C] tensor whose rows start 16-byte aligned: contiguous, or with
// rows apart by C rounded up.
Tensor rows_like(const Tensor& like, at::ScalarType type, int64_t B, int64_t T, int64_t C) {
    const int64_t n = 16 / static_cast<int64_t>(c10::elementSize(type)), pitch = (C + n - 1) / n * n;
    if (pitch == C) return empty(like, {B, T, C}, type);
    return at::detail::empty_strided_cuda({B, T, C}, {T * pitch, pitch, 1}, type, like.device());
}
Tensor scratch(const Tensor& like, size_t bytes) { return empty(like, {static_cast<int64_t>(bytes)}, at::kByte); }
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return empty(like, shape, at::kFloat); }
template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
need_view view(const Tensor& t) { return need_view{t.const_data_ptr(), t.stride(0), 0, t.stride(1)}; }

// The current stream of t's device, which is made current for the guard's life.
struct On {
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index())) {}
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream stream;
};

bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Whether one of them carries a forward-mode tangent.  A node refuses it; a plain launch
// would drop it.
bool has_tangent(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) return true;
    return false;
}

// Under create_graph: gradients of these gradients raise instead of being left out.
variable_list once(variable_list g) {
    if (!at::GradMode::is_enabled()) return g;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "need_b200: the training operators have no second derivative", static_cast<int>(g.size()));
    variable_list in;
    for (Tensor& t : g) in.push_back(t.defined() ? t.detach().requires_grad_() : t);
    return (*node)(std::move(in));
}

// ------------------------------------------------------------------ the recurrences
struct ScanShape {
    int64_t form, B, T, C;
    double dt_min, dt_max;
    bool ckpt;
};

need_scan_train_args scan_args(const ScanShape& s, int32_t dtype, const Tensor& seg, const Tensor& d_skip,
                               const Tensor& states) {
    need_scan_train_args a{};
    a.form = static_cast<int32_t>(s.form), a.dtype = dtype, a.checkpoint = s.ckpt ? 1 : 0;
    a.nb = s.B, a.T = s.T, a.C = s.C, a.dt_min = s.dt_min, a.dt_max = s.dt_max;
    a.d_skip = ptr<float>(d_skip), a.states = ptr<float>(states);
    if (seg.defined()) a.seg_start = ptr<uint8_t>(seg), a.seg_stride_b = seg.stride(0), a.seg_stride_t = seg.stride(1);
    return a;
}

struct ScanOut {
    Tensor out, final, states, q, qs;
};

// Runs the forward; x: the streams in in[] order, each as channels() gives it.
ScanOut scan_forward(const ScanShape& s, const variable_list& x, const Tensor& seg, const Tensor& h0,
                     const Tensor& d_skip) {
    On on(x[0]);
    ScanOut r;
    const int64_t nin = static_cast<int64_t>(x.size());
    r.out = rows_like(x[0], x[0].scalar_type(), s.B, s.T, s.C);
    r.final = floats(x[0], {s.B, s.C});
    r.states = floats(x[0], {s.B, (s.T + kSpan - 1) / kSpan, s.C});
    need_scan_train_args a = scan_args(s, dtype_of(x[0]), seg, d_skip, r.states);
    for (int64_t k = 0; k < nin; ++k) a.in[k] = view(x[k]);
    if (s.ckpt) {
        const int64_t groups = (s.C + kGroup - 1) / kGroup;
        r.q = scratch(x[0], nin * s.B * s.T * groups * kGroup);
        r.qs = scratch(x[0], nin * s.B * s.T * groups);
        a.ckpt_values = ptr<uint8_t>(r.q), a.ckpt_scales = ptr<uint8_t>(r.qs);
    }
    a.h0 = ptr<float>(h0);
    a.out = r.out.data_ptr(), a.out_stride_b = r.out.stride(0), a.out_stride_t = r.out.stride(1);
    a.h_final = ptr<float>(r.final);
    const Tensor ws = scratch(x[0], need_scan_train_workspace_size(a.form, a.dtype, a.checkpoint, 0, s.B, s.T, s.C));
    a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    check("need_scan_train_forward", need_scan_train_forward(&a, on.stream));
    return r;
}

struct ScanTrain : torch::autograd::Function<ScanTrain> {
    static variable_list forward(AutogradContext* ctx, int64_t form, bool ckpt, double dt_min, double dt_max,
                                 const OptTensor& seg_, const OptTensor& h0_, const OptTensor& d_skip_,
                                 const Tensor& x0, const Tensor& x1, const Tensor& x2, const OptTensor& x3_,
                                 const OptTensor& x4_) {
        const Tensor seg = or_none(seg_), h0 = or_none(h0_), d_skip = or_none(d_skip_);
        const Tensor x3 = or_none(x3_), x4 = or_none(x4_);  // none for the GATED form
        variable_list x{channels(x0), channels(x1), channels(x2)};
        if (x3.defined()) x.insert(x.end(), {channels(x3), channels(x4)});
        const ScanShape s{form, x0.size(0), x0.size(1), x0.size(2), dt_min, dt_max, ckpt};
        ScanOut r = scan_forward(s, x, seg, h0, d_skip);
        variable_list saved{r.states, seg, d_skip};
        if (ckpt) saved.insert(saved.end(), {r.q, r.qs});
        else saved.insert(saved.end(), x.begin(), x.end());
        ctx->save_for_backward(std::move(saved));
        auto& d = ctx->saved_data;
        d["form"] = form, d["ckpt"] = ckpt, d["lo"] = dt_min, d["hi"] = dt_max, d["h0"] = h0.defined();
        d["B"] = s.B, d["T"] = s.T, d["C"] = s.C, d["dtype"] = static_cast<int64_t>(x0.scalar_type());
        ctx->set_materialize_grads(false);
        return {r.out, r.final};
    }

    static variable_list backward(AutogradContext* ctx, variable_list go) {
        auto& d = ctx->saved_data;
        const ScanShape s{d["form"].toInt(),    d["B"].toInt(),     d["T"].toInt(), d["C"].toInt(),
                          d["lo"].toDouble(), d["hi"].toDouble(), d["ckpt"].toBool()};
        variable_list saved = ctx->get_saved_variables();
        const Tensor &states = saved[0], &seg = saved[1], &d_skip = saved[2];
        On on(states);
        const auto type = static_cast<at::ScalarType>(d["dtype"].toInt());
        const int nin = s.form == NEED_FORM_GATED ? 3 : 5;
        const Tensor gout = go[0].defined() ? channels(go[0]) : at::zeros({s.B, s.T, s.C}, states.options().dtype(type));
        const Tensor gfin = go[1].defined() ? go[1].contiguous() : Tensor();
        need_scan_train_args a = scan_args(s, dtype_of(gout), seg, d_skip, states);
        if (s.ckpt) a.ckpt_values = ptr<uint8_t>(saved[3]), a.ckpt_scales = ptr<uint8_t>(saved[4]);
        else
            for (int k = 0; k < nin; ++k) a.in[k] = view(saved[3 + k]);
        a.gout = view(gout), a.g_final = ptr<float>(gfin);
        variable_list g(12);  // as forward's arguments
        for (int k = 0; k < nin; ++k) {
            g[7 + k] = rows_like(states, type, s.B, s.T, s.C);
            a.grad[k] = g[7 + k].data_ptr();
        }
        a.grad_stride_b = g[7].stride(0), a.grad_stride_t = g[7].stride(1);
        if (d["h0"].toBool()) g[5] = floats(states, {s.B, s.C}), a.grad_h0 = ptr<float>(g[5]);
        if (d_skip.defined()) g[6] = floats(states, {s.C}), a.grad_d = ptr<float>(g[6]);
        const Tensor ws = scratch(states, need_scan_train_workspace_size(a.form, a.dtype, a.checkpoint, 1, s.B, s.T, s.C));
        a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
        check("need_scan_train_backward", need_scan_train_backward(&a, on.stream));
        return once(std::move(g));
    }
};

// (out, final state); x in the C ABI's in[] order, of one shape and device.
variable_list scan_train(int64_t form, variable_list x, const Tensor& seg_, Tensor h0, Tensor d_skip,
                         double dt_min, double dt_max, bool ckpt) {
    const Tensor& x2 = x[2];  // x or u
    const int64_t B = x2.size(0), T = x2.size(1), C = x2.size(2);
    if (h0.defined()) {
        check_value(h0.dim() == 2 && h0.size(0) == B && h0.size(1) == C, "h0 must be [B, C] = [", B, ", ", C, "]; got ",
                    h0.sizes());
        h0 = h0.to(at::kFloat).contiguous();
    }
    if (d_skip.defined()) d_skip = d_skip.to(at::kFloat).contiguous();
    const Tensor seg = mask_of(seg_, B, T);
    if (x2.numel() == 0) {  // nothing to scan: the state passes through
        Tensor out = x[0];
        for (size_t k = 1; k < x.size(); ++k) out = out * x[k];
        if (d_skip.defined()) out = (out * d_skip).to(x2.scalar_type());
        return {out, h0.defined() ? h0.clone() : at::zeros({B, C}, x2.options().dtype(at::kFloat))};
    }
    const Tensor none;
    const Tensor &x3 = x.size() > 3 ? x[3] : none, &x4 = x.size() > 4 ? x[4] : none;
    const std::initializer_list<const Tensor*> all{&h0, &d_skip, &x[0], &x[1], &x2, &x3, &x4};
    if (!wants_grad(all) && !has_tangent(all)) {  // nothing to keep
        at::NoGradGuard no_grad;
        for (Tensor& t : x) t = channels(t);
        ScanOut r = scan_forward({form, B, T, C, dt_min, dt_max, false}, x, seg, h0, d_skip);
        return {r.out, r.final};
    }
    return ScanTrain::apply(form, ckpt, dt_min, dt_max, opt(seg), opt(h0), opt(d_skip), x[0], x[1], x2, opt(x3), opt(x4));
}

variable_list gated_scan_train(const Tensor& x, const Tensor& z, const Tensor& g, const OptTensor& seg_,
                               const OptTensor& h0_, bool ckpt) {
    const Tensor seg = or_none(seg_), h0 = or_none(h0_);
    check_tensors("gated_scan_train", x, {&z, &g, &seg, &h0});
    check_value(x.dim() == 3 && z.sizes() == x.sizes() && g.sizes() == x.sizes(),
                "x, decay_logit and gate_logit must have the same [B, T, C] shape");
    const auto ty = x.scalar_type();
    return scan_train(NEED_FORM_GATED, {z.to(ty), g.to(ty), x}, seg, h0, Tensor(), 0.0, 0.0, ckpt);
}

variable_list ssd_scan_train(const Tensor& u, const Tensor& bg, const Tensor& cg, const Tensor& dt, const Tensor& og,
                             const Tensor& d_skip, double dt_min, double dt_max, const OptTensor& seg_,
                             const OptTensor& h0_, bool ckpt) {
    const Tensor seg = or_none(seg_), h0 = or_none(h0_);
    check_tensors("ssd_scan_train", u, {&bg, &cg, &dt, &og, &d_skip, &seg, &h0});
    bool same = u.dim() == 3;
    for (const Tensor* t : {&bg, &cg, &dt, &og}) same = same && t->sizes() == u.sizes();
    check_value(same, "u, b_gate, c_gate, dt_raw and out_gate must have the same [B, T, D] shape");
    check_value(d_skip.numel() == u.size(2), "d_skip must have D=", u.size(2), " elements; got ", d_skip.sizes());
    check_value(dt_min >= 0.0 && dt_max >= dt_min && dt_max <= 1e30, "0 <= dt_min <= dt_max (finite) expected; got ", dt_min, ", ",
                dt_max);
    const auto ty = u.scalar_type();
    return scan_train(NEED_FORM_SSD, {dt.to(ty), bg.to(ty), u, cg.to(ty), og.to(ty)}, seg, h0,
                      d_skip.dim() == 1 ? d_skip : d_skip.reshape(-1), dt_min, dt_max, ckpt);
}

// ------------------------------------------------------------------ the conv
need_conv_train_args conv_args(const Tensor& u, const Tensor& w, const Tensor& b, const Tensor& seg) {
    need_conv_train_args a{};
    a.dtype = dtype_of(u), a.K = static_cast<int32_t>(w.size(-1));
    a.nb = u.size(0), a.T = u.size(1), a.C = u.size(2);
    a.u = u.const_data_ptr(), a.u_stride_b = u.stride(0), a.u_stride_t = u.stride(1);
    a.weight = ptr<float>(w), a.bias = ptr<float>(b);
    if (seg.defined()) a.seg_start = ptr<uint8_t>(seg), a.seg_stride_b = seg.stride(0), a.seg_stride_t = seg.stride(1);
    return a;
}

struct ConvTrain : torch::autograd::Function<ConvTrain> {
    static Tensor forward(AutogradContext* ctx, const Tensor& u_, const Tensor& w_, const OptTensor& b_,
                          const OptTensor& seg_) {
        // the weight [C, K] or [C, 1, K], as it is
        const Tensor u = channels(u_), w = w_.contiguous(), seg = or_none(seg_);
        const Tensor b = b_.has_value() ? b_->contiguous() : Tensor();
        On on(u);
        Tensor out = rows_like(u, u.scalar_type(), u.size(0), u.size(1), u.size(2));
        need_conv_train_args a = conv_args(u, w, b, seg);
        a.out = out.data_ptr(), a.out_stride_b = out.stride(0), a.out_stride_t = out.stride(1);
        check("need_conv_silu_train_forward", need_conv_silu_train_forward(&a, on.stream));
        ctx->save_for_backward({u, w, b, seg});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list go) {
        variable_list s = ctx->get_saved_variables();
        const Tensor &u = s[0], &w = s[1], &b = s[2], &seg = s[3];
        On on(u);
        const Tensor gout = channels(go[0]);
        need_conv_train_args a = conv_args(u, w, b, seg);
        a.gout = gout.const_data_ptr(), a.gout_stride_b = gout.stride(0), a.gout_stride_t = gout.stride(1);
        Tensor gu = rows_like(u, u.scalar_type(), a.nb, a.T, a.C), gwb = floats(u, {a.C, a.K + 1});
        const Tensor ws = scratch(u, need_conv_silu_train_workspace_size(a.K, a.nb, a.T, a.C));
        a.grad_u = gu.data_ptr(), a.out_stride_b = gu.stride(0), a.out_stride_t = gu.stride(1);
        a.grad_wb = ptr<float>(gwb);
        a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
        check("need_conv_silu_train_backward", need_conv_silu_train_backward(&a, on.stream));
        const Tensor gw = w.dim() == 3 ? gwb.unsqueeze(1).narrow(2, 0, a.K) : gwb.narrow(1, 0, a.K);
        return once({gu, gw, b.defined() ? gwb.select(1, a.K) : Tensor(), Tensor()});
    }
};

Tensor conv_train(const Tensor& u, const Tensor& weight, const OptTensor& bias, const OptTensor& seg_) {
    Tensor b = or_none(bias), seg = or_none(seg_);
    check_tensors("ssd_conv_silu_train", u, {&weight, &b, &seg});
    check_value(u.dim() == 3, "u must be [B, T, C]; got ", u.sizes());
    const int64_t B = u.size(0), T = u.size(1), C = u.size(2);
    check_value((weight.dim() == 2 || (weight.dim() == 3 && weight.size(1) == 1)) && weight.size(0) == C,
                "weight must be [C, 1, K] or [C, K] with C=", C, "; got ", weight.sizes());
    check_value(weight.size(-1) >= 1 && weight.size(-1) <= 4, "1 to 4 taps expected; got ", weight.size(-1));
    check_value(!b.defined() || (b.dim() == 1 && b.size(0) == C), "bias must be [C] = [", C, "]; got ",
                b.defined() ? b.sizes() : u.sizes());
    seg = mask_of(seg, B, T);
    const Tensor w = weight.to(at::kFloat);
    if (b.defined()) b = b.to(at::kFloat);
    if (u.numel() == 0) {
        Tensor out = u * w.flatten(1).sum(1);
        return (b.defined() ? out + b : out).to(u.scalar_type());
    }
    return ConvTrain::apply(u, w, opt(b), opt(seg));
}

// ------------------------------------------------------------------ the norm
need_norm_train_args norm_args(int32_t dtype, int64_t n, int64_t C, const Tensor& w, const Tensor& rstd, double eps,
                               bool ckpt) {
    need_norm_train_args a{};
    a.dtype = dtype, a.checkpoint = ckpt ? 1 : 0, a.rows = n, a.C = C;
    a.weight = ptr<float>(w), a.rstd = ptr<float>(rstd), a.eps = eps;
    return a;
}
// The distance of t's rows (all dims but the last, as one) where they are evenly
// apart with channel stride 1; else 0.
int64_t row_stride(const Tensor& t) {
    if (t.stride(-1) != 1 && t.size(-1) > 1) return 0;
    int64_t step = 0, next = 0;  // of the innermost dim of more than one, and what the next must be
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (step == 0) step = t.stride(d);
        else if (t.stride(d) != next) return 0;
        if (step <= 0) return 0;
        next = t.stride(d) * t.size(d);
    }
    return step == 0 ? t.size(-1) : step;
}
Tensor even_rows(const Tensor& t) { return row_stride(t) != 0 ? t : t.clone(at::MemoryFormat::Contiguous); }

struct NormTrain : torch::autograd::Function<NormTrain> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, double eps, bool ckpt) {
        const Tensor x = even_rows(x_), w = w_.contiguous();
        const int64_t C = x.size(-1), n = x.numel() / C;
        On on(x);
        Tensor out = empty(x, x.sizes(), x.scalar_type()), rstd = floats(x, {n}), q, qs;
        need_norm_train_args a = norm_args(dtype_of(x), n, C, w, rstd, eps, ckpt);
        a.x = x.const_data_ptr(), a.x_stride = row_stride(x), a.out = out.data_ptr(), a.out_stride = C;
        if (ckpt) {
            const int64_t groups = (C + kGroup - 1) / kGroup;
            q = scratch(x, n * groups * kGroup), qs = scratch(x, n * groups);
            a.ckpt_values = ptr<uint8_t>(q), a.ckpt_scales = ptr<uint8_t>(qs);
        }
        check("need_rms_norm_train_forward", need_rms_norm_train_forward(&a, on.stream));
        if (ckpt) ctx->save_for_backward({w, rstd, q, qs});
        else ctx->save_for_backward({w, rstd, x});
        ctx->saved_data["eps"] = eps;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list go) {
        variable_list s = ctx->get_saved_variables();
        const bool ckpt = s.size() == 4;
        On on(s[0]);
        const Tensor gout = even_rows(go[0]);
        const int64_t C = gout.size(-1), n = s[1].numel();
        need_norm_train_args a = norm_args(dtype_of(gout), n, C, s[0], s[1], ctx->saved_data["eps"].toDouble(), ckpt);
        if (ckpt) a.ckpt_values = ptr<uint8_t>(s[2]), a.ckpt_scales = ptr<uint8_t>(s[3]);
        else a.x = s[2].const_data_ptr(), a.x_stride = row_stride(s[2]);
        a.gout = gout.const_data_ptr(), a.gout_stride = row_stride(gout);
        Tensor gx = empty(gout, gout.sizes(), gout.scalar_type()), gw = floats(gout, s[0].sizes());
        const Tensor ws = scratch(gout, need_rms_norm_train_workspace_size(n, C));
        a.grad_x = gx.data_ptr(), a.out_stride = C, a.grad_weight = ptr<float>(gw);
        a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
        check("need_rms_norm_train_backward", need_rms_norm_train_backward(&a, on.stream));
        return once({gx, gw, Tensor(), Tensor()});
    }
};

Tensor norm_train(const Tensor& x, const Tensor& weight, double eps, bool ckpt) {
    check_tensors("rms_norm_train", x, {&weight});
    check_value(x.dim() >= 1 && weight.numel() == x.size(-1),
                "weight must have as many elements as x's last dim; got ", weight.sizes(), " for ", x.sizes());
    check_value(eps >= 0.0, "eps must be >= 0; got ", eps);
    const Tensor w = weight.to(at::kFloat);
    if (x.numel() == 0) return (x * w.flatten()).to(x.scalar_type());
    return NormTrain::apply(x, w, eps, ckpt && wants_grad({&x, &w}));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("gated_scan_train", &gated_scan_train, nogil);
    m.def("ssd_scan_train", &ssd_scan_train, nogil);
    m.def("conv_train", &conv_train, nogil);
    m.def("norm_train", &norm_train, nogil);
}
