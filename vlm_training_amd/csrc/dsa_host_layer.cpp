// Host side of the operators of a gated-delta-rule layer: argument checks, allocations, the C-ABI calls and the autograd
// nodes, as dsa_host.cpp has them for the attention.
#include "dsa_host.h"

#include <torch/csrc/autograd/functions/utils.h>

namespace {

using at::ScalarType;

// The tensor itself where its rows can be read 16 bytes at a time in place, a contiguous copy otherwise
Tensor rows16(const Tensor &x) {
    const bool ok = x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) % 8 == 0) && (x.size(0) == 1 || (x.stride(0) % 8 == 0 && x.stride(0) <= DSA_DELTA_MAX_ROW)) &&
                    aligned16(x));
    if (ok) return x;
    const Tensor c = x.contiguous();
    return aligned16(c) ? c : c.clone();
}
bool half_or_float(const Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// With create_graph a backward's results carry this node: it leads to all that they depend on - the operator's inputs and the gradients that came in - and stands for
// second derivatives, which the operators do not have.  Asked for them it raises; first derivatives are what they are without it.
struct NoSecondDerivative : torch::autograd::Node {
    const char *what;
    NoSecondDerivative(const char *what, torch::autograd::edge_list &&next) : Node(std::move(next)), what(what) {}
    variable_list apply(variable_list &&) override {
        TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": second derivatives are not implemented");
    }
};
variable_list once(variable_list results, const variable_list &grads, const char *what) {
    if (!at::GradMode::is_enabled()) return results;
    const auto node = torch::autograd::get_current_node();
    torch::autograd::edge_list next = node->next_edges();
    for (const Tensor &g : grads)
        if (g.defined() && g.requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(g));
    const auto end = std::make_shared<NoSecondDerivative>(what, std::move(next));
    for (Tensor &t : results)
        if (t.defined()) torch::autograd::set_history(t, end);
    return results;
}

// ---- gated delta rule ---------------------------------------------------------------------------------------------------
struct DeltaInputs {
    Tensor q, k, v, a, b, a_log, dt_bias, cu;
    dsa_delta_args args;
};

DeltaInputs delta_inputs(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &a, const Tensor &b, const Tensor &a_log, const Tensor &dt_bias,
                         const Tensor &cu, std::optional<double> scale, bool l2_norm) {
    for (const Tensor *t : {&q, &k, &v, &a, &b, &a_log, &dt_bias, &cu}) {
        need_gpu(*t);
        if (t->defined()) same_device(q, *t, "a tensor");
    }
    check_bf16_thd(q, "q");
    check_bf16_thd(k, "k");
    check_bf16_thd(v, "v");
    const int64_t T = q.size(0), Hk = q.size(1), Dk = q.size(2), Hv = v.size(1), Dv = v.size(2);
    TORCH_CHECK_VALUE(k.sizes() == q.sizes() && v.size(0) == T, "q/k/v shapes disagree: ", q.sizes(), " ", k.sizes(), " ", v.sizes());
    TORCH_CHECK_VALUE(Hk >= 1 && Hv >= 1 && Hv % Hk == 0, "the value heads (", Hv, ") must be a multiple of the key heads (", Hk, ")");
    TORCH_CHECK_VALUE(T <= INT32_MAX, "too many rows: ", T);
    TORCH_CHECK_VALUE(a.dim() == 2 && a.size(0) == T && a.size(1) == Hv && b.sizes() == a.sizes() && half_or_float(a) && half_or_float(b),
                      "a and b must be (", T, ", ", Hv, ") bf16 or fp32 tensors");
    TORCH_CHECK_VALUE(a_log.dim() == 1 && a_log.size(0) == Hv && dt_bias.sizes() == a_log.sizes() && half_or_float(a_log) && half_or_float(dt_bias),
                      "a_log and dt_bias must be (", Hv, ") bf16 or fp32 tensors");
    TORCH_CHECK_VALUE(!scale || *scale != 0., "scale must not be zero");
    DeltaInputs in;
    in.q = rows16(q);
    in.k = rows16(k);
    in.v = rows16(v);
    in.a = a.stride(1) == 1 || Hv == 1 ? a : a.contiguous();
    in.b = b.stride(1) == 1 || Hv == 1 ? b : b.contiguous();
    const bool mixed = a_log.scalar_type() != dt_bias.scalar_type();
    in.a_log = (mixed ? a_log.to(at::kFloat) : a_log).contiguous();
    in.dt_bias = (mixed ? dt_bias.to(at::kFloat) : dt_bias).contiguous();
    in.cu = cu;
    in.args = dsa_delta_args{ptr(in.q), ptr(in.k), ptr(in.v), ptr(in.a), ptr(in.b), ptr(in.a_log), ptr(in.dt_bias),
                             tok_of(in.q), head_of(in.q), tok_of(in.k), head_of(in.k), tok_of(in.v), head_of(in.v), tok_of(in.a), tok_of(in.b),
                             iptr(cu), (int)T, cu.defined() ? (int)cu.numel() - 1 : 0, (int)Hk, (int)Hv, (int)Dk, (int)Dv,
                             (float)(scale ? *scale : std::pow((double)Dk, -0.5)), l2_norm, in.a.scalar_type() == at::kFloat, in.b.scalar_type() == at::kFloat,
                             in.a_log.scalar_type() == at::kFloat};
    return in;
}

Tensor state_input(const Tensor &s, const Tensor &like, at::IntArrayRef sizes) {
    need_gpu(s);
    same_device(like, s, "the state");
    TORCH_CHECK_VALUE(s.sizes() == sizes && s.scalar_type() == at::kFloat, "the state must be a ", sizes, " fp32 tensor, not ", s.sizes(), " ", s.scalar_type());
    return s;
}

class DeltaNode : public torch::autograd::Function<DeltaNode> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &a, const Tensor &b, const Tensor &a_log,
                                 const Tensor &dt_bias, const Tensor &cu, const OptTensor &initial_, std::optional<double> scale, bool l2_norm, bool want_final, bool save) {
        at::AutoDispatchBelowADInplaceOrView below;
        const DeltaInputs in = delta_inputs(q, k, v, a, b, a_log, dt_bias, cu, scale, l2_norm);
        const int64_t N = in.args.N, Hv = in.args.Hv, Dk = in.args.Dk, Dv = in.args.Dv;
        Tensor initial;
        if (initial_) initial = state_input(*initial_, q, {N, Hv, Dk, Dv}).contiguous();
        const Tensor out = empty(v.sizes(), at::kBFloat16, q);
        const Tensor last = want_final ? empty({N, Hv, Dk, Dv}, at::kFloat, q) : Tensor();
        const size_t bytes = dsa_delta_workspace_bytes(&in.args, save);
        const Tensor ws = empty_bytes(bytes, q);
        check(dsa_delta_fwd(&in.args, fptr(initial), ptr(out), fptr(last), save, ptr(ws), bytes, stream_of(q)), "dsa_delta_fwd");
        if (save) {
            ctx->save_for_backward({in.q, in.k, in.v, in.a, in.b, in.a_log, in.dt_bias, in.cu, ws});
            ctx->saved_data["s"] = (double)in.args.scale;
            ctx->saved_data["l"] = l2_norm;
            ctx->saved_data["i"] = (bool)initial_;
            ctx->saved_data["pa"] = (int64_t)a_log.scalar_type();
            ctx->saved_data["pd"] = (int64_t)dt_bias.scalar_type();
            ctx->set_materialize_grads(false);
        }
        return want_final ? variable_list{out, last} : variable_list{out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list s = ctx->get_saved_variables();
        const c10::OptionalDeviceGuard guard(s[0].device());
        DeltaInputs in = delta_inputs(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["s"].toDouble(), ctx->saved_data["l"].toBool());
        const int64_t N = in.args.N, Hv = in.args.Hv, Dk = in.args.Dk, Dv = in.args.Dv;
        const Tensor &q = in.q, &v = in.v;
        const Tensor dout = grads[0].defined() ? as_bf16(grads[0]) : at::zeros(v.sizes(), v.options());
        const Tensor dfinal = grads.size() > 1 && grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : Tensor();
        const Tensor dq = empty(q.sizes(), at::kBFloat16, q), dk = empty(q.sizes(), at::kBFloat16, q), dv = empty(v.sizes(), at::kBFloat16, q);
        const Tensor da = empty(in.a.sizes(), in.a.scalar_type(), q), db = empty(in.b.sizes(), in.b.scalar_type(), q);
        const Tensor dlog = empty({Hv}, in.a_log.scalar_type(), q), ddt = empty({Hv}, in.a_log.scalar_type(), q);
        const Tensor dinitial = ctx->saved_data["i"].toBool() ? empty({N, Hv, Dk, Dv}, at::kFloat, q) : Tensor();
        const size_t bytes = dsa_delta_scratch_bytes(&in.args);
        const Tensor scratch = empty_bytes(bytes, q);
        check(dsa_delta_bwd(&in.args, ptr(dout), fptr(dfinal), ptr(s[8]), (size_t)s[8].numel(), ptr(dq), ptr(dk), ptr(dv), ptr(da), ptr(db), ptr(dlog), ptr(ddt),
                            fptr(dinitial), ptr(scratch), bytes, stream_of(q)), "dsa_delta_bwd");
        return once({dq, dk, dv, da, db, dlog.to((ScalarType)ctx->saved_data["pa"].toInt()), ddt.to((ScalarType)ctx->saved_data["pd"].toInt()), Tensor(), dinitial,
                     Tensor(), Tensor(), Tensor(), Tensor()}, grads, "gated_delta_rule");
    }
};

variable_list gated_delta_rule(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &a, const Tensor &b, const Tensor &a_log, const Tensor &dt_bias,
                               const Tensor &cu_, std::optional<double> scale, bool l2_norm, const OptTensor &initial, bool want_final) {
    const Tensor none;
    const Tensor &first = initial ? *initial : none;
    no_forward_mode({&q, &k, &v, &a, &b, &a_log, &dt_bias, &first}, "gated_delta_rule");
    need_gpu(q);
    need_gpu(cu_);
    const c10::OptionalDeviceGuard guard(q.device());
    bool save = false;                                   // (the node's forward runs with gradients off)
    if (at::GradMode::is_enabled())
        for (const Tensor *t : {&q, &k, &v, &a, &b, &a_log, &dt_bias, &first}) save |= t->defined() && t->requires_grad();
    return DeltaNode::apply(q, k, v, a, b, a_log, dt_bias, checked_cu(cu_), initial, scale, l2_norm, want_final, save);
}

Tensor gated_delta_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &a, const Tensor &b, const Tensor &a_log, const Tensor &dt_bias,
                        const Tensor &state, std::optional<double> scale, bool l2_norm) {
    no_forward_mode({&q, &k, &v, &a, &b, &a_log, &dt_bias, &state}, "gated_delta_step");
    no_graph({&q, &k, &v, &a, &b, &a_log, &dt_bias, &state}, "gated_delta_step");
    need_gpu(q);
    const c10::OptionalDeviceGuard guard(q.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const DeltaInputs in = delta_inputs(q, k, v, a, b, a_log, dt_bias, Tensor(), scale, l2_norm);
    const int64_t B = in.args.T, Hv = in.args.Hv, Dk = in.args.Dk, Dv = in.args.Dv;
    state_input(state, q, {B, Hv, Dk, Dv});
    TORCH_CHECK_VALUE(B == 0 || (state.select(0, 0).is_contiguous() && aligned16(state) && (B == 1 || (state.stride(0) % 4 == 0 && state.stride(0) >= Hv * Dk * Dv))),
                      "the state is updated in place: each request's part must be contiguous, on a 16-byte boundary and apart from the others");
    const Tensor out = empty(v.sizes(), at::kBFloat16, q);
    check(dsa_delta_step(&in.args, fptr(state), B > 1 ? state.stride(0) : 0, ptr(out), stream_of(q)), "dsa_delta_step");
    torch::autograd::impl::bump_version(state);
    return out;
}

// ---- short convolution ------------------------------------------------------------------------------------------------------
struct ConvInputs { Tensor x, w, bias; int64_t T, C, W; int f32, bias_f32; };
ConvInputs conv_inputs(const Tensor &x, const Tensor &w, const OptTensor &bias) {
    need_gpu(x);
    need_gpu(w);
    same_device(x, w, "weight");
    TORCH_CHECK_VALUE(x.dim() == 2 && x.scalar_type() == at::kBFloat16 && x.size(0) <= INT32_MAX, "x must be a bf16 (T, channels) tensor");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == x.size(1) && half_or_float(w), "weight must be (", x.size(1), ", width) bf16 or fp32");
    ConvInputs in{x, w.contiguous(), Tensor(), x.size(0), x.size(1), w.size(1), w.scalar_type() == at::kFloat, 0};
    if (!(x.numel() == 0 || (x.stride(1) == 1 && (in.T == 1 || x.stride(0) % 8 == 0) && aligned16(x)))) {
        in.x = x.contiguous();
        if (!aligned16(in.x)) in.x = in.x.clone();
    }
    if (bias) {
        need_gpu(*bias);
        same_device(x, *bias, "bias");
        TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == in.C && half_or_float(*bias), "bias must be (", in.C, ") bf16 or fp32");
        in.bias = bias->contiguous();
        in.bias_f32 = bias->scalar_type() == at::kFloat;
    }
    return in;
}
void check_conv_state(const Tensor &s, const Tensor &x, at::IntArrayRef sizes) {
    need_gpu(s);
    same_device(x, s, "the state");
    TORCH_CHECK_VALUE(s.sizes() == sizes && s.scalar_type() == at::kBFloat16, "the state must be a ", sizes, " bf16 tensor, not ", s.sizes(), " ", s.scalar_type());
}

class ConvNode : public torch::autograd::Function<ConvNode> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &bias, const Tensor &cu, const OptTensor &initial_, bool silu,
                                 bool want_final) {
        at::AutoDispatchBelowADInplaceOrView below;
        const ConvInputs in = conv_inputs(x, w, bias);
        const int64_t N = cu.numel() - 1;
        Tensor initial;
        if (initial_) {
            check_conv_state(*initial_, x, {N, in.C, in.W - 1});
            initial = initial_->contiguous();
        }
        const Tensor y = empty({in.T, in.C}, at::kBFloat16, x), last = want_final ? empty({N, in.C, in.W - 1}, at::kBFloat16, x) : Tensor();
        check(dsa_conv_fwd(ptr(in.x), in.T > 1 ? in.x.stride(0) : 0, ptr(in.w), in.f32, ptr(in.bias), in.bias_f32, silu, iptr(cu), (int)in.T, (int)N, (int)in.C, (int)in.W,
                           ptr(initial), ptr(y), ptr(last), stream_of(x)), "dsa_conv_fwd");
        ctx->save_for_backward({in.x, in.w, in.bias, cu, initial});
        ctx->saved_data["s"] = silu;
        ctx->set_materialize_grads(false);
        if (!want_final) return {y};
        ctx->mark_non_differentiable({last});
        return {y, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        if (!grads[0].defined()) return variable_list(7);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &bias = s[2], &cu = s[3], &initial = s[4];
        const c10::OptionalDeviceGuard guard(x.device());
        const int64_t T = x.size(0), C = x.size(1), W = w.size(1);
        const Tensor dy = as_bf16(grads[0]), dx = empty({T, C}, at::kBFloat16, x), dw = empty(w.sizes(), w.scalar_type(), x);
        const Tensor dbias = bias.defined() ? empty({C}, bias.scalar_type(), x) : Tensor();
        const size_t bytes = dsa_conv_bwd_workspace_bytes((int)T, (int)C, (int)W);
        const Tensor ws = empty_bytes(bytes, x);
        check(dsa_conv_bwd(ptr(x), T > 1 ? x.stride(0) : 0, ptr(dy), C, ptr(w), w.scalar_type() == at::kFloat, ptr(bias), bias.defined() && bias.scalar_type() == at::kFloat,
                           ctx->saved_data["s"].toBool(), iptr(cu), (int)T, (int)cu.numel() - 1, (int)C, (int)W, ptr(initial), ptr(dx), ptr(dw), ptr(dbias), ptr(ws), bytes,
                           stream_of(x)), "dsa_conv_bwd");
        return once({dx, dw, dbias, Tensor(), Tensor(), Tensor(), Tensor()}, grads, "short_conv");
    }
};

variable_list short_conv(const Tensor &x, const Tensor &w, const OptTensor &bias, const Tensor &cu, bool silu, const OptTensor &initial, bool want_final) {
    const Tensor none;
    no_forward_mode({&x, &w, bias ? &*bias : &none, initial ? &*initial : &none}, "short_conv");
    need_gpu(x);
    need_gpu(cu);
    same_device(x, cu, "cu_seqlens");
    TORCH_CHECK_VALUE(!initial || !initial->requires_grad(), "initial_state takes no part in the backward pass: detach it");
    const c10::OptionalDeviceGuard guard(x.device());
    return ConvNode::apply(x, w, bias, checked_cu(cu), initial, silu, want_final);
}

Tensor short_conv_step(const Tensor &x, const Tensor &state, const Tensor &w, const OptTensor &bias, bool silu) {
    const Tensor none;
    no_forward_mode({&x, &w, bias ? &*bias : &none, &state}, "short_conv_step");
    no_graph({&x, &state, &w, bias ? &*bias : &none}, "short_conv_step");
    need_gpu(x);
    const c10::OptionalDeviceGuard guard(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const ConvInputs in = conv_inputs(x, w, bias);
    const int64_t B = in.T, per = in.C * (in.W - 1);
    check_conv_state(state, x, {B, in.C, in.W - 1});
    TORCH_CHECK_VALUE(B == 0 || (state.select(0, 0).is_contiguous() && aligned16(state) && (B == 1 || (state.stride(0) % 8 == 0 && state.stride(0) >= per))),
                      "the state is updated in place: each request's part must be contiguous, on a 16-byte boundary and apart from the others");
    const Tensor y = empty({B, in.C}, at::kBFloat16, x);
    check(dsa_conv_step(ptr(in.x), B > 1 ? in.x.stride(0) : 0, ptr(in.w), in.f32, ptr(in.bias), in.bias_f32, silu, (int)B, (int)in.C, (int)in.W, ptr(state),
                        B > 1 ? state.stride(0) : 0, ptr(y), stream_of(x)), "dsa_conv_step");
    torch::autograd::impl::bump_version(state);
    return y;
}

// ---- norms behind and between blocks -------------------------------------------------------------------------------------------
class GatedNormNode : public torch::autograd::Function<GatedNormNode> {
public:
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &gate, const Tensor &weight, double eps, bool offset) {
        at::AutoDispatchBelowADInplaceOrView below;
        for (const Tensor *t : {&x_, &gate, &weight}) {
            need_gpu(*t);
            same_device(x_, *t, "a tensor");
        }
        check_bf16_thd(x_, "x");
        check_bf16_thd(gate, "gate");
        TORCH_CHECK_VALUE(gate.sizes() == x_.sizes(), "gate must have the shape of x");
        const int64_t T = x_.size(0), H = x_.size(1), D = x_.size(2);
        TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == D && half_or_float(weight), "weight must be (", D, ") bf16 or fp32");
        TORCH_CHECK_VALUE(T <= INT32_MAX, "too many rows: ", T);
        const Tensor x = rows16(x_), z = rows16(gate), w = weight.contiguous();
        const Tensor y = empty(x.sizes(), at::kBFloat16, x), rstd = empty({T, H}, at::kFloat, x);
        check(dsa_gated_norm_fwd(ptr(x), tok_of(x), head_of(x), ptr(z), tok_of(z), head_of(z), ptr(w), w.scalar_type() == at::kFloat, (float)eps, offset ? 1.f : 0.f, (int)T,
                                 (int)H, (int)D, ptr(y), fptr(rstd), stream_of(x)), "dsa_gated_norm_fwd");
        ctx->save_for_backward({x, z, w, rstd});
        ctx->saved_data["o"] = offset;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &z = s[1], &w = s[2], &rstd = s[3];
        const c10::OptionalDeviceGuard guard(x.device());
        const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
        const Tensor dy = as_bf16(grads[0]), dx = empty(x.sizes(), at::kBFloat16, x), dz = empty(x.sizes(), at::kBFloat16, x), dw = empty({D}, w.scalar_type(), x);
        const size_t bytes = dsa_gated_norm_bwd_workspace_bytes((int)T, (int)H, (int)D);
        const Tensor ws = empty_bytes(bytes, x);
        check(dsa_gated_norm_bwd(ptr(dy), ptr(x), tok_of(x), head_of(x), ptr(z), tok_of(z), head_of(z), ptr(w), w.scalar_type() == at::kFloat,
                                 ctx->saved_data["o"].toBool() ? 1.f : 0.f, (int)T, (int)H, (int)D, fptr(rstd), ptr(dx), ptr(dz), ptr(dw), ptr(ws), bytes, stream_of(x)),
              "dsa_gated_norm_bwd");
        return once({dx, dz, dw, Tensor(), Tensor()}, grads, "gated_rms_norm");
    }
};

Tensor gated_rms_norm(const Tensor &x, const Tensor &gate, const Tensor &weight, double eps, bool offset) {
    no_forward_mode({&x, &gate, &weight}, "gated_rms_norm");
    need_gpu(x);
    const c10::OptionalDeviceGuard guard(x.device());
    return GatedNormNode::apply(x, gate, weight, eps, offset);
}

Tensor packed_rows(const Tensor &x) {
    const Tensor c = x.contiguous();
    return aligned16(c) ? c : c.clone();
}

class ResidualNormNode : public torch::autograd::Function<ResidualNormNode> {
public:
    // everything (T, C) and (C)
    static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &y_, const Tensor &weight, const OptTensor &post_, const OptTensor &gate_,
                                 const OptTensor &scale_, double eps, bool offset) {
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t T = x_.size(0), C = x_.size(1);
        auto parameter = [&](const OptTensor &t, const char *name) {
            if (!t) return Tensor();
            need_gpu(*t);
            same_device(x_, *t, name);
            TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == C && half_or_float(*t), name, " must be (", C, ") bf16 or fp32");
            return t->contiguous();
        };
        const Tensor w = parameter(weight, "weight"), post = parameter(post_, "post_weight"), scale = parameter(scale_, "scale");
        const Tensor x = packed_rows(x_), y = packed_rows(y_), gate = gate_ ? packed_rows(*gate_) : Tensor();
        auto f32 = [](const Tensor &t) { return t.defined() && t.scalar_type() == at::kFloat; };
        const Tensor xn = empty({T, C}, x.scalar_type(), x), h = empty({T, C}, at::kBFloat16, x), rstd = empty({T}, at::kFloat, x);
        const Tensor rstd_y = post.defined() ? empty({T}, at::kFloat, x) : Tensor();
        check(dsa_residual_norm_fwd(ptr(x), f32(x), ptr(y), ptr(gate), ptr(w), f32(w), ptr(post), f32(post), ptr(scale), f32(scale), (float)eps, offset ? 1.f : 0.f, (int)T,
                                    (int)C, ptr(xn), ptr(h), fptr(rstd), fptr(rstd_y), stream_of(x)), "dsa_residual_norm_fwd");
        // (the norm reads x' before it is rounded: of a bf16 stream x and y are kept, from which it is formed again; of an fp32 stream x', and y where it is read)
        const bool before = !f32(x), through = post.defined() || gate.defined() || scale.defined();
        ctx->save_for_backward({before ? x : xn, before || through ? y : Tensor(), gate, w, post, scale, rstd, rstd_y});
        ctx->saved_data["o"] = offset;
        ctx->set_materialize_grads(false);
        return {xn, h};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list s = ctx->get_saved_variables();
        const Tensor &xn = s[0], &y = s[1], &gate = s[2], &w = s[3], &post = s[4], &scale = s[5], &rstd = s[6], &rstd_y = s[7];
        const c10::OptionalDeviceGuard guard(xn.device());
        const int64_t T = xn.size(0), C = xn.size(1);
        auto f32 = [](const Tensor &t) { return t.defined() && t.scalar_type() == at::kFloat; };
        auto like = [&](const Tensor &t) { return t.defined() ? empty(t.sizes(), t.scalar_type(), xn) : Tensor(); };
        const Tensor dxn = grads[0].defined() ? packed_rows(grads[0].to(xn.scalar_type())) : Tensor(), dh = grads[1].defined() ? as_bf16(grads[1]) : Tensor();
        const Tensor dx = like(xn), dy = empty({T, C}, at::kBFloat16, xn), dgate = like(gate), dw = like(w), dpost = like(post), dscale = like(scale);
        const size_t bytes = dsa_residual_norm_bwd_workspace_bytes((int)T, (int)C);
        const Tensor ws = empty_bytes(bytes, xn);
        check(dsa_residual_norm_bwd(ptr(dxn), ptr(dh), ptr(xn), f32(xn) ? DSA_STREAM_F32 : DSA_STREAM_BF16_BEFORE, ptr(y), ptr(gate), ptr(w), f32(w), ptr(post), f32(post), ptr(scale), f32(scale),
                                    ctx->saved_data["o"].toBool() ? 1.f : 0.f, (int)T, (int)C, fptr(rstd), fptr(rstd_y), ptr(dx), ptr(dy), ptr(dgate), ptr(dw), ptr(dpost),
                                    ptr(dscale), ptr(ws), bytes, stream_of(xn)), "dsa_residual_norm_bwd");
        return once({dx, dy, dw, dpost, dgate, dscale, Tensor(), Tensor()}, grads, "residual_rms_norm");
    }
};

variable_list residual_rms_norm(const Tensor &x, const Tensor &y, const Tensor &weight, const OptTensor &post, const OptTensor &gate, const OptTensor &scale, double eps,
                                bool offset) {
    const Tensor none;
    no_forward_mode({&x, &y, &weight, post ? &*post : &none, gate ? &*gate : &none, scale ? &*scale : &none}, "residual_rms_norm");
    need_gpu(x);
    need_gpu(y);
    same_device(x, y, "y");
    TORCH_CHECK_VALUE(x.dim() >= 1 && half_or_float(x), "x must be bf16 or fp32");
    TORCH_CHECK_VALUE(y.sizes() == x.sizes() && y.scalar_type() == at::kBFloat16, "y must be bf16 and have the shape of x");
    const int64_t C = x.size(-1), T = C ? x.numel() / C : 0;
    TORCH_CHECK_VALUE(T <= INT32_MAX, "too many rows: ", T);
    OptTensor rows_of_gate;
    if (gate) {
        need_gpu(*gate);
        same_device(x, *gate, "gate");
        TORCH_CHECK_VALUE(gate->sizes() == x.sizes() && gate->scalar_type() == at::kBFloat16, "gate must be bf16 and have the shape of x");
        rows_of_gate = gate->dim() == 2 ? *gate : gate->reshape({T, C});
    }
    const c10::OptionalDeviceGuard guard(x.device());
    // (rows as they are where they are rows: a view is a node of its own, 3 us each way)
    const bool flat = x.dim() == 2;
    variable_list out = ResidualNormNode::apply(flat ? x : x.reshape({T, C}), flat ? y : y.reshape({T, C}), weight, post, rows_of_gate, scale, eps, offset);
    if (!flat)
        for (Tensor &t : out) t = t.view(x.sizes());
    return out;
}

}  // namespace

void bind_layer(py::module_ &m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("gated_delta_rule", &gated_delta_rule, nogil);
    m.def("gated_delta_step", &gated_delta_step, nogil);
    m.def("short_conv", &short_conv, nogil);
    m.def("short_conv_step", &short_conv_step, nogil);
    m.def("gated_rms_norm", &gated_rms_norm, nogil);
    m.def("residual_rms_norm", &residual_rms_norm, nogil);
}
