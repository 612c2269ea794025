// Host side of the operators of a gated-delta-rule layer: argument checks, allocations, the C-ABI calls and the autograd
// nodes, as dsa_host.cpp has them for the attention.
#include "dsa_host.h"

namespace {

using at::ScalarType;

void check_bf16_thd(const Tensor &x, const char *name) {
    TORCH_CHECK_VALUE(x.dim() == 3 && x.scalar_type() == at::kBFloat16, name, " must be a bf16 (T, H, D) tensor");
}
void same_device(const Tensor &a, const Tensor &b, const char *name) {
    TORCH_CHECK_VALUE(a.device() == b.device(), name, " is on ", b.device().str(), ", the other tensors on ", a.device().str());
}
// The tensor itself where its rows can be read 16 bytes at a time in place, a contiguous copy otherwise
Tensor rows16(const Tensor &x) {
    const bool ok = x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) % 8 == 0) && (x.size(0) == 1 || x.stride(0) % 8 == 0) && aligned16(x));
    if (ok) return x;
    const Tensor c = x.contiguous();
    return aligned16(c) ? c : c.clone();
}
int64_t tok_of(const Tensor &x) { return x.size(0) > 1 ? x.stride(0) : 0; }
int64_t head_of(const Tensor &x) { return x.size(1) > 1 ? x.stride(1) : 0; }
bool half_or_float(const Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
void no_graph(std::initializer_list<const Tensor *> inputs, const char *what) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor *t : inputs)
        TORCH_CHECK_VALUE(!t->defined() || !t->requires_grad(), what, " has no backward pass: call it under torch.no_grad() or with detached tensors");
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
        return {dq, dk, dv, da, db, dlog.to((ScalarType)ctx->saved_data["pa"].toInt()), ddt.to((ScalarType)ctx->saved_data["pd"].toInt()), Tensor(), dinitial,
                Tensor(), Tensor(), Tensor(), Tensor()};
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

}  // namespace

void bind_layer(py::module_ &m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("gated_delta_rule", &gated_delta_rule, nogil);
    m.def("gated_delta_step", &gated_delta_step, nogil);
}
