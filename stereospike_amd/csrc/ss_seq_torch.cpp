// ss_seq_torch.cpp — the sequence operators as PyTorch calls: argument checks, allocation, launch through the C-ABI (ss_sequence.h), autograd nodes.
//
// In C++ because a small call is bound by the host: an autograd node in Python costs 65 us a pass before it launches anything, and checking and launching from
// Python twice what a launch itself does.  Every function returns None where an operand is not what its documentation says (nothing has been launched then);
// stereospike_amd/sequence.py turns that into the error that names the operand.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <tuple>

#include "ss_sequence.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

constexpr int64_t kMaxHead = 256, kMaxWidth = 16384, kMaxK = 131071, kMaxStates = 65535, kMaxSteps = 1 << 30, kMaxSide = 1 << 27, kMaxTiles = 1 << 24;

struct SeqError : std::runtime_error { using std::runtime_error::runtime_error; };

int code_of(at::ScalarType t) { return t == at::kFloat ? SS_SEQ_F32 : t == at::kHalf ? SS_SEQ_F16 : t == at::kBFloat16 ? SS_SEQ_BF16 : -1; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void check(int rc, const char* name)
{
    if (rc) throw SeqError(std::string(name) + " failed with code " + std::to_string(rc) + " (-22 = invalid argument, -5 = HIP launch error)");
}
bool is(const Tensor& t, const Tensor& ref, at::ScalarType dt, at::IntArrayRef shape) { return t.defined() && t.device() == ref.device() && t.scalar_type() == dt && t.sizes() == shape; }
Tensor last_contiguous(const Tensor& t) { return t.stride(-1) == 1 || t.is_contiguous() ? t : t.contiguous(); }
const Tensor& given(const Maybe& t)
{
    static const Tensor none;
    return t.has_value() ? *t : none;
}
template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor floats(int64_t n, const Tensor& like) { return n ? at::empty({n}, like.options().dtype(at::kFloat)) : Tensor(); }
bool records(std::initializer_list<Tensor> ts)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts) if (t.defined() && t.requires_grad()) return true;
    return false;
}
// A recording that would hold the outputs' allocation without the launch (torch.jit.trace, a proxy tracer), or a forward-mode tangent, which the outputs would not have.
bool recorded(std::initializer_list<Tensor> ts)
{
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value()) return true;
    for (const Tensor& t : ts) if (t.defined() && t._fw_grad(0).defined()) return true;
    return false;
}
// gradients that raise when they are differentiated again (only under create_graph)
variable_list once_only(variable_list g)
{
    if (!at::GradMode::is_enabled()) return g;
    variable_list in;
    for (const Tensor& t : g) in.push_back(t.defined() ? t.detach().requires_grad_(true) : t);
    auto err = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a sequence operator: its gradients are computed by kernels without a graph",
                                                               (int64_t)in.size());
    variable_list out = (*err)(std::move(in));
    return out;
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// leaky attention
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// q [lead..., B, H, Dk], k [lead..., B, Hk, Dk], v [lead..., B, Hk, Dv]
bool attention_ok(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const Tensor& lengths, int64_t dims)
{
    if (!q.is_cuda() || code_of(q.scalar_type()) < 0 || q.dim() != dims || k.dim() != dims || v.dim() != dims) return false;
    const auto dt = q.scalar_type();
    const int64_t B = q.size(-3), H = q.size(-2), Dk = q.size(-1), Hk = v.size(-2), Dv = v.size(-1);
    if (k.device() != q.device() || v.device() != q.device() || k.scalar_type() != dt || v.scalar_type() != dt) return false;
    for (int64_t i = 0; i < dims - 2; ++i) if (k.size(i) != q.size(i) || v.size(i) != q.size(i)) return false;
    if (k.size(-2) != Hk || k.size(-1) != Dk || H < 1 || Hk < 1 || H % Hk || Dk < 1 || Dk > kMaxHead || Dv < 1 || Dv > kMaxHead || B * H > kMaxStates) return false;
    if (dims == 4 && q.size(0) > kMaxSteps) return false;
    if (!is(log_decay, q, at::kFloat, {H})) return false;
    if (state.defined() && !is(state, q, at::kFloat, {B, H, Dk, Dv})) return false;
    return !lengths.defined() || is(lengths, q, at::kInt, {B});
}

// the forward pass; returns its workspace (the states between segments), undefined where there is none
Tensor attention_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& log_decay, double scale, const Tensor& lengths,
                     const Tensor& s_in, const Tensor& s_out)
{
    const bool seq = q.dim() == 4;
    ss_seq_leaky_desc d{};
    d.size = sizeof(d);
    d.dtype = d.out_dtype = code_of(q.scalar_type());
    d.T = seq ? (int)q.size(0) : 1;
    d.B = (int)q.size(-3); d.H = (int)q.size(-2); d.DA = (int)q.size(-1); d.DC = (int)v.size(-1);
    d.b_scale = 1.f; d.o_scale = (float)scale;
    d.a = q.data_ptr(); d.b = k.data_ptr(); d.c = v.data_ptr(); d.out = out.data_ptr();
    d.a_t = seq ? q.stride(0) : 0; d.a_b = q.stride(-3); d.a_h = q.stride(-2);
    d.b_t = seq ? k.stride(0) : 0; d.b_b = k.stride(-3); d.b_h = k.stride(-2);
    d.c_t = seq ? v.stride(0) : 0; d.c_b = v.stride(-3); d.c_h = v.stride(-2);
    d.o_h = d.DC; d.o_b = (long long)d.H * d.DC; d.o_t = d.B * d.o_b;
    d.a_group = 1; d.b_group = d.c_group = d.H / (int)k.size(-2);
    d.log_decay = ptr<float>(log_decay); d.lengths = ptr<int>(lengths); d.s_in = ptr<float>(s_in); d.s_out = ptr<float>(s_out);
    d.s_in_row = d.s_out_row = d.DC; d.s_in_col = d.s_out_col = 1;
    const Tensor ws = floats(ss_seq_leaky_ws_floats(&d), q);
    d.ws = ptr<float>(ws);
    check(ss_seq_leaky(&d, stream_of(q)), "ss_seq_leaky");
    return ws;
}

// no step, or no stream: outputs that are empty or zeros, the state as it is, and nothing to launch
variable_list attention_none(const Tensor& q, const Tensor& v, const Tensor& log_decay, const Tensor& state)
{
    return {at::zeros({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options()),
            state.defined() ? state.clone() : at::zeros({q.size(1), q.size(2), q.size(3), v.size(3)}, log_decay.options())};
}

struct LeakyAttention : torch::autograd::Function<LeakyAttention> {
    // (an operand that is not there has no edge: the state's, if it is there, is the fifth)
    static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, Tensor log_decay, Maybe state0, Maybe lengths0, double scale)
    {
        const Tensor &state = given(state0), &lengths = given(lengths0);
        ctx->set_materialize_grads(false);
        if (q.numel() == 0) {
            ctx->save_for_backward({q, k, v, state});
            return attention_none(q, v, log_decay, state);
        }
        const Tensor out = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options()),
                     last = at::empty({q.size(1), q.size(2), q.size(3), v.size(3)}, log_decay.options());
        const Tensor states = attention_run(q, k, v, out, log_decay, scale, lengths, state, last);
        ctx->save_for_backward({q, k, v, state, log_decay, lengths, states});
        ctx->saved_data["scale"] = scale;
        return {out, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        if (s[0].numel() == 0) {
            const Tensor g_s = !s[3].defined() || !ctx->needs_input_grad(4) ? Tensor() : grads[1].defined() ? grads[1] : at::zeros_like(s[3]);
            return {at::zeros_like(s[0]), at::zeros_like(s[1]), at::zeros_like(s[2]), Tensor(), g_s, Tensor(), Tensor()};
        }
        const Tensor &q = s[0], &k = s[1], &v = s[2], &state = s[3], &log_decay = s[4], &lengths = s[5], &states = s[6];
        const c10::DeviceGuard guard(q.device());
        const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2), need_s = state.defined() && ctx->needs_input_grad(4);
        Tensor g_q, g_k, g_v, g_s;
        {
            const at::NoGradGuard plain;
            const Tensor g = grads[0].defined() ? last_contiguous(grads[0]) : at::zeros({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options()),
                         g_last = grads[1].defined() ? grads[1].contiguous() : Tensor();
            if (need_q) g_q = at::empty(q.sizes(), q.options());
            if (need_k) g_k = at::empty(k.sizes(), k.options());
            if (need_v || need_s) g_v = at::empty(v.sizes(), v.options());
            if (need_s) g_s = at::empty(state.sizes(), state.options());
            ss_seq_leaky_bwd_desc d{};
            d.size = sizeof(d);
            d.dtype = code_of(q.scalar_type());
            d.T = (int)q.size(0); d.B = (int)q.size(1); d.H = (int)q.size(2); d.Hk = (int)k.size(2); d.Dk = (int)q.size(3); d.Dv = (int)v.size(3);
            d.scale = (float)ctx->saved_data["scale"].toDouble();
            d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr(); d.g = g.data_ptr();
            d.q_t = q.stride(0); d.q_b = q.stride(1); d.q_h = q.stride(2);
            d.k_t = k.stride(0); d.k_b = k.stride(1); d.k_h = k.stride(2);
            d.v_t = v.stride(0); d.v_b = v.stride(1); d.v_h = v.stride(2);
            d.g_t = g.stride(0); d.g_b = g.stride(1); d.g_h = g.stride(2);
            d.g_q = ptr<void>(g_q); d.g_k = ptr<void>(g_k); d.g_v = ptr<void>(g_v); d.g_s = ptr<float>(g_s);
            d.log_decay = ptr<float>(log_decay); d.lengths = ptr<int>(lengths); d.s_in = ptr<float>(state); d.g_last = ptr<float>(g_last);
            d.states = ptr<float>(states);
            const Tensor ws = floats(ss_seq_leaky_bwd_ws_floats(&d), q);
            d.ws = ptr<float>(ws);
            check(ss_seq_leaky_bwd(&d, stream_of(q)), "ss_seq_leaky_bwd");
        }
        variable_list out = once_only({g_q, g_k, need_v ? g_v : Tensor(), g_s});
        return {out[0], out[1], out[2], Tensor(), out[3], Tensor(), Tensor()};
    }
};

std::optional<std::tuple<Tensor, Tensor>> leaky_attention(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& log_decay0, std::optional<double> scale0,
                                                          const Maybe& state0, const Maybe& lengths0)
{
    const Tensor& st = given(state0);
    if (!attention_ok(q0, k0, v0, log_decay0, st, given(lengths0), 4)) return std::nullopt;
    if ((at::GradMode::is_enabled() && log_decay0.requires_grad()) || recorded({q0, k0, v0, log_decay0, st})) return std::nullopt;
    const c10::DeviceGuard guard(q0.device());
    const double scale = scale0.has_value() ? *scale0 : 1. / std::sqrt((double)q0.size(3));
    const int64_t T = q0.size(0), B = q0.size(1), H = q0.size(2), Dk = q0.size(3), Dv = v0.size(3);
    const Tensor q = last_contiguous(q0), k = last_contiguous(k0), v = last_contiguous(v0), log_decay = log_decay0.contiguous(),
                 state = st.defined() ? st.contiguous() : Tensor(), lengths = lengths0.has_value() ? lengths0->contiguous() : Tensor();
    if (records({q, k, v, state})) {
        const variable_list r = LeakyAttention::apply(q, k, v, log_decay, st.defined() ? Maybe(state) : Maybe(), lengths.defined() ? Maybe(lengths) : Maybe(), scale);
        return std::make_tuple(r[0], r[1]);
    }
    if (T == 0 || B == 0) {
        const variable_list r = attention_none(q, v, log_decay, state);
        return std::make_tuple(r[0], r[1]);
    }
    const Tensor out = at::empty({T, B, H, Dv}, q.options()), last = at::empty({B, H, Dk, Dv}, log_decay.options());
    attention_run(q, k, v, out, log_decay, scale, lengths, state, last);
    return std::make_tuple(out, last);
}

std::optional<Tensor> leaky_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, std::optional<double> scale)
{
    if (!state.defined() || !attention_ok(q, k, v, log_decay, state, Tensor(), 3) || !state.is_contiguous() || recorded({q, k, v, log_decay, state})) return std::nullopt;
    if (state.requires_grad() || records({q, k, v, log_decay})) return std::nullopt;
    const c10::DeviceGuard guard(q.device());
    const at::NoGradGuard plain;
    const Tensor out = at::empty({q.size(0), q.size(1), v.size(2)}, q.options());
    if (q.size(0)) {
        attention_run(last_contiguous(q), last_contiguous(k), last_contiguous(v), out, log_decay.contiguous(),
                      scale.has_value() ? *scale : 1. / std::sqrt((double)q.size(2)), Tensor(), state, state);
        if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();       // an autograd graph that saved this state must notice
    }
    return out;
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// add + root-mean-square norm
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
bool norm_ok(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps)
{
    if (!x.is_cuda() || code_of(x.scalar_type()) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kMaxWidth || !(eps >= 0.)) return false;
    if (!is(weight, x, at::kFloat, {x.size(-1)})) return false;
    return !residual.defined() || is(residual, x, x.scalar_type(), x.sizes());
}
// [rows][C] with a contiguous last axis
Tensor rows_of(const Tensor& t)
{
    const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

// y and, with a residual, the sum; rstd if defined
void norm_run(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& y, const Tensor& sum, const Tensor& rstd, double eps)
{
    const Tensor xr = rows_of(x), rr = residual.defined() ? rows_of(residual) : Tensor();
    if (xr.size(0) == 0) return;
    check(ss_seq_rms_norm_fwd(xr.data_ptr(), xr.stride(0), ptr<void>(rr), rr.defined() ? rr.stride(0) : 0, ptr<float>(weight), y.data_ptr(), ptr<void>(sum),
                              ptr<float>(rstd), xr.size(0), (int)xr.size(1), (float)eps, code_of(x.scalar_type()), stream_of(x)), "ss_seq_rms_norm_fwd");
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, Maybe residual0, double eps)
    {
        const Tensor& residual = given(residual0);
        ctx->set_materialize_grads(false);
        if (!residual.defined()) x = x.contiguous();       // kept for the backward
        const Tensor y = at::empty(x.sizes(), x.options()), sum = residual.defined() ? at::empty(x.sizes(), x.options()) : Tensor(),
                     rstd = at::empty({x.numel() / x.size(-1)}, weight.options());
        norm_run(x, residual, weight, y, sum, rstd, eps);
        ctx->save_for_backward({residual.defined() ? sum : x, weight, rstd});
        return residual.defined() ? variable_list{y, sum} : variable_list{y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &h = s[0], &weight = s[1], &rstd = s[2];
        const c10::DeviceGuard guard(h.device());
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_r = grads.size() > 1 && ctx->needs_input_grad(2);
        Tensor g_h, g_w;
        {
            const at::NoGradGuard plain;
            const int64_t rows = rstd.size(0), C = h.size(-1);
            const int dt = code_of(h.scalar_type());
            const Tensor g_y = grads[0].defined() ? grads[0].contiguous() : Tensor(), g_sum = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
            g_h = at::empty(h.sizes(), h.options());
            if (need_w) g_w = rows ? at::empty(weight.sizes(), weight.options()) : at::zeros(weight.sizes(), weight.options());
            if (rows) {
                const Tensor ws = need_w ? floats(ss_seq_rms_norm_ws_floats(rows, (int)C, dt), h) : Tensor();
                check(ss_seq_rms_norm_bwd(ptr<void>(g_y), ptr<void>(g_sum), h.data_ptr(), ptr<float>(weight), ptr<float>(rstd), g_h.data_ptr(), ptr<float>(g_w),
                                          ptr<float>(ws), rows, (int)C, dt, stream_of(h)), "ss_seq_rms_norm_bwd");
            }
        }
        variable_list out = once_only({need_x ? g_h : Tensor(), g_w, need_r ? g_h : Tensor()});
        out.resize(4);
        return out;
    }
};

std::optional<std::tuple<Tensor, Tensor>> add_rms_norm(const Tensor& x, const Tensor& weight, const Maybe& residual0, double eps)
{
    const Tensor& residual = given(residual0);
    if (!norm_ok(x, weight, residual, eps) || recorded({x, weight, residual})) return std::nullopt;
    const c10::DeviceGuard guard(x.device());
    if (records({x, residual, weight})) {
        const variable_list r = AddRmsNorm::apply(x, weight.contiguous(), residual.defined() ? Maybe(residual) : Maybe(), eps);
        return std::make_tuple(r[0], residual.defined() ? r[1] : x);
    }
    const Tensor y = at::empty(x.sizes(), x.options()), sum = residual.defined() ? at::empty(x.sizes(), x.options()) : Tensor();
    norm_run(x, residual, weight.contiguous(), y, sum, Tensor(), eps);
    return std::make_tuple(y, residual.defined() ? sum : x);
}

// codes, scales and, with a residual, the sum
variable_list norm_int8_run(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps)
{
    const at::NoGradGuard plain;
    const Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar)), scales = at::empty(x.sizes().slice(0, x.dim() - 1), weight.options()),
                 sum = residual.defined() ? at::empty(x.sizes(), x.options()) : Tensor();
    const Tensor xr = rows_of(x), rr = residual.defined() ? rows_of(residual) : Tensor();
    if (xr.size(0))
        check(ss_seq_rms_norm_int8(xr.data_ptr(), xr.stride(0), ptr<void>(rr), rr.defined() ? rr.stride(0) : 0, ptr<float>(weight.contiguous()),
                                   static_cast<signed char*>(codes.data_ptr()), ptr<float>(scales), ptr<void>(sum), xr.size(0), (int)xr.size(1), (float)eps,
                                   code_of(x.scalar_type()), stream_of(x)), "ss_seq_rms_norm_int8");
    return {codes, scales, sum};
}

// codes and scales have no gradient; the sum has an addition's
struct AddRmsNormInt8 : torch::autograd::Function<AddRmsNormInt8> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor residual, Tensor weight, double eps)
    {
        ctx->set_materialize_grads(false);
        const variable_list r = norm_int8_run(x, weight, residual, eps);
        ctx->mark_non_differentiable({r[0], r[1]});
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        return {ctx->needs_input_grad(0) ? grads[2] : Tensor(), ctx->needs_input_grad(1) ? grads[2] : Tensor(), Tensor(), Tensor()};
    }
};

std::optional<std::tuple<Tensor, Tensor, Tensor>> add_rms_norm_int8(const Tensor& x, const Tensor& weight, const Maybe& residual0, double eps)
{
    const Tensor& residual = given(residual0);
    if (!norm_ok(x, weight, residual, eps) || recorded({x, weight, residual})) return std::nullopt;
    const c10::DeviceGuard guard(x.device());
    const variable_list r = residual.defined() && records({x, residual}) ? AddRmsNormInt8::apply(x, residual, weight.detach(), eps) : norm_int8_run(x, weight, residual, eps);
    return std::make_tuple(r[0], r[1], residual.defined() ? r[2] : x);
}

std::optional<Tensor> dequantize_int8(const Tensor& codes, const Tensor& scales, at::ScalarType dtype)
{
    if (!codes.is_cuda() || codes.scalar_type() != at::kChar || codes.dim() < 1 || codes.size(-1) < 1 || code_of(dtype) < 0) return std::nullopt;
    if (!is(scales, codes, at::kFloat, codes.sizes().slice(0, codes.dim() - 1)) || records({scales}) || recorded({scales})) return std::nullopt;
    const c10::DeviceGuard guard(codes.device());
    const at::NoGradGuard plain;
    const Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype)), c = codes.contiguous(), s = scales.contiguous();
    if (out.numel())
        check(ss_seq_dequant_int8(static_cast<const signed char*>(c.data_ptr()), ptr<float>(s), out.data_ptr(), c.numel() / c.size(-1), (int)c.size(-1), code_of(dtype),
                                  stream_of(codes)), "ss_seq_dequant_int8");
    return out;
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// 8-bit integer product
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
std::optional<Tensor> int8_linear(const Tensor& codes, const Tensor& scales, const Tensor& weight, const Tensor& weight_scale, const Maybe& bias0, at::ScalarType out_dtype)
{
    const Tensor& bias = given(bias0);
    if (!codes.is_cuda() || codes.scalar_type() != at::kChar || codes.dim() < 1 || weight.dim() != 2 || code_of(out_dtype) < 0) return std::nullopt;
    const int64_t N = weight.size(0), K = weight.size(1);
    if (!is(weight, codes, at::kChar, {N, K}) || codes.size(-1) != K || N < 1 || N > kMaxSide || K < 1 || K > kMaxK || codes.numel() / K > kMaxSide) return std::nullopt;
    if ((codes.numel() / K + 127) / 128 * ((N + 127) / 128) >= kMaxTiles) return std::nullopt;
    if (!is(scales, codes, at::kFloat, codes.sizes().slice(0, codes.dim() - 1)) || !is(weight_scale, codes, at::kFloat, {N})) return std::nullopt;
    if (bias.defined() && !is(bias, codes, at::kFloat, {N})) return std::nullopt;
    if (records({scales, weight_scale, bias}) || recorded({scales, weight_scale, bias})) return std::nullopt;
    const c10::DeviceGuard guard(codes.device());
    const at::NoGradGuard plain;
    auto shape = codes.sizes().vec();
    shape.back() = N;
    const Tensor out = at::empty(shape, codes.options().dtype(out_dtype));
    const Tensor a = rows_of(codes), w = rows_of(weight), as = scales.contiguous(), wsc = weight_scale.contiguous(), b = bias.defined() ? bias.contiguous() : Tensor();
    const int64_t M = a.size(0);
    if (M == 0) return out;
    const signed char *pa = static_cast<const signed char*>(a.data_ptr()), *pw = static_cast<const signed char*>(w.data_ptr());
    const int64_t n = ss_seq_int8_linear_ws_ints(pa, a.stride(0), pw, w.stride(0), M, (int)N, (int)K);
    const Tensor ws = n ? at::empty({n}, codes.options().dtype(at::kInt)) : Tensor();
    check(ss_seq_int8_linear(pa, a.stride(0), ptr<float>(as), pw, w.stride(0), ptr<float>(wsc), ptr<float>(b), out.data_ptr(), M, (int)N, (int)K, code_of(out_dtype),
                             ptr<int>(ws), stream_of(codes)), "ss_seq_int8_linear");
    return out;
}

PyObject* error_class = nullptr;

}  // namespace

PYBIND11_MODULE(ss_seq_torch, m)
{
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const SeqError& e) {
            PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
        }
    });
    m.def("set_error", [](py::object c) { error_class = c.release().ptr(); });
    m.def("abi_version", [] { return ss_seq_abi_version(); });
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("leaky_attention", &leaky_attention, nogil);
    m.def("leaky_attention_step", &leaky_attention_step, nogil);
    m.def("add_rms_norm", &add_rms_norm, nogil);
    m.def("add_rms_norm_int8", &add_rms_norm_int8, nogil);
    m.def("dequantize_int8", &dequantize_int8, nogil);
    m.def("int8_linear", &int8_linear, nogil);
}
