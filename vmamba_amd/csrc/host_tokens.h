// The host's share of token_scan.py, causal_conv.py and group_norm.py in C++, as host_attention.h is for linear attention: a call whose arguments are not what the
// kernels take is left to the Python callers (None), which say what is wrong with them.  Through ctypes one token's convolution of one request took 16 us of
// the host, its scan 27, a training step's norm 147.
#pragma once
#include "host_attention.h"

namespace tokens {

using attention::dense_last;
using attention::expect;
using attention::fresh;
using attention::fresh_like;
using attention::gradient;
using attention::launch;
using attention::Maybe;
using attention::maybe;
using attention::on_gpu;
using attention::recorded;
using attention::refuse_capture;
using attention::workspace;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline at::Tensor of(const Maybe &t) { return t.value_or(at::Tensor()); }
inline bool counted(const at::Tensor &t) {
    for (int64_t n : t.sizes())
        if (n > INT32_MAX) return false;
    return true;
}
inline bool weights_fit(const at::Tensor &t, const at::Tensor &x, at::ScalarType type, at::IntArrayRef shape) {
    return !t.defined() || (on_gpu(t, x) && t.scalar_type() == type && has_shape(t, shape) && t.is_contiguous());
}
inline bool places_fit(const at::Tensor &cu, const at::Tensor &x) {
    return !cu.defined() || (on_gpu(cu, x) && cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.numel() >= 2 && cu.numel() <= INT32_MAX && cu.is_contiguous() && x.size(0) == 1);
}
inline int64_t sequences(const at::Tensor &x, const at::Tensor &cu) { return cu.defined() ? cu.numel() - 1 : x.size(0); }
// A state that is updated in place: dense but for the batch's stride, which keeps the states apart
inline bool in_place(const at::Tensor &state, const at::Tensor &x, at::ScalarType type, at::IntArrayRef shape) {
    if (!on_gpu(state, x) || state.scalar_type() != type || !has_shape(state, shape) || state.numel() == 0) return false;
    if (shape[0] > 1 && state.stride(0) < shape[1] * shape[2]) return false;
    return state.is_contiguous() || state[0].is_contiguous();
}
inline bool silu_of(const py::object &activation, bool &ok) {
    if (activation.is_none()) return false;
    ok = ok && py::isinstance<py::str>(activation) && activation.cast<std::string>() == "silu";
    return true;
}
// Which of a function's tensors want their gradients: its edges are those of the tensors that there are
struct Wanted {
    AutogradContext *ctx;
    int edge = 0;
    bool operator()(const at::Tensor &t) { return t.defined() && ctx->needs_input_grad(edge++); }
};
inline void *made(const at::Tensor &t) { return const_cast<void *>(ptr_of(t)); }

// ---- selective scan ----------------------------------------------------------------------------------------------------------------
struct Scan {
    at::Tensor u, delta, A, B, C, D, z, bias;
    bool softplus;
    int code = -1;

    bool read(int64_t rank) {
        if (!u.defined() || !u.is_cuda() || !plain(u) || !on_gpu(delta, u) || !on_gpu(A, u) || !on_gpu(B, u) || !on_gpu(C, u) || (z.defined() && !on_gpu(z, u))) return false;
        code = dtype_code(u.scalar_type());
        if (code < 0 || u.dim() != rank || A.dim() != 2 || B.dim() != rank + 1 || C.dim() != rank + 1 || !counted(u)) return false;
        for (const at::Tensor *t : {&u, &delta, &z, &B, &C})
            if (t->defined() && (t->scalar_type() != u.scalar_type() || !dense_last(*t))) return false;
        if (delta.sizes() != u.sizes() || (z.defined() && z.sizes() != u.sizes()) || B.sizes() != C.sizes()) return false;
        for (int64_t i = 0; i < rank - 1; ++i)
            if (B.size(i) != u.size(i)) return false;
        const int64_t dim = u.size(-1), N = A.size(1), groups = B.size(-2);
        if (A.size(0) != dim || N < 1 || N > 64 || B.size(-1) != N || groups < 1 || groups > INT32_MAX || dim % groups) return false;
        return A.scalar_type() == at::kFloat && A.is_contiguous() && weights_fit(D, u, at::kFloat, {dim}) && weights_fit(bias, u, at::kFloat, {dim});
    }
    bool sequences_fit(const at::Tensor &state, const at::Tensor &cu) const {
        return places_fit(cu, u) && weights_fit(state, u, at::kFloat, {sequences(u, cu), u.size(2), A.size(1)});
    }
    ss2d_token_scan_params describe(const at::Tensor &state, const at::Tensor &cu) const {
        ss2d_token_scan_params p = {};
        p.batch = (int)u.size(0); p.seqlen = (int)u.size(1); p.dim = (int)u.size(2); p.dstate = (int)A.size(1); p.n_groups = (int)B.size(2);
        p.dtype = code; p.delta_softplus = softplus;
        p.u = u.data_ptr(); p.delta = delta.data_ptr(); p.B = B.data_ptr(); p.C = C.data_ptr(); p.z = ptr_of(z);
        p.A = (const float *)A.data_ptr(); p.D = (const float *)ptr_of(D); p.delta_bias = (const float *)ptr_of(bias); p.initial_state = (const float *)ptr_of(state);
        if (cu.defined()) { p.cu_seqlens = (const int32_t *)cu.data_ptr(); p.n_seqs = (int)cu.numel() - 1; }
        p.u_batch_stride = u.stride(0); p.u_token_stride = u.stride(1);
        p.delta_batch_stride = delta.stride(0); p.delta_token_stride = delta.stride(1);
        if (z.defined()) { p.z_batch_stride = z.stride(0); p.z_token_stride = z.stride(1); }
        attention::strides3(B, p.B_batch_stride, p.B_token_stride, p.B_group_stride);
        attention::strides3(C, p.C_batch_stride, p.C_token_stride, p.C_group_stride);
        return p;
    }
    // {out}, {out, final state}, with `keep` the kept states behind them
    variable_list run(const at::Tensor &state, const at::Tensor &cu, bool want_final, at::Tensor *keep) const {
        variable_list out = {fresh_like(u)};
        ss2d_token_scan_params p = describe(state, cu);
        p.out = out[0].data_ptr();
        if (want_final) {
            out.push_back(fresh({sequences(u, cu), u.size(2), A.size(1)}, at::kFloat, u));
            p.final_state = (float *)out[1].data_ptr();
        }
        if (keep) {
            const int64_t n = ss2d_token_scan_kept_states(&p);
            expect(n < 0 ? (int)n : SS2D_OK, "ss2d_token_scan_fwd");
            *keep = fresh({n}, at::kFloat, u);
            p.kept_states = (float *)keep->data_ptr();
        }
        const int64_t need = ss2d_token_scan_workspace_bytes(&p);
        at::Tensor space;
        if (need) space = workspace(need, u, "ss2d_token_scan_fwd");
        expect(launch(u, [&](void *stream) { return ss2d_token_scan_fwd(&p, made(space), need, stream); }), "ss2d_token_scan_fwd");
        return out;
    }
};

struct SelectiveScanTokens : torch::autograd::Function<SelectiveScanTokens> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &u, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B, const at::Tensor &C, const Maybe &D,
                                 const Maybe &z, const Maybe &bias, const Maybe &state, const Maybe &cu, bool softplus, bool want_final) {
        Scan s = {u, delta, A, B, C, of(D), of(z), of(bias), softplus};
        s.read(3);                                                   // (it has been: for the type)
        at::Tensor kept;
        const variable_list out = s.run(of(state), of(cu), want_final, &kept);
        ctx->save_for_backward({u, delta, A, B, C, s.D, s.z, s.bias, of(state), of(cu), kept});
        ctx->saved_data["softplus"] = softplus;
        ctx->set_materialize_grads(false);
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "selective_scan_tokens_fn is differentiable once: its gradients have none (create_graph)");
        const variable_list saved = ctx->get_saved_variables();
        Scan s = {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], ctx->saved_data["softplus"].toBool()};
        const at::Tensor &state = saved[8], &cu = saved[9], &kept = saved[10];
        TORCH_CHECK(s.read(3) && s.sequences_fit(state, cu), "selective_scan_tokens_fn: what a hook made of its saved tensors is not what it saved");
        variable_list result(12);
        at::Tensor dout = grads[0], dfinal = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!dout.defined() && !dfinal.defined()) return result;
        if (!dout.defined()) dout = at::zeros(s.u.sizes(), s.u.options());
        dout = gradient(dout, s.u, s.u.sizes(), s.u.scalar_type(), "dout");
        if (dfinal.defined()) dfinal = gradient(dfinal, s.u, {sequences(s.u, cu), s.u.size(2), s.A.size(1)}, at::kFloat, "dfinal").contiguous();
        ss2d_token_scan_bwd_params p = {};
        p.fwd = s.describe(state, cu);
        TORCH_CHECK(on_gpu(kept, s.u) && kept.scalar_type() == at::kFloat && kept.is_contiguous() && kept.numel() == ss2d_token_scan_kept_states(&p.fwd),
                    "selective_scan_tokens_fn: the states kept for the gradients are not what was kept");
        p.fwd.kept_states = (float *)kept.data_ptr();
        Wanted wanted = {ctx};
        for (int i = 0; i < 9; ++i) {
            const bool want = wanted(saved[i]), always = i < 2 || i == 3 || i == 4 || i == 6;      // (the kernels write these in any case)
            if (saved[i].defined() && (want || always)) result[i] = fresh_like(saved[i]);
        }
        if (s.u.size(2) == 0)                                        // (without channels no kernel runs, and B and C may have gradients)
            for (int i : {3, 4}) result[i].zero_();
        p.dout = dout.data_ptr(); p.dfinal_state = (const float *)ptr_of(dfinal);
        p.dout_batch_stride = dout.stride(0); p.dout_token_stride = dout.stride(1);
        p.du = made(result[0]); p.ddelta = made(result[1]); p.dA = (float *)made(result[2]); p.dB = made(result[3]); p.dC = made(result[4]); p.dD = (float *)made(result[5]);
        p.dz = made(result[6]); p.ddelta_bias = (float *)made(result[7]); p.dinitial_state = (float *)made(result[8]);
        const at::Tensor space = workspace(ss2d_token_scan_bwd_workspace_bytes(&p), s.u, "ss2d_token_scan_bwd");
        expect(launch(s.u, [&](void *stream) { return ss2d_token_scan_bwd(&p, space.data_ptr(), space.numel(), stream); }), "ss2d_token_scan_bwd");
        return result;
    }
};

// token_scan.py:selective_scan_tokens_fn -- out or (out, final state), or None
static py::object token_scan(const py::tuple &kinds, const py::object &u, const py::object &delta, const py::object &A, const py::object &B, const py::object &C, const py::object &D,
                             const py::object &z, const py::object &bias, bool softplus, const py::object &state_in, bool want_final, const py::object &cu_in) {
    bool ok = true;
    Scan s = {exactly(u, kinds, ok), exactly(delta, kinds, ok), exactly(A, kinds, ok), exactly(B, kinds, ok), exactly(C, kinds, ok), exactly(D, kinds, ok), exactly(z, kinds, ok),
              exactly(bias, kinds, ok), softplus};
    const at::Tensor state = exactly(state_in, kinds, ok), cu = exactly(cu_in, kinds, ok);
    if (!ok || !s.read(3) || !s.sequences_fit(state, cu)) return py::none();
    const std::initializer_list<const at::Tensor *> leaves = {&s.u, &s.delta, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &state};
    const bool record = recorded(leaves);
    if (record) refuse_capture(leaves, "selective_scan_tokens_fn");
    const variable_list out = record ? SelectiveScanTokens::apply(s.u, s.delta, s.A, s.B, s.C, maybe(s.D), maybe(s.z), maybe(s.bias), maybe(state), maybe(cu), softplus, want_final)
                                     : s.run(state, cu, want_final, nullptr);
    return want_final ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

// token_scan.py:selective_scan_step_fn -- out, None, or a status
static py::object token_scan_step(const py::tuple &kinds, const py::object &u, const py::object &delta, const py::object &A, const py::object &B, const py::object &C,
                                  const py::object &state_in, const py::object &D, const py::object &z, const py::object &bias, bool softplus) {
    bool ok = true;
    Scan s = {exactly(u, kinds, ok), exactly(delta, kinds, ok), exactly(A, kinds, ok), exactly(B, kinds, ok), exactly(C, kinds, ok), exactly(D, kinds, ok), exactly(z, kinds, ok),
              exactly(bias, kinds, ok), softplus};
    const at::Tensor state = exactly(state_in, kinds, ok);
    if (!ok || !s.read(2) || !state.defined() || !in_place(state, s.u, at::kFloat, {s.u.size(0), s.u.size(1), s.A.size(1)})) return py::none();
    if (recorded({&s.u, &s.delta, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &state})) return py::none();
    const at::Tensor out = fresh_like(s.u);
    ss2d_token_scan_step_params p = {};
    p.batch = (int)s.u.size(0); p.dim = (int)s.u.size(1); p.dstate = (int)s.A.size(1); p.n_groups = (int)s.B.size(1); p.dtype = s.code; p.delta_softplus = softplus;
    p.u = s.u.data_ptr(); p.delta = s.delta.data_ptr(); p.B = s.B.data_ptr(); p.C = s.C.data_ptr(); p.z = ptr_of(s.z);
    p.A = (const float *)s.A.data_ptr(); p.D = (const float *)ptr_of(s.D); p.delta_bias = (const float *)ptr_of(s.bias);
    p.state = (float *)state.data_ptr(); p.out = out.data_ptr();
    p.u_batch_stride = s.u.stride(0); p.delta_batch_stride = s.delta.stride(0); p.z_batch_stride = s.z.defined() ? s.z.stride(0) : 0;
    p.B_batch_stride = s.B.stride(0); p.B_group_stride = s.B.stride(1); p.C_batch_stride = s.C.stride(0); p.C_group_stride = s.C.stride(1);
    p.state_batch_stride = p.batch > 1 ? state.stride(0) : (int64_t)p.dim * p.dstate;
    state.unsafeGetTensorImpl()->bump_version();                     // (written in place, behind autograd's back)
    const int rc = launch(s.u, [&](void *stream) { return ss2d_token_scan_step(&p, stream); });
    return rc == SS2D_OK ? py::cast(out) : py::object(py::int_(rc));
}

// ---- causal convolution --------------------------------------------------------------------------------------------------------------
struct Conv {
    at::Tensor x, weight, bias;
    bool silu;
    int code = -1;

    bool read(int64_t rank) {
        if (!x.defined() || !x.is_cuda() || !plain(x) || x.dim() != rank || !dense_last(x) || !counted(x) || !on_gpu(weight, x)) return false;
        code = dtype_code(x.scalar_type());
        if (code < 0 || weight.dim() != 2 || weight.size(0) != x.size(-1) || weight.size(1) < 2 || weight.size(1) > 4 || !weight.is_contiguous()) return false;
        return (weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type()) && weights_fit(bias, x, weight.scalar_type(), {x.size(-1)});
    }
    bool sequences_fit(const at::Tensor &state, const at::Tensor &cu) const {
        return places_fit(cu, x) && weights_fit(state, x, x.scalar_type(), {sequences(x, cu), weight.size(1) - 1, x.size(2)});
    }
    ss2d_causal_conv_params describe(const at::Tensor &state, const at::Tensor &cu) const {
        ss2d_causal_conv_params p = {};
        p.batch = (int)x.size(0); p.seqlen = (int)x.size(1); p.dim = (int)x.size(2); p.width = (int)weight.size(1);
        p.dtype = code; p.weight_dtype = dtype_code(weight.scalar_type()); p.silu = silu;
        p.x = x.data_ptr(); p.weight = weight.data_ptr(); p.bias = ptr_of(bias); p.initial_state = ptr_of(state);
        if (cu.defined()) { p.cu_seqlens = (const int32_t *)cu.data_ptr(); p.n_seqs = (int)cu.numel() - 1; }
        p.x_batch_stride = x.stride(0); p.x_token_stride = x.stride(1);
        return p;
    }
    variable_list run(const at::Tensor &state, const at::Tensor &cu, bool want_final) const {
        variable_list out = {fresh_like(x)};
        ss2d_causal_conv_params p = describe(state, cu);
        p.out = out[0].data_ptr();
        if (want_final) {
            out.push_back(fresh({sequences(x, cu), weight.size(1) - 1, x.size(2)}, x.scalar_type(), x));
            p.final_state = out[1].data_ptr();
        }
        expect(launch(x, [&](void *stream) { return ss2d_causal_conv_fwd(&p, stream); }), "ss2d_causal_conv_fwd");
        return out;
    }
};

struct CausalConv : torch::autograd::Function<CausalConv> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const Maybe &bias, const Maybe &state, const Maybe &cu, bool silu, bool want_final) {
        Conv c = {x, weight, of(bias), silu};
        c.read(3);                                                   // (it has been: for the type)
        ctx->save_for_backward({x, weight, c.bias, of(state), of(cu)});
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        return c.run(of(state), of(cu), want_final);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "causal_conv_fn is differentiable once: its gradients have none (create_graph)");
        const variable_list saved = ctx->get_saved_variables();
        Conv c = {saved[0], saved[1], saved[2], ctx->saved_data["silu"].toBool()};
        const at::Tensor &state = saved[3], &cu = saved[4];
        TORCH_CHECK(c.read(3) && c.sequences_fit(state, cu), "causal_conv_fn: what a hook made of its saved tensors is not what it saved");
        variable_list result(7);
        at::Tensor dout = grads[0], dfinal = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!dout.defined() && !dfinal.defined()) return result;
        if (!dout.defined()) dout = at::zeros(c.x.sizes(), c.x.options());
        dout = gradient(dout, c.x, c.x.sizes(), c.x.scalar_type(), "dout");
        if (dfinal.defined()) dfinal = gradient(dfinal, c.x, {sequences(c.x, cu), c.weight.size(1) - 1, c.x.size(2)}, c.x.scalar_type(), "dfinal").contiguous();
        ss2d_causal_conv_bwd_params p = {};
        p.fwd = c.describe(state, cu);
        Wanted wanted = {ctx};
        for (int i = 0; i < 4; ++i) {
            const bool want = wanted(saved[i]);
            if (saved[i].defined() && (want || i == 0)) result[i] = fresh_like(saved[i]);
        }
        p.dout = dout.data_ptr(); p.dfinal_state = ptr_of(dfinal);
        p.dout_batch_stride = dout.stride(0); p.dout_token_stride = dout.stride(1);
        p.dx = made(result[0]); p.dweight = made(result[1]); p.dbias = made(result[2]); p.dinitial_state = made(result[3]);
        const at::Tensor space = workspace(ss2d_causal_conv_bwd_workspace_bytes(&p), c.x, "ss2d_causal_conv_bwd");
        expect(launch(c.x, [&](void *stream) { return ss2d_causal_conv_bwd(&p, space.data_ptr(), space.numel(), stream); }), "ss2d_causal_conv_bwd");
        return result;
    }
};

// causal_conv.py:causal_conv_fn -- out or (out, final state), or None
static py::object causal_conv(const py::tuple &kinds, const py::object &x, const py::object &weight, const py::object &bias, const py::object &activation, const py::object &state_in,
                              bool want_final, const py::object &cu_in) {
    bool ok = true;
    Conv c = {exactly(x, kinds, ok), exactly(weight, kinds, ok), exactly(bias, kinds, ok), silu_of(activation, ok)};
    const at::Tensor state = exactly(state_in, kinds, ok), cu = exactly(cu_in, kinds, ok);
    if (!ok || !c.read(3) || !c.sequences_fit(state, cu)) return py::none();
    const std::initializer_list<const at::Tensor *> leaves = {&c.x, &c.weight, &c.bias, &state};
    const bool record = recorded(leaves);
    if (record) refuse_capture(leaves, "causal_conv_fn");
    const variable_list out = record ? CausalConv::apply(c.x, c.weight, maybe(c.bias), maybe(state), maybe(cu), c.silu, want_final) : c.run(state, cu, want_final);
    return want_final ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

// causal_conv.py:causal_conv_step_fn -- out, None, or a status
static py::object causal_conv_step(const py::tuple &kinds, const py::object &x, const py::object &state_in, const py::object &weight, const py::object &bias, const py::object &activation) {
    bool ok = true;
    Conv c = {exactly(x, kinds, ok), exactly(weight, kinds, ok), exactly(bias, kinds, ok), silu_of(activation, ok)};
    const at::Tensor state = exactly(state_in, kinds, ok);
    if (!ok || !c.read(2) || !state.defined() || !in_place(state, c.x, c.x.scalar_type(), {c.x.size(0), c.weight.size(1) - 1, c.x.size(1)})) return py::none();
    if (recorded({&c.x, &c.weight, &c.bias, &state})) return py::none();
    const at::Tensor out = fresh_like(c.x);
    ss2d_causal_conv_step_params p = {};
    p.batch = (int)c.x.size(0); p.dim = (int)c.x.size(1); p.width = (int)c.weight.size(1); p.dtype = c.code; p.weight_dtype = dtype_code(c.weight.scalar_type()); p.silu = c.silu;
    p.x = c.x.data_ptr(); p.weight = c.weight.data_ptr(); p.bias = ptr_of(c.bias); p.state = state.data_ptr(); p.out = out.data_ptr();
    p.x_batch_stride = c.x.stride(0); p.state_batch_stride = p.batch > 1 ? state.stride(0) : (int64_t)(p.width - 1) * p.dim;
    state.unsafeGetTensorImpl()->bump_version();                     // (written in place, behind autograd's back)
    const int rc = launch(c.x, [&](void *stream) { return ss2d_causal_conv_step(&p, stream); });
    return rc == SS2D_OK ? py::cast(out) : py::object(py::int_(rc));
}

// ---- group norm ------------------------------------------------------------------------------------------------------------------------
struct GroupNormArgs {
    at::Tensor x, weight, bias;
    int64_t groups;
    double eps;
    bool silu;

    bool read() const {
        if (!x.defined() || !x.is_cuda() || !plain(x) || x.dim() < 2 || x.numel() == 0 || !x.is_contiguous() || dtype_code(x.scalar_type()) < 0) return false;
        const int64_t C = x.size(-1);
        if (groups < 1 || groups > C || C % groups || C > 1 << 30 || x.size(0) > INT32_MAX || x.numel() / C / x.size(0) > INT32_MAX - 65536) return false;
        const at::Tensor &w = weight.defined() ? weight : bias;
        for (const at::Tensor *t : {&weight, &bias})
            if (t->defined() && (!weights_fit(*t, x, w.scalar_type(), {C}) || (t->scalar_type() != at::kFloat && t->scalar_type() != x.scalar_type()))) return false;
        return true;
    }
    ss2d_group_norm_params describe() const {
        ss2d_group_norm_params p = {};
        p.batch = x.size(0); p.channels = (int)x.size(-1); p.positions = x.numel() / p.channels / p.batch; p.groups = (int)groups;
        const at::Tensor &w = weight.defined() ? weight : bias;
        p.dtype = dtype_code(x.scalar_type()); p.weight_dtype = w.defined() ? dtype_code(w.scalar_type()) : SS2D_F32; p.silu = silu; p.eps = (float)eps;
        p.x = x.data_ptr(); p.weight = ptr_of(weight); p.bias = ptr_of(bias);
        return p;
    }
    at::Tensor run(at::Tensor *stats) const {
        const at::Tensor out = fresh_like(x);
        ss2d_group_norm_params p = describe();
        p.out = out.data_ptr();
        if (stats) {
            *stats = fresh({x.size(0), groups, 2}, at::kFloat, x);
            p.stats = (float *)stats->data_ptr();
        }
        const int64_t need = ss2d_group_norm_workspace_bytes(&p);
        at::Tensor space;
        if (need) space = workspace(need, x, "ss2d_group_norm_fwd");
        expect(launch(x, [&](void *stream) { return ss2d_group_norm_fwd(&p, made(space), need, stream); }), "ss2d_group_norm_fwd");
        return out;
    }
};

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const Maybe &weight, const Maybe &bias, int64_t groups, double eps, bool silu) {
        at::Tensor stats;
        const at::Tensor out = GroupNormArgs{x, of(weight), of(bias), groups, eps, silu}.run(&stats);
        ctx->save_for_backward({x, of(weight), of(bias), stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["silu"] = silu;
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "group_norm_fn is differentiable once: its gradients have none (create_graph)");
        const variable_list saved = ctx->get_saved_variables();
        const GroupNormArgs a = {saved[0], saved[1], saved[2], ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["silu"].toBool()};
        const at::Tensor &stats = saved[3];
        TORCH_CHECK(a.read() && on_gpu(stats, a.x) && stats.scalar_type() == at::kFloat && stats.is_contiguous() && has_shape(stats, {a.x.size(0), a.groups, 2}),
                    "group_norm_fn: what a hook made of its saved tensors is not what it saved");
        const at::Tensor dout = gradient(grads[0], a.x, a.x.sizes(), a.x.scalar_type(), "dout").contiguous();
        variable_list result(6);
        ss2d_group_norm_bwd_params p = {};
        p.fwd = a.describe();
        p.fwd.stats = (float *)stats.data_ptr();
        Wanted wanted = {ctx};
        for (int i = 0; i < 3; ++i) {
            const bool want = wanted(saved[i]);
            if (saved[i].defined() && (want || i == 0)) result[i] = fresh_like(saved[i]);
        }
        p.dout = dout.data_ptr(); p.dx = made(result[0]); p.dweight = made(result[1]); p.dbias = made(result[2]);
        const at::Tensor space = workspace(ss2d_group_norm_bwd_workspace_bytes(&p), a.x, "ss2d_group_norm_bwd");
        expect(launch(a.x, [&](void *stream) { return ss2d_group_norm_bwd(&p, space.data_ptr(), space.numel(), stream); }), "ss2d_group_norm_bwd");
        return result;
    }
};

// group_norm.py:group_norm_fn -- out, or None
static py::object group_norm(const py::tuple &kinds, const py::object &x, int64_t groups, const py::object &weight, const py::object &bias, double eps, const py::object &activation) {
    bool ok = true;
    const GroupNormArgs a = {exactly(x, kinds, ok), exactly(weight, kinds, ok), exactly(bias, kinds, ok), groups, eps, silu_of(activation, ok)};
    if (!ok || !a.read()) return py::none();
    const std::initializer_list<const at::Tensor *> leaves = {&a.x, &a.weight, &a.bias};
    const bool record = recorded(leaves);
    if (record) refuse_capture(leaves, "group_norm_fn");
    return py::cast(record ? GroupNorm::apply(a.x, maybe(a.weight), maybe(a.bias), a.groups, a.eps, a.silu) : a.run(nullptr));
}

}  // namespace tokens
