// The host's share of linear_attention.py and qk_norm.py in C++, included by host_ext.cpp: their tensors' checks, outputs, workspaces and calls
// into the C ABI, and the nodes of their gradients.  A call whose arguments are not what the kernels take is left to the Python callers (None), which
// say what is wrong with them.  One token of one request took 23 us of the host through ctypes, queries and keys of a token 28.
#pragma once
#include <ATen/hip/EmptyTensor.h>
#include <torch/csrc/autograd/custom_function.h>

namespace attention {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Maybe = c10::optional<at::Tensor>;
inline Maybe maybe(const at::Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

// fn() on x's device and PyTorch's current stream there; by whoever holds Python's lock or does not
template <typename F> int launch(const at::Tensor &x, F fn) {
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    return fn((void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
}

// at::empty on x's device without the way through the dispatcher (a microsecond a tensor): nobody follows these calls' operators
inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &x) { return at::detail::empty_cuda(sizes, type, x.device(), c10::nullopt); }
inline at::Tensor fresh_like(const at::Tensor &t) { return fresh(t.sizes(), t.scalar_type(), t); }

inline bool dense_last(const at::Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }
inline bool on_gpu(const at::Tensor &t, const at::Tensor &x) { return t.defined() && on(t, x) && plain(t); }
inline void expect(int rc, const char *what) { TORCH_CHECK(rc == SS2D_OK, what, ": ", ss2d_strerror(rc), " (ss2d status ", rc, ")"); }
inline bool recorded(std::initializer_list<const at::Tensor *> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// A call with gradients that is captured: an eager graph of the same leaves that still lives holds their gradients' nodes on another stream, and the engine,
// which would have the two streams wait for one another at the backward's end, cannot inside a capture and takes the process with it.
inline void refuse_capture(at::ArrayRef<const at::Tensor *> tensors, const char *what) {
    const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(tensors.front()->device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status != hipStreamCaptureStatusActive) return;
    for (const at::Tensor *t : tensors) {
        if (!t->defined() || !t->requires_grad() || t->grad_fn()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        TORCH_CHECK(!node || !node->stream().has_value() || *node->stream() == stream.unwrap(), what,
                    ": this capture's leaves belong to an autograd graph that was recorded on another stream and still lives; drop it first");
    }
}
// The same for a call that goes through Python: tensors or None, the first one on the call's device
static void refuse_capture_of(const std::vector<Maybe> &tensors, const std::string &what) {
    std::vector<const at::Tensor *> leaves;
    for (const Maybe &t : tensors)
        if (t.has_value()) leaves.push_back(&*t);
    refuse_capture(leaves, what.c_str());
}
template <typename P> void strides3(const at::Tensor &t, P &batch, P &token, P &head) { batch = t.stride(0); token = t.stride(1); head = t.stride(2); }
// What comes into a backward: memory on the inputs' device, its last dimension dense, its type that of what it is the gradient of (the inputs' may have
// changed since: a hook brought them back as something else)
inline at::Tensor gradient(const at::Tensor &g, const at::Tensor &x, at::IntArrayRef shape, at::ScalarType type, const char *name) {
    TORCH_CHECK(on_gpu(g, x) && has_shape(g, shape) && g.scalar_type() == type, name,
                " must be a plain tensor with memory of its own, on the device of the inputs and of the shape and type of what it is the gradient of");
    return dense_last(g) ? g : g.contiguous();
}

constexpr int64_t kMaxHead = 256, kMaxNorm = 512;

// ---- linear attention ----------------------------------------------------------------------------------------------------------------
struct Sides {
    at::Tensor q, k, v, decay;
    int64_t heads = 0;
    int code = -1;

    // rank 4: (batch, tokens, heads, dim), 3 without the tokens
    bool read(int64_t rank) {
        if (!q.defined() || !q.is_cuda() || !plain(q) || !on_gpu(k, q) || !on_gpu(v, q)) return false;
        code = dtype_code(q.scalar_type());
        if (code < 0 || q.dim() != rank || k.dim() != rank || v.dim() != rank || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
        for (int64_t i = 0; i < rank - 2; ++i)
            if (k.size(i) != q.size(i) || v.size(i) != q.size(i) || q.size(i) > INT32_MAX) return false;
        if (k.size(-1) != q.size(-1)) return false;
        for (const at::Tensor *t : {&q, &k, &v}) {
            if (!dense_last(*t) || t->size(-1) < 1 || t->size(-1) > kMaxHead || t->size(-2) < 1 || t->size(-2) > INT32_MAX) return false;
            heads = std::max(heads, t->size(-2));
        }
        for (const at::Tensor *t : {&q, &k, &v})
            if (heads % t->size(-2) != 0) return false;
        if (!decay.defined()) return true;
        if (!on_gpu(decay, q) || (decay.scalar_type() != at::kFloat && decay.scalar_type() != q.scalar_type())) return false;
        if (decay.dim() == 1) return decay.size(0) == heads;
        if (decay.dim() != rank - 1 || decay.size(-1) != heads) return false;
        for (int64_t i = 0; i < rank - 2; ++i)
            if (decay.size(i) != q.size(i)) return false;
        return true;
    }
};

inline ss2d_linear_attention_params describe(const Sides &s, const at::Tensor &state, const at::Tensor &cu, double scale) {
    ss2d_linear_attention_params p = {};
    p.batch = (int)s.q.size(0); p.seqlen = (int)s.q.size(1); p.heads = (int)s.heads;
    p.q_heads = (int)s.q.size(2); p.k_heads = (int)s.k.size(2); p.v_heads = (int)s.v.size(2);
    p.key_dim = (int)s.q.size(3); p.value_dim = (int)s.v.size(3);
    p.dtype = s.code; p.scale = (float)scale;
    p.q = s.q.data_ptr(); p.k = s.k.data_ptr(); p.v = s.v.data_ptr();
    p.initial_state = (const float *)ptr_of(state);
    if (cu.defined()) { p.cu_seqlens = (const int32_t *)cu.data_ptr(); p.n_seqs = (int)cu.numel() - 1; }
    if (s.decay.defined()) {
        p.decay = s.decay.data_ptr(); p.decay_dtype = dtype_code(s.decay.scalar_type());
        if (s.decay.dim() == 1) p.decay_head_stride = s.decay.stride(0);
        else strides3(s.decay, p.decay_batch_stride, p.decay_token_stride, p.decay_head_stride);
    }
    strides3(s.q, p.q_batch_stride, p.q_token_stride, p.q_head_stride);
    strides3(s.k, p.k_batch_stride, p.k_token_stride, p.k_head_stride);
    strides3(s.v, p.v_batch_stride, p.v_token_stride, p.v_head_stride);
    return p;
}

inline at::Tensor workspace(int64_t need, const at::Tensor &x, const char *what) {
    expect(need < 0 ? (int)need : SS2D_OK, what);
    return fresh({need}, at::kByte, x);
}

inline variable_list attend(const Sides &s, const at::Tensor &state, const at::Tensor &cu, double scale, bool want_final) {
    const at::Tensor out = fresh({s.q.size(0), s.q.size(1), s.heads, s.v.size(3)}, s.q.scalar_type(), s.q);
    variable_list made = {out};
    ss2d_linear_attention_params p = describe(s, state, cu, scale);
    p.out = out.data_ptr();
    if (want_final) {
        made.push_back(fresh({cu.defined() ? cu.numel() - 1 : s.q.size(0), s.heads, s.q.size(3), s.v.size(3)}, at::kFloat, s.q));
        p.final_state = (float *)made[1].data_ptr();
    }
    const at::Tensor space = workspace(ss2d_linear_attention_workspace_bytes(&p), s.q, "ss2d_linear_attention_fwd");
    expect(launch(s.q, [&](void *stream) { return ss2d_linear_attention_fwd(&p, space.data_ptr(), space.numel(), stream); }), "ss2d_linear_attention_fwd");
    return made;
}

inline bool state_fits(const at::Tensor &state, const at::Tensor &q, at::IntArrayRef shape) {
    return !state.defined() || (on_gpu(state, q) && state.scalar_type() == at::kFloat && has_shape(state, shape));
}

inline bool sequences_fit(const Sides &s, const at::Tensor &state, const at::Tensor &cu) {
    if (cu.defined() && (!on_gpu(cu, s.q) || cu.scalar_type() != at::kInt || cu.dim() != 1 || cu.numel() < 2 || cu.numel() > INT32_MAX || !cu.is_contiguous() || s.q.size(0) != 1))
        return false;
    return state_fits(state, s.q, {cu.defined() ? cu.numel() - 1 : s.q.size(0), s.heads, s.q.size(3), s.v.size(3)}) && (!state.defined() || state.is_contiguous());
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const Maybe &decay_in, const Maybe &state_in,
                                 const Maybe &cu_in, double scale, bool want_final) {
        const at::Tensor decay = decay_in.value_or(at::Tensor()), state = state_in.value_or(at::Tensor()), cu = cu_in.value_or(at::Tensor());
        Sides s = {q, k, v, decay};
        s.read(4);                                                   // (it has been: for the heads and the type)
        ctx->save_for_backward({q, k, v, decay, state, cu});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return attend(s, state, cu, scale, want_final);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_attention_fn is differentiable once: its gradients have none (create_graph)");
        const variable_list saved = ctx->get_saved_variables();
        Sides s = {saved[0], saved[1], saved[2], saved[3]};
        const at::Tensor &state = saved[4], &cu = saved[5];
        TORCH_CHECK(s.read(4) && sequences_fit(s, state, cu), "linear_attention_fn: what a hook made of its saved tensors is not what it saved");
        variable_list result(8);
        at::Tensor dout = grads[0], dfinal = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!dout.defined() && !dfinal.defined()) return result;
        const int64_t n_seqs = cu.defined() ? cu.numel() - 1 : s.q.size(0), out_shape[4] = {s.q.size(0), s.q.size(1), s.heads, s.v.size(3)},
                      state_shape[4] = {n_seqs, s.heads, s.q.size(3), s.v.size(3)};
        if (!dout.defined()) dout = at::zeros(out_shape, s.q.options());
        dout = gradient(dout, s.q, out_shape, s.q.scalar_type(), "dout");
        if (dfinal.defined()) dfinal = gradient(dfinal, s.q, state_shape, at::kFloat, "dfinal").contiguous();
        ss2d_linear_attention_bwd_params p = {};
        p.fwd = describe(s, state, cu, ctx->saved_data["scale"].toDouble());
        for (int i = 0; i < 3; ++i) result[i] = fresh_like(saved[i]);
        int edge = 3;                                                // (of the tensors that there are)
        for (int i = 3; i < 5; ++i)
            if (saved[i].defined() && ctx->needs_input_grad(edge++)) result[i] = fresh_like(saved[i]);
        p.dout = dout.data_ptr(); p.dfinal_state = (const float *)ptr_of(dfinal);
        p.dq = result[0].data_ptr(); p.dk = result[1].data_ptr(); p.dv = result[2].data_ptr();
        p.ddecay = const_cast<void *>(ptr_of(result[3])); p.dinitial_state = (float *)ptr_of(result[4]);
        strides3(dout, p.dout_batch_stride, p.dout_token_stride, p.dout_head_stride);
        p.decay_per_head = s.decay.defined() && s.decay.dim() == 1;
        const at::Tensor space = workspace(ss2d_linear_attention_bwd_workspace_bytes(&p), s.q, "ss2d_linear_attention_bwd");
        expect(launch(s.q, [&](void *stream) { return ss2d_linear_attention_bwd(&p, space.data_ptr(), space.numel(), stream); }), "ss2d_linear_attention_bwd");
        return result;
    }
};

// linear_attention.py:linear_attention_fn -- (out,) or (out, final state), or None
static py::object linear_attention(const py::tuple &kinds, const py::object &q, const py::object &k, const py::object &v, const py::object &decay, const py::object &state_in,
                                   const py::object &cu_in, c10::optional<double> scale_in, bool want_final) {
    bool ok = true;
    Sides s = {exactly(q, kinds, ok), exactly(k, kinds, ok), exactly(v, kinds, ok), exactly(decay, kinds, ok)};
    const at::Tensor state = exactly(state_in, kinds, ok), cu = exactly(cu_in, kinds, ok);
    if (!ok || !s.read(4) || !sequences_fit(s, state, cu)) return py::none();
    const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt((double)s.q.size(3));
    const bool record = recorded({&s.q, &s.k, &s.v, &s.decay, &state});
    if (record) refuse_capture({&s.q, &s.k, &s.v, &s.decay, &state}, "linear_attention_fn");
    const variable_list made = record ? LinearAttention::apply(s.q, s.k, s.v, maybe(s.decay), maybe(state), maybe(cu), scale, want_final)
                                      : attend(s, state, cu, scale, want_final);
    return want_final ? py::object(py::make_tuple(made[0], made[1])) : py::cast(made[0]);
}

// linear_attention.py:linear_attention_step_fn -- out, or None
static py::object linear_attention_step(const py::tuple &kinds, const py::object &q, const py::object &k, const py::object &v, const py::object &decay, const py::object &state_in,
                                        c10::optional<double> scale) {
    bool ok = true;
    Sides s = {exactly(q, kinds, ok), exactly(k, kinds, ok), exactly(v, kinds, ok), exactly(decay, kinds, ok)};
    const at::Tensor state = exactly(state_in, kinds, ok);
    if (!ok || !s.read(3) || !state.defined()) return py::none();
    const int64_t B = s.q.size(0), dk = s.q.size(2), dv = s.v.size(2), each = s.heads * dk * dv;
    if (B == 0 || !state_fits(state, s.q, {B, s.heads, dk, dv}) || recorded({&s.q, &s.k, &s.v, &s.decay, &state})) return py::none();
    if ((B > 1 && state.stride(0) < each) || !(state.is_contiguous() || state[0].is_contiguous())) return py::none();
    const at::Tensor out = fresh({B, s.heads, dv}, s.q.scalar_type(), s.q);
    ss2d_linear_attention_step_params p = {};
    p.batch = (int)B; p.heads = (int)s.heads; p.q_heads = (int)s.q.size(1); p.k_heads = (int)s.k.size(1); p.v_heads = (int)s.v.size(1);
    p.key_dim = (int)dk; p.value_dim = (int)dv; p.dtype = s.code;
    p.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)dk));
    p.q = s.q.data_ptr(); p.k = s.k.data_ptr(); p.v = s.v.data_ptr(); p.state = (float *)state.data_ptr(); p.out = out.data_ptr();
    if (s.decay.defined()) {
        p.decay = s.decay.data_ptr(); p.decay_dtype = dtype_code(s.decay.scalar_type());
        p.decay_head_stride = s.decay.stride(-1); p.decay_batch_stride = s.decay.dim() == 2 ? s.decay.stride(0) : 0;
    }
    p.q_batch_stride = s.q.stride(0); p.q_head_stride = s.q.stride(1); p.k_batch_stride = s.k.stride(0); p.k_head_stride = s.k.stride(1);
    p.v_batch_stride = s.v.stride(0); p.v_head_stride = s.v.stride(1);
    p.state_batch_stride = B > 1 ? state.stride(0) : each;
    state.unsafeGetTensorImpl()->bump_version();                     // (written in place, behind autograd's back)
    const int rc = launch(s.q, [&](void *stream) { return ss2d_linear_attention_step(&p, stream); });
    return rc == SS2D_OK ? py::cast(out) : py::object(py::int_(rc));
}

// ---- norm and rotation -----------------------------------------------------------------------------------------------------------------
struct NormArgs {
    at::Tensor q, k, q_weight, k_weight, positions, frequencies;
    double eps;
    bool interleaved;

    bool read() const {
        if (!q.defined() || !q.is_cuda() || !plain(q) || !on_gpu(k, q) || dtype_code(q.scalar_type()) < 0 || k.scalar_type() != q.scalar_type()) return false;
        if (q.dim() != 4 || k.dim() != 4 || k.size(0) != q.size(0) || k.size(1) != q.size(1) || k.size(3) != q.size(3)) return false;
        if (q.size(3) < 1 || q.size(3) > kMaxNorm || !dense_last(q) || !dense_last(k)) return false;
        for (int i = 0; i < 3; ++i)
            if (q.size(i) > INT32_MAX || k.size(i) > INT32_MAX) return false;
        const at::Tensor &w = q_weight.defined() ? q_weight : k_weight;
        for (const at::Tensor *t : {&q_weight, &k_weight})
            if (t->defined() && (!on_gpu(*t, q) || t->scalar_type() != w.scalar_type() || (w.scalar_type() != at::kFloat && w.scalar_type() != q.scalar_type()) ||
                                 !has_shape(*t, {q.size(3)}) || !t->is_contiguous()))
                return false;
        if (positions.defined() != frequencies.defined()) return false;
        if (!positions.defined()) return true;
        const int64_t several = frequencies.dim() == 2, rank = positions.dim() - several;
        if (!on_gpu(positions, q) || !on_gpu(frequencies, q) || (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong)) return false;
        if ((frequencies.scalar_type() != at::kFloat && frequencies.scalar_type() != at::kDouble) || frequencies.dim() < 1 || frequencies.dim() > 2 || !frequencies.is_contiguous())
            return false;
        if ((rank != 1 && rank != 2) || positions.size(rank - 1) != q.size(1) || (rank == 2 && positions.size(0) != q.size(0))) return false;
        return (!several || positions.size(rank) == frequencies.size(0)) && 2 * frequencies.numel() <= q.size(3);
    }

    ss2d_qk_norm_rotate_params describe() const {
        ss2d_qk_norm_rotate_params p = {};
        p.batch = (int)q.size(0); p.seqlen = (int)q.size(1); p.q_heads = (int)q.size(2); p.k_heads = (int)k.size(2); p.dim = (int)q.size(3);
        p.dtype = dtype_code(q.scalar_type());
        const at::Tensor &w = q_weight.defined() ? q_weight : k_weight;
        p.weight_dtype = w.defined() ? dtype_code(w.scalar_type()) : SS2D_F32;
        p.eps = (float)eps; p.interleaved = interleaved;
        p.q = q.data_ptr(); p.k = k.data_ptr(); p.q_weight = ptr_of(q_weight); p.k_weight = ptr_of(k_weight);
        strides3(q, p.q_batch_stride, p.q_token_stride, p.q_head_stride);
        strides3(k, p.k_batch_stride, p.k_token_stride, p.k_head_stride);
        if (positions.defined() && frequencies.numel()) {
            const bool several = frequencies.dim() == 2;
            p.axes = several ? (int)frequencies.size(0) : 1; p.per_axis = (int)frequencies.size(-1);
            p.positions = positions.data_ptr(); p.frequencies = frequencies.data_ptr();
            p.positions_int64 = positions.scalar_type() == at::kLong; p.frequencies_float64 = frequencies.scalar_type() == at::kDouble;
            const int64_t rank = positions.dim() - several;
            p.position_axis_stride = several ? positions.stride(rank) : 0;
            p.position_token_stride = positions.stride(rank - 1);
            p.position_batch_stride = rank == 2 ? positions.stride(0) : 0;
        }
        return p;
    }
};

inline variable_list norm_rotate(const NormArgs &a) {
    const variable_list made = {fresh_like(a.q), fresh_like(a.k)};
    ss2d_qk_norm_rotate_params p = a.describe();
    p.q_out = made[0].data_ptr(); p.k_out = made[1].data_ptr();
    expect(launch(a.q, [&](void *stream) { return ss2d_qk_norm_rotate(&p, stream); }), "ss2d_qk_norm_rotate");
    return made;
}

struct QkNormRotate : torch::autograd::Function<QkNormRotate> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const Maybe &q_weight_in, const Maybe &k_weight_in, const Maybe &positions_in,
                                 const Maybe &frequencies_in, double eps, bool interleaved) {
        const at::Tensor q_weight = q_weight_in.value_or(at::Tensor()), k_weight = k_weight_in.value_or(at::Tensor()), positions = positions_in.value_or(at::Tensor()),
                         frequencies = frequencies_in.value_or(at::Tensor());
        ctx->save_for_backward({q, k, q_weight, k_weight, positions, frequencies});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        return norm_rotate(NormArgs{q, k, q_weight, k_weight, positions, frequencies, eps, interleaved});
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rotate_fn is differentiable once: its gradients have none (create_graph)");
        const variable_list saved = ctx->get_saved_variables();
        const NormArgs a = {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool()};
        TORCH_CHECK(a.read(), "qk_norm_rotate_fn: what a hook made of its saved tensors is not what it saved");
        const at::Tensor dq = gradient(grads[0], a.q, a.q.sizes(), a.q.scalar_type(), "dq_out"),
                         dk = gradient(grads[1], a.q, a.k.sizes(), a.q.scalar_type(), "dk_out");
        variable_list result(8);
        result[0] = fresh_like(a.q);
        result[1] = fresh_like(a.k);
        int edge = 2;                                                // (of the tensors that there are)
        for (int i = 2; i < 4; ++i)
            if (saved[i].defined() && ctx->needs_input_grad(edge++)) result[i] = fresh_like(saved[i]);
        ss2d_qk_norm_rotate_bwd_params g = {};
        g.fwd = a.describe();
        g.dq_out = dq.data_ptr(); g.dk_out = dk.data_ptr();
        g.dq = result[0].data_ptr(); g.dk = result[1].data_ptr();
        g.dq_weight = const_cast<void *>(ptr_of(result[2])); g.dk_weight = const_cast<void *>(ptr_of(result[3]));
        strides3(dq, g.dq_batch_stride, g.dq_token_stride, g.dq_head_stride);
        strides3(dk, g.dk_batch_stride, g.dk_token_stride, g.dk_head_stride);
        const at::Tensor space = workspace(ss2d_qk_norm_rotate_bwd_workspace_bytes(g.fwd.dim), a.q, "ss2d_qk_norm_rotate_bwd");
        expect(launch(a.q, [&](void *stream) { return ss2d_qk_norm_rotate_bwd(&g, space.data_ptr(), space.numel(), stream); }), "ss2d_qk_norm_rotate_bwd");
        return result;
    }
};

// qk_norm.py:qk_norm_rotate_fn -- (q, k), or None
static py::object qk_norm_rotate(const py::tuple &kinds, const py::object &q, const py::object &k, const py::object &q_weight, const py::object &k_weight, const py::object &positions,
                                 const py::object &frequencies, double eps, bool interleaved) {
    bool ok = true;
    NormArgs a = {exactly(q, kinds, ok),         exactly(k, kinds, ok),           exactly(q_weight, kinds, ok), exactly(k_weight, kinds, ok),
                  exactly(positions, kinds, ok), exactly(frequencies, kinds, ok), eps,                          interleaved};
    if (!ok || !a.read()) return py::none();
    const bool record = recorded({&a.q, &a.k, &a.q_weight, &a.k_weight});
    if (record) refuse_capture({&a.q, &a.k, &a.q_weight, &a.k_weight}, "qk_norm_rotate_fn");
    const variable_list made = record ? QkNormRotate::apply(a.q, a.k, maybe(a.q_weight), maybe(a.k_weight), maybe(a.positions), maybe(a.frequencies), eps, interleaved) : norm_rotate(a);
    return py::make_tuple(made[0], made[1]);
}

}  // namespace attention
