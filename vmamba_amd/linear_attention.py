"""Linear attention with a decay for each head: the selective scan whose state is a matrix per head and whose decay is one for all of it.

    S_t = exp(log_decay_t) S_(t-1) + k_t v_t^T,   out_t = scale q_t^T S_t          S (key_dim, value_dim), S_0 = initial_state or 0

``linear_attention_fn`` is the chunked form, for prompts and training (the reference's scan over chunks with a matrix state,
classification/models/mamba2/ssd_minimal.py:144); ``linear_attention_step_fn`` the recurrence itself, for single tokens,
its state updated in place.  Both run on the HIP kernels of libss2d_hip.so (ss2d_linear_attention_*); GPU tensors only: there is no CPU path
here.  Arguments are checked as csms6s.py does and fail with RuntimeError.
"""
import torch
from torch.autograd import forward_ad

from . import _lib
from .norm import TENSOR_KINDS, native_stands, untraced

_DTYPE_CODE = {torch.float32: _lib.SS2D_F32, torch.bfloat16: _lib.SS2D_BF16, torch.float16: _lib.SS2D_F16}
MAX_HEAD_DIM = 256
MAX_SIZE = 2 ** 31 - 1               # of batch, tokens, heads and sequences, which the C entries count in 32 bits


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _ptr(t):
    return None if t is None else t.data_ptr()


def check_plain(like, /, **tensors):
    """GPU tensors with memory of their own, all on the device of `like` (q)."""
    for name, t in tensors.items():
        if t is None:
            continue
        _check(isinstance(t, torch.Tensor), f"{name} must be a tensor")
        _check(t.is_cuda, f"{name} must be a GPU tensor: vmamba_amd has no CPU path")
        _check(t.device == like.device, f"{name} must be on the device of q ({like.device}), not on {t.device}")
        _check(type(t) in TENSOR_KINDS and torch._C._has_storage(t) and not t.is_neg(), f"{name} must be a plain tensor with memory of its own")


def _dense_last(t):
    return t.stride(-1) == 1 or t.size(-1) <= 1


def _check_sides(q, k, v, what, rank):
    check_plain(q, q=q, k=k, v=v)
    _check(q.dtype in _DTYPE_CODE, f"{what} not implemented for input type '{q.dtype}'")
    _check(k is not None and v is not None and k.dtype == q.dtype and v.dtype == q.dtype, "k and v must have q's dtype")
    layout = "(batch, tokens, heads, dim)" if rank == 4 else "(batch, heads, dim)"
    _check(q.dim() == rank and k.dim() == rank and v.dim() == rank, f"q, k, v must be {layout}")
    _check(k.shape[:-2] == q.shape[:-2] and v.shape[:-2] == q.shape[:-2], f"q, k, v must agree in {'batch and tokens' if rank == 4 else 'batch'}")
    _check(k.shape[-1] == q.shape[-1], "k must have q's head dimension")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(_dense_last(t), f"{name} must be contiguous in its last dimension")
        _check(max(t.shape) <= MAX_SIZE, f"{name} must have no dimension of more than {MAX_SIZE}")
        _check(t.shape[-2] >= 1 and 1 <= t.shape[-1] <= MAX_HEAD_DIM, f"{name} must have heads of 1 to {MAX_HEAD_DIM} values")
    heads = max(q.shape[-2], k.shape[-2], v.shape[-2])
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(heads % t.shape[-2] == 0, f"the heads of {name} must divide those of the others")
    return heads


def _check_decay(log_decay, q, heads, shape):
    if log_decay is None:
        return
    check_plain(q, log_decay=log_decay)
    _check(log_decay.dtype in (torch.float32, q.dtype), "log_decay must be float32 or have q's dtype")
    _check(tuple(log_decay.shape) in (shape, (heads,)), f"log_decay must have shape {shape} or ({heads},)")


def _check_state(state, q, shape, name):
    if state is None:
        return
    check_plain(q, **{name: state})
    _check(state.dtype == torch.float32 and tuple(state.shape) == shape, f"{name} must be float32 of shape {shape}")


def _check_sequences(q, k, v, log_decay, initial_state, cu_seqlens):
    heads = _check_sides(q, k, v, "linear_attention_fn", 4)
    _check_decay(log_decay, q, heads, (q.shape[0], q.shape[1], heads))
    n_seqs = q.shape[0]
    if cu_seqlens is not None:
        check_plain(q, cu_seqlens=cu_seqlens)
        _check(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, "cu_seqlens must be int32 of shape (sequences + 1,)")
        _check(cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous")
        _check(q.shape[0] == 1, "packed sequences (cu_seqlens) must stand in a batch of one")
        n_seqs = cu_seqlens.numel() - 1
        _check(n_seqs <= MAX_SIZE, f"cu_seqlens must have no more than {MAX_SIZE} sequences")
    _check_state(initial_state, q, (n_seqs, heads, q.shape[3], v.shape[3]), "initial_state")
    return heads, n_seqs


def _params(q, k, v, log_decay, scale, initial_state, cu_seqlens, heads, out, final_state):
    p = _lib.LinearAttentionParams()
    p.batch, p.seqlen, p.heads = q.shape[0], q.shape[1], heads
    p.q_heads, p.k_heads, p.v_heads, p.key_dim, p.value_dim = q.shape[2], k.shape[2], v.shape[2], q.shape[3], v.shape[3]
    p.dtype, p.scale = _DTYPE_CODE[q.dtype], scale
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(out)
    p.initial_state, p.final_state = _ptr(initial_state), _ptr(final_state)
    if cu_seqlens is not None:
        p.cu_seqlens, p.n_seqs = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
    if log_decay is not None:
        p.decay, p.decay_dtype = log_decay.data_ptr(), _DTYPE_CODE[log_decay.dtype]
        p.decay_batch_stride, p.decay_token_stride, p.decay_head_stride = (0, 0, *log_decay.stride()) if log_decay.dim() == 1 else log_decay.stride()
    p.q_batch_stride, p.q_token_stride, p.q_head_stride = q.stride()[:3]
    p.k_batch_stride, p.k_token_stride, p.k_head_stride = k.stride()[:3]
    p.v_batch_stride, p.v_token_stride, p.v_head_stride = v.stride()[:3]
    return p


def _workspace(need, what, device):
    _lib.check(min(need, 0), what)
    return torch.empty(need, dtype=torch.uint8, device=device)


def linear_attention_fwd(q, k, v, log_decay, scale, initial_state, cu_seqlens, want_final):
    """(out, final state or None) of arguments that linear_attention_fn has checked."""
    heads = max(q.shape[2], k.shape[2], v.shape[2])
    n_seqs = q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
    out = torch.empty((*q.shape[:2], heads, v.shape[3]), dtype=q.dtype, device=q.device)
    final = torch.empty((n_seqs, heads, q.shape[3], v.shape[3]), dtype=torch.float32, device=q.device) if want_final else None
    p = _params(q, k, v, log_decay, scale, initial_state, cu_seqlens, heads, out, final)
    L = _lib.lib()
    workspace = _workspace(L.ss2d_linear_attention_workspace_bytes(p), "ss2d_linear_attention_fwd", q.device)
    _lib.check(_lib.launch(q, L.ss2d_linear_attention_fwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_linear_attention_fwd")
    return out, final


def linear_attention_bwd(q, k, v, log_decay, scale, initial_state, cu_seqlens, dout, dfinal_state, want_decay, want_state):
    """(dq, dk, dv, dlog_decay or None, dinitial_state or None) of arguments that linear_attention_fn has checked."""
    heads = max(q.shape[2], k.shape[2], v.shape[2])
    p = _lib.LinearAttentionBwdParams()
    p.fwd = _params(q, k, v, log_decay, scale, initial_state, cu_seqlens, heads, None, None)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    ddecay = torch.empty(log_decay.shape, dtype=log_decay.dtype, device=q.device) if want_decay else None
    dstate = torch.empty(initial_state.shape, dtype=torch.float32, device=q.device) if want_state else None
    p.dout, p.dfinal_state = dout.data_ptr(), _ptr(dfinal_state)
    p.dq, p.dk, p.dv, p.ddecay, p.dinitial_state = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ddecay), _ptr(dstate)
    p.dout_batch_stride, p.dout_token_stride, p.dout_head_stride = dout.stride()[:3]
    p.decay_per_head = int(log_decay is not None and log_decay.dim() == 1)
    L = _lib.lib()
    workspace = _workspace(L.ss2d_linear_attention_bwd_workspace_bytes(p), "ss2d_linear_attention_bwd", q.device)
    _lib.check(_lib.launch(q, L.ss2d_linear_attention_bwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_linear_attention_bwd")
    return dq, dk, dv, ddecay, dstate


class LinearAttentionHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, scale, cu_seqlens, want_final):
        with untraced():                                             # (a trace holds this call, with whatever tensors it is given when it runs)
            _check_sequences(q, k, v, log_decay, initial_state, cu_seqlens)
            if ctx.next_functions:                                   # (gradients are recorded)
                _lib.host().refuse_capture([q, k, v, log_decay, initial_state], "linear_attention_fn")
            ctx.scale = q.shape[3] ** -0.5 if scale is None else float(scale)
            initial_state = initial_state if initial_state is None else initial_state.contiguous()
            out, final = linear_attention_fwd(q, k, v, log_decay, ctx.scale, initial_state, cu_seqlens, want_final)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, cu_seqlens)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, dout, dfinal):
        _check(not torch.is_grad_enabled(), "linear_attention_fn is differentiable once: its gradients have none (create_graph)")
        q, k, v, log_decay, initial_state, cu_seqlens = ctx.saved_tensors
        heads, n_seqs = _check_sequences(q, k, v, log_decay, initial_state, cu_seqlens)          # (a hook may have made something else of them)
        if dout is None:
            if dfinal is None:
                return (None,) * 8
            dout = q.new_zeros((*q.shape[:2], heads, v.shape[3]))
        check_plain(q, dout=dout, dfinal=dfinal)
        _check(tuple(dout.shape) == (*q.shape[:2], heads, v.shape[3]) and dout.dtype == q.dtype, "dout must have out's shape and type")
        _check_state(dfinal, q, (n_seqs, heads, q.shape[3], v.shape[3]), "dfinal")
        if not _dense_last(dout):
            dout = dout.contiguous()
        dfinal, initial_state = (t if t is None else t.contiguous() for t in (dfinal, initial_state))
        want = ctx.needs_input_grad
        dq, dk, dv, ddecay, dstate = linear_attention_bwd(q, k, v, log_decay, ctx.scale, initial_state, cu_seqlens, dout, dfinal,
                                                          log_decay is not None and want[3], initial_state is not None and want[4])
        return dq, dk, dv, ddecay, dstate, None, None, None


def linear_attention_fn(q, k, v, log_decay=None, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Linear attention over sequences, differentiable in q, k, v, log_decay and initial_state.

    q (batch, tokens, q_heads, key_dim), k (batch, tokens, k_heads, key_dim), v (batch, tokens, v_heads, value_dim): one dtype (bfloat16, float16 or
    float32), contiguous in the last dimension, any other strides, dimensions up to 256.  The most heads of the three is the number of
    heads; each of the three numbers divides it and neighbouring heads share.
    log_decay: the logarithm of the decay, (batch, tokens, heads) or one for each head (heads,), float32 or q's dtype, None for no
    decay; -inf forgets everything before its token.  scale: key_dim ** -0.5 by default.
    cu_seqlens: int32 (sequences + 1,) on the GPU, the places in a batch of one at which packed sequences begin and the last one ends, ascending;
    sequences may be empty.  Rows of none of them come out as zeros, and so do their gradients.
    initial_state (sequences, heads, key_dim, value_dim) float32.

    Returns out (batch, tokens, heads, value_dim) in q's dtype, with ``output_final_state`` (out, final_state): the states behind the last tokens,
    float32, which linear_attention_step_fn carries on.  In bfloat16 the states are then summed to 24 bits in place of 16, and out may be another by a rounding.

    Differentiable once.  Captured into a graph with gradients, its leaves may belong to no autograd graph that was recorded on another stream and still lives."""
    _check(isinstance(q, torch.Tensor) and q.is_cuda, "q must be a GPU tensor: vmamba_amd has no CPU path")
    if native_stands(q) and not torch.jit.is_tracing():              # (its memory is made where a tracer does not see it)
        native = _lib.host().linear_attention(TENSOR_KINDS, q, k, v, log_decay, initial_state, cu_seqlens, scale, bool(output_final_state))
        if native is not None:
            return native
    out, final = LinearAttentionHip.apply(q, k, v, log_decay, initial_state, scale, cu_seqlens, bool(output_final_state))
    return (out, final) if output_final_state else out


def linear_attention_step_fn(q, k, v, log_decay, state, scale=None):
    """One token of each sequence: state (batch, heads, key_dim, value_dim) float32 is updated in place, and out (batch, heads, value_dim) returned.

    q (batch, q_heads, key_dim), k, v and log_decay ((batch, heads), (heads,) or None) as in linear_attention_fn, without the tokens.  The states have to
    be dense but for the batch's stride, which keeps them apart.  For inference: it refuses tensors that require a gradient while
    gradients are recorded, and to be traced (torch.jit.trace), since a trace would not hold what becomes of the state."""
    _check(isinstance(q, torch.Tensor) and q.is_cuda, "q must be a GPU tensor: vmamba_amd has no CPU path")
    _check(not torch.jit.is_tracing(), "linear_attention_step_fn changes its state behind a tracer's back: it cannot be traced")
    if native_stands(q):
        native = _lib.host().linear_attention_step(TENSOR_KINDS, q, k, v, log_decay, state, scale)
        if native is not None:
            return _lib.result(native, "ss2d_linear_attention_step")
    heads = _check_sides(q, k, v, "linear_attention_step_fn", 3)
    _check_decay(log_decay, q, heads, (q.shape[0], heads))
    shape = (q.shape[0], heads, q.shape[2], v.shape[2])
    _check(state is not None, "state must be a tensor")
    _check_state(state, q, shape, "state")
    per_sequence = shape[1] * shape[2] * shape[3]
    _check(state.shape[0] == 0 or state[0].is_contiguous(), "state must be contiguous but for its batch's stride")
    _check(state.shape[0] <= 1 or state.stride(0) >= per_sequence, "the states of a batch must not overlap")
    _check(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, state))),
           "linear_attention_step_fn has no gradient: call it under torch.no_grad(), or linear_attention_fn")
    _check(forward_ad._current_level < 0 or all(t is None or forward_ad.unpack_dual(t).tangent is None for t in (q, k, v, log_decay, state)),
           "linear_attention_step_fn has no derivative forward either")
    p = _lib.LinearAttentionStepParams()
    out = torch.empty((shape[0], heads, shape[3]), dtype=q.dtype, device=q.device)
    p.batch, p.heads, p.q_heads, p.k_heads, p.v_heads, p.key_dim, p.value_dim = q.shape[0], heads, q.shape[1], k.shape[1], v.shape[1], shape[2], shape[3]
    p.dtype, p.scale = _DTYPE_CODE[q.dtype], q.shape[2] ** -0.5 if scale is None else float(scale)
    p.q, p.k, p.v, p.state, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), state.data_ptr(), out.data_ptr()
    if log_decay is not None:
        p.decay, p.decay_dtype = log_decay.data_ptr(), _DTYPE_CODE[log_decay.dtype]
        p.decay_batch_stride, p.decay_head_stride = (0, log_decay.stride(0)) if log_decay.dim() == 1 else log_decay.stride()
    p.q_batch_stride, p.q_head_stride = q.stride()[:2]
    p.k_batch_stride, p.k_head_stride = k.stride()[:2]
    p.v_batch_stride, p.v_head_stride = v.stride()[:2]
    p.state_batch_stride = state.stride(0) if state.shape[0] > 1 else per_sequence
    torch.autograd.graph.increment_version(state)                # (written in place, behind autograd's back)
    _lib.check(_lib.launch(q, _lib.lib().ss2d_linear_attention_step, p), "ss2d_linear_attention_step")
    return out
