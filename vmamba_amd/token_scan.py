"""The selective scan of token sequences: tokens are rows and channels neighbours, states come in and go out, and a gate is folded in.

    step = softplus(delta + delta_bias),   h_t = exp(step_t A) h_(t-1) + step_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t)

``selective_scan_tokens_fn`` is for prompts and training (the recurrence of selective_scan_fn, classification/models/csms6s.py:29-68, whose rows are
positions of maps); ``selective_scan_step_fn`` for single tokens, its state updated in place.  causal_conv.py has the short convolution that goes
before it.  Both run on the HIP kernels of libss2d_hip.so (ss2d_token_scan_*); GPU tensors only: there is no CPU path here.  Arguments are checked
as csms6s.py does and fail with RuntimeError.
"""
import torch
from torch.autograd import forward_ad

from . import _lib
from .norm import TENSOR_KINDS, native_stands, untraced

_DTYPE_CODE = {torch.float32: _lib.SS2D_F32, torch.bfloat16: _lib.SS2D_BF16, torch.float16: _lib.SS2D_F16}
MAX_STATE = 64
MAX_SIZE = 2 ** 31 - 1               # of dimensions, which the C entries count in 32 bits


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _ptr(t):
    return None if t is None else t.data_ptr()


def check_plain(like, what, /, **tensors):
    """GPU tensors with memory of their own, all on the device of `like`, the argument called `what`."""
    for name, t in tensors.items():
        if t is None:
            continue
        _check(isinstance(t, torch.Tensor), f"{name} must be a tensor")
        _check(t.is_cuda, f"{name} must be a GPU tensor: vmamba_amd has no CPU path")
        _check(t.device == like.device, f"{name} must be on the device of {what} ({like.device}), not on {t.device}")
        _check(type(t) in TENSOR_KINDS and torch._C._has_storage(t) and not t.is_neg(), f"{name} must be a plain tensor with memory of its own")


def dense_last(t):
    return t.stride(-1) == 1 or t.size(-1) <= 1


def check_places(x, what, cu_seqlens):
    """The number of sequences of x (batch, tokens, ..)."""
    if cu_seqlens is None:
        return x.shape[0]
    check_plain(x, what, cu_seqlens=cu_seqlens)
    _check(cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, "cu_seqlens must be int32 of shape (sequences + 1,)")
    _check(cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous")
    _check(x.shape[0] == 1, "packed sequences (cu_seqlens) must stand in a batch of one")
    _check(cu_seqlens.numel() - 1 <= MAX_SIZE, f"cu_seqlens must have no more than {MAX_SIZE} sequences")
    return cu_seqlens.numel() - 1


def check_unseen(what, tensors):
    """What a call in place refuses: gradients and derivatives forward, which it has none of."""
    _check(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)),
           f"{what} has no gradient: call it under torch.no_grad(), or the operator for sequences")
    _check(forward_ad._current_level < 0 or all(t is None or forward_ad.unpack_dual(t).tangent is None for t in tensors), f"{what} has no derivative forward either")


def _check_sides(u, delta, A, B, C, D, z, delta_bias, what, rank):
    check_plain(u, "u", u=u, delta=delta, A=A, B=B, C=C, D=D, z=z, delta_bias=delta_bias)
    _check(u.dtype in _DTYPE_CODE, f"{what} not implemented for input type '{u.dtype}'")
    for name, t in (("delta", delta), ("A", A), ("B", B), ("C", C)):
        _check(t is not None, f"{name} must be a tensor")
    for name, t in (("delta", delta), ("B", B), ("C", C), ("z", z)):
        _check(t is None or t.dtype == u.dtype, f"{name} must have u's dtype")
    layout = "(batch, tokens, dim)" if rank == 3 else "(batch, dim)"
    _check(u.dim() == rank, f"u must be {layout}")
    for name, t in (("delta", delta), ("z", z)):
        _check(t is None or t.shape == u.shape, f"{name} must have u's shape")
    dim = u.shape[-1]
    _check(A.dtype == torch.float32 and A.dim() == 2 and A.shape[0] == dim, "A must be float32 of shape (dim, dstate)")
    dstate = A.shape[1]
    _check(1 <= dstate <= MAX_STATE, f"{what} takes 1 to {MAX_STATE} states per channel")
    for name, t in (("B", B), ("C", C)):
        _check(t.dim() == rank + 1 and t.shape[:rank - 1] == u.shape[:rank - 1] and t.shape[-1] == dstate and t.shape[-2] == B.shape[-2],
               f"{name} must be {layout[:-4]}groups, dstate), of one number of groups")
    _check(B.shape[-2] >= 1 and dim % B.shape[-2] == 0, "dims should be dividable by the groups")
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        _check(t is None or (t.dtype == torch.float32 and tuple(t.shape) == (dim,)), f"{name} must be float32 of shape (dim,)")
    for name, t in (("u", u), ("delta", delta), ("z", z), ("B", B), ("C", C)):
        _check(t is None or dense_last(t), f"{name} must be contiguous in its last dimension")
        _check(t is None or max(t.shape) <= MAX_SIZE, f"{name} must have no dimension of more than {MAX_SIZE}")
    return dstate


def _check_state(state, u, shape, name):
    if state is None:
        return
    check_plain(u, "u", **{name: state})
    _check(state.dtype == torch.float32 and tuple(state.shape) == shape, f"{name} must be float32 of shape {shape}")


def _check_sequences(u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens):
    dstate = _check_sides(u, delta, A, B, C, D, z, delta_bias, "selective_scan_tokens_fn", 3)
    n_seqs = check_places(u, "u", cu_seqlens)
    _check_state(initial_state, u, (n_seqs, u.shape[2], dstate), "initial_state")
    return n_seqs


def _params(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, cu_seqlens):
    p = _lib.TokenScanParams()
    p.batch, p.seqlen, p.dim = u.shape
    p.dstate, p.n_groups, p.dtype, p.delta_softplus = A.shape[1], B.shape[2], _DTYPE_CODE[u.dtype], int(softplus)
    p.u, p.delta, p.B, p.C, p.z = u.data_ptr(), delta.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z)
    p.A, p.D, p.delta_bias, p.initial_state = A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(initial_state)
    if cu_seqlens is not None:
        p.cu_seqlens, p.n_seqs = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
    p.u_batch_stride, p.u_token_stride = u.stride()[:2]
    p.delta_batch_stride, p.delta_token_stride = delta.stride()[:2]
    if z is not None:
        p.z_batch_stride, p.z_token_stride = z.stride()[:2]
    p.B_batch_stride, p.B_token_stride, p.B_group_stride = B.stride()[:3]
    p.C_batch_stride, p.C_token_stride, p.C_group_stride = C.stride()[:3]
    return p


def workspace_of(need, what, device):
    _lib.check(min(need, 0), what)
    return torch.empty(need, dtype=torch.uint8, device=device)


def token_scan_fwd(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, cu_seqlens, want_final, want_kept):
    """(out, final state or None, kept states or None) of arguments that selective_scan_tokens_fn has checked, the weights and states dense."""
    n_seqs = u.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
    p = _params(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, cu_seqlens)
    L = _lib.lib()
    out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    final = torch.empty((n_seqs, *A.shape), dtype=torch.float32, device=u.device) if want_final else None
    kept = None
    if want_kept:
        need = L.ss2d_token_scan_kept_states(p)
        _lib.check(min(need, 0), "ss2d_token_scan_fwd")
        kept = torch.empty(need, dtype=torch.float32, device=u.device)
    p.out, p.final_state, p.kept_states = out.data_ptr(), _ptr(final), _ptr(kept)
    workspace = workspace_of(L.ss2d_token_scan_workspace_bytes(p), "ss2d_token_scan_fwd", u.device)
    _lib.check(_lib.launch(u, L.ss2d_token_scan_fwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_token_scan_fwd")
    return out, final, kept


class SelectiveScanTokensHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, initial_state, softplus, cu_seqlens, want_final):
        with untraced():                                             # (a trace holds this call, with whatever tensors it is given when it runs)
            _check_sequences(u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens)
            record = bool(ctx.next_functions)
            if record:                                               # (gradients are recorded)
                _lib.host().refuse_capture([u, delta, A, B, C, D, z, delta_bias, initial_state], "selective_scan_tokens_fn")
            A, D, delta_bias, initial_state = (t if t is None else t.contiguous() for t in (A, D, delta_bias, initial_state))
            out, final, kept = token_scan_fwd(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, cu_seqlens, want_final, record)
        ctx.softplus = softplus
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens, kept)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, dout, dfinal):
        _check(not torch.is_grad_enabled(), "selective_scan_tokens_fn is differentiable once: its gradients have none (create_graph)")
        u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens, kept = ctx.saved_tensors
        n_seqs = _check_sequences(u, delta, A, B, C, D, z, delta_bias, initial_state, cu_seqlens)        # (a hook may have made something else of them)
        if dout is None:
            if dfinal is None:
                return (None,) * 12
            dout = u.new_zeros(u.shape)
        check_plain(u, "u", dout=dout, dfinal=dfinal, kept=kept)
        _check(dout.shape == u.shape and dout.dtype == u.dtype, "dout must have out's shape and type")
        _check_state(dfinal, u, (n_seqs, *A.shape), "dfinal")
        if not dense_last(dout):
            dout = dout.contiguous()
        A, D, delta_bias, initial_state, dfinal = (t if t is None else t.contiguous() for t in (A, D, delta_bias, initial_state, dfinal))
        p = _lib.TokenScanBwdParams()
        p.fwd = _params(u, delta, A, B, C, D, z, delta_bias, ctx.softplus, initial_state, cu_seqlens)
        L = _lib.lib()
        need = L.ss2d_token_scan_kept_states(p.fwd)
        _check(kept is not None and kept.dtype == torch.float32 and kept.is_contiguous() and kept.numel() == need, "the states kept for the gradients are not what was kept")
        p.fwd.kept_states = kept.data_ptr()
        want = ctx.needs_input_grad
        grads = [torch.empty(t.shape, dtype=t.dtype, device=u.device) if t is not None and (always or want[i]) else None
                 for i, (t, always) in enumerate(((u, True), (delta, True), (A, False), (B, True), (C, True), (D, False), (z, True), (delta_bias, False), (initial_state, False)))]
        if u.shape[2] == 0:                                          # (without channels no kernel runs, and B and C may have gradients)
            grads[3].zero_(), grads[4].zero_()
        p.dout, p.dfinal_state = dout.data_ptr(), _ptr(dfinal)
        p.dout_batch_stride, p.dout_token_stride = dout.stride()[:2]
        p.du, p.ddelta, p.dA, p.dB, p.dC, p.dD, p.dz, p.ddelta_bias, p.dinitial_state = (_ptr(t) for t in grads)
        workspace = workspace_of(L.ss2d_token_scan_bwd_workspace_bytes(p), "ss2d_token_scan_bwd", u.device)
        _lib.check(_lib.launch(u, L.ss2d_token_scan_bwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_token_scan_bwd")
        return *grads, None, None, None


def selective_scan_tokens_fn(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, initial_state=None, output_final_state=False, cu_seqlens=None):
    """The selective scan over sequences of tokens, differentiable in u, delta, A, B, C, D, z, delta_bias and initial_state.

    u, delta, z (batch, tokens, dim), B, C (batch, tokens, groups, dstate): one dtype (bfloat16, float16 or float32), contiguous in the last dimension, any
    other strides; z may be None (no gate).  Channel d belongs to group d // (dim // groups).  A (dim, dstate), D (dim,) or None,
    delta_bias (dim,) or None: float32.  dstate up to 64.  Without delta_softplus the step is delta + delta_bias itself.
    cu_seqlens: int32 (sequences + 1,) on the GPU, the places in a batch of one at which packed sequences begin and the last one ends, ascending;
    sequences may be empty.  Rows of none of them come out as zeros, and so do their gradients.
    initial_state (sequences, dim, dstate) float32.

    Returns out (batch, tokens, dim) in u's dtype, with ``output_final_state`` (out, final_state): the states behind the last tokens, float32, which
    selective_scan_step_fn carries on.  States and sums are float32; recorded for gradients the call keeps the states before
    every 16th token (dstate up to 16; 32nd up to 32, else 64th): 4 bytes for each token and channel.

    Differentiable once.  Captured into a graph with gradients, its leaves may belong to no autograd graph that was recorded on another stream and still lives."""
    _check(isinstance(u, torch.Tensor) and u.is_cuda, "u must be a GPU tensor: vmamba_amd has no CPU path")
    if native_stands(u) and not torch.jit.is_tracing():              # (its memory is made where a tracer does not see it)
        native = _lib.host().token_scan(TENSOR_KINDS, u, delta, A, B, C, D, z, delta_bias, bool(delta_softplus), initial_state, bool(output_final_state), cu_seqlens)
        if native is not None:
            return native
    out, final = SelectiveScanTokensHip.apply(u, delta, A, B, C, D, z, delta_bias, initial_state, bool(delta_softplus), cu_seqlens, bool(output_final_state))
    return (out, final) if output_final_state else out


def selective_scan_step_fn(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True):
    """One token of each sequence: state (batch, dim, dstate) float32 is updated in place, and out (batch, dim) returned.

    u, delta, z (batch, dim), B, C (batch, groups, dstate), A, D and delta_bias as in selective_scan_tokens_fn, without the tokens.  The states have to be
    dense but for the batch's stride, which keeps them apart.  For inference: it refuses tensors that require a gradient while gradients
    are recorded, and to be traced (torch.jit.trace), since a trace would not hold what becomes of the state."""
    _check(isinstance(u, torch.Tensor) and u.is_cuda, "u must be a GPU tensor: vmamba_amd has no CPU path")
    _check(not torch.jit.is_tracing(), "selective_scan_step_fn changes its state behind a tracer's back: it cannot be traced")
    if native_stands(u):
        native = _lib.host().token_scan_step(TENSOR_KINDS, u, delta, A, B, C, state, D, z, delta_bias, bool(delta_softplus))
        if native is not None:
            return _lib.result(native, "ss2d_token_scan_step")
    dstate = _check_sides(u, delta, A, B, C, D, z, delta_bias, "selective_scan_step_fn", 2)
    shape = (*u.shape, dstate)
    _check(state is not None, "state must be a tensor")
    _check_state(state, u, shape, "state")
    _check(state.shape[0] == 0 or state[0].is_contiguous(), "state must be contiguous but for its batch's stride")
    _check(state.shape[0] <= 1 or state.stride(0) >= shape[1] * dstate, "the states of a batch must not overlap")
    check_unseen("selective_scan_step_fn", (u, delta, A, B, C, state, D, z, delta_bias))
    A, D, delta_bias = (t if t is None else t.contiguous() for t in (A, D, delta_bias))
    p = _lib.TokenScanStepParams()
    out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    p.batch, p.dim, p.dstate, p.n_groups, p.dtype, p.delta_softplus = u.shape[0], u.shape[1], dstate, B.shape[1], _DTYPE_CODE[u.dtype], int(bool(delta_softplus))
    p.u, p.delta, p.B, p.C, p.z, p.state, p.out = u.data_ptr(), delta.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), state.data_ptr(), out.data_ptr()
    p.A, p.D, p.delta_bias = A.data_ptr(), _ptr(D), _ptr(delta_bias)
    p.u_batch_stride, p.delta_batch_stride, p.z_batch_stride = u.stride(0), delta.stride(0), 0 if z is None else z.stride(0)
    p.B_batch_stride, p.B_group_stride = B.stride()[:2]
    p.C_batch_stride, p.C_group_stride = C.stride()[:2]
    p.state_batch_stride = state.stride(0) if state.shape[0] > 1 else shape[1] * dstate
    torch.autograd.graph.increment_version(state)                # (written in place, behind autograd's back)
    _lib.check(_lib.launch(u, _lib.lib().ss2d_token_scan_step, p), "ss2d_token_scan_step")
    return out
