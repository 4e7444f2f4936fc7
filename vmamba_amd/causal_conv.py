"""The short causal convolution of token sequences, each channel for itself, that goes before a selective scan.

    y_t = act(bias + sum_j weight[:, j] x_(t - width + 1 + j))

``causal_conv_fn`` is for prompts and training (a block's depthwise convolution, classification/models/vmamba.py:654-658, along tokens); its state is
the last width - 1 inputs, which ``causal_conv_step_fn`` carries on token by token, in place.  Both run on the HIP kernels of libss2d_hip.so
(ss2d_causal_conv_*); GPU tensors only: there is no CPU path here.  Arguments are checked as csms6s.py does and fail with RuntimeError.
"""
import torch

from . import _lib
from .norm import TENSOR_KINDS, native_stands, untraced
from .token_scan import MAX_SIZE, _check, _ptr, check_places, check_plain, check_unseen, dense_last, workspace_of

_DTYPE_CODE = {torch.float32: _lib.SS2D_F32, torch.bfloat16: _lib.SS2D_BF16, torch.float16: _lib.SS2D_F16}
ACTIVATIONS = (None, "silu")


def _check_sides(x, weight, bias, activation, what, rank):
    check_plain(x, "x", x=x, weight=weight, bias=bias)
    _check(x.dtype in _DTYPE_CODE, f"{what} not implemented for input type '{x.dtype}'")
    _check(x.dim() == rank, f"x must be {'(batch, tokens, dim)' if rank == 3 else '(batch, dim)'}")
    dim = x.shape[-1]
    _check(weight is not None and weight.dim() == 2 and weight.shape[0] == dim and 2 <= weight.shape[1] <= 4, "weight must have shape (dim, width) of width 2, 3 or 4")
    _check(weight.dtype in (torch.float32, x.dtype), "weight must be float32 or have x's dtype")
    _check(bias is None or (bias.dtype == weight.dtype and tuple(bias.shape) == (dim,)), "bias must have shape (dim,) and weight's dtype")
    _check(activation in ACTIVATIONS, "activation must be None or 'silu'")
    _check(dense_last(x), "x must be contiguous in its last dimension")
    _check(max(x.shape) <= MAX_SIZE, f"x must have no dimension of more than {MAX_SIZE}")


def _check_state(state, x, shape, name):
    if state is None:
        return
    check_plain(x, "x", **{name: state})
    _check(state.dtype == x.dtype and tuple(state.shape) == shape, f"{name} must have x's dtype and shape {shape}")


def _check_sequences(x, weight, bias, activation, initial_state, cu_seqlens):
    _check_sides(x, weight, bias, activation, "causal_conv_fn", 3)
    n_seqs = check_places(x, "x", cu_seqlens)
    _check_state(initial_state, x, (n_seqs, weight.shape[1] - 1, x.shape[2]), "initial_state")
    return n_seqs


def _params(x, weight, bias, activation, initial_state, cu_seqlens):
    p = _lib.CausalConvParams()
    p.batch, p.seqlen, p.dim = x.shape
    p.width, p.dtype, p.weight_dtype, p.silu = weight.shape[1], _DTYPE_CODE[x.dtype], _DTYPE_CODE[weight.dtype], int(activation == "silu")
    p.x, p.weight, p.bias, p.initial_state = x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial_state)
    if cu_seqlens is not None:
        p.cu_seqlens, p.n_seqs = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
    p.x_batch_stride, p.x_token_stride = x.stride()[:2]
    return p


class CausalConvHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, activation, cu_seqlens, want_final):
        with untraced():                                             # (a trace holds this call, with whatever tensors it is given when it runs)
            n_seqs = _check_sequences(x, weight, bias, activation, initial_state, cu_seqlens)
            if ctx.next_functions:                                   # (gradients are recorded)
                _lib.host().refuse_capture([x, weight, bias, initial_state], "causal_conv_fn")
            weight, bias, initial_state = (t if t is None else t.contiguous() for t in (weight, bias, initial_state))
            p = _params(x, weight, bias, activation, initial_state, cu_seqlens)
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            final = torch.empty((n_seqs, weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device) if want_final else None
            p.out, p.final_state = out.data_ptr(), _ptr(final)
            _lib.check(_lib.launch(x, _lib.lib().ss2d_causal_conv_fwd, p), "ss2d_causal_conv_fwd")
        ctx.activation = activation
        ctx.save_for_backward(x, weight, bias, initial_state, cu_seqlens)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, dout, dfinal):
        _check(not torch.is_grad_enabled(), "causal_conv_fn is differentiable once: its gradients have none (create_graph)")
        x, weight, bias, initial_state, cu_seqlens = ctx.saved_tensors
        n_seqs = _check_sequences(x, weight, bias, ctx.activation, initial_state, cu_seqlens)        # (a hook may have made something else of them)
        if dout is None:
            if dfinal is None:
                return (None,) * 7
            dout = x.new_zeros(x.shape)
        check_plain(x, "x", dout=dout, dfinal=dfinal)
        _check(dout.shape == x.shape and dout.dtype == x.dtype, "dout must have out's shape and type")
        _check_state(dfinal, x, (n_seqs, weight.shape[1] - 1, x.shape[2]), "dfinal")
        if not dense_last(dout):
            dout = dout.contiguous()
        weight, bias, initial_state, dfinal = (t if t is None else t.contiguous() for t in (weight, bias, initial_state, dfinal))
        p = _lib.CausalConvBwdParams()
        p.fwd = _params(x, weight, bias, ctx.activation, initial_state, cu_seqlens)
        want = ctx.needs_input_grad
        grads = [torch.empty(t.shape, dtype=t.dtype, device=x.device) if t is not None and (i == 0 or want[i]) else None
                 for i, t in enumerate((x, weight, bias, initial_state))]
        p.dout, p.dfinal_state = dout.data_ptr(), _ptr(dfinal)
        p.dout_batch_stride, p.dout_token_stride = dout.stride()[:2]
        p.dx, p.dweight, p.dbias, p.dinitial_state = (_ptr(t) for t in grads)
        L = _lib.lib()
        workspace = workspace_of(L.ss2d_causal_conv_bwd_workspace_bytes(p), "ss2d_causal_conv_bwd", x.device)
        _lib.check(_lib.launch(x, L.ss2d_causal_conv_bwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_causal_conv_bwd")
        return *grads, None, None, None


def causal_conv_fn(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """The causal convolution over sequences of tokens, differentiable in x, weight, bias and initial_state.

    x (batch, tokens, dim): bfloat16, float16 or float32, contiguous in the last dimension, any other strides.  weight (dim, width) of width 2, 3 or 4, the
    newest token's last, and bias (dim,) or None: one dtype, float32 or x's.  activation: None or "silu".
    cu_seqlens: int32 (sequences + 1,) on the GPU, the places in a batch of one at which packed sequences begin and the last one ends, ascending;
    sequences may be empty.  Rows of none of them come out as zeros, and so do their gradients.
    initial_state (sequences, width - 1, dim) in x's dtype: the inputs before the first token, the oldest first; None: zeros.

    Returns out (batch, tokens, dim) in x's dtype, with ``output_final_state`` (out, final_state): the last width - 1 inputs, which causal_conv_step_fn carries on.

    Differentiable once.  Captured into a graph with gradients, its leaves may belong to no autograd graph that was recorded on another stream and still lives."""
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a GPU tensor: vmamba_amd has no CPU path")
    if native_stands(x) and not torch.jit.is_tracing():              # (its memory is made where a tracer does not see it)
        native = _lib.host().causal_conv(TENSOR_KINDS, x, weight, bias, activation, initial_state, bool(output_final_state), cu_seqlens)
        if native is not None:
            return native
    out, final = CausalConvHip.apply(x, weight, bias, initial_state, activation, cu_seqlens, bool(output_final_state))
    return (out, final) if output_final_state else out


def causal_conv_step_fn(x, state, weight, bias=None, activation=None):
    """One token of each sequence: out (batch, dim) returned, and state (batch, width - 1, dim), in x's dtype, moved up by a row in place.

    x (batch, dim), weight, bias and activation as in causal_conv_fn, without the tokens.  The states have to be dense but for the batch's stride, which
    keeps them apart.  For inference: it refuses tensors that require a gradient while gradients are recorded, and to be traced
    (torch.jit.trace), since a trace would not hold what becomes of the state."""
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a GPU tensor: vmamba_amd has no CPU path")
    _check(not torch.jit.is_tracing(), "causal_conv_step_fn changes its state behind a tracer's back: it cannot be traced")
    if native_stands(x):
        native = _lib.host().causal_conv_step(TENSOR_KINDS, x, state, weight, bias, activation)
        if native is not None:
            return _lib.result(native, "ss2d_causal_conv_step")
    _check_sides(x, weight, bias, activation, "causal_conv_step_fn", 2)
    shape = (x.shape[0], weight.shape[1] - 1, x.shape[1])
    _check(state is not None, "state must be a tensor")
    _check_state(state, x, shape, "state")
    _check(state.shape[0] == 0 or state[0].is_contiguous(), "state must be contiguous but for its batch's stride")
    _check(state.shape[0] <= 1 or state.stride(0) >= shape[1] * shape[2], "the states of a batch must not overlap")
    check_unseen("causal_conv_step_fn", (x, state, weight, bias))
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    p = _lib.CausalConvStepParams()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    p.batch, p.dim, p.width, p.dtype, p.weight_dtype, p.silu = *x.shape, weight.shape[1], _DTYPE_CODE[x.dtype], _DTYPE_CODE[weight.dtype], int(activation == "silu")
    p.x, p.weight, p.bias, p.state, p.out = x.data_ptr(), weight.data_ptr(), _ptr(bias), state.data_ptr(), out.data_ptr()
    p.x_batch_stride, p.state_batch_stride = x.stride(0), state.stride(0) if state.shape[0] > 1 else shape[1] * shape[2]
    torch.autograd.graph.increment_version(state)                # (written in place, behind autograd's back)
    _lib.check(_lib.launch(x, _lib.lib().ss2d_causal_conv_step, p), "ss2d_causal_conv_step")
    return out
