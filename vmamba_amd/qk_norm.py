"""Norm of each head of an attention's queries and keys, and their rotation by position, in one pass (ss2d_qk_norm_rotate, with its gradients).

    n = x / sqrt(mean(x^2) + eps) * weight        over a head's dim values, statistics in float32
    (a, b) -> (a cos - b sin, b cos + a sin)      for the pairs of n's first values, by position * frequency

What linear_attention_fn reads as q and k.  Besides places in a text a position may have several axes, as a token of a map has a row and a column.
GPU tensors only: there is no CPU path here.  Arguments are checked as csms6s.py does and fail with RuntimeError.
"""
import torch

from . import _lib
from .linear_attention import MAX_SIZE, _check, _dense_last, _ptr, check_plain
from .norm import TENSOR_KINDS, native_stands, untraced

_DTYPE_CODE = {torch.float32: _lib.SS2D_F32, torch.bfloat16: _lib.SS2D_BF16, torch.float16: _lib.SS2D_F16}
MAX_DIM = 512


def _check_all(q, k, q_weight, k_weight, positions, frequencies):
    check_plain(q, q=q, k=k, q_weight=q_weight, k_weight=k_weight, positions=positions, frequencies=frequencies)
    _check(q.dtype in _DTYPE_CODE, f"qk_norm_rotate_fn not implemented for input type '{q.dtype}'")
    _check(k is not None and k.dtype == q.dtype, "k must have q's dtype")
    _check(q.dim() == 4 and k.dim() == 4 and k.shape[:2] == q.shape[:2] and k.shape[3] == q.shape[3],
           "q and k must be (batch, tokens, heads, dim) and agree in batch, tokens and dim")
    _check(1 <= q.shape[3] <= MAX_DIM, f"heads must have 1 to {MAX_DIM} values")
    for name, t in (("q", q), ("k", k)):
        _check(_dense_last(t), f"{name} must be contiguous in its last dimension")
        _check(max(t.shape) <= MAX_SIZE, f"{name} must have no dimension of more than {MAX_SIZE}")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        _check(w.dtype in (torch.float32, q.dtype) and w.dtype == weights[0].dtype, "weights must be of one type, float32 or q's dtype")
        _check(tuple(w.shape) == (q.shape[3],), f"weights must have shape ({q.shape[3]},)")
    _check((positions is None) == (frequencies is None), "positions and frequencies go together")
    if positions is not None:
        _check(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
        _check(frequencies.dtype in (torch.float32, torch.float64) and frequencies.dim() in (1, 2), "frequencies must be float32 or float64 of shape (pairs,) or (axes, pairs)")
        axes = (frequencies.shape[0],) if frequencies.dim() == 2 else ()
        _check(tuple(positions.shape) in ((*q.shape[:2], *axes), (q.shape[1], *axes)),
               f"positions must have shape {(*q.shape[:2], *axes)} or {(q.shape[1], *axes)}")
        _check(2 * frequencies.numel() <= q.shape[3], f"a head of {q.shape[3]} values has no {frequencies.numel()} pairs")


def _params(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
    p = _lib.QkNormRotateParams()
    p.batch, p.seqlen, p.q_heads, p.dim = q.shape
    p.k_heads = k.shape[2]
    weight = q_weight if q_weight is not None else k_weight
    p.dtype, p.weight_dtype = _DTYPE_CODE[q.dtype], _DTYPE_CODE[weight.dtype] if weight is not None else _lib.SS2D_F32
    p.eps, p.interleaved = eps, int(bool(interleaved))
    p.q, p.k, p.q_weight, p.k_weight = q.data_ptr(), k.data_ptr(), _ptr(q_weight), _ptr(k_weight)
    p.q_batch_stride, p.q_token_stride, p.q_head_stride = q.stride()[:3]
    p.k_batch_stride, p.k_token_stride, p.k_head_stride = k.stride()[:3]
    if positions is not None and frequencies.numel():
        p.axes, p.per_axis = frequencies.shape if frequencies.dim() == 2 else (1, frequencies.shape[0])
        p.positions, p.frequencies = positions.data_ptr(), frequencies.data_ptr()
        p.positions_int64, p.frequencies_float64 = int(positions.dtype == torch.int64), int(frequencies.dtype == torch.float64)
        strides = positions.stride() if frequencies.dim() == 2 else (*positions.stride(), 0)
        p.position_batch_stride, p.position_token_stride, p.position_axis_stride = strides if len(strides) == 3 else (0, *strides)
    return p


def qk_norm_rotate_fwd(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
    """(q, k) of arguments that qk_norm_rotate_fn has checked."""
    outs = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    p = _params(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved)
    p.q_out, p.k_out = (t.data_ptr() for t in outs)
    _lib.check(_lib.launch(q, _lib.lib().ss2d_qk_norm_rotate, p), "ss2d_qk_norm_rotate")
    return outs


class QkNormRotateHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
        with untraced():                                             # (a trace holds this call, with whatever tensors it is given when it runs)
            _check_all(q, k, q_weight, k_weight, positions, frequencies)
            if ctx.next_functions:                                   # (gradients are recorded)
                _lib.host().refuse_capture([q, k, q_weight, k_weight], "qk_norm_rotate_fn")
            q_weight, k_weight, frequencies = (t if t is None else t.contiguous() for t in (q_weight, k_weight, frequencies))
            outs = qk_norm_rotate_fwd(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.eps, ctx.interleaved = eps, interleaved
        return outs

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        _check(not torch.is_grad_enabled(), "qk_norm_rotate_fn is differentiable once: its gradients have none (create_graph)")
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        _check_all(q, k, q_weight, k_weight, positions, frequencies)               # (a hook may have made something else of them)
        q_weight, k_weight, frequencies = (t if t is None else t.contiguous() for t in (q_weight, k_weight, frequencies))
        check_plain(q, dq_out=dq_out, dk_out=dk_out)
        _check(dq_out.shape == q.shape and dk_out.shape == k.shape and dq_out.dtype == dk_out.dtype == q.dtype, "gradients must have the outputs' shapes and type")
        dq_out, dk_out = (t if _dense_last(t) else t.contiguous() for t in (dq_out, dk_out))
        g = _lib.QkNormRotateBwdParams()
        g.fwd = _params(q, k, q_weight, k_weight, positions, frequencies, ctx.eps, ctx.interleaved)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
        grads += [torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None and want else None
                  for w, want in zip((q_weight, k_weight), ctx.needs_input_grad[2:4])]
        g.dq_out, g.dk_out = dq_out.data_ptr(), dk_out.data_ptr()
        g.dq, g.dk, g.dq_weight, g.dk_weight = (_ptr(t) for t in grads)
        g.dq_batch_stride, g.dq_token_stride, g.dq_head_stride = dq_out.stride()[:3]
        g.dk_batch_stride, g.dk_token_stride, g.dk_head_stride = dk_out.stride()[:3]
        L = _lib.lib()
        need = L.ss2d_qk_norm_rotate_bwd_workspace_bytes(q.shape[3])
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        _lib.check(_lib.launch(q, L.ss2d_qk_norm_rotate_bwd, g, workspace.data_ptr(), need), "ss2d_qk_norm_rotate_bwd")
        return *grads, None, None, None, None


def qk_norm_rotate_fn(q, k, q_weight=None, k_weight=None, positions=None, frequencies=None, eps=1e-6, interleaved=False):
    """(q, k) with each head normalised and rotated, differentiable in q, k and the weights.

    q (batch, tokens, q_heads, dim), k (batch, tokens, k_heads, dim): one dtype (bfloat16, float16 or float32), contiguous in the last dimension, any
    other strides, dim up to 512.  q_weight, k_weight (dim,): float32 or q's dtype, either may be None (ones).
    positions int32 or int64 with frequencies float32 or float64: (batch, tokens) or (tokens,) with (pairs,), or several axes (batch, tokens, axes) or
    (tokens, axes) with (axes, pairs): pair a * pairs + i of a head turns by positions[.., a] * frequencies[a, i], a product in 64 bits.  Pair
    i is values (i, i + R / 2) of the first R = 2 * frequencies.numel() values of a head, with ``interleaved`` values (2 i, 2 i + 1); what is behind them is
    not turned.  Without positions nothing is.

    Differentiable once.  Captured into a graph with gradients, its leaves may belong to no autograd graph that was recorded on another stream and still lives."""
    _check(isinstance(q, torch.Tensor) and q.is_cuda, "q must be a GPU tensor: vmamba_amd has no CPU path")
    if native_stands(q) and not torch.jit.is_tracing():              # (its memory is made where a tracer does not see it)
        native = _lib.host().qk_norm_rotate(TENSOR_KINDS, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved)
        if native is not None:
            return native
    return QkNormRotateHip.apply(q, k, q_weight, k_weight, positions, frequencies, float(eps), bool(interleaved))
