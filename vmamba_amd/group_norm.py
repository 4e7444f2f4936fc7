"""Group norm of channel-last activations with an activation behind it, and its gradients (ss2d_group_norm).

    y = act((x - mean) / sqrt(var + eps) * weight + bias)       mean and var over the positions and a group's channels of one sample

Tokens (tokens, channels) are normalised each by itself, as behind a mixer of tokens; feature maps (batch, height, width, channels) over all their
positions.  norm.py has the norms over all channels of a position.  GPU tensors only: there is no CPU path here.  Arguments are checked as csms6s.py
does and fail with RuntimeError.
"""
import torch

from . import _lib
from .causal_conv import ACTIVATIONS
from .norm import TENSOR_KINDS, native_stands, untraced
from .token_scan import MAX_SIZE, _check, _ptr, check_plain, workspace_of

_DTYPE_CODE = {torch.float32: _lib.SS2D_F32, torch.bfloat16: _lib.SS2D_BF16, torch.float16: _lib.SS2D_F16}


def _check_all(x, num_groups, weight, bias, activation):
    check_plain(x, "x", x=x, weight=weight, bias=bias)
    _check(x.dtype in _DTYPE_CODE, f"group_norm_fn not implemented for input type '{x.dtype}'")
    _check(x.dim() >= 2, "x must be (batch, ..., channels)")
    C = x.shape[-1]
    _check(isinstance(num_groups, int) and num_groups >= 1 and C >= 1 and C % num_groups == 0, "channels must be dividable by num_groups")
    for name, t in (("weight", weight), ("bias", bias)):
        _check(t is None or tuple(t.shape) == (C,), f"{name} must have shape ({C},)")
        _check(t is None or t.dtype in (torch.float32, x.dtype), f"{name} must be float32 or have x's dtype")
    _check(weight is None or bias is None or weight.dtype == bias.dtype, "weight and bias must be of one type")
    _check(activation in ACTIVATIONS, "activation must be None or 'silu'")
    positions = x[0].numel() // C if x.shape[0] else 0
    _check(x.shape[0] <= MAX_SIZE and positions <= MAX_SIZE - 65536 and C <= 1 << 30, "x must have no more samples or positions than 32 bits count")
    return positions


def _params(x, positions, num_groups, weight, bias, eps, activation):
    p = _lib.GroupNormParams()
    p.batch, p.positions, p.channels, p.groups = x.shape[0], positions, x.shape[-1], num_groups
    weights = weight if weight is not None else bias
    p.dtype, p.weight_dtype = _DTYPE_CODE[x.dtype], _DTYPE_CODE[weights.dtype] if weights is not None else _lib.SS2D_F32
    p.silu, p.eps = int(activation == "silu"), eps
    p.x, p.weight, p.bias = x.data_ptr(), _ptr(weight), _ptr(bias)
    return p


class GroupNormHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, activation):
        with untraced():                                             # (a trace holds this call, with whatever tensors it is given when it runs)
            positions = _check_all(x, num_groups, weight, bias, activation)
            record = bool(ctx.next_functions)
            if record:                                               # (gradients are recorded)
                _lib.host().refuse_capture([x, weight, bias], "group_norm_fn")
            x, weight, bias = (t if t is None else t.contiguous() for t in (x, weight, bias))
            p = _params(x, positions, num_groups, weight, bias, eps, activation)
            L = _lib.lib()
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            stats = torch.empty((x.shape[0], num_groups, 2), dtype=torch.float32, device=x.device) if record else None
            p.out, p.stats = out.data_ptr(), _ptr(stats)
            workspace = workspace_of(L.ss2d_group_norm_workspace_bytes(p), "ss2d_group_norm_fwd", x.device)
            _lib.check(_lib.launch(x, L.ss2d_group_norm_fwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_group_norm_fwd")
        ctx.num_groups, ctx.eps, ctx.activation = num_groups, eps, activation
        ctx.save_for_backward(x, weight, bias, stats)
        return out

    @staticmethod
    def backward(ctx, dout):
        _check(not torch.is_grad_enabled(), "group_norm_fn is differentiable once: its gradients have none (create_graph)")
        x, weight, bias, stats = ctx.saved_tensors
        positions = _check_all(x, ctx.num_groups, weight, bias, ctx.activation)         # (a hook may have made something else of them)
        check_plain(x, "x", dout=dout, stats=stats)
        _check(dout.shape == x.shape and dout.dtype == x.dtype, "dout must have out's shape and type")
        _check(stats is not None and stats.dtype == torch.float32 and stats.is_contiguous() and tuple(stats.shape) == (x.shape[0], ctx.num_groups, 2),
               "the statistics kept for the gradients are not what was kept")
        x, weight, bias, dout = (t if t is None else t.contiguous() for t in (x, weight, bias, dout))
        p = _lib.GroupNormBwdParams()
        p.fwd = _params(x, positions, ctx.num_groups, weight, bias, ctx.eps, ctx.activation)
        p.fwd.stats, p.dout = stats.data_ptr(), dout.data_ptr()
        grads = [torch.empty(t.shape, dtype=t.dtype, device=x.device) if t is not None and (i == 0 or ctx.needs_input_grad[i]) else None for i, t in enumerate((x, weight, bias))]
        p.dx, p.dweight, p.dbias = (_ptr(t) for t in grads)
        L = _lib.lib()
        workspace = workspace_of(L.ss2d_group_norm_bwd_workspace_bytes(p), "ss2d_group_norm_bwd", x.device)
        _lib.check(_lib.launch(x, L.ss2d_group_norm_bwd, p, workspace.data_ptr(), workspace.numel()), "ss2d_group_norm_bwd")
        return *grads, None, None, None


def group_norm_fn(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Group norm over the last dimension's groups, differentiable in x, weight and bias.

    x (batch, ..., channels): bfloat16, float16 or float32; what is not contiguous is copied.  Group g is the channels / num_groups channels from
    g * channels / num_groups on; each sample's group has its own statistics, over all dimensions between the first and the last too.  weight, bias (channels,): of one
    type, float32 or x's, either may be None.  activation: None or "silu".  Statistics are float32, squares those of centred values.

    Differentiable once.  Captured into a graph with gradients, its leaves may belong to no autograd graph that was recorded on another stream and still lives."""
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a GPU tensor: vmamba_amd has no CPU path")
    if type(num_groups) is int and native_stands(x) and not torch.jit.is_tracing():             # (its memory is made where a tracer does not see it)
        native = _lib.host().group_norm(TENSOR_KINDS, x, num_groups, weight, bias, eps, activation)
        if native is not None:
            return native
    return GroupNormHip.apply(x, weight, bias, num_groups, float(eps), activation)
