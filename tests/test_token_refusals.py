"""What the selective scan of tokens, the causal convolution, their single tokens and the group norm refuse: every case on the CPU first, where nothing can be
launched (tensors that say they are the GPU's; a launch fails the test), then on the GPU through the native host calls; and the checks of the C entries, which are made
before anything is launched."""
import ctypes

import pytest
import torch

import vmamba_amd
from vmamba_amd import _lib, causal_conv, group_norm, token_scan

F32, F16, BF16, F64, INT = torch.float32, torch.float16, torch.bfloat16, torch.float64, torch.int32
HERE = ctypes.c_void_p(256)          # an aligned address, never read: the calls with it are refused first


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is the GPU's."""
    is_cuda = property(lambda self: True)


def on_cpu(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def on_gpu(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype, device="cuda:0")


def made(make, a, change):
    return a | {n: c(make) if callable(c) else c for n, c in change.items()}


def scan(make, *, b=2, t=5, d=12, n=4, g=2, **change):
    return made(make, dict(u=make(b, t, d), delta=make(b, t, d), A=make(d, n), B=make(b, t, g, n), C=make(b, t, g, n), D=None, z=None, delta_bias=None, initial_state=None,
                           cu_seqlens=None), change)


SCAN = {
    "no u": dict(u=None), "u a number": dict(u=3), "delta none": dict(delta=None), "A none": dict(A=None), "B a list": dict(B=[1.0]), "C none": dict(C=None),
    "rank of u": dict(u=lambda m: m(5, 12)), "64 bits": dict(u=lambda m: m(2, 5, 12, dtype=F64)), "whole numbers": dict(u=lambda m: m(2, 5, 12, dtype=INT)),
    "delta's type": dict(delta=lambda m: m(2, 5, 12, dtype=BF16)), "delta's shape": dict(delta=lambda m: m(2, 5, 1)), "z's type": dict(z=lambda m: m(2, 5, 12, dtype=F16)),
    "z's shape": dict(z=lambda m: m(2, 4, 12)), "B's type": dict(B=lambda m: m(2, 5, 2, 4, dtype=F16)), "B's rank": dict(B=lambda m: m(2, 5, 4)), "C's tokens": dict(C=lambda m: m(2, 6, 2, 4)),
    "C's groups": dict(C=lambda m: m(2, 5, 1, 4)), "C's states": dict(C=lambda m: m(2, 5, 2, 5)), "groups that do not divide": dict(g=5), "no groups": dict(g=0),
    "A's type": dict(A=lambda m: m(12, 4, dtype=BF16)), "A's shape": dict(A=lambda m: m(4, 12)), "no states": dict(n=0), "too many states": dict(n=65),
    "D's type": dict(D=lambda m: m(12, dtype=BF16)), "D's shape": dict(D=lambda m: m(1)), "bias' type": dict(delta_bias=lambda m: m(12, dtype=F16)), "bias' shape": dict(delta_bias=lambda m: m(11)),
    "u not dense": dict(u=lambda m: m(2, 12, 5).transpose(1, 2)), "B not dense": dict(B=lambda m: m(2, 5, 4, 2).transpose(2, 3)), "z not dense": dict(z=lambda m: m(2, 5, 24)[..., ::2]),
    "state's type": dict(initial_state=lambda m: m(2, 12, 4, dtype=BF16)), "state's shape": dict(initial_state=lambda m: m(2, 4, 12)), "state's sequences": dict(initial_state=lambda m: m(1, 12, 4)),
    "places in a batch of two": dict(cu_seqlens=lambda m: m(3, dtype=INT)), "places of 64 bits": dict(b=1, cu_seqlens=lambda m: m(3, dtype=torch.int64)),
    "one place": dict(b=1, cu_seqlens=lambda m: m(1, dtype=INT)), "places' rank": dict(b=1, cu_seqlens=lambda m: m(1, 3, dtype=INT)),
    "every other place": dict(b=1, cu_seqlens=lambda m: m(6, dtype=INT)[::2]), "state of packed sequences": dict(b=1, cu_seqlens=lambda m: m(3, dtype=INT), initial_state=lambda m: m(1, 12, 4)),
}


def scan_step(make, *, b=2, d=12, n=4, g=2, **change):
    return made(make, dict(u=make(b, d), delta=make(b, d), A=make(d, n), B=make(b, g, n), C=make(b, g, n), state=make(b, d, n), D=None, z=None, delta_bias=None), change)


SCAN_STEP = {
    "with tokens": dict(u=lambda m: m(2, 1, 12)), "batch": dict(b=3, u=lambda m: m(2, 12)), "no state": dict(state=None), "state's type": dict(state=lambda m: m(2, 12, 4, dtype=F16)),
    "state's shape": dict(state=lambda m: m(2, 4, 12)), "states in one place": dict(state=lambda m: m(1, 12, 4).expand(2, 12, 4)),
    "states that overlap": dict(state=lambda m: m(200).as_strided((2, 12, 4), (47, 4, 1))), "a state turned": dict(state=lambda m: m(2, 4, 12).transpose(1, 2)),
    "gradients": dict(B=lambda m: m(2, 2, 4).requires_grad_()), "a state with a gradient": dict(state=lambda m: m(2, 12, 4).requires_grad_()), "too many states": dict(n=100),
    "B's rank": dict(B=lambda m: m(2, 4)), "z's type": dict(z=lambda m: m(2, 12, dtype=BF16)), "D's shape": dict(D=lambda m: m(4)),
}


def conv(make, *, b=2, t=5, d=12, w=4, **change):
    return made(make, dict(x=make(b, t, d), weight=make(d, w), bias=None, activation=None, initial_state=None, cu_seqlens=None), change)


CONV = {
    "no x": dict(x=None), "no weight": dict(weight=None), "rank": dict(x=lambda m: m(5, 12)), "64 bits": dict(x=lambda m: m(2, 5, 12, dtype=F64)), "one tap": dict(w=1), "five taps": dict(w=5),
    "weight's shape": dict(weight=lambda m: m(4, 12)), "weight's rank": dict(weight=lambda m: m(12, 1, 4)), "weight's type": dict(weight=lambda m: m(12, 4, dtype=BF16)),
    "bias' shape": dict(bias=lambda m: m(11)), "bias' type": dict(x=lambda m: m(2, 5, 12, dtype=BF16), weight=lambda m: m(12, 4), bias=lambda m: m(12, dtype=BF16)),
    "another activation": dict(activation="gelu"), "an activation that is true": dict(activation=True), "not dense": dict(x=lambda m: m(2, 12, 5).transpose(1, 2)),
    "state's type": dict(initial_state=lambda m: m(2, 3, 12, dtype=F16)), "state's shape": dict(initial_state=lambda m: m(2, 12, 3)), "state's sequences": dict(initial_state=lambda m: m(1, 3, 12)),
    "places in a batch of two": dict(cu_seqlens=lambda m: m(3, dtype=INT)), "places of floats": dict(b=1, cu_seqlens=lambda m: m(3)), "one place": dict(b=1, cu_seqlens=lambda m: m(1, dtype=INT)),
}


def conv_step(make, *, b=2, d=12, w=4, **change):
    return made(make, dict(x=make(b, d), state=make(b, w - 1, d), weight=make(d, w), bias=None, activation=None), change)


CONV_STEP = {
    "with tokens": dict(x=lambda m: m(2, 1, 12)), "no state": dict(state=None), "state's type": dict(state=lambda m: m(2, 3, 12, dtype=BF16)), "state's rows": dict(state=lambda m: m(2, 4, 12)),
    "state's batch": dict(state=lambda m: m(3, 3, 12)), "states in one place": dict(state=lambda m: m(1, 3, 12).expand(2, 3, 12)), "states that overlap": dict(state=lambda m: m(99).as_strided((2, 3, 12), (35, 12, 1))),
    "a state turned": dict(state=lambda m: m(2, 12, 3).transpose(1, 2)), "gradients": dict(weight=lambda m: m(12, 4).requires_grad_()), "five taps": dict(w=5), "another activation": dict(activation="relu"),
}


def norm(make, *, b=2, p=5, c=12, g=3, **change):
    return made(make, dict(x=make(b, p, c), num_groups=g, weight=None, bias=None, activation=None), change)


NORM = {
    "no x": dict(x=None), "rank": dict(x=lambda m: m(12)), "64 bits": dict(x=lambda m: m(2, 5, 12, dtype=F64)), "groups that do not divide": dict(g=5), "no groups": dict(g=0), "half a group": dict(g=1.5),
    "minus a group": dict(g=-3), "no channels": dict(c=0), "weight's shape": dict(weight=lambda m: m(3)), "bias' shape": dict(bias=lambda m: m(1, 12)), "weight's type": dict(weight=lambda m: m(12, dtype=F16)),
    "weights of two types": dict(x=lambda m: m(2, 5, 12, dtype=BF16), weight=lambda m: m(12), bias=lambda m: m(12, dtype=BF16)), "another activation": dict(activation="tanh"),
}
CALLS = [(vmamba_amd.selective_scan_tokens_fn, scan, SCAN), (vmamba_amd.selective_scan_step_fn, scan_step, SCAN_STEP), (vmamba_amd.causal_conv_fn, conv, CONV),
         (vmamba_amd.causal_conv_step_fn, conv_step, CONV_STEP), (vmamba_amd.group_norm_fn, norm, NORM)]
CASES = [pytest.param(call, build, change, id=f"{build.__name__}: {name}") for call, build, changes in CALLS for name, change in changes.items()]
NAMES = [build.__name__ for _, build, _ in CALLS]


def alike(like, what, /, **tensors):
    for n, t in tensors.items():
        token_scan._check(t is None or isinstance(t, torch.Tensor), f"{n} must be a tensor")


@pytest.mark.parametrize("call,build,change", CASES)
def test_refused_before_anything_runs(call, build, change, monkeypatch):
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    for module in (token_scan, causal_conv, group_norm):
        monkeypatch.setattr(module, "check_plain", alike)
    with pytest.raises(RuntimeError) as error:
        call(**build(on_cpu, **change))
    assert "ss2d_" not in str(error.value), "said by the kernels' entry, not by the caller's checks"


@pytest.mark.gpu
@pytest.mark.parametrize("call,build,change", CASES)
def test_refused_on_the_gpu(call, build, change):
    print("CASE refused", build.__name__, sorted(change), flush=True)
    with pytest.raises(RuntimeError) as error:
        call(**build(on_gpu, **change))
    assert "ss2d_" not in str(error.value)


@pytest.mark.gpu
@pytest.mark.parametrize("call,build,changes", CALLS, ids=NAMES)
def test_tensors_elsewhere_are_refused(call, build, changes):
    """Each tensor in turn on the CPU, of a class of its own, or without memory."""
    full = build(on_gpu)
    more = dict(D=on_gpu(12), z=on_gpu(*full["u"].shape), delta_bias=on_gpu(12)) if "u" in full else dict(bias=on_gpu(12))
    more |= dict(weight=on_gpu(12)) if "num_groups" in full else {}
    more |= dict(initial_state=on_gpu(2, 12, 4) if "u" in full else on_gpu(2, 3, 12)) if "initial_state" in full else {}
    full |= more
    with torch.no_grad():
        call(**full)
        for name, t in full.items():
            if not isinstance(t, torch.Tensor):
                continue
            for other in (t.cpu(), t.as_subclass(OnGpu), torch.empty(t.shape, dtype=t.dtype, device="meta")):
                with pytest.raises(RuntimeError):
                    call(**full | {name: other})


@pytest.mark.parametrize("call,build,changes", CALLS, ids=NAMES)
def test_no_cpu_path(call, build, changes):
    with pytest.raises(RuntimeError, match="GPU tensor"):
        call(**build(torch.zeros))


@pytest.mark.parametrize("call,build,changes", [c for c in CALLS if "step" in c[1].__name__], ids=["scan", "conv"])
def test_a_traced_step_is_refused(call, build, changes, monkeypatch):
    monkeypatch.setattr(torch.jit, "is_tracing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        call(**build(on_cpu))


# ---- the C entries -------------------------------------------------------------------------------------------------------------------
def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_lib.TokenScanParams) == 8 * 4 + 13 * 8 + 12 * 8 and _lib.TokenScanParams.u.offset == 32 and _lib.TokenScanParams.u_batch_stride.offset == 136
    assert ctypes.sizeof(_lib.TokenScanBwdParams) == 232 + 11 * 8 + 2 * 8 and _lib.TokenScanBwdParams.dout.offset == 232
    assert ctypes.sizeof(_lib.TokenScanStepParams) == 6 * 4 + 10 * 8 + 8 * 8 and _lib.TokenScanStepParams.u_batch_stride.offset == 104
    assert ctypes.sizeof(_lib.CausalConvParams) == 8 * 4 + 7 * 8 + 2 * 8 and ctypes.sizeof(_lib.CausalConvBwdParams) == 104 + 6 * 8 + 2 * 8
    assert ctypes.sizeof(_lib.CausalConvStepParams) == 6 * 4 + 5 * 8 + 2 * 8
    assert ctypes.sizeof(_lib.GroupNormParams) == 2 * 8 + 6 * 4 + 5 * 8 and ctypes.sizeof(_lib.GroupNormBwdParams) == 80 + 4 * 8


def fill(p, **values):
    for name, value in values.items():
        setattr(p, name, value)
    return p


def scan_params(**change):
    return fill(_lib.TokenScanParams(), **(dict(batch=2, seqlen=500, dim=64, dstate=16, n_groups=2, dtype=_lib.SS2D_BF16, delta_softplus=1, u=256, delta=256, A=256, B=256, C=256, out=256,
                                                u_token_stride=64, delta_token_stride=64, B_token_stride=32, C_token_stride=32) | change))


def scan_grads(fwd, **change):
    return fill(_lib.TokenScanBwdParams(), **(dict(fwd=fwd, dout=256, du=256, ddelta=256, dB=256, dC=256) | change))


@pytest.mark.parametrize("change", [dict(batch=-1), dict(seqlen=-1), dict(dim=-2), dict(dstate=0), dict(n_groups=0), dict(n_groups=3), dict(dtype=7), dict(dtype=-1), dict(n_seqs=-1),
                                    dict(cu_seqlens=256, n_seqs=3), dict(batch=1, cu_seqlens=256, n_seqs=0)], ids=str)
def test_scans_of_bad_arguments(change):
    L, p = _lib.lib(), scan_params(**change)
    g = scan_grads(p)
    assert L.ss2d_token_scan_workspace_bytes(p) == L.ss2d_token_scan_kept_states(p) == L.ss2d_token_scan_fwd(p, HERE, 1 << 40, None) == _lib.SS2D_EINVAL
    assert L.ss2d_token_scan_bwd_workspace_bytes(g) == L.ss2d_token_scan_bwd(g, HERE, 1 << 40, None) == _lib.SS2D_EINVAL


def test_scans_of_too_much():
    L = _lib.lib()
    for change in (dict(dstate=65), dict(seqlen=2 ** 31 - 1), dict(batch=2 ** 31 - 1, dim=4096), dict(dim=2 ** 30)):
        p = scan_params(**change)
        g = scan_grads(p)
        assert L.ss2d_token_scan_workspace_bytes(p) == L.ss2d_token_scan_fwd(p, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change
        assert L.ss2d_token_scan_bwd_workspace_bytes(g) == L.ss2d_token_scan_bwd(g, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change


def test_scans_workspace_and_results():
    L = _lib.lib()
    for call in (L.ss2d_token_scan_fwd, L.ss2d_token_scan_bwd, L.ss2d_causal_conv_bwd, L.ss2d_group_norm_fwd, L.ss2d_group_norm_bwd):
        assert call(None, HERE, 1 << 20, None) == _lib.SS2D_EINVAL
    for call in (L.ss2d_token_scan_step, L.ss2d_causal_conv_fwd, L.ss2d_causal_conv_step):
        assert call(None, None) == _lib.SS2D_EINVAL
    p = scan_params()
    g = scan_grads(p)
    p_kept = fill(scan_params(), kept_states=256)
    g_kept = scan_grads(p_kept)
    need, need_bwd = L.ss2d_token_scan_workspace_bytes(p), L.ss2d_token_scan_bwd_workspace_bytes(g)
    assert need > 0 and need_bwd >= 2 * 500 * 2 * 16 * 8 and L.ss2d_token_scan_kept_states(p) == 2 * 32 * 64 * 16
    for call, params, bytes_ in ((L.ss2d_token_scan_fwd, p, need), (L.ss2d_token_scan_bwd, g_kept, need_bwd)):
        assert call(params, None, bytes_, None) == call(params, ctypes.c_void_p(264), bytes_, None) == _lib.SS2D_EINVAL
        assert call(params, HERE, bytes_ - 1, None) == _lib.SS2D_ENOMEM
    for missing in ("u", "delta", "A", "B", "C", "out"):
        assert L.ss2d_token_scan_fwd(scan_params(**{missing: None}), HERE, need, None) == _lib.SS2D_EINVAL, missing
    assert L.ss2d_token_scan_bwd(g, HERE, need_bwd, None) == _lib.SS2D_EINVAL                      # without the kept states
    for missing in ("dout", "du", "ddelta", "dB", "dC"):
        assert L.ss2d_token_scan_bwd(scan_grads(p_kept, **{missing: None}), HERE, need_bwd, None) == _lib.SS2D_EINVAL, missing
    assert L.ss2d_token_scan_bwd(scan_grads(fill(scan_params(), kept_states=256, z=256)), HERE, need_bwd, None) == _lib.SS2D_EINVAL      # a gate without its gradient
    for empty in (dict(batch=0), dict(dim=0)):
        p = scan_params(**empty, u=None, delta=None, B=None, C=None)
        assert L.ss2d_token_scan_workspace_bytes(p) == 0 and L.ss2d_token_scan_fwd(p, None, 0, None) == _lib.SS2D_OK
    p = scan_params(dim=0, u=None)
    assert L.ss2d_token_scan_bwd_workspace_bytes(scan_grads(p)) == 0 and L.ss2d_token_scan_bwd(scan_grads(p), None, 0, None) == _lib.SS2D_OK


def test_scan_steps_of_bad_arguments():
    L = _lib.lib()
    make = lambda **change: fill(_lib.TokenScanStepParams(), **(dict(batch=2, dim=64, dstate=16, n_groups=2, dtype=_lib.SS2D_F16, u=256, delta=256, A=256, B=256, C=256, state=256,  # noqa: E731
                                                                     out=256, state_batch_stride=1024) | change))
    for change in (dict(batch=-1), dict(dim=-1), dict(dstate=0), dict(n_groups=0), dict(n_groups=5), dict(dtype=3), dict(u=None), dict(delta=None), dict(A=None), dict(B=None), dict(C=None),
                   dict(state=None), dict(out=None), dict(state_batch_stride=1023), dict(state_batch_stride=0)):
        assert L.ss2d_token_scan_step(make(**change), None) == _lib.SS2D_EINVAL, change
    for change in (dict(dstate=65), dict(batch=2 ** 31 - 1, dim=2 ** 20)):
        assert L.ss2d_token_scan_step(make(**change, state_batch_stride=1 << 40), None) == _lib.SS2D_ENOTSUP, change
    assert L.ss2d_token_scan_step(make(batch=0, u=None), None) == L.ss2d_token_scan_step(make(dim=0, u=None), None) == _lib.SS2D_OK


def test_convolutions_of_bad_arguments():
    L = _lib.lib()
    make = lambda **change: fill(_lib.CausalConvParams(), **(dict(batch=2, seqlen=50, dim=64, width=4, dtype=_lib.SS2D_BF16, weight_dtype=_lib.SS2D_F32, x=256, weight=256, out=256,  # noqa: E731
                                                                  x_token_stride=64, x_batch_stride=3200) | change))
    back = lambda fwd, **change: fill(_lib.CausalConvBwdParams(), **(dict(fwd=fwd, dout=256, dx=256) | change))  # noqa: E731
    for change in (dict(batch=-1), dict(seqlen=-1), dict(dim=-1), dict(dtype=4), dict(weight_dtype=_lib.SS2D_F16), dict(n_seqs=-1), dict(cu_seqlens=256, n_seqs=2), dict(batch=1, cu_seqlens=256)):
        assert L.ss2d_causal_conv_fwd(make(**change), None) == L.ss2d_causal_conv_bwd(back(make(**change)), HERE, 1 << 40, None) == _lib.SS2D_EINVAL, change
        assert L.ss2d_causal_conv_bwd_workspace_bytes(back(make(**change))) == _lib.SS2D_EINVAL
    for change in (dict(x=None), dict(weight=None), dict(out=None)):
        assert L.ss2d_causal_conv_fwd(make(**change), None) == _lib.SS2D_EINVAL, change
    for change in (dict(width=1), dict(width=5), dict(seqlen=2 ** 31 - 1), dict(batch=2 ** 31 - 1, dim=2 ** 20), dict(dim=2 ** 30 + 1)):
        assert L.ss2d_causal_conv_fwd(make(**change), None) == L.ss2d_causal_conv_bwd(back(make(**change)), HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change
    need = L.ss2d_causal_conv_bwd_workspace_bytes(back(make()))
    assert need >= 5 * 64 * 4
    for change in (dict(dout=None), dict(dx=None)):
        assert L.ss2d_causal_conv_bwd(back(make(), **change), HERE, need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_causal_conv_bwd(back(make()), None, need, None) == L.ss2d_causal_conv_bwd(back(make()), ctypes.c_void_p(260), need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_causal_conv_bwd(back(make()), HERE, need - 1, None) == _lib.SS2D_ENOMEM
    for empty in (dict(batch=0), dict(dim=0)):
        assert L.ss2d_causal_conv_fwd(make(**empty, x=None, out=None), None) == _lib.SS2D_OK
    step = lambda **change: fill(_lib.CausalConvStepParams(), **(dict(batch=2, dim=64, width=4, dtype=_lib.SS2D_F32, weight_dtype=_lib.SS2D_F32, x=256, weight=256, state=256, out=256,  # noqa: E731
                                                                      state_batch_stride=192) | change))
    for change in (dict(batch=-1), dict(dim=-1), dict(dtype=5), dict(weight_dtype=_lib.SS2D_BF16), dict(x=None), dict(weight=None), dict(state=None), dict(out=None), dict(state_batch_stride=191)):
        assert L.ss2d_causal_conv_step(step(**change), None) == _lib.SS2D_EINVAL, change
    assert L.ss2d_causal_conv_step(step(width=5), None) == L.ss2d_causal_conv_step(step(dim=2 ** 30 + 1, state_batch_stride=1 << 40), None) == _lib.SS2D_ENOTSUP
    assert L.ss2d_causal_conv_step(step(batch=0, x=None), None) == _lib.SS2D_OK


def test_norms_of_bad_arguments():
    L = _lib.lib()
    make = lambda **change: fill(_lib.GroupNormParams(), **(dict(batch=4, positions=5000, channels=64, groups=4, dtype=_lib.SS2D_F16, weight_dtype=_lib.SS2D_F16, eps=1e-5, x=256, out=256) | change))  # noqa: E731
    back = lambda fwd, **change: fill(_lib.GroupNormBwdParams(), **(dict(fwd=fwd, dout=256, dx=256) | change))  # noqa: E731
    for change in (dict(batch=-1), dict(positions=-1), dict(channels=0), dict(groups=0), dict(groups=3), dict(dtype=4), dict(weight_dtype=_lib.SS2D_BF16)):
        assert L.ss2d_group_norm_workspace_bytes(make(**change)) == L.ss2d_group_norm_fwd(make(**change), HERE, 1 << 40, None) == _lib.SS2D_EINVAL, change
        assert L.ss2d_group_norm_bwd_workspace_bytes(back(make(**change))) == L.ss2d_group_norm_bwd(back(make(**change)), HERE, 1 << 40, None) == _lib.SS2D_EINVAL, change
    for change in (dict(batch=2 ** 31), dict(positions=2 ** 31 - 1), dict(batch=2 ** 30, positions=2 ** 20)):
        assert L.ss2d_group_norm_workspace_bytes(make(**change)) == L.ss2d_group_norm_fwd(make(**change), HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change
    need, kept = L.ss2d_group_norm_workspace_bytes(make()), make(stats=256)
    need_bwd = L.ss2d_group_norm_bwd_workspace_bytes(back(kept))
    assert need > 0 and need_bwd > 0 and L.ss2d_group_norm_workspace_bytes(make(positions=1)) == 0
    assert L.ss2d_group_norm_fwd(make(x=None), HERE, need, None) == L.ss2d_group_norm_fwd(make(out=None), HERE, need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_group_norm_bwd(back(make()), HERE, need_bwd, None) == _lib.SS2D_EINVAL            # without the statistics
    for change in (dict(dout=None), dict(dx=None)):
        assert L.ss2d_group_norm_bwd(back(kept, **change), HERE, need_bwd, None) == _lib.SS2D_EINVAL
    for call, params, bytes_ in ((L.ss2d_group_norm_fwd, make(), need), (L.ss2d_group_norm_bwd, back(kept), need_bwd)):
        assert call(params, None, bytes_, None) == call(params, ctypes.c_void_p(264), bytes_, None) == _lib.SS2D_EINVAL
        assert call(params, HERE, bytes_ - 1, None) == _lib.SS2D_ENOMEM
    assert L.ss2d_group_norm_fwd(make(batch=0, x=None), None, 0, None) == L.ss2d_group_norm_fwd(make(positions=0, x=None), None, 0, None) == _lib.SS2D_OK


# ---- sizes over 32 bits, and what only Python's form sees ---------------------------------------------------------------------------------
def stretched(*shape, dtype=F32):
    """A tensor of any number of rows in the memory of one."""
    return torch.zeros(shape[-1], dtype=dtype).expand(*shape).as_subclass(OnGpu)


@pytest.mark.parametrize("build,sizes", [(scan, dict(t=2 ** 31)), (scan, dict(b=2 ** 31)), (scan_step, dict(b=2 ** 31)), (conv, dict(t=2 ** 31)), (conv_step, dict(b=2 ** 31)),
                                         (norm, dict(b=2 ** 31)), (norm, dict(p=2 ** 31 - 65535))], ids=lambda v: getattr(v, "__name__", str(v)))
def test_sizes_over_32_bits_are_refused(build, sizes, monkeypatch):
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    for module in (token_scan, causal_conv, group_norm):
        monkeypatch.setattr(module, "check_plain", alike)
    call = next(c for c, b, _ in CALLS if b is build)
    with pytest.raises(RuntimeError) as error:
        call(**build(stretched, **sizes))
    print(error.value)


def test_forward_derivatives_are_refused(monkeypatch):
    """A step changes its state in place, and a derivative of it would be dropped."""
    import torch.autograd.forward_ad as fwd
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    for module in (token_scan, causal_conv):
        monkeypatch.setattr(module, "check_plain", alike)
    for call, build in ((vmamba_amd.selective_scan_step_fn, scan_step), (vmamba_amd.causal_conv_step_fn, conv_step)):
        with fwd.dual_level():
            a = build(on_cpu)
            name = "u" if "u" in a else "x"
            a[name] = fwd.make_dual(torch.zeros(2, 12), torch.ones(2, 12))
            monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
            with torch.no_grad(), pytest.raises(RuntimeError, match="derivative forward"):
                call(**a)
