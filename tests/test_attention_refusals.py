"""What linear_attention_fn, linear_attention_step_fn and qk_norm_rotate_fn refuse: every case on the CPU first, where nothing can be launched (tensors that
say they are the GPU's; a launch fails the test), then on the GPU through the native host calls; and the checks of the C entries, which
are made before anything is launched."""
import ctypes

import pytest
import torch

import vmamba_amd
from vmamba_amd import _lib, linear_attention, qk_norm

F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
HERE = ctypes.c_void_p(256)          # an aligned address, never read: the calls with it are refused first


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is the GPU's."""
    is_cuda = property(lambda self: True)


def on_cpu(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def on_gpu(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype, device="cuda:0")


def attention(make, *, B=2, T=5, Hq=4, Hk=2, Hv=4, dk=8, dv=6, **change):
    a = dict(q=make(B, T, Hq, dk), k=make(B, T, Hk, dk), v=make(B, T, Hv, dv), log_decay=None, scale=None, initial_state=None, cu_seqlens=None)
    return a | {n: c(make) if callable(c) else c for n, c in change.items()}


ATTENTION = {
    "no q": dict(q=None), "q a number": dict(q=3), "k none": dict(k=None), "v a list": dict(v=[1.0]),
    "rank of q": dict(q=lambda m: m(5, 4, 8)), "rank of v": dict(v=lambda m: m(2, 5, 4, 6, 1)),
    "64 bits": dict(q=lambda m: m(2, 5, 4, 8, dtype=F64), k=lambda m: m(2, 5, 2, 8, dtype=F64), v=lambda m: m(2, 5, 4, 6, dtype=F64)),
    "whole numbers": dict(q=lambda m: m(2, 5, 4, 8, dtype=torch.int32)), "k's type": dict(k=lambda m: m(2, 5, 2, 8, dtype=BF16)),
    "v's type": dict(v=lambda m: m(2, 5, 4, 6, dtype=F16)), "batch": dict(k=lambda m: m(1, 5, 2, 8)), "tokens": dict(v=lambda m: m(2, 6, 4, 6)),
    "key dimension": dict(k=lambda m: m(2, 5, 2, 7)), "heads that do not divide": dict(Hk=3), "no heads": dict(Hk=0), "no values": dict(dv=0), "no keys": dict(dk=0),
    "keys too wide": dict(dk=257), "values too wide": dict(dv=257), "q not dense": dict(q=lambda m: m(2, 5, 8, 4).transpose(2, 3)),
    "decay's shape": dict(log_decay=lambda m: m(2, 5, 2)), "decay's tokens": dict(log_decay=lambda m: m(2, 1, 4)), "decay's heads": dict(log_decay=lambda m: m(3)),
    "decay's type": dict(log_decay=lambda m: m(2, 5, 4, dtype=BF16)), "decay a number": dict(log_decay=-0.1),
    "state's type": dict(initial_state=lambda m: m(2, 4, 8, 6, dtype=BF16)), "state's shape": dict(initial_state=lambda m: m(2, 4, 6, 8)),
    "state's sequences": dict(initial_state=lambda m: m(1, 4, 8, 6)),
    "places in a batch of two": dict(cu_seqlens=lambda m: m(3, dtype=torch.int32)), "places of 64 bits": dict(B=1, cu_seqlens=lambda m: m(3, dtype=torch.int64)),
    "one place": dict(B=1, cu_seqlens=lambda m: m(1, dtype=torch.int32)), "places' rank": dict(B=1, cu_seqlens=lambda m: m(1, 3, dtype=torch.int32)),
    "every other place": dict(B=1, cu_seqlens=lambda m: m(6, dtype=torch.int32)[::2]),
    "state of packed sequences": dict(B=1, cu_seqlens=lambda m: m(3, dtype=torch.int32), initial_state=lambda m: m(1, 4, 8, 6)),
}


def step(make, *, B=2, Hq=4, Hk=2, Hv=4, dk=8, dv=6, **change):
    a = dict(q=make(B, Hq, dk), k=make(B, Hk, dk), v=make(B, Hv, dv), log_decay=None, state=make(B, 4, dk, dv))
    return a | {n: c(make) if callable(c) else c for n, c in change.items()}


STEP = {
    "with tokens": dict(q=lambda m: m(2, 1, 4, 8)), "k's type": dict(k=lambda m: m(2, 2, 8, dtype=F16)), "batch": dict(v=lambda m: m(3, 4, 6)), "no state": dict(state=None),
    "state's type": dict(state=lambda m: m(2, 4, 8, 6, dtype=F16)), "state's shape": dict(state=lambda m: m(2, 4, 6, 8)), "states in one place": dict(state=lambda m: m(1, 4, 8, 6).expand(2, 4, 8, 6)),
    "states that overlap": dict(state=lambda m: m(400).as_strided((2, 4, 8, 6), (191, 48, 6, 1))), "a state turned": dict(state=lambda m: m(2, 4, 6, 8).transpose(2, 3)),
    "heads of one state": dict(state=lambda m: m(2, 1, 8, 6).expand(2, 4, 8, 6)), "decay's shape": dict(log_decay=lambda m: m(2, 1)), "decay's type": dict(log_decay=lambda m: m(2, 4, dtype=BF16)),
    "gradients": dict(k=lambda m: m(2, 2, 8).requires_grad_()), "a state with a gradient": dict(state=lambda m: m(2, 4, 8, 6).requires_grad_()), "heads": dict(Hq=3), "too wide": dict(dk=300),
}


def norm(make, *, B=2, T=5, Hq=4, Hk=2, D=8, **change):
    a = dict(q=make(B, T, Hq, D), k=make(B, T, Hk, D), q_weight=None, k_weight=None, positions=None, frequencies=None)
    return a | {n: c(make) if callable(c) else c for n, c in change.items()}


INT = torch.int64
NORM = {
    "no k": dict(k=None), "k's type": dict(k=lambda m: m(2, 5, 2, 8, dtype=BF16)), "64 bits": dict(q=lambda m: m(2, 5, 4, 8, dtype=F64)), "rank": dict(q=lambda m: m(2, 5, 8)),
    "tokens": dict(k=lambda m: m(2, 4, 2, 8)), "dimension": dict(k=lambda m: m(2, 5, 2, 6)), "too wide": dict(D=513), "nothing": dict(D=0), "not dense": dict(k=lambda m: m(2, 5, 8, 2).transpose(2, 3)),
    "weight's shape": dict(q_weight=lambda m: m(7)), "weight's type": dict(k_weight=lambda m: m(8, dtype=BF16)), "weights of two types": dict(
        q=lambda m: m(2, 5, 4, 8, dtype=BF16), k=lambda m: m(2, 5, 2, 8, dtype=BF16), q_weight=lambda m: m(8), k_weight=lambda m: m(8, dtype=BF16)),
    "positions alone": dict(positions=lambda m: m(2, 5, dtype=INT)), "frequencies alone": dict(frequencies=lambda m: m(4)),
    "positions of floats": dict(positions=lambda m: m(2, 5), frequencies=lambda m: m(4)), "frequencies of halves": dict(positions=lambda m: m(2, 5, dtype=INT), frequencies=lambda m: m(4, dtype=F16)),
    "positions' shape": dict(positions=lambda m: m(2, 4, dtype=INT), frequencies=lambda m: m(4)), "positions' batch": dict(positions=lambda m: m(1, 5, dtype=INT), frequencies=lambda m: m(4)),
    "axes": dict(positions=lambda m: m(2, 5, 3, dtype=INT), frequencies=lambda m: m(2, 2)), "axes without frequencies": dict(positions=lambda m: m(2, 5, 1, dtype=INT), frequencies=lambda m: m(4)),
    "too many pairs": dict(positions=lambda m: m(5, dtype=INT), frequencies=lambda m: m(5)), "frequencies' rank": dict(positions=lambda m: m(5, dtype=INT), frequencies=lambda m: m(1, 1, 4)),
}
CALLS = [(vmamba_amd.linear_attention_fn, attention, ATTENTION), (vmamba_amd.linear_attention_step_fn, step, STEP), (vmamba_amd.qk_norm_rotate_fn, norm, NORM)]
CASES = [pytest.param(call, build, change, id=f"{build.__name__}: {name}") for call, build, changes in CALLS for name, change in changes.items()]


@pytest.mark.parametrize("call,build,change", CASES)
def test_refused_before_anything_runs(call, build, change, monkeypatch):
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    alike = lambda like, /, **tensors: [linear_attention._check(t is None or isinstance(t, torch.Tensor), f"{n} must be a tensor") for n, t in tensors.items()]  # noqa: E731
    monkeypatch.setattr(linear_attention, "check_plain", alike)
    monkeypatch.setattr(qk_norm, "check_plain", alike)
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
@pytest.mark.parametrize("call,build,changes", CALLS, ids=["attention", "step", "norm"])
def test_tensors_elsewhere_are_refused(call, build, changes):
    """Each tensor in turn on the CPU, of a class of its own, or without memory."""
    full = build(on_gpu)
    full |= dict(log_decay=on_gpu(4)) if "log_decay" in full else dict(q_weight=on_gpu(8), k_weight=on_gpu(8), positions=on_gpu(5, dtype=INT), frequencies=on_gpu(4))
    full |= dict(initial_state=on_gpu(2, 4, 8, 6)) if "initial_state" in full else {}
    with torch.no_grad():
        call(**full)
        for name, t in full.items():
            if not isinstance(t, torch.Tensor):
                continue
            for other in (t.cpu(), t.as_subclass(OnGpu), torch.empty(t.shape, dtype=t.dtype, device="meta")):
                with pytest.raises(RuntimeError):
                    call(**full | {name: other})


@pytest.mark.parametrize("call,build,changes", CALLS, ids=["attention", "step", "norm"])
def test_no_cpu_path(call, build, changes):
    with pytest.raises(RuntimeError, match="GPU tensor"):
        call(**build(torch.zeros))


# ---- the C entries -------------------------------------------------------------------------------------------------------------------
def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_lib.LinearAttentionParams) == 12 * 4 + 8 * 8 + 12 * 8 and _lib.LinearAttentionParams.q.offset == 48
    assert ctypes.sizeof(_lib.LinearAttentionBwdParams) == 208 + 7 * 8 + 3 * 8 + 8 and _lib.LinearAttentionBwdParams.decay_per_head.offset == 288
    assert ctypes.sizeof(_lib.LinearAttentionStepParams) == 10 * 4 + 6 * 8 + 9 * 8 and _lib.LinearAttentionStepParams.state_batch_stride.offset == 152
    assert ctypes.sizeof(_lib.QkNormRotateParams) == 14 * 4 + 8 * 8 + 9 * 8 and _lib.QkNormRotateParams.q_batch_stride.offset == 120
    assert ctypes.sizeof(_lib.QkNormRotateBwdParams) == 192 + 6 * 8 + 6 * 8


def fill(p, **values):
    for name, value in values.items():
        setattr(p, name, value)
    return p


def sequences(**change):
    p = fill(_lib.LinearAttentionParams(), batch=2, seqlen=100, heads=4, q_heads=4, k_heads=2, v_heads=4, key_dim=64, value_dim=64, dtype=_lib.SS2D_BF16, decay_dtype=_lib.SS2D_F32, scale=1.0,
             q=256, k=256, v=256, out=256, q_token_stride=256, k_token_stride=128, v_token_stride=256)
    return fill(p, **change)


INVALID = [dict(batch=-1), dict(seqlen=-1), dict(heads=-4), dict(key_dim=0), dict(value_dim=0), dict(dtype=7), dict(dtype=-1), dict(q_heads=0), dict(k_heads=3), dict(v_heads=-2),
           dict(decay=256, decay_dtype=_lib.SS2D_F16), dict(cu_seqlens=256, n_seqs=3), dict(batch=1, cu_seqlens=256, n_seqs=0), dict(n_seqs=-1), dict(q=None), dict(k=None), dict(v=None)]


@pytest.mark.parametrize("change", INVALID, ids=str)
def test_sequences_of_bad_arguments(change):
    L, p = _lib.lib(), sequences(**change)
    g = fill(_lib.LinearAttentionBwdParams(), fwd=p, dout=256, dq=256, dk=256, dv=256)
    assert L.ss2d_linear_attention_workspace_bytes(p) == _lib.SS2D_EINVAL and L.ss2d_linear_attention_fwd(p, HERE, 1 << 40, None) == _lib.SS2D_EINVAL
    assert L.ss2d_linear_attention_bwd_workspace_bytes(g) == _lib.SS2D_EINVAL and L.ss2d_linear_attention_bwd(g, HERE, 1 << 40, None) == _lib.SS2D_EINVAL


def test_sequences_of_too_much():
    L = _lib.lib()
    for change in (dict(key_dim=257), dict(value_dim=300), dict(batch=2 ** 31 - 1, seqlen=1), dict(seqlen=2 ** 31 - 1, batch=64), dict(batch=1, cu_seqlens=256, n_seqs=2 ** 31 - 1),
                   dict(heads=2 ** 31 - 4, q_heads=1, k_heads=1, v_heads=1, seqlen=1)):
        p = sequences(**change)
        g = fill(_lib.LinearAttentionBwdParams(), fwd=p, dout=256, dq=256, dk=256, dv=256)
        assert L.ss2d_linear_attention_workspace_bytes(p) == _lib.SS2D_ENOTSUP and L.ss2d_linear_attention_fwd(p, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change
        assert L.ss2d_linear_attention_bwd_workspace_bytes(g) == _lib.SS2D_ENOTSUP and L.ss2d_linear_attention_bwd(g, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, change


def test_sequences_workspace_and_results():
    L = _lib.lib()
    assert L.ss2d_linear_attention_workspace_bytes(None) == _lib.SS2D_EINVAL and L.ss2d_linear_attention_bwd(None, HERE, 1, None) == _lib.SS2D_EINVAL
    p = sequences()
    g = fill(_lib.LinearAttentionBwdParams(), fwd=p, dout=256, dq=256, dk=256, dv=256)
    need, need_bwd = L.ss2d_linear_attention_workspace_bytes(p), L.ss2d_linear_attention_bwd_workspace_bytes(g)
    # tables: 2 x 2 chunks of 4 heads; the backward has 2 states of 64 x 64 in bf16 for each at least
    assert need >= 4 * 4 * 64 * 8 and need_bwd >= 2 * 16 * 64 * 64 * 2
    for call, params, bytes_ in ((L.ss2d_linear_attention_fwd, p, need), (L.ss2d_linear_attention_bwd, g, need_bwd)):
        assert call(params, None, bytes_, None) == _lib.SS2D_EINVAL
        assert call(params, ctypes.c_void_p(264), bytes_, None) == _lib.SS2D_EINVAL
        assert call(params, HERE, bytes_ - 1, None) == _lib.SS2D_ENOMEM
    assert L.ss2d_linear_attention_fwd(sequences(out=None), HERE, need, None) == _lib.SS2D_EINVAL
    for missing in ("dout", "dq", "dk", "dv"):
        assert L.ss2d_linear_attention_bwd(fill(_lib.LinearAttentionBwdParams(), **(dict(fwd=p, dout=256, dq=256, dk=256, dv=256) | {missing: None})), HERE, need_bwd, None) == _lib.SS2D_EINVAL
    assert L.ss2d_linear_attention_bwd(fill(_lib.LinearAttentionBwdParams(), fwd=p, dout=256, dq=256, dk=256, dv=256, ddecay=256), HERE, need_bwd, None) == _lib.SS2D_EINVAL
    low = fill(_lib.LinearAttentionBwdParams(), fwd=sequences(decay=256), dout=256, dq=256, dk=256, dv=256, ddecay=256)
    assert L.ss2d_linear_attention_bwd_workspace_bytes(low) >= need_bwd + 2 * 16 * 64 * 64 * 2       # (and what the states' rounding left)
    for empty in (dict(batch=0), dict(heads=0)):
        p = sequences(**empty, q=None, k=None, v=None)
        assert L.ss2d_linear_attention_workspace_bytes(p) == 0 and L.ss2d_linear_attention_fwd(p, None, 0, None) == _lib.SS2D_OK
        assert L.ss2d_linear_attention_bwd(fill(_lib.LinearAttentionBwdParams(), fwd=p), None, 0, None) == _lib.SS2D_OK


def test_step_of_bad_arguments():
    L = _lib.lib()
    make = lambda **change: fill(_lib.LinearAttentionStepParams(), **(dict(  # noqa: E731
        batch=2, heads=4, q_heads=4, k_heads=2, v_heads=4, key_dim=64, value_dim=32, dtype=_lib.SS2D_F16, decay_dtype=_lib.SS2D_F32, scale=1.0, q=256, k=256, v=256, state=256, out=256,
        state_batch_stride=4 * 64 * 32) | change))
    assert L.ss2d_linear_attention_step(None, None) == _lib.SS2D_EINVAL
    for change in (dict(batch=-1), dict(heads=-1), dict(key_dim=0), dict(value_dim=0), dict(k_heads=3), dict(q_heads=0), dict(dtype=9), dict(decay=256, decay_dtype=_lib.SS2D_BF16), dict(q=None),
                   dict(k=None), dict(v=None), dict(state=None), dict(out=None), dict(state_batch_stride=4 * 64 * 32 - 1), dict(state_batch_stride=0)):
        assert L.ss2d_linear_attention_step(make(**change), None) == _lib.SS2D_EINVAL, change
    for change in (dict(key_dim=257), dict(value_dim=1000), dict(batch=2 ** 31 - 1)):
        assert L.ss2d_linear_attention_step(make(**change), None) == _lib.SS2D_ENOTSUP, change
    assert L.ss2d_linear_attention_step(make(batch=0, q=None), None) == _lib.SS2D_OK


def test_norm_of_bad_arguments():
    L = _lib.lib()
    full = dict(batch=2, seqlen=10, q_heads=4, k_heads=2, dim=64, dtype=_lib.SS2D_BF16, weight_dtype=_lib.SS2D_F32, eps=1e-6, q=256, k=256, q_out=256, k_out=256)
    make = lambda **change: fill(_lib.QkNormRotateParams(), **(full | change))  # noqa: E731
    turned = dict(positions=256, frequencies=256, axes=2, per_axis=16)
    assert L.ss2d_qk_norm_rotate(None, None) == _lib.SS2D_EINVAL
    for change in (dict(batch=-1), dict(seqlen=-1), dict(q_heads=-1), dict(k_heads=-1), dict(dim=0), dict(dtype=5), dict(q_weight=256, weight_dtype=_lib.SS2D_F16), dict(q=None), dict(k=None),
                   dict(q_out=None), dict(k_out=None), turned | dict(frequencies=None), turned | dict(axes=0), turned | dict(per_axis=17), turned | dict(axes=2 ** 30, per_axis=4),
                   dict(k_heads=2 ** 30)):
        assert L.ss2d_qk_norm_rotate(make(**change), None) == _lib.SS2D_EINVAL, change
    assert L.ss2d_qk_norm_rotate(make(dim=513), None) == _lib.SS2D_ENOTSUP
    for empty in (dict(batch=0), dict(seqlen=0), dict(q_heads=0, k_heads=0)):
        assert L.ss2d_qk_norm_rotate(make(**empty, q=None, k=None, q_out=None, k_out=None), None) == _lib.SS2D_OK
    need = L.ss2d_qk_norm_rotate_bwd_workspace_bytes(64)
    assert need > 0 and L.ss2d_qk_norm_rotate_bwd_workspace_bytes(0) == _lib.SS2D_EINVAL and L.ss2d_qk_norm_rotate_bwd_workspace_bytes(513) == _lib.SS2D_EINVAL
    grads = dict(dq_out=256, dk_out=256, dq=256, dk=256)
    back = lambda fwd, **change: fill(_lib.QkNormRotateBwdParams(), **(grads | dict(fwd=fwd) | change))  # noqa: E731
    assert L.ss2d_qk_norm_rotate_bwd(None, HERE, need, None) == _lib.SS2D_EINVAL
    for missing in grads:
        assert L.ss2d_qk_norm_rotate_bwd(back(make(), **{missing: None}), HERE, need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_qk_norm_rotate_bwd(back(make(), dq_weight=256), HERE, need, None) == _lib.SS2D_EINVAL          # of a weight that is not there
    weighed = make(q_weight=256)
    assert L.ss2d_qk_norm_rotate_bwd(back(weighed, dq_weight=256), None, need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_qk_norm_rotate_bwd(back(weighed, dq_weight=256), ctypes.c_void_p(260), need, None) == _lib.SS2D_EINVAL
    assert L.ss2d_qk_norm_rotate_bwd(back(weighed, dq_weight=256), HERE, need - 1, None) == _lib.SS2D_ENOMEM


# ---- traced calls ----------------------------------------------------------------------------------------------------------------------
def behind_the_tracer(*like):
    """Results as kernels make them, in memory that no operator of torch's writes: twice the inputs."""
    made = [torch.empty(tuple(map(int, t.shape)), dtype=t.dtype) for t in like]
    for out, t in zip(made, like):
        out.numpy()[...] = 2 * t.detach().numpy()
    return made


@pytest.mark.filterwarnings("ignore")
def test_a_traced_call_is_run_again(monkeypatch):
    """A traced module calls the operator with its own inputs, of other sizes too, instead of giving the example's results back; with tensors that do not
    fit it refuses as the call itself does."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(qk_norm, "check_plain", lambda *a, **b: None)

    class Native:
        @staticmethod
        def linear_attention(kinds, q, k, v, *rest):
            return behind_the_tracer(v)[0]

        @staticmethod
        def qk_norm_rotate(kinds, q, k, *rest):
            return tuple(behind_the_tracer(q, k))

    monkeypatch.setattr(_lib, "host", lambda: Native)
    monkeypatch.setattr(linear_attention, "linear_attention_fwd", lambda q, k, v, *rest: (behind_the_tracer(v)[0], None))
    monkeypatch.setattr(qk_norm, "qk_norm_rotate_fwd", lambda q, k, *rest: tuple(behind_the_tracer(q, k)), raising=False)
    make = lambda B, T: [torch.randn(B, T, 2, 8) for _ in range(3)]  # noqa: E731
    with torch.no_grad():
        attend = torch.jit.trace(lambda q, k, v: vmamba_amd.linear_attention_fn(q, k, v) + 1, make(2, 5))
        rotate = torch.jit.trace(lambda q, k: sum(vmamba_amd.qk_norm_rotate_fn(q, k)), make(2, 5)[:2])
        for sizes in ((2, 5), (1, 7)):
            q, k, v = make(*sizes)
            assert torch.equal(attend(q, k, v), 2 * v + 1) and torch.equal(rotate(q, k), 2 * q + 2 * k)
        with pytest.raises(RuntimeError, match="agree"):
            attend(q, k[:, :5], v)
        with pytest.raises(RuntimeError, match="agree"):
            rotate(q, k[:, :5])


def test_a_traced_step_is_refused(monkeypatch):
    monkeypatch.setattr(torch.jit, "is_tracing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        vmamba_amd.linear_attention_step_fn(**step(on_cpu))


def test_a_learnt_decay_of_no_sequences_is_not_left_out():
    """A gradient that is asked for without the decays it is of is refused here too."""
    p = fill(_lib.LinearAttentionBwdParams(), fwd=sequences(batch=0, q=None, k=None, v=None), ddecay=256, decay_per_head=1)
    assert _lib.lib().ss2d_linear_attention_bwd(p, None, 0, None) == _lib.SS2D_EINVAL


class Kept:
    """What a backward is given besides the gradients."""
    scale, eps, interleaved, needs_input_grad = 1.0, 1e-6, False, (True,) * 8

    def __init__(self, *saved):
        self.saved_tensors = saved


def test_gradients_of_another_type_are_refused(monkeypatch):
    """Saved tensors that a hook brought back in single precision: the gradients, which are still bf16, are not read as that."""
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(qk_norm, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(linear_attention, "linear_attention_bwd", lambda *a: pytest.fail("called"))
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    q, k, v = on_cpu(2, 5, 4, 8), on_cpu(2, 5, 2, 8), on_cpu(2, 5, 4, 6)
    with torch.no_grad():
        for dout, dfinal in ((on_cpu(2, 5, 4, 6, dtype=BF16), None), (None, on_cpu(2, 4, 8, 6, dtype=BF16)), (on_cpu(2, 5, 4, 6), on_cpu(2, 4, 8, 6, dtype=BF16))):
            with pytest.raises(RuntimeError):
                linear_attention.LinearAttentionHip.backward(Kept(q, k, v, None, None, None), dout, dfinal)
        for dq, dk in ((BF16, F32), (F32, BF16), (BF16, BF16)):
            with pytest.raises(RuntimeError):
                qk_norm.QkNormRotateHip.backward(Kept(q, k, None, None, None, None), on_cpu(*q.shape, dtype=dq), on_cpu(*k.shape, dtype=dk))


MANY = 2 ** 32 + 64                  # 64, counted in 32 bits


def stretched(*shape, dtype=F32):
    """A tensor of this shape in the memory of one value a row, whatever the number of rows."""
    return on_cpu(*(1 if n > 2 ** 20 else n for n in shape), dtype=dtype).expand(*shape)


@pytest.mark.parametrize("build,sizes", [(attention, dict(T=MANY)), (attention, dict(B=MANY)), (attention, dict(Hv=MANY)), (attention, dict(Hq=MANY, Hk=MANY, Hv=MANY)),
                                         (attention, dict(B=1, cu_seqlens=lambda m: torch.empty(MANY, dtype=torch.int32, device="meta"))),
                                         (norm, dict(T=MANY)), (norm, dict(B=MANY)), (norm, dict(Hk=MANY))],
                         ids=["tokens", "batch", "heads of v", "heads", "sequences", "norm tokens", "norm batch", "norm heads"])
def test_sizes_over_32_bits_are_refused(build, sizes, monkeypatch):
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(qk_norm, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(linear_attention, "linear_attention_fwd", lambda *a: pytest.fail("called"))
    monkeypatch.setattr(qk_norm, "qk_norm_rotate_fwd", lambda *a: pytest.fail("called"))
    with pytest.raises(RuntimeError, match="no dimension of more|no more than"):
        {attention: vmamba_amd.linear_attention_fn, norm: vmamba_amd.qk_norm_rotate_fn}[build](**build(stretched, **sizes))


def test_a_step_of_more_sequences_than_32_bits_is_refused(monkeypatch):
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    with pytest.raises(RuntimeError, match="no dimension of more"):
        vmamba_amd.linear_attention_step_fn(**step(stretched, B=MANY))


@pytest.mark.parametrize("dtype,chunk", [(_lib.SS2D_BF16, 64), (_lib.SS2D_F16, 32), (_lib.SS2D_F32, 32)], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("sequences_", [0, 1, 100_000])
def test_tokens_at_the_end_of_32_bits(sequences_, dtype, chunk):
    """Places of tokens, rounded up to chunks and with a chunk for each packed sequence behind them, stay 32-bit numbers, or the call is refused."""
    L = _lib.lib()
    one = dict(batch=1, heads=1, q_heads=1, k_heads=1, v_heads=1, key_dim=8, value_dim=8, dtype=dtype) | (dict(cu_seqlens=256, n_seqs=sequences_) if sequences_ else {})
    most = 2 ** 31 - 1 - (sequences_ + 3) * chunk
    assert L.ss2d_linear_attention_workspace_bytes(sequences(seqlen=most, **one)) > 8 * most
    for tokens in (most + 1, 2 ** 31 - chunk, 2 ** 31 - 2, 2 ** 31 - 1):
        p = sequences(seqlen=tokens, **one)
        assert L.ss2d_linear_attention_workspace_bytes(p) == _lib.SS2D_ENOTSUP and L.ss2d_linear_attention_fwd(p, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP, tokens


def test_norm_of_tokens_at_the_end_of_32_bits():
    """A round of 16 tokens that begins in front of a batch's last one counts past it before it goes on in the next batch."""
    L = _lib.lib()
    for tokens in (2 ** 31 - 16, 2 ** 31 - 1):
        p = fill(_lib.QkNormRotateParams(), batch=2, seqlen=tokens, q_heads=1, k_heads=1, dim=8, dtype=_lib.SS2D_BF16, eps=1e-6)
        assert L.ss2d_qk_norm_rotate(p, None) == _lib.SS2D_ENOTSUP
        assert L.ss2d_qk_norm_rotate_bwd(fill(_lib.QkNormRotateBwdParams(), fwd=p), HERE, 1 << 40, None) == _lib.SS2D_ENOTSUP
    p.seqlen = 2 ** 31 - 17
    assert L.ss2d_qk_norm_rotate(p, None) == _lib.SS2D_EINVAL        # (no queries: refused for that)


def test_captures_are_looked_at_through_python(monkeypatch):
    """A call with gradients asks whether it may be captured before anything is launched, with its own leaves and not with copies of them; one without does not."""
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(qk_norm, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(linear_attention, "linear_attention_fwd", lambda *a: pytest.fail("called"))
    monkeypatch.setattr(qk_norm, "qk_norm_rotate_fwd", lambda *a: pytest.fail("called"))
    asked = []

    class Native:
        @staticmethod
        def refuse_capture(tensors, what):
            asked.append((tensors, what))
            raise RuntimeError("still lives")

    monkeypatch.setattr(_lib, "host", lambda: Native)
    leaf = on_cpu(2, 4, 6, 8).transpose(2, 3).requires_grad_()       # (not dense: this one is what brings the call through Python)
    weight = on_cpu(16)[::2].requires_grad_()
    with pytest.raises(RuntimeError, match="still lives"):
        vmamba_amd.linear_attention_fn(**attention(on_cpu, initial_state=leaf))
    with pytest.raises(RuntimeError, match="still lives"):
        vmamba_amd.qk_norm_rotate_fn(**norm(on_cpu, q_weight=weight))
    assert [what for _, what in asked] == ["linear_attention_fn", "qk_norm_rotate_fn"] and asked[0][0][4] is leaf and asked[1][0][2] is weight
    monkeypatch.setattr(linear_attention, "linear_attention_fwd", lambda q, k, v, *a: (torch.zeros_like(v), None))
    with torch.no_grad():
        vmamba_amd.linear_attention_fn(**attention(on_cpu, initial_state=leaf))
    assert len(asked) == 2


def test_forward_derivatives_are_refused(monkeypatch):
    """A token's step has no derivative of either kind: a tangent that comes in is not dropped."""
    from torch.autograd import forward_ad
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    monkeypatch.setattr(linear_attention, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(qk_norm, "check_plain", lambda *a, **b: None)
    monkeypatch.setattr(linear_attention, "linear_attention_fwd", lambda q, k, v, *a: (torch.zeros_like(v), None))
    monkeypatch.setattr(qk_norm, "qk_norm_rotate_fwd", lambda q, k, *a: (torch.zeros_like(q), torch.zeros_like(k)))
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))
    with forward_ad.dual_level():
        for call, build, _ in CALLS:
            args = build(torch.zeros)
            for name in ("q", "k", "v", "state"):
                if name in args:
                    with pytest.raises(RuntimeError):
                        call(**args | {name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))})


@pytest.mark.parametrize("dtype,decay,parts", [(_lib.SS2D_BF16, None, 2), (_lib.SS2D_BF16, 256, 6), (_lib.SS2D_F32, 256, 3)], ids=["bf16", "bf16, decays' gradients", "fp32"])
def test_a_backward_asks_for_the_states_that_it_keeps(dtype, decay, parts):
    """Both states of each chunk, in bf16 with what their rounding left where decays' gradients are in single precision; what is behind a chunk in both
    orders only where it is read so.  Besides them the tables: a few values a token and head."""
    L, T, H, D = _lib.lib(), 6400, 16, 128
    p = sequences(batch=1, seqlen=T, heads=H, q_heads=H, k_heads=H, v_heads=H, key_dim=D, value_dim=D, dtype=dtype, decay=decay)
    g = fill(_lib.LinearAttentionBwdParams(), fwd=p, dout=256, dq=256, dk=256, dv=256, ddecay=decay)
    chunk, size = (64, 2) if dtype == _lib.SS2D_BF16 else (32, 4)
    states = parts * (T // chunk) * H * D * D * size
    segments = 2 * 4 * (D * D + 1) * H * (512 // (H * 2 * 4) + 1)    # their own sums: two workgroups to a CU, of both walks
    tables = T * H * 8 + (T // chunk) * (H * 8 + 16)
    assert states <= L.ss2d_linear_attention_bwd_workspace_bytes(g) <= states + segments + tables + 16 * 256
