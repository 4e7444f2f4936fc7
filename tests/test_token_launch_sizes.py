"""Sizes that the C entries of the token operators refuse because a launch of theirs, or an index inside it, could not count them: said before anything is launched, so that the tests run
on the CPU, where a launch would be another status."""
import ctypes

import pytest

from vmamba_amd import _lib

HERE = ctypes.c_void_p(256)          # an aligned address, never read


def fill(p, **values):
    for name, value in values.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("dim", [2 ** 31 - 1, 2 ** 31 - 255])
@pytest.mark.parametrize("dtype", [_lib.SS2D_F32, _lib.SS2D_BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dstate", [1, 16])
def test_a_step_of_more_channels_than_a_workgroup_rounds_up_to(dim, dtype, dstate):
    """A workgroup takes up to 256 channels: within as many of 2^31 its last channel's index does not fit 32 bits."""
    p = fill(_lib.TokenScanStepParams(), batch=1, dim=dim, dstate=dstate, n_groups=1, dtype=dtype, u=256, delta=256, A=256, B=256, C=256, state=256, out=256)
    assert _lib.lib().ss2d_token_scan_step(p, None) == _lib.SS2D_ENOTSUP


@pytest.mark.parametrize("sizes", [dict(batch=4, seqlen=16384, n_groups=4096, dim=4096, dstate=16), dict(batch=1, seqlen=2 ** 26, n_groups=1, dim=1, dstate=64), dict(batch=1, seqlen=1, n_groups=1, dim=1500000000, dstate=1)],
                         ids=["2^32 values of B", "one channel", "values of A, D and the bias"])
def test_gradients_whose_sums_are_more_than_a_launch_counts(sizes):
    """The forward is taken; with states kept for gradients it says at once that there are none."""
    L = _lib.lib()
    p = fill(_lib.TokenScanParams(), **sizes, dtype=_lib.SS2D_BF16, delta_softplus=1, u=256, delta=256, A=256, B=256, C=256, out=256)
    g = fill(_lib.TokenScanBwdParams(), fwd=fill(p, kept_states=256), dout=256, du=256, ddelta=256, dB=256, dC=256)
    assert L.ss2d_token_scan_workspace_bytes(p) >= 0
    assert L.ss2d_token_scan_kept_states(p) == L.ss2d_token_scan_bwd_workspace_bytes(g) == L.ss2d_token_scan_bwd(g, HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP


def test_a_convolutions_gradients_of_more_channels_than_their_sums_launch_counts():
    L = _lib.lib()
    make = lambda dim: fill(_lib.CausalConvBwdParams(), fwd=fill(_lib.CausalConvParams(), batch=1, seqlen=1, dim=dim, width=2, dtype=_lib.SS2D_BF16, weight_dtype=_lib.SS2D_BF16, x=256,  # noqa: E731
                                                                weight=256, out=256), dout=256, dx=256)
    for dim in (2 ** 30, 2 ** 30 - 63):
        assert L.ss2d_causal_conv_bwd_workspace_bytes(make(dim)) == L.ss2d_causal_conv_bwd(make(dim), HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP
    assert L.ss2d_causal_conv_bwd_workspace_bytes(make(2 ** 30 - 64)) == 3 * (2 ** 30 - 64) * 4


@pytest.mark.parametrize("weights", [dict(dweight=256), dict(dbias=256), dict(dweight=256, dbias=256)], ids=lambda v: " and ".join(v))
def test_a_norms_gradients_of_more_channels_than_their_sums_launch_counts(weights):
    """Without its weights' gradients it is taken as before."""
    L = _lib.lib()
    make = lambda channels, **grads: fill(_lib.GroupNormBwdParams(), fwd=fill(_lib.GroupNormParams(), batch=1, positions=1, channels=channels, groups=channels // 64, dtype=_lib.SS2D_BF16,  # noqa: E731
                                                                              weight_dtype=_lib.SS2D_BF16, eps=1e-5, x=256, out=256, stats=256), dout=256, dx=256, **grads)
    most = 2 ** 28 - 64
    assert L.ss2d_group_norm_bwd_workspace_bytes(make(most + 64, **weights)) == L.ss2d_group_norm_bwd(make(most + 64, **weights), HERE, 1 << 62, None) == _lib.SS2D_ENOTSUP
    assert L.ss2d_group_norm_bwd_workspace_bytes(make(most, **weights)) == 8 * most and L.ss2d_group_norm_bwd_workspace_bytes(make(most + 64)) == 8 * (most + 64)
