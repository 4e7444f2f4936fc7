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
