"""Tokens of no channels: the selective scan's B and C have gradients all the same."""
import contextlib

import pytest
import torch

from vmamba_amd import selective_scan_tokens_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Seen(torch.overrides.TorchFunctionMode):
    """A mode that follows operators: the calls then go through Python."""
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("mode", [contextlib.nullcontext, Seen])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("packed", [False, True])
def test_the_gradients_of_B_and_C_are_zeros(packed, dtype, mode):
    """... not what their memory held."""
    B, T, G, N = (1 if packed else 2), 300, 2, 16
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=DEV) if packed else None
    new = lambda *s, dtype=dtype: torch.zeros(*s, dtype=dtype, device=DEV).requires_grad_()  # noqa: E731
    leaves = dict(u=new(B, T, 0), delta=new(B, T, 0), A=new(0, N, dtype=torch.float32), B=new(B, T, G, N), C=new(B, T, G, N), D=new(0, dtype=torch.float32), z=new(B, T, 0),
                  delta_bias=new(0, dtype=torch.float32), initial_state=new(2, 0, N, dtype=torch.float32))
    with mode():
        out, final = selective_scan_tokens_fn(**leaves, output_final_state=True, cu_seqlens=cu)
        spoiled = [torch.full((B, T, G, N), float("nan"), dtype=dtype, device=DEV) for _ in range(16)]          # (what new tensors of that size are given next)
        del spoiled
        grads = torch.autograd.grad([out, final], list(leaves.values()), [torch.zeros_like(out), torch.zeros_like(final)])
    assert out.shape == (B, T, 0) and final.shape == (2, 0, N)
    for (name, t), g in zip(leaves.items(), grads):
        assert g.shape == t.shape and g.dtype == t.dtype and not bool(g.any()), name
