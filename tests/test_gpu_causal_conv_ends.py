"""The causal convolution's gradients at the ends of sequences: tokens that are not there have no part in them, whatever the weights are."""
import pytest
import torch

from vmamba_amd import causal_conv_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,dim", [(2, 5), (37, 16), (130, 40), (5000, 2048)], ids=str)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("packed", [False, True])
def test_an_infinite_tap_reaches_its_own_tokens_only(packed, W, T, dim, dtype):
    """Tap j takes part in dx of a token whose W - 1 - j next ones are there.  x and dout are of 1s, so that no infinity meets another or a 0."""
    for j in range(W):
        weight = torch.ones(dim, W, dtype=dtype, device=DEV)
        weight[:, j] = float("inf")
        x, state = torch.ones(1, T, dim, dtype=dtype, device=DEV, requires_grad=True), torch.ones(2 if packed else 1, W - 1, dim, dtype=dtype, device=DEV, requires_grad=True)
        lengths = [T - T // 3, T // 3] if packed else [T]
        starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        cu = torch.tensor(starts, dtype=torch.int32, device=DEV) if packed else None
        dout = torch.ones_like(x)
        dx, dstate = torch.autograd.grad(causal_conv_fn(x, weight, None, None, initial_state=state, cu_seqlens=cu), [x, state], dout)
        for n, length in enumerate(lengths):
            line = torch.cat([dstate[n], dx[0, starts[n]:starts[n + 1]]]).float()                      # of the state's rows and the tokens: row r is token r - (W - 1)
            at = torch.arange(length + W - 1, device=DEV)
            first, last = at - (W - 1), at                                                             # tokens whose window has the row, tap W - 1 first
            mine = (first + W - 1 - j >= 0) & (first + W - 1 - j < length)
            count = (last.clamp(max=length - 1) - first.clamp(min=0) + 1).float()
            want = torch.where(mine, torch.full_like(count, float("inf")), count)
            assert torch.equal(line, want[:, None].expand_as(line)), (W, j, n)
