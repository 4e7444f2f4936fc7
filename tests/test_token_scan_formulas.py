"""The formulas that the GPU's tests of the selective scan of tokens compare with (one_sequence in test_gpu_token_scan.py), checked by themselves in 64 bits on the CPU: their gradients
against central differences of their own forward.  Over h = 2^-17 a difference is off by h^2 / 6 of the third derivative and 2^-53 / h of the loss: below 1e-8 of the size of either."""
import pytest
import torch

from test_gpu_token_scan import NAMES, one_sequence

F64 = torch.float64


def inputs(T, dim, N, G, seed, gate, extra, state):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    return {"u": normal(T, dim), "delta": normal(T, dim) - 1, "A": -torch.exp(0.7 * normal(dim, N)), "B": normal(T, G, N), "C": normal(T, G, N), "D": normal(dim) if extra else None,
            "z": normal(T, dim) if gate else None, "delta_bias": normal(dim) if extra else None, "state": normal(dim, N) if state else None}, normal(T, dim), normal(dim, N), normal


@pytest.mark.parametrize("T,dim,N,G,gate,extra,state,softplus", [(1, 3, 2, 1, True, True, True, True), (9, 6, 4, 2, True, False, True, True), (33, 8, 5, 4, False, True, False, True),
                                                                 (70, 4, 16, 1, True, True, True, True), (1, 3, 2, 1, True, True, True, False), (9, 6, 4, 2, False, False, True, False)])
def test_gradients_are_those_of_the_forward(T, dim, N, G, gate, extra, state, softplus):
    a, dout, dfinal, normal = inputs(T, dim, N, G, T + N, gate, extra, state)
    if not softplus:                                                 # (steps of both signs, decays of at most e: a few tokens, or they grow past everything else)
        a["delta"], a["delta_bias"] = 0.1 * a["delta"], None
    found = one_sequence(a, dout, dfinal, softplus, False)

    def loss(values):
        made = one_sequence(values, None, None, softplus, False)
        return ((made["out"] * dout).sum() + (made["final"] * dfinal).sum()).item()

    h = 2.0 ** -17
    for name in NAMES:
        if a[name] is None:
            continue
        along = normal(*a[name].shape) * (a[name].abs() if name == "A" else 1.0)
        difference = (loss(a | {name: a[name] + h * along}) - loss(a | {name: a[name] - h * along})) / (2 * h)
        want = (found["d" + name] * along).sum().item()
        size = (found["d" + name].abs() * along.abs()).sum().item() + abs(loss(a))
        assert abs(want) > 1e-4 * size, name                          # (a gradient of nothing would not do)
        assert abs(difference - want) <= 1e-7 * size, (name, difference, want)
