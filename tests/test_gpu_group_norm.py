"""group_norm_fn against the formula in 64 bits.

Sums are fp32, over at most K = 300 + positions / 64 roundings in a row (a lane's values, then trees).  With u = 2^-24: the mean is off by K u mean|x|, so a centred value by
K u (|x| + mean|x|); the variance, relatively, by K u (1 + S), S = (rms x + |mean|) / std; a normalised value n therefore by K u N, N = (|x| + mean|x|) / std + |n| (1 + S).  What is
made of n carries N for |n| in its sum of magnitudes.  SiLU's slope is at most 1.1 and its derivative changes by at most half of what y is off by.  The weights' gradients add up
as many terms as there are samples and positions.  A result is rounded once, by half a step at most."""
import pytest
import torch

from vmamba_amd import group_norm_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def reference(x, G, weight, bias, eps, act, dout):
    B, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(B, -1, G, C // G)
    w = torch.ones(G, C // G, dtype=v.dtype, device=DEV) if weight is None else weight.double().view(G, -1)
    b = torch.zeros_like(w) if bias is None else bias.double().view(G, -1)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    rstd = (var + eps).rsqrt()
    n = (v - mean) * rstd
    S = (v.square().mean((1, 3), keepdim=True).sqrt() + mean.abs()) * rstd
    N = (v.abs() + v.abs().mean((1, 3), keepdim=True)) * rstd + n.abs() * (1 + S)
    y, y_size = n * w + b, N * w.abs() + b.abs()
    sig = torch.sigmoid(y)
    d = dout.double().view(v.shape) * (sig * (1 + y * (1 - sig)) if act else 1)
    d_size = dout.double().view(v.shape).abs() * ((1 + y_size) if act else 1)
    over = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    dw_, dws = d * w, d_size * w.abs()
    dx = rstd * (dw_ - over(dw_) - n * over(dw_ * n))
    dx_size = rstd * (1 + S) * (dws + over(dws) + N * over(dws * N))
    flat = lambda t: t.sum((0, 1)).flatten()  # noqa: E731
    return ({"out": (y * sig if act else y).view(x.shape), "dx": dx.view(x.shape), "dweight": flat(d * n), "dbias": flat(d)},
            {"out": (1.1 * y_size + 1e-3 if act else y_size).view(x.shape), "dx": dx_size.view(x.shape), "dweight": flat(d_size * N), "dbias": flat(d_size)})


def check(name, got, want, size, x):
    rows = x.numel() // x.shape[-1]
    terms = 300 + rows / x.shape[0] / 64 + (rows if name in ("dweight", "dbias") else 0)
    bound = terms * 2.0 ** -24 * size + HALF[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == F16 else 1e-38)     # (fp16's smallest step)
    off = (got.double() - want).abs()
    assert got.shape == want.shape, name
    assert bool((off <= bound).all()), (name, (off / bound).max().item())


def run_all(x, G, weight, bias, eps, act, dout):
    leaves = {n: t.detach().requires_grad_() for n, t in (("x", x), ("weight", weight), ("bias", bias)) if t is not None}
    out = group_norm_fn(leaves["x"], G, leaves.get("weight"), leaves.get("bias"), eps, act)
    grads = torch.autograd.grad(out, list(leaves.values()), dout)
    return {"out": out.detach(), **{"d" + n: d for n, d in zip(leaves, grads)}}


SHAPES = [  # shape, groups
    ((1, 8), 1), ((3, 20), 2), ((70, 2048), 16), ((5, 96), 32), ((9, 1000), 8), ((2, 6000), 3), ((3, 4099), 1), ((2, 9000), 1), ((300, 33), 3), ((4, 7, 64), 4), ((2, 5, 5, 48), 8),
    ((3, 49, 40), 8), ((2, 300, 96), 32), ((1, 5000, 24), 3), ((2, 56, 56, 192), 32), ((1, 700, 1030), 2), ((2, 33, 2050), 1), ((1, 4000, 3), 1), ((40, 17, 130), 13), ((2, 1, 20000), 2),
    ((3, 400, 515), 103), ((1, 64, 5), 5),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,G", SHAPES, ids=str)
def test_values_and_gradients(shape, G, dtype):
    print("CASE group_norm", shape, G, dtype, flush=True)
    gen = torch.Generator().manual_seed(len(shape) * 100 + G)
    C = shape[-1]
    offset = 0.5 * torch.randn(C, generator=gen)
    x = (1.5 * torch.randn(*shape, generator=gen) + offset).to(DEV, dtype)
    wide = F32 if G % 2 else dtype
    weight = None if C == 1000 else torch.randn(C, generator=gen).to(DEV, wide)
    bias = None if C in (1000, 96) else torch.randn(C, generator=gen).to(DEV, wide)
    dout = torch.randn(*shape, generator=gen).to(DEV, dtype)
    act = "silu" if (C + G) % 2 else None
    got = run_all(x, G, weight, bias, 1e-5, act, dout)
    want, size = reference(x, G, weight, bias, 1e-5, act, dout)
    for name in got:
        check(name, got[name], want[name], size[name], x)
    with torch.no_grad():
        assert torch.equal(group_norm_fn(x, G, weight, bias, 1e-5, act), got["out"])


@pytest.mark.parametrize("shape,G", [((4, 64), 2), ((2, 3000, 64), 4)], ids=str)
def test_far_from_zero(shape, G):
    """Values of 1000 +- 1, the first of each group far from all others: the variance is that of centred values."""
    gen = torch.Generator().manual_seed(7)
    x = 1000 + torch.randn(*shape, generator=gen)
    x.view(shape[0], -1, shape[-1])[:, 0, ::shape[-1] // G] = -4000.0
    x = x.to(DEV)
    dout = torch.randn(*shape, generator=gen).to(DEV)
    got = run_all(x, G, None, None, 1e-5, "silu", dout)
    want, size = reference(x, G, None, None, 1e-5, "silu", dout)
    for name in got:
        check(name, got[name], want[name], size[name], x)
    flat = torch.full(shape, 3.0, device=DEV)                        # no variance at all
    assert not group_norm_fn(flat, G).any()
