"""group_norm_fn of values far from zero beside their spread: 4000 +- 1, where squares that are not of centred values lose everything in fp32.

u = 2^-24, M = |mean| / std.  K = 24 roundings in a row at most make a mean here (8 values of a lane or rows of a thread, then sums over 16 threads or lanes): its error, and those of the parts it is
joined of, is e = K u M standard deviations at most.  The variance, of values centred by such means, is off by 4 e relatively at most (twice where a part's squares are about its own mean, twice where
parts' means are joined) and 8 u.  So a normalised value n is off by dn = e + |n| (2 e + 8 u), a gradient dx = rstd (d - mean(d) - n mean(d n)) by
    |dx| (2 e + 8 u) + rstd (K u mean|d| + |n| (mean(|d| dn) + K u mean|d n|) + dn |mean(d n)| + 4 u (|d| + |mean d| + |n mean(d n)|)),
the weight's, sum d n, by sum(|d| dn) and as many roundings as it has terms.  The test asserts that squares of uncentred values, and a gradient of zeros, would break these bounds."""
import pytest
import torch

from vmamba_amd import group_norm_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U, K, EPS = 2.0 ** -24, 24, 1e-5


@pytest.mark.parametrize("offset", [4000.0, -4000.0])
@pytest.mark.parametrize("shape,G", [((4, 64), 2), ((3, 2048), 16), ((2, 7, 96), 3), ((2, 3000, 64), 4), ((3, 56, 56, 48), 8), ((3, 500, 1030), 2)], ids=str)
def test_far_from_zero(shape, G, offset):
    gen = torch.Generator().manual_seed(7)
    C = shape[-1]
    x = (offset + torch.randn(*shape, generator=gen)).to(DEV)
    dout = torch.randn(*shape, generator=gen).to(DEV) + (x - offset)             # (so that the weight's gradient is not a sum of terms that cancel)
    leaves = [t.requires_grad_() for t in (x, torch.ones(C, device=DEV), torch.zeros(C, device=DEV))]
    out = group_norm_fn(leaves[0], G, leaves[1], leaves[2], EPS)
    dx, dweight, dbias = torch.autograd.grad(out, leaves, dout)

    v, d = x.detach().double().view(shape[0], -1, G, C // G), dout.double().view(shape[0], -1, G, C // G)
    over = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mean = over(v)
    rstd = (over((v - mean).square()) + EPS).rsqrt()
    n = (v - mean) * rstd
    e = K * U * mean.abs() * rstd
    dn = e + n.abs() * (2 * e + 8 * U)
    m1, m2 = over(d), over(d * n)
    want = rstd * (d - m1 - n * m2)
    off = want.abs() * (2 * e + 8 * U) + rstd * (K * U * over(d.abs()) + n.abs() * (over(d.abs() * dn) + K * U * over((d * n).abs())) + dn * m2.abs() + 4 * U * (d.abs() + m1.abs() + (n * m2).abs()))
    rows = v.shape[0] * v.shape[1]
    per_channel = lambda t: t.sum((0, 1)).flatten()  # noqa: E731
    for name, got, is_, bound in (("out", out, n, dn + 2 * U * n.abs()), ("dx", dx, want, off), ("dweight", dweight, per_channel(d * n), per_channel(d.abs() * dn) + rows * U * per_channel((d * n).abs())),
                                  ("dbias", dbias, per_channel(d), rows * U * per_channel(d.abs()))):
        wrong = (got.detach().double().view(is_.shape) - is_).abs()
        assert bool((wrong <= bound).all()), (name, (wrong / bound).max().item())
        assert bool((is_.abs() > 10 * bound).double().mean() > 0.5), (name, "zeros would pass")
    # the formula that is not to be used
    f = x.detach().view(v.shape)
    naive = (f - f.mean((1, 3), keepdim=True)) * (f.square().mean((1, 3), keepdim=True) - f.mean((1, 3), keepdim=True).square() + EPS).clamp(min=EPS).rsqrt()
    assert bool(((naive.double() - n).abs() > dn + 2 * U * n.abs()).any()), "squares of uncentred values would pass"
