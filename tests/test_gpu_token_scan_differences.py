"""The selective scan's gradients against differences of the definition, and what segments hand on against bounds that one lost segment would break.

Differences: the definition in 64 bits (one_sequence in test_gpu_token_scan.py, its forward alone) moved by h = 2^-17 both ways is off by parts in 1e8 of its size; the gradients are fp32, each off
by at most its number of roundings of 2^-24 of its sum of magnitudes, as that file has them, so their sum along a direction by the sum of those bounds along it.  The derivatives are many times
that, which the test asserts: a gradient of zeros, of another sign or twice as large would be seen.

Long sequences: the bounds of that file add every rounding up, 20 for each token.  Roundings are of both signs, so that the root of the mean square of the errors grows with the root of their number:
40 that all values share (the rounded products A log2 e and steps, whose errors a term has at most once, since it weighs exp(-sum |x|)) and sqrt(20 T + 4 N + 200) of the others, in units of 2^-24 of
the magnitudes' root mean square.  What is lost of one of eight segments is an eighth of a value, or all of it; the bound is 2e-5."""
import pytest
import torch

from test_gpu_token_scan import DEV, F32, NAMES, inputs, one_sequence, reference, run_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,dim,N,G", [(70, 24, 16, 2), (45, 9, 5, 3), (33, 16, 40, 1)])
def test_gradients_against_differences_of_the_definition(T, dim, N, G):
    args, dout, dfinal, normal = inputs(1, T, dim, N, G, F32, 3)
    got = run_all(args, dout, dfinal)
    pieces = [(0, 0, T)]
    formula, size = reference(args, pieces, dout, dfinal)

    def loss(name, step):
        a = {k: t.double() for k, t in args.items()}
        a[name] = a[name] + step
        a |= {k: a[k][0] for k in ("u", "delta", "B", "C", "z", "state")}
        made = one_sequence(a, None, None, True, False)
        return ((made["out"] * dout[0].double()).sum() + (made["final"] * dfinal[0].double()).sum()).item()

    h = 2.0 ** -17
    for name in NAMES:
        # up the formula's gradient, by chance how far: along any other direction terms cancel
        along = normal(*args[name].shape).to(DEV).double().abs() * formula["d" + name].view_as(args[name]).sign() * (args[name].double().abs() if name == "A" else 1.0)
        want = (loss(name, h * along) - loss(name, -h * along)) / (2 * h)
        found = (got["d" + name].double() * along).sum().item()
        terms = 20 * T + 4 * N + 200 + (dim // G if name in ("B", "C") else 0) + (T if name in ("A", "D", "delta_bias") else 0)
        tol = terms * 2.0 ** -24 * (size["d" + name].view_as(along) * along.abs()).sum().item() + 1e-6 * abs(want)
        assert abs(want) > 2 * tol, (name, want, tol)                 # (or the test would test nothing)
        assert abs(found - want) <= tol, (name, found, want, tol)


SHAPES = [((1, 2000, 64, 16, 1), None), ((2, 1500, 128, 16, 2), None), ((1, 3000, 16, 16, 1), None), ((1, 1500, 1024, 16, 1), [700, 1, 0, 95, 160, 444, 100]), ((2, 700, 256, 12, 1), None),
          ((1, 1500, 32, 64, 1), None), ((1, 1500, 64, 32, 2), [640, 800]), ((1, 900, 256, 4, 1), None), ((1, 1100, 130, 8, 1), None)]


@pytest.mark.parametrize("slow", [True, False])
@pytest.mark.parametrize("shape,lengths", SHAPES, ids=str)
def test_what_segments_hand_on(shape, lengths, slow):
    print("CASE handed on", shape, lengths, slow, flush=True)
    B, T, dim, N, G = shape
    starts = None if lengths is None else [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    pieces = [(b, 0, T) for b in range(B)] if starts is None else [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    args, dout, dfinal, _ = inputs(*shape, F32, T, n_seqs=len(pieces))
    if slow:
        args["A"] = 0.02 * args["A"]                                 # (decays slow enough that a segment hands on what came in)
    got = run_all(args, dout, dfinal, None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV))
    want, size = reference(args, pieces, dout, dfinal)
    rms = lambda t: t.double().square().mean().sqrt().item()  # noqa: E731
    for name in got:
        terms = 20 * T + 4 * N + 200 + (dim // G if name in ("dB", "dC") else 0) + (B * T if name in ("dA", "dD", "ddelta_bias") else 0)
        bound = (40 + terms ** 0.5) * 2.0 ** -24 * rms(size[name])
        off = rms(got[name].double() - want[name])
        print(name, "%.2g of %.2g" % (off, bound), "values", "%.2g" % rms(want[name]), flush=True)
        assert off <= bound, (name, off, bound)
        assert rms(want[name]) > 20 * bound, name                     # (an eighth of the values and less would be seen)


@pytest.mark.parametrize("shape,lengths", SHAPES, ids=str)
def test_sums_over_tokens_are_those_of_the_tokens(shape, lengths):
    """The gradients of D and of the bias are the sums of what the tokens have: of dout silu(z) u, and of ddelta, as it came out in single precision.  A lane adds at most every fourth token of a
    segment up, then lanes and segments are: T / 4 + 64 + 4096 / 16 roundings of 2^-24 of the magnitudes' sum at most, and the terms' own of 2^-20."""
    B, T, dim, N, G = shape
    starts = None if lengths is None else [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    args, dout, dfinal, _ = inputs(*shape, F32, T + 1, n_seqs=B if lengths is None else len(lengths))
    args["A"] = 0.02 * args["A"]
    got = run_all(args, dout, dfinal, None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV))
    z = args["z"].double()
    for name, terms in (("ddelta_bias", got["ddelta"].double()), ("dD", dout.double() * z * torch.sigmoid(z) * args["u"].double())):
        if lengths is not None:
            terms = terms[:, :starts[-1]]
        want, size = terms.sum((0, 1)), terms.abs().sum((0, 1))
        bound = ((T / 4 + 320) * 2.0 ** -24 + 2.0 ** -20) * size
        assert bool(((got[name].double() - want).abs() <= bound).all()), name
