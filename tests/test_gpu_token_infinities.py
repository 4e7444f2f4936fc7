"""Infinite values in the selective scan of tokens: results and gradients are infinite and undefined where the formulas in 64 bits are, and nowhere else -- however many states and channels
lanes have beside those that there are, wherever tiles, segments and sequences end, and whether a skip term is there.

All other inputs are positive (A negative), so that infinities meet no others of the other sign but where the formulas have them do so.  What is finite is compared as in
test_gpu_token_scan.py: off by at most 20 T + 4 N + 200 roundings of 2^-24 of the sum of magnitudes, more where tokens or channels are summed."""
import pytest
import torch

from vmamba_amd import selective_scan_step_fn, selective_scan_tokens_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = torch.float32
INF = float("inf")
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")


def one_sequence(a, dout, dfinal, size):
    """The formulas, token by token; with `size` of the magnitudes of A's terms (all others are positive)."""
    u, B, C, A, D, z = a["u"], a["B"], a["C"], a["A"], a["D"], a["z"]
    T, dim = u.shape
    group = torch.arange(dim, device=u.device) // (dim // B.shape[1])
    raw = a["delta"] if a["delta_bias"] is None else a["delta"] + a["delta_bias"]
    step, slope = torch.where(raw > 60, raw, torch.log1p(torch.exp(raw.clamp(max=60)))), torch.sigmoid(raw)
    sig = None if z is None else torch.sigmoid(z)
    gate, turn = (1.0, None) if z is None else (z * sig, sig * (1 + z * (1 - sig)))
    h = torch.zeros(dim, A.shape[1], dtype=u.dtype, device=u.device) if a["state"] is None else a["state"]
    before, inner = [], torch.zeros_like(u)
    for t in range(T):
        before.append(h)
        h = torch.exp(step[t][:, None] * A) * h + (step[t] * u[t])[:, None] * B[t][group]
        inner[t] = (h * C[t][group]).sum(1)
    inner = inner if D is None else inner + D * u
    dy = dout * gate
    du = torch.zeros_like(u) if D is None else D * dy
    dstep, dB, dC, dA = torch.zeros_like(u), torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    ga = torch.zeros_like(h) if dfinal is None else dfinal
    for t in reversed(range(T)):
        g = ga + dy[t][:, None] * C[t][group]
        fed, decay = (step[t] * u[t])[:, None], torch.exp(step[t][:, None] * A)
        dC[t].index_add_(0, group, dy[t][:, None] * (decay * before[t] + fed * B[t][group]))
        dB[t].index_add_(0, group, fed * g)
        s, ga = (g * B[t][group]).sum(1), decay * g
        w = ga * before[t]
        du[t] += step[t] * s
        dstep[t] = u[t] * s + (w * (A.abs() if size else A)).sum(1)
        dA += w * step[t][:, None]
    made = {"out": inner * gate, "final": h, "du": du, "ddelta": dstep * slope, "dA": dA, "dB": dB, "dC": dC, "dstate": ga, "ddelta_bias": (dstep * slope).sum(0), "dD": (dy * u).sum(0)}
    return made if turn is None else made | {"dz": dout * inner * turn}


def reference(args, pieces, dout, dfinal):
    both = []
    for size in (False, True):
        made = {}
        for n, (b, lo, hi) in enumerate(pieces):
            a = {k: None if t is None else t.double() for k, t in args.items()}
            a |= {k: a[k][b, lo:hi] for k in ("u", "delta", "B", "C", "z") if a[k] is not None}
            a["state"] = None if a["state"] is None else a["state"][n]
            for k, v in one_sequence(a, dout[b, lo:hi].double(), None if dfinal is None else dfinal[n].double(), size).items():
                if k in ("final", "dstate"):
                    made.setdefault(k, []).append(v)
                elif k in ("dA", "dD", "ddelta_bias"):
                    made[k] = made.get(k, 0) + v
                else:
                    like = args["B"] if k in ("dB", "dC") else args["u"]
                    made.setdefault(k, torch.zeros(like.shape, dtype=torch.float64, device=DEV))[b, lo:hi] = v
        both.append({k: torch.stack(v) if isinstance(v, list) else v for k, v in made.items()})
    return both


def kinds(t):
    return torch.where(t.isnan(), 2, torch.where(t.isinf(), t.sign(), torch.zeros_like(t))).int()


def check(name, got, want, size, args, pieces):
    assert got.shape == want.shape, name
    got = got.double()
    other = kinds(got) != kinds(want)
    assert not bool(other.any()), (name, int(other.sum()), [(got[tuple(i)].item(), want[tuple(i)].item(), i.tolist()) for i in other.nonzero()[:3]])
    dim, N = args["A"].shape
    terms = 20 * max([hi - lo for _, lo, hi in pieces] + [1]) + 4 * N + 200
    terms += dim // args["B"].shape[2] if name in ("dB", "dC") else 0
    terms += sum(hi - lo for _, lo, hi in pieces) if name in ("dA", "dD", "ddelta_bias") else 0
    off, bound = (got - want).abs(), terms * 2.0 ** -24 * size + 1e-30
    finite = want.isfinite()
    assert bool((off <= bound)[finite].all()), (name, (off / bound)[finite].max().item())


def inputs(B, T, dim, N, G, seed, gate, extra, state, n_seqs):
    gen = torch.Generator().manual_seed(seed)
    some = lambda *s: (0.5 + torch.rand(*s, generator=gen)).to(DEV)  # noqa: E731 -- 0.5 to 1.5
    return {"u": some(B, T, dim), "delta": some(B, T, dim) - 2, "A": -0.25 * some(dim, N), "B": some(B, T, G, N), "C": some(B, T, G, N), "D": some(dim) if extra else None,
            "z": some(B, T, dim) if gate else None, "delta_bias": some(dim) - 1 if extra else None, "state": some(n_seqs, dim, N) if state else None}, some(B, T, dim), some(n_seqs, dim, N)


def compare(args, dout, dfinal, lengths):
    """The operator against the formulas; lengths: of packed sequences, or None."""
    B, T = args["u"].shape[:2]
    starts = None if lengths is None else [3 + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    pieces = [(b, 0, T) for b in range(B)] if starts is None else [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    cu = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV)
    leaves = {n: None if t is None else t.detach().requires_grad_() for n, t in args.items()}
    out, final = selective_scan_tokens_fn(*(leaves[n] for n in NAMES[:8]), True, leaves["state"], True, cu)
    wanted = {n: t for n, t in leaves.items() if t is not None}
    outs, douts = ([out], [dout]) if dfinal is None else ([out, final], [dout, dfinal])
    grads = torch.autograd.grad(outs, list(wanted.values()), douts)
    got = {"out": out.detach(), "final": final.detach(), **{"d" + n: d for n, d in zip(wanted, grads)}}
    want, size = reference(args, pieces, dout, dfinal)
    return got, want, size, pieces


# (sequence, token, channel) of the infinite value, and tokens: one walk of the token axis, several segments (of 16 channels and fewer from 256 tokens on), packed
SIDES = {"results": ("out", "final"), "gradients": ("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dstate")}
LAYOUTS = {"short": (2, 45, 2, 1, 20, None), "cut": (1, 700, 1, 0, 333, None), "packed": (1, 420, 4, 2, 130, [70, 0, 309, 33])}
STATES = [1, 3, 12, 16, 20, 50]


@pytest.mark.parametrize("side,where", [*(("results", n) for n in ("u", "delta", "B", "C", "state")), *(("gradients", n) for n in ("u", "delta", "B", "C", "state", "dout", "dfinal"))])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("N", STATES)
def test_one_infinite_value(N, layout, side, where):
    B, T, n_seqs, seq, t, lengths = LAYOUTS[layout]
    print("CASE infinite", side, where, layout, N, flush=True)
    dim = 5 if N != 16 else 16                                       # (lanes without channels, and none)
    args, dout, dfinal = inputs(B, T, dim, N, 1, N, gate=True, extra=N % 2 == 0, state=True, n_seqs=n_seqs)
    at = (seq if lengths is None else 0, t)
    {"state": args["state"], "dfinal": dfinal}.get(where, dout if where == "dout" else args.get(where))[(seq, 2, N // 2) if where in ("state", "dfinal") else (*at, 0, N // 2) if where in ("B", "C") else (*at, 2)] = INF
    got, want, size, pieces = compare(args, dout, dfinal, lengths)
    assert any(not bool(want[name].isfinite().all()) for name in got if name in SIDES[side])
    for name in got:
        if name in SIDES[side]:
            check(name, got[name], want[name], size[name], args, pieces)


@pytest.mark.parametrize("side,where", [("results", "state"), ("results", "u"), ("gradients", "dfinal"), ("gradients", "dout")])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("N", [3, 16])
def test_an_infinite_step_forgets_nothing_infinite(N, layout, side, where):
    """A decay of 0 of an infinite state, or of an infinite gradient of one, is NaN -- from the infinite step on, though a segment before or behind it hands the state on by its steps' sum."""
    B, T, n_seqs, seq, t, lengths = LAYOUTS[layout]
    args, dout, dfinal = inputs(B, T, 16, N, 1, N, gate=True, extra=True, state=True, n_seqs=n_seqs)
    b = seq if lengths is None else 0
    args["delta"][b, t, 2] = INF
    if where in ("state", "dfinal"):
        (args["state"] if where == "state" else dfinal)[seq, 2, N // 2] = INF
    else:
        (args["u"] if where == "u" else dout)[b, t + (-15 if where == "u" else 20), 2] = INF
    got, want, size, pieces = compare(args, dout, dfinal, lengths)
    assert any(bool(want[name].isnan().any()) for name in got if name in SIDES[side])
    for name in got:
        if name in SIDES[side]:
            check(name, got[name], want[name], size[name], args, pieces)


@pytest.mark.parametrize("side", SIDES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("N", STATES)
@pytest.mark.parametrize("dim,G", [(5, 1), (32, 2), (128, 1)], ids=str)
def test_states_that_forget_at_once(dim, G, N, layout, side):
    """A of -inf for two states, one of them of a last channel: a decay of 0, in tiles that sequences begin and end in as elsewhere."""
    B, T, n_seqs, _, _, lengths = LAYOUTS[layout]
    print("CASE forgets", dim, G, N, layout, flush=True)
    args, dout, dfinal = inputs(B, T, dim, N, G, N + dim, gate=N != 12, extra=N % 2 == 0, state=True, n_seqs=n_seqs)
    args["A"][dim // 2, 0] = args["A"][dim - 1, N - 1] = -INF
    got, want, size, pieces = compare(args, dout, dfinal, lengths)
    for name in got:
        if name in SIDES[side]:
            check(name, got[name], want[name], size[name], args, pieces)


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dim", [16, 64])
def test_no_skip_term_is_no_term(dim, gate):
    """Without D an infinite u (and an infinite gradient) meets no 0 D."""
    for where in ("u", "dout"):
        args, dout, dfinal = inputs(1, 48, dim, 16, 1, 7, gate=gate, extra=False, state=True, n_seqs=1)
        (dout if where == "dout" else args["u"])[0, 20, 2] = INF
        got, want, size, pieces = compare(args, dout, dfinal, None)
        assert not bool(want["out"].isnan().any()) and not bool(want["du"].isnan().any())
        for name in got:
            check(name, got[name], want[name], size[name], args, pieces)


def test_no_skip_term_of_a_step():
    args, _, _ = inputs(2, 1, 6, 16, 2, 3, gate=True, extra=False, state=True, n_seqs=2)
    a = {n: t if t is None or n in ("A", "state") else t[:, 0] for n, t in args.items()}
    a["u"][1, 2] = INF
    out = selective_scan_step_fn(*(a[n] for n in ("u", "delta", "A", "B", "C")), a["state"], None, a["z"])
    assert out[1, 2] == INF and int(out.isfinite().sum()) == 11


@pytest.mark.parametrize("extra", [True, False])
@pytest.mark.parametrize("N", [1, 3, 12, 16, 33])
def test_a_step_is_a_prompt_of_one_token(N, extra):
    for where in ("u", "delta", "B", "state", "A"):
        args, dout, _ = inputs(2, 1, 6, N, 2, N, gate=True, extra=extra, state=True, n_seqs=2)
        args[where][{"u": (1, 0, 2), "delta": (1, 0, 2), "B": (1, 0, 0, 0), "state": (1, 2, 0), "A": (2, N - 1)}[where]] = -INF if where == "A" else INF
        got, want, size, pieces = compare(args, dout, None, None)
        state, a = args["state"].clone(), {n: t if t is None or n in ("A", "D", "delta_bias", "state") else t[:, 0] for n, t in args.items()}
        one = selective_scan_step_fn(*(a[n] for n in ("u", "delta", "A", "B", "C")), state, a["D"], a["z"], a["delta_bias"])
        for name, t in (("out", one), ("final", state)):
            check(name, t, want[name].reshape(t.shape), size[name].reshape(t.shape), args, pieces)
            check(name, got[name], want[name], size[name], args, pieces)
