"""selective_scan_tokens_fn and selective_scan_step_fn against the recurrence in 64 bits, token by token, with its gradients by the formulas.

Every result is a sum of products of the inputs, of steps, decays and gates; `size` is the same sum of their magnitudes (every factor but the decays, which are
positive, by its magnitude).  All is fp32, so a result is off by a number of roundings of 2^-24 each, relative to size:
  a decay exp(x) is off by 2^-22 + |x| 2^-22 (its argument is a product of rounded factors, the step itself a softplus good to 2^-22), and a term passes at most T of
  them, each with two roundings, but weighs exp(-sum |x|), and s exp(-s) < 0.4: 10 T + 8 in all, and as much for the products around it; sums of N states, of T tokens (dA, dD, bias) and
  of the channels of a group (dB, dC) and B rows add their lengths.
The last rounding is half a step of the result's type: 2^-8 in bf16, 2^-11 in fp16, 2^-24 in fp32 (a step without softplus and its decays can
grow to results over fp16's range)."""
import pytest
import torch

from vmamba_amd import selective_scan_step_fn, selective_scan_tokens_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")


def one_sequence(a, dout, dfinal, softplus, size):
    """Results and gradients of one sequence (T, dim) in 64 bits; with `size` the sums of magnitudes."""
    mag = (lambda t: t.abs()) if size else (lambda t: t)
    u, B, C = mag(a["u"]), mag(a["B"]), mag(a["C"])
    T, dim = u.shape
    group = torch.arange(dim, device=u.device) // (dim // B.shape[1])
    raw = a["delta"] + (0 if a["delta_bias"] is None else a["delta_bias"])
    step = torch.nn.functional.softplus(raw, threshold=60) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    A, fed = a["A"], mag(step) * u
    D = torch.zeros(dim, dtype=u.dtype, device=u.device) if a["D"] is None else mag(a["D"])
    if a["z"] is None:
        gate, turn = torch.ones_like(u), None
    else:
        sig = torch.sigmoid(a["z"])
        gate, turn = mag(a["z"] * sig), (1 + a["z"].abs() if size else sig * (1 + a["z"] * (1 - sig)))
    h = torch.zeros(dim, A.shape[1], dtype=u.dtype, device=u.device) if a["state"] is None else mag(a["state"])
    before, y = [], torch.zeros_like(u)
    for t in range(T):
        before.append(h)
        h = torch.exp(step[t][:, None] * A) * h + fed[t][:, None] * B[t][group]
        y[t] = (h * C[t][group]).sum(1)
    inner = y + D * u
    found = {"out": inner * gate, "final": h}
    if dout is None:
        return found
    dout = mag(dout)
    dy = dout * gate
    du, dstep, dB, dC, dA = D * dy, torch.zeros_like(u), torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    ga = torch.zeros_like(h) if dfinal is None else mag(dfinal)
    for t in reversed(range(T)):
        g = ga + dy[t][:, None] * C[t][group]
        decay = torch.exp(step[t][:, None] * A)
        now = decay * before[t] + fed[t][:, None] * B[t][group]
        dC[t].index_add_(0, group, dy[t][:, None] * now)
        dB[t].index_add_(0, group, fed[t][:, None] * g)
        s = (g * B[t][group]).sum(1)
        ga = decay * g
        w = ga * before[t]
        du[t] += mag(step[t]) * s
        dstep[t] = u[t] * s + (w * mag(A)).sum(1)
        dA += w * mag(step[t])[:, None]
    ddelta = dstep * slope
    found |= {"du": du, "ddelta": ddelta, "dA": dA, "dB": dB, "dC": dC, "dD": (dy * u).sum(0), "ddelta_bias": ddelta.sum(0), "dstate": ga}
    if turn is not None:
        found["dz"] = dout * inner * turn
    return found


def reference(args, pieces, dout=None, dfinal=None, softplus=True):
    """Two dicts, results and sizes; pieces: (batch, start, end) of each sequence."""
    both = []
    for size in (False, True):
        made = {}
        for n, (b, lo, hi) in enumerate(pieces):
            a = {k: None if t is None else t.double() for k, t in args.items()}
            for k in ("u", "delta", "B", "C", "z"):
                a[k] = None if a[k] is None else a[k][b, lo:hi]
            a["state"] = None if a["state"] is None else a["state"][n]
            one = one_sequence(a, None if dout is None else dout[b, lo:hi].double(), None if dfinal is None else dfinal[n].double(), softplus, size)
            for k, v in one.items():
                if k in ("final", "dstate"):
                    made.setdefault(k, []).append(v)
                elif k in ("dA", "dD", "ddelta_bias"):
                    made[k] = made.get(k, 0) + v
                else:
                    like = args["u"] if v.shape[1:] == args["u"].shape[2:] else args["B"]
                    made.setdefault(k, torch.zeros(like.shape, dtype=torch.float64, device=DEV))[b, lo:hi] = v
        both.append({k: torch.stack(v) if isinstance(v, list) else v for k, v in made.items()})
    return both


def check(name, got, want, size, args, pieces):
    dim, N = args["A"].shape
    longest = max([hi - lo for _, lo, hi in pieces] + [1])
    terms = 20 * longest + 4 * N + 200
    terms += dim // args["B"].shape[2] if name in ("dB", "dC") else 0
    terms += sum(hi - lo for _, lo, hi in pieces) if name in ("dA", "dD", "ddelta_bias") else 0
    bound = terms * 2.0 ** -24 * size + HALF[got.dtype] * want.abs() + 1e-30 + (2.0 ** -25 if got.dtype == F16 else 0.0)     # (fp16's smallest step)
    off = (got.double() - want).abs()
    over = want.abs() + bound > torch.finfo(got.dtype).max            # what is behind the type's largest value rounds to infinity
    right = (off <= bound) | (over & (got.double() == want.sign() * float("inf")))
    assert got.shape == want.shape, name
    assert bool(right.all()), (name, (off / bound)[~right].max().item())


def inputs(B, T, dim, N, G, dtype, seed=0, gate=True, state=True, extra=True, n_seqs=None):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    a = {"u": normal(B, T, dim).to(DEV, dtype), "delta": (normal(B, T, dim) - 1).to(DEV, dtype), "A": -torch.exp(0.7 * normal(dim, N)).to(DEV),
         "B": normal(B, T, G, N).to(DEV, dtype), "C": normal(B, T, G, N).to(DEV, dtype), "D": normal(dim).to(DEV) if extra else None,
         "z": normal(B, T, dim).to(DEV, dtype) if gate else None, "delta_bias": normal(dim).to(DEV) if extra else None,
         "state": normal(n_seqs or B, dim, N).to(DEV) if state else None}
    return a, normal(B, T, dim).to(DEV, dtype), normal(n_seqs or B, dim, N).to(DEV), normal


def run_all(args, dout, dfinal, cu=None, softplus=True):
    leaves = {n: None if t is None else t.detach().requires_grad_() for n, t in args.items()}
    out, final = selective_scan_tokens_fn(*(leaves[n] for n in NAMES[:8]), softplus, leaves["state"], True, cu)
    wanted = {n: t for n, t in leaves.items() if t is not None}
    outs, douts = ([out, final], [dout, dfinal]) if dfinal is not None else ([out], [dout])
    grads = torch.autograd.grad(outs, list(wanted.values()), douts)
    return {"out": out.detach(), "final": final.detach(), **{"d" + n: d for n, d in zip(wanted, grads)}}


SHAPES = [  # B, T, dim, N, groups
    (1, 1, 1, 1, 1), (2, 2, 16, 16, 1), (1, 15, 17, 16, 1), (2, 16, 64, 4, 2), (1, 17, 40, 8, 1), (3, 31, 66, 16, 3), (1, 63, 100, 12, 2), (1, 64, 33, 32, 1), (2, 65, 70, 64, 2),
    (1, 130, 130, 16, 1), (1, 200, 19, 3, 1), (2, 129, 96, 20, 4), (1, 300, 24, 50, 1), (2, 77, 6, 2, 6), (1, 70, 260, 7, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences(shape, dtype):
    print("CASE token_scan", shape, dtype, flush=True)
    B, T, dim, N, G = shape
    args, dout, dfinal, _ = inputs(*shape, dtype, T, gate=T % 2 == 0 or T == 1, state=(T + N) % 3 != 0, extra=T % 5 != 0)
    dfinal = dfinal if T % 3 else None
    softplus = T % 4 != 3
    if not softplus:                                                 # (steps of both signs, decays of at most e)
        args["delta"], args["delta_bias"] = args["delta"] * 0.1, None
    got = run_all(args, dout, dfinal, softplus=softplus)
    pieces = [(b, 0, T) for b in range(B)]
    want, size = reference(args, pieces, dout, dfinal, softplus)
    for name in got:
        check(name, got[name], want[name], size[name], args, pieces)


def test_gradients_against_differences():
    """Along u, B, C, D, z (a gate's curvature aside) and the state the loss is a polynomial of degree one or, along z, delta, A and the bias, smooth: over a step h a
    central difference is off by h^2 / 6 of the third derivative, which along these directions is below 100 times the magnitudes' sum.  The loss is summed in 64 bits of
    results in fp32."""
    args, dout, _, normal = inputs(1, 70, 24, 16, 2, F32, 3)
    grads = run_all(args, dout, None)
    _, size = reference(args, [(0, 0, 70)], dout)
    loss_size = (size["out"] * dout.double().abs()).sum().item()
    for name in NAMES:
        along = normal(*args[name].shape).to(DEV) * (0.1 * args[name].abs() if name == "A" else 1.0)
        h, curved = (2.0 ** -7, 1.0) if name in ("z", "delta", "delta_bias", "A") else (0.5, 0.0)
        values = []
        for sign in (1, -1):
            moved = {**args, name: args[name] + sign * h * along}
            out = selective_scan_tokens_fn(*(moved[n] for n in NAMES[:8]), True, moved["state"])
            values.append((out.double() * dout.double()).sum().item())
        got, want = (values[0] - values[1]) / (2 * h), (grads["d" + name].double() * along.double()).sum().item()
        grown = 4.0                                                  # the moved inputs' magnitudes: |x| + h |along| for |x|
        assert abs(got - want) <= grown * loss_size * (20 * 70 + 300) * 2.0 ** -24 / h + curved * h * h / 6 * 100 * loss_size, name


PACKED = [[0, 1, 70, 0, 0, 64, 129, 5, 0], [16, 48, 64, 1, 63], [300], [0, 0, 0], [7] * 30, [1000, 3, 0, 500, 40]]


@pytest.mark.parametrize("lengths", PACKED, ids=lambda v: str(len(v)) + "x" + str(sum(v)))
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 90)])
def test_packed(lengths, before, behind):
    """Sequences one behind another, empty ones and rows of none before and behind: as each alone, zeros elsewhere."""
    print("CASE token_scan packed", lengths, before, behind, flush=True)
    T = before + sum(lengths) + behind
    if T == 0:
        T = behind = 5
    starts = [before + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
    args, dout, dfinal, _ = inputs(1, T, 36, 16, 1, F32, 5, n_seqs=len(lengths))
    got = run_all(args, dout, dfinal, cu)
    pieces = [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    want, size = reference(args, pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], args, pieces)
    for name in ("out", "du", "ddelta", "dz", "dB", "dC"):
        assert not got[name][0, :before].any() and not got[name][0, starts[-1]:].any(), name
    for i, n in enumerate(lengths):
        if n == 0:
            assert torch.equal(got["final"][i], args["state"][i]) and torch.equal(got["dstate"][i], dfinal[i])


def step_args(args):
    return {n: t if t is None or n in ("A", "D", "delta_bias", "state") else t[:, 0].contiguous() for n, t in args.items()}


def take_step(a, state, softplus=True):
    return selective_scan_step_fn(*(a[n] for n in ("u", "delta", "A", "B", "C")), state, a["D"], a["z"], a["delta_bias"], softplus)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,dim,N,G", [(1, 1, 1, 1), (3, 64, 16, 1), (5, 100, 12, 2), (2, 33, 3, 1), (70, 520, 16, 4), (4, 6, 64, 3), (1, 1000, 8, 1), (300, 1024, 16, 1), (2, 40, 23, 1)], ids=str)
def test_step(B, dim, N, G, dtype):
    print("CASE token_scan step", B, dim, N, G, dtype, flush=True)
    args, _, _, _ = inputs(B, 1, dim, N, G, dtype, B + N, gate=N != 12, extra=dim != 33)
    want, size = reference(args, [(b, 0, 1) for b in range(B)])
    state = args["state"].clone()
    out = take_step(step_args(args), state)
    pieces = [(0, 0, 1)]
    check("out", out, want["out"][:, 0], size["out"][:, 0], args, pieces)
    check("final", state, want["final"], size["final"], args, pieces)


def test_prompt_then_tokens():
    """A prompt and then tokens one by one are the whole sequence."""
    args, _, _, _ = inputs(3, 90, 48, 16, 2, F32, 9)
    whole, final = selective_scan_tokens_fn(*(args[n] for n in NAMES[:8]), True, args["state"], True)
    cut = {n: t[:, :77] if n in ("u", "delta", "B", "C", "z") else t for n, t in args.items()}
    out, state = selective_scan_tokens_fn(*(cut[n] for n in NAMES[:8]), True, args["state"], True)
    outs = [out]
    for t in range(77, 90):
        a = {n: v[:, t] if n in ("u", "delta", "B", "C", "z") else v for n, v in args.items()}
        outs.append(take_step(a, state)[:, None])
    want, size = reference(args, [(b, 0, 90) for b in range(3)])
    check("out", torch.cat(outs, 1), want["out"], size["out"], args, [(0, 0, 90)])
    check("final", state, want["final"], size["final"], args, [(0, 0, 90)])
    check("final", final, want["final"], size["final"], args, [(0, 0, 90)])
    check("out", whole, want["out"], size["out"], args, [(0, 0, 90)])


@pytest.mark.parametrize("shape", [(1, 2000, 64, 16, 1), (2, 700, 128, 16, 2), (1, 3000, 16, 16, 1), (1, 600, 32, 64, 1), (2, 500, 64, 32, 2), (1, 900, 256, 4, 1), (1, 1100, 1, 1, 1), (9, 333, 640, 16, 1)],
                         ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_long_sequences(shape, dtype):
    """Many segments, of channels and states that fill their lanes and of those that do not."""
    print("CASE token_scan long", shape, dtype, flush=True)
    args, dout, dfinal, _ = inputs(*shape, dtype, shape[1])
    got = run_all(args, dout, dfinal)
    pieces = [(b, 0, shape[1]) for b in range(shape[0])]
    want, size = reference(args, pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], args, pieces)


@pytest.mark.parametrize("N", [16, 32, 64, 4])
def test_packed_where_lanes_are_full(N):
    """As test_packed, with segments' ends inside and at the ends of sequences, and a lone row before them."""
    lengths = [255, 0, 1, 256, 16, 17, 700, 0, 64, 31]
    starts = [1 + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    T = starts[-1] + 40
    cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
    args, dout, dfinal, _ = inputs(1, T, 128, N, 2, BF16, 6, n_seqs=len(lengths))
    got = run_all(args, dout, dfinal, cu)
    pieces = [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    want, size = reference(args, pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], args, pieces)
    for name in ("out", "du", "ddelta", "dz", "dB", "dC"):
        assert not got[name][0, :1].any() and not got[name][0, starts[-1]:].any(), name


@pytest.mark.parametrize("shape,lengths", [((4, 512, 2048, 16, 1), None), ((4, 601, 1024, 8, 2), None), ((1, 2400, 2048, 16, 1), [700, 1, 0, 95, 160, 900, 444]), ((2, 700, 1100, 16, 1), None),
                                           ((1, 1500, 2048, 32, 1), [640, 860])], ids=str)
def test_what_segments_hand_back_from_shorter_ones(shape, lengths):
    """Sizes at which what is handed from behind is found from shorter segments than the gradients' own."""
    print("CASE token_scan handed back", shape, lengths, flush=True)
    B, T = shape[:2]
    starts = None if lengths is None else [50 + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    pieces = [(b, 0, T) for b in range(B)] if starts is None else [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    args, dout, dfinal, _ = inputs(*shape, BF16, T, n_seqs=len(pieces))
    args["A"] = 0.02 * args["A"]                                     # (decays slow enough that a segment hands on what came in)
    got = run_all(args, dout, dfinal, None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV))
    want, size = reference(args, pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], args, pieces)
