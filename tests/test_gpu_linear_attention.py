"""linear_attention_fn and linear_attention_step_fn against the recurrence in 64 bits, token by token.

Every result is a sum of products of the inputs, of decays and, for gradients, of the gradients that come in; `size` below is the same sum of
their magnitudes (the same formula of |q|, |k|, |v|, ...: no term is negative then).  A relative rounding u of an operand or a
partial sum moves a result by at most u * size.  Half a step is 2^-8 in bf16, 2^-11 in fp16, 2^-24 in fp32.
  bf16: an operand that is computed (a pair's weight, a state) is rounded once, and the result once: 2^-8 size + 2^-8 |result|.  What is kept in 32 bits (states,
        decays' gradients in fp32) comes of operands split in two at least: 2^-16 size for each of at most three such splits; in three: 2^-24.
  fp16, fp32: fp32 throughout; fp16 results are rounded once.
  Sums in fp32: a result passes at most N = dk + dv + 4 C + 4 (chunks) + 64 additions and products; an exp of x is good to 2^-22 + |x| 2^-23, and
  x below -40 contributes nothing to speak of.  (N + 200) 2^-24 size in all."""
import pytest
import torch

from vmamba_amd import linear_attention_fn, linear_attention_step_fn, qk_norm_rotate_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def recur(q, k, v, g, state, scale, pieces):
    """(out, final states) of (B, T, H, D) in 64 bits; pieces: (batch, start, end) of each sequence."""
    H = max(t.shape[2] for t in (q, k, v))
    q, k, v = (t.repeat_interleave(H // t.shape[2], 2) for t in (q, k, v))
    out = [[torch.zeros(H, v.shape[3], dtype=torch.float64)] * q.shape[1] for _ in range(q.shape[0])]
    finals = []
    for n, (b, lo, hi) in enumerate(pieces):
        S = torch.zeros(H, q.shape[3], v.shape[3], dtype=torch.float64) if state is None else state[n]
        for t in range(lo, hi):
            if g is not None:
                S = (g if g.dim() == 1 else g[b, t]).exp()[:, None, None] * S
            S = S + k[b, t][:, :, None] * v[b, t][:, None, :]
            out[b][t] = (q[b, t][:, :, None] * S).sum(1) * scale
        finals.append(S)
    return torch.stack([torch.stack(row) if row else torch.zeros(0, H, v.shape[3], dtype=torch.float64) for row in out]), torch.stack(finals)


def reference(q, k, v, g, state, scale, pieces, dout=None, dfinal=None):
    """Results and gradients in 64 bits, and the sums of magnitudes behind them: two dicts."""
    both = []
    for size in (False, True):
        leaves = {n: None if t is None else (t.double().cpu().abs() if size and n != "g" else t.double().cpu()).requires_grad_()
                  for n, t in (("q", q), ("k", k), ("v", v), ("g", g), ("state", state))}
        out, final = recur(*leaves.values(), scale, pieces)
        found = {"out": out.detach(), "final": final.detach()}
        if dout is not None:
            pick = lambda t: t.double().cpu().abs() if size else t.double().cpu()  # noqa: E731
            loss = (out * pick(dout)).sum() + (0 if dfinal is None else (final * pick(dfinal)).sum())
            wanted = {n: t for n, t in leaves.items() if t is not None}
            grads = torch.autograd.grad(loss, list(wanted.values()), allow_unused=True)
            found |= {"d" + n: torch.zeros_like(t) if d is None else d for (n, t), d in zip(wanted.items(), grads)}
        both.append(found)
    return both


def check(name, got, want, size, dtype, dims, tokens, split=2.0 ** -16):
    C = 64 if dtype == BF16 else 32
    terms = (sum(dims) + 4 * C + 4 * (tokens // C + 1) + 264) * 2.0 ** -24
    kept = got.dtype == F32 and dtype == BF16
    operand = 3 * split if kept else 2.0 ** -8 if dtype == BF16 else 0.0
    bound = (operand + terms) * size + HALF[got.dtype] * want.abs() + 1e-30 + (2.0 ** -25 if got.dtype == F16 else 0.0)     # (fp16's smallest step)
    off = (got.double().cpu() - want).abs()
    assert got.shape == want.shape, name
    assert bool((off <= bound).all()), (name, (off / bound).max().item())


def inputs(B, T, Hq, Hk, Hv, dk, dv, dtype, decay, seed=0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    H = max(Hq, Hk, Hv)
    q, k, v = (normal(B, T, h, d).to(DEV, dtype) for h, d in ((Hq, dk), (Hk, dk), (Hv, dv)))
    g = {"none": None, "head": -torch.rand(H, generator=gen) * 0.3, "token": -torch.nn.functional.softplus(normal(B, T, H) - 2)}[decay[0]]
    g = None if g is None else g.to(DEV, F32 if decay[1] else dtype)
    dout = normal(B, T, H, dv).to(DEV, dtype)
    return q, k, v, g, dout, normal


def run_all(q, k, v, g, state, dout, dfinal, cu=None, scale=None):
    leaves = {n: None if t is None else t.detach().requires_grad_() for n, t in (("q", q), ("k", k), ("v", v), ("g", g), ("state", state))}
    out, final = linear_attention_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], scale, leaves["state"], True, cu)
    wanted = {n: t for n, t in leaves.items() if t is not None}
    outs, douts = ([out, final], [dout, dfinal]) if dfinal is not None else ([out], [dout])
    grads = torch.autograd.grad(outs, list(wanted.values()), douts)
    return {"out": out.detach(), "final": final.detach(), **{"d" + n: d for n, d in zip(wanted, grads)}}


SHAPES = [  # B, T, Hq, Hk, Hv, dk, dv
    (1, 1, 1, 1, 1, 16, 16), (2, 2, 2, 2, 2, 64, 64), (1, 31, 4, 2, 4, 32, 48), (2, 33, 3, 1, 3, 20, 36), (1, 63, 2, 2, 2, 128, 64), (1, 64, 2, 2, 2, 64, 128),
    (2, 65, 4, 4, 1, 17, 5), (1, 129, 1, 1, 6, 64, 32), (1, 200, 2, 2, 2, 128, 128), (1, 97, 2, 1, 2, 256, 256), (1, 70, 1, 1, 1, 1, 1), (1, 130, 6, 3, 2, 96, 130),
]


@pytest.mark.parametrize("decay", [("none", 0), ("head", 1), ("token", 0), ("token", 1)], ids=["no", "head", "own", "fp32"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences(shape, dtype, decay):
    print("CASE linear_attention", shape, dtype, decay, flush=True)
    B, T, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, dout, normal = inputs(*shape, dtype, decay, T)
    H = max(Hq, Hk, Hv)
    carried = (T + H) % 2 == 0
    state = normal(B, H, dk, dv).to(DEV) if carried else None
    dfinal = normal(B, H, dk, dv).to(DEV) if T % 3 else None
    scale = None if T % 5 else 0.7
    got = run_all(q, k, v, g, state, dout, dfinal, scale=scale)
    want, size = reference(q, k, v, g, state, dk ** -0.5 if scale is None else scale, [(b, 0, T) for b in range(B)], dout, dfinal)
    for name in got:
        # a decay of its own type is rounded once; one that a head's tokens share is a sum of theirs
        check(name, got[name], want[name], size[name], dtype, (dk, dv, B * T if name == "dg" else 0), T)


def test_gradients_against_differences():
    """Along one input at a time the loss is linear (q, k, v, state), so a difference over any step is its derivative; along the decays over a step h it is
    off by h^2 / 6 of the third derivative.  The loss itself is summed in 64 bits from results in fp32: 2^-22 of the magnitudes' sum covers it."""
    q, k, v, g, dout, normal = inputs(1, 90, 2, 1, 2, 32, 48, F32, ("token", 1), 3)
    state = normal(1, 2, 32, 48).to(DEV)
    grads = run_all(q, k, v, g, state, dout, None)
    args = {"q": q, "k": k, "v": v, "g": g, "state": state}
    _, size = reference(q, k, v, g, state, 32 ** -0.5, [(0, 0, 90)], dout)
    loss_size = (size["out"] * dout.double().cpu().abs()).sum().item()
    for name in args:
        along = normal(*args[name].shape).to(DEV)
        h = 2.0 ** -7 if name == "g" else 1.0
        values = []
        for sign in (1, -1):
            moved = {**args, name: args[name] + sign * h * along}
            out = linear_attention_fn(moved["q"], moved["k"], moved["v"], moved["g"], None, moved["state"])
            values.append((out.double() * dout.double()).sum().item())
        got, want = (values[0] - values[1]) / (2 * h), (grads["d" + name].double() * along.double()).sum().item()
        grown = 4.0 * (2 if name == "g" else 1)                       # the moved inputs' magnitudes: |x| + |along| for |x|
        assert abs(got - want) <= grown * loss_size * (600 * 2.0 ** -24 / h + (h * h * 90 if name == "g" else 0)), name


def test_packed():
    """Sequences one behind another, empty ones and rows of none before, between and behind: as each alone, zeros elsewhere."""
    lengths, before, behind = [0, 1, 70, 0, 0, 64, 129, 5, 0], 3, 90
    T = before + sum(lengths) + behind
    starts = [before + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
    pieces = [(0, a, a + n) for a, n in zip(starts, lengths)]
    for dtype in (BF16, F16, F32):
        q, k, v, g, dout, normal = inputs(1, T, 3, 1, 3, 32, 40, dtype, ("token", 1), 5)
        q[:, :before], v[:, -behind:], g[:, -1] = float("nan"), float("inf"), float("nan")         # rows of nobody
        state, dfinal = normal(len(lengths), 3, 32, 40).to(DEV), normal(len(lengths), 3, 32, 40).to(DEV)
        for state_, dfinal_ in ((state, dfinal), (None, None)):
            got = run_all(q, k, v, g, state_, dout, dfinal_, cu)
            clean = [torch.nan_to_num(t, 0, 0, 0) for t in (q, k, v, g)]
            want, size = reference(*clean, state_, 32 ** -0.5, pieces, dout, dfinal_)
            for name in got:
                check(name, got[name], want[name], size[name], dtype, (32, 40), 129)
            for name in ("out", "dq", "dk", "dv", "dg"):
                assert not got[name][:, :before].any() and not got[name][:, T - behind:].any(), name
    # a learnt decay's gradient leaves the rows of nobody out
    q, k, v, g, dout, normal = inputs(1, T, 3, 1, 3, 32, 40, F32, ("head", 1), 5)
    got = run_all(q, k, v, g, None, dout, None, cu)
    want, size = reference(q, k, v, g, None, 32 ** -0.5, pieces, dout)
    check("dg", got["dg"], want["dg"], size["dg"], F32, (32, 40, T), 129)


@pytest.mark.parametrize("count", [1, 255, 256, 257, 700])
def test_many_packed(count):
    """More sequences than the table's kernel takes at once, and one long enough to be cut into segments."""
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 9, (count,), generator=gen).tolist()
    lengths[count // 2] = 2500
    starts = [sum(lengths[:i]) for i in range(count + 1)]
    q, k, v, g, dout, normal = inputs(1, starts[-1], 2, 2, 2, 16, 32, F32, ("token", 1), 1)
    out, final = linear_attention_fn(q, k, v, g, output_final_state=True, cu_seqlens=torch.tensor(starts, dtype=torch.int32, device=DEV))
    for n in {0, 1 % count, count // 2, (count // 2 + 1) % count, 254 % count, 255 % count, 256 % count, count - 1}:
        lo, hi = starts[n], starts[n + 1]
        if hi > lo:
            alone, state = linear_attention_fn(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], g[:, lo:hi], output_final_state=True)
            assert torch.allclose(out[:, lo:hi], alone, rtol=1e-4, atol=1e-5) and torch.allclose(final[n], state[0], rtol=1e-4, atol=1e-4)
        else:
            assert not final[n].any()


@pytest.mark.parametrize("places", [[0, 50, 30, 90], [-5, 20, 300, 90], [90, 10, 10, 10], [200, 200, 200, 200], [0, 0, 0, 0], [40, 2 ** 31 - 1, -2 ** 31, 60]], ids=str)
def test_places_that_are_none(places):
    """Places outside the rows are moved into them, descending ones are the ones before: no row is read or written that is not there."""
    T = 100
    q, k, v, g, dout, _ = inputs(1, T, 2, 2, 2, 16, 16, BF16, ("token", 1))
    cu, most = [], 0
    for c in places:
        most = max(most, min(max(c, 0), T))
        cu.append(most)
    got, want = (run_all(q, k, v, g, None, dout, None, torch.tensor(c, dtype=torch.int32, device=DEV)) for c in (places, cu))
    for name in got:
        assert torch.equal(got[name], want[name]), name


def test_segments():
    """A long sequence of one head, cut into segments that are walked on their own and joined: as in pieces that hand their states on."""
    for dtype, T in ((BF16, 5003), (F32, 2777)):
        q, k, v, g, dout, normal = inputs(1, T, 1, 1, 1, 64, 64, dtype, ("token", 1), 2)
        g = g * 0.02                                                  # horizons beyond a segment
        state, dfinal = normal(1, 1, 64, 64).to(DEV), normal(1, 1, 64, 64).to(DEV)
        got = run_all(q, k, v, g, state, dout, dfinal)
        exact = [t.double().requires_grad_() for t in (q, k, v, g, state)]
        qd, kd, vd, gd, sd = exact
        G = gd[0, :, 0].cumsum(0)
        seen = torch.ones(T, T, dtype=torch.bool, device=DEV).tril()
        decay = (G[:, None] - G[None]).masked_fill(~seen, -1e30).exp()
        out = ((qd[0, :, 0] @ kd[0, :, 0].t()) * decay) @ vd[0, :, 0] + (qd[0, :, 0] * G.exp()[:, None]) @ sd[0, 0]
        final = (kd[0, :, 0] * (G[-1] - G).exp()[:, None]).t() @ vd[0, :, 0] + G[-1].exp() * sd[0, 0]
        grads = torch.autograd.grad([out / 8, final], exact, [dout[0, :, 0].double(), dfinal[0, 0].double()])
        near = lambda a, b: ((a.double().reshape(-1) - b.reshape(-1)).norm() / b.norm()).item()  # noqa: E731
        # in norm: a rounding's 2^-8 and an operand's, one of them at their worst
        limit = 2 * 2.0 ** -8 if dtype == BF16 else 2e-6
        assert near(got["out"], out / 8) <= limit
        for name, want in zip(("dq", "dk", "dv"), grads):
            assert near(got[name], want) <= limit, name
        kept = 3 * 2.0 ** -16 if dtype == BF16 else 2e-6
        assert near(got["final"], final) <= kept and near(got["dstate"], grads[4]) <= kept and near(got["dg"], grads[3]) <= 4 * kept


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_layouts(dtype):
    """Other strides and alignments than dense ones: the same bits."""
    B, T, H, dk, dv = 2, 100, 4, 32, 24
    q, k, v, g, dout, normal = inputs(B, T, H, H, H, dk, dv, dtype, ("token", 1))
    dense = run_all(q, k, v, g, None, dout, None)

    def moved(t, how):
        if how == "heads first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if how == "tokens first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        if how == "slice":
            return torch.cat([t, t, t], -1)[..., t.shape[-1]:2 * t.shape[-1]]
        odd = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return odd.copy_(t)

    for how in ("heads first", "tokens first", "slice", "odd address"):
        got = run_all(moved(q, how), moved(k, how), moved(v, how), moved(g, how), None, moved(dout, how), None)
        for name in dense:
            assert torch.equal(got[name], dense[name]), (how, name)
    # a head and a batch that are expanded, and the gradient of such a broadcast
    one = k[:1, :, :1].detach().requires_grad_()
    out, _ = linear_attention_fn(q, one.expand(B, T, H, dk), v, g, output_final_state=True)
    dk_one, = torch.autograd.grad(out, one, dout)
    shared = run_all(q, k[:1, :, :1].expand(B, T, 1, dk), v, g, None, dout, None)
    assert torch.equal(out, shared["out"])
    assert ((dk_one.double() - shared["dk"].double().sum((0,), keepdim=True)).norm() / dk_one.double().norm()).item() <= 4 * HALF[dtype] + 1e-6
    # a gradient that is dense in another order, and one that is expanded
    for d in (dout.transpose(-1, -2).contiguous().transpose(-1, -2), dout[:1, :1, :1, :1].expand_as(dout)):
        a, b = run_all(q, k, v, g, None, d, None), run_all(q, k, v, g, None, d.contiguous(), None)
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_resets_and_extremes(dtype):
    """Decays of -inf, of the lowest value and long sums: what is behind them is as if the sequence began there."""
    q, k, v, g, dout, normal = inputs(1, 200, 2, 2, 2, 32, 32, dtype, ("token", 1))
    state = normal(1, 2, 32, 32).to(DEV)
    for at, low in ((0, -float("inf")), (70, -float("inf")), (64, torch.finfo(F32).min), (199, -1e5), (100, -700.0)):
        cut = g.clone()
        cut[:, at] = low
        got, final = linear_attention_fn(q, k, v, cut, initial_state=state, output_final_state=True)
        alone, state_alone = linear_attention_fn(q[:, at:], k[:, at:], v[:, at:], g[:, at:], output_final_state=True)
        near = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
        assert near(got[:, at:], alone) <= 3 * HALF[dtype] + 2e-6 and near(final, state_alone) <= 2.0 ** -14
        grads = run_all(q, k, v, cut, state, dout, None)
        assert all(bool(t.isfinite().all()) for t in grads.values())
        if at:
            assert near(grads["dq"][:, at:], run_all(q[:, at:], k[:, at:], v[:, at:], g[:, at:], None, dout[:, at:], None)["dq"]) <= 3 * HALF[dtype] + 2e-6


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("at", [20, 40, 100])
def test_values_that_are_none(dtype, at):
    """An infinity or NaN in a token reaches no token in front of it, in its own chunk either; in other sequences nothing."""
    q, k, v, g, dout, _ = inputs(2, 128, 2, 2, 2, 32, 32, dtype, ("token", 1))
    clean = linear_attention_fn(q, k, v, g)
    for which in range(3):
        for bad in (float("nan"), float("inf")):
            args = [q.clone(), k.clone(), v.clone()]
            args[which][0, at, 1, 3] = bad
            out = linear_attention_fn(*args, g)
            near = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
            assert near(out[0, :at], clean[0, :at]) <= 2 * HALF[dtype] and torch.equal(out[1], clean[1]) and torch.equal(out[0, :, 0], clean[0, :, 0])
            if which == 2:                                            # one column of the values alone
                assert bool(out[0, :, 1, 4:].isfinite().all()) and not bool(out[0, at:, 1, 3].isfinite().any())
            # a loss of the tokens in front alone, whatever stands behind: its gradient too
            d = dout.clone()
            d[0, at:] = 0
            if which == 0:                                            # (0 times a key or value that is none is none)
                grads = run_all(*args, g, None, d, None)
                good = run_all(q, k, v, g, None, d, None)
                assert near(grads["dq"][0, :at], good["dq"][0, :at]) <= 2 * HALF[dtype]


def test_empty():
    for B, T in ((0, 5), (2, 0)):
        q, k, v = (torch.zeros(B, T, 2, 16, device=DEV, requires_grad=True) for _ in range(3))
        state = torch.randn(B, 2, 16, 16, device=DEV, requires_grad=True)
        out, final = linear_attention_fn(q, k, v, None, None, state, True)
        assert out.shape == (B, T, 2, 16) and torch.equal(final, state)
        grads = torch.autograd.grad([out, final], [q, k, v, state], [torch.ones_like(out), torch.ones_like(final)])
        assert torch.equal(grads[3], torch.ones_like(state)) and all(t.shape == q.shape for t in grads[:3])
    with torch.no_grad():
        assert linear_attention_step_fn(*(torch.zeros(0, 2, 16, device=DEV) for _ in range(3)), None, torch.zeros(0, 2, 16, 16, device=DEV)).shape == (0, 2, 16)


def test_which_gradients():
    """Only those that are asked for, from the output, the final state or both."""
    q, k, v, g, dout, normal = inputs(1, 70, 2, 2, 2, 16, 16, F32, ("token", 1))
    state, dfinal = normal(1, 2, 16, 16).to(DEV), normal(1, 2, 16, 16).to(DEV)
    whole = run_all(q, k, v, g, state, dout, dfinal)
    leaf = v.clone().requires_grad_()
    out, final = linear_attention_fn(q, k, leaf, g, None, state, True)
    assert torch.equal(torch.autograd.grad([out, final], leaf, [dout, dfinal])[0], whole["dv"])
    out, final = linear_attention_fn(q, k, leaf, g, None, state, True)
    of_final, = torch.autograd.grad(final, leaf, dfinal)
    out, final = linear_attention_fn(q, k, leaf, g, None, state, True)
    of_out, = torch.autograd.grad(out, leaf, dout)
    assert torch.allclose(of_final + of_out, whole["dv"], rtol=1e-4, atol=1e-4)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(linear_attention_fn(q, k, leaf, g), leaf, dout, create_graph=True)


# ---- single tokens -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,Hq,Hk,Hv,dk,dv", [(1, 1, 1, 1, 1, 1), (1, 8, 8, 8, 64, 64), (3, 4, 2, 4, 20, 36), (2, 6, 1, 6, 128, 50), (1, 2, 2, 2, 256, 256), (130, 8, 2, 8, 96, 128),
                                              (5, 1, 1, 4, 33, 17), (260, 2, 2, 2, 16, 80)])
def test_step(B, Hq, Hk, Hv, dk, dv, dtype):
    print("CASE step", B, Hq, Hk, Hv, dk, dv, dtype, flush=True)
    H = max(Hq, Hk, Hv)
    for decay in (("none", 0), ("head", 1), ("token", 0), ("token", 1)):
        q, k, v, g, _, normal = inputs(B, 1, Hq, Hk, Hv, dk, dv, dtype, decay, B)
        state = normal(B, H, dk, dv).to(DEV)
        want, size = reference(q, k, v, g, state, dk ** -0.5, [(b, 0, 1) for b in range(B)])
        mine = state.clone()
        out = linear_attention_step_fn(q[:, 0], k[:, 0], v[:, 0], g if g is None or g.dim() == 1 else g[:, 0], mine)
        check("out", out, want["out"][:, 0], size["out"][:, 0], F32, (dk,), 1)
        check("state", mine, want["final"], size["final"], F32, (0,), 1)


def test_step_layouts():
    """States inside a larger pool, whatever is around them left alone; tokens as slices of one projection."""
    B, H, dk, dv = 5, 4, 32, 48
    pool = torch.randn(B, 3, H, dk, dv, device=DEV)
    before = pool.clone()
    both = torch.randn(B, H, 2 * dk + dv, device=DEV)
    q, k, v = both.split([dk, dk, dv], -1)
    g = -torch.rand(H, B, device=DEV).t()
    alone = pool[:, 1].clone()
    want = linear_attention_step_fn(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), alone)
    got = linear_attention_step_fn(q, k, v, g, pool[:, 1])
    assert torch.equal(got, want) and torch.equal(pool[:, 1], alone) and torch.equal(pool[:, ::2], before[:, ::2])
    odd = torch.empty(B * H * dk * dv + 1, device=DEV)[1:].view(B, H, dk, dv).copy_(before[:, 1])
    assert torch.allclose(linear_attention_step_fn(q, k, v, g, odd), want, rtol=1e-5, atol=1e-5) and torch.equal(odd, alone)


def test_prompt_then_tokens():
    """A prompt in two calls and tokens one by one are the whole in one."""
    for dtype in (BF16, F16, F32):
        q, k, v, g, _, normal = inputs(2, 150, 4, 2, 4, 64, 32, dtype, ("token", 1), 9)
        whole, end = linear_attention_fn(q, k, v, g, output_final_state=True)
        part = lambda lo, hi: [t[:, lo:hi] for t in (q, k, v, g)]  # noqa: E731
        a, state = linear_attention_fn(*part(0, 77), output_final_state=True)
        b, state = linear_attention_fn(*part(77, 140), initial_state=state, output_final_state=True)
        outs = [a, b]
        for t in range(140, 150):
            outs.append(linear_attention_step_fn(q[:, t], k[:, t], v[:, t], g[:, t], state)[:, None])
        near = lambda x, y: ((x.double() - y.double()).norm() / y.double().norm()).item()  # noqa: E731
        assert near(torch.cat(outs, 1), whole) <= 2 * HALF[dtype] + 2e-6
        assert near(state, end) <= 3 * 2.0 ** -16


# ---- streams, graphs, repetition -------------------------------------------------------------------------------------------------------

def test_same_bits_every_time():
    q, k, v, g, dout, normal = inputs(2, 700, 6, 2, 6, 64, 48, BF16, ("head", 1))
    first = run_all(q, k, v, g, None, dout, None)
    for _ in range(3):
        again = run_all(q, k, v, g, None, dout, None)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_two_streams_and_graphs():
    """Two graphs of the same call, forward and backward, replayed side by side on their own streams between eager calls: each has its own workspace."""
    sets = []
    for seed in (1, 2):
        q, k, v, g, dout, normal = inputs(1, 1100, 2, 1, 2, 64, 64, BF16, ("token", 1), seed)
        leaves = [t.requires_grad_() for t in (q, k, v, g)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                out, final = linear_attention_fn(*leaves, output_final_state=True)
                torch.autograd.grad(out, leaves, dout)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, final = linear_attention_fn(*leaves, output_final_state=True)
            grads = torch.autograd.grad(out, leaves, dout)
        sets.append((leaves, dout, stream, graph, [out, final, *grads]))
    for turn in range(4):
        wants = []
        for leaves, dout, stream, graph, results in sets:
            with torch.no_grad():
                for t in leaves[:3]:
                    t.copy_(torch.randn_like(t))
            out, final = linear_attention_fn(*leaves, output_final_state=True)
            wants.append([out.detach(), final.detach(), *torch.autograd.grad(out, leaves, dout)])
            for t in results:
                t.detach().fill_(float("nan"))
        torch.cuda.synchronize()
        for _, _, stream, graph, _ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, results), want in zip(sets, wants):
            assert all(torch.equal(a, b) for a, b in zip(results, want)), turn
    state = torch.randn(2, 2, 64, 64, device=DEV)
    token = [torch.randn(2, 2, 64, device=DEV) for _ in range(3)]
    mine, graph = state.clone(), torch.cuda.CUDAGraph()
    linear_attention_step_fn(*token, None, state.clone())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = linear_attention_step_fn(*token, None, mine)
    mine.copy_(state)
    for _ in range(3):
        want = linear_attention_step_fn(*token, None, state)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(mine, state)


@pytest.mark.parametrize("shape", [(1, 70, 2, 1, 2, 65, 64), (2, 70, 2, 2, 2, 64, 129), (1, 129, 1, 1, 1, 200, 33), (1, 65, 2, 2, 1, 128, 96), (1, 40, 1, 1, 3, 48, 80), (1, 70, 2, 1, 2, 9, 11),
                                   (2, 66, 1, 1, 1, 13, 8), (1, 90, 1, 2, 2, 66, 71), (1, 33, 1, 1, 1, 7, 4)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_dimensions_between_the_kernels(shape, dtype):
    """Both sides of the dimensions at which another kernel is taken, with all that the backward can be asked for."""
    print("CASE dimensions", shape, dtype, flush=True)
    B, T, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, dout, normal = inputs(*shape, dtype, ("token", 1), 3)
    state, dfinal = (normal(B, max(Hq, Hk, Hv), dk, dv).to(DEV) for _ in range(2))
    got = run_all(q, k, v, g, state, dout, dfinal)
    want, size = reference(q, k, v, g, state, dk ** -0.5, [(b, 0, T) for b in range(B)], dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], dtype, (dk, dv, 0), T)


def test_far_apart_in_memory():
    """Tokens 2^24 bytes apart, and batches more than 2^31 values apart: the same bits as side by side."""
    q, k, v, g, dout, normal = inputs(2, 40, 2, 2, 2, 32, 16, BF16, ("token", 1), 5)
    want = run_all(q, k, v, g, None, dout, None)
    memory = torch.zeros(2 ** 31 + 2 ** 20, dtype=BF16, device=DEV)
    far = memory.as_strided(k.shape, (2 ** 31 + 64, 80, 32, 1)).copy_(k)
    again = run_all(q, far, v, g, None, dout, None)
    assert far.stride(0) > 2 ** 31 and all(torch.equal(want[n], again[n]) for n in want)
    far = memory.as_strided(v.shape, (40 * 2 ** 23 + 64, 2 ** 23, 16, 1)).copy_(v)
    assert far.stride(1) * 2 == 2 ** 24
    again = run_all(q, k, far, g, None, dout, None)
    assert all(torch.equal(want[n], again[n]) for n in want)
    again = run_all(q, k, v, g, None, memory.as_strided(dout.shape, (40 * 2 ** 23 + 64, 2 ** 23, 16, 1)).copy_(dout), None)
    assert all(torch.equal(want[n], again[n]) for n in want)


def test_a_long_sequence_behind_many_empty_ones():
    """More pieces of states to join than a launch has workgroups; the same bits as of the long sequence alone."""
    q, k, v, g, dout, normal = inputs(1, 5000, 4, 4, 4, 16, 16, BF16, ("token", 1), 9)
    alone = torch.tensor([0, 5000], dtype=torch.int32, device=DEV)
    many = torch.tensor([0] * 70000 + [5000], dtype=torch.int32, device=DEV)
    dfinal = normal(1, 4, 16, 16).to(DEV)
    want = run_all(q, k, v, g, None, dout, dfinal, cu=alone)
    got = run_all(q, k, v, g, None, dout, torch.cat([torch.zeros(69999, 4, 16, 16, device=DEV), dfinal]), cu=many)
    for name in want:
        assert torch.equal(want[name], got[name][-1:] if name == "final" else got[name]), name
    assert not got["final"][:-1].any()


def test_broadcast_inputs_and_gradients():
    """Inputs that repeat one row of memory, and gradients that do (sum().backward()): those of the same values laid out whole."""
    q, k, v, g, dout, normal = inputs(3, 80, 4, 1, 4, 32, 24, BF16, ("head", 1), 11)
    leaf = k[:1].detach().requires_grad_()
    out = linear_attention_fn(q, leaf.expand(3, -1, 4, -1), v, g)
    out.sum().backward()
    whole = k[:1].repeat(3, 1, 4, 1).requires_grad_()
    other = linear_attention_fn(q, whole, v, g)
    assert torch.equal(out, other)
    other.backward(torch.ones_like(other))
    assert torch.equal(leaf.grad, whole.grad.sum((0, 2), keepdim=True))


class Seen(torch.overrides.TorchFunctionMode):
    """A mode that follows operators: the calls then go through Python."""
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_through_python_as_through_the_extension():
    from vmamba_amd.norm import native_stands
    q, k, v, g, dout, normal = inputs(1, 90, 4, 2, 4, 40, 24, BF16, ("token", 1), 13)
    state, dfinal = normal(2, 4, 40, 24).to(DEV), normal(2, 4, 40, 24).to(DEV)
    cu = torch.tensor([3, 50, 85], dtype=torch.int32, device=DEV)
    want = run_all(q, k, v, g, state, dout, dfinal, cu=cu)
    with Seen():
        assert not native_stands(q)
        got = run_all(q, k, v, g, state, dout, dfinal, cu=cu)
    assert all(torch.equal(want[n], got[n]) for n in want)
    token, mine, theirs = (q[0, 0, None], k[0, 0, None], v[0, 0, None], g[0, 0]), state[:1].clone(), state[:1].clone()
    want = linear_attention_step_fn(*token, mine)
    with Seen():
        got = linear_attention_step_fn(*token, theirs)
    assert torch.equal(want, got) and torch.equal(mine, theirs)


@pytest.mark.parametrize("seen", [False, True])
def test_gradients_that_are_refused(seen):
    """Second derivatives, a batch of gradients at once, and saved tensors of which a hook made something else; what a hook brings back whole is taken."""
    import contextlib
    q, k, v, g, dout, normal = inputs(1, 50, 2, 2, 2, 16, 16, F32, ("token", 1), 17)
    want = run_all(q, k, v, g, None, dout, None)
    with Seen() if seen else contextlib.nullcontext():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
        out = linear_attention_fn(*leaves)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out, leaves, dout, create_graph=True)
        out = linear_attention_fn(*leaves)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaves, torch.stack([dout, dout]), is_grads_batched=True)
        with torch.autograd.graph.save_on_cpu():
            out = linear_attention_fn(*leaves)
        for d, name in zip(torch.autograd.grad(out, leaves, dout), ("dq", "dk", "dv", "dg")):
            assert torch.equal(d, want[name])
        for spoil in (lambda t: t.cpu(), lambda t: t[:, :7], lambda t: t.double(), lambda t: t.transpose(0, 1)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil):
                out = linear_attention_fn(*leaves)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(out, leaves, dout)


@pytest.mark.parametrize("seen", [False, True])
def test_step_and_autograd(seen):
    """The state's change is seen by what saved it; inference mode and its tensors are taken."""
    import contextlib
    token = [torch.randn(2, 2, 16, device=DEV) for _ in range(3)]
    state, w = torch.randn(2, 2, 16, 16, device=DEV), torch.randn(2, 2, 16, 16, device=DEV, requires_grad=True)
    with Seen() if seen else contextlib.nullcontext():
        product = state * w
        linear_attention_step_fn(*token, None, state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
        with torch.inference_mode():
            mine = state.clone()
            out = linear_attention_step_fn(*token, None, mine)
        want = linear_attention_step_fn(*token, None, state)
    assert torch.equal(out, want) and torch.equal(mine, state)


def test_capture_beside_an_eager_graph():
    """An eager graph of the same leaves on another stream: the captured call says so before anything of it is recorded; without it the capture goes through."""
    q, k, v, g, dout, normal = inputs(1, 100, 2, 2, 2, 32, 32, BF16, ("token", 1), 19)
    leaves = [t.requires_grad_() for t in (q, k, v, g)]
    stream = torch.cuda.Stream()
    eager = linear_attention_fn(*leaves)
    want = [eager.detach(), *torch.autograd.grad(eager, leaves, dout, retain_graph=True)]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            held = torch.zeros(8, device=DEV)
            with pytest.raises(RuntimeError, match="still lives"):
                linear_attention_fn(*leaves)
            with pytest.raises(RuntimeError, match="still lives"):
                qk_norm_rotate_fn(q, k)
            linear_attention_fn(*[t.detach() for t in leaves])       # (without gradients nothing is in the way)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = linear_attention_fn(*leaves)
        got = [out, *torch.autograd.grad(out, leaves, dout)]
    for _ in range(2):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del held


@pytest.mark.parametrize("decay", [("head", 1), ("token", 1)], ids=["head", "own"])
@pytest.mark.parametrize("shape", [(1, 31, 4, 2, 4, 32, 48), (4, 8, 3, 3, 3, 64, 36), (1, 200, 2, 2, 2, 128, 128), (1, 97, 2, 1, 2, 256, 256), (2, 300, 2, 1, 2, 64, 16)], ids=str)
def test_what_16_bit_inputs_leave_in_32(shape, decay):
    """States and the gradients of states and of single precision decays, of bf16 inputs: three parts of each operand, 24 bits."""
    print("CASE kept", shape, decay, flush=True)
    B, T, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, dout, normal = inputs(*shape, BF16, decay, T + 1)
    state, dfinal = (normal(B, max(Hq, Hk, Hv), dk, dv).to(DEV) for _ in range(2))
    got = run_all(q, k, v, g, state, dout, dfinal)
    want, size = reference(q, k, v, g, state, dk ** -0.5, [(b, 0, T) for b in range(B)], dout, dfinal)
    for name in ("final", "dg", "dstate"):
        check(name, got[name], want[name], size[name], BF16, (dk, dv, B * T if name == "dg" else 0), T, split=2.0 ** -24)


def test_a_learnt_decay_over_many_chunks():
    """One decay for all tokens of a head: what rounding does to it is the same in every chunk.  A sum of 32 maps' tokens in single precision, against 64 bits."""
    gen = torch.Generator().manual_seed(21)
    q, k, v, dout = (torch.randn(8, 784, h, d, generator=gen).to(DEV) for h, d in ((1, 64), (1, 64), (2, 32), (2, 32)))
    g = torch.tensor([-0.004, -0.02], device=DEV)
    got = run_all(q, k, v, g, None, dout, None)["dg"].double()
    at = torch.arange(784, device=DEV, dtype=torch.float64)
    apart = at[:, None] - at[None]
    pairs = (q[:, :, 0].double() @ k[:, :, 0].double().transpose(1, 2).contiguous())[:, None] * (dout.double().transpose(1, 2) @ v.double().permute(0, 2, 3, 1).contiguous())
    terms = pairs * (apart * (apart * g.double()[:, None, None]).clamp(max=0).exp()).tril() * 64 ** -0.5
    want, size = terms.sum((0, 2, 3)), terms.abs().sum((0, 2, 3))
    # of 32-term sums of products, added over 25 chunks and 8 maps; each step's half step at most
    assert bool(((got - want).abs() <= (64 + 32 + 32 + 25 + 8) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 20), (37, 50)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_rows_off_the_grid(dtype, dk, dv):
    """Views that begin one value behind a 16-byte boundary, their rows an odd number of values apart, with NaN all around: the same bits as of copies."""
    q, k, v, g, dout, normal = inputs(2, 77, 2, 2, 2, dk, dv, dtype, ("token", 1), 23)
    want = run_all(q, k, v, g, None, dout, None)

    def off(t):
        B, T, H, d = t.shape
        memory = torch.full((B * T * (H * d + 3) + 9,), float("nan"), dtype=dtype, device=DEV)
        return memory.as_strided(t.shape, (T * (H * d + 3), H * d + 3, d, 1), 1).copy_(t)

    got = run_all(off(q), off(k), off(v), g, None, off(dout), None)
    assert all(torch.equal(want[n], got[n]) for n in want)


@pytest.mark.filterwarnings("ignore")
def test_traced():
    """A traced call is the call, for inputs of other values and sizes too, whatever stands behind it; a token's state is not left to a trace."""
    def layer(q, k, v, g):
        q, k = qk_norm_rotate_fn(q, k)
        out, final = linear_attention_fn(q, k, v, g, output_final_state=True)
        return out + 1, final * 2

    with torch.no_grad():
        q, k, v, g, _, _ = inputs(2, 50, 4, 2, 4, 32, 24, BF16, ("token", 1), 29)
        traced = torch.jit.trace(layer, (q, k, v, g))
        for sizes in ((2, 50), (1, 131)):
            q, k, v, g, _, _ = inputs(*sizes, 4, 2, 4, 32, 24, BF16, ("token", 1), 31)
            assert all(torch.equal(a, b) for a, b in zip(traced(q, k, v, g), layer(q, k, v, g)))
        with pytest.raises(RuntimeError, match="agree"):
            traced(q, k, v[:, :100], g)
        state = torch.zeros(1, 4, 32, 24, device=DEV)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(linear_attention_step_fn, (q[:, 0], k[:, 0], v[:, 0], g[:, 0], state))


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("own", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
def test_a_learnt_decay_without_sequences(own, seen):
    """The gradient of what all tokens of a head share is zero where there are none, not what its memory held before."""
    import contextlib
    for B, T in ((0, 5), (2, 0)):
        q, k, v = (torch.zeros(B, T, 7, 16, device=DEV, dtype=own) for _ in range(3))
        g = torch.full((7,), -0.5, device=DEV, dtype=own, requires_grad=True)
        with Seen() if seen else contextlib.nullcontext():
            out = linear_attention_fn(q, k, v, g)
            dout = torch.zeros_like(out)
            spoiled = [torch.full((7,), float("nan"), device=DEV, dtype=own) for _ in range(64)]    # (what a new tensor of that size is given next)
            del spoiled
            dg, = torch.autograd.grad(out, g, dout)
        assert dg.shape == (7,) and not dg.any(), (B, T)


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("other", [F32, F16], ids=["fp32", "fp16"])
def test_saved_tensors_of_another_type(other, seen):
    """A hook that brings bf16 back as another type: the gradients that come in are bf16 still, and are not read as what they are not."""
    import contextlib
    q, k, v, g, dout, normal = inputs(1, 50, 2, 2, 2, 16, 16, BF16, ("token", 0), 37)
    with Seen() if seen else contextlib.nullcontext():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.to(other)):
            out = linear_attention_fn(*leaves)
            turned = qk_norm_rotate_fn(*leaves[:2])
        with pytest.raises(RuntimeError, match="type"):
            torch.autograd.grad(out, leaves, dout)
        with pytest.raises(RuntimeError, match="type"):
            torch.autograd.grad(turned, leaves[:2], [torch.ones_like(t) for t in turned])


def test_capture_beside_an_eager_graph_through_python():
    """As through the extension: of a mode that follows operators, and of leaves that are not dense, whose copies are no leaves.  Nothing of such a call is launched, so no
    backward comes to it."""
    import contextlib
    import gc
    q, k, v, g, dout, normal = inputs(1, 100, 2, 2, 2, 32, 32, BF16, ("token", 1), 41)
    state, weight = normal(1, 2, 32, 32).to(DEV).transpose(2, 3).requires_grad_(), normal(64).to(DEV)[::2].requires_grad_()
    qg = q.detach().requires_grad_()
    with Seen():
        eager = [linear_attention_fn(qg, k, v, g), linear_attention_fn(q, k, v, g, initial_state=state), *qk_norm_rotate_fn(q, k, weight)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
        held = torch.zeros(8, device=DEV)
        for mode, call in ((Seen, lambda: linear_attention_fn(qg, k, v, g)), (Seen, lambda: qk_norm_rotate_fn(qg, k)),
                           (contextlib.nullcontext, lambda: linear_attention_fn(q, k, v, g, initial_state=state)), (contextlib.nullcontext, lambda: qk_norm_rotate_fn(q, k, weight))):
            with mode(), pytest.raises(RuntimeError, match="still lives"):
                call()
            with mode(), torch.no_grad():
                call()                                               # (without gradients nothing is in the way)
    del eager
    gc.collect()                                                     # (the refusals' tracebacks hold the refused calls)
    # their graph gone, the same leaves are captured, and replayed
    want = linear_attention_fn(q, k, v, g, initial_state=state)
    want = [want.detach(), *torch.autograd.grad(want, state, dout)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = linear_attention_fn(q, k, v, g, initial_state=state)
        got = [out, *torch.autograd.grad(out, state, dout)]
    for _ in range(2):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del held


def quadratic(q, k, v, g, state, scale, pieces):
    """(out, final states) of a batch of one in 64 bits, as sums over the pairs of tokens of each piece and head."""
    H = v.shape[2]
    outs, finals = [], []
    for n, (lo, hi) in enumerate(pieces):
        for h in range(H):
            qh, kh, vh = q[0, lo:hi, h * q.shape[2] // H], k[0, lo:hi, h * k.shape[2] // H], v[0, lo:hi, h]
            G = g[0, lo:hi, h].cumsum(0)
            apart = (G[:, None] - G[None]).masked_fill(~torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=q.device).tril(), -float("inf"))
            end = G[-1] if hi > lo else G.sum()
            outs.append((((qh @ kh.t()) * apart.exp()) @ vh + (qh * G.exp()[:, None]) @ state[n, h]) * scale)
            finals.append((kh * (end - G).exp()[:, None]).t() @ vh + end.exp() * state[n, h])
    rows = [torch.stack(outs[n * H:(n + 1) * H], 1) for n in range(len(pieces))]
    return torch.cat(rows)[None], torch.stack(finals).view(len(pieces), H, q.shape[3], v.shape[3])


@pytest.mark.parametrize("packed", [False, True], ids=["one", "packed"])
@pytest.mark.parametrize("Hk,H,dk,dv", [(1, 1, 64, 64), (2, 2, 128, 128), (1, 2, 192, 256), (1, 1, 130, 96), (1, 3, 80, 144), (2, 2, 33, 200)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_segments_of_states_in_several_pieces(Hk, H, dk, dv, dtype, packed):
    """Sequences that are cut, of heads whose states take more than one workgroup: what comes into a segment is read back by pieces, in either order.  Decays of which
    a segment leaves something; all that is kept in 32 bits comes of operands in three parts."""
    print("CASE pieces", Hk, H, dk, dv, dtype, packed, flush=True)
    lengths = [0, 700, 37, 411, 0, 64, 330] if packed else [1301]
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    T, pieces = starts[-1], list(zip(starts, starts[1:]))
    q, k, v, g, dout, normal = inputs(1, T, Hk, Hk, H, dk, dv, dtype, ("token", 1), 43)
    g = g * 0.05
    state, dfinal = (normal(len(lengths), H, dk, dv).to(DEV) for _ in range(2))
    got = run_all(q, k, v, g, state, dout, dfinal, torch.tensor(starts, dtype=torch.int32, device=DEV) if packed else None)
    both = []
    for size in (False, True):
        of = lambda t: t.double().abs() if size else t.double()  # noqa: E731
        leaves = [t.detach().requires_grad_() for t in (of(q), of(k), of(v), g.double(), of(state))]
        out, final = quadratic(*leaves, dk ** -0.5, pieces)
        grads = torch.autograd.grad((out * of(dout)).sum() + (final * of(dfinal)).sum(), leaves)
        both.append({n: t.detach().cpu() for n, t in zip(("out", "final", "dq", "dk", "dv", "dg", "dstate"), (out, final, *grads))})
    for name in got:
        check(name, got[name], both[0][name], both[1][name], dtype, (dk, dv), max(lengths), split=2.0 ** -24)


def test_what_is_not_dense_may_change_behind_the_forward():
    """Of a state, weights and frequencies that are not dense it is a copy that is kept for the gradients: writing into them later, as a token's step does, changes none."""
    q, k, v, g, dout, normal = inputs(1, 60, 2, 2, 2, 16, 16, F32, ("token", 1), 47)
    state, weight, f = normal(1, 2, 16, 16).to(DEV).transpose(2, 3), normal(32).to(DEV)[::2], torch.rand(16, device=DEV)[::2]
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def both(spoil):
        turned = qk_norm_rotate_fn(*leaves[:2], weight, None, torch.arange(60, device=DEV), f)
        out = linear_attention_fn(*turned, leaves[2], g, initial_state=state)
        if spoil:
            for t in (state, weight, f):
                t.fill_(7.0)
        return torch.autograd.grad(out, leaves, dout)

    assert all(torch.equal(a, b) for a, b in zip(both(False), both(True)))
