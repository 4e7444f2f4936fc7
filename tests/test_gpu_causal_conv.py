"""causal_conv_fn and causal_conv_step_fn against the sums in 64 bits.

y is a sum of width + 1 terms in fp32: off by (width + 4) 2^-24 of the sum of their magnitudes, `size`.  SiLU's slope is at most 1.1 and its own
rounding, like its derivative's, 2^-21 relative to 1 + size; the derivative changes by at most half of what y is off by.  Gradients of the weights add up all tokens: as many
roundings more.  A result is rounded once, by half a step at most: 2^-8 in bf16, 2^-11 in fp16, 2^-24 in fp32."""
import pytest
import torch

from vmamba_amd import causal_conv_fn, causal_conv_step_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def reference(x, weight, bias, state, act, pieces, dout=None, dfinal=None):
    """(results, sizes): out, final and, with dout, dx, dweight, dbias and dstate."""
    W = weight.shape[1]
    x, weight = x.double(), weight.double()
    both = []
    for size in (False, True):
        mag = (lambda t: t.abs()) if size else (lambda t: t)
        w, b = mag(weight), 0 if bias is None else mag(bias.double())
        out, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w[:, 0])
        finals, dstates = [], []
        for n, (k, lo, hi) in enumerate(pieces):
            T = hi - lo
            line = torch.cat([torch.zeros(W - 1, x.shape[2], dtype=x.dtype, device=DEV) if state is None else mag(state[n].double()), mag(x[k, lo:hi])])
            finals.append(line[T:])
            y = b + sum(w[:, j] * line[j:j + T] for j in range(W))
            sig = torch.sigmoid(y)
            out[k, lo:hi] = (1.1 * y if size else y * sig) if act else y
            if dout is None:
                continue
            g = mag(dout[k, lo:hi].double()) * (((1 + y) if size else sig * (1 + y * (1 - sig))) if act else 1)
            dline = torch.zeros_like(line)
            for j in range(W):
                dline[j:j + T] += w[:, j] * g
                dw[:, j] += (g * line[j:j + T]).sum(0)
            db += g.sum(0)
            if dfinal is not None:
                dline[T:] += mag(dfinal[n].double())
            dx[k, lo:hi] = dline[W - 1:]
            dstates.append(dline[:W - 1])
        made = {"out": out, "final": torch.stack(finals)}
        if dout is not None:
            made |= {"dx": dx, "dweight": dw, "dbias": db, "dstate": torch.stack(dstates)}
        both.append(made)
    return both


def check(name, got, want, size, pieces):
    terms = 40 + (sum(hi - lo for _, lo, hi in pieces) if name in ("dweight", "dbias") else 0)
    bound = terms * 2.0 ** -24 * (size + 1e-30) + HALF[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == F16 else 1e-38)     # (fp16's smallest step)
    off = (got.double() - want).abs()
    assert got.shape == want.shape, name
    assert bool((off <= bound).all()), (name, (off / bound).max().item())


def inputs(B, T, dim, W, dtype, wide=False, bias=True, state=True, n_seqs=None, seed=0):
    gen = torch.Generator().manual_seed(seed + T * 7 + dim)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    wd = F32 if wide else dtype
    a = {"x": normal(B, T, dim).to(DEV, dtype), "weight": normal(dim, W).to(DEV, wd), "bias": normal(dim).to(DEV, wd) if bias else None,
         "state": normal(n_seqs or B, W - 1, dim).to(DEV, dtype) if state else None}
    return a, normal(B, T, dim).to(DEV, dtype), normal(n_seqs or B, W - 1, dim).to(DEV, dtype)


def run_all(a, act, dout, dfinal, cu=None):
    leaves = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
    out, final = causal_conv_fn(leaves["x"], leaves["weight"], leaves["bias"], act, leaves["state"], True, cu)
    wanted = {n: t for n, t in leaves.items() if t is not None}
    outs, douts = ([out, final], [dout, dfinal]) if dfinal is not None else ([out], [dout])
    return {"out": out.detach(), "final": final.detach(), **{"d" + n: d for n, d in zip(wanted, torch.autograd.grad(outs, list(wanted.values()), douts))}}


SHAPES = [(1, 1, 1), (2, 2, 3), (1, 3, 8), (2, 5, 9), (3, 37, 64), (1, 65, 100), (2, 130, 515), (1, 300, 7), (5, 8, 1000), (1, 1000, 96)]       # B, T, dim


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences(shape, W, dtype):
    print("CASE causal_conv", shape, W, dtype, flush=True)
    B, T, dim = shape
    act = "silu" if (T + W) % 3 else None
    a, dout, dfinal = inputs(*shape, W, dtype, wide=T % 2 == 0, bias=dim != 100, state=(T + W) % 2 == 0)
    dfinal = dfinal if T % 3 != 2 else None
    got = run_all(a, act, dout, dfinal)
    pieces = [(b, 0, T) for b in range(B)]
    want, size = reference(a["x"], a["weight"], a["bias"], a["state"], act, pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], pieces)


@pytest.mark.parametrize("lengths", [[0, 1, 70, 0, 0, 2, 3, 64, 129, 5, 0], [16, 48, 64, 1, 63], [0, 0], [1] * 40, [1000, 3, 0, 500]], ids=lambda v: str(len(v)) + "x" + str(sum(v)))
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 50)])
def test_packed(lengths, before, behind):
    """Sequences one behind another, empty ones and rows of none before and behind: as each alone, zeros elsewhere."""
    print("CASE causal_conv packed", lengths, before, behind, flush=True)
    T = before + sum(lengths) + behind
    if T == 0:
        T = behind = 5
    starts = [before + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
    a, dout, dfinal = inputs(1, T, 43, 4, F32, n_seqs=len(lengths))
    got = run_all(a, "silu", dout, dfinal, cu)
    pieces = [(0, lo, lo + n) for lo, n in zip(starts, lengths)]
    want, size = reference(a["x"], a["weight"], a["bias"], a["state"], "silu", pieces, dout, dfinal)
    for name in got:
        check(name, got[name], want[name], size[name], pieces)
    for name in ("out", "dx"):
        assert not got[name][0, :before].any() and not got[name][0, starts[-1]:].any(), name
    assert torch.equal(got["final"].double(), want["final"])


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,dim,W", [(1, 1, 2), (3, 7, 4), (2, 8, 3), (5, 100, 4), (1, 1025, 4), (600, 4096, 4), (300, 2047, 3)], ids=str)
def test_step(B, dim, W, dtype):
    print("CASE causal_conv step", B, dim, W, dtype, flush=True)
    act = "silu" if dim % 2 else None
    a, _, _ = inputs(B, 1, dim, W, dtype, wide=B == 5)
    want, size = reference(a["x"], a["weight"], a["bias"], a["state"], act, [(b, 0, 1) for b in range(B)])
    state = a["state"].clone()
    out = causal_conv_step_fn(a["x"][:, 0], state, a["weight"], a["bias"], act)
    check("out", out, want["out"][:, 0], size["out"][:, 0], [(0, 0, 1)])
    assert torch.equal(state.double(), want["final"])


def test_prompt_then_tokens():
    a, _, _ = inputs(3, 40, 70, 4, BF16)
    whole, final = causal_conv_fn(a["x"], a["weight"], a["bias"], "silu", a["state"], True)
    for cut in (1, 2, 3, 33):
        out, state = causal_conv_fn(a["x"][:, :cut], a["weight"], a["bias"], "silu", a["state"], True)
        assert torch.equal(out, whole[:, :cut])
        for t in range(cut, 40):
            out = causal_conv_step_fn(a["x"][:, t], state, a["weight"], a["bias"], "silu")
            assert bool(((out - whole[:, t]).float().abs() <= 2.0 ** -7 * whole[:, t].float().abs() + 1e-5).all())       # (sums in another order: a rounding apart)
        assert torch.equal(state, final)
