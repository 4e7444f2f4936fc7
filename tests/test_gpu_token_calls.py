"""How the selective scan of tokens, the causal convolution, the group norm and the single tokens are called: layouts, empties, streams and graphs, hooks, traces, and a token
mixer made of them, prompt and single tokens, with its gradients."""
import contextlib
import gc

import pytest
import torch

from vmamba_amd import causal_conv_fn, causal_conv_step_fn, group_norm_fn, selective_scan_step_fn, selective_scan_tokens_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Op:
    """One of the operators with its inputs: `args` by name, of which all but `fixed` are differentiable."""
    def __init__(self, name, B, T, dtype, seed=0, state=True, cu=None, dim=40, N=16, G=2):
        gen = torch.Generator().manual_seed(seed * 1000 + T)
        normal = lambda *s, dtype=dtype: torch.randn(*s, generator=gen).to(DEV, dtype)  # noqa: E731
        self.name, n = name, B if cu is None else len(cu) - 1
        self.cu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
        if name == "scan":
            self.args = dict(u=normal(B, T, dim), delta=normal(B, T, dim), A=-torch.exp(normal(dim, N, dtype=F32)), B=normal(B, T, G, N), C=normal(B, T, G, N), D=normal(dim, dtype=F32),
                             z=normal(B, T, dim), delta_bias=normal(dim, dtype=F32), initial_state=normal(n, dim, N, dtype=F32) if state else None)
            self.douts = [normal(B, T, dim), normal(n, dim, N, dtype=F32)]
        elif name == "conv":
            self.args = dict(x=normal(B, T, dim), weight=normal(dim, 4), bias=normal(dim), initial_state=normal(n, 3, dim) if state else None)
            self.douts = [normal(B, T, dim), normal(n, 3, dim)]
        else:
            self.args = dict(x=normal(B, T, dim), weight=normal(dim), bias=normal(dim))
            self.douts = [normal(B, T, dim)]

    def call(self, args):
        if self.name == "scan":
            return selective_scan_tokens_fn(**args, output_final_state=True, cu_seqlens=self.cu)
        if self.name == "conv":
            return causal_conv_fn(**args, activation="silu", output_final_state=True, cu_seqlens=self.cu)
        return (group_norm_fn(**args, num_groups=5, activation="silu"),)

    def leaves(self):
        return {n: None if t is None else t.detach().requires_grad_() for n, t in self.args.items()}

    def run(self, leaves=None, douts=None):
        leaves = leaves or self.leaves()
        outs = self.call(leaves)
        there = {n: t for n, t in leaves.items() if t is not None}
        grads = torch.autograd.grad(outs, list(there.values()), douts or self.douts)
        return {**{f"out{i}": o.detach() for i, o in enumerate(outs)}, **{"d" + n: g for n, g in zip(there, grads)}}


OPS = ["scan", "conv", "norm"]


class Seen(torch.overrides.TorchFunctionMode):
    """A mode that follows operators: the calls then go through Python."""
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def through(seen):
    return Seen() if seen else contextlib.nullcontext()


def same(a, b):
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("name", OPS)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_same_bits_every_time(name, dtype):
    for B, T, dim in ((2, 700, 40), (3, 300, 640)):
        op = Op(name, B, T, dtype, dim=dim)
        first = op.run()
        for _ in range(3):
            same(first, op.run())


@pytest.mark.parametrize("name", OPS)
def test_through_python_as_through_the_extension(name):
    from vmamba_amd.norm import native_stands
    for cu in (None, [3, 50, 50, 85]):
        op = Op(name, 1, 90, BF16, 1, cu=cu)
        want = op.run()
        with Seen():
            assert not native_stands(op.douts[0])
            got = op.run()
        same(want, got)
    with torch.no_grad():
        for mode in (Seen, contextlib.nullcontext):
            with mode():
                assert torch.equal(op.call(op.args)[0], want["out0"])


def steps(B, dim=40, N=16, G=2, dtype=BF16, seed=0):
    scan, conv = Op("scan", B, 1, dtype, seed, dim=dim, N=N, G=G).args, Op("conv", B, 1, dtype, seed, dim=dim).args
    a = {n: scan[n][:, 0] if n in ("u", "delta", "B", "C", "z") else scan[n] for n in scan}
    take_scan = lambda state, **k: selective_scan_step_fn(**{n: t for n, t in a.items() if n != "initial_state"} | k, state=state)  # noqa: E731
    take_conv = lambda state, **k: causal_conv_step_fn(**dict(x=conv["x"][:, 0], weight=conv["weight"], bias=conv["bias"], activation="silu") | k, state=state)  # noqa: E731
    return (take_scan, scan["initial_state"], a), (take_conv, conv["initial_state"], dict(x=conv["x"][:, 0], weight=conv["weight"], bias=conv["bias"]))


@pytest.mark.parametrize("seen", [False, True])
def test_steps_in_places_of_a_larger_memory(seen):
    """States of which only the batch's stride is not dense, and one-token views of longer tensors: the same bits, and nothing else is written."""
    for take, state, a in steps(5):
        mine, memory = state.clone(), torch.full((5, 3, *state.shape[1:]), 7.0, dtype=state.dtype, device=DEV)
        theirs = memory[:, 1]
        theirs.copy_(state)
        wide = {n: torch.cat([t, t, t], -1)[..., t.shape[-1]:2 * t.shape[-1]] for n, t in a.items() if n in ("u", "x", "delta", "z", "B", "C")}
        with through(seen):
            want, got = take(mine), take(theirs, **wide)
        assert torch.equal(want, got) and torch.equal(mine, theirs) and bool((memory[:, ::2] == 7).all())
        for b in (0, 3):                                             # and one sequence alone, whatever its stride
            with through(seen):
                one = take(state[b:b + 1], **{n: t[b:b + 1] for n, t in a.items() if n in wide})
            assert torch.equal(one, want[b:b + 1]) and torch.equal(state[b], mine[b])


@pytest.mark.parametrize("seen", [False, True])
def test_step_and_autograd(seen):
    """The state's change is seen by what saved it; inference mode and its tensors are taken; a batch of none is one."""
    for take, state, a in steps(2):
        w = torch.randn_like(state).requires_grad_()
        with through(seen):
            product = state * w
            take(state)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                product.sum().backward()
            with torch.inference_mode():
                mine = state.clone()
                out = take(mine)
            want = take(state)
            assert torch.equal(out, want) and torch.equal(mine, state)
            none = take(state[:0], **{n: t[:0] for n, t in a.items() if n in ("u", "x", "delta", "z", "B", "C")})
            assert none.shape == want[:0].shape
            with pytest.raises(RuntimeError, match="no gradient"):
                take(state, **{"u" if "u" in a else "x": a["u" if "u" in a else "x"].detach().requires_grad_()})


@pytest.mark.parametrize("name", OPS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [64, 37, 129])
def test_rows_off_the_grid(name, dtype, dim):
    """Views that begin one value behind a 16-byte boundary, their rows an odd number of values apart, with NaN all around: the same bits as of copies."""
    op = Op(name, 2, 77, dtype, dim=dim if name != "norm" else dim // 5 * 5, G=1)
    want = op.run()

    def off(t):
        if t.dim() < 3 or t.dtype != dtype or t.shape[1] != 77:
            return t
        B, T, rest = t.shape[0], t.shape[1], t[0, 0].numel()
        memory = torch.full((B * T * (rest + 3) + 9,), float("nan"), dtype=dtype, device=DEV)
        strides = (T * (rest + 3), rest + 3, 1) if t.dim() == 3 else (T * (rest + 3), rest + 3, t.shape[3], 1)
        return memory.as_strided(t.shape, strides, 1).copy_(t)

    leaves = {n: t if t is None else off(t).detach().requires_grad_() for n, t in op.args.items()}
    same(want, op.run(leaves, [off(d) for d in op.douts]))


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_splits_turned_and_broadcast(name, seen):
    """Parts of one projection, time-first memory, inputs and gradients broadcast over batch or tokens: as their copies, and their leaves' gradients are the sums."""
    op = Op(name, 3, 50, F32)
    for layout in ("split", "time first", "one batch", "one token"):
        made, args = {}, dict(op.args)
        for n, t in op.args.items():
            if t is None or t.dim() < 3 or t.shape[1] != 50:
                continue
            if layout == "split":
                made[n] = torch.cat([t, t], -1).requires_grad_()
                args[n] = made[n][..., t.shape[-1]:]
            elif layout == "time first":
                made[n] = t.transpose(0, 1).contiguous().requires_grad_()
                args[n] = made[n].transpose(0, 1)
            elif layout == "one batch":
                made[n] = t[:1].clone().requires_grad_()
                args[n] = made[n].expand_as(t)
            else:
                made[n] = t[:, :1].clone().requires_grad_()
                args[n] = made[n].expand_as(t)
        douts = [op.douts[0][:, :1].expand_as(op.douts[0]) if layout == "one token" else op.douts[0].transpose(0, 1).contiguous().transpose(0, 1), *op.douts[1:]]
        copies = {n: t if t is None else t.detach().contiguous().requires_grad_() for n, t in args.items()}
        want = op.run(copies, [d.contiguous() for d in douts])
        with through(seen):
            outs = op.call(args)
            grads = dict(zip(made, torch.autograd.grad(outs, list(made.values()), douts)))
        assert all(torch.equal(o, want[f"out{i}"]) for i, o in enumerate(outs)), layout
        for n, g in grads.items():
            whole = torch.autograd.grad(args[n], made[n], want["d" + n], retain_graph=True)[0]
            assert torch.equal(g, whole), (layout, n)


@pytest.mark.parametrize("name", ["scan", "conv"])
def test_memory_far_apart(name):
    """Tokens over 2^24 values apart, memory behind 2^32 bytes: the same bits as of copies."""
    B, T, dim = 2, 70, 24
    op = Op(name, B, T, BF16, dim=dim)
    want = op.run()
    step = 2 ** 24 + 4
    memory = torch.empty(B * T * step, dtype=BF16, device=DEV)                # (4.7 GB, of which only the rows are written)
    args, at = dict(op.args), 0
    for n, t in op.args.items():
        if t is not None and t.dim() >= 3 and t.shape[1] == T:
            inner = (1,) if t.dim() == 3 else (t.shape[3], 1)
            args[n] = memory.as_strided(t.shape, (T * step, step, *inner), at).copy_(t)
            at += 1024
    dout = memory.as_strided(op.douts[0].shape, (T * step, step, 1), at).copy_(op.douts[0])
    far = {n: t if t is None else t.detach().requires_grad_() for n, t in args.items()}
    same(want, op.run(far, [dout, *op.douts[1:]]))


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_nothing_in_it(name, seen):
    """No sequence, no token, packed sequences all empty: states go through, the weights' gradients are zero, not what their memory held before."""
    for B, T, cu in ((0, 5, None), (2, 0, None), (1, 0, [0, 0, 0]), (1, 6, [2, 2, 2, 2])):
        if name == "norm" and cu is not None:
            continue
        op = Op(name, B, T, BF16, cu=cu)
        spoiled = [torch.full_like(t, float("nan")) for t in op.args.values() if t is not None for _ in range(8)]        # (what new tensors of those sizes are given next)
        del spoiled
        with through(seen):
            got = op.run()
        assert got["out0"].shape == op.douts[0].shape and not got["out0"].any()
        for n, t in op.args.items():
            if n == "initial_state":
                assert torch.equal(got["out1"], t) and torch.equal(got["d" + n], op.douts[1])
            else:
                assert got["d" + n].shape == t.shape and not got["d" + n].any(), (n, B, T, cu)


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_which_gradients(name, seen):
    """One leaf at a time, one result at a time: the same bits as with all of them."""
    op = Op(name, 2, 60, BF16)
    want = op.run()
    with through(seen):
        for n, t in op.args.items():
            leaf = t.detach().requires_grad_()
            outs = op.call(op.args | {n: leaf})
            assert torch.equal(torch.autograd.grad(outs, leaf, op.douts)[0], want["d" + n]), n
        zeros = [torch.zeros_like(d) for d in op.douts]
        for i, d in enumerate(op.douts):
            for n in op.args:
                leaf = op.args[n].detach().requires_grad_()
                outs = op.call(op.args | {n: leaf})
                got, = torch.autograd.grad(outs[i], leaf, d, allow_unused=True)
                leaf = op.args[n].detach().requires_grad_()
                full, = torch.autograd.grad(op.call(op.args | {n: leaf}), leaf, [*zeros[:i], d, *zeros[i + 1:]])
                assert torch.equal(got, full), (n, i)
        if "initial_state" in op.args:                               # no optional input at all
            bare = {n: t for n, t in op.leaves().items() if n in ("u", "delta", "A", "B", "C", "x", "weight")}
            outs = op.call(bare)
            torch.autograd.grad(outs[0], list(bare.values()), op.douts[0])


@pytest.mark.parametrize("name", OPS)
def test_two_streams_and_graphs(name):
    """Two graphs of the same call, forward and backward, replayed side by side on their own streams between eager calls: each has its own workspace."""
    sets = []
    for seed in (1, 2):
        op = Op(name, 2, 1100, BF16, seed, dim=80)
        leaves = op.leaves()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                op.run(leaves)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results = op.run(leaves)
        sets.append((op, leaves, stream, graph, results))
    for turn in range(4):
        wants = []
        for op, leaves, stream, graph, results in sets:
            with torch.no_grad():
                for n in ("u", "z", "B", "x", "bias"):
                    if n in leaves:
                        leaves[n].copy_(torch.randn_like(leaves[n]))
            wants.append(op.run(leaves))
            for t in results.values():
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for _, _, stream, graph, _ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, results), want in zip(sets, wants):
            same(results, want)


def test_steps_in_a_graph():
    for take, state, _ in steps(3):
        mine, graph = state.clone(), torch.cuda.CUDAGraph()
        take(state.clone())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = take(mine)
        mine.copy_(state)
        for _ in range(4):
            want = take(state)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(mine, state)


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_capture_beside_an_eager_graph(name, seen):
    """An eager graph of the same leaves on another stream: the captured call says so before anything of it is recorded; without it the capture goes through."""
    op = Op(name, 1, 100, BF16, 3)
    leaves = op.leaves()
    with through(seen):
        eager = op.call(leaves)
        want = [*(e.detach() for e in eager), *torch.autograd.grad(eager, list(leaves.values()), op.douts, retain_graph=True)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
        held = torch.zeros(8, device=DEV)
        with through(seen):
            with pytest.raises(RuntimeError, match="still lives"):
                op.call(leaves)
            op.call({n: t.detach() for n, t in leaves.items()})      # (without gradients nothing is in the way)
    del eager
    gc.collect()                                                     # (the refusals' tracebacks hold the refused calls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream), through(seen):
        outs = op.call(leaves)
        got = [*outs, *torch.autograd.grad(outs, list(leaves.values()), op.douts)]
    for _ in range(2):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del held


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_gradients_that_are_refused(name, seen):
    """Second derivatives, a batch of gradients at once, and saved tensors of which a hook made something else; what a hook brings back whole is taken."""
    op = Op(name, 2, 50, BF16)
    want = op.run()
    with through(seen):
        leaves = op.leaves()
        wanted = list(leaves.values())
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(op.call(leaves), wanted, op.douts, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(op.call(leaves), wanted, [torch.stack([d, d]) for d in op.douts], is_grads_batched=True)
        with torch.autograd.graph.save_on_cpu():
            outs = op.call(leaves)
        for d, n in zip(torch.autograd.grad(outs, wanted, op.douts), leaves):
            assert torch.equal(d, want["d" + n])
        for spoil in (lambda t: t.cpu(), lambda t: t[:1], lambda t: t.double(), lambda t: t.unsqueeze(0), lambda t: t.to(F32), lambda t: t.to(F16)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil):
                outs = op.call(leaves)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(outs, wanted, op.douts)


@pytest.mark.filterwarnings("ignore")
def test_traced():
    """A traced call is the call, for inputs of other values and sizes too, whatever stands behind it."""
    def layer(u, delta, A, B, C, z, x, weight):
        x, last = causal_conv_fn(x, weight, None, "silu", None, True)
        out, final = selective_scan_tokens_fn(u, delta, A, B, C, None, z, output_final_state=True)
        return group_norm_fn(x + out, 5, activation="silu") + 1, final * 2, last

    with torch.no_grad():
        args = lambda B, T, seed: [v for k, v in (Op("scan", B, T, BF16, seed).args | {"x": Op("conv", B, T, BF16, seed).args["x"], "weight": Op("conv", B, 1, BF16).args["weight"]}).items()  # noqa: E731
                                   if k not in ("D", "delta_bias", "initial_state")]
        traced = torch.jit.trace(layer, args(2, 50, 1))
        for sizes in ((2, 50, 2), (1, 131, 3)):
            a = args(*sizes)
            for got, want in zip(traced(*a), layer(*a)):
                assert torch.equal(got, want)
        with pytest.raises(RuntimeError):
            traced(*a[:3], a[3][:, :100], *a[4:])


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("name", ["scan", "conv"])
def test_spoiled_neighbours(name, seen):
    """NaN and infinities in one packed sequence, in the rows of none and in another sequence of a batch stay where they are: all else has the same bits."""
    starts = [5, 70, 70, 103, 190]
    op = Op(name, 1, 200, BF16, cu=starts)
    clean = op.run()
    for value in (float("nan"), float("inf"), -float("inf")):
        args, douts = {n: t if t is None else t.clone() for n, t in op.args.items()}, [d.clone() for d in op.douts]
        for t in [*args.values(), douts[0]]:
            if t.dim() >= 3 and t.shape[1] == 200:
                t[:, :5] = t[:, 190:] = value
                t[:, 70:103] = value
        args["initial_state"][2], douts[1][2] = value, value
        with through(seen):
            got = op.run({n: t.requires_grad_() for n, t in args.items()}, douts)
        for n in got:
            a, b = got[n], clean[n]
            if a.dim() >= 3 and a.shape[1] == 200:
                assert torch.equal(a[:, 5:70], b[:, 5:70]) and torch.equal(a[:, 103:190], b[:, 103:190]), n
                assert not a[:, :5].any() and not a[:, 190:].any(), n
            elif n in ("out1", "dinitial_state"):
                assert all(torch.equal(a[i], b[i]) for i in (0, 1, 3)), n
    op = Op(name, 3, 130, F32)
    clean = op.run()
    args = {n: t.clone() for n, t in op.args.items()}
    for n in ("u", "delta", "z", "B", "C", "x", "initial_state"):
        if n in args:
            args[n][1] = float("nan")
    with through(seen):
        got = op.run({n: t.requires_grad_() for n, t in args.items()})
    for n in got:
        if got[n].shape[0] == 3:
            assert torch.equal(got[n][::2], clean[n][::2]), n


def test_a_spoiled_channel_of_the_norm():
    """NaN in one group of one sample: the other groups and samples have the same bits."""
    for shape in ((3, 200, 40), (3, 40)):
        x = torch.randn(*shape, device=DEV)
        want = group_norm_fn(x, 5)
        for value in (float("nan"), float("inf")):
            y = x.clone()
            y.view(3, -1, 40)[1, 0, 17] = value
            got = group_norm_fn(y, 5).view(3, -1, 5, 8)
            assert torch.equal(got[::2], want.view(3, -1, 5, 8)[::2])
            assert torch.equal(got[1][:, [0, 1, 3, 4]], want.view(3, -1, 5, 8)[1][:, [0, 1, 3, 4]]) and bool(got[1, :, 2].isnan().all())


def test_steps_of_decay_and_gates_out_of_range():
    """Steps, gates and pre-activations far out of exp's range: softplus, SiLU and their slopes have their limits there, not NaN."""
    T, dim, N = 40, 16, 16
    one = torch.ones(1, T, dim, device=DEV)
    B = torch.ones(1, T, 1, N, device=DEV)
    A = -torch.ones(dim, N, device=DEV)
    for raw, gate in ((-200.0, 1.0), (200.0, -200.0), (200.0, 200.0), (1e30, 200.0), (200.0, -1e30), (-3e38, -3e38), (-float("inf"), 2.0)):
        leaves = [(one * 0.5).requires_grad_(), (one * raw).requires_grad_(), A.clone().requires_grad_(), B.clone().requires_grad_(), B.clone().requires_grad_(), (one * gate).requires_grad_()]
        out = selective_scan_tokens_fn(*leaves[:5], None, leaves[5])
        want = 0.5 * max(raw, 0.0) * N * (gate if gate > 100 else 0.0)                  # (a decay of exp(-200) leaves one token's part)
        assert bool((out.double() - want).abs().max() <= 1e-5 * want + 1e-30), (raw, gate)
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
        assert all(bool(g.isfinite().all()) for g in grads), (raw, gate)
    x = torch.tensor([-3e38, -200.0, 200.0, 1e38], device=DEV).view(1, 1, 4).requires_grad_()
    w = torch.tensor([[0.0, 1.0]] * 4, device=DEV)
    out = causal_conv_fn(x, w, None, "silu")
    assert not out[0, 0, :2].any() and torch.equal(out[0, 0, 2:], x[0, 0, 2:])
    assert torch.autograd.grad(out, x, torch.ones_like(out))[0][0, 0].abs().tolist() == pytest.approx([0, 0, 1, 1], abs=1e-30)


@pytest.mark.parametrize("name", ["scan", "conv"])
@pytest.mark.parametrize("places", [[0, 500, 90], [-40, 20, 200], [50, 20, 60], [90, 0], [2 ** 31 - 1, -2 ** 31, 40], [0, 40, 30, 80]], ids=str)
def test_places_that_are_not_places(name, places):
    """Descending places and places out of the tensor are the caller's mistake and have no right result; the calls end, touch nothing but their own memory and leave the sequences in order as they
    are.  (The kernels bring every place into 0..tokens before they use it.)"""
    print("CASE places", name, places, flush=True)
    op = Op(name, 1, 90, F32, cu=places)
    op.run()
    torch.cuda.synchronize()
    good = Op(name, 1, 90, F32, cu=[0, 40, 90])
    first = good.run()
    op.run()
    same(first, good.run())


# ---- together ----------------------------------------------------------------------------------------------------------------------
class Mixer(torch.nn.Module):
    """A token mixer: projection in, causal convolution, selective scan, group norm, projection out."""
    def __init__(self, width, dim, N, groups, dtype):
        super().__init__()
        gen = torch.Generator().manual_seed(11)
        normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.dim, self.N, self.G = dim, N, groups
        self.inner = torch.nn.Parameter((normal(width, 2 * dim) / width ** 0.5).to(DEV, dtype))
        self.taps, self.taps_bias = (torch.nn.Parameter(t.to(DEV, dtype)) for t in (normal(dim, 4) / 2, normal(dim) / 4))
        self.select = torch.nn.Parameter((normal(dim, dim + 2 * groups * N) / dim ** 0.5).to(DEV, dtype))
        self.A, self.D, self.bias = (torch.nn.Parameter(t.to(DEV)) for t in (-torch.exp(normal(dim, N) / 2), normal(dim), normal(dim) - 1))
        self.weight, self.shift = (torch.nn.Parameter(t.to(DEV, dtype)) for t in (1 + normal(dim) / 8, normal(dim) / 8))
        self.outer = torch.nn.Parameter((normal(dim, width) / dim ** 0.5).to(DEV, dtype))

    def split(self, y):
        delta, B, C = y.split([self.dim, self.G * self.N, self.G * self.N], -1)
        return delta, B.unflatten(-1, (self.G, self.N)), C.unflatten(-1, (self.G, self.N))

    def forward(self, x, states=(None, None), cu=None):
        u, z = (x @ self.inner).chunk(2, -1)
        u, taps = causal_conv_fn(u, self.taps, self.taps_bias, "silu", states[0], True, cu)
        delta, B, C = self.split(u @ self.select)
        y, state = selective_scan_tokens_fn(u, delta, self.A, B, C, self.D, z, self.bias, True, states[1], True, cu)
        return group_norm_fn(y.flatten(0, 1), 4, self.weight, self.shift).view_as(y) @ self.outer, taps, state

    @torch.no_grad()
    def step(self, x, taps, state):
        u, z = (x @ self.inner).chunk(2, -1)
        u = causal_conv_step_fn(u, taps, self.taps, self.taps_bias, "silu")
        delta, B, C = self.split(u @ self.select)
        y = selective_scan_step_fn(u, delta, self.A, B, C, state, self.D, z, self.bias)
        return group_norm_fn(y, 4, self.weight, self.shift) @ self.outer


class Plain(Mixer):
    """The same in plain operations."""
    def forward(self, x):
        F = torch.nn.functional
        T = x.shape[1]
        u, z = (x @ self.inner).chunk(2, -1)
        line = F.pad(u, (0, 0, 3, 0))
        u = F.silu(self.taps_bias + sum(self.taps[:, j] * line[:, j:j + T] for j in range(4)))
        delta, B, C = self.split(u @ self.select)
        each = self.dim // self.G
        step = F.softplus(delta + self.bias)
        h, ys = u.new_zeros(x.shape[0], self.dim, self.N), []
        for t in range(T):
            h = torch.exp(step[:, t, :, None] * self.A) * h + (step[:, t] * u[:, t])[..., None] * B[:, t].repeat_interleave(each, 1)
            ys.append((h * C[:, t].repeat_interleave(each, 1)).sum(-1))
        y = (torch.stack(ys, 1) + self.D * u) * F.silu(z)
        y = y.unflatten(-1, (4, -1))                                 # (torch's own group norm of one position has given wrong gradients of its weights here, in 64 bits)
        y = (y - y.mean(-1, keepdim=True)) * (y.var(-1, keepdim=True, correction=0) + 1e-5).rsqrt()
        return (y.flatten(-2) * self.weight + self.shift) @ self.outer


def test_a_mixer_with_its_gradients():
    """All together in single precision against the plain operations in 64 bits, results and the gradients of the input and of every parameter.  Each operator of the chain (products,
    convolution, scan, norm) is off by at most a few hundred roundings of 2^-24 of its own terms; ten of them in a row, each with a growth below 8 of its input's error through norm and scan,
    stay below 2^-24 * 300 * 10 * 8 = 1.4e-3 of the largest value."""
    mixer, plain = Mixer(24, 48, 16, 2, F32), Plain(24, 48, 16, 2, F32).double()
    gen = torch.Generator().manual_seed(2)
    x, dout = (torch.randn(3, 45, 24, generator=gen).to(DEV) for _ in range(2))
    mine, theirs = x.clone().requires_grad_(), x.double().requires_grad_()
    out, want = mixer(mine)[0], plain(theirs)
    out.backward(dout)
    want.backward(dout.double())
    for a, b in ((out, want), (mine.grad, theirs.grad), *((p.grad, q.grad) for p, q in zip(mixer.parameters(), plain.parameters()))):
        assert bool((a.double() - b).abs().max() <= 1.4e-3 * b.abs().max()) and bool(b.abs().max() > 0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_a_mixers_prompt_and_tokens(dtype):
    """Prompts packed, then one token a step of all sequences at once, a captured step among them: as each whole sequence.  In bf16 each of the nine roundings of the chain is half a step,
    2^-8, of values that norm and scan make at most 8 times larger: 0.3 of the largest value at the worst; in single precision the bound above."""
    mixer = Mixer(24, 48, 16, 2, dtype)
    gen = torch.Generator().manual_seed(3)
    lengths, more = [9, 0, 31, 2], 12
    lines = [torch.randn(n + more, 24, generator=gen).to(DEV, dtype) for n in lengths]
    bound = 0.3 if dtype == BF16 else 1.4e-3
    with torch.no_grad():
        whole = [mixer(line[None])[0][0] for line in lines]
        starts = [sum(lengths[:i]) for i in range(5)]
        cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
        out, taps, state = mixer(torch.cat([line[:n] for line, n in zip(lines, lengths)])[None], cu=cu)
        for i, n in enumerate(lengths):
            assert bool(((out[0, starts[i]:starts[i + 1]] - whole[i][:n]).float().abs() <= bound * whole[i].float().abs().max()).all())
        x = torch.empty(4, 24, dtype=dtype, device=DEV)
        held = taps.clone(), state.clone()
        mixer.step(x.zero_(), *held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mixer.step(x, taps, state)
        for t in range(more):
            x.copy_(torch.stack([line[n + t] for line, n in zip(lines, lengths)]))
            if t % 3 == 1:
                got = mixer.step(x, taps, state)
            else:
                graph.replay()
                got = y
            torch.cuda.synchronize()
            for i, n in enumerate(lengths):
                assert bool(((got[i] - whole[i][n + t]).float().abs() <= bound * whole[i].float().abs().max()).all()), (t, i)


@pytest.mark.parametrize("name", ["scan", "conv"])
def test_more_places_than_half_of_what_32_bits_count(name):
    """Over 2^30 sequences of which the last two have tokens: as those two alone."""
    op = Op(name, 1, 90, F32, state=False, cu=[0, 40, 90])
    many = torch.zeros(2 ** 30 + 101, dtype=torch.int32, device=DEV)
    many[-2], many[-1] = 40, 90
    found = []
    for cu in (op.cu, many):
        leaves = {n: t for n, t in op.leaves().items() if t is not None}
        out = selective_scan_tokens_fn(**leaves, cu_seqlens=cu) if name == "scan" else causal_conv_fn(**leaves, activation="silu", cu_seqlens=cu)
        found.append({"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), op.douts[0])))})
    same(*found)
