"""qk_norm_rotate_fn against the definition in 64 bits, forward and backward.

Every value passes a sum of squares of dim terms, a root, two or three products and, turned, two products and a sum with a sine and a cosine (each
good to 2^-22 with the angle's own rounding): (dim / 2 + 40) 2^-24 of the magnitudes that it is a sum of, and the rounding to its type.  A weight's gradient
is a sum of `rows` such terms."""
import pytest
import torch

from vmamba_amd import linear_attention_fn, linear_attention_step_fn, qk_norm_rotate_fn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def define(x, w, positions, frequencies, eps, interleaved, size=False):
    """One side in 64 bits; size: of magnitudes, for the bound."""
    D = x.shape[-1]
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = n if w is None else n * w
    n = n.abs() if size else n
    if positions is None:
        return n
    f = frequencies.double()
    angle = (positions.double()[..., None] * f).flatten(-2) if f.dim() == 2 else positions.double()[..., None] * f
    cos, sin = angle.cos().unsqueeze(-2), angle.sin().unsqueeze(-2)
    R = 2 * f.numel()
    a, b = (n[..., 0:R:2], n[..., 1:R:2]) if interleaved else (n[..., :R // 2], n[..., R // 2:R])
    if size:
        a, b = a + b, a + b
    else:
        a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, n[..., R:]], -1)


def case(B, T, Hq, Hk, D, dtype, wdtype, turned, axes, seed=0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k = ((normal(B, T, h, D) * 2).to(DEV, dtype) for h in (Hq, Hk))
    ws = [None if wdtype is None else (1 + 0.3 * normal(D)).to(DEV, wdtype) for _ in range(2)]
    if not turned:
        return q, k, ws, None, None, normal
    pairs = turned // (2 * axes)
    f = 100000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    at = torch.randint(-50, 2 ** 20, (B, T) if axes == 1 else (B, T, axes), generator=gen)
    return q, k, ws, at.to(DEV), (f if axes == 1 else f.expand(axes, pairs) * torch.arange(1, axes + 1)[:, None]).to(DEV), normal


def check(name, got, want, size, terms):
    off, bound = (got.double() - want).abs(), terms * 2.0 ** -24 * size + HALF[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == F16 else 1e-30)
    assert got.shape == want.shape and bool((off <= bound).all()), (name, (off / bound).max().item())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,D,turned,axes", [
    (1, 1, 1, 1, 64, 64, 1), (2, 7, 4, 2, 128, 128, 1), (1, 33, 3, 1, 32, 32, 2), (3, 5, 6, 6, 64, 48, 2), (1, 300, 2, 2, 256, 256, 1), (2, 9, 5, 1, 80, 40, 1),
    (1, 4, 2, 1, 8, 8, 1), (1, 6, 3, 3, 512, 512, 4), (2, 11, 2, 2, 20, 12, 1), (1, 13, 2, 1, 33, 10, 1), (1, 3, 1, 1, 1, 0, 1), (2, 5, 2, 2, 96, 0, 1), (1, 2, 40, 8, 130, 130, 1),
    (1, 2500, 16, 4, 64, 64, 1)])
def test_against_the_definition(B, T, Hq, Hk, D, turned, axes, interleaved, dtype):
    print("CASE qk_norm", B, T, Hq, Hk, D, turned, axes, interleaved, dtype, flush=True)
    for wdtype in (None, F32) if dtype == F32 else (dtype, F32):
        q, k, ws, at, f, normal = case(B, T, Hq, Hk, D, dtype, wdtype, turned, axes, T)
        leaves = [t for t in (q, k, *ws) if t is not None]
        for t in leaves:
            t.requires_grad_()
        outs = qk_norm_rotate_fn(q, k, *ws, at, f, 1e-5, interleaved)
        douts = [normal(*t.shape).to(DEV, dtype) for t in outs]
        grads = torch.autograd.grad(outs, leaves, douts)
        exact = [t.detach().double().requires_grad_() for t in leaves]
        wd = exact[2:] if wdtype else [None, None]
        wants = [define(x, w, at, f, 1e-5, interleaved) for x, w in zip(exact, wd)]
        dwants = torch.autograd.grad(wants, exact, [d.double() for d in douts])
        for i in range(2):
            with torch.no_grad():
                x, w = exact[i].detach(), None if wd[i] is None else wd[i].detach()
                check("out", outs[i], wants[i], define(x, w, at, f, 1e-5, interleaved, size=True), D / 2 + 40)
                r = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
                back = define(douts[i].double(), None, None if at is None else -at, f, 0.0, interleaved, size=True)         # |turned back|, up to its norm
                back = back * (douts[i].double().square().mean(-1, keepdim=True)).sqrt()
                g = back.abs() * (1 if w is None else w.abs())
                check("dx", grads[i], dwants[i], r * (g + (x * r).abs() * (g * (x * r).abs()).mean(-1, keepdim=True)), 2 * D + 80)
                if w is not None:
                    check("dw", grads[2 + i], dwants[2 + i], (back.abs() * (x * r).abs()).flatten(0, 2).sum(0), D / 2 + 80 + B * T * Hq / 64 + 1100)


def test_differences():
    """Along a weight the result is linear; along x a difference over h is off by h^2."""
    q, k, ws, at, f, normal = case(1, 20, 2, 2, 64, F32, F32, 64, 1)
    leaves = [t.requires_grad_() for t in (q, k, *ws)]
    douts = [normal(1, 20, 2, 64).to(DEV) for _ in range(2)]
    grads = torch.autograd.grad(qk_norm_rotate_fn(*leaves, at, f), leaves, douts)
    for i, leaf in enumerate(leaves):
        along, h = normal(*leaf.shape).to(DEV), 1.0 if i >= 2 else 2.0 ** -7
        values = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * h * along if j == i else 0) for j, t in enumerate(leaves)]
            values.append(sum((o.double() * d.double()).sum().item() for o, d in zip(qk_norm_rotate_fn(*moved, at, f), douts)))
        size = 2 * 2 * 20 * 2 * 64 * 2.0                              # values of unit size, of both sides, with the move
        want = (grads[i].double() * along.double()).sum().item()
        assert abs((values[0] - values[1]) / (2 * h) - want) <= size * (100 * 2.0 ** -24 / h + (4 * h * h if i < 2 else 0))


def test_far_positions():
    """Places of 2^40 and frequencies in single precision: the angle keeps its digits."""
    at = torch.tensor([[0, 1, 2 ** 20 + 1, 2 ** 40 + 12345, -(2 ** 33) - 7]], device=DEV)
    q = torch.randn(1, 5, 2, 64, device=DEV)
    f = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(DEV)
    out, _ = qk_norm_rotate_fn(q, q[:, :, :1], None, None, at, f, 0.0)
    # a product's rounding to 53 bits: 2^40 * 2^-53, next to the results' 2^-22
    assert (out.double() - define(q.double(), None, at, f, 0.0, False)).abs().max().item() <= 8 * (2.0 ** -13 + 2.0 ** -20)
    near, _ = qk_norm_rotate_fn(q[:, :3], q[:, :3, :1], None, None, at[:, :3].int(), f, 0.0)
    assert torch.equal(near, out[:, :3])
    assert (near.double() - define(q[:, :3].double(), None, at[:, :3], f, 0.0, False)).abs().max().item() <= 8 * 2.0 ** -20


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_layouts(dtype):
    """Slices of one projection, transposed heads, odd addresses, positions by broadcast strides: the same values."""
    q, k, ws, at, f, normal = case(2, 12, 4, 2, 64, dtype, F32, 64, 1)
    at = torch.arange(12, device=DEV)
    dq, dk = normal(2, 12, 4, 64).to(DEV, dtype), normal(2, 12, 2, 64).to(DEV, dtype)

    def both(q, k, at, dq, dk):
        leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]
        outs = qk_norm_rotate_fn(*leaves, at, f)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [dq, dk]))

    want = both(q, k, at, dq, dk)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)  # noqa: E731
    first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    joined = torch.cat([q, k, k], 2)
    wide = torch.cat([q, q], -1)
    for args in ((joined[:, :, :4], joined[:, :, 4:6], at, dq, dk), (first(q), first(k), at[None].expand(2, 12), first(dq), first(dk)),
                 (wide[..., 64:], k, at[None].repeat(2, 1).int(), dq, dk.transpose(-1, -2).contiguous().transpose(-1, -2))):
        assert all(torch.equal(a, b) for a, b in zip(both(*args), want))
    for a, b in zip(both(odd(q), odd(k), at, odd(dq), odd(dk)), want):
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() <= 2 * HALF[dtype] + 2e-6
    # each token on its own: the same values as in the batch
    for t in (0, 5, 11):
        alone = qk_norm_rotate_fn(q[:, t:t + 1], k[:, t:t + 1], *ws, at[t:t + 1], f)
        assert torch.equal(alone[0], want[0][:, t:t + 1]) and torch.equal(alone[1], want[1][:, t:t + 1])


def test_rows_without_size():
    """A row of zeros stays zeros (with eps), an infinite or NaN value stays in its row."""
    q, k, ws, at, f, normal = case(1, 6, 2, 2, 64, F32, F32, 64, 1)
    clean = qk_norm_rotate_fn(q, k, *ws, at, f)
    q[0, 2, 1], q[0, 3, 0, 5], q[0, 4, 1, 9] = 0.0, float("nan"), float("inf")
    out, key = qk_norm_rotate_fn(q, k, *ws, at, f)
    assert not out[0, 2, 1].any() and torch.equal(key, clean[1]) and not bool(out[0, 3, 0].isfinite().any())
    for t, h in ((0, 0), (0, 1), (2, 0), (3, 1), (4, 0), (5, 1)):
        assert torch.equal(out[0, t, h], clean[0][0, t, h])


def test_empty():
    for B, T in ((0, 3), (2, 0)):
        q = torch.zeros(B, T, 2, 32, device=DEV, requires_grad=True)
        w = torch.ones(32, device=DEV, requires_grad=True)
        outs = qk_norm_rotate_fn(q, q, w, w, torch.zeros(B, T, dtype=torch.int64, device=DEV), torch.ones(16, device=DEV))
        grads = torch.autograd.grad(outs, [q, w], [torch.ones_like(t) for t in outs])
        assert outs[0].shape == q.shape and grads[0].shape == q.shape and not grads[1].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
def test_an_attention_of_them(dtype):
    """Queries and keys of one projection normalised and rotated, attended to with a learnt gate, then token by token; and trained."""
    gen = torch.Generator().manual_seed(0)
    B, T, H, Hk, D = 2, 100, 4, 2, 32
    normal = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    qkv = normal(B, T, (H + 2 * Hk) * D).to(dtype).requires_grad_()
    gate = (-torch.nn.functional.softplus(normal(B, T, H) - 2)).requires_grad_()
    wq, wk = (1 + 0.1 * normal(D)).requires_grad_(), (1 + 0.1 * normal(D)).requires_grad_()
    f = 10000.0 ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2))

    def layer(qkv, gate, wq, wk, at, **more):
        q, k, v = qkv.unflatten(-1, (-1, D)).split([H, Hk, Hk], -2)
        q, k = qk_norm_rotate_fn(q, k, wq, wk, at, f)
        return linear_attention_fn(q, k, v, gate, **more)

    at = torch.arange(T, device=DEV)
    out, state = layer(qkv, gate, wq, wk, at, output_final_state=True)
    dout = normal(*out.shape).to(dtype)
    grads = torch.autograd.grad(out, [qkv, gate, wq, wk], dout)
    # the same in 64 bits, as one matrix of weights
    exact = [t.detach().double().requires_grad_() for t in (qkv, gate, wq, wk)]
    q, k, v = exact[0].unflatten(-1, (-1, D)).split([H, Hk, Hk], -2)
    q, k = (define(x, w, at, f, 1e-6, False) for x, w in ((q, exact[2]), (k, exact[3])))
    G = exact[1].cumsum(1)
    decay = (G[:, :, None] - G[:, None]).masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1)[None, :, :, None], -1e30).exp()     # (B, t, s, H)
    weights = (q[:, :, None] * k.repeat_interleave(2, 2)[:, None]).sum(-1) * decay * D ** -0.5
    want = (weights[..., None] * v.repeat_interleave(2, 2)[:, None]).sum(2)
    dwant = torch.autograd.grad(want, exact, dout.double())
    near = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
    # in norm: q, k, the weights or states and the result are rounded once each on the way, and as many gradients
    assert near(out, want) <= 4 * HALF[dtype] + 4e-6
    for a, b in zip(grads, dwant):
        assert near(a, b) <= 8 * HALF[dtype] + 8e-6
    with torch.no_grad():
        part, carried = layer(qkv[:, :90], gate[:, :90], wq, wk, at[:90], output_final_state=True)
        for t in range(90, T):
            q, k, v = qkv[:, t:t + 1].unflatten(-1, (-1, D)).split([H, Hk, Hk], -2)
            q, k = qk_norm_rotate_fn(q, k, wq, wk, at[t:t + 1], f)
            token = linear_attention_step_fn(q[:, 0], k[:, 0], v[:, 0], gate[:, t], carried)
            assert near(token, out[:, t]) <= 3 * HALF[dtype] + 4e-6
        assert near(carried, state) <= 2.0 ** -13


def test_graph():
    """Forward and backward captured, replayed between eager calls with other inputs."""
    q, k, ws, at, f, normal = case(2, 64, 8, 2, 64, BF16, F32, 64, 1)
    leaves = [t.requires_grad_() for t in (q, k, *ws)]
    douts = [normal(*t.shape).to(DEV, BF16) for t in (q, k)]

    def step():
        outs = qk_norm_rotate_fn(*leaves, at, f)
        return [*outs, *torch.autograd.grad(outs, leaves, douts)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
        want = step()
        for t in held:
            t.detach().fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


class Seen(torch.overrides.TorchFunctionMode):
    """A mode that follows operators: the calls then go through Python."""
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("seen", [False, True])
def test_through_python_and_what_is_refused(seen):
    """The Python path gives the extension's bits; second derivatives, batches of gradients and saved tensors of which a hook made something else are refused."""
    import contextlib
    q, k, ws, at, f, normal = case(2, 33, 4, 2, 40, BF16, F32, 32, 2)
    douts = [normal(*t.shape).to(DEV, BF16) for t in (q, k)]

    def step(**more):
        leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]
        outs = qk_norm_rotate_fn(*leaves, at, f)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, **{"grad_outputs": douts} | more))

    want = step()
    with Seen() if seen else contextlib.nullcontext():
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
        with pytest.raises(RuntimeError, match="differentiable once"):
            step(create_graph=True)
        with pytest.raises(RuntimeError):
            step(grad_outputs=[torch.stack([t, t]) for t in douts], is_grads_batched=True)
        with torch.autograd.graph.save_on_cpu():
            assert all(torch.equal(a, b) for a, b in zip(step(), want))
        for spoil in (lambda t: t.cpu(), lambda t: t[:, :7] if t.dim() > 2 else t, lambda t: t.double()):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil), pytest.raises(RuntimeError):
                step()


def test_one_gradient_alone():
    """Of queries alone, of a weight alone, and of one output's gradient alone."""
    q, k, ws, at, f, normal = case(2, 20, 4, 2, 32, F32, F32, 32, 1)
    dq, dk = (normal(*t.shape).to(DEV) for t in (q, k))
    leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]
    outs = qk_norm_rotate_fn(*leaves, at, f)
    whole = torch.autograd.grad(outs, leaves, [dq, torch.zeros_like(dk)], retain_graph=True)
    alone = torch.autograd.grad(outs[0], leaves, dq, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, alone))
    for i, leaf in enumerate(leaves):
        args = [t.detach() for t in (q, k, *ws)]
        args[i] = leaf
        out = qk_norm_rotate_fn(*args, at, f)
        assert torch.equal(torch.autograd.grad(out[0] if i in (0, 2) else out[1], leaf, dq if i in (0, 2) else dk)[0],
                           torch.autograd.grad(outs, leaf, [dq, dk], retain_graph=True)[0])


def test_more_rows_than_a_launch_has_workgroups():
    """2^26 and some tokens, 16 to a workgroup's round: the last ones as they come alone."""
    T = 2 ** 26 + 1000
    q = torch.zeros(1, T, 1, 8, dtype=BF16, device=DEV)
    q[:, -3000:] = torch.randn(1, 3000, 1, 8, device=DEV)
    weight = torch.randn(8, device=DEV)
    outs = qk_norm_rotate_fn(q, q, weight, weight)
    alone = qk_norm_rotate_fn(q[:, -3000:], q[:, -3000:], weight, weight)
    for out, want in zip(outs, alone):
        assert torch.equal(out[:, -3000:], want) and not out[:, :-3000].any()
