"""A selective scan of token sequences with its short causal convolution -- for prompts, for training and for single tokens -- and the group norm
of channel-last activations, as cases that can be timed.

A case is a plain dict; ``prepare`` makes what a program holds before the call, ``run`` is one pass: the operators' plain forms in
elementary torch operations, or, where ``own`` is true, the package's operators; ``exact`` is the definition in 64 bits.

  convolution   y_t = act(bias + sum_j weight[j] x_(t - width + 1 + j)), each channel for itself, the state being the last width - 1 inputs
  scan          h_t = exp(step_t A) h_(t-1) + step_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t),   step = softplus(delta + bias), for each channel
  group norm    y = act((x - mean) / sqrt(var + eps) * weight + bias), mean and var over the positions and a group's channels of one sample
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_CHUNK = 64
_EPS = 1e-5


def _conv(name, kind, dtype, batch, tokens, dim, width, silu=True, state=False, sequences=0):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, tokens=tokens, dim=dim, width=width, silu=silu, state=state, sequences=sequences)


def _scan(name, kind, dtype, batch, tokens, dim, dstate, groups=1, gate=True, state=False, sequences=0):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, tokens=tokens, dim=dim, dstate=dstate, groups=groups, gate=gate, state=state, sequences=sequences)


def _norm(name, kind, dtype, batch, positions, channels, groups, silu):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, positions=positions, channels=channels, groups=groups, silu=silu)


def listed():
    return [
        # The convolution of one short prompt of an online request, its state kept for the tokens that follow: latency counts.
        _conv("conv_37_b1_bf16", "conv", "bf16", 1, 37, 1024, 4, state=True),
        # Training of a language model's layer: forward and all gradients, sequences of one batch.
        _conv("conv_train_4096_b8_bf16", "conv_train", "bf16", 8, 4096, 2048, 4),
        # One token of one request in half precision.
        _conv("conv_step_b1_fp16", "conv_step", "fp16", 1, 1, 1536, 4),
        # One token for each of many requests.
        _conv("conv_step_b512_bf16", "conv_step", "bf16", 512, 1, 4096, 4),
        # Prompts of different lengths one behind another, an empty one among them, each with a state from before.
        _scan("scan_packed_bf16", "scan", "bf16", 1, 12011, 1536, 16, state=True, sequences=16),
        # One long document: the sequence itself has to fill the chip.
        _scan("scan_32768_b1_bf16", "scan", "bf16", 1, 32768, 2048, 16, state=True),
        # Training of a language model's layer.
        _scan("scan_train_2048_b4_bf16", "scan_train", "bf16", 4, 2048, 2048, 16),
        # Training on the tokens of 28 x 28 maps in single precision, four groups of channels with keys of their own, no gate.
        _scan("scan_train_784_b8_fp32", "scan_train", "fp32", 8, 784, 768, 8, groups=4, gate=False),
        # One token of one request: latency.
        _scan("scan_step_b1_bf16", "scan_step", "bf16", 1, 1, 1536, 16),
        # One token for each of many requests: the states pass through memory once.
        _scan("scan_step_b256_fp16", "scan_step", "fp16", 256, 1, 4096, 16),
        # Groups of each token behind a mixer of tokens, in training.
        _norm("norm_train_tokens_bf16", "norm_train", "bf16", 8192, 1, 2048, 16, False),
        # Feature maps of 56 x 56 with their activation, few channels to a group.
        _norm("norm_56x56_b32_fp16", "norm", "fp16", 32, 3136, 192, 32, True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for c in listed():
        w, key = work(c), (c["kind"].split("_")[0], c["kind"].endswith("step"))
        old = most.get(key, (0, 0))
        most[key] = max(old[0], w["bytes"]), max(old[1], w["flops"])
    while True:
        kind = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan", "scan_train", "scan_train", "scan_step", "norm", "norm_train"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        batch, tokens = _between(rng, 1, 64), _between(rng, 1, 32768)
        dim = rng.choice([64, 96, 192, 200, 384, 520, 768, 1000, 1024, 1536, 2048, 2560, 4096])
        if kind.endswith("step"):
            batch, tokens = _between(rng, 1, 512), 1
        packed = rng.randint(2, 40) if rng.random() < 0.3 and not kind.endswith("step") else 0
        if packed:
            batch, tokens = 1, max(tokens, 4 * packed)
        if kind.startswith("conv"):
            case = _conv(None, kind, dtype, batch, tokens, dim - rng.choice([0, 0, 0, 1, 6]), rng.choice([2, 3, 4, 4]), rng.random() < 0.8, rng.random() < 0.5, packed)
        elif kind.startswith("scan"):
            case = _scan(None, kind, dtype, batch, tokens, dim, rng.choice([1, 4, 8, 12, 16, 16, 16, 32, 64]), rng.choice([1, 1, 2, 4]), rng.random() < 0.7, rng.random() < 0.5, packed)
        else:
            positions = rng.choice([1, 1, _between(rng, 1, 65536)])
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            case = _norm(None, kind, dtype, _between(rng, 1, 8192 if positions == 1 else 64), positions, groups * rng.choice([1, 3, 4, 6, 8, 16, 20, 32, 64, 128]), groups, rng.random() < 0.5)
            if case["positions"] * (case["channels"] // groups) < 8:       # (statistics of a few values say nothing)
                continue
        del case["name"]
        limit = most[(kind.split("_")[0], kind.endswith("step"))]
        w = work(case)
        if w["bytes"] <= limit[0] and w["flops"] <= limit[1]:
            return case


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _lengths(case):
    """Lengths of the packed sequences: skewed, an empty one and a single token among them where there are several."""
    rng = random.Random(case["tokens"] * 64 + case["sequences"])
    n, total = case["sequences"], case["tokens"]
    fixed = [0, 1] if n > 3 and total > 8 else []
    shares = [rng.random() ** 2 + 0.02 for _ in range(n - len(fixed))]
    left = total - sum(fixed)
    lengths = [int(left * s / sum(shares)) for s in shares]
    lengths[0] += left - sum(lengths)
    lengths += fixed
    rng.shuffle(lengths)
    return lengths


def prepare(case, seed):
    dev, dtype = "cuda", _DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=dev, generator=gen)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, device=dev, generator=gen)  # noqa: E731
    s, kind = {"case": case}, case["kind"]
    if kind.startswith("norm"):
        B, P, C = case["batch"], case["positions"], case["channels"]
        shape = (B, C) if P == 1 else (B, P, C)
        s["x"] = (normal(*shape) * 1.5 + 0.5 * normal(C)).to(dtype)
        s["weight"], s["bias"] = (1 + 0.2 * normal(C)).to(dtype), (0.2 * normal(C)).to(dtype)
        if kind == "norm_train":
            s["dout"] = normal(*shape).to(dtype)
        return s
    B, T, D = case["batch"], case["tokens"], case["dim"]
    N = case["sequences"] or B
    middle = () if kind.endswith("step") else (T,)
    if case["sequences"]:
        lengths = _lengths(case)
        s["longest"] = max(lengths)
        s["cu_seqlens"] = torch.tensor([sum(lengths[:i]) for i in range(N + 1)], device=dev, dtype=torch.int32)
    with_state = case["state"] or kind.endswith("step")
    if kind.startswith("conv"):
        W = case["width"]
        s["x"] = normal(B, *middle, D).to(dtype)
        bound = W ** -0.5
        s["weight"], s["bias"] = (bound * (2 * uniform(D, W) - 1)).to(dtype), (bound * (2 * uniform(D) - 1)).to(dtype)
        s["state"] = normal(N, W - 1, D).to(dtype) if with_state else None
        if kind == "conv_train":
            s["dout"] = normal(B, T, D).to(dtype)
        return s
    G, S = case["groups"], case["dstate"]
    s["u"] = normal(B, *middle, D).to(dtype)
    s["z"] = normal(B, *middle, D).to(dtype) if case["gate"] else None
    # what projections of u leave: the step's offset sets steps of 0.001 to 0.1
    s["delta"] = (0.7 * normal(B, *middle, D)).to(dtype)
    step = torch.exp(uniform(D) * math.log(100.0) + math.log(0.001))
    s["delta_bias"] = step + torch.log(-torch.expm1(-step))
    s["A"] = -torch.arange(1, S + 1, device=dev, dtype=torch.float32) * torch.exp(0.1 * normal(D, S))
    s["B"], s["C"] = normal(B, *middle, G, S).to(dtype), normal(B, *middle, G, S).to(dtype)
    s["D"] = 1 + 0.1 * normal(D)
    s["state"] = normal(N, D, S) if with_state else None
    if kind == "scan_train":
        s["dout"] = normal(B, T, D).to(dtype)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _silu(x):
    return x * torch.sigmoid(x)


def _softplus(x):
    return torch.logaddexp(x, torch.zeros((), device=x.device))


def _apart(s):
    """Gather from the packed tokens to one sequence a row, zeros behind it, and back: two functions."""
    cu, T = s["cu_seqlens"].long(), s["case"]["tokens"]
    at = cu[:-1, None] + torch.arange(s["longest"], device=cu.device)
    inside = at < cu[1:, None]
    token = torch.arange(T, device=cu.device)
    which = torch.searchsorted(cu, token, right=True) - 1
    rows = lambda t: torch.where(inside.view(*inside.shape, *(1,) * (t.dim() - 2)), t[0][at.clamp(max=T - 1)], 0)  # noqa: E731
    return rows, lambda t: t[which, token - cu[which]][None]


def _plain_conv(s):
    case = s["case"]
    dtype, W = _DTYPES[case["dtype"]], case["width"]
    train = case["kind"] == "conv_train"
    names = [n for n in ("x", "weight", "bias", "state") if s[n] is not None]
    leaves = {n: s[n].detach().float().requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        x, (rows, back) = leaves["x"], _apart(s) if case["sequences"] else (None, None)
        lengths = torch.diff(s["cu_seqlens"].long()) if rows else torch.full((x.shape[0],), x.shape[1], device=x.device)
        x = rows(x) if rows else x
        before = leaves["state"] if "state" in leaves else x.new_zeros(x.shape[0], W - 1, x.shape[2])
        padded = torch.cat([before, x], 1)
        y = leaves["bias"] + sum(leaves["weight"][:, j] * padded[:, j:j + x.shape[1]] for j in range(W))
        y = _silu(y) if case["silu"] else y
        out = (back(y) if back else y).to(dtype)
        if not train:
            last = lengths[:, None] + torch.arange(W - 1, device=x.device)
            return [out, padded[torch.arange(x.shape[0], device=x.device)[:, None], last].to(dtype)]
        grads = torch.autograd.grad(out, list(leaves.values()), s["dout"])
    return [out.detach()] + [d.to(dtype) for d in grads]


def _plain_conv_step(s):
    case = s["case"]
    window = torch.cat([s["state"], s["x"][:, None]], 1)
    y = s["bias"].float() + (window.float() * s["weight"].float().t()).sum(1)
    s["state"].copy_(window[:, 1:])
    return [(_silu(y) if case["silu"] else y).to(s["x"].dtype), s["state"]]


def _scanned(u, step, A, B, C, state):
    """(C . h of all tokens, final state) of (R, T, D) in single precision: all chunks at once, token by token within them."""
    R, T, D = u.shape
    n = max(1, -(-T // _CHUNK))
    cut = lambda t: torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, n * _CHUNK - T)).unflatten(1, (n, _CHUNK))  # noqa: E731
    per = D // B.shape[2]
    step, fed, B, C = cut(step), cut(step * u), cut(B), cut(C)
    spread = lambda t, i: t[:, :, i].repeat_interleave(per, 2)  # noqa: E731 -- (R, n, D, N)
    zero = torch.zeros(R, n, D, A.shape[1], device=u.device)
    turn = lambda h, i: torch.exp(step[:, :, i, :, None] * A) * h + fed[:, :, i, :, None] * spread(B, i)  # noqa: E731
    h = zero
    for i in range(_CHUNK):
        h = turn(h, i)
    whole = torch.exp(step.sum(2)[..., None] * A)
    enters = [zero[:, 0] if state is None else state]
    for c in range(n):
        enters.append(whole[:, c] * enters[-1] + h[:, c])
    h, ys = torch.stack(enters[:-1], 1), []
    for i in range(_CHUNK):
        h = turn(h, i)
        ys.append((h * spread(C, i)).sum(-1))
    return torch.stack(ys, 2).flatten(1, 2)[:, :T], enters[-1]


def _plain_scan(s):
    case = s["case"]
    dtype, train = _DTYPES[case["dtype"]], case["kind"] == "scan_train"
    names = [n for n in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state") if s[n] is not None]
    leaves = {n: s[n].detach().float().requires_grad_(train) for n in names}
    with torch.set_grad_enabled(train):
        step = _softplus(leaves["delta"] + leaves["delta_bias"])
        u, B, C = leaves["u"], leaves["B"], leaves["C"]
        rows, back = _apart(s) if case["sequences"] else (lambda t: t, lambda t: t)
        y, final = _scanned(rows(u), rows(step), leaves["A"], rows(B), rows(C), leaves.get("state"))
        y = back(y) + leaves["D"] * u
        out = (y * _silu(leaves["z"]) if case["gate"] else y).to(dtype)
        if not train:
            return [out, final]
        grads = torch.autograd.grad(out, list(leaves.values()), s["dout"])
    return [out.detach()] + [d.to(s[n].dtype) for n, d in zip(names, grads)]


def _plain_scan_step(s):
    case = s["case"]
    per = case["dim"] // case["groups"]
    step = _softplus(s["delta"].float() + s["delta_bias"])
    B, C = s["B"].float().repeat_interleave(per, 1), s["C"].float().repeat_interleave(per, 1)
    u = s["u"].float()
    s["state"].mul_(torch.exp(step[..., None] * s["A"])).add_((step * u)[..., None] * B)
    y = (s["state"] * C).sum(-1) + s["D"] * u
    return [(y * _silu(s["z"].float()) if case["gate"] else y).to(s["u"].dtype), s["state"]]


def _plain_norm(s):
    case = s["case"]
    dtype, train = _DTYPES[case["dtype"]], case["kind"] == "norm_train"
    leaves = [s[n].detach().float().requires_grad_(train) for n in ("x", "weight", "bias")]
    with torch.set_grad_enabled(train):
        x = leaves[0].reshape(case["batch"], case["positions"], case["groups"], -1)
        centred = x - x.mean((1, 3), keepdim=True)
        normal = centred / (centred.square().mean((1, 3), keepdim=True) + _EPS).sqrt()
        y = normal.reshape(s["x"].shape) * leaves[1] + leaves[2]
        out = (_silu(y) if case["silu"] else y).to(dtype)
        if not train:
            return [out]
        grads = torch.autograd.grad(out, leaves, s["dout"])
    return [out.detach()] + [d.to(dtype) for d in grads]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, state["case"], kind)
    return {"conv": _plain_conv, "conv_train": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_train": _plain_scan, "scan_step": _plain_scan_step,
            "norm": _plain_norm, "norm_train": _plain_norm}[kind](state)


def _own(s, case, kind):
    from vmamba_amd import causal_conv_fn, causal_conv_step_fn, group_norm_fn, selective_scan_step_fn, selective_scan_tokens_fn
    act = "silu" if case.get("silu") else None
    if kind == "conv_step":
        return [causal_conv_step_fn(s["x"], s["state"], s["weight"], s["bias"], act), s["state"]]
    if kind == "scan_step":
        return [selective_scan_step_fn(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], s["D"], s["z"], s["delta_bias"]), s["state"]]
    if kind == "norm":
        return [group_norm_fn(s["x"], case["groups"], s["weight"], s["bias"], _EPS, act)]
    if kind == "conv":
        return list(causal_conv_fn(s["x"], s["weight"], s["bias"], act, initial_state=s["state"], output_final_state=True, cu_seqlens=s.get("cu_seqlens")))
    names = {"conv_train": ("x", "weight", "bias", "state"), "norm_train": ("x", "weight", "bias")}.get(kind, ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"))
    if kind == "scan":
        a = s
    else:
        a = {n: s[n].detach().requires_grad_() if s[n] is not None else None for n in names}
    if kind == "conv_train":
        out = causal_conv_fn(a["x"], a["weight"], a["bias"], act, initial_state=a["state"], cu_seqlens=s.get("cu_seqlens"))
    elif kind == "norm_train":
        out = group_norm_fn(a["x"], case["groups"], a["weight"], a["bias"], _EPS, act)
    else:
        out = selective_scan_tokens_fn(a["u"], a["delta"], a["A"], a["B"], a["C"], a["D"], a["z"], a["delta_bias"], initial_state=a["state"],
                                       output_final_state=kind == "scan", cu_seqlens=s.get("cu_seqlens"))
        if kind == "scan":
            return list(out)
    return [out.detach()] + list(torch.autograd.grad(out, [t for t in a.values() if t is not None], s["dout"]))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
    e, B, kind = _SIZE[case["dtype"]], case["batch"], case["kind"]
    train = kind.endswith("train")
    if kind.startswith("norm"):
        values = B * case["positions"] * case["channels"]
        return {"bytes": values * e * (4 if train else 2), "flops": values * (24 if train else 10)}     # x and y; dy and dx (x stays at hand)
    T, D = case["tokens"], case["dim"]
    values, N = B * T * D, case["sequences"] or B
    if kind.startswith("conv"):
        W = case["width"]
        states = N * (W - 1) * D * e
        kept = 2 * states if kind == "conv_step" else states * (2 if train else 1) * int(case["state"]) + states * int(kind == "conv")
        return {"bytes": values * e * (4 if train else 2) + kept + (2 if train else 1) * D * (W + 1) * e, "flops": values * (2 * W + 4) * (3 if train else 1)}
    G, S, gates = case["groups"], case["dstate"], int(case["gate"])
    states = 4 * N * D * S
    inputs = e * (values * (2 + gates) + 2 * B * T * G * S) + 4 * D * (S + 2)
    flops = values * (7 * S + 12)
    if kind == "scan_step":
        return {"bytes": inputs + values * e + 2 * states, "flops": flops}
    if train:                                             # the inputs once, y, its gradient and theirs
        return {"bytes": 2 * inputs + 2 * values * e + 2 * states * int(case["state"]), "flops": 3 * flops}
    return {"bytes": inputs + values * e + states * (1 + int(case["state"])), "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _act(y, silu):
    """(act(y), its derivative)."""
    if not silu:
        return y, torch.ones_like(y)
    sig = 1 / (1 + torch.exp(-y))
    return y * sig, sig * (1 + y * (1 - sig))


def _pieces(case):
    """(batch, start, end) of each sequence."""
    if not case["sequences"]:
        return [(b, 0, case["tokens"]) for b in range(case["batch"])]
    lengths = _lengths(case)
    ends = [sum(lengths[:i + 1]) for i in range(len(lengths))]
    return [(0, end - n, end) for n, end in zip(lengths, ends)]


def _exact_conv(s, case):
    W, train = case["width"], case["kind"] == "conv_train"
    x, w, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    out, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    finals, dstates = [], []
    for n, (b, lo, hi) in enumerate(_pieces(case)):
        T = hi - lo
        line = torch.zeros(T + W - 1, x.shape[2], dtype=torch.float64, device=x.device)
        if s["state"] is not None:
            line[:W - 1] = s["state"][n].double()
        line[W - 1:] = x[b, lo:hi]
        finals.append(line[T:].clone())
        if T == 0:
            dstates.append(torch.zeros_like(line))
            continue
        window = line.unfold(0, W, 1)                      # (T, D, W)
        y, slope = _act((window * w).sum(-1) + bias, case["silu"])
        out[b, lo:hi] = y
        if train:
            d = s["dout"][b, lo:hi].double() * slope
            db += d.sum(0)
            dw += (window * d[..., None]).sum(0)
            dline = torch.zeros_like(line)
            for t in range(W):
                dline[t:t + T] += d * w[:, t]
            dx[b, lo:hi] = dline[W - 1:]
            dstates.append(dline[:W - 1])
    if not train:
        return [out, torch.stack(finals)]
    return [out, dx, dw, db] + ([torch.stack(dstates)] if s["state"] is not None else [])


def _exact_scan(s, case):
    train, G, S, D = case["kind"] == "scan_train", case["groups"], case["dstate"], case["dim"]
    dev, f64 = s["u"].device, torch.float64
    pieces = _pieces(case)
    lengths = [hi - lo for _, lo, hi in pieces]
    R, T = len(pieces), max(lengths)

    def lined(t):                                          # tokens in front, so that a step of all sequences is a slice
        made = torch.zeros(T, R, *t.shape[2:], dtype=f64, device=dev)
        for r, (b, lo, hi) in enumerate(pieces):
            made[:hi - lo, r] = t[b, lo:hi].double()
        return made

    def unlined(t):
        made = torch.zeros(case["batch"], case["tokens"], *t.shape[2:], dtype=f64, device=dev)
        for r, (b, lo, hi) in enumerate(pieces):
            made[b, lo:hi] = t[:hi - lo, r]
        return made

    group = torch.arange(D, device=dev) // (D // G)
    A, skip = s["A"].double(), s["D"].double()
    u, raw = lined(s["u"]), lined(s["delta"]) + s["delta_bias"].double()
    alive = torch.arange(T, device=dev)[:, None] < torch.tensor(lengths, device=dev)
    step = torch.where(alive[..., None], torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30)))), 0)
    B, C = lined(s["B"]), lined(s["C"])
    gate, slope = _act(lined(s["z"]), True) if case["gate"] else (torch.ones_like(u), None)
    h = torch.zeros(R, D, S, dtype=f64, device=dev) if s["state"] is None else s["state"].double()
    y, before = torch.empty_like(u), []
    for t in range(T):
        if train:
            before.append(h)
        h = torch.exp(step[t][..., None] * A) * h + (step[t] * u[t])[..., None] * B[t][:, group]
        y[t] = (h * C[t][:, group]).sum(-1)
    inner = y + skip * u
    if not train:
        return [unlined(inner * gate), h]
    dout = lined(s["dout"])
    dy = dout * gate
    dz = dout * inner * slope if case["gate"] else None
    du, dstep, dB, dC, dA = dy * skip, torch.empty_like(u), torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    behind = torch.zeros_like(before[0])
    for t in reversed(range(T)):
        decay, b, c = torch.exp(step[t][..., None] * A), B[t][:, group], C[t][:, group]
        kept = decay * before[t]
        now = kept + (step[t] * u[t])[..., None] * b
        dC[t].index_add_(1, group, dy[t][..., None] * now)
        behind = behind + dy[t][..., None] * c
        dB[t].index_add_(1, group, behind * (step[t] * u[t])[..., None])
        through = (behind * b).sum(-1)
        du[t] += through * step[t]
        moved = behind * kept
        dstep[t] = through * u[t] + (moved * A).sum(-1)
        dA += (moved * step[t][..., None]).sum(0)
        behind = decay * behind
    ddelta = dstep / (1 + torch.exp(-raw))
    grads = [unlined(du), unlined(ddelta), dA, unlined(dB), unlined(dC), (dy * u).sum((0, 1))]
    grads += ([unlined(dz)] if case["gate"] else []) + [torch.where(alive[..., None], ddelta, 0).sum((0, 1))]
    return [unlined(inner * gate)] + grads + ([behind] if s["state"] is not None else [])


def _exact_norm(s, case):
    B, P, G = case["batch"], case["positions"], case["groups"]
    x = s["x"].double().view(B, P, G, -1)
    w, bias = (s[n].double().view(G, -1) for n in ("weight", "bias"))
    count = P * x.shape[3]
    mean = torch.einsum("bpgc->bg", x)[:, None, :, None] / count
    var = torch.einsum("bpgc->bg", (x - mean) ** 2)[:, None, :, None] / count
    scale = (var + _EPS) ** -0.5
    hat = (x - mean) * scale
    y, slope = _act(hat * w + bias, case["silu"])
    if case["kind"] == "norm":
        return [y.view(s["x"].shape)]
    d = s["dout"].double().view(x.shape) * slope
    dhat = d * w
    along = torch.einsum("bpgc->bg", dhat * hat)[:, None, :, None] / count
    dx = scale * (dhat - torch.einsum("bpgc->bg", dhat)[:, None, :, None] / count - hat * along)
    return [y.view(s["x"].shape), dx.view(s["x"].shape), (d * hat).sum((0, 1)).flatten(), d.sum((0, 1)).flatten()]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "conv_step":
        line = torch.cat([s["state"], s["x"][:, None]], 1).double()
        y = torch.einsum("bjd,dj->bd", line, s["weight"].double()) + s["bias"].double()
        return [_act(y, case["silu"])[0], line[:, 1:]]
    if case["kind"] == "scan_step":
        at = torch.arange(case["dim"], device=s["u"].device) // (case["dim"] // case["groups"])
        raw, u = s["delta"].double() + s["delta_bias"].double(), s["u"].double()
        step = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
        new = torch.exp(step.unsqueeze(-1) * s["A"].double()) * s["state"].double() + (step * u).unsqueeze(-1) * s["B"].double()[:, at]
        y = torch.einsum("bdn,bdn->bd", new, s["C"].double()[:, at]) + s["D"].double() * u
        return [y * _act(s["z"].double(), True)[0] if case["gate"] else y, new]
    return {"c": _exact_conv, "s": _exact_scan, "n": _exact_norm}[case["kind"][0]](s, case)
