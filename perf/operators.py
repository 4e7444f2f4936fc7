"""Linear attention with a decay for each head -- the chunked form for prompts and training, the recurrent form for single
tokens -- and the norm and position rotation of its queries and keys, as cases that can be timed.

A case is a plain dict; ``prepare`` makes what a program holds before the call, ``run`` is one pass: the operators' plain forms in
elementary torch operations, or, where ``own`` is true, the package's operators; ``exact`` is the definition in 64 bits.

  state_t = exp(g_t) state_{t-1} + k_t v_t^T,   out_t = scale q_t^T state_t      for each head, state (Dk, Dv)
  norm and rotation: n = x / sqrt(mean(x^2) + eps) * weight, then each pair of n turned by position * frequency
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_CHUNK = 64
_EPS = 1e-6


def _attention(name, dtype, batch, tokens, heads, q_heads, k_heads, key_dim, value_dim, train, per_head=False, decay="", state=False, sequences=0):
    return dict(name=name, kind="train" if train else "prompt", dtype=dtype, batch=batch, tokens=tokens, heads=heads, q_heads=q_heads, k_heads=k_heads,
                key_dim=key_dim, value_dim=value_dim, per_head=per_head, decay=decay or dtype, state=state, sequences=sequences)


def _token(name, dtype, batch, heads, q_heads, k_heads, key_dim, value_dim):
    return dict(name=name, kind="token", dtype=dtype, batch=batch, heads=heads, q_heads=q_heads, k_heads=k_heads, key_dim=key_dim, value_dim=value_dim)


def _norm(name, dtype, batch, tokens, q_heads, k_heads, dim, rotated, axes, interleaved, train):
    return dict(name=name, kind="norm_train" if train else "norm", dtype=dtype, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim,
                rotated=rotated, axes=axes, interleaved=interleaved)


def listed():
    return [
        # One short prompt of an online request: the smallest call, its latency counts.
        _attention("prompt_37_b1_bf16", "bf16", 1, 37, 8, 8, 8, 64, 64, False, state=True),
        # A batch of ordinary prompts, the state kept for the tokens that follow.
        _attention("prompt_4096_b8_bf16", "bf16", 8, 4096, 16, 16, 16, 128, 128, False, state=True),
        # Prompts of different lengths one behind another, an empty one among them; queries and keys shared by all heads, as
        # state-space models have them.
        _attention("prompt_packed_bf16", "bf16", 1, 12011, 24, 1, 1, 128, 64, False, state=True, sequences=16),
        # One long document with few heads: the sequence itself has to fill the chip.
        _attention("prompt_65536_b1_bf16", "bf16", 1, 65536, 8, 8, 2, 64, 64, False, state=True),
        # Training of a language model's layer: forward and all gradients.
        _attention("train_2048_b4_bf16", "bf16", 4, 2048, 16, 16, 16, 128, 128, True),
        # Training in half precision at odd sizes, keys shared by the queries of a group, decays in single precision.
        _attention("train_1003_b3_fp16", "fp16", 3, 1003, 6, 6, 2, 48, 80, True, decay="fp32"),
        # Training on the tokens of 28 x 28 maps in single precision, one learnt decay for each head.
        _attention("train_784_b16_fp32", "fp32", 16, 784, 6, 1, 1, 64, 32, True, per_head=True),
        # One token of one request: latency.
        _token("token_b1_bf16", "bf16", 1, 8, 8, 8, 64, 64),
        # One token for each of many requests: the states pass through memory once.
        _token("token_b256_bf16", "bf16", 256, 32, 32, 8, 128, 128),
        # Queries and keys of one token of a few requests, far into their texts.
        _norm("norm_1_b8_bf16", "bf16", 8, 1, 32, 8, 128, 128, 1, False, False),
        # Queries and keys of a language model's layer in training, fewer key heads than query heads.
        _norm("norm_train_4096_b4_bf16", "bf16", 4, 4096, 32, 8, 128, 128, 1, False, True),
        # Tokens of 28 x 28 maps, rotated by row and column, neighbours paired, part of the head left unrotated.
        _norm("norm_train_784_b16_fp32", "fp32", 16, 784, 6, 6, 64, 48, 2, True, True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        key = (c["kind"].replace("norm_train", "norm"), c["dtype"] == "fp32")
        old = most.get(key, (0, 0))
        most[key] = max(old[0], w["bytes"]), max(old[1], w["flops"])
    while True:
        kind = rng.choice(["prompt", "prompt", "train", "train", "token", "norm", "norm_train"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        shared = rng.choice([1, 1, 2, 3, 4])
        if kind in ("prompt", "train"):
            heads = shared * rng.choice([1, 2, 3, 4, 5, 8])
            case = _attention(None, dtype, _between(rng, 1, 32), _between(rng, 1, 16384), heads, heads if rng.random() < 0.7 else heads // shared, heads // shared,
                              rng.choice([16, 20, 32, 48, 64, 64, 96, 128, 128, 192, 256]), rng.choice([16, 32, 36, 48, 64, 64, 80, 128, 128, 192, 256]), kind == "train",
                              per_head=rng.random() < 0.25, decay=rng.choice([dtype, "fp32"]), state=rng.random() < 0.5,
                              sequences=rng.randint(2, 40) if rng.random() < 0.3 else 0)
            if case["sequences"]:
                case["batch"], case["tokens"] = 1, max(case["tokens"], 4 * case["sequences"])
            if case["kind"] == "train":                    # (one token has no gradient of its decay)
                case["tokens"] = max(case["tokens"], 8)
            if case["per_head"]:
                case["decay"] = "fp32"
        elif kind == "token":
            heads = shared * rng.choice([1, 2, 4, 8, 16])
            case = _token(None, dtype, _between(rng, 1, 512), heads, heads, heads // shared, rng.choice([16, 32, 64, 96, 128, 256]), rng.choice([20, 32, 64, 80, 128, 256]))
        else:
            k_heads = rng.choice([1, 2, 4, 6, 8])
            dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 192, 256])
            axes = rng.choice([1, 1, 2])
            case = _norm(None, dtype, _between(rng, 1, 32), _between(rng, 1, 16384), k_heads * shared, k_heads, dim, dim if rng.random() < 0.7 else 2 * axes * (dim // (4 * axes)),
                         axes, rng.random() < 0.4, kind == "norm_train")
        del case["name"]
        # single precision where the kind has such a listed case is held to that one, else to a quarter of the others'
        limit = most.get((kind.replace("norm_train", "norm"), dtype == "fp32")) or tuple(v / 4 for v in most[(kind, False)])
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
    s = {"case": case}
    if case["kind"] in ("norm", "norm_train"):
        B, T, D, A = case["batch"], case["tokens"], case["dim"], case["axes"]
        s["q"] = (normal(B, T, case["q_heads"], D) * 2).to(dtype)
        s["k"] = (normal(B, T, case["k_heads"], D) * 2).to(dtype)
        s["q_weight"], s["k_weight"] = (1 + 0.2 * normal(D)).to(dtype), (1 + 0.2 * normal(D)).to(dtype)
        n = case["rotated"] // (2 * A)
        frequencies = 10000.0 ** (-torch.arange(n, device=dev, dtype=torch.float64) / n)
        if A == 1:                                         # each request at its own place in its text
            start = torch.randint(0, 100_000, (B, 1), device=dev, generator=gen)
            s["positions"], s["frequencies"] = start + torch.arange(T, device=dev), frequencies
        else:                                              # row and column of a token of a map
            side = max(1, math.isqrt(T))
            at = torch.arange(T, device=dev)
            s["positions"], s["frequencies"] = torch.stack([at // side, at % side], -1), frequencies.expand(A, n).contiguous()
        if case["kind"] == "norm_train":
            s["dq"], s["dk"] = torch.empty_like(s["q"]).copy_(normal(*s["q"].shape)), torch.empty_like(s["k"]).copy_(normal(*s["k"].shape))
        return s
    B, H, Hq, Hk, Dk, Dv = (case[n] for n in ("batch", "heads", "q_heads", "k_heads", "key_dim", "value_dim"))
    middle = () if case["kind"] == "token" else (case["tokens"],)
    s["q"], s["k"] = normal(B, *middle, Hq, Dk).to(dtype), normal(B, *middle, Hk, Dk).to(dtype)
    s["v"] = normal(B, *middle, H, Dv).to(dtype)
    if case.get("per_head"):                               # spread over horizons of 8 to 512 tokens
        s["g"] = torch.log1p(-torch.exp2(-3 - 6 * torch.rand(H, device=dev, generator=gen)))
    else:                                                  # a gate for each token and head
        s["g"] = -torch.nn.functional.softplus(1.5 * normal(B, *middle, H) - 3).to(_DTYPES[case.get("decay", case["dtype"])])
    if case["kind"] == "token":
        s["state"] = normal(B, H, Dk, Dv)
        return s
    N = case["sequences"] or B
    s["state"] = normal(N, H, Dk, Dv) if case["state"] else None
    if case["sequences"]:
        lengths = _lengths(case)
        s["longest"] = max(lengths)
        s["cu_seqlens"] = torch.tensor([sum(lengths[:i]) for i in range(N + 1)], device=dev, dtype=torch.int32)
    if case["kind"] == "train":
        s["dout"] = normal(*s["v"].shape).to(dtype)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _attend(q, k, v, g, state, scale):
    """(out, final state) of (B, T, H, D) in single precision, g (B, T, H) in double: all chunks at once, the states before them from the
    products of the decays between every two."""
    B, T, H, Dk = q.shape
    n = max(1, -(-T // _CHUNK))
    cut = lambda t: torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, n * _CHUNK - T)).unflatten(1, (n, _CHUNK))  # noqa: E731
    q, k, v = (cut(t).permute(0, 3, 1, 2, 4) for t in (q, k, v))                   # (B, H, n, C, D)
    G = cut(g).permute(0, 3, 1, 2).cumsum(-1)
    later = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).triu(1)
    P = (q @ k.transpose(-1, -2)) * (G[..., :, None] - G[..., None, :]).masked_fill(later, -math.inf).exp().float()
    end = G[..., -1:]
    local = (k * (end - G).exp().float()[..., None]).transpose(-1, -2) @ v         # (B, H, n, Dk, Dv)
    total = end[..., 0].cumsum(-1)                                                 # up to and with a chunk
    before = torch.cat([torch.zeros_like(total[..., :1]), total], -1)              # the n + 1 places between chunks
    after = torch.ones(n + 1, n, dtype=torch.bool, device=q.device).triu()         # a chunk is not behind the place
    between = (before[..., :, None] - total[..., None, :]).masked_fill(after, -math.inf).exp().float()
    states = (between @ local.flatten(-2)).unflatten(-1, local.shape[-2:])         # (B, H, n + 1, Dk, Dv)
    if state is not None:
        states = states + before.exp().float()[..., None, None] * state[:, :, None]
    out = (P @ v + (q * G.exp().float()[..., None]) @ states[:, :, :-1]) * scale
    return out.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :T], states[:, :, -1]


def _plain_attention(s):
    case = s["case"]
    dtype, H, T = _DTYPES[case["dtype"]], case["heads"], case["tokens"]
    spread = lambda t: t.repeat_interleave(H // t.shape[-2], -2)                   # noqa: E731
    leaves = [s[n].detach().float().requires_grad_(case["kind"] == "train") for n in ("q", "k", "v", "g")]
    with torch.set_grad_enabled(case["kind"] == "train"):
        q, k, v = (spread(t) for t in leaves[:3])
        g = leaves[3].double()
        g = g.expand(*q.shape[:2], H) if g.dim() == 1 else g
        if case["sequences"]:                              # one sequence to a row, zeros behind it
            cu = s["cu_seqlens"].long()
            at = cu[:-1, None] + torch.arange(s["longest"], device=cu.device)
            inside = at < cu[1:, None]
            rows = lambda t: torch.where(inside.view(*inside.shape, *(1,) * (t.dim() - 2)), t[0][at.clamp(max=T - 1)], 0)  # noqa: E731
            q, k, v, g = rows(q), rows(k), rows(v), rows(g)
        out, final = _attend(q, k, v, g, s["state"], case["key_dim"] ** -0.5)
        if case["sequences"]:
            token = torch.arange(T, device=cu.device)
            which = torch.searchsorted(cu, token, right=True) - 1
            out = out[which, token - cu[which]][None]
        out = out.to(dtype)
        if case["kind"] == "prompt":
            return [out, final]
        grads = torch.autograd.grad(out, leaves, s["dout"])
    return [out.detach()] + [d.to(s[n].dtype) for d, n in zip(grads, ("q", "k", "v", "g"))]


def _plain_token(s):
    case = s["case"]
    spread = lambda t: t.float().repeat_interleave(case["heads"] // t.shape[-2], -2)  # noqa: E731
    q, k, v = spread(s["q"]), spread(s["k"]), spread(s["v"])
    s["state"].mul_(s["g"].float().exp()[..., None, None]).add_(k[..., :, None] * v[..., None, :])
    out = (q[..., :, None] * s["state"]).sum(-2) * case["key_dim"] ** -0.5
    return [out.to(s["v"].dtype), s["state"]]


def _turned(n, cos, sin, rotated, interleaved):
    turned = n[..., :rotated]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else turned.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, n[..., rotated:]], -1)


def _plain_norm(s):
    case = s["case"]
    train = case["kind"] == "norm_train"
    angle = s["positions"].double()[..., None] * s["frequencies"]                  # (..., T, [axes,] n) in double: far positions
    angle = angle.flatten(-2) if case["axes"] > 1 else angle
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    leaves = [s[n].detach().float().requires_grad_(train) for n in ("q", "k", "q_weight", "k_weight")]
    with torch.set_grad_enabled(train):
        outs = [_turned(x * (x.square().mean(-1, keepdim=True) + _EPS).rsqrt() * w, cos, sin, case["rotated"], case["interleaved"]).to(s["q"].dtype)
                for x, w in zip(leaves[:2], leaves[2:])]
        if not train:
            return outs
        grads = torch.autograd.grad(outs, leaves, [s["dq"], s["dk"]])
    return [t.detach() for t in outs] + [d.to(s[n].dtype) for d, n in zip(grads, ("q", "k", "q_weight", "k_weight"))]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _own(state, case, kind)
    return _plain_token(state) if kind == "token" else _plain_norm(state) if kind in ("norm", "norm_train") else _plain_attention(state)


def _own(s, case, kind):
    from vmamba_amd import linear_attention_fn, linear_attention_step_fn, qk_norm_rotate_fn
    if kind == "token":
        return [linear_attention_step_fn(s["q"], s["k"], s["v"], s["g"], s["state"]), s["state"]]
    if kind == "norm":
        return list(qk_norm_rotate_fn(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["frequencies"], _EPS, case["interleaved"]))
    if kind == "norm_train":
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
        outs = qk_norm_rotate_fn(*leaves, s["positions"], s["frequencies"], _EPS, case["interleaved"])
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [s["dq"], s["dk"]]))
    more = dict(initial_state=s["state"], cu_seqlens=s.get("cu_seqlens"))
    if kind == "prompt":
        return list(linear_attention_fn(s["q"], s["k"], s["v"], s["g"], output_final_state=True, **more))
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    out = linear_attention_fn(*leaves, **more)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, s["dout"]))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
    e, B = _SIZE[case["dtype"]], case["batch"]
    if case["kind"] in ("norm", "norm_train"):
        values = B * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        passes = 4 if case["kind"] == "norm_train" else 2    # x and y, dy and dx (the gradients' weights are small)
        return {"bytes": values * e * passes, "flops": values * (24 if case["kind"] == "norm_train" else 8)}
    H, Hq, Hk, Dk, Dv = (case[n] for n in ("heads", "q_heads", "k_heads", "key_dim", "value_dim"))
    states = 4 * H * Dk * Dv
    if case["kind"] == "token":
        return {"bytes": B * (2 * states + e * ((Hq + Hk) * Dk + 2 * H * Dv)), "flops": 5 * B * H * Dk * Dv}
    T = case["tokens"]
    N = case["sequences"] or B
    sides = e * B * T * ((Hq + Hk) * Dk + H * Dv)             # q, k and v
    out = e * B * T * H * Dv
    decays = 0 if case["per_head"] else _SIZE[case["decay"]] * B * T * H
    kept = N * states * (int(case["state"]) + int(case["kind"] == "prompt"))
    flops = 4 * B * T * H * Dk * Dv                           # k v^T into the state and q^T state, each pair of a key and a value once
    if case["kind"] == "train":                               # and its backward: dout read, the inputs again, their gradients written
        return {"bytes": 2 * sides + 2 * out + 2 * decays + kept + sides, "flops": 3 * flops}
    return {"bytes": sides + out + decays + kept, "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _exact_sequence(q, k, v, g, state, scale, dout):
    """One head's sequence from the quadratic form out_t = scale sum_{s <= t} exp(G_t - G_s) (q_t . k_s) v_s + ..., a block of rows at a time:
    (out, final state, dq, dk, dv, dg)."""
    T = q.shape[0]
    G = torch.cumsum(g, 0)
    out = torch.zeros_like(v)
    dq, dk, dv, dG = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g)
    for lo in range(0, T, 1024):
        hi = min(lo + 1024, T)
        span = G[lo:hi, None] - G[None, :hi]
        seen = torch.arange(lo, hi, device=q.device)[:, None] >= torch.arange(hi, device=q.device)[None]
        decay = torch.where(seen, torch.exp(torch.where(seen, span, 0.0)), 0.0) * scale
        weights = torch.mm(q[lo:hi], k[:hi].t()) * decay
        out[lo:hi] = torch.mm(weights, v[:hi])
        carried = None
        if state is not None:
            carried = torch.mm(q[lo:hi], state) * (scale * torch.exp(G[lo:hi]))[:, None]
            out[lo:hi] += carried
        if dout is not None:
            d = dout[lo:hi]
            through = torch.mm(d, v[:hi].t())
            dv[:hi] += torch.mm(weights.t(), d)
            dq[lo:hi] += torch.mm(through * decay, k[:hi])
            dk[:hi] += torch.mm((through * decay).t(), q[lo:hi])
            both = weights * through
            dG[lo:hi] += both.sum(1)
            dG[:hi] -= both.sum(0)
            if state is not None:
                dq[lo:hi] += torch.mm(d, state.t()) * (scale * torch.exp(G[lo:hi]))[:, None]
                dG[lo:hi] += (carried * d).sum(1)
    final = torch.zeros(q.shape[1], v.shape[1], dtype=q.dtype, device=q.device) if state is None else state.clone()
    if T:
        final = final * torch.exp(G[-1]) + torch.mm((k * torch.exp(G[-1] - G)[:, None]).t(), v)
    return out, final, dq, dk, dv, torch.flip(torch.cumsum(torch.flip(dG, [0]), 0), [0])


def _exact_attention(s, case):
    H, T = case["heads"], case["tokens"]
    train = case["kind"] == "train"
    q, k, v, g = (s[n].double() for n in ("q", "k", "v", "g"))
    B = q.shape[0]
    if case["sequences"]:
        lengths = _lengths(case)
        starts = [sum(lengths[:i]) for i in range(len(lengths))]
        pieces = [(0, a, a + n) for a, n in zip(starts, lengths)]
    else:
        pieces = [(b, 0, T) for b in range(B)]
    out = torch.zeros(B, T, H, case["value_dim"], dtype=torch.float64, device=q.device)
    final = torch.zeros(len(pieces), H, case["key_dim"], case["value_dim"], dtype=torch.float64, device=q.device)
    dq, dk, dv, dg = (torch.zeros_like(t) for t in (q, k, v, g))
    for n, (b, lo, hi) in enumerate(pieces):
        for h in range(H):
            hq, hk = h // (H // q.shape[2]), h // (H // k.shape[2])
            gates = g[h].expand(hi - lo) if g.dim() == 1 else g[b, lo:hi, h]
            state = None if s["state"] is None else s["state"][n, h].double()
            o, f, a, c, d, e = _exact_sequence(q[b, lo:hi, hq], k[b, lo:hi, hk], v[b, lo:hi, h], gates, state, case["key_dim"] ** -0.5,
                                               s["dout"][b, lo:hi, h].double() if train else None)
            out[b, lo:hi, h], final[n, h] = o, f
            if train:
                dq[b, lo:hi, hq] += a
                dk[b, lo:hi, hk] += c
                dv[b, lo:hi, h] += d
                if g.dim() == 1:
                    dg[h] += e.sum()
                else:
                    dg[b, lo:hi, h] = e
    return [out, dq, dk, dv, dg] if train else [out, final]


def _exact_norm(s, case):
    train = case["kind"] == "norm_train"
    n, A, R = case["rotated"] // (2 * case["axes"]), case["axes"], case["rotated"]
    where = s["positions"].double().reshape(*s["positions"].shape[:s["positions"].dim() - (A > 1)], A, 1)
    angle = (where * s["frequencies"].view(A, n)).reshape(*where.shape[:-2], A * n)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)
    place = torch.arange(R // 2, device=angle.device)
    first, second = (2 * place, 2 * place + 1) if case["interleaved"] else (place, place + R // 2)

    def rotate(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs, sides, weights = [], [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + _EPS)
        outs.append(rotate(x / size * w, turn))
        if train:
            d = rotate(s["d" + name].double(), turn.conj())
            weights.append((d * x / size).flatten(0, 2).sum(0))
            d = d * w
            sides.append(d / size - x * (d * x).sum(-1, keepdim=True) / (case["dim"] * size ** 3))
    return outs + sides + weights if train else outs


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "token":
        H = case["heads"]
        pick = lambda t: t.double()[:, torch.arange(H, device=t.device) // (H // t.shape[1])]  # noqa: E731
        q, k, v = pick(s["q"]), pick(s["k"]), pick(s["v"])
        new = torch.exp(s["g"].double())[:, :, None, None] * s["state"].double() + k.unsqueeze(-1) * v.unsqueeze(-2)
        return [torch.matmul(q.unsqueeze(-2), new).squeeze(-2) * case["key_dim"] ** -0.5, new]
    return _exact_norm(s, case) if case["kind"] in ("norm", "norm_train") else _exact_attention(s, case)
