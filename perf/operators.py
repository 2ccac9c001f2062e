"""Cases and plain forms of the sequence operators beside the TTC layer: attention with a fixed
decay for each head (``decay_attention`` for prompts and training, ``decay_attention_step`` for
single tokens over a cache of states), rotary positions (``rotary``) and the group norm of each
token's heads with its gate (``group_norm``).

``own`` false: elementary torch operations in 32 bits (64 for angles), rounded once at the end.
``own`` true: the calls a user makes of ``ttc_b200``.
"""
import math
import os
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CHUNK = 64  # tokens per block of the plain chunked form


def listed():
    return [
        # A batch of long prompts at the width of the layer's LLM-scale configuration (8 x 4096
        # tokens, 32 heads of 128), with the states that the first generated token starts from.
        dict(name="prompt 8x4096 h32 d128 bf16", op="attention", seqs=8, tokens=4096, heads=32, key_heads=32,
             dk=128, dv=128, dtype="bf16", packed=False, start=False, train=False),
        # One long document alone: few sequences, so the work has to be split over its length.
        dict(name="prompt 1x32768 h16 d64 bf16", op="attention", seqs=1, tokens=32768, heads=16, key_heads=16,
             dk=64, dv=64, dtype="bf16", packed=False, start=True, train=False),
        # Prompts of mixed lengths packed into one row as a server batches them, keys shared by
        # four heads, continued from earlier states.
        dict(name="packed 24 to 777 h32/8 d128 bf16", op="attention", seqs=24, tokens=777, heads=32, key_heads=8,
             dk=128, dv=128, dtype="bf16", packed=True, start=True, train=False),
        # One training micro-batch, forward and backward, at the LLM-scale width.
        dict(name="train 2x4096 h32 d128 bf16", op="attention", seqs=2, tokens=4096, heads=32, key_heads=32,
             dk=128, dv=128, dtype="bf16", packed=False, start=False, train=True),
        # A small model trained in 32 bits, odd length, values wider than keys, gradients of shared
        # keys and of the starting state.
        dict(name="train 4x1001 h16/4 d32/64 f32", op="attention", seqs=4, tokens=1001, heads=16, key_heads=4,
             dk=32, dv=64, dtype="f32", packed=False, start=True, train=True),
        # One token for each of 64 running requests, their states in a cache of 96.
        dict(name="token 64 of 96 h32 d128 bf16", op="step", seqs=64, slots=96, heads=32, key_heads=32, dk=128,
             dv=128, dtype="bf16"),
        # One token of a single request: the call's latency.
        dict(name="token 1 h16/4 d64 f32", op="step", seqs=1, slots=1, heads=16, key_heads=4, dk=64, dv=64,
             dtype="f32"),
        # Queries and keys of a training batch, forward and backward, the whole head rotated.
        dict(name="rotary 4x4096 h32/8 d128 bf16", op="rotary", seqs=4, tokens=4096, heads=32, key_heads=8, dim=128,
             rot=128, interleaved=False, scaling="none", first=0, dtype="bf16", train=True),
        # New tokens of 7 requests far into a long context, part of the head, interleaved pairs.
        dict(name="rotary 7x1 far h16/4 d80/32 f32", op="rotary", seqs=7, tokens=1, heads=16, key_heads=4, dim=80,
             rot=32, interleaved=True, scaling="yarn", first=900001, dtype="f32", train=False),
        # The gated norm after attention in a training batch: 32 heads of 128, forward and backward.
        dict(name="norm 16384x32x128 bf16", op="norm", rows=16384, groups=32, size=128, activation="silu", gate=True,
             affine=True, dtype="bf16", train=True),
        # The same norm of the new tokens of 5 requests, heads of an odd size, no gate.
        dict(name="norm 5x12x45 f32", op="norm", rows=5, groups=12, size=45, activation="silu", gate=False,
             affine=True, dtype="f32", train=False),
    ]


def _log(rng, a, b):
    """A whole number from a to b, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "step", "rotary", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    key_heads = rng.choice([1, 2, 4, 5, 8])
    heads = key_heads * rng.choice([1, 1, 2, 4])
    dk, dv = 8 * rng.randint(1, 16), 8 * rng.randint(1, 16)
    if op == "attention":
        train = rng.random() < 0.5
        tokens = _log(rng, 1, 4096 if train else 8192)
        most = (1 << (20 - 2 * train - (dtype == "f32"))) // (heads * tokens)
        return dict(op=op, seqs=_log(rng, 1, max(1, min(64, most))), tokens=tokens, heads=heads, key_heads=key_heads,
                    dk=dk, dv=dv, dtype=dtype, packed=rng.random() < 0.4, start=rng.random() < 0.5, train=train)
    if op == "step":
        seqs = _log(rng, 1, 256)
        return dict(op=op, seqs=seqs, slots=seqs + rng.randint(0, 40), heads=heads, key_heads=key_heads, dk=dk, dv=dv,
                    dtype=dtype)
    if op == "rotary":
        tokens = _log(rng, 1, 4096)
        dim = 2 * rng.randint(4, 128)
        return dict(op=op, seqs=_log(rng, 1, max(1, min(64, (1 << 17) // (heads * tokens)))), tokens=tokens, heads=heads,
                    key_heads=key_heads, dim=dim, rot=2 * rng.randint(1, dim // 2), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), first=_log(rng, 1, 1000000), dtype=dtype,
                    train=rng.random() < 0.5)
    size = _log(rng, 3, 700)
    return dict(op=op, rows=_log(rng, 1, max(2, (1 << 25) // (heads * size))), groups=heads, size=size,
                activation=rng.choice(["none", "silu", "gelu"]), gate=rng.random() < 0.5, affine=rng.random() < 0.7,
                dtype=dtype, train=rng.random() < 0.6)


# --------------------------------------------------------------------------------------------
# What a program has in hand
# --------------------------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the packed sequences: from one token to case["tokens"], an empty one among them."""
    n, most = case["seqs"], case["tokens"]
    lens = [1 + (most - 1) * ((i * 7) % n) // max(1, n - 1) for i in range(n)]
    lens[0] = most
    if n > 2:
        lens[1] = 0
    return lens


def _frequencies(case):
    """Inverse frequencies of the rotated pairs in 64 bits, and the factor on the result."""
    half = case["rot"] // 2
    base, factor, trained = 10000.0, 8.0, 4096.0
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    plain = base ** (-2.0 * i / case["rot"])
    if case["scaling"] == "linear":
        return plain / factor, 1.0
    if case["scaling"] == "ntk":
        if case["rot"] <= 2:
            return plain, 1.0
        return (base * factor ** (case["rot"] / (case["rot"] - 2.0))) ** (-2.0 * i / case["rot"]), 1.0
    if case["scaling"] == "yarn":
        turns = trained * plain / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return plain * keep + plain / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return plain, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = dict(case=dict(case))
    if case["op"] in ("attention", "step"):
        H = case["heads"]
        # decays from 31/32 to 511/512 over the heads: memories of 32 to 512 tokens
        s["log_gamma"] = torch.log1p(-torch.exp2(-5 - 4 * torch.arange(H, device="cuda", dtype=torch.float64)
                                                 / max(1, H - 1))).float()
    if case["op"] == "attention":
        if case["packed"]:
            lens = _lengths(case)
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + n)
            s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
            s["longest"] = max(lens)
            rows = (1, cu[-1])
        else:
            rows = (case["seqs"], case["tokens"])
        s["q"] = normal(*rows, case["key_heads"], case["dk"])
        s["k"] = normal(*rows, case["key_heads"], case["dk"])
        s["v"] = normal(*rows, case["heads"], case["dv"])
        if case["start"]:
            s["start"] = normal(case["seqs"], case["heads"], case["dk"], case["dv"], dtype=torch.float32)
        if case["train"]:
            s["g_o"] = normal(*rows, case["heads"], case["dv"])
    elif case["op"] == "step":
        s["q"] = normal(case["seqs"], case["key_heads"], case["dk"])
        s["k"] = normal(case["seqs"], case["key_heads"], case["dk"])
        s["v"] = normal(case["seqs"], case["heads"], case["dv"])
        s["cache"] = normal(case["slots"], case["heads"], case["dk"], case["dv"], dtype=torch.float32)
        s["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:case["seqs"]].to(torch.int32)
    elif case["op"] == "rotary":
        s["q"] = normal(case["seqs"], case["tokens"], case["heads"], case["dim"])
        s["k"] = normal(case["seqs"], case["tokens"], case["key_heads"], case["dim"])
        first = torch.randint(case["first"], case["first"] + 1000, (case["seqs"], 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(case["tokens"], device="cuda")
        s["inv_freq"], s["magnitude"] = _frequencies(case)
        if case["train"]:
            s["g_q"], s["g_k"] = normal(*s["q"].shape), normal(*s["k"].shape)
    else:
        C = case["groups"] * case["size"]
        # group means away from zero and spreads of their own, as attention's outputs have them
        x = torch.randn(case["rows"], case["groups"], case["size"], generator=g, device="cuda")
        x = x * (0.2 + torch.rand(case["rows"], case["groups"], 1, generator=g, device="cuda"))
        x = x + torch.randn(case["rows"], case["groups"], 1, generator=g, device="cuda")
        s["x"] = x.view(case["rows"], C).to(dt)
        if case["affine"]:
            s["weight"] = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(dt)
            s["bias"] = (0.2 * torch.randn(C, generator=g, device="cuda")).to(dt)
        if case["gate"]:
            s["gate"] = normal(case["rows"], C)
        if case["train"]:
            s["g_y"] = normal(case["rows"], C)
    return s


# --------------------------------------------------------------------------------------------
# Plain forms
# --------------------------------------------------------------------------------------------
def _aligned(x, s):
    """[1, total, ...] packed rows -> [sequences, longest, ...], each sequence at the END of its row,
    zeros before it."""
    cu, L = s["cu"].long(), s["longest"]
    at = cu[1:, None] - L + torch.arange(L, device=x.device)
    there = at >= cu[:-1, None]
    rows = x[0][at.clamp(min=0)]
    return torch.where(there.view(*there.shape, *([1] * (x.dim() - 2))), rows, torch.zeros_like(rows))


def _packed(x, s):
    """The inverse of _aligned for x [sequences, longest, ...]."""
    cu, L = s["cu"].long(), s["longest"]
    t = torch.arange(int(s["q"].shape[1]), device=x.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return x[seq, t - cu[1:][seq] + L][None]


def _attention(q, k, v, s):
    """o and the last states of float32 q, k, v, block by block: inside a block the masked and
    decayed scores, between blocks the decayed sum of the earlier blocks' key-value products."""
    case = s["case"]
    H, rep = case["heads"], case["heads"] // case["key_heads"]
    scale = case["dk"] ** -0.5
    lg = s["log_gamma"].double()
    if case["packed"]:
        lens = s["cu"].long()[1:] - s["cu"].long()[:-1]
        q, k, v = _aligned(q, s), _aligned(k, s), _aligned(v, s)
    B, T = v.shape[:2]
    if not case["packed"]:
        lens = torch.full((B,), T, device=v.device)
    n = -(-T // CHUNK)
    pad = n * CHUNK - T

    def blocks(x, r):  # [B, T, h, d] -> [B, H, n, CHUNK, d], zeros first
        x = torch.nn.functional.pad(x.repeat_interleave(r, dim=2), (0, 0, 0, 0, pad, 0))
        return x.view(B, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v = blocks(q, rep), blocks(k, rep), blocks(v, 1)
    i = torch.arange(CHUNK, device=v.device)
    ahead = (i[:, None] - i[None, :]).double()
    decay = torch.where(ahead >= 0, torch.exp(lg[:, None, None] * ahead.clamp(min=0)), 0.0).float()
    score = q @ k.transpose(-1, -2) * decay[:, None] * scale
    o = score @ v
    left = torch.exp(lg[:, None] * (CHUNK - 1 - i)).float()
    add = (k * left[:, None, :, None]).transpose(-1, -2) @ v  # [B, H, n, dk, dv]
    c = torch.arange(n + 1, device=v.device)
    gap = (c[:, None] - 1 - c[None, :-1]).double()  # blocks between block j's end and block c's start
    carry = torch.where(gap >= 0, torch.exp(lg[:, None, None] * CHUNK * gap.clamp(min=0)), 0.0).float()
    state = torch.einsum("hcj,bhjx->bhcx", carry, add.flatten(-2)).unflatten(-1, add.shape[-2:])
    passed = torch.exp(lg[:, None] * (i + 1)).float()
    o = o + (q * (passed[:, None, :, None] * scale)) @ state[:, :, :-1]
    last = state[:, :, -1]
    if "start" in s:
        t = torch.arange(n * CHUNK, device=v.device) - (n * CHUNK - lens[:, None])  # place in its sequence
        since = torch.exp(lg[None, :, None] * (t[:, None] + 1).clamp(min=0)).float()
        full = q.flatten(2, 3) * (since * scale)[..., None]
        o = o + (full @ s["start_"]).view_as(o)
        last = last + torch.exp(lg[None] * lens[:, None]).float()[..., None, None] * s["start_"]
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, -1)[:, pad:]
    return (_packed(o, s) if case["packed"] else o), last


def _rotated(x, s, back=False):
    """x [B, T, H, D] float32 with its first `rot` values turned by position * inv_freq."""
    case = s["case"]
    rot, half = case["rot"], case["rot"] // 2
    angle = s["positions"].double()[..., None] * s["inv_freq"]
    cos = (angle.cos() * s["magnitude"]).float()[:, :, None]
    sin = (angle.sin() * s["magnitude"]).float()[:, :, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :half], x[..., half:rot])
    if back:
        sin = -sin
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _act(x, kind):
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _norm(x, weight, bias, gate, case):
    """Each token's groups to mean 0 and variance 1, weight and bias, then the activation: of the
    gate, which multiplies, or of the result itself."""
    xg = x.view(case["rows"], case["groups"], case["size"])
    xg = xg - xg.mean(-1, keepdim=True)
    y = (xg * torch.rsqrt(xg.square().mean(-1, keepdim=True) + 1e-5)).view_as(x)
    if weight is not None:
        y = y * weight + bias
    return _act(y, case["activation"]) if gate is None else y * _act(gate, case["activation"])


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "attention":
        names = ["q", "k", "v"] + (["start"] if case["start"] else [])
        ins = {n: s[n].float().requires_grad_(case["train"]) for n in names}
        o, last = _attention(ins["q"], ins["k"], ins["v"], {**s, "start_": ins.get("start")})
        if not case["train"]:
            return {"o": o.to(dt), "state": last}
        grads = torch.autograd.grad(o, list(ins.values()), s["g_o"].float())
        out = {"o": o.detach().to(dt)}
        out.update({"d_" + n: d.to(s[n].dtype) for n, d in zip(names, grads)})
        return out
    if case["op"] == "step":
        rep = case["heads"] // case["key_heads"]
        q, k = s["q"].float().repeat_interleave(rep, 1), s["k"].float().repeat_interleave(rep, 1)
        at = s["slots"].long()
        new = s["cache"][at] * torch.exp(s["log_gamma"].double()).float()[:, None, None]
        new = new + k[..., None] * s["v"].float()[..., None, :]
        s["cache"][at] = new
        o = (q[..., None] * new).sum(-2) * case["dk"] ** -0.5
        return {"o": o.to(dt), "cache": s["cache"]}
    if case["op"] == "rotary":
        out = {"q": _rotated(s["q"].float(), s).to(dt), "k": _rotated(s["k"].float(), s).to(dt)}
        if case["train"]:
            out["d_q"] = torch.cat([_rotated(s["g_q"].float(), s, True)[..., :case["rot"]],
                                    s["g_q"].float()[..., case["rot"]:]], -1).to(dt)
            out["d_k"] = torch.cat([_rotated(s["g_k"].float(), s, True)[..., :case["rot"]],
                                    s["g_k"].float()[..., case["rot"]:]], -1).to(dt)
        return out
    names = [n for n in ("x", "weight", "bias", "gate") if n in s]
    ins = {n: s[n].float().requires_grad_(case["train"]) for n in names}
    y = _norm(ins["x"], ins.get("weight"), ins.get("bias"), ins.get("gate"), case)
    out = {"y": y.detach().to(dt)}
    if case["train"]:
        grads = torch.autograd.grad(y, list(ins.values()), s["g_y"].float())
        out.update({"d_" + n: d.to(dt) for n, d in zip(names, grads)})
    return out


# --------------------------------------------------------------------------------------------
# The framework's calls
# --------------------------------------------------------------------------------------------
def _ops():
    path = os.path.join(REPO, "ttc-net_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ttc_b200
    return ttc_b200


def _leaves(s, names, train):
    return [s[n].detach().requires_grad_(train) for n in names]


def _run_own(s):
    ops, case = _ops(), s["case"]
    if case["op"] == "attention":
        names = ["q", "k", "v"] + (["start"] if case["start"] else [])
        ins = _leaves(s, names, case["train"])
        start = ins[3] if case["start"] else None
        if not case["train"]:
            o, last = ops.decay_attention(*ins[:3], s["log_gamma"], initial_state=start, return_state=True,
                                          cu_seqlens=s.get("cu"))
            return {"o": o, "state": last}
        o = ops.decay_attention(*ins[:3], s["log_gamma"], initial_state=start, cu_seqlens=s.get("cu"))
        grads = torch.autograd.grad(o, ins, s["g_o"])
        return {"o": o.detach(), **{"d_" + n: d for n, d in zip(names, grads)}}
    if case["op"] == "step":
        o = ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_gamma"], s["cache"], slots=s["slots"])
        return {"o": o, "cache": s["cache"]}
    if case["op"] == "rotary":
        ins = _leaves(s, ["q", "k"], case["train"])
        q, k = ops.rotary(*ins, s["positions"], s["inv_freq"], interleaved=case["interleaved"],
                          magnitude=s["magnitude"])
        out = {"q": q.detach(), "k": k.detach()}
        if case["train"]:
            out["d_q"], out["d_k"] = torch.autograd.grad((q, k), ins, (s["g_q"], s["g_k"]))
        return out
    names = [n for n in ("x", "weight", "bias", "gate") if n in s]
    ins = dict(zip(names, _leaves(s, names, case["train"])))
    y = ops.group_norm(ins["x"], case["groups"], ins.get("weight"), ins.get("bias"), gate=ins.get("gate"),
                       activation=case["activation"])
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, list(ins.values()), s["g_y"])
        out.update({"d_" + n: d for n, d in zip(names, grads)})
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------------------------
def _exact_sequence(q, k, v, gamma, scale, start, g_o):
    """One token after the other, [B, T, H, d] in 64 bits; with g_o the gradients as well."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    S = start.clone() if start is not None else torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device)
    gam = gamma[None, :, None, None]
    o = torch.zeros(B, T, H, dv, dtype=torch.float64, device=q.device)
    d_q, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T):
        S = S * gam + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * torch.einsum("bhk,bhkv->bhv", q[:, t], S)
        if g_o is not None:
            d_q[:, t] = scale * torch.einsum("bhkv,bhv->bhk", S, g_o[:, t])
    if g_o is None:
        return o, S
    dS = torch.zeros_like(S)
    for t in reversed(range(T)):
        dS = dS + scale * q[:, t, :, :, None] * g_o[:, t, :, None, :]
        d_k[:, t] = torch.einsum("bhkv,bhv->bhk", dS, v[:, t])
        d_v[:, t] = torch.einsum("bhkv,bhk->bhv", dS, k[:, t])
        dS = dS * gam
    return o, d_q, d_k, d_v, dS


def _exact_attention(s):
    case = s["case"]
    rep = case["heads"] // case["key_heads"]
    q, k = (s[n].double().repeat_interleave(rep, 2) for n in "qk")
    v = s["v"].double()
    start = s["start"].double() if case["start"] else None
    g_o = s["g_o"].double() if case["train"] else None
    gamma = torch.exp(s["log_gamma"].double())
    scale = 1.0 / math.sqrt(case["dk"])

    def call(rows, seq):
        return _exact_sequence(q[rows], k[rows], v[rows], gamma, scale, None if start is None else start[seq],
                               None if g_o is None else g_o[rows])

    if not case["packed"]:
        res = call((slice(None),), slice(None))
    else:
        cu = s["cu"].tolist()
        parts = [call((slice(None), slice(cu[i], cu[i + 1])), slice(i, i + 1)) for i in range(len(cu) - 1)]
        res = [torch.cat(p, 0 if p[0].shape[1:] == (case["heads"], case["dk"], case["dv"]) and j == len(parts[0]) - 1
                         else 1) for j, p in enumerate(zip(*parts))]
    if not case["train"]:
        return {"o": res[0], "state": res[1]}
    shared = lambda d: d.unflatten(2, (case["key_heads"], rep)).sum(3)  # noqa: E731
    out = {"o": res[0], "d_q": shared(res[1]), "d_k": shared(res[2]), "d_v": res[3]}
    if case["start"]:
        out["d_start"] = res[4]
    return out


def _exact_norm(s):
    case = s["case"]
    R, G, n, kind = case["rows"], case["groups"], case["size"], case["activation"]
    x = s["x"].double().reshape(R, G, n)
    one = torch.ones(G * n, dtype=torch.float64, device=x.device)
    w = s["weight"].double() if case["affine"] else one
    b = s["bias"].double() if case["affine"] else 0 * one
    mean = x.sum(-1, keepdim=True) / n
    rstd = 1 / torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / n + 1e-5)
    xhat = ((x - mean) * rstd).reshape(R, G * n)
    z = xhat * w + b

    def act(u):  # the activation and its derivative
        if kind == "silu":
            p = torch.sigmoid(u)
            return u * p, p * (1 + u * (1 - p))
        if kind == "gelu":
            c = 0.5 * torch.erfc(-u / math.sqrt(2))
            return u * c, c + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
        return u, torch.ones_like(u)

    if case["gate"]:
        ga, gd = act(s["gate"].double())
        y = z * ga
    else:
        y, zd = act(z)
    out = {"y": y}
    if not case["train"]:
        return out
    g = s["g_y"].double()
    gz = g * ga if case["gate"] else g * zd
    gx = (gz * w).reshape(R, G, n)
    xh = xhat.reshape(R, G, n)
    out["d_x"] = (rstd * (gx - gx.mean(-1, keepdim=True) - xh * (gx * xh).mean(-1, keepdim=True))).reshape(R, G * n)
    if case["affine"]:
        out["d_weight"], out["d_bias"] = (gz * xhat).sum(0), gz.sum(0)
    if case["gate"]:
        out["d_gate"] = g * z * gd
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        tokens = sum(_lengths(case)) if case["packed"] else case["tokens"]
        # about 15 us for each small operation of a token's step, and the states' traffic
        states = (1 if case["packed"] else case["seqs"]) * case["heads"] * case["dk"] * case["dv"]
        if tokens * (8e-5 + states * 1e-11) * (3 if case["train"] else 1) > 18:
            return None
        return _exact_attention(s)
    if case["op"] == "step":
        rep = case["heads"] // case["key_heads"]
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        cache = s["cache"].double()
        gamma = torch.exp(s["log_gamma"].double())
        o = torch.zeros_like(v)
        for b, slot in enumerate(s["slots"].tolist()):
            for h in range(case["heads"]):
                cache[slot, h] = gamma[h] * cache[slot, h] + torch.outer(k[b, h // rep], v[b, h])
                o[b, h] = q[b, h // rep] @ cache[slot, h] / math.sqrt(case["dk"])
        return {"o": o, "cache": cache}
    if case["op"] == "rotary":
        half, rot = case["rot"] // 2, case["rot"]
        j = torch.arange(half, device="cuda")
        first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
        turn = torch.polar(torch.full_like(s["inv_freq"], s["magnitude"]),
                           s["positions"].double()[:, :, None, None] * s["inv_freq"])

        def turned(x, by):
            y = x.double().clone()
            z = torch.complex(y[..., first], y[..., second]) * by
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
        if case["train"]:
            out["d_q"], out["d_k"] = turned(s["g_q"], turn.conj()), turned(s["g_k"], turn.conj())
        return out
    return _exact_norm(s)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        rows = sum(_lengths(case)) if case["packed"] else case["seqs"] * case["tokens"]
        state = case["seqs"] * case["heads"] * case["dk"] * case["dv"] * 4
        qk, vo = rows * case["key_heads"] * case["dk"] * size, rows * case["heads"] * case["dv"] * size
        # the recurrence: a product with the state and an update of it for each token
        flops = 4 * rows * case["heads"] * case["dk"] * case["dv"]
        if not case["train"]:
            return {"bytes": 2 * qk + 2 * vo + state * (2 if case["start"] else 1), "flops": flops}
        # forward as above without the last state, backward: q, k, v, g_o read, three gradients written
        return {"bytes": 2 * qk + 2 * vo + 4 * qk + 3 * vo + state * (3 if case["start"] else 0), "flops": 3.5 * flops}
    if case["op"] == "step":
        state = case["seqs"] * case["heads"] * case["dk"] * case["dv"]
        rest = case["seqs"] * size * 2 * (case["key_heads"] * case["dk"] + case["heads"] * case["dv"])
        return {"bytes": 8 * state + rest, "flops": 5 * state}
    if case["op"] == "rotary":
        values = case["seqs"] * case["tokens"] * (case["heads"] + case["key_heads"]) * case["dim"]
        both = 2 if case["train"] else 1
        return {"bytes": both * 2 * values * size, "flops": both * 3 * values}
    values = case["rows"] * case["groups"] * case["size"]
    gate = 1 if case["gate"] else 0
    passes = 2 + gate + ((3 + 2 * gate) if case["train"] else 0)
    return {"bytes": passes * values * size, "flops": (10 + (25 if case["train"] else 0)) * values}
