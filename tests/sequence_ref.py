"""The sequence operators from their definitions in 64 bits, and error bounds for the kernels'.

Bounds count roundings: one to bf16 is off by at most 2^-8 of the value, one to fp32 by 2^-24, and a
sum of n terms in fp32 by n 2^-24 (2^-23 where the tensor core cuts) of the sum of their absolute
values.  That sum is the same recurrence on the inputs' absolute values (`absolute`)."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def attention(q, k, v, log_gamma, scale, start=None):
    """o, last state of one batch, token after token: q, k [B, T, Hk, dk], v [B, T, H, dv] in float64."""
    rep = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    gamma = torch.exp(log_gamma.double())[None, :, None, None]
    S = start if start is not None else torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3],
                                                    dtype=torch.float64, device=v.device)
    o = []
    for t in range(v.shape[1]):
        S = gamma * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o.append(scale * (q[:, t, :, :, None] * S).sum(-2))
    return (torch.stack(o, 1) if o else torch.zeros_like(v)), S


def attention_grads(q, k, v, log_gamma, scale, g_o, start=None, g_state=None, cu=None):
    """{name: value} of o, state and the gradients, in float64 by autograd through the recurrence; cu: the
    bounds of packed sequences."""
    ins = {n: t.detach().double().clone().requires_grad_() for n, t in
           dict(q=q, k=k, v=v, start=start).items() if t is not None}
    s = ins.get("start")
    if cu is None:
        o, state = attention(ins["q"], ins["k"], ins["v"], log_gamma, scale, s)
    else:
        parts = [attention(*(ins[n][:, a:b] for n in "qkv"), log_gamma, scale, None if s is None else s[i:i + 1])
                 for i, (a, b) in enumerate(zip(cu, cu[1:]))]
        rest = torch.zeros_like(ins["v"][:, cu[-1]:])
        o, state = torch.cat([p[0] for p in parts] + [rest], 1), torch.cat([p[1] for p in parts])
    loss = (o * g_o.double()).sum()
    if g_state is not None:
        loss = loss + (state * g_state.double()).sum()
    grads = torch.autograd.grad(loss, list(ins.values()), allow_unused=True)
    out = {"o": o.detach(), "state": state.detach()}
    for (n, t), g in zip(ins.items(), grads):
        out["d_" + n] = torch.zeros_like(t) if g is None else g
    return out


def attention_bounds(want, absolute, dtype, dk, dv, blocks, state_f32=True):
    """{name: largest allowed |difference|, elementwise}.  fp32: each product is of three bf16 parts (what is
    left out is below 4 2^-24) and runs through two sums over up to max(dk, dv) and 64 terms and the states of
    `blocks` blocks.  bf16: the scores and the state's copy are rounded once each on the way, and the result."""
    n32 = (max(dk, dv) + 64 + blocks + 32) * 2.0 ** -23
    out = {}
    for name, w in want.items():
        a = absolute[name]
        if dtype == torch.bfloat16 and name not in ("state", "d_start"):
            out[name] = U[dtype] * (w.abs() + 2 * a) * (1 + 2.0 ** -7) + n32 * a
        else:
            out[name] = n32 * a
    return out


def close(got, want, bound, name=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 1e-300, f"{name}: {over:.3g} above its bound (largest difference {(got - want).abs().max():.3g})"


def turned(x, positions, inv_freq, interleaved, magnitude, inverse=False):
    """x [B, T, H, D] in float64 with its pairs turned as complex numbers."""
    half = inv_freq.numel()
    p = torch.arange(half, device=x.device)
    a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
    angle = positions.double().expand(x.shape[:2])[:, :, None, None] * inv_freq
    by = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)
    y = x.double().clone()
    z = torch.complex(y[..., a], y[..., b]) * by
    y[..., a], y[..., b] = z.real, z.imag
    return y


def act(u, kind):
    if kind == "silu":
        return u * torch.sigmoid(u)
    if kind == "gelu":
        return 0.5 * u * torch.erfc(-u / 2 ** 0.5)
    return u


def group_norm(x, groups, weight, bias, gate, activation, eps):
    xg = x.unflatten(-1, (groups, -1))
    xg = xg - xg.mean(-1, keepdim=True)
    z = (xg / torch.sqrt((xg * xg).mean(-1, keepdim=True) + eps)).flatten(-2)
    if weight is not None:
        z = z * weight
    if bias is not None:
        z = z + bias
    return act(z, activation) if gate is None else z * act(gate, activation)
