"""rotary and group_norm against their definitions in 64 bits, and the three sequence operators run
together as a memory layer runs them."""
import pytest
import torch
from sequence_ref import U, attention, close, group_norm, turned

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _rot_bound(x, want, half, interleaved, dtype):
    """Three fp32 roundings of products and sums of a pair and those of the cosine and sine (2 ulp): below
    2^-21 of |a| + |b|; the copied part is exact."""
    p = torch.arange(half, device=x.device)
    a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
    s = torch.zeros_like(want)
    s[..., a] = s[..., b] = x.double()[..., a].abs() + x.double()[..., b].abs()
    return 2.0 ** -21 * s * 2 + (U[dtype] * want.abs() * 1.01 if dtype == torch.bfloat16 else 0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D,half", [(2, 5, 4, 2, 64, 32), (1, 1, 3, 3, 128, 64), (3, 7, 2, 1, 80, 16), (1, 33, 5, 2, 6, 2),
                                             (2, 3, 1, 1, 130, 65), (1, 2, 2, 2, 512, 256), (1, 9, 2, 2, 16, 0),
                                             (1, 400, 8, 8, 32, 16)])
def test_rotary(B, T, H, Hk, D, half, interleaved, dtype):
    from ttc_b200 import rotary
    q, k = _normal(1, B, T, H, D, dtype=dtype), _normal(2, B, T, Hk, D, dtype=dtype)
    gq, gk = _normal(3, B, T, H, D, dtype=dtype), _normal(4, B, T, Hk, D, dtype=dtype)
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
    pos = torch.randint(0, 1 << 20, (B, T), device="cuda")
    ins = [q.requires_grad_(), k.requires_grad_()]
    outs = rotary(*ins, pos, inv, interleaved=interleaved, magnitude=1.25)
    grads = torch.autograd.grad(outs, ins, (gq, gk))
    m = 1.25
    for x, y in zip(ins, outs):
        want = turned(x.detach(), pos, inv, interleaved, m)
        close(y.detach(), want, _rot_bound(x.detach(), want, half, interleaved, dtype))
        assert torch.equal(y[..., 2 * half:], x[..., 2 * half:])
    for g, d in zip((gq, gk), grads):
        want = turned(g, pos, inv, interleaved, m, inverse=True)
        close(d, want, _rot_bound(g, want, half, interleaved, dtype))


def test_rotary_positions_and_strides():
    from ttc_b200 import rotary
    z = _normal(0, 2, 6, 3 * 4 * 32 + 1, dtype=torch.bfloat16)
    inv = torch.tensor([1.0, 0.3, 0.01, 1e-5] * 4, dtype=torch.float64, device="cuda")
    pos = torch.arange(6, device="cuda") + 123456789  # 1e8: 64-bit angles
    q = z[..., 1:1 + 4 * 32].unflatten(-1, (4, 32))  # odd start: rows off the 16-byte grid
    k = z[..., 128:256].unflatten(-1, (4, 32)).transpose(0, 1).contiguous().transpose(0, 1)
    want = rotary(q.contiguous(), k.contiguous(), pos.expand(2, 6).contiguous(), inv)
    for p in (pos, pos[None], pos.int(), pos.expand(2, 6)):
        got = rotary(q, k, p, inv)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    alone, none = rotary(q, None, pos, inv)
    assert none is None and torch.equal(alone, want[0])
    ref = turned(q, pos, inv, False, 1.0)
    close(alone, ref, _rot_bound(q, ref, 16, False, torch.bfloat16))
    neg = rotary(q, None, -pos, inv)[0]
    ref = turned(q, -pos, inv, False, 1.0)
    close(neg, ref, _rot_bound(q, ref, 16, False, torch.bfloat16))
    assert rotary(q[:, :0], k[:, :0], pos[:0], inv)[0].shape == (2, 0, 4, 32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,groups,n", [(5, 4, 64), (300, 3, 128), (1, 1, 1), (17, 5, 45), (64, 2, 1024), (9, 7, 3), (33, 2, 1000),
                                           (700, 1, 16), (3, 2, 513)])
def test_group_norm(rows, groups, n, gated, activation, dtype):
    """Bounds: xhat is off by sums of n terms of values up to max |x| against the spread (n 2^-24 (1 + max |x| rstd)),
    and everything after it by a few roundings more, of terms bounded by their absolute values; slopes of
    the activations are below 1.2."""
    from ttc_b200 import group_norm as gn
    C = groups * n
    x = (_normal(1, rows, groups, n) * 0.7 + _normal(2, rows, groups, 1)).view(rows, C).to(dtype)
    w, b = 1 + 0.3 * _normal(3, C), 0.3 * _normal(4, C)
    if dtype == torch.bfloat16 and n != 64:  # bf16 rows with fp32 parameters at n = 64
        w, b = w.to(dtype), b.to(dtype)
    gate = _normal(5, rows, C, dtype=dtype) * 2 if gated else None
    gy = _normal(6, rows, C, dtype=dtype)
    named = [(k, t) for k, t in (("x", x), ("weight", w), ("bias", b), ("gate", gate)) if t is not None]
    ins = {k: t.detach().requires_grad_() for k, t in named}
    y = gn(ins["x"], groups, ins["weight"], ins["bias"], gate=ins.get("gate"), activation=activation, eps=1e-5)
    grads = torch.autograd.grad(y, list(ins.values()), gy)
    ref = {k: t.detach().double().requires_grad_() for k, t in named}
    yr = group_norm(ref["x"], groups, ref["weight"], ref["bias"], ref.get("gate"), activation, 1e-5)
    want = dict(zip(ref, torch.autograd.grad(yr, list(ref.values()), gy.double())))

    xg = x.double().view(rows, groups, n)
    rstd = (xg.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    rel = ((n + 32) * 2.0 ** -24 * (2 + xg.abs().amax(-1, keepdim=True) * rstd)).expand(-1, -1, n).reshape(rows, C)
    xhat = ((xg - xg.mean(-1, keepdim=True)) * rstd).view(rows, C).abs()
    wd, bd, gyd = w.double().abs(), b.double().abs(), gy.double().abs()
    za = (xhat + 1) * wd + bd
    gab = 1.2 * gate.double().abs() if gated else torch.ones_like(za)
    u = U[dtype] * 1.01

    def bound(value, f32):
        return f32 + (u * value.double().abs() if dtype == torch.bfloat16 else 0)

    close(y.detach(), yr.detach(), bound(yr.detach(), 4 * rel * za * gab), "y")
    gz = gyd * gab * 1.2  # |dL/dz|, and its error relative to this plus that of act'(z): slopes up to 1.2
    gz_err = 8 * rel * gz * (1 + za)
    gx = gz * wd
    mean = lambda t: t.view(rows, groups, n).mean(-1, keepdim=True).expand(-1, -1, n).reshape(rows, C)  # noqa: E731
    r = rstd.expand(-1, -1, n).reshape(rows, C)
    ab = r * (gx * (1 + za) + mean(gx * (1 + za)) + (xhat + 1) * mean(gx * (1 + za) * (xhat + 1)))
    got = dict(zip(ins, grads))
    close(got["x"], want["x"], bound(want["x"], 16 * rel * ab), "d_x")
    n_rows = (rows + 64) * 2.0 ** -24
    wf = w.dtype == torch.float32
    uw = (lambda t: 0 if wf else u * t.abs())  # noqa: E731
    close(got["weight"], want["weight"], (gz_err * (xhat + 1) + gz * (xhat + 1) * (4 * rel + n_rows)).sum(0) + uw(want["weight"]), "d_weight")
    close(got["bias"], want["bias"], (gz_err + gz * n_rows).sum(0) + uw(want["bias"]), "d_bias")
    if gated:
        close(got["gate"], want["gate"], bound(want["gate"], 8 * rel * gyd * za * 1.2), "d_gate")


def test_group_norm_forms():
    """Leading dims, strided rows, one parameter alone, only some gradients, no rows."""
    from ttc_b200 import group_norm as gn
    z = _normal(0, 2, 5, 3 * 64 + 1)
    x, gate = z[..., :64], z[..., 65:129]  # strided rows; the gate's off the 16-byte grid
    w = _normal(1, 64)
    for kw in (dict(weight=w), dict(bias=w), dict(weight=w, bias=w), dict()):
        a = gn(x, 4, **kw, gate=gate, activation="silu")
        b = gn(x.contiguous(), 4, **kw, gate=gate.contiguous(), activation="silu")
        assert a.shape == x.shape
        ref = group_norm(x.double(), 4, None if "weight" not in kw else w.double(), None if "bias" not in kw else w.double(),
                         gate.double(), "silu", 1e-5)
        assert torch.allclose(a.double(), ref, rtol=1e-5, atol=1e-5)  # sums of 16, a few roundings of values below 20
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    g = gate.clone().requires_grad_()
    (d,) = torch.autograd.grad(gn(x, 4, w, gate=g, activation="silu").sum(), [g])
    ga = gate.double().requires_grad_()
    (dr,) = torch.autograd.grad(group_norm(x.double(), 4, w.double(), None, ga, "silu", 1e-5).sum(), [ga])
    assert torch.allclose(d.double(), dr, rtol=1e-5, atol=1e-5)
    p = w.clone().requires_grad_()
    y = gn(x[:0], 4, p)
    assert y.shape == (0, 5, 64)
    (dp,) = torch.autograd.grad(y.sum(), [p])
    assert torch.equal(dp, torch.zeros_like(dp))
    x0 = x.contiguous().requires_grad_()
    a, = torch.autograd.grad(gn(x0, 4, w).square().sum(), [x0], retain_graph=False)
    b, = torch.autograd.grad(gn(x0, 4, w).square().sum(), [x0])
    assert torch.equal(a, b)


def _memory(x, wq, wk, wv, wg, heads, key_heads, log_gamma, pos, inv, weight, ops):
    """A memory layer on x [B, T, C]: projections, rotary positions, attention with decays, gated group norm."""
    B, T, _ = x.shape
    q = (x @ wq).view(B, T, key_heads, -1)
    k = (x @ wk).view(B, T, key_heads, -1)
    v = (x @ wv).view(B, T, heads, -1)
    gate = x @ wg
    q, k = ops["rotary"](q, k, pos, inv)
    o, state = ops["attention"](q, k, v, log_gamma)
    return ops["norm"](o.reshape(B, T, -1), heads, weight, gate), state


def test_memory_layer_together():
    """Prompt forward and gradients against the same layer in 64 bits, and the same tokens one at a time."""
    import ttc_b200 as ours
    B, T, C, H, Hk, d = 2, 100, 64, 4, 2, 32
    names = ("x", "wq", "wk", "wv", "wg", "weight")
    vals = [_normal(i, *s) * c for i, (s, c) in enumerate([((B, T, C), 1.0), ((C, Hk * d), 0.125), ((C, Hk * d), 0.125),
                                                           ((C, H * d), 0.125), ((C, H * d), 0.125), ((H * d,), 1.0)])]
    inv, m = ours.rotary_frequencies(d, scaling="yarn", factor=4.0, original_length=64)
    lg = torch.log1p(-torch.exp2(-2.0 - torch.arange(H, device="cuda")))
    pos = torch.arange(T, device="cuda") + 1000
    gy = _normal(9, B, T, H * d)
    kernel = dict(rotary=lambda q, k, p, f: ours.rotary(q, k, p, f, magnitude=m),
                  attention=lambda q, k, v, g: ours.decay_attention(q, k, v, g, return_state=True),
                  norm=lambda o, n, w, g: ours.group_norm(o, n, w, gate=g, activation="silu"))
    turn = lambda t, p, f: torch.cat([t[..., :16] * torch.cos(p[:, None, None] * f) - t[..., 16:] * torch.sin(p[:, None, None] * f),  # noqa: E731,E501
                                      t[..., :16] * torch.sin(p[:, None, None] * f) + t[..., 16:] * torch.cos(p[:, None, None] * f)], -1) * m
    plain = dict(rotary=lambda q, k, p, f: (turn(q, p, f), turn(k, p, f)),
                 attention=lambda q, k, v, g: attention(q, k, v, g, d ** -0.5),
                 norm=lambda o, n, w, g: group_norm(o, n, w, None, g, "silu", 1e-5))
    torch.backends.cuda.matmul.allow_tf32 = False
    res = []
    for ops, dt in ((kernel, torch.float32), (plain, torch.float64)):
        ins = dict(zip(names, (t.detach().clone().to(dt).requires_grad_() for t in vals)))
        y, state = _memory(ins["x"], ins["wq"], ins["wk"], ins["wv"], ins["wg"], H, Hk, lg, pos, inv, ins["weight"], ops)
        res.append([y.detach(), state.detach(), *torch.autograd.grad(y, list(ins.values()), gy.to(dt))])
    for n, a, b in zip(("y", "state") + names, *res):
        # fp32 throughout, sums of at most B T terms of normalised values, the norm's 1/spread up to about 30: within
        # 2e-4 of the largest value (200 terms, 2^-23 each, through five operators)
        assert (a.double() - b).abs().max() <= 2e-4 * b.abs().max(), n
    # token after token
    x, wq, wk, wv, wg, weight = vals
    state = torch.zeros(B, H, d, d, device="cuda")
    for t in range(T):
        xt = x[:, t:t + 1]
        q, k = ours.rotary((xt @ wq).view(B, 1, Hk, d), (xt @ wk).view(B, 1, Hk, d), pos[t:t + 1], inv, magnitude=m)
        o = ours.decay_attention_step(q[:, 0], k[:, 0], (xt @ wv).view(B, H, d), lg, state)
        y = ours.group_norm(o.reshape(B, -1), H, weight, gate=(xt @ wg)[:, 0], activation="silu")
        assert (y - res[0][0][:, t]).abs().max() <= 2e-4 * res[0][0].abs().max()
    assert (state - res[0][1]).abs().max() <= 2e-4 * state.abs().max()
