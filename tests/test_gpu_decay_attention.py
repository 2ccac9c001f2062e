"""decay_attention (forward, backward, packed and segmented) and decay_attention_step against the
recurrence in 64 bits."""
import pytest
import torch
from sequence_ref import attention, attention_bounds, attention_grads, close

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _inputs(B, T, H, Hk, dk, dv, dtype, seed=0, n_state=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * T + dk)

    def normal(*s, dt=dtype):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    q, k, v, go = normal(B, T, Hk, dk), normal(B, T, Hk, dk), normal(B, T, H, dv), normal(B, T, H, dv)
    n = B if n_state is None else n_state
    start, gs = (normal(n, H, dk, dv, dt=torch.float32) for _ in range(2))
    log_gamma = -torch.rand(H, generator=g, device="cuda") * 0.2
    return q, k, v, log_gamma, go, start, gs


def _bounds(want, q, k, v, lg, scale, go, start, gs, dtype, T, cu=None):
    ab = [None if t is None else t.abs() for t in (go, start, gs)]
    absolute = attention_grads(q.abs(), k.abs(), v.abs(), lg, abs(scale), *ab, cu=cu)
    return attention_bounds(want, absolute, dtype, q.shape[-1], v.shape[-1], T // 64 + 1)


def _check(q, k, v, lg, go, start=None, gs=None, cu=None, scale=None):
    from ttc_b200 import decay_attention
    ins = {n: t.detach().requires_grad_() for n, t in dict(q=q, k=k, v=v, start=start).items() if t is not None}
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    o, state = decay_attention(ins["q"], ins["k"], ins["v"], lg, scale=scale, initial_state=ins.get("start"),
                               return_state=True, cu_seqlens=cut)
    outs, gos = ([o, state], [go, gs]) if gs is not None else ([o], [go])
    grads = torch.autograd.grad(outs, list(ins.values()), gos)
    s = q.shape[-1] ** -0.5 if scale is None else scale
    want = attention_grads(q, k, v, lg, s, go, start, gs, cu)
    bound = _bounds(want, q, k, v, lg, s, go, start, gs, q.dtype, v.shape[1], cu)
    got = {"o": o, "state": state, **{"d_" + n: g for n, g in zip(ins, grads)}}
    for n, x in got.items():
        assert x.dtype == (torch.float32 if n in ("state", "d_start") else q.dtype)
        close(x.detach(), want[n], bound[n], n)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 130])
@pytest.mark.parametrize("H,Hk,dk,dv", [(3, 3, 32, 32), (4, 2, 64, 64), (2, 1, 128, 128), (2, 2, 8, 128), (4, 4, 72, 16)])
def test_against_recurrence(H, Hk, dk, dv, T, dtype):
    q, k, v, lg, go, start, gs = _inputs(2, T, H, Hk, dk, dv, dtype)
    _check(q, k, v, lg, go, start, gs)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_without_states_and_with_a_scale(dtype):
    q, k, v, lg, go, _, _ = _inputs(3, 100, 2, 2, 48, 56, dtype)
    _check(q, k, v, lg, go, scale=-0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lens,tail", [([5, 0, 64, 1, 130], 7), ([0], 3), ([0, 0, 70], 0), ([1] * 40, 1)])
def test_packed(lens, tail, dtype):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v, lg, go, start, gs = _inputs(1, cu[-1] + tail, 4, 2, 40, 64, dtype, n_state=len(lens))
    _check(q, k, v, lg, go, start, gs, cu=cu)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("packed", [False, True])
def test_long_rows_are_split(packed, dtype):
    """Few long sequences: segments whose states are joined; a short and an empty one among them."""
    from ttc_b200 import _lib
    T = 2500
    cu = [0, 1700, 1700, 1765, T] if packed else None
    assert _lib.load().ttc_decay_attn_workspace(T, 4 if packed else 1, packed, 2, 2, 32, 64, 1, 0) > 0
    q, k, v, lg, go, start, gs = _inputs(1, T, 2, 2, 32, 64, dtype, n_state=4 if packed else 1)
    _check(q, k, v, lg * 0.05, go, start, gs, cu=cu)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_strided_operands(dtype):
    """Slices of one projection read in place, an expanded key, operands that have to be copied."""
    from ttc_b200 import decay_attention
    B, T, H, d = 2, 90, 4, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.randn(B, T, 3 * H * d + 3, generator=g, device="cuda").to(dtype)
    lg = torch.full((H,), -0.1, device="cuda")
    parts = {"fused": [z[..., i * H * d:(i + 1) * H * d].unflatten(-1, (H, d)) for i in range(3)],
             "odd": [z[..., 1 + i * H * d:1 + (i + 1) * H * d].unflatten(-1, (H, d)) for i in range(3)]}
    w = torch.randn(T, B, H, 3 * d, generator=g, device="cuda").to(dtype)
    parts["permuted"] = [w[..., i * d:(i + 1) * d].transpose(0, 1) for i in range(3)]
    parts["inner"] = [torch.randn(B, T, d, H, generator=g, device="cuda").to(dtype).transpose(2, 3) for _ in range(3)]
    parts["expanded"] = [parts["permuted"][0][:, :1].expand(-1, T, -1, -1)] + parts["permuted"][1:]
    for name, (q, k, v) in parts.items():
        a = decay_attention(q, k, v, lg)
        b = decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), lg)
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gradient_against_differences(dtype):
    """The loss is linear in v and in the start, bilinear in q and k: a central difference of the kernel's own loss in
    64-bit sums is its derivative up to the forward's roundings (bounded as its outputs are)."""
    from ttc_b200 import decay_attention
    q, k, v, lg, go, start, _ = _inputs(1, 150, 2, 1, 32, 32, dtype)
    go = go.float()
    ins = [t.detach().requires_grad_() for t in (q, k, v, start)]
    o = decay_attention(*ins[:3], lg, initial_state=ins[3])
    grads = torch.autograd.grad(o, ins, go.to(dtype))
    g = torch.Generator(device="cuda").manual_seed(9)
    for i in range(4):
        d = torch.randint(-1, 2, ins[i].shape, generator=g, device="cuda").to(ins[i].dtype)
        # a step of 1 / 2: x +- d / 2 may round in bf16, so the step that was made is used
        hi, lo = [t.detach() for t in ins], [t.detach() for t in ins]
        hi[i], lo[i] = (ins[i].detach() + d / 2).contiguous(), (ins[i].detach() - d / 2).contiguous()
        made = hi[i].double() - lo[i].double()
        outs = [decay_attention(*x[:3], lg, initial_state=x[3]) for x in (hi, lo)]
        diff = ((outs[0].double() - outs[1].double()) * go.to(dtype).double()).sum()
        slack = torch.zeros((), dtype=torch.float64, device="cuda")
        for x in (hi, lo):
            want = attention_grads(*x[:3], lg, 32 ** -0.5, go.to(dtype), x[3])
            b = _bounds(want, *x[:3], lg, 32 ** -0.5, go.to(dtype), x[3], None, dtype, 150)
            slack += (b["o"] * go.double().abs()).sum()
        name = ("d_q", "d_k", "d_v", "d_start")[i]
        slack += (b[name] * made.abs()).sum()
        assert abs((grads[i].double() * made).sum() - diff) <= slack, name


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_decay_limits(dtype):
    """gamma = 1 sums everything, gamma = 0 (log -inf) keeps nothing but the token itself."""
    from ttc_b200 import decay_attention
    q, k, v, _, go, start, _ = _inputs(1, 70, 2, 2, 32, 32, dtype)
    _check(q, k, v, torch.zeros(2, device="cuda"), go, start)
    lg = torch.full((2,), -float("inf"), device="cuda")
    o, state = decay_attention(q, k, v, lg, initial_state=start, return_state=True)
    own = (q.double() * k.double()).sum(-1, keepdim=True) * 32 ** -0.5 * v.double()
    ab = (q.double().abs() * k.double().abs()).sum(-1, keepdim=True) * 32 ** -0.5 * v.double().abs()
    close(o, own, 200 * 2.0 ** -23 * ab + (2.0 ** -8 * (own.abs() + 2 * ab) * 1.01 if dtype == torch.bfloat16 else 0), "o")
    last = k.double()[:, -1, :, :, None] * v.double()[:, -1, :, None, :]
    close(state, last, 2.0 ** -22 * last.abs(), "state")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", [0, 1, 2])
def test_later_tokens_do_not_reach_earlier_ones(where, bad, dtype):
    """Inf or NaN in token 40's q, k or v: tokens before it get what they get without it, token 40 (where it can
    be seen) and later ones something that is not finite; and the other way round in the backward."""
    from ttc_b200 import decay_attention
    q, k, v, lg, go, _, _ = _inputs(1, 100, 2, 2, 64, 64, dtype)
    clean = decay_attention(q, k, v, lg)
    ops = [q.clone(), k.clone(), v.clone()]
    ops[where][0, 40, 0, 3] = bad
    got = decay_attention(*ops, lg)
    # in the token's own block the values' product may run in another order: fp32 sums of 64 terms
    tol = 1e-5 if dtype == torch.float32 else 2.0 ** -7
    scale = clean.float().abs().max()
    assert ((got[:, :40].float() - clean[:, :40].float()).abs() <= tol * scale).all()
    assert torch.equal(got[:, :, 1], clean[:, :, 1])
    assert not torch.isfinite(got[0, 40, 0]).all()
    if where == 0:
        assert torch.equal(got[:, 41:], clean[:, 41:])
    # backward: gradients of tokens after 40 do not see token 40's g_o
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = decay_attention(*ins, lg)
    g2 = go.clone()
    g2[0, 40, 0, 3] = bad
    a = torch.autograd.grad(o, ins, go, retain_graph=True)
    b = torch.autograd.grad(o, ins, g2)
    for x, y in zip(a[1:], b[1:]):  # d_k, d_v of later tokens
        assert ((x[:, 41:].float() - y[:, 41:].float()).abs() <= tol * x.float().abs().max()).all()
    assert torch.isfinite(b[0][:, :40]).all() and torch.isfinite(b[0][:, 41:]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_empty(dtype):
    from ttc_b200 import decay_attention
    q, k, v, lg, go, start, _ = _inputs(2, 0, 4, 2, 32, 64, dtype)
    ins = [t.detach().requires_grad_() for t in (q, k, v, start)]
    o, state = decay_attention(*ins[:3], lg, initial_state=ins[3], return_state=True)
    assert o.shape == (2, 0, 4, 64) and torch.equal(state, start)
    grads = torch.autograd.grad(state, ins, torch.full_like(state, 2.0), allow_unused=True)
    assert torch.equal(grads[3], torch.full_like(start, 2.0))
    o, state = decay_attention(q[:0], k[:0], v[:0], lg, return_state=True)
    assert o.shape == (0, 0, 4, 64) and state.shape == (0, 4, 32, 64)


def test_bad_offsets_stay_inside():
    """Offsets that decrease or pass the row are cut: no sequence reads outside, no value is asked for."""
    from ttc_b200 import decay_attention
    q, k, v, lg, _, _, _ = _inputs(1, 200, 2, 2, 32, 32, torch.bfloat16)
    for cu in ([0, 500, 100], [-7, 90, 60, 1 << 30], [200, 200], [150, 20, 10]):
        o, state = decay_attention(q, k, v, lg, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                   return_state=True)
        torch.cuda.synchronize()
        assert o.shape == v.shape


def test_repeats_bit_by_bit_and_on_another_stream():
    from ttc_b200 import decay_attention
    q, k, v, lg, go, start, _ = _inputs(1, 3000, 4, 2, 64, 64, torch.bfloat16)
    ins = [t.detach().requires_grad_() for t in (q, k, v, start)]

    def call():
        o = decay_attention(*ins[:3], lg, initial_state=ins[3])
        return (o.detach(), *torch.autograd.grad(o, ins, go))

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_captured_forward_and_backward():
    """Two graphs of the same call, replayed in turn on new inputs."""
    from ttc_b200 import decay_attention
    ins = [t.detach().requires_grad_() for t in _inputs(1, 1500, 4, 2, 64, 64, torch.bfloat16)[:3]]
    lg = torch.full((4,), -0.02, device="cuda")
    go = torch.randn(1, 1500, 4, 64, device="cuda").bfloat16()

    def call():
        o = decay_attention(*ins, lg)
        return (o, *torch.autograd.grad(o, ins, go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = call()
        graphs.append((g, outs))
    for seed in (1, 2):
        with torch.no_grad():
            for t, new in zip(ins, _inputs(1, 1500, 4, 2, 64, 64, torch.bfloat16, seed=seed)):
                t.copy_(new)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_more_than_2_31_values():
    """Element offsets past 32 bits: 2^20 tokens of 17 heads of 128, the last tokens against a short call (a memory of 64
    tokens, gamma = e^-1/8: what is 4096 tokens back weighs e^-512)."""
    from ttc_b200 import decay_attention
    T, H = 1 << 20, 17
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(1, T, H, 8, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    v = torch.randn(1, T, H, 128, generator=g, device="cuda", dtype=torch.bfloat16)
    assert v.numel() > 1 << 31
    lg = torch.full((H,), -0.125, device="cuda")
    o = decay_attention(q, k, v, lg)
    tail = decay_attention(q[:, -8192:], k[:, -8192:], v[:, -8192:], lg)
    a, b = o[:, -4096:].float(), tail[:, -4096:].float()
    assert ((a - b).abs() <= 2.0 ** -7 * (b.abs() + b.abs().max())).all()


# --------------------------------------------------------------------------------- single tokens
def _step_inputs(B, n, H, Hk, dk, dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s, dt=dtype):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    return (normal(B, Hk, dk), normal(B, Hk, dk), normal(B, H, dv), -torch.rand(H, generator=g, device="cuda") * 0.2,
            normal(n, H, dk, dv, dt=torch.float32))


def _step_ref(q, k, v, lg, state, slots, scale):
    state, rep = state.double().clone(), v.shape[1] // q.shape[1]
    o = torch.zeros_like(v, dtype=torch.float64)
    for b, s in enumerate(slots):
        if 0 <= s < state.shape[0]:
            ob, new = attention(*(t[b:b + 1, None].double() for t in (q, k, v)), lg, scale, state[s:s + 1])
            o[b], state[s] = ob[0, 0], new[0]
    assert rep >= 1
    return o, state


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("H,Hk,dk,dv", [(4, 4, 64, 64), (6, 2, 128, 128), (1, 1, 8, 8), (5, 1, 40, 72)])
@pytest.mark.parametrize("slots", [None, [2, 0, 4, 1], [3, -1, 5, 1 << 30, 0], [1, 1, 0, 1, 0, 2], [0] * 9],
                         ids=["none", "permuted", "padding", "twice", "one"])
def test_step(H, Hk, dk, dv, slots, dtype):
    from ttc_b200 import decay_attention_step
    at = list(range(4)) if slots is None else slots
    q, k, v, lg, state = _step_inputs(len(at), 5, H, Hk, dk, dv, dtype)
    want_o, want_s = _step_ref(q, k, v, lg, state, at, dk ** -0.5)
    ab_o, ab_s = _step_ref(q.abs(), k.abs(), v.abs(), lg, state.abs(), at, dk ** -0.5)
    o = decay_attention_step(q, k, v, lg, state,
                             slots=None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda"))
    # an update rounds twice for each token of a slot; o sums dk terms and rounds to its type
    close(state, want_s, 3 * len(at) * 2.0 ** -24 * ab_s, "state")
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    close(o, want_o, (dk + 3 * len(at) + 8) * 2.0 ** -24 * ab_o + u * want_o.abs() * 1.01, "o")


def test_step_goes_on_from_a_prompt():
    from ttc_b200 import decay_attention, decay_attention_step
    q, k, v, lg, _, _, _ = _inputs(2, 80, 4, 2, 64, 64, torch.float32)
    whole, last = decay_attention(q, k, v, lg, return_state=True)
    cache = torch.full((5, 4, 64 * 64 + 8), 7.0, device="cuda")[..., :64 * 64].unflatten(-1, (64, 64))
    with pytest.raises(ValueError, match="contiguous"):  # heads of a state have to lie together
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lg, cache)
    cache = torch.full((5, 4 * 64 * 64 + 8), 7.0, device="cuda")[:, :4 * 64 * 64].unflatten(-1, (4, 64, 64))
    slots = torch.tensor([4, 1], dtype=torch.int32, device="cuda")
    _, cache[slots.long()] = decay_attention(q[:, :70], k[:, :70], v[:, :70], lg, return_state=True)
    before = cache._version
    for t in range(70, 80):
        o = decay_attention_step(q[:, t], k[:, t], v[:, t], lg, cache, slots=slots)
        # two orders of the same sums of up to 80 + 64 terms, of values below 100
        assert torch.allclose(o, whole[:, t], rtol=1e-5, atol=1e-4)
    assert cache._version > before
    assert torch.allclose(cache[slots.long()], last, rtol=1e-5, atol=1e-4)
    assert (cache[[0, 2, 3]] == 7).all()


def test_step_in_a_graph():
    from ttc_b200 import decay_attention_step
    q, k, v, lg, state = _step_inputs(3, 4, 4, 2, 64, 64, torch.bfloat16)
    slots = torch.tensor([0, 3, 1], dtype=torch.int32, device="cuda")
    eager = state.clone()
    decay_attention_step(q, k, v, lg, state.clone(), slots=slots)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = decay_attention_step(q, k, v, lg, state, slots=slots)
    for new in ([0, 3, 1], [2, 2, -1]):
        slots.copy_(torch.tensor(new, dtype=torch.int32))
        g.replay()
        want = decay_attention_step(q, k, v, lg, eager, slots=slots)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, eager)


def test_step_offsets_past_32_bits():
    from ttc_b200 import decay_attention_step
    n, H, d = 4200, 32, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    q, k, v, lg, one = _step_inputs(1, 1, H, H, d, d, torch.float32)
    state = torch.empty(n, H, d, d, device="cuda")
    assert state.numel() > 1 << 31
    state[n - 1] = one[0]
    o = decay_attention_step(q, k, v, lg, state, slots=torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    want = decay_attention_step(q, k, v, lg, one)
    assert torch.equal(o, want) and torch.equal(state[n - 1], one[0])
