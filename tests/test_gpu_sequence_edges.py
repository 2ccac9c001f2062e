"""Calls of the sequence operators at the edges of what their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,T,Hk,H", [(1, 1, 1, 1), (1, 5, 2, 4), (1, 1, 1, 3), (3, 1, 1, 1), (2, 0, 2, 2)])
def test_slices_of_odd_projections(B, T, Hk, H, dtype):
    """Dims of one element (and all dims of nothing) count as contiguous whatever their strides: slices of a projection of
    odd width, forward and backward, are what their copies are."""
    from ttc_b200 import decay_attention, decay_attention_step
    dk, dv = 32, 16
    z = _normal(B + T, 3, 7, 2 * Hk * dk + H * dv + 3, dtype=dtype)[:B, :T]
    cuts = [z[..., :Hk * dk].unflatten(-1, (Hk, dk)), z[..., Hk * dk:2 * Hk * dk].unflatten(-1, (Hk, dk)),
            z[..., 2 * Hk * dk:2 * Hk * dk + H * dv].unflatten(-1, (H, dv))]
    lg = torch.linspace(-0.3, -0.1, H, device="cuda")
    start = _normal(9, B, H, dk, dv)
    res = []
    for ops in (cuts, [torch.empty(t.shape, dtype=dtype, device="cuda").copy_(t) for t in cuts]):
        ins = [t.detach().requires_grad_() for t in (*ops, start)]
        o, state = decay_attention(*ins[:3], lg, initial_state=ins[3], return_state=True)
        grads = torch.autograd.grad((o, state), ins, (torch.ones_like(o), torch.ones_like(state)))
        res.append([o.detach(), state.detach(), *grads])
        if T > 0:
            cache = start.clone()
            res[-1] += [decay_attention_step(*(t[:, 0] for t in ops), lg, cache), cache]
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_default_dtype_changes_nothing(default):
    from ttc_b200 import decay_attention, group_norm, rotary, rotary_frequencies
    pos, lg = torch.arange(100, device="cuda"), torch.tensor([-0.1, -0.2], device="cuda")
    ins = [_normal(i, 1, 100, 2, 32).requires_grad_() for i in range(3)] + [_normal(3, 1, 2, 32, 32).requires_grad_()]

    def call():
        f, _ = rotary_frequencies(32)
        q, k = rotary(ins[0], ins[1], pos, f)
        o, state = decay_attention(q, k, ins[2], lg, initial_state=ins[3], return_state=True)
        y = group_norm(o.flatten(2), 2, activation="silu")
        return [y, state, *torch.autograd.grad((y, state), ins, (torch.ones_like(y), torch.ones_like(state)))]

    want = call()
    torch.set_default_dtype(default)
    try:
        got = call()
    finally:
        torch.set_default_dtype(torch.float32)
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and torch.equal(a, b)


def test_a_timeout_is_reported_by_a_step_and_on_request():
    """The status word that a kernel would set, set from the host: a token's step raises and leaves its states alone."""
    import ctypes
    import sys

    import ttc_b200
    module = sys.modules["ttc_b200.decay_attention"]
    q, k, v = (_normal(i, 1, 10, 2, 32, dtype=torch.bfloat16) for i in range(3))
    lg = torch.tensor([-0.1, -0.2], device="cuda")
    _, state = ttc_b200.decay_attention(q, k, v, lg, return_state=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ttc_b200.decay_attention(q, k, v, lg)
    g.replay()
    ttc_b200.check_decay_attention()
    word, before = ctypes.c_int.from_address(module._status_word()), state.clone()
    word.value = 16
    with pytest.raises(RuntimeError, match="ran out"):
        ttc_b200.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lg, state)
    assert torch.equal(state, before)
    ttc_b200.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lg, state)
    assert not torch.equal(state, before)
    word.value = 16
    with pytest.raises(RuntimeError, match="ran out"):
        ttc_b200.check_decay_attention("cuda")
    ttc_b200.check_decay_attention(state.device)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("Hk", [1, 2])
def test_losses_on_some_of_the_outputs(monkeypatch, Hk, dtype):
    """Of (o, state): a loss on one is a loss on both with zeros for the other, and what is not there reaches the C
    entry as NULL."""
    import sys

    from ttc_b200 import decay_attention
    module = sys.modules["ttc_b200.decay_attention"]
    lg, seen, backward = torch.tensor([-0.1, -0.2], device="cuda"), [], module._backward

    def spy(*args):
        seen.append(args[8] is not None)  # the last state's gradient
        return backward(*args)

    monkeypatch.setattr(module, "_backward", spy)
    ins = [_normal(i, 2, 70, h, 32, dtype=dtype).requires_grad_() for i, h in enumerate((Hk, Hk, 2))]
    ins.append(_normal(7, 2, 2, 32, 32).requires_grad_())
    go, gs = _normal(8, 2, 70, 2, 32, dtype=dtype), _normal(9, 2, 2, 32, 32)

    def grads(outs, gos):
        o, state = decay_attention(*ins[:3], lg, initial_state=ins[3], return_state=True)
        return torch.autograd.grad([(o, state)[i] for i in outs], ins, gos)

    for outs, gos, both in (([0], [go], [go, torch.zeros_like(gs)]), ([1], [gs], [torch.zeros_like(go), gs])):
        for a, b in zip(grads(outs, gos), grads([0, 1], both)):
            assert torch.equal(a, b)
    assert seen == [False, True, True, True]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_losses_on_one_of_rotarys_outputs(dtype):
    from ttc_b200 import rotary, rotary_frequencies
    f, _ = rotary_frequencies(32)
    ins = [_normal(i, 2, 9, h, 32, dtype=dtype).requires_grad_() for i, h in enumerate((4, 2))]
    g = [_normal(5 + i, *t.shape, dtype=dtype) for i, t in enumerate(ins)]
    pos = torch.arange(9, device="cuda")
    want = torch.autograd.grad(rotary(*ins, pos, f), ins, g)
    for i in range(2):
        got = torch.autograd.grad(rotary(*ins, pos, f)[i], ins, g[i])
        assert torch.equal(got[i], want[i]) and got[1 - i].dtype == dtype and torch.equal(got[1 - i], torch.zeros_like(ins[1 - i]))
    # neither: an operator behind them that forms no gradient

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, b):
            return a.sum()

        @staticmethod
        def backward(ctx, g):
            return None, None

    for x in torch.autograd.grad(Nothing.apply(*rotary(*ins, pos, f)), ins, allow_unused=True):
        assert x is None


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [5, 1500])
def test_decays_that_are_not_numbers_show(T, dtype):
    """gamma = NaN: S_0 = NaN 0 + k v and all that follows, of this head alone; not the head without memory that a
    logarithm of -inf is."""
    from ttc_b200 import decay_attention, decay_attention_step
    q, k, v = (_normal(i, 1, T, 3, 32, dtype=dtype) for i in range(3))
    lg, clean = torch.tensor([-0.1, float("nan"), -0.2], device="cuda"), torch.tensor([-0.1, -0.3, -0.2], device="cuda")
    res = []
    for x in (lg, clean):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        o, state = decay_attention(*ins, x, return_state=True)
        step = state.detach().clone()
        one = decay_attention_step(q[:, 0], k[:, 0], v[:, 0], x, step)
        res.append([o.detach(), *torch.autograd.grad(o, ins, torch.ones_like(o)), state.detach().transpose(0, 1)[None],
                    one[:, None], step.transpose(0, 1)[None]])
    for i, (a, b) in enumerate(zip(*res)):  # heads are dim 2, of the states dim 1
        a, b = (a, b) if i not in (4, 6) else (a.transpose(1, 2), b.transpose(1, 2))
        assert torch.isnan(a[:, :, 1]).all()
        for h in (0, 2):
            assert torch.equal(a[:, :, h], b[:, :, h])


def test_default_device_changes_nothing(monkeypatch):
    """A program that builds its tensors on the GPU by default, from its first call on."""
    import sys

    import ttc_b200
    monkeypatch.setattr(sys.modules["ttc_b200.decay_attention"], "_status", {})
    q, k, v = (_normal(i, 1, 10, 2, 32, dtype=torch.bfloat16) for i in range(3))
    lg, pos = torch.tensor([-0.1, -0.2], device="cuda"), torch.arange(10, device="cuda")

    def call():
        f, _ = ttc_b200.rotary_frequencies(32, scaling="yarn", factor=2.0, original_length=100)
        a, b = ttc_b200.rotary(q, k, pos, f)
        return ttc_b200.group_norm(ttc_b200.decay_attention(a, b, v, lg).flatten(2), 2)

    with torch.device("cuda"):
        got = call()
    assert torch.equal(got, call())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [61, 8192, 30001])
@pytest.mark.parametrize("H,Hk,dk,dv", [(3, 3, 16, 40), (4, 2, 128, 64)])
def test_many_rows_behind_the_last_sequence(H, Hk, dk, dv, T, dtype):
    """A buffer of fixed size with a few rows in use: zeros behind them, in o and in every gradient, in memory that held
    something else, and the rows in use as they are alone."""
    from ttc_b200 import decay_attention
    cu = torch.tensor([0, 7, 7, 50], dtype=torch.int32, device="cuda")
    lg = torch.linspace(-0.3, -0.1, H, device="cuda")
    ins = [_normal(i, 1, T, h, d, dtype=dtype).requires_grad_() for i, (h, d) in enumerate(((Hk, dk), (Hk, dk), (H, dv)))]
    go = _normal(5, 1, T, H, dv, dtype=dtype)

    def call(ts, go):
        o = decay_attention(*ts, lg, cu_seqlens=cu)
        return [o.detach(), *torch.autograd.grad(o, ts, go)]

    want = call([t.detach()[:, :50].requires_grad_() for t in ins], go[:, :50])
    stale = [torch.full_like(t, float("nan")) for t in (*ins, *ins, go, go)]
    torch.cuda.synchronize()
    del stale  # what the outputs are allocated from
    for a, b in zip(call(ins, go), want):
        assert torch.equal(a[:, :50], b) and (a[:, 50:] == 0).all()


def _room(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB")


def test_gradients_of_more_than_2_31_values():
    """The last tokens of 2^20 against a short call: of decays by e^-1/8 a token, what is 4096 tokens away weighs e^-512."""
    from ttc_b200 import decay_attention
    _room(48)
    T, H = 1 << 20, 17
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(1, T, H, 8, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    v, go = (torch.randn(1, T, H, 128, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert v.numel() > 1 << 31
    lg, res = torch.full((H,), -0.125, device="cuda"), []
    for n in (T, 8192):
        ins = [t[:, -n:].detach().requires_grad_() for t in (q, k, v)]
        res.append([t[:, -4096:].float() for t in torch.autograd.grad(decay_attention(*ins, lg), ins, go[:, -n:])])
    for a, b in zip(*res):
        assert ((a - b).abs() <= 2.0 ** -7 * (b.abs() + b.abs().max())).all()


def test_rotary_of_more_than_2_31_values():
    from ttc_b200 import rotary, rotary_frequencies
    _room(24)
    T, H, D = (1 << 17) + 3, 129, 128
    q = torch.randn(1, T, H, D, device="cuda", dtype=torch.bfloat16).requires_grad_()
    assert q.numel() > 1 << 31
    f, _ = rotary_frequencies(64)
    pos = torch.arange(T, device="cuda")
    tail = q.detach()[:, -50:].requires_grad_()
    y, _ = rotary(q, None, pos, f)
    z, _ = rotary(tail, None, pos[-50:], f)
    assert torch.equal(y[:, -50:], z)
    a, = torch.autograd.grad(y, q, y.detach())
    b, = torch.autograd.grad(z, tail, z.detach())
    assert torch.equal(a[:, -50:], b)


@pytest.mark.parametrize("shift", [0, 1])
def test_group_norm_of_more_than_2_31_values(shift):
    """With 16-byte accesses, and one value at a time (rows off the 16-byte grid)."""
    from ttc_b200 import group_norm
    _room(40)
    rows, groups, n = (1 << 17) + 5, 41, 400
    C = groups * n
    x = torch.randn(rows * C + 1, device="cuda", dtype=torch.bfloat16)[shift:shift + rows * C].view(rows, C).requires_grad_()
    assert x.numel() > 1 << 31
    w = _normal(3, C, dtype=torch.bfloat16)
    tail = torch.empty(20 * C + 1, device="cuda", dtype=torch.bfloat16)[shift:shift + 20 * C].view(20, C).copy_(x.detach()[-20:]).requires_grad_()
    y, z = (group_norm(t, groups, w, activation="silu") for t in (x, tail))
    assert torch.equal(y[-20:], z)
    a, = torch.autograd.grad(y, x, y.detach())
    b, = torch.autograd.grad(z, tail, z.detach())
    assert torch.equal(a[-20:], b)
