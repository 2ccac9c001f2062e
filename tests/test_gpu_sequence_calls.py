"""The sequence operators as programs call them: packed neighbours that are not finite, two streams at once,
graphs whose offsets and inputs change, a first call inside a capture, a reported timeout."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch
from test_gpu_decay_attention import _check, _inputs

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _normal(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _decays(H):
    return torch.linspace(-0.3, -0.01, H, device="cuda")


def _cut(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 40), (24, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_packed_neighbours_do_not_reach_each_other(dtype, dk, dv, bad):
    """Sequences between others (and in front of rows behind the last) that hold nothing but NaN or Inf, states and
    output gradients among it: bit for bit what they are beside finite ones."""
    from ttc_b200 import decay_attention
    lens, poisoned, tail, H = [70, 64, 33, 1, 130, 5, 200], (1, 3, 4, 6), 9, 2
    cu, T = _cut(lens), sum(lens) + tail
    clean = [_normal(i, 1, T, H, d, dtype=dtype) for i, d in enumerate((dk, dk, dv, dv))]  # q, k, v, g_o
    clean += [_normal(9 + i, len(lens), H, dk, dv, dtype=torch.float32) for i in range(2)]  # start, its end's gradient
    rows = torch.zeros(T, dtype=torch.bool, device="cuda")
    rows[sum(lens):] = True
    for n in poisoned:
        rows[sum(lens[:n]):sum(lens[:n + 1])] = True

    def call(ts):
        q, k, v, go, start, gs = ts
        ins = [t.detach().requires_grad_() for t in (q, k, v, start)]
        o, end = decay_attention(*ins[:3], _decays(H), initial_state=ins[3], cu_seqlens=cu, return_state=True)
        return [o.detach(), end.detach(), *torch.autograd.grad((o, end), ins, (go, gs))]

    dirty = [t.clone() for t in clean]
    for t in dirty[:4]:
        t[0, rows] = bad
    for t in dirty[4:]:
        t[list(poisoned)] = bad
    others = [n for n in range(len(lens)) if n not in poisoned]
    for i, (a, b) in enumerate(zip(call(clean), call(dirty))):
        if i in (1, 5):
            assert torch.equal(a[others], b[others])
        else:
            assert torch.equal(a[0, ~rows], b[0, ~rows])
            assert (b[0, sum(lens):] == 0).all()


def test_two_streams_at_once():
    """Calls that run beside each other, segmented ones with workspaces among them, give what they give alone."""
    from ttc_b200 import decay_attention, group_norm, rotary, rotary_frequencies
    lg, (f, _) = _decays(4), rotary_frequencies(64)
    pos = torch.arange(3000, device="cuda")

    def call(x):
        q, k, v = (t.detach().requires_grad_() for t in x)
        a, b = rotary(q, k, pos, f)
        o = decay_attention(a, b, v, lg)
        y = group_norm(o.flatten(2), 4, gate=v.flatten(2), activation="silu")
        return [y.detach(), *torch.autograd.grad(y, (q, k, v), torch.ones_like(y))]

    inputs = [[_normal(10 * s + i, 1, 3000, 4, 64) for i in range(3)] for s in range(2)]
    want = [call(x) for x in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = []
        for s, x in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_captured_packed_call_with_other_offsets(dtype):
    """The offsets are read on the device: a graph takes other lengths and values at its replay."""
    from ttc_b200 import decay_attention
    q, k, v = (_normal(i, 1, 700, 2, 32, dtype=dtype) for i in range(3))
    cu, lg = _cut([100, 500, 64, 36]), _decays(2)

    def call():
        return decay_attention(q, k, v, lg, cu_seqlens=cu, return_state=True)

    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = call()
    for lens in ([100, 500, 64, 36], [0, 700, 0, 0], [1, 2, 3, 4], [175] * 4):
        cu.copy_(_cut(lens))
        v.copy_(_normal(len(lens) + lens[0], *v.shape, dtype=dtype))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call()):
            assert torch.equal(a, b)


def test_captured_rotary_and_norm():
    from ttc_b200 import group_norm, rotary, rotary_frequencies
    f, _ = rotary_frequencies(32)
    pos = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    q, k = (_normal(i, 2, 5, 3, 48).requires_grad_() for i in range(2))
    w = _normal(3, 144).requires_grad_()

    def call():
        a, b = rotary(q, k, pos, f, interleaved=True)
        y = group_norm(a.flatten(2), 3, weight=w, activation="gelu")
        return [y, *torch.autograd.grad((y, b), (q, k, w), (torch.ones_like(y), torch.ones_like(b)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = call()
    for first in (0, 1 << 33):
        pos.copy_(first + torch.arange(10, device="cuda").view(2, 5))
        with torch.no_grad():
            q.copy_(_normal(first % 97, *q.shape))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call()):
            assert torch.equal(a, b)


def test_first_call_inside_a_capture():
    """Nothing that a first call sets up is forbidden in a capture."""
    code = """
import torch, ttc_b200
q, k, v = (torch.randn(1, 100, 2, 64, device="cuda").bfloat16() for _ in range(3))
lg = torch.full((2,), -0.05, device="cuda")
st = torch.zeros(1, 2, 64, 64, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o = ttc_b200.decay_attention(q, k, v, lg)
    s = ttc_b200.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lg, st)
g.replay()
torch.cuda.synchronize()
assert torch.equal(o, ttc_b200.decay_attention(q, k, v, lg))
print("same")
"""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ttc-net_b200")
    env = dict(os.environ, PYTHONPATH=root + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_a_timeout_is_reported_at_the_next_call():
    """The status word that a kernel would set, set from the host: one call raises, the next one works."""
    import ttc_b200
    module = sys.modules["ttc_b200.decay_attention"]
    q, k, v = (_normal(i, 1, 10, 2, 32) for i in range(3))
    want = ttc_b200.decay_attention(q, k, v, _decays(2))
    torch.cuda.synchronize()
    ctypes.c_int.from_address(module._status_word()).value = 1
    with pytest.raises(RuntimeError, match="ran out"):
        ttc_b200.decay_attention(q, k, v, _decays(2))
    assert torch.equal(ttc_b200.decay_attention(q, k, v, _decays(2)), want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lens", [[3] * 50 + [2100] + [70] * 9, [7] * 333])
def test_many_packed_sequences(lens, dtype):
    """More sequences than a warp looks at in one turn, one of them cut into segments; and more than there are CTAs."""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v, lg, go, start, gs = _inputs(1, cu[-1] + 2, 1, 1, 32, 64, dtype, n_state=len(lens))
    _check(q, k, v, lg, go, start, gs, cu=cu)


def test_autocast_changes_nothing():
    """Types are the operands' own, forward and backward, whatever autocast is set around either."""
    from ttc_b200 import decay_attention, group_norm, rotary, rotary_frequencies
    f, _ = rotary_frequencies(32)
    pos, lg = torch.arange(90, device="cuda"), _decays(2)
    ins = [_normal(i, 2, 90, 2, 32, dtype=torch.float32).requires_grad_() for i in range(3)]

    def call():
        q, k = rotary(ins[0], ins[1], pos, f)
        y = group_norm(decay_attention(q, k, ins[2], lg).flatten(2), 2, activation="silu")
        return [y, *torch.autograd.grad(y, ins, torch.ones_like(y))]

    want = call()
    with torch.autocast("cuda", torch.bfloat16):
        got = call()
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and torch.equal(a, b)
