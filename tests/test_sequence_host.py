"""What decay_attention, decay_attention_step, rotary and group_norm refuse, on the CPU: the C entry points before any
launch, the Python calls before the library; and the rotary frequencies against their formulas."""
import ctypes
import math

import pytest
import torch

P = 16  # a pointer that is never read: the calls are rejected before any launch


@pytest.fixture(scope="module")
def lib():
    import build as ttc_build
    from ttc_b200 import _lib
    ttc_build.build()
    return _lib.load()


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_decay_attention_abi_rejects_bad_arguments(lib):
    from ttc_b200 import _lib

    def fwd(q=P, o=P, fin=None, T=8, n=1, H=4, Hk=2, dk=16, dv=16, dtype=0, strides=_i64(*[64] * 9), cu=None, ws=None,
            nbytes=0):
        return lib.ttc_decay_attn_fwd(q, P, P, strides, P, 1.0, None, cu, T, n, H, Hk, dk, dv, dtype, o, fin, ws, nbytes,
                                      None, None)

    def bwd(g=P, dq=P, T=8, n=1, H=4, Hk=4, nbytes=0):
        return lib.ttc_decay_attn_bwd(P, P, P, _i64(*[64] * 9), g, P, 1.0, None, None, None, T, n, H, Hk, 16, 16, 0, dq, P, P,
                                      None, None, nbytes, None, None)

    assert fwd(T=-1) == _lib.ERR_INVALID
    assert fwd(T=1 << 31) == _lib.ERR_INVALID
    assert fwd(H=4, Hk=3) == _lib.ERR_INVALID
    assert fwd(H=0, Hk=1) == _lib.ERR_INVALID
    assert fwd(n=1 << 20, H=4) == _lib.ERR_INVALID
    assert fwd(dtype=3) == _lib.ERR_INVALID
    assert fwd(dk=12) == _lib.ERR_UNSUPPORTED
    assert fwd(dv=136) == _lib.ERR_UNSUPPORTED
    assert b"multiples of 8" in lib.ttc_last_error()
    assert fwd(q=None) == _lib.ERR_INVALID
    assert fwd(q=8) == _lib.ERR_INVALID                      # misaligned
    assert fwd(strides=_i64(*[6] * 9)) == _lib.ERR_INVALID   # rows off the 16-byte grid
    assert fwd(n=0, cu=P) == _lib.ERR_INVALID                # packed rows without a sequence
    assert fwd(n=0) == _lib.OK
    assert fwd(q=None, o=None, T=0) == _lib.OK               # no token and no state asked for
    assert fwd(T=1 << 20, H=1, Hk=1) == _lib.ERR_INVALID     # a long row needs a workspace
    assert b"workspace" in lib.ttc_last_error()
    assert bwd(g=None) == _lib.ERR_INVALID
    assert bwd(dq=None) == _lib.ERR_INVALID
    assert bwd(Hk=2) == _lib.ERR_INVALID                     # shared heads need a workspace
    assert bwd(n=0) == _lib.OK


def test_decay_attention_workspace(lib):
    from ttc_b200 import _lib
    size = lib.ttc_decay_attn_workspace
    assert size(64, 1, 0, 4, 4, 16, 16, 1, 0) == 0
    assert size(64, 3, 0, 4, 2, 16, 16, 1, 1) == 2 * 3 * 64 * 4 * 16 * 4  # the shared heads' gradients
    long_ = size(1 << 20, 1, 0, 1, 1, 64, 64, 1, 0)
    assert long_ > 0 and long_ % (64 * 64 * 4) == 0
    assert size(64, 1, 0, 4, 3, 16, 16, 1, 0) == -_lib.ERR_INVALID
    assert size(64, 1, 0, 4, 4, 20, 16, 1, 0) == -_lib.ERR_UNSUPPORTED


def test_step_abi_rejects_bad_arguments(lib):
    from ttc_b200 import _lib

    def step(state=P, stride=4096, slots=P, B=2, n=2, H=4, Hk=4, dk=16, dv=16, dtype=0, o=P):
        return lib.ttc_decay_attn_step(P, P, P, _i64(*[3] * 6), P, 1.0, state, stride, slots, B, n, H, Hk, dk, dv, dtype, o,
                                       None)

    assert step(B=-1) == _lib.ERR_INVALID
    assert step(n=1, slots=None) == _lib.ERR_INVALID
    assert step(state=8) == _lib.ERR_INVALID
    assert step(stride=4097) == _lib.ERR_INVALID
    assert step(dk=4) == _lib.ERR_UNSUPPORTED
    assert step(o=None) == _lib.ERR_INVALID
    assert step(B=0) == _lib.OK


def test_rotary_abi_rejects_bad_arguments(lib):
    from ttc_b200 import _lib

    def rot(q=P, Hq=2, k=P, Hk=2, B=1, T=4, D=16, half=8, dtype=0, pos=P, inv=P, out=P):
        s = _i64(64, 32, 16)
        return lib.ttc_rotary(q, s, Hq, k, s, Hk, pos, _i64(4, 1), 1, inv, B, T, D, half, 0, 0, 1.0, dtype, out, P, None)

    assert rot(B=-1) == _lib.ERR_INVALID
    assert rot(B=1 << 20, T=1 << 20) == _lib.ERR_INVALID
    assert rot(Hq=0) == _lib.ERR_INVALID
    assert rot(D=16, half=9) == _lib.ERR_UNSUPPORTED
    assert rot(D=514, half=8) == _lib.ERR_UNSUPPORTED
    assert rot(dtype=2) == _lib.ERR_INVALID
    assert rot(k=None) == _lib.ERR_INVALID
    assert rot(inv=None) == _lib.ERR_INVALID
    assert rot(out=None) == _lib.ERR_INVALID
    assert rot(T=0) == _lib.OK


def test_group_norm_abi_rejects_bad_arguments(lib):
    from ttc_b200 import _lib

    def fwd(x=P, rows=2, groups=2, n=8, act=0, dtype=0, y=P):
        return lib.ttc_group_norm_fwd(x, 16, None, 0, None, None, 0, rows, groups, n, act, 1e-5, dtype, y, None)

    def bwd(g=P, gate=None, dgate=None, dw=None, ws=None, nbytes=0, rows=2):
        return lib.ttc_group_norm_bwd(P, 16, gate, 16, None, None, 0, g, rows, 2, 8, 0, 1e-5, 0, P, dgate, dw, None, ws, nbytes,
                                      None)

    assert fwd(rows=-1) == _lib.ERR_INVALID
    assert fwd(groups=0) == _lib.ERR_INVALID
    assert fwd(n=1025) == _lib.ERR_UNSUPPORTED
    assert fwd(groups=70000) == _lib.ERR_UNSUPPORTED
    assert fwd(act=3) == _lib.ERR_INVALID
    assert fwd(dtype=9) == _lib.ERR_INVALID
    assert fwd(x=None) == _lib.ERR_INVALID
    assert fwd(y=None) == _lib.ERR_INVALID
    assert fwd(rows=0) == _lib.OK
    assert bwd(g=None) == _lib.ERR_INVALID
    assert bwd(dgate=P) == _lib.ERR_INVALID          # a gate's gradient without the gate
    assert bwd(dw=P) == _lib.ERR_INVALID             # no workspace
    assert bwd(rows=0) == _lib.OK
    assert lib.ttc_group_norm_workspace(16384, 32, 128, 1) > 0


def _qkv(B=2, T=3, Hk=2, H=4, dk=16, dv=8, dtype=torch.float32):
    return torch.zeros(B, T, Hk, dk, dtype=dtype), torch.zeros(B, T, Hk, dk, dtype=dtype), torch.zeros(B, T, H, dv, dtype=dtype)


def test_decay_attention_refuses():
    from ttc_b200 import decay_attention
    q, k, v = _qkv()
    lg = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        decay_attention(q, k, v, lg)
    with pytest.raises(TypeError):
        decay_attention(q.half(), k.half(), v.half(), lg)
    with pytest.raises(TypeError, match="one dtype"):
        decay_attention(q.bfloat16(), k, v, lg)
    with pytest.raises(ValueError, match="dimensions"):
        decay_attention(q[0], k[0], v[0], lg)
    with pytest.raises(ValueError, match="match"):
        decay_attention(q, k[:, :2], v, lg)
    with pytest.raises(ValueError, match="multiple"):
        decay_attention(q, k, v[:, :, :3], torch.zeros(3))
    with pytest.raises(ValueError, match="log_gamma"):
        decay_attention(q, k, v, torch.zeros(2))
    with pytest.raises(ValueError, match="gradient"):
        decay_attention(q, k, v, lg.requires_grad_())
    lg = torch.zeros(4)
    with pytest.raises(ValueError, match="initial_state"):
        decay_attention(q, k, v, lg, initial_state=torch.zeros(2, 4, 8, 16))
    with pytest.raises(ValueError, match="batch of 1"):
        decay_attention(q, k, v, lg, cu_seqlens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32"):
        decay_attention(q[:1], k[:1], v[:1], lg, cu_seqlens=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="int32"):
        decay_attention(q[:1], k[:1], v[:1], lg, cu_seqlens=torch.zeros(1, dtype=torch.int32))


def test_decay_attention_step_refuses():
    from ttc_b200 import decay_attention_step
    q, k, v = (t[:, 0] for t in _qkv())
    lg, state = torch.zeros(4), torch.zeros(3, 4, 16, 8)
    with pytest.raises(ValueError, match="CUDA"):
        decay_attention_step(q, k, v, lg, state)
    with pytest.raises(ValueError, match="states"):
        decay_attention_step(q, k, v, lg, state[:1])
    with pytest.raises(ValueError, match="float32"):
        decay_attention_step(q, k, v, lg, state.double())
    with pytest.raises(ValueError, match="contiguous"):
        decay_attention_step(q, k, v, lg, state.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="contiguous"):
        decay_attention_step(q, k, v, lg, state[:1].expand(3, -1, -1, -1))  # one state under three numbers
    with pytest.raises(ValueError, match="slots"):
        decay_attention_step(q, k, v, lg, state, slots=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="gradient"):
        decay_attention_step(q.clone().requires_grad_(), k, v, lg, state)


def test_rotary_refuses():
    from ttc_b200 import rotary
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 1, 16)
    pos, f = torch.arange(3), torch.ones(8, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        rotary(q, k, pos, f)
    with pytest.raises(TypeError):
        rotary(q.double(), None, pos, f)
    with pytest.raises(TypeError, match="positions"):
        rotary(q, k, pos.float(), f)
    with pytest.raises(ValueError, match="positions"):
        rotary(q, k, torch.arange(2), f)
    with pytest.raises(ValueError, match="match"):
        rotary(q, k[:, :2], pos, f)
    with pytest.raises(ValueError, match="inv_freq"):
        rotary(q, k, pos, f.float())
    with pytest.raises(ValueError, match="inv_freq"):
        rotary(q, k, pos, torch.ones(9, dtype=torch.float64))
    with pytest.raises(ValueError, match="heads"):
        rotary(q[0], None, pos, f)


def test_group_norm_refuses():
    from ttc_b200 import group_norm
    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    with pytest.raises(ValueError, match="CUDA"):
        group_norm(x, 4, w)
    with pytest.raises(TypeError):
        group_norm(x.half(), 4)
    with pytest.raises(ValueError, match="groups"):
        group_norm(x, 3)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 4, activation="relu")
    with pytest.raises(ValueError, match="gate"):
        group_norm(x, 4, gate=x[:1])
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, 4, w[:4])
    with pytest.raises(ValueError, match="weight"):
        group_norm(x.bfloat16(), 4, w, w.bfloat16())


def test_rotary_frequencies():
    from ttc_b200 import rotary_frequencies
    f, m = rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    lin, _ = rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, f / 4)
    ntk, _ = rotary_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4 / f[-1] - 1) < 1e-12  # first pair kept, last divided by the factor
    yarn, m = rotary_frequencies(8, scaling="yarn", factor=4.0, original_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert yarn[0] == f[0] and turns[0] > 32            # many turns: kept
    assert abs(yarn[3] * 4 / f[3] - 1) < 1e-12 and turns[3] < 1  # under one turn: divided
    assert f[2] / 4 < yarn[2] < f[2]
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-15
    for bad in (dict(rot_dim=7), dict(rot_dim=8, scaling="x"), dict(rot_dim=8, scaling="yarn", factor=2.0),
                dict(rot_dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad, device="cpu")
