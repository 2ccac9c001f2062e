"""What decay_attention hands to the C entries for states, on the CPU with the launch taken out."""
import sys

import pytest
import torch


@pytest.fixture
def module(monkeypatch):
    import build as ttc_build
    import ttc_b200  # noqa: F401
    ttc_build.build()
    m = sys.modules["ttc_b200.decay_attention"]
    monkeypatch.setattr(m, "launch", lambda *a: None)
    monkeypatch.setattr(m, "_status_word", lambda *a: 0)
    return m


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_states_are_float32_whatever_the_default_dtype(module, default):
    """The kernels write 4 bytes for each element of a state: fewer in its buffer would be written over."""
    q, k, v = torch.zeros(1, 3, 2, 16), torch.zeros(1, 3, 2, 16), torch.zeros(1, 3, 2, 8)
    lg, start = torch.zeros(2), torch.zeros(1, 2, 16, 8)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        o, state = module._forward(q, k, v, lg, 1.0, None, None, True)
        grads = module._backward(q, k, v, lg, 1.0, start, None, torch.zeros_like(v), None, True)
    finally:
        torch.set_default_dtype(before)
    assert state.dtype == torch.float32 and state.shape == start.shape
    assert all(t.dtype == torch.float32 for t in (o, *grads)) and grads[3].shape == start.shape


def test_a_timeout_belongs_to_its_device(monkeypatch):
    """Two devices' words, held in ordinary memory: a report is raised for the device that has it, once."""
    import ctypes

    import ttc_b200
    m = sys.modules["ttc_b200.decay_attention"]
    words = [torch.zeros(1, dtype=torch.int32) for _ in range(2)]
    monkeypatch.setattr(m, "_status", {i: (w, ctypes.c_int.from_address(w.data_ptr()), w.data_ptr())
                                       for i, w in enumerate(words)})
    synced = []
    monkeypatch.setattr(torch.cuda, "synchronize", synced.append)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    assert m._status_word(0) == words[0].data_ptr() and m._status_word() == words[0].data_ptr()
    words[1][0] = 16
    assert m._status_word(0) == words[0].data_ptr()
    m._raise_timeout(0)
    m._raise_timeout(7)  # a device that had no call
    ttc_b200.check_decay_attention()
    with pytest.raises(RuntimeError, match="ran out.*cuda:1"):
        m._status_word(1)
    assert m._status_word(1) == words[1].data_ptr()
    for device in ("cuda:1", torch.device("cuda", 1), 1):
        words[1][0] = 16
        with pytest.raises(RuntimeError, match="ran out.*cuda:1"):
            ttc_b200.check_decay_attention(device)
        ttc_b200.check_decay_attention(device)
    assert synced == [0] + [1] * 6
    q, state = torch.zeros(1, 1, 8), torch.zeros(1, 1, 8, 8)
    q_on_1 = type("OnOne", (), {"device": torch.device("cuda", 1), "new_empty": None})
    words[1][0] = 16
    with pytest.raises(RuntimeError, match="ran out.*cuda:1"):  # a token's step, before anything else
        m._step(q_on_1, q, q, None, 1.0, state, 64, None, ())


def test_sizes_of_packed_rows_are_the_rows(module):
    """A packed row has T tokens in all: a long one of many sequences is no larger than its blocks and sequences."""
    from ttc_b200 import _lib
    size = _lib.load().ttc_decay_attn_workspace
    assert size(1 << 21, 131000, 1, 8, 8, 16, 16, _lib.DTYPE_BF16, 0) == 0
    assert size(1 << 28, 1000, 1, 8, 8, 16, 16, _lib.DTYPE_F32, 0) == 0
    assert size((1 << 31) - 65, 1 << 20, 1, 1, 1, 16, 16, _lib.DTYPE_F32, 0) == -_lib.ERR_INVALID  # sequences x heads
    assert size(1 << 21, 131000, 0, 8, 8, 16, 16, _lib.DTYPE_BF16, 0) == -_lib.ERR_INVALID  # 2^38 tokens
    assert size((1 << 31) - 65, 1000, 1, 8, 8, 16, 16, _lib.DTYPE_F32, 0) == 0


def test_outputs_off_the_16_byte_grid_are_rejected():
    """Before any launch: the pointers are never read."""
    import ctypes

    from ttc_b200 import _lib
    lib, strides = _lib.load(), (ctypes.c_int64 * 9)(*[64] * 9)
    for dtype in (_lib.DTYPE_F32, _lib.DTYPE_BF16):
        assert lib.ttc_decay_attn_fwd(16, 16, 16, strides, 16, 1.0, None, None, 8, 1, 4, 4, 16, 16, dtype, 8, None, None, 0, None,
                                      None) == _lib.ERR_INVALID
        for at in range(3):
            outs = [16 if i != at else 24 for i in range(3)]
            assert lib.ttc_decay_attn_bwd(16, 16, 16, strides, 16, 16, 1.0, None, None, None, 8, 1, 4, 4, 16, 16, dtype, *outs, None,
                                          None, 0, None, None) == _lib.ERR_INVALID
        assert b"aligned" in lib.ttc_last_error()
