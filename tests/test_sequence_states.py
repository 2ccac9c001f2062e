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
