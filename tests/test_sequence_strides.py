"""Strides that go to the C entries, on the CPU."""
import sys

import pytest
import torch


def _operands(dt):
    z = torch.zeros(2, 6, 101, dtype=dt)
    return [z[:1, :1, :32].unsqueeze(2),                                             # one token of one sequence and head
            torch.zeros(3, 161, dtype=dt)[:, :160].unflatten(1, (5, 2, 16))[:1],  # one sequence
            z[:1, :1, 1:33].unsqueeze(2),                                            # off the 16-byte grid, copied
            z[:, :0, :32].unsqueeze(2),                                              # nothing
            z[:, :, :32].unsqueeze(2),                                               # copied
            torch.zeros(6, 2, 3, 32, dtype=dt).transpose(0, 1),                      # read in place
            torch.zeros(2, 6, 3, 32, dtype=dt)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("at", range(7))
def test_strides_are_multiples_of_16_bytes(at, dtype):
    """What decay_attention passes on: the C entry refuses anything else.  Dims of more than one element keep theirs."""
    import ttc_b200  # noqa: F401
    module = sys.modules["ttc_b200.decay_attention"]
    t = module._operand(_operands(dtype)[at])
    strides = list(module._strides(t))
    assert len(strides) == 3 and all(s * t.element_size() % 16 == 0 for s in strides)
    assert t.numel() == 0 or all(s == r for s, r, n in zip(strides, t.stride(), t.shape) if n > 1)
