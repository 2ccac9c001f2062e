"""Derivatives that the sequence operators do not form are refused, not left out: on the CPU, before the library."""
import sys

import pytest
import torch
from torch.autograd import forward_ad


def _attention():
    g = torch.zeros
    return dict(q=g(2, 3, 2, 16), k=g(2, 3, 2, 16), v=g(2, 3, 4, 8), log_gamma=g(4), initial_state=g(2, 4, 16, 8))


def _step():
    g = torch.zeros
    return dict(q=g(2, 2, 16), k=g(2, 2, 16), v=g(2, 4, 8), log_gamma=g(4), state=g(2, 4, 16, 8))


def _rotary():
    return dict(q=torch.zeros(2, 3, 4, 16), k=torch.zeros(2, 3, 1, 16), positions=torch.arange(3),
                inv_freq=torch.ones(8, dtype=torch.float64))


def _norm():
    return dict(x=torch.zeros(2, 16), num_groups=2, weight=torch.ones(16), bias=torch.zeros(16), gate=torch.zeros(2, 16))


OPERATORS = [("decay_attention", _attention), ("decay_attention_step", _step), ("rotary", _rotary), ("group_norm", _norm)]
CASES = [(name, make, n) for name, make in OPERATORS for n, t in make().items()
         if isinstance(t, torch.Tensor) and t.is_floating_point()]


@pytest.mark.parametrize("name,make,operand", CASES, ids=[f"{c[0]}-{c[2]}" for c in CASES])
def test_tangents_are_refused(name, make, operand):
    """A dual tensor needs no gradient in the backward's sense, so nothing else stops a result without its tangent."""
    import ttc_b200
    call, args = getattr(ttc_b200, name), make()
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="CUDA"):  # without tangents it gets as far as the device
            call(**args)
        args[operand] = forward_ad.make_dual(args[operand], torch.ones_like(args[operand]))
        with pytest.raises(NotImplementedError, match=f"{name}.*{operand}.*tangent"):
            call(**args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):  # which leaves tangents alone
            call(**args)
        with torch.inference_mode(), pytest.raises(ValueError, match="CUDA"):  # which does not
            call(**args)


@pytest.mark.parametrize("name,function,grads", [("decay_attention", "DecayAttentionFunction", 2), ("rotary", "RotaryFunction", 2),
                                                 ("group_norm", "GroupNormFunction", 1)])
def test_tangents_of_gradients_are_refused(name, function, grads):
    """Forward over reverse: a gradient that comes in with a tangent, at the first thing that a backward does."""
    import ttc_b200  # noqa: F401
    backward = getattr(sys.modules[f"ttc_b200.{name}"], function).backward
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        for at in range(grads):
            gs = [None] * grads
            gs[at] = dual
            with pytest.raises(NotImplementedError, match=f"{name}.*tangent"):
                backward(None, *gs)


FIXED = [("rotary", _rotary, "inv_freq"), ("rotary", _rotary, "magnitude"), ("decay_attention", _attention, "log_gamma"),
         ("decay_attention", _attention, "scale"), ("decay_attention_step", _step, "log_gamma"),
         ("decay_attention_step", _step, "scale"), ("group_norm", _norm, "eps")]


@pytest.mark.parametrize("name,make,operand", FIXED, ids=[f"{c[0]}-{c[2]}" for c in FIXED])
def test_what_has_no_gradient_may_not_ask_for_one(name, make, operand):
    """Decays, frequencies and factors are fixed: a leaf in their place would get no gradient."""
    import ttc_b200
    call, args = getattr(ttc_b200, name), make()
    args[operand] = args.get(operand, torch.tensor(0.5)).clone()
    with pytest.raises(ValueError, match="CUDA"):
        call(**args)
    args[operand].requires_grad_()
    with pytest.raises(ValueError, match=f"{operand}.* gradient"):
        call(**args)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(**args)
    with forward_ad.dual_level():
        args[operand] = forward_ad.make_dual(args[operand].detach(), torch.ones_like(args[operand]))
        with pytest.raises(NotImplementedError, match="tangent"):
            call(**args)
