"""Calls of the sequence operators into the library: latency counts for single tokens, so a call is made with
the raw handle of the current stream, and autograd's machinery only where a gradient is asked for.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib, solver


def launch(name, dev, fn, *args) -> None:
    """fn(*args, stream) on the current stream of ``dev``, which has to be the current device; reported to the
    solver's kernel timer where one is installed."""
    if solver._timer is not None:
        solver._launch(name, dev, fn, *args)
        return
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _lib.check(rc)


def on_device(dev, f, *args):
    """f(*args) with ``dev`` as the current device."""
    if torch._C._cuda_getDevice() == dev.index:
        return f(*args)
    with torch.cuda.device(dev):
        return f(*args)


def refuse_tangents(name, **operands) -> None:
    """Raises where an operand carries a forward-mode tangent.  The kernels write into new tensors, which
    have none, and a dual tensor need not require a gradient: the result would pass for a constant."""
    # the number of the innermost dual level, negative outside of all (this costs 0.13 us there)
    if forward_ad._current_level < 0 or not torch._C._is_fwd_grad_enabled():
        return
    for n, t in operands.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"ttc_b200 {name} has no forward-mode derivative: {n} carries a tangent")


def refuse_gradient(name, **fixed) -> None:
    """Raises where one of ``fixed`` (numbers, or tensors in their place) asks for a gradient: there is none."""
    for n, t in fixed.items():
        if isinstance(t, torch.Tensor):
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"ttc_b200 {name}: {n} is fixed, it must not require a gradient")
            refuse_tangents(name, **{n: t})


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
