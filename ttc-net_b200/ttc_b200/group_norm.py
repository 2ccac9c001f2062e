"""Group norm over the channels of each token, with an activation or a gate: the norm of the
heads' outputs behind ``decay_attention``, beside the l2norm of the TTC layer's epilogue
(``epilogue.py``).  One CUDA kernel forward (``ttc_group_norm_fwd``), one backward and a small sum over
rows for the parameters (``ttc_group_norm_bwd``, which recomputes the statistics).  No counterpart in the reference;
no fallback: without the CUDA library this raises.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import launch, on_device, refuse_gradient, refuse_tangents, wants_grad
from .decay_attention import _workspace
from .solver import _DTYPES, _ptr

_ACTS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}


def _rows(t, C):
    """t as [rows, C] with contiguous channels, a view where its strides allow."""
    t = t if t.dim() == 2 else t.reshape(-1, C)
    return t if t.stride(1) == 1 or C == 1 else t.contiguous()


def _dims(x, weight, bias, groups, act, eps):
    """((rows, groups, channels of a group, act, eps, dtype code), whether the parameters are float32)"""
    some = weight if weight is not None else bias
    return ((x.shape[0], groups, x.shape[1] // groups, act, eps, _DTYPES[x.dtype]),
            int(some is not None and some.dtype == torch.float32))


def _forward(x, weight, bias, gate, groups, act, eps):
    dims, f32 = _dims(x, weight, bias, groups, act, eps)
    y = x.new_empty(x.shape)
    launch("ttc_group_norm_fwd", x.device, _lib.load().ttc_group_norm_fwd, _ptr(x), x.stride(0), _ptr(gate),
           0 if gate is None else gate.stride(0), _ptr(weight), _ptr(bias), f32, *dims, _ptr(y))
    return y


def _backward(x, weight, bias, gate, groups, act, eps, g, needs):
    """(dx, dweight, dbias, dgate), None where not needed."""
    dev, lib = x.device, _lib.load()
    dims, f32 = _dims(x, weight, bias, groups, act, eps)
    dx, dw, db, dgate = (t.new_empty(t.shape) if need and t is not None else None
                         for need, t in zip(needs, (x, weight, bias, gate)))
    nbytes = lib.ttc_group_norm_workspace(*dims[:3], dims[5]) if dw is not None or db is not None else 0
    ws = _workspace(nbytes, dev)
    launch("ttc_group_norm_bwd", dev, lib.ttc_group_norm_bwd, _ptr(x), x.stride(0), _ptr(gate),
           0 if gate is None else gate.stride(0), _ptr(weight), _ptr(bias), f32, _ptr(g), *dims, _ptr(dx), _ptr(dgate),
           _ptr(dw), _ptr(db), _ptr(ws), nbytes)
    return dx, dw, db, dgate


class GroupNormFunction(torch.autograd.Function):
    """(x, weight, bias, gate) -> y for x and gate [rows, C], all but x may be None."""

    @staticmethod
    def forward(ctx, x, weight, bias, gate, groups, act, eps):
        ctx.save_for_backward(x, weight, bias, gate)
        ctx.how = (groups, act, eps)
        return on_device(x.device, _forward, x, weight, bias, gate, groups, act, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        refuse_tangents("group_norm", g=g)
        saved = ctx.saved_tensors
        g = g.contiguous()
        return (*on_device(g.device, _backward, *saved, *ctx.how, g, ctx.needs_input_grad[:4]), None, None, None)


def group_norm(x, num_groups: int, weight=None, bias=None, gate=None, activation: str = "none", eps: float = 1e-5):
    """y, shaped like x [..., C] (float32 or bfloat16): the C channels of each row in ``num_groups`` groups (heads) of
    at most 1024, each to mean 0 and variance 1 (fp32), times ``weight`` [C] plus ``bias`` [C] (x's dtype
    or float32), then ``activation`` ("none", "silu" or "gelu", the exact one).  With ``gate`` (x's
    shape) the activation is of the gate and multiplies: norm(x) * act(gate).  Rows do not mix, so a
    token's result does not depend on other tokens.  fp32 arithmetic; bfloat16's silu uses the approximate
    exponential and reciprocal, below its rounding.  Differentiable in x, weight, bias and gate, once and in
    reverse mode."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"ttc_b200 group_norm supports float32 and bfloat16, got {x.dtype}")
    if activation not in _ACTS:
        raise ValueError(f"ttc_b200 group_norm: unknown activation {activation!r}")
    if x.dim() < 1 or num_groups < 1 or x.shape[-1] < 1 or x.shape[-1] % num_groups:
        raise ValueError(f"ttc_b200 group_norm: {tuple(x.shape)} channels do not divide into {num_groups} groups")
    C = x.shape[-1]
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError(f"ttc_b200 group_norm: gate must be {x.dtype} {tuple(x.shape)}, got "
                         f"{gate.dtype} {tuple(gate.shape)}")
    params = [p for p in (weight, bias) if p is not None]
    for p in params:
        if p.shape != (C,) or p.dtype not in (x.dtype, torch.float32) or p.dtype != params[0].dtype:
            raise ValueError(f"ttc_b200 group_norm: weight and bias must be [{C}] in {x.dtype} or both float32")
    if isinstance(eps, torch.Tensor):
        refuse_gradient("group_norm", eps=eps)
    refuse_tangents("group_norm", x=x, weight=weight, bias=bias, gate=gate)
    dev = x.device
    for t, n in ((weight, "weight"), (bias, "bias"), (gate, "gate")):
        if t is not None and t.device != dev:
            raise ValueError(f"ttc_b200 group_norm: {n} is on {t.device}, x on {dev}")
    if not x.is_cuda:
        raise ValueError("ttc_b200 group_norm needs CUDA tensors (there is no CPU path)")
    args = (_rows(x, C), *(p if p is None or p.is_contiguous() else p.contiguous() for p in (weight, bias)),
            None if gate is None else _rows(gate, C), int(num_groups), _ACTS[activation], float(eps))
    if wants_grad(x, weight, bias, gate):
        y = GroupNormFunction.apply(*args)
    else:
        y = on_device(dev, _forward, *args)
    return y if x.dim() == 2 else y.view(x.shape)
