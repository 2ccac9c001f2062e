"""Rotary positions of queries and keys: one CUDA kernel (``ttc_rotary``) for both, each way.

Pair p of the first ``2 len(inv_freq)`` values of a head turns by position * inv_freq[p], the others
are copied.  Angles are formed in 64 bits (a position of 10^6 has 0.03 rad of rounding in
32).  ``rotary_frequencies`` gives the frequencies, plain or scaled for contexts longer than the trained
one.  No counterpart in the reference; no fallback: without the CUDA library this raises.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import launch, on_device, refuse_gradient, refuse_tangents, wants_grad
from .solver import _DTYPES, _ptr


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device="cuda"):
    """(inv_freq float64 [rot_dim // 2], magnitude) for ``rotary``: inv_freq[p] = base^(-2p / rot_dim) and 1.
    ``scaling`` for a context ``factor`` times the trained ``original_length``:
    "linear" divides the frequencies by factor; "ntk" raises the base to
    base * factor^(rot_dim / (rot_dim - 2)), which leaves the first pair and divides the last by factor;
    "yarn" keeps pairs of more than beta_fast turns in original_length, divides those of fewer than beta_slow
    by factor, interpolates between, and scales the result by 0.1 ln(factor) + 1."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary_frequencies: rot_dim must be even and at least 2, got {rot_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if not (factor > 0 and base > 0):
        raise ValueError("rotary_frequencies: base and factor must be positive")
    p = torch.arange(rot_dim // 2, dtype=torch.float64, device="cpu")
    if scaling == "ntk" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2.0))
    f = float(base) ** (-2.0 * p / rot_dim)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if original_length is None or not beta_fast > beta_slow:
            raise ValueError("rotary_frequencies: yarn needs original_length and beta_fast > beta_slow")
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return f.to(device), magnitude


_TWO, _THREE = ctypes.c_int64 * 2, ctypes.c_int64 * 3


def _dense(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _turn(q, k, positions, inv_freq, interleaved, magnitude, inverse):
    q, k = _dense(q), None if k is None else _dense(k)
    B, T, H, D = shape = q.shape
    q_out, k_out = q.new_empty(shape), None if k is None else k.new_empty(k.shape)
    ps = positions.stride()  # [T] and [1, T] are shared by the batch
    launch("ttc_rotary", q.device, _lib.load().ttc_rotary, q.data_ptr(), _THREE(*q.stride()[:3]), H, _ptr(k),
           None if k is None else _THREE(*k.stride()[:3]), 0 if k is None else k.shape[2], positions.data_ptr(),
           _TWO(0 if len(ps) == 1 or positions.shape[0] == 1 else ps[0], ps[-1]), positions.dtype == torch.int64,
           inv_freq.data_ptr(), B, T, D, inv_freq.shape[0], interleaved, inverse, magnitude, _DTYPES[q.dtype],
           q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


class RotaryFunction(torch.autograd.Function):
    """(q, k or None) -> both turned; the backward turns the gradients back.  No autocast wrappers, here as in the other
    sequence operators: nothing inside depends on its state."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, magnitude):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (interleaved, magnitude)
        ctx.like = q.shape, None if k is None else k.shape, q.dtype
        return on_device(q.device, _turn, q, k, positions, inv_freq, *ctx.how, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_q, g_k):
        refuse_tangents("rotary", g_q=g_q, g_k=g_k)
        if g_q is None and g_k is None:
            return (None,) * 6
        positions, inv_freq = ctx.saved_tensors
        q_shape, k_shape, dtype = ctx.like
        # what the loss sees is turned back, the other's gradient is zeros
        some, other = (g_k, None) if g_q is None else (g_q, g_k)
        d_some, d_other = on_device(positions.device, _turn, some, other, positions, inv_freq, *ctx.how, True)
        d_q, d_k = (None, d_some) if g_q is None else (d_some, d_other)
        if d_q is None:
            d_q = torch.zeros(q_shape, dtype=dtype, device=positions.device)
        if d_k is None and k_shape is not None:
            d_k = torch.zeros(k_shape, dtype=dtype, device=positions.device)
        return d_q, d_k, None, None, None, None


def rotary(q, k, positions, inv_freq, interleaved: bool = False, magnitude: float = 1.0):
    """(q', k') for q [B, T, H, D] and k [B, T, Hk, D] (or None; float32 or bfloat16, D <= 512), turned at ``positions``
    (int32 or int64, [T] or [B, T], any values) by ``inv_freq`` [R / 2] float64: the first R <= D values of
    each head in pairs (p, p + R / 2), or (2p, 2p + 1) where ``interleaved``, multiplied by ``magnitude``; the
    other D - R are copied.  Differentiable in q and k, once and in reverse mode (the frequencies
    and the factor are fixed).  The head dim is read in place where it is contiguous, whatever the
    other strides."""
    for t, n in ((q, "q"), (k, "k")):
        if t is None and n == "k":
            continue
        if t.dtype not in _DTYPES:
            raise TypeError(f"ttc_b200 rotary supports float32 and bfloat16, got {t.dtype} for {n}")
        if t.dim() != 4:
            raise ValueError(f"ttc_b200 rotary: {n} must be [B, T, heads, D], got {tuple(t.shape)}")
    B, T, H, D = q.shape
    if k is not None and (k.dtype != q.dtype or k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise ValueError(f"ttc_b200 rotary: q {q.dtype} {tuple(q.shape)} and k {k.dtype} {tuple(k.shape)} do not match")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ttc_b200 rotary: positions must be int32 or int64, got {positions.dtype}")
    if positions.shape not in ((T,), (1, T), (B, T)):
        raise ValueError(f"ttc_b200 rotary: positions must be [{T}] or [{B},{T}], got {tuple(positions.shape)}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or 2 * inv_freq.numel() > D:
        raise ValueError(f"ttc_b200 rotary: inv_freq must be float64 [R / 2] with R <= {D}, got "
                         f"{inv_freq.dtype} {tuple(inv_freq.shape)}")
    if inv_freq.requires_grad or isinstance(magnitude, torch.Tensor):
        refuse_gradient("rotary", inv_freq=inv_freq, magnitude=magnitude)
    refuse_tangents("rotary", q=q, k=k, inv_freq=inv_freq)
    dev = q.device
    for t, n in ((k, "k"), (positions, "positions"), (inv_freq, "inv_freq")):
        if t is not None and t.device != dev:
            raise ValueError(f"ttc_b200 rotary: {n} is on {t.device}, q on {dev}")
    if not q.is_cuda:
        raise ValueError("ttc_b200 rotary needs CUDA tensors (there is no CPU path)")
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    args = (q, k, positions, inv_freq, bool(interleaved), float(magnitude))
    if wants_grad(q, k):
        return RotaryFunction.apply(*args)
    return on_device(dev, _turn, *args, False)
