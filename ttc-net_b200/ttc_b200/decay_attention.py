"""Attention with a fixed decay for each head: the memory over tokens that stands beside the
TTC layer, which mixes none.

    S_t = gamma_h S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   gamma_h = exp(log_gamma[h])

``decay_attention`` takes whole sequences (prompts and training; ``ttc_decay_attn_fwd`` / ``_bwd``,
blocks of 64 tokens on the tensor cores, the state in fp32 registers), ``decay_attention_step`` one token
for each row over a cache of states (``ttc_decay_attn_step``).  No counterpart in the reference; no
fallback: without the CUDA library these raise.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import launch, on_device, refuse_gradient, refuse_tangents, wants_grad
from .solver import _DTYPES, _aligned, _ptr


def _workspace(nbytes: int, dev) -> torch.Tensor | None:
    """Scratch memory of one call, on the call's stream."""
    if nbytes < 0:
        _lib.check(-nbytes)
    return torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None


# For each device one word of pinned host memory that its kernels can reach, a view of it and its address: it is
# read at the next call without waiting for the GPU.
_status: dict[int, tuple[torch.Tensor, ctypes.c_int, int]] = {}

WAIT_TIMEOUT_MSG = ("ttc_b200 decay_attention: a wait inside an earlier call's kernel ran out "
                    "(that call's results are not valid)")


def _raise_timeout(device: int) -> None:
    """Raises if a call on the device reported a timeout since the last time this raised."""
    held = _status.get(device)
    if held is not None and held[1].value:
        held[1].value = 0
        raise RuntimeError(f"{WAIT_TIMEOUT_MSG[:-1]}, on cuda:{device})")


def _status_word(device: int | None = None) -> int:
    """The address of the device's status word (None: of the current device's); raises as `_raise_timeout`."""
    device = torch.cuda.current_device() if device is None else device
    held = _status.get(device)
    if held is None:
        word = torch.zeros(1, dtype=torch.int32, device="cpu", pin_memory=True)
        at = word.data_ptr()
        held = _status.setdefault(device, (word, ctypes.c_int.from_address(at), at))
    if held[1].value:
        _raise_timeout(device)
    return held[2]


def check_decay_attention(device=None) -> None:
    """Waits for the device (None: the current one) and raises RuntimeError if a wait inside a
    ``decay_attention`` kernel ran out on it since the last report; that call's results, and states that went
    on from them, are not valid.  Calls report it by themselves, but only what was known when they were made:
    ask here behind replays of a captured call and before results leave the program."""
    device = torch.cuda.current_device() if device is None else torch.device(device).index
    device = torch.cuda.current_device() if device is None else device
    torch.cuda.synchronize(device)
    _raise_timeout(device)


def _operand(t: torch.Tensor) -> torch.Tensor:
    """t itself if its head dim is contiguous and its rows start on 16-byte boundaries (a slice of
    a fused projection), else a contiguous copy (an expanded tensor among these: tensor maps know no
    stride of 0)."""
    if t.is_contiguous():
        return _aligned(t)
    es = t.element_size()
    ok = t.stride(-1) == 1 and all(n == 1 or (s > 0 and s * es % 16 == 0) for n, s in zip(t.shape[:-1], t.stride()))
    return _aligned(t if ok else t.contiguous())


_SIX, _NINE = ctypes.c_int64 * 6, ctypes.c_int64 * 9


def _strides(t: torch.Tensor):
    """Strides of the dims before the head dim of t [B, T, heads, D], as the C entries want them: multiples of 16 bytes.
    Those of a dim of one element, and all of an empty tensor, may be anything, in a contiguous tensor too."""
    if t.is_contiguous():
        _, T, H, D = t.shape
        return T * H * D, H * D, D
    return [s if n > 1 else 0 for n, s in zip(t.shape[:-1], t.stride())]


def _check_qkv(name, q, k, v, log_gamma, lead):
    """Types, devices and shapes of q, k [*lead, Hk, dk], v [*lead, H, dv], log_gamma [H]."""
    qs, vs, dt = q.shape, v.shape, q.dtype
    if not (dt in _DTYPES and k.dtype == dt and v.dtype == dt and len(qs) == lead + 2 and qs == k.shape
            and len(vs) == lead + 2 and qs[:lead] == vs[:lead]):
        for t, n in ((q, "q"), (k, "k"), (v, "v")):
            if t.dtype not in _DTYPES:
                raise TypeError(f"ttc_b200 {name} supports float32 and bfloat16, got {t.dtype} for {n}")
            if t.dim() != lead + 2:
                raise ValueError(f"ttc_b200 {name}: {n} must have {lead + 2} dimensions, got {tuple(t.shape)}")
        if not q.dtype == k.dtype == v.dtype:
            raise TypeError(f"ttc_b200 {name}: q, k and v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
        raise ValueError(f"ttc_b200 {name}: q {tuple(qs)}, k {tuple(k.shape)} and v {tuple(vs)} do not match")
    Hk, dk = qs[lead:]
    H, dv = vs[lead:]
    if Hk < 1 or H % Hk:
        raise ValueError(f"ttc_b200 {name}: {H} value heads are not a multiple of {Hk} key heads")
    if log_gamma.shape != (H,) or not log_gamma.dtype.is_floating_point:
        raise ValueError(f"ttc_b200 {name}: log_gamma must be [{H}] floating point, got {tuple(log_gamma.shape)}")
    if log_gamma.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"ttc_b200 {name}: the decays are fixed, log_gamma must not require a gradient")
    return H, Hk, dk, dv


def _decays(log_gamma):
    return log_gamma if log_gamma.dtype == torch.float32 and log_gamma.is_contiguous() else log_gamma.float().contiguous()


def _check_device(name, dev, **tensors):
    for n, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"ttc_b200 {name}: {n} is on {t.device}, q on {dev}")
    if dev.type != "cuda":
        raise ValueError(f"ttc_b200 {name} needs CUDA tensors (there is no CPU path)")


def _dims(q, v, cu_seqlens):
    """(T, sequences, H, Hk, dk, dv, dtype code) of the C calls."""
    B, T, Hk, dk = q.shape
    return T, B if cu_seqlens is None else cu_seqlens.numel() - 1, v.shape[2], Hk, dk, v.shape[3], _DTYPES[q.dtype]


def _forward(q, k, v, log_gamma, scale, initial_state, cu_seqlens, want_state):
    dev, lib, dims = q.device, _lib.load(), _dims(q, v, cu_seqlens)
    status = _status_word(dev.index)
    T, n_seq, H, _, dk, dv, _ = dims
    o = v.new_empty(v.shape)
    state = torch.empty(n_seq, H, dk, dv, device=dev, dtype=torch.float32) if want_state else None
    nbytes = lib.ttc_decay_attn_workspace(T, n_seq, cu_seqlens is not None, *dims[2:], 0)
    ws = _workspace(nbytes, dev)
    launch("ttc_decay_attn_fwd", dev, lib.ttc_decay_attn_fwd, _ptr(q), _ptr(k), _ptr(v),
           _NINE(*_strides(q), *_strides(k), *_strides(v)), _ptr(log_gamma), scale,
           _ptr(initial_state), _ptr(cu_seqlens), *dims, _ptr(o), _ptr(state), _ptr(ws), nbytes, status)
    return o, state


def _backward(q, k, v, log_gamma, scale, initial_state, cu_seqlens, g_o, g_state, want_start):
    dev, lib, dims = q.device, _lib.load(), _dims(q, v, cu_seqlens)
    status = _status_word(dev.index)
    d_q, d_k, d_v = (t.new_empty(t.shape) for t in (q, k, v))
    d_s = torch.empty(initial_state.shape, device=dev, dtype=torch.float32) if want_start else None
    nbytes = lib.ttc_decay_attn_workspace(*dims[:2], cu_seqlens is not None, *dims[2:], 1)
    ws = _workspace(nbytes, dev)
    launch("ttc_decay_attn_bwd", dev, lib.ttc_decay_attn_bwd, _ptr(q), _ptr(k), _ptr(v),
           _NINE(*_strides(q), *_strides(k), *_strides(v)), _ptr(g_o), _ptr(log_gamma), scale,
           _ptr(initial_state), _ptr(g_state), _ptr(cu_seqlens), *dims, _ptr(d_q), _ptr(d_k), _ptr(d_v), _ptr(d_s),
           _ptr(ws), nbytes, status)
    return d_q, d_k, d_v, d_s


def _step(q, k, v, log_gamma, scale, state, slot_stride, slots, dims):
    _raise_timeout(q.device.index)  # before the states advance
    o = v.new_empty(v.shape)
    launch("ttc_decay_attn_step", q.device, _lib.load().ttc_decay_attn_step, q.data_ptr(), k.data_ptr(), v.data_ptr(),
           _SIX(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2]), log_gamma.data_ptr(), scale,
           state.data_ptr(), slot_stride, _ptr(slots), *dims, o.data_ptr())
    return o


class DecayAttentionFunction(torch.autograd.Function):
    """(q, k, v, initial_state) -> (o, last state or None)."""

    @staticmethod
    def forward(ctx, q, k, v, log_gamma, scale, initial_state, cu_seqlens, want_state):
        ctx.set_materialize_grads(False)  # None for an output that the loss does not see, a state's above all
        ctx.save_for_backward(q, k, v, log_gamma, initial_state, cu_seqlens)
        ctx.scale = scale
        return on_device(q.device, _forward, q, k, v, log_gamma, scale, initial_state, cu_seqlens, want_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_o, g_state):
        refuse_tangents("decay_attention", g_o=g_o, g_state=g_state)
        if g_o is None and g_state is None:
            return (None,) * 8
        q, k, v, log_gamma, initial_state, cu_seqlens = ctx.saved_tensors
        g_o = torch.zeros_like(v) if g_o is None else g_o
        g_o = _aligned(g_o.contiguous())
        g_state = None if g_state is None else g_state.float().contiguous()
        want = initial_state is not None and ctx.needs_input_grad[5]
        d_q, d_k, d_v, d_s = on_device(q.device, _backward, q, k, v, log_gamma, ctx.scale, initial_state, cu_seqlens, g_o,
                                       g_state, want)
        return d_q, d_k, d_v, None, None, d_s, None, None


def decay_attention(q, k, v, log_gamma, scale: float | None = None, initial_state=None, return_state: bool = False,
                    cu_seqlens=None):
    """o [B, T, H, dv] for q, k [B, T, Hk, dk] and v [B, T, H, dv] (float32 or bfloat16; H a multiple of
    Hk, head h reads key head h // (H // Hk); dk, dv multiples of 8 up to 128), log_gamma [H] the logarithm
    of each head's decay (fixed: no gradient; -inf is no memory).  ``scale`` defaults to
    dk ** -0.5.  Differentiable in q, k, v and ``initial_state`` [B, H, dk, dv] float32, once and
    in reverse mode.

    ``return_state``: (o, state), the states behind the last tokens, float32, from which
    ``decay_attention_step`` or another call goes on.

    ``cu_seqlens`` (int32 [n + 1] on the device, from 0, non-decreasing): packed sequences, B = 1 and
    sequence i the tokens cu_seqlens[i] .. cu_seqlens[i + 1] - 1; states are [n, H, dk, dv].  Rows
    behind the last sequence get zeros.  Offsets past the row are cut to it.

    A token's output depends on no later token, whatever that holds.  What an Inf or NaN in k or v
    reaches, later outputs and states of its heads, is not finite, and NaN also where the definition has an infinity.
    Any strides with a contiguous head dim are read in place if rows start on 16-byte boundaries.  At most
    2^20 - 16 sequences times heads.

    Sums and states are float32.  float32 operands are used with all their 24 bits.  For bfloat16 the scores times
    decays, and every 64 tokens the copy of the state that queries multiply, are rounded to bfloat16 once on the way, in the
    backward too: for random operands o, d_q, d_k and d_v are 2.35e-3 from the definition as a whole, where rounding
    them alone is 1.66e-3.  With ``return_state`` (or a gradient to ``initial_state``) the state is updated with 24 bits of
    the decayed values, without it with 16, which can show in the last bit of o."""
    name = "decay_attention"
    H, Hk, dk, dv = _check_qkv(name, q, k, v, log_gamma, 2)
    n_seq = q.shape[0]
    if cu_seqlens is not None:
        if q.shape[0] != 1:
            raise ValueError(f"ttc_b200 {name}: packed sequences need a batch of 1, got {q.shape[0]}")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
            raise ValueError(f"ttc_b200 {name}: cu_seqlens must be int32 [n + 1] with n >= 1")
        n_seq = cu_seqlens.numel() - 1
    if initial_state is not None and (initial_state.dtype != torch.float32
                                      or tuple(initial_state.shape) != (n_seq, H, dk, dv)):
        raise ValueError(f"ttc_b200 {name}: initial_state must be float32 [{n_seq},{H},{dk},{dv}], got "
                         f"{initial_state.dtype} {tuple(initial_state.shape)}")
    if isinstance(scale, torch.Tensor):
        refuse_gradient(name, scale=scale)
    refuse_tangents(name, q=q, k=k, v=v, log_gamma=log_gamma, initial_state=initial_state)
    _check_device(name, q.device, k=k, v=v, log_gamma=log_gamma, initial_state=initial_state, cu_seqlens=cu_seqlens)
    args = (_operand(q), _operand(k), _operand(v), _decays(log_gamma),
            dk ** -0.5 if scale is None else float(scale), None if initial_state is None else initial_state.contiguous(),
            None if cu_seqlens is None else cu_seqlens.contiguous(), bool(return_state))
    if wants_grad(q, k, v, initial_state):
        o, state = DecayAttentionFunction.apply(*args)
    else:
        o, state = on_device(q.device, _forward, *args)
    return (o, state) if return_state else o


def decay_attention_step(q, k, v, log_gamma, state, slots=None, scale: float | None = None) -> torch.Tensor:
    """One token for each row: q, k [B, Hk, dk], v [B, H, dv] -> o [B, H, dv].  ``state`` [n, H, dk, dv]
    float32 is the cache of states, advanced in place; row b goes on from state ``slots[b]`` (int32 on the
    device; b without ``slots``).  Rows of one slot are consecutive tokens in the rows' order; a row whose slot
    is outside [0, n) is padding, its output is zeros.  At most 2^20 - 16 rows times heads.  float32 arithmetic.
    Records no gradient."""
    name = "decay_attention_step"
    H, Hk, dk, dv = _check_qkv(name, q, k, v, log_gamma, 1)
    if state.dtype != torch.float32 or state.dim() != 4 or state.shape[1:] != (H, dk, dv):
        raise ValueError(f"ttc_b200 {name}: state must be float32 [n,{H},{dk},{dv}], got "
                         f"{state.dtype} {tuple(state.shape)}")
    B, n = q.shape[0], state.shape[0]
    slot_stride, *inner = state.stride()
    size = H * dk * dv
    if n <= 1:
        slot_stride = size
    if (inner != [dk * dv, dv, 1] and not state[:1].is_contiguous()) or slot_stride < size or slot_stride % 4 \
            or state.data_ptr() % 16:
        raise ValueError(f"ttc_b200 {name}: each state must be contiguous and start on a 16-byte boundary")
    if slots is not None and (slots.dtype != torch.int32 or slots.shape != (B,)):
        raise ValueError(f"ttc_b200 {name}: slots must be int32 [{B}], got {slots.dtype} {tuple(slots.shape)}")
    if slots is None and n < B:
        raise ValueError(f"ttc_b200 {name}: {B} rows and {n} states")
    if (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad) and torch.is_grad_enabled():
        raise ValueError(f"ttc_b200 {name} records no gradient: call it under torch.no_grad()")
    if isinstance(scale, torch.Tensor):
        refuse_gradient(name, scale=scale)
    refuse_tangents(name, q=q, k=k, v=v, log_gamma=log_gamma, state=state)
    dev = q.device
    _check_device(name, dev, k=k, v=v, log_gamma=log_gamma, state=state, slots=slots)
    if not (q.stride(-1) == k.stride(-1) == v.stride(-1) == 1):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if slots is not None and not slots.is_contiguous():
        slots = slots.contiguous()
    o = on_device(dev, _step, q, k, v, _decays(log_gamma), dk ** -0.5 if scale is None else float(scale), state,
                  slot_stride, slots, (B, n, H, Hk, dk, dv, _DTYPES[q.dtype]))
    torch.autograd.graph.increment_version(state)
    return o
