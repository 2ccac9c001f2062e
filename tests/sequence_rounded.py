"""The block form of attention with a decay in 64 bits, with the roundings below 32 bits that the bf16 kernels document
and no others, or with operands cut to fewer bf16 parts: how far results may be off as a whole, and how far they
would be off if a part were lost.

Every test uses relative errors of whole tensors, |got - want| / |want| in the norm of all elements.  For random
operands the kernels' roundings are as good as independent, so their squares add and what a single value may be
off by does not: with tens of thousands of values the ratio of two such errors is known to a few per cent."""
import torch

C = 64


def bf16(x):
    return x.float().bfloat16().double()


def parts(x, n):
    """x as the sum of its first n bf16 parts."""
    s = torch.zeros_like(x)
    for _ in range(n):
        s = s + bf16(x - s)
    return s


def recurrence(q, k, v, log_gamma, a, b, u, e, start, scores=bf16, copy=bf16, update=lambda x: x):
    """o [B, T, H, dv] and the last state for q, k [B, T, H, dk], v [B, T, H, dv] in float64, in blocks of 64 tokens:
    o_i = sum_{j <= i} scores(a gamma^(i-j) q_i . k_j) v_j + b gamma^(i+1-e) q_i copy(S),
    S' = gamma^rows S + sum_j k_j^T update(u gamma^(rows-1-j+e) v_j)."""
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    lg = log_gamma.double()[None, :, None]
    S = start if start is not None else q.new_zeros(*q.shape[:2], q.shape[-1], v.shape[-1])
    out = []
    for c in range(0, q.shape[2], C):
        qc, kc, vc = (t[:, :, c:c + C] for t in (q, k, v))
        n = qc.shape[2]
        i = torch.arange(n, device=q.device, dtype=torch.float64)
        ahead = i[:, None] - i[None, :]
        P = a * torch.where(ahead >= 0, torch.exp(lg[..., None] * ahead.clamp(min=0)), 0.0) * (qc @ kc.transpose(-1, -2))
        out.append(scores(P) @ vc + b * torch.exp(lg * (i + 1 - e))[..., None] * (qc @ copy(S)))
        S = torch.exp(lg * n)[..., None] * S + kc.transpose(-1, -2) @ update(u * torch.exp(lg * (n - 1 - i + e))[..., None] * vc)
    return torch.cat(out, 2).transpose(1, 2), S


def rounded(q, k, v, log_gamma, scale, g_o, start, g_state, dtype, **how):
    """{name: value} of o, state, d_q, d_k, d_v, d_start as `recurrence` forms them, in the results' types."""
    Hk, H = q.shape[2], v.shape[2]
    q, k = (t.double().repeat_interleave(H // Hk, 2) for t in (q, k))
    v, g = v.double(), g_o.double()
    start, end = (None if t is None else t.double() for t in (start, g_state))
    swapped = (lambda t: None if t is None else t.transpose(-1, -2))  # noqa: E731
    back = (lambda *ts: [t.flip(1) for t in ts])  # noqa: E731
    o, state = recurrence(q, k, v, log_gamma, scale, scale, 1.0, 0, start, **how)
    d_q, _ = recurrence(g, v, k, log_gamma, scale, scale, 1.0, 0, swapped(start), **how)
    d_v, d_start = recurrence(*back(k, q, g), log_gamma, scale, 1.0, scale, 1, end, **how)
    d_k, _ = recurrence(*back(v, g, q), log_gamma, scale, 1.0, scale, 1, swapped(end), **how)
    shared = (lambda t: t.unflatten(2, (Hk, H // Hk)).sum(3))  # noqa: E731
    out = dict(o=o, d_q=shared(d_q), d_k=shared(d_k.flip(1)), d_v=d_v.flip(1))
    out = {n: bf16(t) if dtype == torch.bfloat16 else t for n, t in out.items()}
    return dict(out, state=state, d_start=d_start)


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# bf16 results: the roundings of `rounded`.  What the kernels add to them, two parts of the decayed values (2^-18 of a
# term as a rule) and sums in 32 bits, adds its square, below 10^-5 of theirs; 4 % are left for the scatter of errors
# over the tens of thousands of values of a test.
BF16_OVER_MODEL = 1.04


def f32_limit(width):
    """Relative error of fp32 results and of states, heads of up to ``width``.  Three products in a row (scores, scores
    times values, state times queries) leave out at most 2^-23 of their terms each; their sums run over width / 16, 64 / 16
    and width / 16 additions in the tensor core, each cut by 0 to 2^-23, half of that on average.  (A result
    that lost the last of three parts anywhere is off by 9 to 21 2^-23, see test_sequence_rounded.py.)"""
    return (3 + (2 * width / 16 + 4) / 2) * 2.0 ** -23
