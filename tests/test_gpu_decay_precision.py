"""decay_attention's errors as a whole against those of its documented roundings, in every form of a call: with and
without a last state and a first one, alone, segmented and packed."""
import pytest
import torch
from sequence_ref import attention_grads
from sequence_rounded import BF16_OVER_MODEL, f32_limit, off, rounded

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
# (B, T, H, Hk, dk, dv, lengths of packed sequences); one of 2 500 tokens in 2 heads is cut into segments, packed or not
SHAPES = [(1, 700, 4, 2, 64, 64, None), (3, 331, 4, 4, 32, 64, None), (1, 2500, 2, 1, 32, 32, None), (1, 2510, 2, 2, 64, 32, (2300, 0, 65, 135)),
          (1, 1200, 6, 2, 32, 64, (300, 64, 1, 335, 500))]


def _whole(f, q, k, v, go, start, end, cuts):
    """f on each of the packed sequences, joined; rows behind the last one are zeros."""
    if cuts is None:
        return f(q, k, v, go, start, end)
    at, got = 0, []
    for i, n in enumerate(cuts):
        if n:
            got.append(f(*(t[:, at:at + n] for t in (q, k, v, go)), *(None if t is None else t[i:i + 1] for t in (start, end))))
        else:  # the last state is the first one
            none = {n: t.new_zeros(1, 0, *t.shape[2:], dtype=torch.float64) for n, t in (("o", v), ("d_q", q), ("d_k", k), ("d_v", v))}
            first = (lambda t: v.new_zeros(1, v.shape[2], q.shape[3], v.shape[3], dtype=torch.float64) if t is None else t[i:i + 1].double())  # noqa: E731
            got.append(dict(none, state=first(start), d_start=first(end)))
        at += n
    out = {n: torch.cat([x[n] for x in got], 0 if n in ("state", "d_start") else 1) for n in got[0] if all(n in x for x in got)}
    for n in ("o", "d_q", "d_k", "d_v"):
        out[n] = torch.cat([out[n], out[n].new_zeros(1, q.shape[1] - at, *out[n].shape[2:])], 1)
    return out


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("decay", [-0.02, -0.002])
@pytest.mark.parametrize("states", ["none", "first", "last", "both"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}-{s[2]}-{s[3]}-{s[4]}-{s[5]}" + ("-packed" if s[6] else ""))
def test_errors_as_a_whole(shape, states, decay, dtype):
    from ttc_b200 import decay_attention
    B, T, H, Hk, dk, dv, lens = shape
    n = B if lens is None else len(lens)
    g = torch.Generator(device="cuda").manual_seed(T + dk)

    def normal(*s, dt=dtype):
        return torch.randn(*s, generator=g, device="cuda").to(dt)

    q, k, v, go = normal(B, T, Hk, dk), normal(B, T, Hk, dk), normal(B, T, H, dv), normal(B, T, H, dv)
    start = normal(n, H, dk, dv, dt=torch.float32) if states in ("first", "both") else None
    end = normal(n, H, dk, dv, dt=torch.float32) if states in ("last", "both") else None
    lg, scale = torch.full((H,), decay, device="cuda"), dk ** -0.5
    cu = None if lens is None else torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")

    ins = {n: t.detach().requires_grad_() for n, t in (("q", q), ("k", k), ("v", v), ("start", start)) if t is not None}
    got = decay_attention(ins["q"], ins["k"], ins["v"], lg, initial_state=ins.get("start"), return_state=end is not None,
                          cu_seqlens=cu)
    outs = got if end is not None else (got,)
    grads = torch.autograd.grad(outs, list(ins.values()), (go, end)[:len(outs)])
    got = dict(zip(("o", "state"), (t.detach() for t in outs)), **{"d_" + n: t for n, t in zip(ins, grads)})

    want = _whole(lambda q, k, v, go, s, e: attention_grads(q, k, v, lg, scale, go, s, e), q, k, v, go, start, end, lens)
    model = _whole(lambda q, k, v, go, s, e: rounded(q, k, v, lg, scale, go, s, e, dtype), q, k, v, go, start, end, lens)
    for name, t in got.items():
        limit = f32_limit(64)
        if dtype == torch.bfloat16 and name not in ("state", "d_start"):
            limit = BF16_OVER_MODEL * off(model[name], want[name])
        assert off(t, want[name]) <= limit, (name, off(t, want[name]), limit)
