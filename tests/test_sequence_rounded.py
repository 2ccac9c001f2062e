"""The oracle of the precision tests: it is the definition, and a part lost anywhere is beyond the tests' limits.  CPU."""
import pytest
import torch
from sequence_ref import attention_grads
from sequence_rounded import BF16_OVER_MODEL, f32_limit, off, parts, rounded

EXACT = dict(scores=lambda x: x, copy=lambda x: x)


def _inputs(dtype, width, T=500, H=4, Hk=2):
    g = torch.Generator().manual_seed(width)

    def normal(*s, dt=dtype):
        return torch.randn(*s, generator=g).to(dt)

    return (normal(1, T, Hk, width), normal(1, T, Hk, width), normal(1, T, H, width), normal(1, T, H, width),
            normal(1, H, width, width, dt=torch.float32), normal(1, H, width, width, dt=torch.float32))


def test_without_roundings_it_is_the_definition():
    q, k, v, go, start, gs = _inputs(torch.float32, 16, T=150)
    lg = torch.tensor([-0.3, -0.1, -0.02, 0.0])
    want = attention_grads(q, k, v, lg, 0.3, go, start, gs)
    got = rounded(q, k, v, lg, 0.3, go, start, gs, torch.float32, **EXACT)
    assert set(got) == set(want) and all(off(got[n], want[n]) < 1e-13 for n in want)


@pytest.mark.parametrize("width", [32, 64])
def test_a_lost_part_shows_in_fp32(width):
    q, k, v, go, start, gs = _inputs(torch.float32, width)
    lg, two = torch.full((4,), -0.02), lambda x: parts(x, 2)
    want = attention_grads(q, k, v, lg, width ** -0.5, go, start, gs)
    limit = f32_limit(width)
    seen = {"q": ("o", "d_k", "d_v", "d_start"), "k": ("o", "d_q", "d_v", "state"), "v": ("o", "d_q", "d_k", "state"),
            "scores": ("o", "d_q", "d_k", "d_v"), "copy": ("o", "d_q", "d_k", "d_v"),
            "update": ("o", "d_q", "d_k", "d_v", "state", "d_start")}
    for where, names in seen.items():
        ops = [two(t.double()) if n == where else t for n, t in (("q", q), ("k", k), ("v", v))]
        how = dict(EXACT, **({where: two} if where in ("scores", "copy", "update") else {}))
        got = rounded(*ops, lg, width ** -0.5, go, start, gs, torch.float32, **how)
        for n in names:
            assert off(got[n], want[n]) > limit, (where, n)
    whole = rounded(*(parts(t.double(), 3) for t in (q, k, v)), lg, width ** -0.5, go, start, gs, torch.float32, **EXACT)
    assert all(off(whole[n], want[n]) < 2.0 ** -23 for n in want)


@pytest.mark.parametrize("width", [32, 64])
def test_a_lost_part_shows_in_bf16(width):
    q, k, v, go, start, gs = _inputs(torch.bfloat16, width)
    lg = torch.full((4,), -0.002)
    want = attention_grads(q, k, v, lg, width ** -0.5, go, start, gs)
    res = [rounded(q, k, v, lg, width ** -0.5, go, start, gs, torch.bfloat16, update=lambda x, n=n: parts(x, n)) for n in (1, 2, 3)]
    for n in ("o", "d_q", "d_k", "d_v"):
        one, two, three = (off(r[n], want[n]) for r in res)
        assert one > BF16_OVER_MODEL * three and two < 1.002 * three and three < 3.2e-3
        assert off(1.03 * res[2][n], want[n]) > BF16_OVER_MODEL * three
    for n in ("state", "d_start"):  # updated with three parts
        assert off(res[1][n], want[n]) > f32_limit(width) > 4 * off(res[2][n], want[n])
