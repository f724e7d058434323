"""Sampling at the ends of its parameters' ranges, against the definition in 64 bits as in
test_serving_sample.py (tokens equal, log-probabilities within 2^-20 (1 + |lp|))."""
import math

import pytest
import torch

from tests.test_serving_sample import DT, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("V", [50, 5003])
@pytest.mark.parametrize("kw", [{}, dict(top_k=9), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=40, top_p=0.9, min_p=0.01)],
                         ids=["none", "k", "p", "min", "all"])
@pytest.mark.parametrize("t", [math.inf, 3e38, 1e30, 1e-30, 1e-39, 1e-42])
def test_temperatures_whose_inverse_is_no_normal_number(dt, V, kw, t):
    """At infinity every token that is not masked weighs the same; near zero all but the largest
    logits, which race, weigh nothing.  Masked tokens stay out."""
    x, e = _inputs(4, V, DT[dt], seed=48 + V)
    x[1, ::3] = -math.inf
    x[2, :] = -math.inf
    x[2, [3, 11]] = torch.tensor([0.5, -2.0], dtype=x.dtype)
    x[3, [5, 17, 40]] = 30.0
    if t > 1 and kw.get("top_p", 1.0) < 1:
        kw = {**kw, "top_p": 0.6003}  # no mass of equal weights ends there
    _check(x, e, t, **kw)
    _check(x, e, torch.full((4,), t), **kw)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("V", [700, 40000])
@pytest.mark.parametrize("kw", [{}, dict(top_k=20), dict(top_k=2000), dict(top_p=0.9), dict(min_p=0.02)],
                         ids=["none", "k", "general", "p", "min"])
def test_random_numbers_of_zero(dt, V, kw):
    """w / 0 beats every number, and of several such tokens the lowest index wins, each time."""
    x, e = _inputs(6, V, DT[dt], seed=49 + V, spread=1.0)
    best = x.float().argsort(1, descending=True)
    e[0, best[0, 3]] = 0.0
    e[1, best[1, :18]] = 0.0        # the first of the ranking among them
    e[2, best[2, 2:18]] = 0.0
    e[3, best[3, 4:6]] = 0.0
    e[4, best[4, -3:]] = 0.0        # mostly filtered out
    e[5] = 0.0
    for _ in range(4):
        want, _ = _check(x, e, 0.7, **{**kw, "top_k": min(kw.get("top_k", 0), V - 1)})
    assert want[0] == best[0, 3] and want[1] == best[1, :18].min() and want[2] == best[2, 2:18].min()


@pytest.mark.parametrize("kw", [dict(min_p=0.05), dict(top_p=0.9)], ids=["min", "p"])
def test_two_random_numbers_of_zero_in_warps_of_unequal_pace(kw):
    """A warp whose tokens are all filtered out but one reaches that one, late in the row, before
    a warp of kept tokens reaches its own in the middle."""
    B, V = 200, 32760
    x, e = _inputs(1, V, torch.bfloat16, seed=50, spread=0.2)
    chunk = torch.arange(V) // 8
    x[0, chunk % 512 < 480] = -20.0
    late, middle = (7 * 512 + 3) * 8 + 1, (4 * 512 + 490) * 8 + 2
    x[0, late] = x[0, middle] = 0.5
    x[0, 490 * 8] = 1.0  # the first of the ranking
    e[0, late] = e[0, middle] = 0.0
    from co_alibi_attn import sample_tokens
    for _ in range(5):
        tok, _ = sample_tokens(x.cuda().expand(B, V).contiguous(), e.cuda().expand(B, V).contiguous(), **kw)
        assert (tok == middle).all()
