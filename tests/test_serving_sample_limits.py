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
