"""Sampling against its definition in 64 bits.  Tokens must be equal: the inputs come from
fixed seeds, and two scores, or a mass and its limit, lie within float32's rounding of each
other in about one row of 10^5.  Log-probabilities: 2^-20 (1 + |lp|), a few
roundings of float32 in the scaled logit and in the logarithm of the sum."""
import ctypes
import math

import pytest
import torch

from tests import _serving_ref as ref

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _inputs(B, V, dt, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, V, generator=g) * spread).to(dt)
    e = torch.empty(B, V).exponential_(generator=g).clamp_(min=1e-9)
    return x, e


def _check(x, e, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, device_x=None, device_e=None):
    from co_alibi_attn import sample_tokens
    B = x.shape[0]
    dev = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v  # noqa: E731
    tok, lp = sample_tokens(x.cuda() if device_x is None else device_x, e.cuda() if device_e is None else device_e,
                            temperature=dev(temperature), top_k=dev(top_k), top_p=dev(top_p), min_p=dev(min_p))
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (B,)
    rows = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [torch.tensor(v).item()] * B  # noqa: E731
    want, want_lp, kept = ref.sample(x, e, rows(temperature), rows(top_k), rows(top_p), rows(min_p))
    assert tok.tolist() == want
    for a, b in zip(lp.tolist(), want_lp):
        assert a == b or abs(a - b) <= 2.0 ** -20 * (1 + abs(b)), (a, b)
    return want, kept


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 37), (5, 1000), (2, 4099), (1, 50304), (3, 70001)])
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (1, 1.0, 0.0), (5, 1.0, 0.0), (40, 0.9, 0.0), (0, 0.7, 0.0),
                                               (0, 0.995, 0.0), (0, 1.0, 0.05), (300, 0.95, 0.01), (10 ** 9, 0.5, 0.0)])
def test_matches_definition(dt, B, V, top_k, top_p, min_p):
    x, e = _inputs(B, V, DT[dt], seed=V + top_k % 97)
    _check(x, e, 0.8, top_k, top_p, min_p)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("B,V,top_k,top_p", [(2, 50304, 1025, 1.0), (2, 4099, 3000, 0.9), (1, 1_000_003, 50, 1.0),
                                             (2, 1_000_003, 0, 0.9), (1, 600_001, 1024, 0.5), (150, 2500, 1024, 0.99),
                                             (40, 9000, 385, 1.0), (1, 2 ** 21, 3, 1.0), (75, 33333, 0, 0.5)])
def test_large_k_and_vocabularies(dt, B, V, top_k, top_p):
    """k past the lists, slices that stay in global memory or exceed the bins' 16-bit halves, and
    row counts on either side of the cluster sizes."""
    x, e = _inputs(B, V, DT[dt], seed=V % 1000 + top_k)
    _check(x, e, 0.9, top_k, top_p)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50304, 333])
def test_each_row_its_own_parameters(V):
    B = 24
    x, e = _inputs(B, V, torch.float32, seed=41)
    r = torch.arange(B)
    _check(x, e, torch.where(r % 5 == 0, 0.0, 0.3 + 0.1 * (r % 9)).float(), (r * 7 % 60).int(),
           torch.where(r % 4 == 1, 1.0, 0.3 + 0.025 * r).float(), torch.where(r % 3 == 0, 0.0, 0.002 * r).float())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("V", [64, 5000, 40000])
def test_ties_go_to_the_lowest_index(dt, V):
    _, e = _inputs(4, V, torch.float32, seed=42)
    flat = torch.full((4, V), 1.25).to(DT[dt])
    flat[1, V // 2:] = -3.0
    flat[2, ::3] = 2.0
    flat[3] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)  # zeros of either sign are equal
    for k in (1, 7, V // 3 + 1, V - 1):
        _, kept = _check(flat, e, 1.0, k)
        assert sorted(kept[0]) == list(range(k)) and sorted(kept[3]) == list(range(k))
    _check(flat, e, 1.0, 0, 0.49993)
    _check(flat, e, 0.0)
    want, _ = _check(flat, torch.ones_like(e))  # equal scores too
    assert want == [0, 0, 0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_masked_infinite_and_nan_logits(dt):
    V = 3001
    x, e = _inputs(10, V, DT[dt], seed=43)
    low, keep = torch.finfo(DT[dt]).min, torch.tensor([5, 77, 2999])
    for row, value in ((0, -math.inf), (1, low), (2, math.nan)):
        some = x[row, keep].clone()
        x[row] = value
        x[row, keep] = some
    x[3] = -math.inf          # nothing to draw
    x[4] = math.nan
    x[5] = low                # all at the type's lowest value: equal, so all stay
    x[6, [9, 11, 500]] = math.inf
    x[7] = -math.inf
    x[7, 1234] = low          # one token left
    x[8, 1::2] = math.nan
    for kw in ({}, dict(top_k=2), dict(top_p=0.8), dict(top_k=50, top_p=0.9, min_p=0.1), dict(temperature=0.0),
               dict(min_p=1.0), dict(top_p=0.0), dict(top_k=1000)):
        want, _ = _check(x, e, **kw)
        assert want[3] == want[4] == -1 and want[7] == 1234 and want[6] in (9, 11, 500)
        assert all(want[r] in keep.tolist() for r in (0, 1, 2))


@pytest.mark.gpu
def test_extreme_temperatures_and_noise():
    x, e = _inputs(6, 2000, torch.float32, seed=44)
    _check(x, e, 1e-3)
    _check(x, e, 50.0, top_p=0.9)
    x2 = x * 1e3
    _check(x2, e, 1.0, top_k=7)
    from co_alibi_attn import sample_tokens
    tok, lp = sample_tokens(x.cuda(), e.cuda(), temperature=-1.0)
    assert tok.tolist() == x.argmax(1).tolist() and (lp == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides_and_alignment(dt):
    x, e = _inputs(5, 777, DT[dt], seed=45)
    wide = torch.zeros(5, 1001, dtype=DT[dt], device="cuda")[:, 3:780]
    wide.copy_(x)
    we = torch.zeros(5, 790, device="cuda")[:, 1:778]
    we.copy_(e)
    _check(x, e, 0.9, 30, 0.9, device_x=wide, device_e=we)
    _check(x, e, 0.9, 0, 0.9, device_x=x.t().contiguous().cuda().t(), device_e=e.t().contiguous().cuda().t())
    one = x[:1].cuda().expand(5, 777)  # one row for all
    _check(x[:1].expand(5, 777), e, 0.9, 30, device_x=one)


@pytest.mark.gpu
def test_draws_follow_the_distribution():
    from co_alibi_attn import sample_tokens
    n, logits = 200_000, torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -2.0, 1.5, 0.2])
    noise = torch.empty(n, 8, device="cuda").exponential_(generator=torch.Generator(device="cuda").manual_seed(46))
    tok, _ = sample_tokens(logits.cuda().expand(n, 8), noise, temperature=0.9, top_k=6, top_p=0.93)
    p = torch.softmax(logits.double() / 0.9, 0)
    order = p.argsort(descending=True)[:6]
    mass = p[order] / p[order].sum()
    order = order[(mass.cumsum(0) - mass) < 0.93]
    want = torch.zeros(8, dtype=torch.float64)
    want[order] = p[order] / p[order].sum()
    got = torch.bincount(tok, minlength=8).double().cpu() / n
    assert ((got - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all()


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_in_a_graph():
    from co_alibi_attn import sample_tokens
    x, e = (t.cuda() for t in _inputs(33, 20011, torch.float32, seed=47))
    first = sample_tokens(x, e, top_p=0.9)
    for _ in range(3):
        again = sample_tokens(x, e, top_p=0.9)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, e, top_p=0.9)
    graph.replay()
    assert torch.equal(out[0], first[0]) and torch.equal(out[1], first[1])
    x.copy_(x.flip(0).clone())
    e.copy_(e.flip(0).clone())
    graph.replay()
    assert torch.equal(out[0], first[0].flip(0))


def test_refusals_of_the_c_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_sample(None, None) == 1
    base = dict(logits=16, noise=16, temperature=None, top_k=None, top_p=None, min_p=None, tokens=16, logprobs=16,
                logits_stride=100, noise_stride=100, B=2, V=100, dtype=2, temperature_all=1.0, top_k_all=0,
                top_p_all=1.0, min_p_all=0.0)
    code = lambda **kw: lib.coalibi_sample(ctypes.byref(_lib.CoalibiSampleArgs(**{**base, **kw})), None)  # noqa: E731
    for field in ("logits", "noise", "tokens", "logprobs"):
        assert code(**{field: None}) == 1
    assert code(dtype=3) == 3
    for bad in (dict(B=0), dict(V=0), dict(V=(1 << 21) + 1), dict(logits_stride=-1)):
        assert code(**bad) == 4
    for bad in (dict(logits=18), dict(noise=17), dict(tokens=20), dict(logprobs=18)):
        assert code(**bad) == 5


def test_refuses_cpu_tensors():
    from co_alibi_attn import sample_tokens
    with pytest.raises(AssertionError):
        sample_tokens(torch.zeros(1, 4), torch.ones(1, 4))


@pytest.mark.gpu
def test_refusals():
    from co_alibi_attn import sample_tokens
    x, e = torch.zeros(2, 8, device="cuda"), torch.ones(2, 8, device="cuda")
    sample_tokens(x, e)
    assert sample_tokens(x[:0], e[:0])[0].shape == (0,)
    for kind, a, b, kw in (
            (ValueError, x[0], e[0], {}), (ValueError, x, e[:1], {}), (TypeError, x.double(), e, {}),
            (TypeError, x, e.half(), {}), (ValueError, x, e.cpu(), {}), (ValueError, x[:, :0], e[:, :0], {}),
            (TypeError, x, e, dict(top_k=torch.ones(2, dtype=torch.int64, device="cuda"))),
            (TypeError, x, e, dict(temperature=torch.ones(2, dtype=torch.float64, device="cuda"))),
            (ValueError, x, e, dict(top_p=torch.ones(3, device="cuda"))),
            (ValueError, x, e, dict(min_p=torch.ones(2)))):
        with pytest.raises(kind):
            sample_tokens(a, b, **kw)
