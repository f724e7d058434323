"""A cache in 8 bits whose scales another program wrote, or that holds blocks of zeros: a value is its code
times the scale of its block, whatever that is.  Against the definitions in 64 bits."""
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_quant_attention import FORMS, IDS, _case, _check, _run, _widen

f16, bf16 = torch.float16, torch.bfloat16


def _bounded(q, kc, vc, ks, vs, table, ctx, words, slopes, scale):
    """(o, bound) of tests/_quant_ref.py, whose bound takes the size of a block's scale, 2^-100 at least."""
    o, _ = qr.attention(q, kc, vc, ks, vs, table, ctx, words, slopes, scale)
    size, bound = qr.attention(q, kc, vc, ks, vs.abs().clamp(min=2.0 ** -100), table, ctx, words, slopes, scale)
    return o, bound + ref.U[q.dtype] * (o.abs() - size.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("kind", ["zeros", "signs", "small", "all zero"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_attention_takes_any_scale(form, kind, width):
    """Blocks of scale 0 (with any codes), of negative scales, and of scales that flush to 0 beside ordinary ones."""
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx, kc, vc, ks, vs, table, words, q, slopes = _case(form, width, 90)
    g = torch.Generator().manual_seed(91)
    pick = lambda n: torch.randint(0, n, vs.shape, generator=g)  # noqa: E731
    if kind == "zeros":
        ks, vs = torch.where(pick(4) == 0, 0.0, ks), torch.where(pick(3) == 0, 0.0, vs)
    elif kind == "signs":
        ks, vs = torch.where(pick(2) == 0, -ks, ks), torch.where(pick(2) == 0, -1.375 * vs, vs)
    elif kind == "small":
        vs = torch.where(pick(2) == 0, torch.tensor([1e-45, -1e-38, 2.0 ** -120, -2.0 ** -101, 2.0 ** -90, 1e-13])[pick(6)], vs)
    else:
        vs = torch.where(pick(2) == 0, -0.0, 0.0)
    o = _run(q, kc, vc, ks, vs, _widen(table, 4096) if width == "wide" else table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    _check(o, *_bounded(q, kc, vc, ks, vs, table, ctx, words, slopes, 1 / math.sqrt(D)))
    if kind == "all zero":
        assert (o == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_keys_of_zero_values_keep_their_weight(form, width):
    """Blocks of zeros as the append writes them, scale 2^-100, beside values of 2^25: their keys count in the sum
    of the weights, though what they add to the result is 2^-120 of the others'."""
    Hq, Hkv, Sq, D, _ = form
    ctx, kc, vc, ks, vs, table, words, q, _ = _case((Hq, Hkv, Sq, D, bf16), width, 92)
    g = torch.Generator().manual_seed(93)
    none = torch.randint(0, 2, vs.shape, generator=g) == 0
    vs = torch.where(none, 2.0 ** -100, vs * 2.0 ** 24)
    vc = torch.where(none.repeat_interleave(16, 2)[..., None], 0, vc)
    slopes, scale = torch.full((Hq,), 0.02), 0.5
    o = _run(q, kc, vc, ks, vs, _widen(table, 4096) if width == "wide" else table, ctx, words, slopes=slopes.cuda(), sm_scale=scale)
    _check(o, *_bounded(q, kc, vc, ks, vs, table, ctx, words, slopes, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [f16, bf16])
def test_reading_takes_any_scale(dt):
    """A code times its block's scale, rounded once; past the type's largest, that, of either sign."""
    import co_alibi_attn
    Hkv, D, page, n = 3, 64, 48, 200
    kc, vc, ks, vs, table = qr.pool([n], Hkv, D, page, 94)
    sizes = torch.tensor([0.0, 1.0, 0.3, 1e-9, 129.0, 7e4, 1e30, 7.1e35, 3e38, 2.0 ** -130])
    sizes = torch.cat((sizes, -sizes))  # (19 blocks apart: every page and head has others)
    for i, s in enumerate((ks, vs)):
        s.copy_(sizes[(torch.arange(s.numel()) * 19 + i) % len(sizes)].view(s.shape))
    at = torch.arange(n, dtype=torch.int32)[None]
    got = co_alibi_attn.read_paged_kv(qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda(), at.cuda(), (ks.cuda(), vs.cuda()), dtype=dt)
    top = torch.finfo(dt).max
    for x, c, s in zip(got, (kc, vc), (ks, vs)):
        assert torch.equal(x[0].cpu(), ref.gather(qr.dequantised(c, s), table, 0, n).clamp(-top, top).to(dt))
