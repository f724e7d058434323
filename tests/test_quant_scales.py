"""A cache in 8 bits whose scales another program wrote, or that holds blocks of zeros: a value is its code
times the scale of its block, whatever that is.  Against the definitions in 64 bits."""
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_quant_append import _new, _same, _tables
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


@pytest.mark.gpu
def test_new_tokens_by_a_scale_that_is_no_power_of_two():
    """A block keeps such a scale where it is large enough, and its new codes are the nearest ones: borders between codes
    fall to the even one, and what lies off them by less than a float32 quotient tells, to its own side."""
    import co_alibi_attn
    D, Hkv = 64, 4
    border = (qr.GRID[1:] + qr.GRID[:-1])[7:].div(2).float()  # (5 bits each)
    scales = torch.tensor([k / 32 for k in range(33, 64)] + [0.7, 1 / 3, 3e-5, 1.1e4])
    S, pages = 15, len(scales)
    x = torch.empty(pages, Hkv, S, D)
    for p, s in enumerate(scales):
        y = (border * s)[border * s < 60000]
        x[p] = y[torch.arange(x[p].numel()) % len(y)].view(x[p].shape)
    x = (x * (1 - 2 * (torch.arange(S) % 2))[None, None, :, None])
    codes = torch.randint(0, 127, (pages, Hkv, 16, D), dtype=torch.uint8, generator=torch.Generator().manual_seed(96))
    was = scales[:, None, None].expand(pages, Hkv, 1).contiguous()
    table = torch.arange(pages, dtype=torch.int32)[:, None]
    for dt in (f16, bf16):  # a border times k / 32 is a float16; the rest are what they round to
        new = x.to(dt)
        want = codes.clone(), was.clone()
        qr.append(new, *want, table, [1] * pages, [S] * pages)
        kd, vd, ks, vs = qr.e4m3(codes.cuda()), qr.e4m3(codes.cuda()), was.cuda(), was.cuda()
        co_alibi_attn.append_paged_kv(new.cuda(), new.cuda(), kd, vd, table.cuda(), torch.ones(pages, dtype=torch.int32).cuda(), scales=(ks, vs))
        assert torch.equal(ks.cpu(), want[1]) and torch.equal(vs.cpu(), want[1])
        assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("D,dt,rot", [(64, f16, 0), (128, bf16, 64)])
def test_old_tokens_move_from_any_scale(D, dt, rot):
    """Codes under a smaller scale that is no power of two, 0 or negative go to the new one with one rounding of the exact
    product; larger scales stay, rotated keys among the new ones."""
    import co_alibi_attn
    Hkv, S, B = 3, 6, 40
    g = torch.Generator().manual_seed(97)
    kc, vc, ks, vs, table = qr.pool([30] * B, Hkv, D, 32, 98)
    for s in (ks, vs):
        s.copy_(torch.tensor([1 / 448, 1.5 / 512, 0.0, -0.01, 1e-9, 0.3, 1.75, 1.0, 123.4, 2e-38])[torch.randint(0, 10, s.shape, generator=g)]
                * (1 + torch.rand(s.shape, generator=g) * (torch.rand(s.shape, generator=g) < 0.5)))
    start = [5 + b % 17 for b in range(B)]
    q, k, v = _new(B, 4, Hkv, S, D, dt, 99)
    rotary, k_in = None, k.double()
    if rot:
        cos, sin = _tables(60, rot)
        at = torch.tensor(start)[:, None] + torch.arange(S)
        k_in, rotary = qr.rotated32(k, cos[at][:, None], sin[at][:, None], False), (cos.cuda(), sin.cuda())
    want = [x.clone() for x in (kc, vc, ks, vs)]
    qr.append(k_in, want[0], want[2], table, start, [S] * B)
    qr.append(v, want[1], want[3], table, start, [S] * B)
    kd, vd, ksd, vsd = qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), ks.cuda(), vs.cuda()
    co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), torch.tensor(start, dtype=torch.int32).cuda(), rotary=rotary, scales=(ksd, vsd))
    assert torch.equal(ksd.cpu(), want[2]) and torch.equal(vsd.cpu(), want[3])
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[1])
