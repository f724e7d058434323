"""Bad data in every form of the attention kernel: drafts that are not finite, pages outside the
pool, stale slots; over 4, 24, 32 (warp-level), 48 (tcgen05, rows twice in the tile) and 132
rows per kv head (tcgen05), with tables cut to the requests (items whole) and tables of 4096
keys (items split over CTAs and joined).  Tolerances as in test_serving_attention.py."""
import math

import pytest
import torch

from tests import _serving_ref as ref
from tests.test_serving_attention import _check, _q, _run, _slopes

pytestmark = pytest.mark.gpu

f16, bf16 = torch.float16, torch.bfloat16
PAGE = 16
FORMS = [(4, 2, 2, 128, bf16), (4, 2, 12, 64, f16), (8, 2, 8, 128, f16), (8, 2, 12, 128, bf16), (8, 2, 12, 64, f16),
         (8, 2, 33, 128, f16), (8, 2, 33, 64, bf16)]
IDS = [f"rows{h // g * s}D{d}" for h, g, s, d, _ in FORMS]
# (narrow tables: at most 512 keys, so that no form splits)
CTX = {"cut": [0, 5, 21, 37, 58, 64, 100, 233, 470], "wide": [0, 5, 37, 64, 100, 470, 1023, 1500, 2222]}


def _widen(table, keys):
    wide = torch.full((table.shape[0], keys // PAGE), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


def _definition(q, k, v, table, ctx, words, slopes, lost=()):
    """(o, P @ |V|) in float64; keys of the (request, page) pairs in ``lost`` are seen by no row."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    o, pav = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        n = ctx[b] + Sq
        safe = table[b:b + 1].clamp(0, k.shape[0] - 1)
        kb, vb = (ref.gather(x, safe, 0, n).double().repeat_interleave(G, 0) for x in (k, v))
        see = torch.ones(Sq, n, dtype=torch.bool)
        see[:, ctx[b]:] = torch.tensor([[bool(w >> t & 1) for t in range(Sq)] for w in words[b]])
        for c, page in lost:
            if c == b:
                see[:, page * PAGE:(page + 1) * PAGE] = False
        p = q[b].double() @ kb.transpose(1, 2) / math.sqrt(D)
        z = torch.where(see, torch.sigmoid(p), 0.0).flip(-1).cumsum(-1).flip(-1)
        x = (p - slopes.double()[:, None, None] * z).masked_fill(~see, -math.inf)
        w = torch.softmax(x, -1).masked_fill(~see.any(1)[:, None], 0.0)
        o[b], pav[b] = w @ vb, w @ vb.abs()
    return o, pav


def _case(form, width, seed):
    Hq, Hkv, Sq, D, dt = form
    ctx = [c for c in CTX[width] if width == "wide" or c + Sq <= 512]
    k, v, table = ref.pool([c + Sq for c in ctx], Hkv, D, PAGE, dt, seed=seed)
    words = [ref.tree(Sq, seed + 1 + b) for b in range(len(ctx))]
    return ctx, k, v, table, words, _q(len(ctx), Hq, Sq, D, dt, seed + 50), _slopes(Hq)(dt)


@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_drafts_that_are_not_finite(form, bad, width):
    """In the contexts' places the draft falls into either half of a step, or a partial last one."""
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx, k, v, table, words, q, slopes = _case(form, width, 60)
    o_ref, pav = _definition(q, k, v, table, ctx, words, slopes)
    t = 1 if Sq < 5 else 4
    places = [(t, slice(3, 5))]
    if Sq > 2:  # and the last draft in another column
        places.append((Sq - 1, slice(D - 1, D)))
    for b, c in enumerate(ctx):
        for draft, cols in places:
            v[table[b, (c + draft) // PAGE], :, (c + draft) % PAGE, cols] = bad
    o = _run(q, k, v, _widen(table, 4096) if width == "wide" else table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    for b in range(len(ctx)):
        for i in range(Sq):
            for draft, cols in places:
                if words[b][i] >> draft & 1:
                    got = o[b, :, i, cols].cpu().float()
                    assert (got.isnan() if math.isnan(bad) else got == bad).all(), (b, i, draft)
                    o[b, :, i, cols] = o_ref[b, :, i, cols].to(o)
    _check(o, o_ref, pav, dt)


@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("entry", [-1, 1 << 30])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_pages_outside_the_pool(form, entry, width):
    """First, middle, neighbouring and last pages of the requests: their keys count for no row."""
    import co_alibi_attn
    ctx, k, v, table, words, q, slopes = _case(form, width, 70)
    Sq, lost = form[2], []
    for b, c in enumerate(ctx):
        n = -(-(c + Sq) // PAGE)
        some = [[], [0], [n - 1], [n // 2], [n // 2, min(n // 2 + 1, n - 1)], [0, n // 3, n - 1], list(range(0, n, 2)), [1], [n - 2]]
        for page in some[b % len(some)]:
            if 0 <= page < n and (b, page) not in lost:
                lost.append((b, page))
    t2 = table.clone()
    for b, page in lost:
        t2[b, page] = entry
    o = _run(q, k, v, _widen(t2, 4096) if width == "wide" else t2, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 11
    o_ref, pav = _definition(q, k, v, table, ctx, words, slopes, lost)
    _check(o, o_ref, pav, form[4])


@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_stale_slots_and_unseen_drafts(form, width):
    """Keys and values that no row sees hold NaN; rows of words 0 see the context alone."""
    import co_alibi_attn
    ctx, k, v, table, words, q, slopes = _case(form, width, 80)
    Sq = form[2]
    words = [[(w & ~0b1000) if i % 3 else 0 for i, w in enumerate(ws)] for ws in words]  # draft 3 unseen
    o_ref, pav = _definition(q, k, v, table, ctx, words, slopes)
    used = torch.zeros(k.shape[0], PAGE, dtype=torch.bool)
    for b, c in enumerate(ctx):
        any_word = 0
        for w in words[b]:
            any_word |= w
        for t in [*range(c), *(c + t for t in range(Sq) if any_word >> t & 1)]:
            used[table[b, t // PAGE], t % PAGE] = True
    hole = ~used[:, None, :, None].expand_as(k)
    k, v = k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan)
    o = _run(q, k, v, _widen(table, 4096) if width == "wide" else table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    _check(o, o_ref, pav, form[4])
