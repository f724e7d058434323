"""Co-ALiBi attention over a paged cache in 8 bits, against its definition in 64 bits; the bound of
the error is derived in tests/_quant_ref.py."""
import ctypes
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_quant_append import _device, _scales
from tests.test_serving_attention import CASES, _chain, _q, _slopes

f16, bf16 = torch.float16, torch.bfloat16


def _run(q, kc, vc, ks, vs, table, ctx, words=None, token_major=False, **kw):
    import co_alibi_attn
    mask = None if words is None else torch.tensor([ref.as_int64(w) for w in words], dtype=torch.int64).cuda()
    o = co_alibi_attn.paged_tree_attention(q.cuda(), _device(kc, token_major), _device(vc, token_major), table.cuda(),
                                           torch.tensor(ctx, dtype=torch.int32).cuda(), tree_mask=mask, scales=(ks.cuda(), vs.cuda()), **kw)
    torch.cuda.synchronize()
    return o


def _check(o, want, bound):
    assert torch.isfinite(o).all()
    err = (o.cpu().double() - want).abs()
    assert (err <= bound).all(), f"worst excess {(err - bound).max().item():.3e}, error {err.max().item():.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"H{c[0]}-{c[1]}D{c[2]}Sq{c[3]}L{max(c[4])}p{c[5]}" for c in CASES])
def test_matches_definition(case):
    import co_alibi_attn
    Hq, Hkv, D, Sq, ctx, page, dt, token_major, is_tree = case
    B = len(ctx)
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, page, 5, spread=1.0)
    q = _q(B, Hq, Sq, D, dt, 6)
    words = [ref.tree(Sq, 7 + b) for b in range(B)] if is_tree else _chain(B, Sq)
    o = _run(q, kc, vc, ks, vs, table, ctx, words if is_tree else None, token_major)
    assert co_alibi_attn.device_status(reset=True) == 0
    _check(o, *qr.attention(q, kc, vc, ks, vs, table, ctx, words, _slopes(Hq)(dt), 1 / math.sqrt(D)))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,Sq,dt", [(8, 2, 128, 1, bf16), (4, 4, 64, 1, f16), (8, 2, 64, 4, bf16), (8, 2, 128, 8, f16), (8, 2, 64, 16, bf16)])
@pytest.mark.parametrize("spread", [6.0, 24.0])
def test_blocks_of_unlike_scales(Hq, Hkv, D, Sq, dt, spread):
    """Blocks of V whose sizes differ by far more than float16 spans; whole and split items."""
    ctx = [900, 3, 17, 2300]
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, 16, 21)
    g = torch.Generator().manual_seed(22)
    vs = vs * 2.0 ** torch.randint(-int(spread), int(spread) + 1, vs.shape, generator=g)
    ks = ks * 2.0 ** torch.randint(-3, 2, ks.shape, generator=g)
    q = _q(4, Hq, Sq, D, dt, 23)
    slopes = torch.full((Hq,), 0.02)  # far keys keep weight
    o = _run(q, kc, vc, ks, vs, table, ctx, slopes=slopes.cuda())
    want, bound = qr.attention(q, kc, vc, ks, vs, table, ctx, _chain(4, Sq), slopes, 1 / math.sqrt(D))
    inside = want.abs() < 0.99 * torch.finfo(dt).max  # (others may be infinite in float16)
    err = (o.cpu().double() - want).abs()
    assert (err <= bound)[inside].all(), f"worst excess {(err - bound)[inside].max().item():.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e5, 1e30])
def test_queries_of_any_size(size):
    """bfloat16 queries go through float16 scaled by a power of two; the scale of the scores takes them back."""
    Hq, Hkv, D, ctx = 4, 2, 64, [200, 31]
    kc, vc, ks, vs, table = qr.pool([c + 1 for c in ctx], Hkv, D, 16, 24)
    q = _q(2, Hq, 1, D, torch.float32, 25)
    q[0, 1] = 0
    q = (q * size * 2.0 ** torch.tensor([0, 0, -7, 5])[None, :, None, None]).to(bf16)
    scale = 0.1 / size
    o = _run(q, kc, vc, ks, vs, table, ctx, sm_scale=scale)
    _check(o, *qr.attention(q, kc, vc, ks, vs, table, ctx, _chain(2, 1), _slopes(Hq)(bf16), scale))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,L,dt", [(8, 2, 128, 20000, bf16), (4, 4, 64, 9000, f16)])
def test_long_context_with_spread_weights(Hq, Hkv, D, L, dt):
    kc, vc, ks, vs, table = qr.pool([L + 1], Hkv, D, 32, 4)
    q = _q(1, Hq, 1, D, dt, 3)
    slopes = torch.full((Hq,), 0.002)
    o = _run(q, kc, vc, ks, vs, table, [L], slopes=slopes.cuda(), sm_scale=0.02)
    _check(o, *qr.attention(q, kc, vc, ks, vs, table, [L], _chain(1, 1), slopes, 0.02))


@pytest.mark.gpu
@pytest.mark.parametrize("short", [False, True])  # short tables: items are not split
@pytest.mark.parametrize("Hq,Hkv,D,Sq", [(24, 8, 128, 1), (32, 8, 64, 3), (32, 8, 64, 5), (32, 8, 128, 16), (16, 4, 64, 12), (24, 4, 128, 20)])
def test_many_ragged_requests(Hq, Hkv, D, Sq, short):
    dt, page = bf16, 16
    ctx = [0, 1, 15, 16, 31, 33] + (list(range(40, 470, 19)) if short else list(range(40, 620, 29)) + [1500, 2047])
    B = len(ctx)
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, page, 24)
    q = _q(B, Hq, Sq, D, dt, 25)
    words = [ref.tree(Sq, 26 + b) for b in range(B)]
    o = _run(q, kc, vc, ks, vs, table, ctx, words)
    want, bound = qr.attention(q, kc, vc, ks, vs, table, ctx, words, _slopes(Hq)(dt), 1 / math.sqrt(D))
    _check(o, want, bound)
    if Sq == 1:  # more requests than threads that sum the lengths; tables as views of wider ones
        import co_alibi_attn
        many = torch.randint(0, B, (300,), generator=torch.Generator().manual_seed(27))
        wide = torch.full((300, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
        wide[:, 2:-3] = table[many].cuda()
        got = co_alibi_attn.paged_tree_attention(q[many].cuda(), qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), wide[:, 2:-3],
                                                 torch.tensor(ctx, dtype=torch.int32)[many].cuda(), scales=(ks.cuda(), vs.cuda()))
        _check(got, want[many], bound[many])


PAGE = 16
FORMS = [(4, 2, 2, 128, bf16), (4, 2, 8, 64, f16), (4, 2, 12, 64, f16), (8, 2, 8, 128, f16), (8, 2, 12, 128, bf16), (8, 2, 12, 64, f16),
         (8, 2, 33, 128, f16), (8, 2, 33, 64, bf16)]
IDS = [f"rows{h // g * s}D{d}" for h, g, s, d, _ in FORMS]
CTX = {"cut": [0, 5, 21, 37, 58, 64, 100, 233, 470], "wide": [0, 5, 37, 64, 100, 470, 1023, 1500, 2222]}


def _widen(table, keys):
    wide = torch.full((table.shape[0], keys // PAGE), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


def _case(form, width, seed):
    Hq, Hkv, Sq, D, dt = form
    ctx = [c for c in CTX[width] if width == "wide" or c + Sq <= 512]
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, PAGE, seed)
    words = [ref.tree(Sq, seed + 1 + b) for b in range(len(ctx))]
    return ctx, kc, vc, ks, vs, table, words, _q(len(ctx), Hq, Sq, D, dt, seed + 50), _slopes(Hq)(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_drafts_of_nan(form, width):
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx, kc, vc, ks, vs, table, words, q, slopes = _case(form, width, 60)
    want, bound = qr.attention(q, kc, vc, ks, vs, table, ctx, words, slopes, 1 / math.sqrt(D))
    t = 1 if Sq < 5 else 4
    places = [(t, slice(3, 5))] + ([(Sq - 1, slice(D - 1, D))] if Sq > 2 else [])
    for b, c in enumerate(ctx):
        for draft, cols in places:
            vc[table[b, (c + draft) // PAGE], :, (c + draft) % PAGE, cols] = 0x7f if b % 2 else 0xff
    o = _run(q, kc, vc, ks, vs, _widen(table, 4096) if width == "wide" else table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    for b in range(len(ctx)):
        for i in range(Sq):
            for draft, cols in places:
                if words[b][i] >> draft & 1:
                    assert o[b, :, i, cols].isnan().all(), (b, i, draft)
                    o[b, :, i, cols] = want[b, :, i, cols].to(o)
    _check(o, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_what_no_row_sees_may_hold_anything(form, width):
    """Slots behind the drafts, drafts that no word names, and blocks of them alone, with any code and scale."""
    Hq, Hkv, Sq, D, dt = form
    ctx, kc, vc, ks, vs, table, words, q, slopes = _case(form, width, 65)
    hide = [t for t in range(Sq) if t % 3 == 2] + ([Sq - 1] if Sq > 2 else [])
    words = [[w & ~sum(1 << t for t in set(hide)) for w in ws] for ws in words]
    want, bound = qr.attention(q, kc, vc, ks, vs, table, ctx, words, slopes, 1 / math.sqrt(D))
    for b, c in enumerate(ctx):
        unseen = [c + t for t in range(Sq) if not any(w >> t & 1 for w in words[b])]
        unseen += list(range(c + Sq, -(-(c + Sq) // PAGE) * PAGE))
        for x in (kc, vc):
            for t in unseen:
                x[table[b, t // PAGE], :, t % PAGE] = 0x7f
        for n in range(-(-(c + Sq) // PAGE)):
            if all(t in unseen for t in range(n * PAGE, (n + 1) * PAGE)):
                ks[table[b, n]], vs[table[b, n]] = math.nan, math.inf if b % 2 else math.nan
    o = _run(q, kc, vc, ks, vs, _widen(table, 4096) if width == "wide" else table, ctx, words)
    _check(o, want, bound)
    for b, ws in enumerate(words):
        for i, w in enumerate(ws):
            if w == 0 and ctx[b] == 0:
                assert (o[b, :, i] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("entry", [-1, 1 << 30])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_pages_outside_the_pool(form, entry, width):
    """Their keys count for no row: as if the request did not have them."""
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx, kc, vc, ks, vs, table, words, q, slopes = _case(form, width, 70)
    keep, ctx2, t2, words2 = [], [], table.clone(), []
    for b, c in enumerate(ctx):
        n = c // PAGE  # whole pages of the context
        lost = {page for page in [[], [0], [n - 1], [n // 2], [n // 2, n // 2 + 1], [0, n // 3, n - 1], list(range(0, n, 2))][b % 7] if 0 <= page < n}
        t2[b, sorted(lost)] = entry
        keep.append([p for p in range(table.shape[1]) if p not in lost])
        ctx2.append(c - PAGE * len(lost))
    short = torch.full_like(table, -1)
    for b, pages in enumerate(keep):
        short[b, :len(pages)] = table[b, pages]
    want, bound = qr.attention(q, kc, vc, ks, vs, short, ctx2, words, slopes, 1 / math.sqrt(D))
    o = _run(q, kc, vc, ks, vs, _widen(t2, 4096) if width == "wide" else t2, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 11
    _check(o, want, bound)


@pytest.mark.gpu
def test_lengths_out_of_range():
    """Negative lengths count as 0; a request longer than its table ends there and is reported."""
    import co_alibi_attn
    Hq, Hkv, D, dt = 4, 2, 64, f16
    kc, vc, ks, vs, table = qr.pool([48, 48, 48], Hkv, D, 16, 31)
    q = _q(3, Hq, 1, D, dt, 32)
    o = _run(q, kc, vc, ks, vs, table, [-5, 47, 0])
    assert co_alibi_attn.device_status(reset=True) == 0
    _check(o, *qr.attention(q, kc, vc, ks, vs, table, [0, 47, 0], _chain(3, 1), _slopes(Hq)(dt), 1 / math.sqrt(D)))
    o = _run(q, kc, vc, ks, vs, table, [20, 48, (1 << 31) - 1])
    assert co_alibi_attn.device_status(reset=True) == 11
    words = [[1], [0], [0]]
    _check(o, *qr.attention(q, kc, vc, ks, vs, torch.cat((table, table[:, :1]), 1), [20, 48, 48], words, _slopes(Hq)(dt), 1 / math.sqrt(D)))
    empty = _run(q[:0], kc, vc, ks, vs, table[:0], [])
    assert empty.shape == (0, Hq, 1, D)


@pytest.mark.gpu
def test_strides_of_queries_and_scales():
    import co_alibi_attn
    Hq, Hkv, D, Sq, dt, ctx = 8, 2, 64, 3, bf16, [20, 33]
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, 32, 19)
    q = _q(2, Sq, Hq + 2, D, dt, 20).cuda().transpose(1, 2)[:, :Hq]
    wide = torch.full((2, ks.shape[0], 5, ks.shape[2] + 3), math.nan, device="cuda")
    wide[0, :, 1:3, 1:-2], wide[1, :, 1:3, 1:-2] = ks.cuda(), vs.cuda()
    lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    o = co_alibi_attn.paged_tree_attention(q, qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda(), lens,
                                           scales=(wide[0, :, 1:3, 1:-2], wide[1, :, 1:3, 1:-2]))
    assert o.transpose(1, 2).is_contiguous()
    assert torch.equal(o, _run(q, kc, vc, ks, vs, table, ctx))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Sq", [(8, 4), (8, 12), (2, 1)])
def test_repeats_bit_for_bit_on_any_stream_and_in_a_graph(Hq, Sq):
    import co_alibi_attn
    Hkv, D, dt = 2, 128, bf16
    ctx = [3000, 17, 0, 800]
    kc, vc, ks, vs, table = (x.cuda() for x in qr.pool([c + Sq for c in ctx], Hkv, D, 64, 22))
    k, v = qr.e4m3(kc), qr.e4m3(vc)
    q = _q(4, Hq, Sq, D, dt, 23).cuda()
    lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    run = lambda q, lens: co_alibi_attn.paged_tree_attention(q, k, v, table, lens, scales=(ks, vs))  # noqa: E731
    want = [run(q, lens) for _ in range(3)]
    other = run(q, (lens - 5).clamp(min=0))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q2 = q * 1.0  # written on the same stream right before
        want.append(run(q2, lens))
    torch.cuda.current_stream().wait_stream(s)
    static = lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(q, static)
    for lengths, expect in ((lens, want[0]), ((lens - 5).clamp(min=0), other), (lens, want[0])):
        static.copy_(lengths)
        graph.replay()
        assert torch.equal(out, expect)
    assert all(torch.equal(w, want[0]) for w in want)


def test_refusals_of_the_c_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_paged_attention8(None, None, None, 0, None) == 1
    strides = ("q_stride", "o_stride", "k_page_stride", "v_page_stride")
    base = dict(q=16, o=16, k_pages=16, v_pages=16, slopes=16, page_table=16, ctx_lens=16, tree_mask=None, status=None,
                q_stride=(512, 128, 128), o_stride=(512, 128, 128), k_page_stride=(4096, 2048, 128),
                v_page_stride=(4096, 2048, 128), table_stride=4, mask_stride=0, B=2, Hq=4, Hkv=2, Sq=1, D=128,
                page_size=16, max_pages=4, n_pages=8, dtype=0, slopes_dtype=0, sm_scale=0.1)

    def code(ws=256, bytes_=1 << 40, scales=None, **kw):
        d = {**base, **kw}
        for f in strides:
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        return lib.coalibi_paged_attention8(ctypes.byref(_lib.CoalibiPagedAttentionArgs(**d)),
                                            ctypes.byref(_scales(_lib, **(scales or {}))), ws, bytes_, None)

    for field in ("q", "o", "k_pages", "v_pages", "slopes", "page_table", "ctx_lens"):
        assert code(**{field: None}) == 1
    assert code(scales=dict(v=None)) == 1 and code(scales=dict(v=2)) == 5 and code(scales=dict(v_stride=(0, 1))) == 4
    assert code(D=96) == 2 and code(dtype=3) == 3 and code(slopes_dtype=5) == 3
    for bad in (dict(B=0), dict(Hq=3), dict(Sq=65), dict(Sq=0), dict(page_size=24), dict(page_size=0), dict(n_pages=0),
                dict(max_pages=1 << 28), dict(mask_stride=-1), dict(table_stride=-4)):
        assert code(**bad) == 4, bad
    for bad in (dict(q=24), dict(o=8), dict(k_pages=24), dict(q_stride=(512, 130, 128)), dict(tree_mask=20),
                dict(v_page_stride=(4096, 2056, 128)), dict(v_page_stride=(-4096, 2048, 128))):
        assert code(**bad) == 5, bad
    need = lib.coalibi_paged_attention8_workspace_bytes(2, 4, 2, 1, 128)
    assert need > 0 and code(ws=None) == 8 and code(ws=264) == 8 and code(bytes_=need - 1) == 8
    for bad in ((2, 4, 2, 65, 128), (2, 4, 3, 1, 128), (2, 4, 2, 1, 80), (0, 4, 2, 1, 64)):
        assert lib.coalibi_paged_attention8_workspace_bytes(*bad) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("page", [32, 64, 48])  # whole steps of 32 keys in a page, or not
@pytest.mark.parametrize("form", [f for f in FORMS if f[0] // f[1] * f[2] <= 32], ids=[i for i, f in zip(IDS, FORMS) if f[0] // f[1] * f[2] <= 32])
def test_stale_halves_of_steps(form, page):
    """Split items, one step to a load: codes and scales of NaN behind the last token, drafts of NaN that some rows see,
    pages outside the pool."""
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx = [0, 3, 16, 17, 31, 32, 47, 100, 480, 1011, 1500, 2222]
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, page, 80)
    words = [ref.tree(Sq, 81 + b) for b in range(len(ctx))]
    q, slopes = _q(len(ctx), Hq, Sq, D, dt, 82), _slopes(Hq)(dt)
    lost = {7: 100 // page - 1, 9: 0, 10: 7, 11: 2222 // page - 1}  # whole pages of the context
    t2, short, ctx2 = table.clone(), torch.full_like(table, -1), list(ctx)
    for b in range(len(ctx)):
        keep = [n for n in range(table.shape[1]) if n != lost.get(b)]
        if b in lost:
            t2[b, lost[b]] = -1 if b % 2 else 1 << 30
            ctx2[b] -= page
        short[b, :len(keep)] = table[b, keep]
    want, bound = qr.attention(q, kc, vc, ks, vs, short, ctx2, words, slopes, 1 / math.sqrt(D))
    t = 1 if Sq < 5 else 4
    for b, c in enumerate(ctx):
        vc[table[b, (c + t) // page], :, (c + t) % page, 3:5] = 0xff
        end = c + Sq
        last = table[b, (end - 1) // page]
        if end % page:
            kc[last, :, end % page:] = vc[last, :, end % page:] = 0x7f
            ks[last, :, -(-(end % page) // 16):] = vs[last, :, -(-(end % page) // 16):] = math.nan
    wide = torch.full((len(ctx), -(-16384 // page)), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = t2
    o = _run(q, kc, vc, ks, vs, wide, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 11
    for b in range(len(ctx)):
        for i in range(Sq):
            if words[b][i] >> t & 1:
                assert o[b, :, i, 3:5].isnan().all(), (b, i)
                o[b, :, i, 3:5] = want[b, :, i, 3:5].to(o)
    _check(o, want, bound)
