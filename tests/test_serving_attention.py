"""Co-ALiBi attention of one token or a drafted tree over a paged cache, against its
definition in 64 bits.

Tolerance, per element: u |o| (the output's rounding) + (u + 2^-12) (P @ |V|) + 2^-20,
with u half an ulp of the type: the weights are rounded to it before the product with V,
and 2^-12 bounds what a float32 score, sigmoid sum and exponential may move a weight by
(scores up to ~16 and slope * z up to ~60 where weights matter, a few ulp of 2^-18 each)."""
import ctypes
import math

import pytest
import torch

from tests import _serving_ref as ref


def _slopes(H):
    from co_alibi_attn.co_alibi_attn import _api_slopes
    return lambda dt: _api_slopes(H, 8.0, dt, torch.device("cpu"))


def _check(o, o_ref, pav, dt):
    u = ref.U[dt]
    err = (o.cpu().double() - o_ref).abs()
    bound = u * o_ref.abs() + (u + 2.0 ** -12) * pav + 2.0 ** -20
    assert torch.isfinite(o).all()
    assert (err <= bound).all(), f"worst excess {(err - bound).max().item():.3e}, error {err.max().item():.3e}"


def _run(q, k, v, table, ctx, words=None, **kw):
    import co_alibi_attn
    mask = None if words is None else torch.tensor([ref.as_int64(w) for w in words], dtype=torch.int64).cuda()
    o = co_alibi_attn.paged_tree_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(),
                                           torch.tensor(ctx, dtype=torch.int32).cuda(), tree_mask=mask, **kw)
    torch.cuda.synchronize()
    return o


def _chain(B, Sq):
    return [[(2 << i) - 1 for i in range(Sq)] for _ in range(B)]


def _q(B, Hq, Sq, D, dt, seed):
    return torch.randn(B, Hq, Sq, D, generator=torch.Generator().manual_seed(seed)).to(dt)


f16, bf16 = torch.float16, torch.bfloat16
CASES = [
    # Hq, Hkv, D, Sq, context lengths, page, dtype, token-major pool, tree
    (12, 12, 64, 1, [0], 16, f16, False, False),                 # the first token of all
    (12, 12, 64, 1, [1, 0, 15, 16, 17], 16, bf16, False, False),
    (8, 2, 128, 1, [31, 32, 33, 63, 64, 65, 127, 128, 129], 32, f16, False, False),
    (8, 2, 128, 1, [1000, 0, 77, 511], 48, bf16, True, False),   # pages that are no power of two
    (8, 1, 128, 1, [2500], 64, bf16, False, False),
    (4, 4, 64, 1, [4097], 128, f16, True, False),
    (16, 1, 64, 1, [300, 5], 16, f16, False, False),             # 16 rows share each key
    (24, 1, 128, 1, [300, 5], 16, bf16, False, False),           # 24
    (6, 3, 64, 5, [0, 3, 200], 16, bf16, False, False),          # a chain of 5
    (8, 8, 128, 7, [0, 100, 13], 32, f16, False, True),
    (8, 2, 128, 8, [40, 0, 999], 16, bf16, True, True),          # 32 rows
    (8, 2, 64, 16, [257, 16], 64, f16, False, True),             # 64 rows
    (32, 8, 128, 16, [700, 1], 16, bf16, False, True),
    (4, 1, 128, 33, [0, 95], 16, f16, False, True),              # 132 rows
    (2, 2, 64, 64, [0, 129], 16, bf16, False, True),             # bit 63 of the words
    (8, 1, 64, 64, [50], 48, f16, False, True),                  # 512 rows
    (1, 1, 128, 63, [31], 16, f16, False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"H{c[0]}-{c[1]}D{c[2]}Sq{c[3]}L{max(c[4])}p{c[5]}" for c in CASES])
def test_matches_definition(case):
    import co_alibi_attn
    Hq, Hkv, D, Sq, ctx, page, dt, token_major, is_tree = case
    B = len(ctx)
    k, v, table = ref.pool([c + Sq for c in ctx], Hkv, D, page, dt, seed=5, token_major=token_major)
    q = _q(B, Hq, Sq, D, dt, 6)
    words = [ref.tree(Sq, 7 + b) for b in range(B)] if is_tree else _chain(B, Sq)
    if token_major:  # keep the strides on the device
        kd, vd = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (k, v))
    else:
        kd, vd = k.cuda(), v.cuda()
    o = _run(q, kd, vd, table, ctx, words if is_tree else None)
    assert co_alibi_attn.device_status(reset=True) == 0
    o_ref, pav = ref.attention(q, k, v, table, ctx, words, _slopes(Hq)(dt), 1 / math.sqrt(D))
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,L,dt", [(8, 2, 128, 20000, bf16), (4, 4, 64, 9000, f16)])
def test_long_context_with_spread_weights(Hq, Hkv, D, L, dt):
    """Mostly negative scores: the sigmoid sums grow slowly, so keys of every part of the
    cache keep weight and every join of the pieces shows."""
    g = torch.Generator().manual_seed(3)
    k, v, table = ref.pool([L + 1], Hkv, D, 32, dt, seed=4)
    lean = torch.randn(D, generator=g)
    k = (k.float() + 0.8 * lean).to(dt)
    q = (torch.randn(1, Hq, 1, D, generator=g) - 0.8 * lean).to(dt)
    slopes = torch.full((Hq,), 0.01)
    o = _run(q, k, v, table, [L], slopes=slopes.cuda())
    o_ref, pav = ref.attention(q, k, v, table, [L], _chain(1, 1), slopes, 1 / math.sqrt(D))
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("short", [False, True])  # short tables: items are not split
@pytest.mark.parametrize("Hq,Hkv,D,Sq", [(24, 8, 128, 1), (32, 8, 64, 5), (32, 8, 128, 16), (16, 4, 64, 12), (24, 4, 128, 20)])
def test_many_ragged_requests(Hq, Hkv, D, Sq, short):
    """More items than CTAs, of every length modulo the steps: items that end and begin within
    one CTA's run, pieces of unequal steps, masked steps before plain ones.  Float64 on the GPU."""
    dt, page = bf16, 16
    ctx = [0, 1, 15, 16, 31, 33] + (list(range(40, 470, 9)) if short else list(range(40, 620, 13)) + [1500, 2047])
    B = len(ctx)
    k, v, table = (x.cuda() for x in ref.pool([c + Sq for c in ctx], Hkv, D, page, dt, seed=24))
    q = _q(B, Hq, Sq, D, dt, 25).cuda()
    words = [ref.tree(Sq, 26 + b) for b in range(B)]
    slopes = _slopes(Hq)(dt).cuda()
    o = _run(q, k, v, table, ctx, words)
    if Sq == 1:  # more requests than threads that sum the lengths; tables as views of wider ones
        many = torch.randint(0, B, (300,), generator=torch.Generator().manual_seed(27))
        wide = torch.full((300, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
        wide[:, 2:-3] = table[many.cuda()]
        import co_alibi_attn
        got = co_alibi_attn.paged_tree_attention(q[many.cuda()], k, v, wide[:, 2:-3],
                                                 torch.tensor(ctx, dtype=torch.int32)[many].cuda())
        assert torch.allclose(got.float(), o[many.cuda()].float(), atol=2e-2, rtol=2e-2)  # split elsewhere
    for b, c in enumerate(ctx):
        kb, vb = (ref.gather(x, table, b, c + Sq).double() for x in (k, v))
        hidden = torch.zeros(Sq, c + Sq, dtype=torch.bool, device="cuda")
        hidden[:, c:] = torch.tensor([[not w >> t & 1 for t in range(Sq)] for w in words[b]], device="cuda")
        p = q[b].double() @ kb.repeat_interleave(Hq // Hkv, 0).transpose(1, 2) / math.sqrt(D)
        z = torch.sigmoid(p).masked_fill(hidden, 0).flip(-1).cumsum(-1).flip(-1)
        w = torch.softmax((p - slopes.double()[:, None, None] * z).masked_fill(hidden, -math.inf), -1)
        vv = vb.repeat_interleave(Hq // Hkv, 0)
        _check(o[b], (w @ vv).cpu(), (w @ vv.abs()).cpu(), dt)


@pytest.mark.gpu
def test_rows_that_see_nothing_and_unseen_drafts():
    """Words of 0 with an empty context give zero rows; drafts no word names are not read,
    so their slots may hold NaN, and their pages need not exist."""
    import co_alibi_attn
    Hq, Hkv, D, Sq, dt = 4, 2, 128, 20, f16
    ctx = [0, 0, 30]
    k, v, table = ref.pool([16, 16, 48], Hkv, D, 16, dt, seed=8)
    words = [[0] * Sq, [0, 1 << 2] + [0] * (Sq - 2), [1, 3] + [0] * (Sq - 2)]
    for t in (0, 1, 3, 4, 15):  # request 1 names draft 2 alone
        k[table[1, 0], :, t] = math.nan
        v[table[1, 0], :, t] = math.inf
    k[table[0, 0]] = math.nan
    v[table[0, 0]] = math.nan
    v[table[2, 2]] = math.nan  # past request 2's two drafts
    q = _q(3, Hq, Sq, D, dt, 9)
    o = _run(q, k, v, table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    assert (o[0] == 0).all() and (o[1, :, 0] == 0).all() and (o[1, :, 2:] == 0).all()
    assert torch.equal(o[1, :, 1].cpu(), v[table[1, 0], :, 2].repeat_interleave(Hq // Hkv, 0))
    k2, v2 = (torch.where(x.isfinite(), x, torch.zeros_like(x)) for x in (k, v))
    o_ref, pav = ref.attention(q, k2, v2, table, ctx, words, _slopes(Hq)(dt), 1 / math.sqrt(D))
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("D,bad", [(128, math.nan), (64, math.inf), (128, -math.inf)])
def test_a_draft_that_is_not_finite_stays_with_the_rows_that_see_it(D, bad):
    Hq, Hkv, Sq, dt, ctx = 4, 2, 12, bf16, [37, 0]
    k, v, table = ref.pool([c + Sq for c in ctx], Hkv, D, 16, dt, seed=10)
    words = [ref.tree(Sq, 11 + b) for b in range(2)]
    q = _q(2, Hq, Sq, D, dt, 12)
    o_ref, pav = ref.attention(q, k, v, table, ctx, words, _slopes(Hq)(dt), 1 / math.sqrt(D))
    for b in range(2):
        t = ctx[b] + 4
        v[table[b, t // 16], :, t % 16, 3:5] = bad
    o = _run(q, k, v, table, ctx, words)
    for b in range(2):
        for i in range(Sq):
            if words[b][i] >> 4 & 1:
                got = o[b, :, i, 3:5].cpu().float()
                assert (got.isnan() if math.isnan(bad) else got == bad).all()
                o[b, :, i, 3:5] = o_ref[b, :, i, 3:5].to(o)
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
def test_stale_slots_and_table_entries_do_not_matter():
    """Slots past a request's end hold NaN and the table's tail names pages of others."""
    Hq, Hkv, D, dt, ctx = 8, 2, 128, bf16, [9, 100]
    k, v, table = ref.pool([c + 1 for c in ctx], Hkv, D, 16, dt, seed=13)
    for b, c in enumerate(ctx):
        k[table[b, c // 16], :, c % 16 + 1:] = math.nan
        v[table[b, c // 16], :, c % 16 + 1:] = math.nan
    table[0, 1:] = 1 << 30
    q = _q(2, Hq, 1, D, dt, 14)
    o = _run(q, k, v, table, ctx)
    import co_alibi_attn
    assert co_alibi_attn.device_status(reset=True) == 0
    o_ref, pav = ref.attention(q, k, v, table, ctx, _chain(2, 1), _slopes(Hq)(dt), 1 / math.sqrt(D))
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
def test_pages_outside_the_pool_are_skipped_and_reported():
    import co_alibi_attn
    Hq, Hkv, D, dt, ctx = 4, 2, 64, f16, [70, 70]
    k, v, table = ref.pool([c + 1 for c in ctx], Hkv, D, 16, dt, seed=15)
    q = _q(2, Hq, 1, D, dt, 16)
    for bad in (-1, k.shape[0], 1 << 30):
        t2 = table.clone()
        t2[1, 2] = bad
        o = _run(q, k, v, t2, ctx)
        assert co_alibi_attn.device_status(reset=True) == 11
        assert torch.isfinite(o).all()
        assert torch.equal(o[0], _run(q, k, v, table, ctx)[0])
    # a length past the table's end
    o = _run(q, k, v, table, [70, 5000])
    assert co_alibi_attn.device_status(reset=True) == 11
    assert torch.isfinite(o).all()
    o = _run(q, k, v, table, [70, -5])  # a negative length is an empty context
    o_ref, pav = ref.attention(q, k, v, table, [70, 0], _chain(2, 1), _slopes(Hq)(dt), 1 / math.sqrt(D))
    co_alibi_attn.device_status(reset=True)
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the request's pages lie at its far end."""
    Hq, Hkv, D, page, dt, ctx = 8, 4, 128, 64, bf16, [150]
    n = (1 << 32) // (Hkv * page * D) + 8
    big = [torch.empty(n, Hkv, page, D, dtype=dt, device="cuda") for _ in range(2)]
    k, v, table = ref.pool([151], Hkv, D, page, dt, seed=17, spare=0)
    for x, y in zip(big, (k, v)):
        x[n - 3:] = y.cuda()
    q = _q(1, Hq, 1, D, dt, 18)
    o = _run(q, big[0], big[1], table + (n - 3), ctx)
    o_ref, pav = ref.attention(q, k, v, table, ctx, _chain(1, 1), _slopes(Hq)(dt), 1 / math.sqrt(D))
    _check(o, o_ref, pav, dt)


@pytest.mark.gpu
def test_query_strides_and_layout():
    """Queries as views of a fused projection; the result keeps their token-major order."""
    Hq, Hkv, D, Sq, dt, ctx = 8, 2, 64, 3, f16, [20, 33]
    k, v, table = ref.pool([c + Sq for c in ctx], Hkv, D, 16, dt, seed=19)
    qkv = _q(2, Sq, Hq + 2 * Hkv, D, dt, 20).cuda()
    q = qkv.transpose(1, 2)[:, :Hq]
    o = _run(q, k, v, table, ctx)
    assert o.transpose(1, 2).is_contiguous()
    assert torch.equal(o, _run(q.contiguous(), k, v, table, ctx))
    odd = torch.zeros(2 * Hq * Sq * D + 1, dtype=dt, device="cuda")[1:].view(2, Hq, Sq, D)  # rows off 16 bytes
    odd.copy_(q)
    assert torch.equal(o, _run(odd, k, v, table, ctx))


@pytest.mark.gpu
def test_agrees_with_the_causal_operator():
    """The last rows of a causal forward are a chain of drafted tokens over the others."""
    import co_alibi_attn
    Hq, Hkv, D, S, Sq, dt = 8, 2, 128, 300, 20, f16
    g = torch.Generator().manual_seed(21)
    q, k, v = (torch.randn(1, h, S, D, generator=g).to(dt).cuda() for h in (Hq, Hkv, Hkv))
    full = co_alibi_attn.co_alibi_attention(q, k, v, causal=True)[:, :, S - Sq:]
    kp, vp = (torch.zeros(19, Hkv, 16, D, dtype=dt, device="cuda") for _ in range(2))
    table = torch.arange(19, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    co_alibi_attn.append_paged_kv(k, v, kp, vp, table, zero)
    o = co_alibi_attn.paged_tree_attention(q[:, :, S - Sq:], kp, vp, table, zero + (S - Sq))
    assert (o.float() - full.float()).abs().max() <= 2 * 2e-3  # two results of the operator's own 2e-3


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_any_stream_and_in_a_graph():
    import co_alibi_attn
    Hq, Hkv, D, Sq, dt = 8, 2, 128, 4, bf16
    ctx = [3000, 17, 0, 800]
    k, v, table = (x.cuda() for x in ref.pool([c + Sq for c in ctx], Hkv, D, 64, dt, seed=22))
    q = _q(4, Hq, Sq, D, dt, 23).cuda()
    lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    want = [co_alibi_attn.paged_tree_attention(q, k, v, table, lens - d) for d in (0, 0, 0)]
    other = co_alibi_attn.paged_tree_attention(q, k, v, table, (lens - 5).clamp(min=0))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q2 = q * 1.0  # written on the same stream right before
        want.append(co_alibi_attn.paged_tree_attention(q2, k, v, table, lens))
    torch.cuda.current_stream().wait_stream(s)
    static = lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = co_alibi_attn.paged_tree_attention(q, k, v, table, static)
    for lengths, expect in ((lens, want[0]), ((lens - 5).clamp(min=0), other), (lens, want[0])):
        static.copy_(lengths)
        graph.replay()
        assert torch.equal(out, expect)
    assert all(torch.equal(w, want[0]) for w in want)


def test_refusals_of_the_c_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_paged_attention(None, None, 0, None) == 1
    base = dict(q=16, o=16, k_pages=16, v_pages=16, slopes=16, page_table=16, ctx_lens=16, tree_mask=None, status=None,
                q_stride=(512, 128, 128), o_stride=(512, 128, 128), k_page_stride=(4096, 2048, 128),
                v_page_stride=(4096, 2048, 128), table_stride=4, mask_stride=0, B=2, Hq=4, Hkv=2, Sq=1, D=128,
                page_size=16, max_pages=4, n_pages=8, dtype=0, slopes_dtype=0, sm_scale=0.1)

    def code(ws=256, **kw):
        d = {**base, **kw}
        for f in ("q_stride", "o_stride", "k_page_stride", "v_page_stride"):
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        a = _lib.CoalibiPagedAttentionArgs(**d)
        return lib.coalibi_paged_attention(ctypes.byref(a), ws, 1 << 40, None)

    for field in ("q", "o", "k_pages", "v_pages", "slopes", "page_table", "ctx_lens"):
        assert code(**{field: None}) == 1
    assert code(D=96) == 2
    assert code(dtype=2) == 3 and code(slopes_dtype=5) == 3
    for bad in (dict(B=0), dict(Hq=3), dict(Sq=65), dict(Sq=0), dict(page_size=24), dict(page_size=0), dict(n_pages=0),
                dict(max_pages=1 << 28), dict(mask_stride=-1), dict(table_stride=-4)):
        assert code(**bad) == 4, bad
    for bad in (dict(q=24), dict(o=8), dict(k_pages=18), dict(q_stride=(512, 130, 128)), dict(tree_mask=20),
                dict(v_page_stride=(-4096, 2048, 128))):
        assert code(**bad) == 5, bad
    assert code(ws=None) == 8 and code(ws=264) == 8
    need = lib.coalibi_paged_attention_workspace_bytes(2, 4, 2, 1, 128)
    assert need > 0 and lib.coalibi_paged_attention_workspace_bytes(2, 4, 2, 65, 128) == 0
    assert lib.coalibi_paged_attention_workspace_bytes(2, 4, 3, 1, 128) == 0
    d = dict(base)
    for f in ("q_stride", "o_stride", "k_page_stride", "v_page_stride"):
        d[f] = (ctypes.c_longlong * 3)(*d[f])
    assert lib.coalibi_paged_attention(ctypes.byref(_lib.CoalibiPagedAttentionArgs(**d)), 256, need - 1, None) == 8


def test_refuses_cpu_tensors():
    from co_alibi_attn import paged_tree_attention
    x = torch.zeros(1, 2, 1, 64, dtype=f16)
    with pytest.raises(AssertionError):
        paged_tree_attention(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals():
    from co_alibi_attn import paged_tree_attention
    z = lambda *s, dt=f16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    good = dict(q=z(2, 4, 1, 64), k_pages=z(3, 2, 16, 64), v_pages=z(3, 2, 16, 64),
                page_table=z(2, 1, dt=torch.int32), ctx_lens=z(2, dt=torch.int32))
    assert paged_tree_attention(**good).shape == (2, 4, 1, 64)
    for kind, kw in (
            (TypeError, dict(q=z(2, 4, 1, 64, dt=torch.float32))), (TypeError, dict(k_pages=z(3, 2, 16, 64, dt=bf16))),
            (ValueError, dict(q=z(2, 4, 1, 96))), (ValueError, dict(q=z(2, 4, 65, 64))), (ValueError, dict(q=z(4, 1, 64))),
            (ValueError, dict(q=z(2, 3, 1, 64))), (ValueError, dict(v_pages=z(4, 2, 16, 64))),
            (ValueError, dict(k_pages=z(3, 2, 24, 64), v_pages=z(3, 2, 24, 64))),
            (ValueError, dict(k_pages=z(3, 2, 64, 16).transpose(2, 3))),
            (TypeError, dict(page_table=z(2, 1, dt=torch.int64))), (ValueError, dict(page_table=z(3, 1, dt=torch.int32))),
            (TypeError, dict(ctx_lens=z(2, dt=torch.int64))), (ValueError, dict(ctx_lens=z(3, dt=torch.int32))),
            (ValueError, dict(ctx_lens=z(2, dt=torch.int32).cpu())),
            (TypeError, dict(tree_mask=z(2, 1, dt=torch.int32))), (ValueError, dict(tree_mask=z(2, 2, dt=torch.int64))),
            (ValueError, dict(slopes=z(3))), (TypeError, dict(slopes=z(4, dt=torch.float64)))):
        with pytest.raises(kind):
            paged_tree_attention(**{**good, **kw})
