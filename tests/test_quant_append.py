"""Appending to a paged cache in 8 bits and reading it back, against the definition in 64 bits:
codes and scales are equal bit for bit (a block's scale is exact, a code is one rounding of the
value; rotated keys go through float32, products and their sum rounded one by one, which the
definition follows)."""
import ctypes
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref

f16, bf16 = torch.float16, torch.bfloat16


def _tables(n, R):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float(), a.sin().float()


def _int(x):
    return torch.tensor(x, dtype=torch.int32)


def _new(B, Hq, Hkv, S, D, dt, seed, spread=3.0):
    """A fused projection's heads; tokens differ in size by 2^+-spread."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g) * 2.0 ** (spread * (2 * torch.rand(B, S, 1, 1, generator=g) - 1))
    x = x.to(dt).transpose(1, 2)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


def _same(got, want):
    """Codes are equal, zeros of either sign and NaNs of any code alike."""
    a, b = qr.values_of(got.cpu()), qr.values_of(want)
    return torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9))


CASES = [
    # Hkv, D, S, start, count, page, dtype, rot, interleaved, token-major pool
    (12, 64, 1, [0], None, 16, f16, 0, False, False),
    (2, 128, 1, [0, 1, 15, 16, 17, 31, 63, 64], None, 32, bf16, 0, False, False),
    (2, 64, 1, [5, 900, 47, 48], None, 48, bf16, 64, False, True),
    (1, 128, 2, [15, 31, 14], None, 16, f16, 128, True, False),
    (3, 64, 5, [12, 0, 13, 100], [5, 0, 3, 1], 16, f16, 16, True, False),
    (2, 128, 17, [0, 15, 16, 9], None, 64, bf16, 48, False, False),
    (2, 128, 70, [3, 0, 33], [70, 1, 64], 32, f16, 64, True, True),
    (4, 64, 300, [1, 17], [300, 299], 128, bf16, 32, False, False),
    (8, 128, 40, [0, 0, 0], [40, 16, 17], 16, f16, 128, False, False),
]


def _device(codes, token_major):
    if token_major:  # keep the strides on the device
        return qr.e4m3(codes.transpose(1, 2).contiguous().cuda()).transpose(1, 2)
    return qr.e4m3(codes.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"H{c[0]}D{c[1]}S{c[2]}p{c[5]}r{c[7]}" for c in CASES])
def test_append_matches_definition(case):
    import co_alibi_attn
    Hkv, D, S, start, count, page, dt, rot, interleaved, token_major = case
    B, Hq = len(start), 2 * Hkv
    n = [S] * B if count is None else count
    kc, vc, ks, vs, table = qr.pool([a + b for a, b in zip(start, n)], Hkv, D, page, 1, spread=3.0)
    q, k, v = _new(B, Hq, Hkv, S, D, dt, 2)
    cos = sin = None
    k_in = k.double()
    if rot:
        cos, sin = _tables(max(start) + S, rot)
        at = _int(start)[:, None].long() + torch.arange(S)
        k_in = qr.rotated32(k, cos[at][:, None], sin[at][:, None], interleaved)
    want = [x.clone() for x in (kc, vc, ks, vs)]
    qr.append(k_in, want[0], want[2], table, start, n)
    qr.append(v, want[1], want[3], table, start, n)
    kd, vd, ksd, vsd = _device(kc, token_major), _device(vc, token_major), ks.cuda(), vs.cuda()
    q_out = co_alibi_attn.append_paged_kv(
        k.cuda(), v.cuda(), kd, vd, table.cuda(), _int(start).cuda(), count=None if count is None else _int(count).cuda(),
        q=q.cuda() if rot else None, rotary=(cos.cuda(), sin.cuda()) if rot else None, interleaved=interleaved, scales=(ksd, vsd))
    assert co_alibi_attn.device_status(reset=True) == 0
    assert torch.equal(ksd.cpu(), want[2]) and torch.equal(vsd.cpu(), want[3])
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[1])
    if rot:  # as the 16-bit append rotates them: one rounding of a float32 sum of two products
        y = ref.rotated(q.double(), cos.double()[at][:, None], sin.double()[at][:, None], interleaved)
        y = y * (torch.arange(S) < _int(n)[:, None])[:, None, :, None]
        bound = ref.U[dt] * y.abs() + 2.0 ** -22 * q.double().abs().amax(-1, keepdim=True) + 2.0 ** -24
        assert ((q_out.cpu().double() - y).abs() <= bound).all()
    else:
        assert q_out is None
    # the same call again writes the same
    before = [x.clone() for x in (kd.view(torch.uint8), vd.view(torch.uint8), ksd, vsd)]
    co_alibi_attn.append_paged_kv(
        k.cuda(), v.cuda(), kd, vd, table.cuda(), _int(start).cuda(), count=None if count is None else _int(count).cuda(),
        rotary=(cos.cuda(), sin.cuda()) if rot else None, interleaved=interleaved, scales=(ksd, vsd))
    assert all(torch.equal(a, b) for a, b in zip(before, (kd.view(torch.uint8), vd.view(torch.uint8), ksd, vsd)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [f16, bf16])
def test_extreme_values(dt):
    """Zeros, the type's smallest and largest, borders of the scale, infinities and NaN, each in blocks of its own."""
    import co_alibi_attn
    D, Hkv = 64, 1
    fi = torch.finfo(dt)
    sizes = [0.0, fi.smallest_normal * 2.0 ** -5, fi.smallest_normal, 448.0, 450.0, 447.0, 224.0, 225.0, 1.0, 3.5, 3.515625, fi.max,
             448 * 2.0 ** -100 if dt == bf16 else 1e-7, 450 * 2.0 ** -100 if dt == bf16 else 2e-7]
    S = BLOCKS = len(sizes) * 16
    g = torch.Generator().manual_seed(3)
    x = (2 * torch.rand(1, Hkv, S, D, generator=g) - 1) * torch.tensor(sizes).repeat_interleave(16)[None, None, :, None]
    x = x.to(dt)
    x[0, 0, ::16, 5] = torch.tensor(sizes).to(dt)  # the block's largest is that
    x[0, 0, 3 * 16 + 2, 7], x[0, 0, 5 * 16 + 1, 9], x[0, 0, 8 * 16 + 15, 0] = math.inf, -math.inf, math.nan
    pages = BLOCKS // 16
    codes = torch.randint(0, 255, (pages, Hkv, 16, D), dtype=torch.uint8, generator=g)
    scales = torch.full((pages, Hkv, 1), math.nan)
    table = torch.randperm(pages, generator=g, dtype=torch.int32)[None]
    want = codes.clone(), scales.clone()
    qr.append(x, *want, table, [0], [S])
    kd, vd, ks, vs = qr.e4m3(codes.cuda()), qr.e4m3(codes.cuda()), scales.cuda(), scales.cuda()
    co_alibi_attn.append_paged_kv(x.cuda(), x.cuda(), kd, vd, table.cuda(), _int([0]).cuda(), scales=(ks, vs))
    assert torch.equal(ks.cpu(), want[1]) and torch.equal(vs.cpu(), want[1])
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[0])
    for out in (f16, bf16):
        k, _ = co_alibi_attn.read_paged_kv(kd, vd, table.cuda(), torch.arange(S, dtype=torch.int32)[None].cuda(), (ks, vs), dtype=out)
        y = ref.gather(qr.dequantised(*want), table, 0, S)
        top = torch.finfo(out).max
        y = torch.where(y.isnan(), y, y.clamp(-top, top)).to(out)
        assert torch.equal(torch.nan_to_num(k[0].cpu(), nan=123.0), torch.nan_to_num(y, nan=123.0))


@pytest.mark.gpu
def test_growing_blocks_token_by_token():
    """Tokens of growing and shrinking size one at a time: old codes follow the scale, and one that
    comes back after reading gets the same code."""
    import co_alibi_attn
    D, Hkv, dt, n = 128, 2, bf16, 40
    g = torch.Generator().manual_seed(4)
    size = 2.0 ** torch.tensor([0, 1, -3, 4, 4, 2, 9, -8, 9, 12, 3, 0, 13, -2, 5, 14] * 3)[:n].float()
    x = [(torch.randn(1, Hkv, n, D, generator=g) * size[None, None, :, None]).to(dt) for _ in range(2)]
    codes = torch.zeros(4, Hkv, 16, D, dtype=torch.uint8)
    scales = torch.zeros(4, Hkv, 1)
    table = _int([[2, 0, 3, 1]])
    want = [codes.clone(), codes.clone(), scales.clone(), scales.clone()]
    kd, vd, ks, vs = qr.e4m3(codes.cuda()), qr.e4m3(codes.cuda()), scales.cuda(), scales.cuda()
    cache = (kd, vd, table.cuda())
    for t in range(n):
        for i in range(2):
            qr.append(x[i][:, :, t:t + 1], want[i], want[2 + i], table, [t], [1])
        co_alibi_attn.append_paged_kv(*(y[:, :, t:t + 1].cuda() for y in x), *cache, _int([t]).cuda(), scales=(ks, vs))
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[1])
    assert torch.equal(ks.cpu(), want[2]) and torch.equal(vs.cpu(), want[3])
    before = [t.clone() for t in (kd.view(torch.uint8), vd.view(torch.uint8), ks, vs)]
    k, v = co_alibi_attn.read_paged_kv(*cache, torch.arange(n, dtype=torch.int32)[None].cuda(), (ks, vs))
    co_alibi_attn.append_paged_kv(k[:, :, 5:], v[:, :, 5:], *cache, _int([5]).cuda(), scales=(ks, vs))
    after = [t for t in (kd.view(torch.uint8), vd.view(torch.uint8), ks, vs)]
    a, b = (co_alibi_attn.read_paged_kv(qr.e4m3(s[0]), qr.e4m3(s[1]), cache[2], torch.arange(n, dtype=torch.int32)[None].cuda(), tuple(s[2:])) for s in (before, after))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_what_is_not_stored_is_reported_and_touches_nothing():
    import co_alibi_attn
    D, Hkv, page, S = 64, 2, 16, 20
    kc, vc, ks, vs, table = qr.pool([64, 64, 64], Hkv, D, page, 5)
    table[0, 1], table[1, 2] = -1, 1 << 30
    start, count = [10, 30, 50], [20, 20, 20]  # the last one leaves the table
    q, k, v = _new(3, 4, Hkv, S, D, f16, 6)
    want = [x.clone() for x in (kc, vc, ks, vs)]
    qr.append(k, want[0], want[2], table, start, count)
    qr.append(v, want[1], want[3], table, start, count)
    kd, vd, ksd, vsd = qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), ks.cuda(), vs.cuda()
    co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), _int(start).cuda(), scales=(ksd, vsd))
    assert co_alibi_attn.device_status(reset=True) == 11
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[1])
    assert torch.equal(ksd.cpu(), want[2]) and torch.equal(vsd.cpu(), want[3])
    for bad in ([-1, -5, -(1 << 31)], [(1 << 31) - 1] * 3):
        co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), _int(bad).cuda(), scales=(ksd, vsd))
        assert co_alibi_attn.device_status(reset=True) == 11
    for none in ([0] * 3, [-7] * 3):
        co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), _int(start).cuda(), count=_int(none).cuda(), scales=(ksd, vsd))
        assert co_alibi_attn.device_status(reset=True) == 0
    assert _same(kd.view(torch.uint8), want[0]) and torch.equal(ksd.cpu(), want[2])
    # a position without angles: stored unrotated, and reported
    cos, sin = _tables(12, 32)
    kd, vd, ksd, vsd = qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), ks.cuda(), vs.cuda()
    co_alibi_attn.append_paged_kv(k[:1, :, :4].cuda(), v[:1, :, :4].cuda(), kd, vd, table[2:].cuda(), _int([10]).cuda(),
                                  rotary=(cos.cuda(), sin.cuda()), scales=(ksd, vsd))
    assert co_alibi_attn.device_status(reset=True) == 11
    turned = k[:1, :, :4].double()
    turned[:, :, :2] = qr.rotated32(k[:1, :, :2], cos[10:12], sin[10:12], False)
    want = kc.clone(), ks.clone()
    qr.append(turned, *want, table[2:], [10], [4])
    assert _same(kd.view(torch.uint8), want[0]) and torch.equal(ksd.cpu(), want[1])


@pytest.mark.gpu
def test_positions_apart_from_slots():
    import co_alibi_attn
    D, Hkv, S = 128, 2, 6
    kc, vc, ks, vs, table = qr.pool([40, 40], Hkv, D, 32, 7)
    q, k, v = _new(2, 4, Hkv, S, D, bf16, 8)
    cos, sin = _tables(64, 64)
    pos = torch.randint(0, 64, (2, S), generator=torch.Generator().manual_seed(9), dtype=torch.int32)
    want = kc.clone(), ks.clone()
    qr.append(qr.rotated32(k, cos[pos.long()][:, None], sin[pos.long()][:, None], False), *want, table, [13, 30], [S, S])
    kd, ksd = qr.e4m3(kc.cuda()), ks.cuda()
    co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, qr.e4m3(vc.cuda()), table.cuda(), _int([13, 30]).cuda(), q=q.cuda(),
                                  rotary=(cos.cuda(), sin.cuda()), positions=pos.cuda(), scales=(ksd, vs.cuda()))
    assert _same(kd.view(torch.uint8), want[0]) and torch.equal(ksd.cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("D,page,dt,token_major", [(64, 16, f16, False), (128, 48, bf16, True), (128, 64, f16, False)])
def test_read_matches_definition(D, page, dt, token_major):
    import co_alibi_attn
    Hkv, B = 3, 3
    kc, vc, ks, vs, table = qr.pool([100, 7, 250], Hkv, D, page, 10, spread=20.0 if dt == bf16 else 6.0)
    pos = torch.randint(-20, 100, (B, 37), generator=torch.Generator().manual_seed(11), dtype=torch.int32)
    pos[1] %= 7
    pos[2, 5] = 249
    want = []
    for c, s in ((kc, ks), (vc, vs)):
        d = qr.dequantised(c, s)
        y = torch.stack([ref.gather(d, table.clamp(min=0), b, table.shape[1] * page)[:, pos[b].clamp(min=0).long()] for b in range(B)])
        want.append(torch.where((pos >= 0)[:, None, :, None], y, 0.0).to(dt))
    # scales in a wider tensor, positions as a view
    wide = torch.full((2, ks.shape[0], Hkv + 1, ks.shape[2]), math.nan, device="cuda")
    wide[0, :, 1:], wide[1, :, 1:] = ks.cuda(), vs.cuda()
    args = (_device(kc, token_major), _device(vc, token_major), table.cuda())
    got = co_alibi_attn.read_paged_kv(*args, pos.cuda(), (wide[0, :, 1:], wide[1, :, 1:]), dtype=dt)
    assert co_alibi_attn.device_status(reset=True) == 0
    for a, b in zip(got, want):
        assert a.is_contiguous() and torch.equal(a.cpu(), b)
    # without a page: zero rows, reported
    pos[0, 0], pos[0, 1] = 1 << 30, table.shape[1] * page
    got = co_alibi_attn.read_paged_kv(*args, pos.cuda(), (ks.cuda(), vs.cuda()), dtype=dt)
    assert co_alibi_attn.device_status(reset=True) == 11
    assert (got[0][0, :, :2] == 0).all() and torch.equal(got[1][0, :, 2:].cpu(), want[1][0, :, 2:])
    empty = co_alibi_attn.read_paged_kv(*args, pos[:, :0].cuda(), (ks.cuda(), vs.cuda()), dtype=dt)
    assert empty[0].shape == (B, Hkv, 0, D)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    import co_alibi_attn
    dt, D, Hkv, page = bf16, 128, 4, 64
    n = (1 << 32) // (Hkv * page * D) + 4
    kp, vp = (torch.empty(n, Hkv, page, D, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(n, Hkv, page // 16, device="cuda") for _ in range(2))
    k, v = (torch.randn(1, Hkv, 20, D, device="cuda").to(dt) for _ in range(2))
    table = torch.tensor([[n - 1, n - 2]], dtype=torch.int32, device="cuda")
    co_alibi_attn.append_paged_kv(k, v, kp, vp, table, _int([48]).cuda(), scales=(ks, vs))
    got = co_alibi_attn.read_paged_kv(kp, vp, table, torch.arange(48, 68, dtype=torch.int32)[None].cuda(), (ks, vs))
    for a, b in zip(got, (k, v)):
        assert ((a.float() - b.float()).abs() <= 2.0 ** -4 * b.float().abs() + 2.0 ** -17 * b.float().abs().max()).all()
    o = co_alibi_attn.paged_tree_attention(k[:, :, 19:], kp, vp, table, _int([0]).cuda(), scales=(ks, vs))
    assert o.shape == (1, Hkv, 1, D)


@pytest.mark.gpu
def test_in_a_graph_and_on_another_stream():
    import co_alibi_attn
    D, Hkv = 64, 4
    kc, vc, ks, vs, table = qr.pool([50, 50], Hkv, D, 16, 12)
    _, k, v = _new(2, 4, Hkv, 1, D, bf16, 13)
    k, v, start = k.cuda(), v.cuda(), _int([20, 7]).cuda()

    def fresh():
        return qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda(), (ks.cuda(), vs.cuda())

    a, b = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in range(12):
            co_alibi_attn.append_paged_kv(k * (t + 1), v * (t + 1), *a[:3], start + t, scales=a[3])
    torch.cuda.current_stream().wait_stream(side)
    at, kk, vv = start.clone(), k.clone(), v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        co_alibi_attn.append_paged_kv(kk, vv, *b[:3], at, scales=b[3])
        out = co_alibi_attn.read_paged_kv(*b[:3], at[:, None], b[3])
    for t in range(12):
        kk.copy_(k * (t + 1)), vv.copy_(v * (t + 1)), at.copy_(start + t)
        graph.replay()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[:2], b[:2]))
    assert all(torch.equal(x, y) for x, y in zip(a[3], b[3]))
    assert torch.equal(out[0], co_alibi_attn.read_paged_kv(*a[:3], at[:, None], a[3])[0])


STRIDES = ("k_stride", "v_stride", "q_stride", "q_out_stride", "k_page_stride", "v_page_stride")


def _scales(_lib, **kw):
    d = dict(k=16, v=16, k_stride=(8, 1), v_stride=(8, 1))
    d.update(kw)
    for f in ("k_stride", "v_stride"):
        d[f] = (ctypes.c_longlong * 2)(*d[f])
    return _lib.CoalibiCacheScales(**d)


def test_refusals_of_the_append_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_paged_append8(None, None, None) == 1
    base = dict(k=16, v=16, q=None, q_out=None, k_pages=16, v_pages=16, page_table=16, start=16, count=None,
                positions=None, cos=None, sin=None, status=None, table_stride=4, B=2, Hq=0, Hkv=2, S=3, D=64,
                page_size=16, max_pages=4, n_pages=8, rot=0, n_pos=0, interleaved=0, dtype=1,
                **{s: (384, 192, 64) for s in STRIDES})

    def code(scales=None, **kw):
        d = {**base, **kw}
        for f in STRIDES:
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        return lib.coalibi_paged_append8(ctypes.byref(_lib.CoalibiPagedAppendArgs(**d)), ctypes.byref(_scales(_lib, **(scales or {}))), None)

    for field in ("k", "v", "k_pages", "v_pages", "page_table", "start"):
        assert code(**{field: None}) == 1
    for field in ("k", "v"):
        assert code(scales={field: None}) == 1 and code(scales={field: 18}) == 5
    assert code(q=16) == 1 and code(q_out=16) == 1
    assert code(D=80) == 2 and code(dtype=2) == 3 and code(dtype=3) == 3
    for bad in (dict(B=0), dict(S=0), dict(page_size=8), dict(rot=8), dict(rot=80), dict(rot=-16), dict(rot=16),
                dict(q=16, q_out=16, Hq=0), dict(n_pages=0), dict(B=1 << 15, S=1 << 17), dict(B=60000, S=30000, Hkv=60000),
                dict(scales=dict(k_stride=(0, 1))), dict(scales=dict(v_stride=(8, 0))), dict(scales=dict(v_stride=(-8, 1)))):
        assert code(**bad) == 4, bad
    assert code(rot=16, n_pos=4) == 1
    for bad in (dict(k=8), dict(k_pages=24), dict(k_stride=(384, 193, 64)), dict(k_page_stride=(384, 200, 64)),
                dict(v_page_stride=(384, 192, 72)), dict(rot=16, n_pos=4, cos=8, sin=16), dict(q=16, q_out=16, Hq=2, q_stride=(1, 8, 8))):
        assert code(**bad) == 5, bad


def test_refusals_of_the_read_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_paged_read8(None, None, None) == 1
    base = dict(k_pages=16, v_pages=16, page_table=16, positions=16, k=32, v=32, status=None, k_page_stride=(2048, 1024, 64),
                v_page_stride=(2048, 1024, 64), table_stride=4, B=2, Hkv=2, S=3, D=64, page_size=16, max_pages=4, n_pages=8, dtype=1)

    def code(scales=None, **kw):
        d = {**base, **kw}
        for f in ("k_page_stride", "v_page_stride"):
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        return lib.coalibi_paged_read8(ctypes.byref(_lib.CoalibiPagedReadArgs(**d)), ctypes.byref(_scales(_lib, **(scales or {}))), None)

    for field in ("k_pages", "v_pages", "page_table", "positions", "k", "v"):
        assert code(**{field: None}) == 1
    assert code(scales=dict(k=None)) == 1 and code(D=96) == 2 and code(dtype=2) == 3
    for bad in (dict(B=0), dict(S=0), dict(S=-4), dict(page_size=24), dict(max_pages=1 << 28), dict(B=65535, Hkv=65535, S=1 << 20),
                dict(scales=dict(k_stride=(0, 1)))):
        assert code(**bad) == 4, bad
    for bad in (dict(k=16), dict(v=18), dict(k_pages=8), dict(positions=18), dict(v_page_stride=(2048, 1032, 64))):
        assert code(**bad) == 5, bad


def test_refuses_cpu_tensors():
    from co_alibi_attn import read_paged_kv
    x = torch.zeros(1, 2, 16, 64, dtype=torch.float8_e4m3fn)
    with pytest.raises(AssertionError):
        read_paged_kv(x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), (x, x))


@pytest.mark.gpu
def test_refusals():
    from co_alibi_attn import append_paged_kv, paged_tree_attention, read_paged_kv
    z = lambda *s, dt=f16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    e = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    f = lambda *s: z(*s, dt=torch.float32)  # noqa: E731
    cache = dict(k_pages=e(3, 2, 32, 64), v_pages=e(3, 2, 32, 64), page_table=z(2, 1, dt=torch.int32), scales=(f(3, 2, 2), f(3, 2, 2)))
    calls = ((append_paged_kv, dict(k=z(2, 2, 3, 64), v=z(2, 2, 3, 64), start=z(2, dt=torch.int32))),
             (paged_tree_attention, dict(q=z(2, 4, 1, 64), ctx_lens=z(2, dt=torch.int32))),
             (read_paged_kv, dict(positions=z(2, 3, dt=torch.int32))))
    bad = [
        (TypeError, dict(scales=None)), (TypeError, dict(scales=(f(3, 2, 2),))), (TypeError, dict(scales=[f(3, 2, 2), f(3, 2, 2)])),
        (TypeError, dict(scales=(f(3, 2, 2), z(3, 2, 2)))), (ValueError, dict(scales=(f(3, 2, 1), f(3, 2, 2)))),
        (ValueError, dict(scales=(f(3, 2, 4)[..., ::2], f(3, 2, 2)))), (ValueError, dict(scales=(f(3, 1, 2).expand(3, 2, 2), f(3, 2, 2)))),
        (ValueError, dict(scales=(f(3, 2, 2), torch.zeros(3, 2, 2)))),
        (TypeError, dict(k_pages=z(3, 2, 32, 64), v_pages=z(3, 2, 32, 64))), (TypeError, dict(v_pages=z(3, 2, 32, 64))),
        (TypeError, dict(k_pages=e(3, 2, 32, 64).view(torch.uint8), v_pages=e(3, 2, 32, 64).view(torch.uint8))),
        (ValueError, dict(v_pages=e(3, 2, 16, 64))), (ValueError, dict(k_pages=e(3, 2, 32, 72)[..., :64], v_pages=e(3, 2, 32, 72)[..., :64])),
        (ValueError, dict(page_table=z(3, 1, dt=torch.int32))),
        (RuntimeError, dict(scales=(f(3, 2, 2).requires_grad_(), f(3, 2, 2)))),
    ]
    for call, own in calls:
        call(**cache, **own)
        for kind, kw in bad:
            with pytest.raises(kind):
                call(**{**cache, **own, **kw})
    with pytest.raises(TypeError):
        read_paged_kv(**cache, positions=z(2, 3, dt=torch.int32), dtype=torch.float32)
    for pos in (z(2, dt=torch.int32), z(3, 1, dt=torch.int32)):
        with pytest.raises(ValueError):
            read_paged_kv(**cache, positions=pos)
    with pytest.raises(TypeError):
        read_paged_kv(**cache, positions=z(2, 3, dt=torch.int64))
    # an append counts as a write of pools and scales
    versions = [t._version for t in (cache["k_pages"], cache["v_pages"], *cache["scales"])]
    append_paged_kv(**cache, **calls[0][1])
    assert all(t._version > v for t, v in zip((cache["k_pages"], cache["v_pages"], *cache["scales"]), versions))


@pytest.mark.gpu
@pytest.mark.parametrize("B,S", [(1, 1), (3, 801), (3, 1975)])  # a token to a CTA, two, and queries in a launch of their own
@pytest.mark.parametrize("rot,interleaved", [(0, False), (32, True), (64, False)])
def test_queries_are_those_of_the_16_bit_append(B, S, rot, interleaved):
    import co_alibi_attn
    D, Hkv, Hq, page, dt = 64, 1, 3, 16, bf16
    q, k, v = (t.cuda() for t in _new(B, Hq, Hkv, S, D, dt, 41))
    width = -(-S // page)
    table = torch.arange(B * width, dtype=torch.int32, device="cuda").view(B, width)
    start, count = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.tensor([S, S // 2, 0][:B], dtype=torch.int32, device="cuda")
    rotary = tuple(t.cuda() for t in _tables(S, rot)) if rot else None
    pool = torch.zeros(B * width, Hkv, page, D, dtype=dt, device="cuda")
    codes = [qr.e4m3(torch.zeros(pool.shape, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    scales = tuple(torch.ones(B * width, Hkv, 1, device="cuda") for _ in range(2))
    for more in (dict(rotary=rotary, interleaved=interleaved), dict()):
        want = co_alibi_attn.append_paged_kv(k, v, pool, pool.clone(), table, start, count=count, q=q if more.get("rotary") else None, **more)
        got = co_alibi_attn.append_paged_kv(k, v, *codes, table, start, count=count, q=q if more.get("rotary") else None, scales=scales, **more)
        assert (want is None and got is None) or torch.equal(want, got)
    assert co_alibi_attn.device_status(reset=True) == 0
