"""Appending to a paged cache, with and without the rotation, against its definition in
64 bits.  Values that are only moved must be equal bit for bit; a rotated one is within
its one rounding, u |x|, plus 2^-22 (|a| + |b|) for float32 products and their sum."""
import ctypes

import pytest
import torch

from tests import _serving_ref as ref

f16, bf16 = torch.float16, torch.bfloat16
CASES = [
    # Hq (0: no queries), Hkv, D, S, starts, counts, page, dtype, rotary dim, interleaved, token-major
    (0, 12, 64, 1, [0, 5, 15, 16, 100], None, 16, bf16, 0, False, False),
    (8, 2, 128, 1, [0, 31, 32, 47], None, 48, f16, 128, False, False),
    (8, 2, 128, 1, [7, 0], None, 16, bf16, 128, True, True),
    (4, 4, 64, 37, [0, 3, 60], [37, 0, 5], 32, f16, 16, False, False),
    (6, 3, 128, 19, [11, 2], [19, 1], 16, bf16, 80, True, False),
    (0, 1, 128, 70, [1], None, 64, f16, 32, False, True),
    (8, 8, 64, 5, [0, 1], [9, -1], 16, f16, 64, False, False),  # counts are held to 0 .. S
    (0, 2, 64, 300, [0, 40], [300, 213], 16, bf16, 0, False, False),
]


def _angles(table, pos):
    return table.double()[pos]


@pytest.mark.gpu
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("case", CASES, ids=[f"H{c[0]}-{c[1]}D{c[2]}S{c[3]}r{c[8]}{'i' if c[9] else 'h'}" for c in CASES])
def test_matches_definition(case, explicit):
    import co_alibi_attn
    from co_alibi_attn.serving import rotary_tables
    Hq, Hkv, D, S, starts, counts, page, dt, rot, inter, token_major = case
    if explicit and not rot:
        pytest.skip("positions matter to the rotation alone")
    B, u = len(starts), ref.U[dt]
    k0, v0, table = ref.pool([s + S for s in starts], Hkv, D, page, dt, seed=31, token_major=token_major)
    dense = lambda x: x.transpose(1, 2).contiguous().cuda().transpose(1, 2) if token_major else x.cuda()  # noqa: E731
    kp, vp = dense(k0), dense(v0)
    g = torch.Generator().manual_seed(32)
    qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g).to(dt).transpose(1, 2)
    dev = qkv.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    pos = torch.randint(0, 512, (B, S), generator=g, dtype=torch.int32)
    tables = rotary_tables(rot, 512, scale=2.0) if rot else None
    int32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    q_out = co_alibi_attn.append_paged_kv(
        dev[:, Hq:Hq + Hkv], dev[:, Hq + Hkv:], kp, vp, table.cuda(), int32(starts), count=int32(counts),
        q=dev[:, :Hq] if Hq else None, rotary=tuple(t.cuda() for t in tables) if rot else None, interleaved=inter,
        positions=pos.cuda() if explicit else None)
    torch.cuda.synchronize()
    assert co_alibi_attn.device_status(reset=True) == 0
    want_k, want_v = k0.double(), v0.double()
    room_k = torch.zeros_like(want_k)  # what the rotation's rounding may be off by
    want_q, room_q = torch.zeros(B, Hq, S, D, dtype=torch.float64), torch.zeros(B, Hq, S, D, dtype=torch.float64)
    for b in range(B):
        n = S if counts is None else max(0, min(S, counts[b]))
        for i in range(n):
            t = starts[b] + i
            at = table[b, t // page].item(), slice(None), t % page
            kk, qq = k[b, :, i].double(), q[b, :, i].double()
            rk, rq = torch.zeros_like(kk), torch.zeros_like(qq)
            if rot:
                p = int(pos[b, i]) if explicit else t
                for x, r in ((kk, rk), (qq, rq)):
                    c, s = _angles(tables[0], p), _angles(tables[1], p)
                    y = ref.rotated(x, c, s, inter)
                    a = ref.rotated(x.abs(), c.abs(), -s.abs(), inter).abs() + x.abs()
                    r[:, :rot] = (u * y.abs() + 2.0 ** -22 * (2 * a + 1e-3))[:, :rot]
                    x.copy_(y)
            want_k[at], room_k[at], want_v[at] = kk, rk, v[b, :, i].double()
            want_q[b, :, i], room_q[b, :, i] = qq, rq
    assert torch.equal(vp.cpu().double(), want_v)
    assert ((kp.cpu().double() - want_k).abs() <= room_k).all()
    if Hq:
        assert ((q_out.cpu().double() - want_q).abs() <= room_q).all()
    else:
        assert q_out is None


@pytest.mark.gpu
def test_tokens_without_a_page_or_an_angle_are_reported():
    import co_alibi_attn
    from co_alibi_attn.serving import rotary_tables
    dt, D = f16, 64
    x = torch.ones(1, 2, 3, D, dtype=dt, device="cuda")
    for start, entry, n_pos, rot in ((30, 0, 64, 0), (-1, 0, 64, 0), (14, -1, 64, 0), (14, 5, 64, 0), (0, 0, 2, 16)):
        kp, vp = (torch.zeros(5, 2, 16, D, dtype=dt, device="cuda") for _ in range(2))
        table = torch.tensor([[4, entry]], dtype=torch.int32, device="cuda")
        co_alibi_attn.append_paged_kv(x, x, kp, vp, table, torch.tensor([start], dtype=torch.int32, device="cuda"),
                                      rotary=tuple(t.cuda() for t in rotary_tables(rot, n_pos)) if rot else None)
        assert co_alibi_attn.device_status(reset=True) == 11
        stored = sum(0 <= t < 32 and 0 <= [4, entry][t // 16] < 5 for t in range(start, start + 3)) if start >= 0 else 0
        assert int(vp.sum()) == stored * 2 * D
    co_alibi_attn.append_paged_kv(x[:, :, :0], x[:, :, :0], kp, vp, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert co_alibi_attn.device_status(reset=True) == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    import co_alibi_attn
    dt, D, Hkv, page = bf16, 128, 4, 64
    n = (1 << 32) // (Hkv * page * D) + 4
    kp, vp = (torch.empty(n, Hkv, page, D, dtype=dt, device="cuda") for _ in range(2))
    k, v = (torch.randn(1, Hkv, 2, D, device="cuda").to(dt) for _ in range(2))
    table = torch.tensor([[n - 1, n - 2]], dtype=torch.int32, device="cuda")
    co_alibi_attn.append_paged_kv(k, v, kp, vp, table, torch.tensor([63], dtype=torch.int32, device="cuda"))
    for pool, x in ((kp, k), (vp, v)):
        assert torch.equal(pool[n - 1, :, 63], x[0, :, 0]) and torch.equal(pool[n - 2, :, 0], x[0, :, 1])


def test_rotary_tables():
    from co_alibi_attn.serving import rotary_tables
    cos, sin = rotary_tables(16, 10, base=100.0, scale=2.0)
    assert cos.shape == sin.shape == (10, 8) and cos.dtype == torch.float32
    a = 7 / 2.0 * 100.0 ** (-2 * 3 / 16)
    import math
    assert abs(cos[7, 3].item() - math.cos(a)) < 1e-7 and abs(sin[7, 3].item() - math.sin(a)) < 1e-7
    for bad in ((0, 4), (7, 4), (16, 0)):
        with pytest.raises(ValueError):
            rotary_tables(*bad)


def test_refusals_of_the_c_entry():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_paged_append(None, None) == 1
    strides = ("k_stride", "v_stride", "q_stride", "q_out_stride", "k_page_stride", "v_page_stride")
    base = dict(k=16, v=16, q=None, q_out=None, k_pages=16, v_pages=16, page_table=16, start=16, count=None,
                positions=None, cos=None, sin=None, status=None, table_stride=4, B=2, Hq=0, Hkv=2, S=3, D=64,
                page_size=16, max_pages=4, n_pages=8, rot=0, n_pos=0, interleaved=0, dtype=1,
                **{s: (384, 192, 64) for s in strides})

    def code(**kw):
        d = {**base, **kw}
        for f in strides:
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        a = _lib.CoalibiPagedAppendArgs(**d)
        return lib.coalibi_paged_append(ctypes.byref(a), None)

    for field in ("k", "v", "k_pages", "v_pages", "page_table", "start"):
        assert code(**{field: None}) == 1
    assert code(q=16) == 1 and code(q_out=16) == 1
    assert code(D=80) == 2 and code(dtype=2) == 3
    for bad in (dict(B=0), dict(S=0), dict(page_size=8), dict(rot=8), dict(rot=80), dict(rot=-16), dict(rot=16),
                dict(q=16, q_out=16, Hq=0), dict(n_pages=0), dict(B=1 << 15, S=1 << 17)):
        assert code(**bad) == 4, bad
    assert code(rot=16, n_pos=4) == 1
    for bad in (dict(k=8), dict(k_pages=20), dict(k_stride=(384, 193, 64)), dict(rot=16, n_pos=4, cos=8, sin=16),
                dict(q=16, q_out=16, Hq=2, q_stride=(1, 8, 8))):
        assert code(**bad) == 5, bad


def test_refuses_cpu_tensors():
    from co_alibi_attn import append_paged_kv
    x = torch.zeros(1, 2, 16, 64, dtype=f16)
    with pytest.raises(AssertionError):
        append_paged_kv(x, x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals():
    from co_alibi_attn import append_paged_kv
    z = lambda *s, dt=f16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    good = dict(k=z(2, 2, 3, 64), v=z(2, 2, 3, 64), k_pages=z(3, 2, 16, 64), v_pages=z(3, 2, 16, 64),
                page_table=z(2, 1, dt=torch.int32), start=z(2, dt=torch.int32))
    tab = lambda n, r, dt=torch.float32: z(n, r, dt=dt)  # noqa: E731
    append_paged_kv(**good)
    for kind, kw in (
            (TypeError, dict(k=z(2, 2, 3, 64, dt=torch.float32))), (TypeError, dict(v=z(2, 2, 3, 64, dt=bf16))),
            (ValueError, dict(v=z(2, 2, 2, 64))), (ValueError, dict(k=z(2, 4, 3, 64), v=z(2, 4, 3, 64))),
            (ValueError, dict(q=z(2, 4, 2, 64))), (TypeError, dict(q=z(2, 4, 3, 64, dt=bf16))),
            (TypeError, dict(start=z(2, dt=torch.int64))), (ValueError, dict(count=z(3, dt=torch.int32))),
            (ValueError, dict(positions=z(2, 2, dt=torch.int32))), (ValueError, dict(rotary=(tab(4, 4), tab(4, 4)))),
            (ValueError, dict(rotary=(tab(4, 40), tab(4, 40)))), (ValueError, dict(rotary=(tab(4, 8), tab(5, 8)))),
            (TypeError, dict(rotary=(tab(4, 8, f16), tab(4, 8, f16)))),
            (ValueError, dict(page_table=z(2, 0, dt=torch.int32)))):
        with pytest.raises(kind):
            append_paged_kv(**{**good, **kw})
