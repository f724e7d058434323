"""Broadcast, shared and oddly laid out inputs of the 8-bit cache and of the heads."""
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_heads import _pairs
from tests.test_quant_append import _same, _tables
from tests.test_quant_attention import _check
from tests.test_serving_attention import _q, _slopes

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


def _int(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 80, 112])
def test_append_and_read_of_shared_heads_and_odd_strides(page):
    """One key and value for all heads (expanded), queries off 16 bytes, a pool inside a larger one, tables as views,
    positions and counts with steps."""
    import co_alibi_attn
    Hkv, D, S, dt, start, count = 4, 64, 21, bf16, [7, 0, 33], [21, 0, 16]
    B = len(start)
    g = torch.Generator().manual_seed(50)
    kc, vc, ks, vs, table = qr.pool([60] * B, Hkv, D, page, 51)
    one = [torch.randn(B, 1, S, D, generator=g).to(dt) for _ in range(2)]
    cos, sin = _tables(90, 32)
    pos = torch.randint(0, 90, (B, S), generator=g, dtype=torch.int32)
    k = one[0].expand(B, Hkv, S, D)
    want = [x.clone() for x in (kc, vc, ks, vs)]
    qr.append(qr.rotated32(k, cos[pos.long()][:, None], sin[pos.long()][:, None], False), want[0], want[2], table, start, count)
    qr.append(one[1].expand(B, Hkv, S, D), want[1], want[3], table, start, count)
    big = torch.zeros(2, kc.shape[0] + 1, Hkv + 2, page, D + 16, dtype=torch.uint8, device="cuda")
    pools = [qr.e4m3(big)[i, 1:, 1:-1, :, 16:] for i in range(2)]
    for p, c in zip(pools, (kc, vc)):
        p.view(torch.uint8).copy_(c)
    q = torch.randn(B * 3 * S * D + 1, generator=g).to(dt).cuda()[1:].view(B, 3, S, D)
    wide = torch.full((B, 2 * table.shape[1] + 3), -9, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + table.shape[1]] = table.cuda()
    view = wide[:, 1:1 + table.shape[1]]
    ksd, vsd = ks.cuda(), vs.cuda()
    got = co_alibi_attn.append_paged_kv(one[0].cuda().expand(B, Hkv, S, D), one[1].cuda().expand(B, Hkv, S, D), *pools, view, _int(start).cuda(),
                                        count=torch.stack((_int(count), _int(count)), 1).cuda()[:, 0], q=q, rotary=(cos.cuda(), sin.cuda()),
                                        positions=pos.t().contiguous().cuda().t(), scales=(ksd, vsd))
    assert co_alibi_attn.device_status(reset=True) == 0
    assert _same(pools[0].view(torch.uint8), want[0]) and _same(pools[1].view(torch.uint8), want[1])
    assert torch.equal(ksd.cpu(), want[2]) and torch.equal(vsd.cpu(), want[3])
    assert (big[:, 0] == 0).all() and (big[:, :, 0] == 0).all() and (big[:, :, -1] == 0).all() and (big[..., :16] == 0).all()
    y = ref.rotated(q.cpu().double(), cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None], False)
    y = y * (torch.arange(S) < _int(count)[:, None])[:, None, :, None]
    bound = ref.U[dt] * y.abs() + 2.0 ** -22 * q.cpu().double().abs().amax(-1, keepdim=True) + 2.0 ** -24
    assert ((got.cpu().double() - y).abs() <= bound).all()
    at = torch.randint(-3, 60, (12, B), generator=g, dtype=torch.int32)
    back = co_alibi_attn.read_paged_kv(*pools, view, at.cuda().t(), (ksd, vsd))
    for a, c, s in zip(back, want[:2], want[2:]):
        d = qr.dequantised(c, s)
        for b in range(B):
            rows = ref.gather(d, table, b, 60)[:, at[:, b].clamp(min=0).long()] * (at[:, b] >= 0)[:, None]
            assert torch.equal(a[b].cpu(), rows.to(bf16))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,Sq", [(1, 1, 64, 1), (1, 1, 128, 64), (6, 2, 128, 64), (8, 1, 64, 3)])
def test_attention_of_one_mask_and_shared_queries(Hq, Hkv, D, Sq):
    """The same queries for all requests (expanded), one mask for all, the largest tree."""
    import co_alibi_attn
    dt, ctx = f16, [5, 700, 0]
    kc, vc, ks, vs, table = qr.pool([c + Sq for c in ctx], Hkv, D, 48, 52)
    q, words = _q(1, Hq, Sq, D, dt, 53), ref.tree(Sq, 54)
    mask = torch.tensor(ref.as_int64(words), dtype=torch.int64).cuda()
    o = co_alibi_attn.paged_tree_attention(q.cuda().expand(3, Hq, Sq, D), qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda(), _int(ctx).cuda(),
                                           tree_mask=mask, scales=(ks.cuda(), vs.cuda()))
    assert co_alibi_attn.device_status(reset=True) == 0 and o.shape == (3, Hq, Sq, D)
    _check(o, *qr.attention(q.expand(3, Hq, Sq, D), kc, vc, ks, vs, table, ctx, [words] * 3, _slopes(Hq)(dt), 1 / math.sqrt(D)))


@pytest.mark.gpu
@pytest.mark.parametrize("rot,interleaved", [(16, True), (48, False)])
def test_gradients_of_broadcast_projections_and_shared_weights(rot, interleaved):
    """One row for a batch and a sequence, a weight for queries and keys both, and gradients that are views: autograd adds
    up what the operator gives each.  Rounded gradients of the operator, added in float32 by autograd."""
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 3, 7, 5, 2, 64, f16
    g = torch.Generator().manual_seed(55)
    x = torch.randn(1, 1, Hq + 2 * Hkv, D, generator=g).to(dt)
    w = 1 + 0.3 * torch.randn(D, generator=g)
    grads = [torch.randn(B, S, H, D, generator=g).to(dt) for H in (Hq, Hkv, Hkv)]
    cos, sin = _tables(20, rot)
    xd, wd = x.float().cuda().requires_grad_(), w.cuda().requires_grad_()
    out = co_alibi_attn.norm_rotate_qkv(xd.expand(B, S, -1, -1).to(dt), Hq, Hkv, wd, wd, rotary=(cos.cuda(), sin.cuda()), interleaved=interleaved)
    got = torch.autograd.grad(out, (xd, wd), [t.cuda().transpose(1, 2) for t in grads])
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    each = x64.expand(B, S, -1, -1)
    want = qr.heads(each, Hq, Hkv, w64, w64, 1e-6, cos, sin, torch.arange(S).expand(B, S), interleaved)
    rows, gw = torch.autograd.grad(want, (each, w64), [t.double().transpose(1, 2) for t in grads])
    # each row's gradient is off by u and a float32 share of it (tests/test_heads.py); at most 21 are added
    assert ((got[0].cpu().double() - rows.sum((0, 1), keepdim=True)).abs() <= (ref.U[dt] + 2.0 ** -18) * rows.abs().sum((0, 1), keepdim=True) + 2.0 ** -14).all()
    n = x.double()[:, :, :Hq + Hkv] / (x.double()[:, :, :Hq + Hkv].square().mean(-1, keepdim=True) + 1e-6).sqrt()
    size = (_pairs(torch.cat(grads[:2], 2).double(), rot, interleaved) * n.abs()).sum((0, 1, 2))
    assert ((got[1].cpu().double() - gw).abs() <= 2.0 ** -18 * size + 2.0 ** -23 * size).all()  # (two sums, and their own)
