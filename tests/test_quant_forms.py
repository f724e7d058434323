"""The 8-bit cache's append and read in the forms that their launches choose: many heads to a CTA, heads that do not
fill their warps, the longest batch."""
import pytest
import torch

from tests import _quant_ref as qr
from tests.test_quant_append import _new, _same, _tables

f16, bf16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
def test_as_many_tokens_as_an_int_counts():
    """All padding but one page's: an expanded row, so that nothing of the size is held."""
    import co_alibi_attn
    D, S = 64, (1 << 31) - 1
    row = torch.linspace(-2, 2, D, device="cuda").to(f16)
    x = row.expand(1, 1, S, D)
    codes = [qr.e4m3(torch.full((2, 1, 16, D), 0x7f, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    scales = tuple(torch.ones(2, 1, 1, device="cuda") for _ in range(2))
    table = torch.ones(1, 1, dtype=torch.int32, device="cuda")
    start, count = torch.full((1,), 3, dtype=torch.int32, device="cuda"), torch.full((1,), 13, dtype=torch.int32, device="cuda")
    co_alibi_attn.append_paged_kv(x, x, *codes, table, start, count=count, scales=scales)
    assert co_alibi_attn.device_status(reset=True) == 0
    want = qr.codes_of(row.cpu().double())
    for c in codes:
        got = c.view(torch.uint8).cpu()
        assert (qr.values_of(got[1, 0, 3:]) == qr.values_of(want)).all() and (got[0] == 0x7f).all() and (got[1, 0, :3] == 0x7f).all()


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D,chunks,per", [(5, 128, 300, 10), (8, 64, 300, 16), (3, 64, 150, 3), (5, 128, 100, 3), (8, 128, 100, 4)])
@pytest.mark.parametrize("dt", [f16, bf16])
def test_reads_of_many_heads_to_a_cta(Hkv, D, chunks, per, dt):
    """`per` of the keys' and values' heads to a CTA, in rounds of eight: rounds that are not full, and with keys and
    values in one.  B * chunks CTAs of 4096 / D tokens side by side."""
    import co_alibi_attn
    n, have = 2 * Hkv, 2 * Hkv
    while have > 1 and chunks * (n // have) < 2 * _sms():
        have = (have + 1) // 2
    assert have == per
    B, page = 2, 48
    S = chunks // B * (4096 // D) - 5
    kc, vc, ks, vs, table = qr.pool([700, 333], Hkv, D, page, 10, spread=6.0)
    g = torch.Generator().manual_seed(11)
    pos = torch.stack([torch.randint(-20, top, (S,), generator=g, dtype=torch.int32) for top in (700, 333)])
    want = []
    for c, s in ((kc, ks), (vc, vs)):
        d, at = qr.dequantised(c, s).to(dt), pos.clamp(min=0).long()
        y = torch.stack([d[table[b].long()[at[b] // page], :, at[b] % page].transpose(0, 1) for b in range(B)])
        want.append(torch.where((pos >= 0)[:, None, :, None], y, 0.0))
    got = co_alibi_attn.read_paged_kv(qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda(), pos.cuda(), (ks.cuda(), vs.cuda()), dtype=dt)
    assert co_alibi_attn.device_status(reset=True) == 0
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D,rot,interleaved", [(9, 64, 0, False), (9, 128, 64, True), (11, 64, 64, False), (17, 64, 32, False)])
def test_heads_that_do_not_fill_their_warps(Hkv, D, rot, interleaved):
    """More heads than warps of a CTA, some of whose warps have none."""
    import co_alibi_attn
    start, S, page, dt = [0, 13, 31], 20, 32, bf16
    kc, vc, ks, vs, table = qr.pool([s + S for s in start], Hkv, D, page, 12, spread=3.0)
    q, k, v = _new(3, 2 * Hkv, Hkv, S, D, dt, 13)
    k_in, rotary = k.double(), None
    if rot:
        cos, sin = _tables(60, rot)
        at = torch.tensor(start)[:, None] + torch.arange(S)
        k_in, rotary = qr.rotated32(k, cos[at][:, None], sin[at][:, None], interleaved), (cos.cuda(), sin.cuda())
    want = [x.clone() for x in (kc, vc, ks, vs)]
    qr.append(k_in, want[0], want[2], table, start, [S] * 3)
    qr.append(v, want[1], want[3], table, start, [S] * 3)
    kd, vd, ksd, vsd = qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), ks.cuda(), vs.cuda()
    co_alibi_attn.append_paged_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), torch.tensor(start, dtype=torch.int32).cuda(), q=q.cuda() if rot else None,
                                  rotary=rotary, interleaved=interleaved, scales=(ksd, vsd))
    assert co_alibi_attn.device_status(reset=True) == 0
    assert torch.equal(ksd.cpu(), want[2]) and torch.equal(vsd.cpu(), want[3])
    assert _same(kd.view(torch.uint8), want[0]) and _same(vd.view(torch.uint8), want[1])
