"""Normed and rotated heads of batches whose CTAs go over several groups of tokens, as those of training do: rows of the
next group on their way while the last one's are taken, angles that change between groups, groups across two sequences,
a last CTA with fewer.  The definition in 64 bits, on the GPU.

Tolerances as in tests/test_heads.py, but for the weights' gradients, whose chains are longer: of a lane at most 5 groups
of 3 heads, 3 + 8 additions of its warp and CTA, 56 of a column's rows and 5 more: 87 of 2^-24 each of the sum of |d n|,
below 2^-17.5 of it; with n and d's own (below 2^-19), 2^-17."""
import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_heads import _inputs, _pairs

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32

CASES = [
    # as in tests/test_heads.py, then groups that a CTA goes over in the forward and in the backward (148 SMs)
    ((7, 12345, 2, 1, 64, bf16, f32, 48, False, "start"), 1, 3),
    ((5, 4011, 3, 3, 128, f16, f16, 64, True, ""), 1, 2),
    ((3, 25323, 1, 1, 128, bf16, None, 128, False, "positions"), 2, 5),
    ((13, 5551, 1, 1, 64, f16, f32, 64, True, "positions"), 1, 2),
]


def _per_cta(case, waves):
    """(groups, groups of a CTA): heads in chunks of up to eight, fewer where CTAs would be fewer than SMs."""
    B, S, Hq, Hkv, D = case[:5]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    groups, most = -(-B * S // (4096 // D)), 8
    chunks = lambda n: -(-Hq // n) + 2 * -(-Hkv // n)  # noqa: E731
    while most > 1 and groups * chunks(most) < sms:
        most //= 2
    return groups, -(-groups // min(groups, max(1, waves * sms // chunks(most))))


@pytest.mark.gpu
@pytest.mark.parametrize("case,forward,backward", CASES, ids=[f"B{c[0]}S{c[1]}H{c[2]}-{c[3]}D{c[4]}r{c[7]}{c[9]}" for c, _, _ in CASES])
def test_ctas_of_several_groups(case, forward, backward):
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt, wdt, rot, interleaved, where = case
    assert _per_cta(case, 48)[1] == forward and _per_cta(case, 12)[1] == backward
    assert any(_per_cta(c, 12)[0] % b for c, _, b in CASES)  # (a last CTA with fewer)
    qkv, weights, grads, rotary, kw, at = _inputs(case, 3)
    qkv, grads, at = qkv.cuda(), [t.cuda() for t in grads], at.cuda()
    weights, rotary, kw = [None if t is None else t.cuda() for t in weights], tuple(t.cuda() for t in rotary), {k: t.cuda() for k, t in kw.items()}
    eps, u = 1e-5, ref.U[dt]
    x, w = qkv.requires_grad_(), [None if t is None else t.requires_grad_() for t in weights]
    out = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, eps=eps, rotary=rotary, interleaved=interleaved, **kw)
    leaves = [x] + [t for t in w if t is not None]
    got = torch.autograd.grad(out, leaves, grads)
    assert co_alibi_attn.device_status(reset=True) == 0
    x64 = qkv.detach().double().requires_grad_()
    w64 = [torch.ones(D, dtype=torch.float64, device="cuda") if t is None else t.detach().double().requires_grad_() for t in w]
    want = qr.heads(x64, Hq, Hkv, *w64, eps, *rotary, at, interleaved)
    want_g = torch.autograd.grad(want, [x64] + [t for t in w64 if t.requires_grad], [t.double() for t in grads])
    for i, (a, b) in enumerate(zip(out, want)):
        b = b.detach()
        bound = u * b.abs() + 2.0 ** -20 * _pairs(b, rot, interleaved) + 2.0 ** -25 if i < 2 else 0 * b
        assert ((a.detach().double() - b).abs() <= bound).all(), f"output {i}"
    Hn = Hq + Hkv
    assert torch.equal(got[0][:, :, Hn:], grads[2].transpose(1, 2))
    xs, d = qkv.detach().double()[:, :, :Hn], torch.cat([t.double().transpose(1, 2) for t in grads[:2]], 2)
    r = (xs.square().mean(-1, keepdim=True) + eps).rsqrt()
    ww = torch.cat([w64[0].detach().expand(Hq, D), w64[1].detach().expand(Hkv, D)]).abs()
    d, n = _pairs(d, rot, interleaved), (xs * r).abs()
    size = r * (d * ww + n * (d * ww * n).mean(-1, keepdim=True))
    bound = u * want_g[0][:, :, :Hn].abs() + 2.0 ** -19 * size + 2.0 ** -25
    assert ((got[0].double() - want_g[0])[:, :, :Hn].abs() <= bound).all()
    for a, b, rows in zip(got[1:], want_g[1:], (slice(0, Hq), slice(Hq, Hn))):
        bound = (u if wdt != f32 else 0) * b.abs() + 2.0 ** -17 * (d * n)[:, :, rows].sum((0, 1, 2)) + 2.0 ** -25
        assert ((a.double() - b).abs() <= bound).all()
    again = torch.autograd.grad(co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, eps=eps, rotary=rotary, interleaved=interleaved, **kw), leaves, grads)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
