"""Normed and rotated heads of a fused projection, forward and backward, against the definition in
64 bits.

Tolerances, with u half an ulp of the type.  Forward: u |y| for the output's rounding; the sum of D
squares, 1 / sqrt and the products are float32: each square and addition is off by 2^-24 of a sum of positive
terms over a chain of at most 8 + 4 additions, 1 / sqrt by 2^-22, four further products and sums by 2^-24
each, together below 2^-20 of the pair's |a| + |b|.  Backward: u |dx| and 2^-19 of r (|w d| + |n| mean |w d n|), d's own
pair |a| + |b| in place of |d|; the weights' gradients: u |dw| and 2^-18 of the sum of |d n| (chains of at most 32
additions here; 2^-24 each, and n and d as above)."""
import ctypes

import pytest
import torch
import torch.utils.checkpoint

from tests import _quant_ref as qr
from tests import _serving_ref as ref

f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


def _tables(n, R):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float(), a.sin().float()


CASES = [
    # B, S, Hq, Hkv, D, dtype, weights' dtype (None: no weights), rot, interleaved, where: "", "start" or "positions"
    (1, 1, 1, 1, 64, f16, f16, 0, False, ""),
    (2, 3, 12, 12, 64, bf16, bf16, 64, False, ""),
    (3, 1, 32, 8, 128, bf16, f32, 128, False, "start"),
    (2, 5, 6, 3, 128, f16, f32, 48, True, "positions"),
    (1, 37, 16, 16, 128, f16, f16, 64, True, ""),
    (2, 17, 8, 1, 64, bf16, None, 16, False, "start"),
    (5, 7, 5, 5, 64, f16, f16, 48, False, "positions"),
    (1, 200, 71, 1, 64, bf16, bf16, 32, True, ""),  # several passes of a CTA, the last one partial
    (1, 3, 100, 20, 128, f16, None, 0, False, ""),
    (4, 900, 3, 1, 128, bf16, f32, 128, False, ""),  # more tokens than CTAs
]


def _inputs(case, seed=0):
    B, S, Hq, Hkv, D, dt, wdt, rot, interleaved, where = case
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(B, S, Hq + 2 * Hkv, D, generator=g) * 2.0 ** (4 * torch.rand(B, S, 1, 1, generator=g) - 2)).to(dt)
    weights = [None if wdt is None else (1 + 0.3 * torch.randn(D, generator=g)).to(wdt) for _ in range(2)]
    grads = [torch.randn(B, H, S, D, generator=g).to(dt) for H in (Hq, Hkv, Hkv)]
    rotary = _tables(S + 50, rot) if rot else None
    kw, at = {}, torch.arange(S).expand(B, S)
    if where == "start":
        kw["start"] = torch.randint(0, 50, (B,), generator=g, dtype=torch.int32)
        at = at + kw["start"][:, None]
    elif where == "positions":
        kw["positions"] = torch.randint(0, S + 50, (B, S), generator=g, dtype=torch.int32)
        at = kw["positions"]
    return qkv, weights, grads, rotary, kw, at.long()


def _pairs(x, rot, interleaved):
    """|a| + |b| of each element's pair, |x| where nothing turns.  x [..., D]."""
    y = x.abs().clone()
    if rot:
        first = torch.arange(rot // 2) * (2 if interleaved else 1)
        second = first + (1 if interleaved else rot // 2)
        both = y[..., first] + y[..., second]
        y[..., first], y[..., second] = both, both
    return y


def _cuda(x):
    return x.cuda() if isinstance(x, torch.Tensor) else tuple(t.cuda() for t in x) if isinstance(x, tuple) else x


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"B{c[0]}S{c[1]}H{c[2]}-{c[3]}D{c[4]}r{c[7]}{c[9]}" for c in CASES])
def test_matches_definition(case):
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt, wdt, rot, interleaved, where = case
    qkv, weights, grads, rotary, kw, at = _inputs(case)
    eps, u = 1e-5, ref.U[dt]
    x = qkv.cuda().requires_grad_()
    w = [None if t is None else t.cuda().requires_grad_() for t in weights]
    out = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, eps=eps, rotary=_cuda(rotary), interleaved=interleaved,
                                        **{k: _cuda(v) for k, v in kw.items()})
    leaves = [x] + [t for t in w if t is not None]
    got = torch.autograd.grad(out, leaves, [t.cuda() for t in grads])
    assert co_alibi_attn.device_status(reset=True) == 0

    x64 = qkv.double().requires_grad_()
    w64 = [torch.ones(D, dtype=torch.float64) if t is None else t.double().requires_grad_() for t in weights]
    cos, sin = rotary or (None, None)
    want = qr.heads(x64, Hq, Hkv, *w64, eps, cos, sin, at, interleaved)
    leaves64 = [x64] + [t for t in w64 if t.requires_grad]
    want_g = torch.autograd.grad(want, leaves64, [t.double() for t in grads])
    for i, (a, b) in enumerate(zip(out, want)):
        assert a.is_contiguous() and a.dtype == dt and a.shape == b.shape
        b = b.detach()
        bound = u * b.abs() + 2.0 ** -20 * _pairs(b, rot, interleaved) + 2.0 ** -25 if i < 2 else 0 * b
        err = (a.detach().cpu().double() - b).abs()
        assert (err <= bound).all(), f"output {i}: worst excess {(err - bound).max().item():.3e}"
    # gradients
    assert got[0].is_contiguous()
    Hn = Hq + Hkv
    err = (got[0].cpu().double() - want_g[0]).abs()
    assert torch.equal(got[0][:, :, Hn:].cpu(), grads[2].transpose(1, 2))
    xs, d = qkv.double()[:, :, :Hn], torch.cat([t.double().transpose(1, 2) for t in grads[:2]], 2)
    r = (xs.square().mean(-1, keepdim=True) + eps).rsqrt()
    ww = torch.cat([w64[0].detach().expand(Hq, D), w64[1].detach().expand(Hkv, D)]).abs()
    d = _pairs(d, rot, interleaved)
    n = (xs * r).abs()
    size = r * (d * ww + n * (d * ww * n).mean(-1, keepdim=True))
    bound = u * want_g[0][:, :, :Hn].abs() + 2.0 ** -19 * size + 2.0 ** -25
    assert (err[:, :, :Hn] <= bound).all(), f"worst excess {(err[:, :, :Hn] - bound).max().item():.3e}"
    for g, want_w, rows in zip(got[1:], want_g[1:], (slice(0, Hq), slice(Hq, Hn))):
        assert g.dtype == wdt
        bound = (u if wdt != f32 else 0) * want_w.abs() + 2.0 ** -18 * (d * n)[:, :, rows].sum((0, 1, 2)) + 2.0 ** -25
        assert ((g.cpu().double() - want_w).abs() <= bound).all()
    # again: the same bits
    again = torch.autograd.grad(co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, eps=eps, rotary=_cuda(rotary), interleaved=interleaved,
                                                              **{k: _cuda(v) for k, v in kw.items()}), leaves, [t.cuda() for t in grads])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("case", [CASES[1], CASES[3], CASES[5]])
def test_the_definitions_gradient_agrees_with_differences(case):
    B, S, Hq, Hkv, D, dt, wdt, rot, interleaved, where = case
    qkv, weights, grads, rotary, kw, at = _inputs(case, 5)
    g = torch.Generator().manual_seed(6)
    leaves = [qkv.double().requires_grad_()] + [(torch.ones(D) if t is None else t).double().requires_grad_() for t in weights]

    def total(x, wq, wk):
        y = qr.heads(x, Hq, Hkv, wq, wk, 1e-5, *(rotary or (None, None)), at, interleaved)
        return sum((a * t.double()).sum() for a, t in zip(y, grads))

    got = torch.autograd.grad(total(*leaves), leaves)
    h = 1e-5
    for i in range(3):
        step = torch.randn(leaves[i].shape, dtype=torch.float64, generator=g)
        moved = [[t.detach() + s * h * step if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1)]
        slope = (total(*moved[0]) - total(*moved[1])) / (2 * h)
        assert abs(slope - (got[i] * step).sum()) <= 1e-6 * (got[i].norm() * step.norm())


@pytest.mark.gpu
def test_gradients_agree_with_differences_of_the_operator():
    """Along a direction of float32 weights, in which the output is linear: its two ends differ by the
    gradient times the step, up to the outputs' own rounding, u of each output times its gradient."""
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 2, 9, 4, 2, 64, f16
    qkv, _, grads, rotary, _, _ = _inputs((B, S, Hq, Hkv, D, dt, f32, 32, False, ""), 7)
    g = torch.Generator().manual_seed(8)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).cuda().requires_grad_() for _ in range(2)]
    steps = [torch.randn(D, generator=g).cuda() for _ in range(2)]
    grads = [t.cuda() for t in grads]
    f = lambda a, b: co_alibi_attn.norm_rotate_qkv(qkv.cuda(), Hq, Hkv, a, b, rotary=_cuda(rotary))  # noqa: E731
    got = torch.autograd.grad(f(*w), w, grads)
    ends = [f(*(t.detach() + s * d for t, d in zip(w, steps))) for s in (0.5, -0.5)]
    change = sum(((a.double() - b.double()) * t.double()).sum() for a, b, t in zip(*ends, grads))
    want = sum((a.double() * d.double()).sum() for a, d in zip(got, steps))
    # (values are moved: no rounding; an error of half the gradient would show beside the noise)
    noise = sum((ref.U[dt] * (a.double().abs() + b.double().abs()) * t.double().abs()).sum() for a, b, t in zip(*(e[:2] for e in ends), grads))
    assert (change - want).abs() <= noise and want.abs() > 2 * noise


@pytest.mark.gpu
def test_layouts_of_projections_and_gradients():
    """A projection with a bias row in front, heads apart, rows off 16 bytes; gradients transposed, expanded or missing."""
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 2, 6, 4, 2, 64, bf16
    qkv, weights, grads, rotary, _, _ = _inputs((B, S, Hq, Hkv, D, dt, bf16, 64, False, ""), 9)
    w = [t.cuda() for t in weights]
    f = lambda x: co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, rotary=_cuda(rotary))  # noqa: E731
    x = qkv.cuda()
    want = f(x)
    wide = torch.zeros(B, S + 3, 2 * (Hq + 2 * Hkv), D + 8, dtype=dt, device="cuda")
    wide[:, 2:-1, ::2, 8:] = x
    odd = torch.zeros(x.numel() + 1, dtype=dt, device="cuda")[1:].view(x.shape)
    odd.copy_(x)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    for y in (wide[:, 2:-1, ::2, 8:], odd, swapped):
        assert all(torch.equal(a, b) for a, b in zip(f(y), want))
    leaf = x.clone().requires_grad_()
    grads = [t.cuda() for t in grads]
    base = torch.autograd.grad(f(leaf), leaf, grads)[0]
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in grads]
    assert torch.equal(torch.autograd.grad(f(leaf), leaf, turned)[0], base)
    ones = torch.autograd.grad(f(leaf), leaf, [torch.ones_like(t) for t in grads])[0]
    assert torch.equal(torch.autograd.grad(sum(t.sum() for t in f(leaf)), leaf)[0], ones)
    only_k = torch.autograd.grad(f(leaf)[1], leaf, grads[1])[0]
    assert torch.equal(only_k[:, :, Hq:Hq + Hkv], base[:, :, Hq:Hq + Hkv]) and (only_k[:, :, :Hq] == 0).all() and (only_k[:, :, -Hkv:] == 0).all()
    # a weight alone
    wq = w[0].clone().requires_grad_()
    out = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, wq, None)
    assert out[0].requires_grad and torch.autograd.grad(out[0], wq, grads[0])[0].shape == (D,)
    with pytest.raises(RuntimeError):  # no second derivative
        first, = torch.autograd.grad(f(leaf)[0].sum(), leaf, create_graph=True)
        first.sum().backward()


@pytest.mark.gpu
def test_rows_of_zeros_and_of_nothing_finite():
    import co_alibi_attn
    qkv = torch.zeros(1, 3, 3, 64, dtype=f16)
    qkv[0, 1], qkv[0, 2, 0, 3], qkv[0, 2, 1, 5] = 60000.0, float("inf"), float("nan")
    x = qkv.cuda().requires_grad_()
    q, k, v = co_alibi_attn.norm_rotate_qkv(x, 1, 1)
    assert (q[0, 0, 0] == 0).all() and (q[0, 0, 1] == 1).all() and q[0, 0, 2].isnan().any() and k[0, 0, 2].isnan().all()
    assert torch.equal(v[0, 0].cpu(), qkv[0, :, 2])
    d, = torch.autograd.grad(q, x, torch.ones_like(q))
    assert (d[0, 0, 0] == 1000).all()  # 1 / sqrt(eps)
    assert (d[0, 1, 0].abs() <= 2.0 ** -24).all()


@pytest.mark.gpu
def test_positions_outside_the_tables_are_reported_and_unrotated():
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 2, 4, 3, 1, 64, f16
    qkv, _, grads, rotary, _, _ = _inputs((B, S, Hq, Hkv, D, dt, None, 64, False, ""), 11)
    at = torch.tensor([[0, -1, 53, 54], [1 << 30, 2, -(1 << 31), 3]], dtype=torch.int32)
    inside = torch.where((at >= 0) & (at < 54), at, -1).long()
    x = qkv.cuda().requires_grad_()
    out = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, rotary=_cuda(rotary), positions=at.cuda())
    assert co_alibi_attn.device_status(reset=True) == 11
    x64 = qkv.double().requires_grad_()
    one = torch.ones(D, dtype=torch.float64)
    want = qr.heads(x64, Hq, Hkv, one, one, 1e-6, *rotary, inside, False)
    for a, b in zip(out, want):
        assert ((a.detach().cpu().double() - b.detach()).abs() <= ref.U[dt] * b.detach().abs() + 2.0 ** -18).all()
    d, = torch.autograd.grad(out, x, [t.cuda() for t in grads])
    d64, = torch.autograd.grad(want, x64, [t.double() for t in grads])
    assert (d.cpu().double() - d64).norm() <= 2 * ref.U[dt] * d64.norm()
    far = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, rotary=_cuda(rotary), start=torch.tensor([(1 << 31) - 1, 0], dtype=torch.int32).cuda())
    assert co_alibi_attn.device_status(reset=True) == 11
    assert torch.equal(far[0][0], co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv)[0][0])


@pytest.mark.gpu
def test_empty_batches():
    import co_alibi_attn
    x = torch.zeros(0, 5, 6, 64, dtype=f16, device="cuda", requires_grad=True)
    w = torch.ones(64, dtype=f16, device="cuda", requires_grad=True)
    q, k, v = co_alibi_attn.norm_rotate_qkv(x, 2, 2, w, w)
    assert q.shape == (0, 2, 5, 64) and v.shape == (0, 2, 5, 64)
    (q.sum() + k.sum()).backward()
    assert x.grad.shape == x.shape and (w.grad == 0).all()
    assert co_alibi_attn.norm_rotate_qkv(x[:, :0], 2, 2)[0].shape == (0, 2, 0, 64)


@pytest.mark.gpu
def test_in_a_graph_and_on_another_stream():
    import co_alibi_attn
    case = (2, 33, 4, 2, 128, bf16, bf16, 64, False, "")
    sets = []
    for seed in (1, 2):
        qkv, weights, grads, rotary, _, _ = _inputs(case, seed)
        sets.append([qkv.cuda(), *(t.cuda() for t in weights), *(t.cuda() for t in grads)])
    rotary = _cuda(rotary)

    def step(qkv, wq, wk, *grads):
        leaves = [t.detach().requires_grad_() for t in (qkv, wq, wk)]
        out = co_alibi_attn.norm_rotate_qkv(leaves[0], 4, 2, *leaves[1:], rotary=rotary)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for s, expect in zip(sets[::-1], want[::-1]):
        for a, b in zip(static, s):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, expect))


def test_refusals_of_the_c_entries():
    from co_alibi_attn import _lib
    lib = _lib.load()
    assert lib.coalibi_heads_fwd(None, None) == 1 and lib.coalibi_heads_bwd(None, None, 0, None) == 1
    strides = ("qkv_stride", "q_stride", "k_stride", "v_stride")
    base = dict(qkv=16, q=16, k=16, v=16, q_weight=None, k_weight=None, cos=None, sin=None, start=None, positions=None, status=None,
                dqkv=16, dq_weight=None, dk_weight=None, B=2, S=3, Hq=2, Hkv=1, D=64, rot=0, n_pos=0, interleaved=0, dtype=1,
                weight_dtype=1, eps=1e-6, **{s: (512, 64, 64) for s in strides})

    def codes(ws=256, bytes_=1 << 40, **kw):
        d = {**base, **kw}
        for f in strides:
            d[f] = (ctypes.c_longlong * 3)(*d[f])
        a = _lib.CoalibiHeadsArgs(**d)
        return lib.coalibi_heads_fwd(ctypes.byref(a), None), lib.coalibi_heads_bwd(ctypes.byref(a), ws, bytes_, None)

    for field in ("qkv", "q", "k", "v"):
        assert codes(**{field: None}) == (1, 1)
    assert codes(dqkv=None)[1] == 1
    assert codes(D=96) == (2, 2) and codes(dtype=2) == (3, 3) and codes(weight_dtype=0) == (3, 3) and codes(weight_dtype=3) == (3, 3)
    for bad in (dict(B=0), dict(S=0), dict(Hq=0), dict(Hkv=-1), dict(Hq=1 << 16), dict(B=1 << 16, S=1 << 16), dict(rot=8), dict(rot=80),
                dict(rot=-16), dict(rot=16)):
        assert codes(**bad) == (4, 4), bad
    assert codes(rot=16, n_pos=4) == (1, 1)
    for bad in (dict(qkv=8), dict(v=18), dict(qkv_stride=(512, 60, 64)), dict(q_stride=(-512, 64, 64)), dict(rot=16, n_pos=4, cos=8, sin=16),
                dict(q_weight=2), dict(start=2)):
        assert codes(**bad) == (5, 5), bad
    assert codes(dqkv=8)[1] == 5 and codes(dk_weight=2)[1] == 5
    need = lib.coalibi_heads_bwd_workspace_bytes(2, 1, 64)
    assert need > 0 and lib.coalibi_heads_bwd_workspace_bytes(2, 1, 96) == 0 and lib.coalibi_heads_bwd_workspace_bytes(0, 1, 64) == 0
    assert codes(ws=None)[1] == 8 and codes(ws=264)[1] == 8 and codes(bytes_=need - 1)[1] == 8


def test_refuses_cpu_tensors():
    from co_alibi_attn import norm_rotate_qkv
    with pytest.raises(AssertionError):
        norm_rotate_qkv(torch.zeros(1, 1, 3, 64, dtype=f16), 1, 1)


@pytest.mark.gpu
def test_refusals():
    from co_alibi_attn import norm_rotate_qkv
    z = lambda *s, dt=f16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    good = dict(qkv=z(2, 3, 6, 64), num_heads=2, num_kv_heads=2)
    norm_rotate_qkv(**good)
    tab = lambda n, r, dt=f32: z(n, r, dt=dt)  # noqa: E731
    for kind, kw in (
            (TypeError, dict(qkv=z(2, 3, 6, 64, dt=f32))), (ValueError, dict(qkv=z(2, 3, 6, 80))), (ValueError, dict(qkv=z(2, 3, 5, 64))),
            (ValueError, dict(qkv=z(2, 3, 384))), (ValueError, dict(num_heads=0, num_kv_heads=3)), (ValueError, dict(num_heads=8, num_kv_heads=-1)),
            (TypeError, dict(q_weight=z(64, dt=bf16))), (ValueError, dict(k_weight=z(128))), (ValueError, dict(q_weight=z(2, 64))),
            (TypeError, dict(q_weight=z(64), k_weight=z(64, dt=f32))), (ValueError, dict(q_weight=torch.zeros(64, dtype=f16))),
            (ValueError, dict(eps=-1.0)), (ValueError, dict(eps=float("nan"))), (TypeError, dict(start=z(2, dt=torch.int64))),
            (ValueError, dict(start=z(3, dt=torch.int32))), (ValueError, dict(positions=z(2, 2, dt=torch.int32))),
            (TypeError, dict(rotary=tab(4, 8))), (ValueError, dict(rotary=(tab(4, 4), tab(4, 4)))), (ValueError, dict(rotary=(tab(4, 40), tab(4, 40)))),
            (ValueError, dict(rotary=(tab(4, 8), tab(5, 8)))), (TypeError, dict(rotary=(tab(4, 8, f16), tab(4, 8, f16)))),
            (RuntimeError, dict(rotary=(tab(4, 8).requires_grad_(), tab(4, 8)))),
            (RuntimeError, dict(rotary=(tab(4, 8), tab(4, 8).requires_grad_()), qkv=z(2, 3, 6, 64).requires_grad_()))):
        with pytest.raises(kind):
            norm_rotate_qkv(**{**good, **kw})


@pytest.mark.gpu
def test_no_eps():
    """Slots of a CTA without a token add nothing to the weights' gradient; tolerances as above."""
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 1, 3, 2, 1, 64, f16
    qkv, weights, grads, _, _, _ = _inputs((B, S, Hq, Hkv, D, dt, f32, 0, False, ""), 21)
    x, w = qkv.cuda().requires_grad_(), [t.cuda().requires_grad_() for t in weights]
    got = torch.autograd.grad(co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, *w, eps=0.0), [x, *w], [t.cuda() for t in grads])
    x64, w64 = qkv.double().requires_grad_(), [t.double().requires_grad_() for t in weights]
    want = torch.autograd.grad(qr.heads(x64, Hq, Hkv, *w64, 0.0, None, None, torch.arange(S).expand(B, S), False), [x64, *w64],
                               [t.double() for t in grads])
    n = qkv.double() * qkv.double().square().mean(-1, keepdim=True).rsqrt()
    for i, h in enumerate((slice(0, Hq), slice(Hq, Hq + Hkv))):
        size = (n[:, :, h] * grads[i].double().transpose(1, 2)).abs().sum((0, 1, 2))
        assert ((got[1 + i].cpu().double() - want[1 + i]).abs() <= 2.0 ** -18 * size + 2.0 ** -25).all()
    assert (got[0].cpu().double() - want[0]).norm() <= 2 * ref.U[dt] * want[0].norm()


@pytest.mark.gpu
def test_a_row_of_zeros_with_an_eps_whose_inverse_overflows():
    import co_alibi_attn
    x = torch.zeros(1, 2, 3, 64, dtype=bf16, device="cuda", requires_grad=True)
    q, _, _ = co_alibi_attn.norm_rotate_qkv(x, 1, 1, eps=1e-39)
    d, = torch.autograd.grad(q, x, torch.full_like(q, 2.0 ** -20))
    want = 2.0 ** -20 * float(torch.tensor(1e-39, dtype=torch.float32).double()) ** -0.5  # 1 / sqrt(eps): about 2^65
    assert ((d[:, :, 0].double() - want).abs() <= 2 * ref.U[bf16] * want).all() and (d[:, :, 1:] == 0).all()


@pytest.mark.gpu
def test_a_backward_that_cannot_run_raises():
    """In the engine's own thread: a saved input written to in between, a graph used twice, a second derivative."""
    import co_alibi_attn
    qkv, weights, grads, rotary, kw, _ = _inputs((2, 5, 3, 1, 64, f16, f16, 32, False, "start"), 31)
    x, w = qkv.cuda().requires_grad_(), [t.cuda().requires_grad_() for t in weights]
    kw, grads = {k: t.cuda() for k, t in kw.items()}, [t.cuda() for t in grads]
    f = lambda: co_alibi_attn.norm_rotate_qkv(x, 3, 1, *w, rotary=_cuda(rotary), **kw)  # noqa: E731
    out = f()
    want = torch.autograd.grad(out, [x, *w], grads)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, grads)
    out = f()
    kw["start"].add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, grads)
    kw["start"].sub_(1)
    out = f()
    assert co_alibi_attn.device_status(reset=True) == 0  # (resets the status word between the two)
    first = torch.autograd.grad(out, [x, *w], grads, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    with pytest.raises(RuntimeError, match="second derivative"):
        first[0].float().square().sum().backward()
    # under saved-tensor hooks, and again with the forward computed anew
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = f()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [x, *w], grads), want))
    out = torch.utils.checkpoint.checkpoint(lambda *a: co_alibi_attn.norm_rotate_qkv(a[0], 3, 1, *a[1:], rotary=_cuda(rotary), **kw), x, *w,
                                            use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [x, *w], grads), want))
