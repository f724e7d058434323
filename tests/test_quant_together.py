"""Calls of the 8-bit cache and of the heads side by side: on several streams at once, out of two graphs that share a pool
of memory, over more elements than 32 bits count, and drafts whose keys are NaN beside rows that do not see them."""
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests.test_quant_attention import FORMS, IDS, _case, _check, _run, _widen

f16, bf16 = torch.float16, torch.bfloat16


def _set(seed, Hq, Hkv, D, Sq, dt, lens):
    """A cache and what a step over it takes, and the step: heads with their gradient, append, attention, read."""
    import co_alibi_attn
    kc, vc, ks, vs, table = (x.cuda() for x in qr.pool([n + Sq for n in lens], Hkv, D, 32, seed))
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    qkv = torch.randn(B, Sq, Hq + 2 * Hkv, D, generator=g).to(dt).cuda()
    weight = (1 + 0.2 * torch.randn(D, generator=g)).to(dt).cuda()
    start = torch.tensor(lens, dtype=torch.int32).cuda()
    grads = [torch.randn(B, H, Sq, D, generator=g).to(dt).cuda() for H in (Hq, Hkv, Hkv)]
    pools = qr.e4m3(kc), qr.e4m3(vc), ks, vs
    keep = [t.clone() for t in pools]

    def step():
        for t, k in zip(pools, keep):
            t.view(torch.uint8).copy_(k.view(torch.uint8)) if t.dtype == torch.float8_e4m3fn else t.copy_(k)
        x, w = qkv.detach().requires_grad_(), weight.detach().requires_grad_()
        q, k, v = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, w, w, start=start)
        out = list(torch.autograd.grad((q, k, v), (x, w), grads))
        with torch.no_grad():
            q, k, v = q.detach(), k.detach(), v.detach()
            co_alibi_attn.append_paged_kv(k, v, *pools[:2], table, start, scales=pools[2:])
            o = co_alibi_attn.paged_tree_attention(q, *pools[:2], table, start, scales=pools[2:])
            back = co_alibi_attn.read_paged_kv(*pools[:2], table, start[:, None], pools[2:], dtype=dt)
        return out + [o, *back]

    return step


SETS = [(1, 32, 8, 128, 1, bf16, [3000, 17, 8000]), (2, 12, 12, 64, 1, f16, [37]), (3, 32, 8, 128, 12, f16, [2000, 900, 4100]),
        (4, 12, 12, 64, 20, bf16, [1500, 0, 333]), (5, 8, 1, 128, 40, bf16, [5000, 2500]), (6, 16, 16, 128, 3, f16, [200, 1, 90, 400])]


@pytest.mark.gpu
def test_on_several_streams_at_once():
    import co_alibi_attn
    steps = [_set(*s) for s in SETS]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        got = [[] for _ in steps]
        for i, (step, stream) in enumerate(zip(steps, streams)):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for _ in range(4):
                    got[i].append(step())
        torch.cuda.synchronize()
        assert co_alibi_attn.device_status(reset=True) == 0
        for i, runs in enumerate(got):
            assert all(torch.equal(a, b) for run in runs for a, b in zip(run, want[i])), f"set {i}"


@pytest.mark.gpu
def test_out_of_graphs_that_share_a_pool():
    steps = [_set(*s) for s in SETS[:4]]
    want = [[t.clone() for t in step()] for step in steps]
    torch.cuda.synchronize()
    graphs, out, pool = [], [], None
    for step in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out.append(step())
        pool = pool or graph.pool()
        graphs.append(graph)
    for i in (0, 1, 2, 3, 2, 0, 0, 3, 1):
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(out[i], want[i])), f"graph {i}"


@pytest.mark.gpu
def test_heads_past_32_bits():
    """2^31 elements and more in the projection and in the queries: the first and the last tokens as by themselves."""
    import co_alibi_attn
    B, S, Hq, Hkv, D, dt = 2, 5600, 1540, 2, 128, bf16
    base = torch.randn(64, Hq + 2 * Hkv, D, device="cuda").to(dt)
    x = base.repeat(-(-B * S // 64), 1, 1)[:B * S].view(B, S, Hq + 2 * Hkv, D)
    assert x.numel() > 1 << 31 and B * S * Hq * D > 1 << 31
    x.requires_grad_()
    weight = (1 + 0.2 * torch.randn(D, device="cuda")).requires_grad_()
    q, k, v = co_alibi_attn.norm_rotate_qkv(x, Hq, Hkv, weight)
    dx, = torch.autograd.grad(q, x, q.detach())
    for sel in (slice(0, 1), slice(B - 1, B)):
        part = x.detach()[sel, -40:].requires_grad_()
        want = co_alibi_attn.norm_rotate_qkv(part, Hq, Hkv, weight)
        for a, b in zip((q, k, v), want):
            assert torch.equal(a[sel, :, -40:], b)
        d, = torch.autograd.grad(want[0], part, want[0].detach())
        assert torch.equal(dx[sel, -40:], d)


@pytest.mark.gpu
@pytest.mark.parametrize("width", ["cut", "wide"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_drafts_whose_keys_are_nan(form, width):
    """A row that sees one is NaN; the others do not know of it."""
    import co_alibi_attn
    Hq, Hkv, Sq, D, dt = form
    ctx, kc, vc, ks, vs, table, words, q, slopes = _case(form, width, 40)
    want, bound = qr.attention(q, kc, vc, ks, vs, table, ctx, words, slopes, 1 / math.sqrt(D))
    t = 1 if Sq < 5 else 4
    for b, c in enumerate(ctx):
        kc[table[b, (c + t) // 16], :, (c + t) % 16, b % D] = 0x7f if b % 2 else 0xff
    o = _run(q, kc, vc, ks, vs, _widen(table, 4096) if width == "wide" else table, ctx, words)
    assert co_alibi_attn.device_status(reset=True) == 0
    sees = [[bool(w >> t & 1) for w in words[b]] for b in range(len(ctx))]
    assert any(not s for row in sees for s in row)
    for b, row in enumerate(sees):
        for i, s in enumerate(row):
            if s:
                assert o[b, :, i].isnan().all(), (b, i)
                o[b, :, i] = want[b, :, i].to(o)
    _check(o, want, bound)
