"""The GPT with normed heads, and generation over a cache in 8 bits: the operators run together, as a
model uses them."""
import math

import pytest
import torch

from tests import _quant_ref as qr
from tests import _serving_ref as ref
from tests.test_gpt import oracle_attention
from tests.test_quant_append import _same

E4M3 = torch.float8_e4m3fn


def plain_heads(qkv, Hq, Hkv, q_weight, k_weight, eps=1e-6, rotary=None, start=None, positions=None, interleaved=False):
    """norm_rotate_qkv in torch operations, in float32 and rounded once; differentiable."""
    B, S, _, D = qkv.shape
    out = []
    for x, w in ((qkv[:, :, :Hq], q_weight), (qkv[:, :, Hq:Hq + Hkv], k_weight)):
        x = x.float()
        y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w.float()
        if rotary is not None:
            at = positions if positions is not None else torch.arange(S, device=x.device) + (0 if start is None else start[:, None])
            c, s = (t[at.long()].view(-1, S, 1, t.shape[1]) for t in rotary)
            r = c.shape[-1]
            a, b = y[..., :r], y[..., r:2 * r]
            y = torch.cat((a * c - b * s, b * c + a * s, y[..., 2 * r:]), -1)
        out.append(y.to(qkv.dtype).transpose(1, 2).contiguous())
    return out[0], out[1], qkv[:, :, Hq + Hkv:].transpose(1, 2).contiguous()


def _cfg(**kw):
    from co_alibi_gpt import GPTConfig
    return GPTConfig(**{**dict(n_layer=2, d_model=128, n_head=2, vocab=331, seq_len=96, init_std=0.15, qk_norm=True), **kw})


def _model(cfg, **kw):
    from co_alibi_gpt import build
    model = build(cfg, "cuda", seed=5, dtype=torch.float16, **kw)[0].eval()
    g = torch.Generator().manual_seed(9)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith(("q_norm", "k_norm")):
                p.copy_(1 + 0.3 * torch.randn(p.shape, generator=g))
    return model


@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_a_normed_model_on_the_cpu(rotary_dim):
    from co_alibi_gpt import build, make_tokens
    cfg = _cfg(rotary_dim=rotary_dim, seq_len=24)
    model, _ = build(cfg, "cpu", seed=1, dtype=torch.float32, attn_fn=oracle_attention, heads_fn=plain_heads)
    plain, _ = build(_cfg(rotary_dim=rotary_dim, seq_len=24, qk_norm=False), "cpu", seed=1, dtype=torch.float32, attn_fn=oracle_attention)
    norms = [n for n, _ in model.named_parameters() if n.endswith(("q_norm", "k_norm"))]
    assert len(norms) == 4 and {n for n, _ in plain.named_parameters()} | set(norms) == {n for n, _ in model.named_parameters()}
    tok = make_tokens(cfg, 2, seed=2)
    tok2 = tok.clone()
    tok2[:, 20] = (tok2[:, 20] + 1) % cfg.vocab
    with torch.no_grad():
        a, b, c = model(tok[:, :-1]), model(tok2[:, :-1]), plain(tok[:, :-1])
    assert torch.allclose(a[:, :20], b[:, :20], atol=1e-5) and not torch.allclose(a, c, atol=1e-2)
    model(tok[:, :-1], targets=tok[:, 1:]).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [0, 64])
def test_a_training_step_agrees_with_plain_heads(rotary_dim):
    """The same weights and attention, heads by the operator and in torch: their float16 results differ by a
    rounding here and there, and what goes through two layers is held to the model tests' tolerances."""
    model, plain = _model(_cfg(rotary_dim=rotary_dim)), _model(_cfg(rotary_dim=rotary_dim), heads_fn=plain_heads)
    tok = torch.randint(0, 331, (3, 97), generator=torch.Generator().manual_seed(3)).cuda()
    losses = [m(tok[:, :-1], targets=tok[:, 1:]) for m in (model, plain)]
    for loss in losses:
        (loss * 64).backward()
    assert (losses[0] - losses[1]).abs() <= 1e-2
    for (name, a), (_, b) in zip(model.named_parameters(), plain.named_parameters()):
        assert (a.grad.float() - b.grad.float()).norm() <= 3e-2 * b.grad.float().norm(), name


@pytest.mark.gpu
def test_a_training_step_of_a_normed_model_can_be_captured():
    model = _model(_cfg(rotary_dim=32))
    tok = torch.randint(0, 331, (2, 25), generator=torch.Generator().manual_seed(2)).cuda()

    def step():
        for p in model.parameters():
            p.grad = None
        loss = model(tok[:, :-1], targets=tok[:, 1:])
        loss.backward()
        return loss.detach(), [p.grad for p in model.parameters()]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [step() for _ in range(2)][-1]
        want = want[0].clone(), [g.clone() for g in want[1]]
    torch.cuda.current_stream().wait_stream(stream)
    for p in model.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    graph.replay()
    assert (loss - want[0]).abs() <= 2e-3
    for g, w in zip(grads, want[1]):
        assert (g.float() - w.float()).abs().max() <= 1e-2 * w.float().abs().max() + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_cached_logits_match_the_causal_forward(rotary_dim):
    """A cache in the model's own type; logits of magnitude ~10 agree to 0.1, as without the norm."""
    from co_alibi_gpt.generate import PagedCache, extend, prefill
    model = _model(_cfg(rotary_dim=rotary_dim))
    tok = torch.randint(0, 331, (3, 90), generator=torch.Generator().manual_seed(6)).cuda()
    counts = torch.tensor([40, 17, 1], dtype=torch.int32).cuda()
    with torch.no_grad():
        full = model(tok)
    b = torch.arange(3, device="cuda")
    cache = PagedCache(model, 3, 90, page_size=16)
    got, want = [prefill(model, cache, tok[:, :40], counts)], [full[b, counts.long() - 1]]
    for _ in range(3):
        at = cache.lens.long()
        got.append(extend(model, cache, tok[b, at][:, None])[:, 0])
        want.append(full[b, at])
        cache.lens += 1
    at = cache.lens.long()[:, None] + torch.arange(7, device="cuda")
    got.append(extend(model, cache, tok.gather(1, at)))
    want.append(full[b[:, None], at])
    for x, y in zip(got, want):
        assert (x.float() - y.float()).abs().max() < 0.1 and y.float().abs().max() > 3


def _read_then_attend(gen):
    """paged_tree_attention of a cache in 8 bits by way of the 16-bit one, over the tokens read back."""
    real = gen.paged_tree_attention

    def attend(q, k_pages, v_pages, table, lens, tree_mask=None, bias_max=8.0, scales=None):
        B, room = table.shape[0], table.shape[1] * k_pages.shape[2]
        at = torch.arange(room, dtype=torch.int32, device=q.device).expand(B, room)
        k, v = gen.read_paged_kv(k_pages, v_pages, table, at, scales, dtype=q.dtype)
        # (slots behind the tokens hold anything, which the operator does not look at)
        own = torch.arange(B, dtype=torch.int32, device=q.device)[:, None]
        return real(q, k, v, own, lens, tree_mask=tree_mask, bias_max=bias_max)

    return attend


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm,rotary_dim", [(False, 0), (False, 32), (True, 32)])
def test_logits_over_a_cache_in_8_bits(qk_norm, rotary_dim, monkeypatch):
    """The operators against the 16-bit attention over the same cache read back (two attention paths with an
    error of 2e-3 each through two layers: 0.1, as above); and near the model's own logits, which e4m3's
    three bits move by far less than they differ between tokens."""
    from co_alibi_gpt import generate as gen
    model = _model(_cfg(qk_norm=qk_norm, rotary_dim=rotary_dim))
    tok = torch.randint(0, 331, (3, 90), generator=torch.Generator().manual_seed(6)).cuda()
    counts = torch.tensor([40, 17, 1], dtype=torch.int32).cuda()
    b = torch.arange(3, device="cuda")

    def run():
        cache = gen.PagedCache(model, 3, 90, page_size=32, kv_dtype=E4M3)
        out = [gen.prefill(model, cache, tok[:, :40], counts)]
        for _ in range(3):
            out.append(gen.extend(model, cache, tok[b, cache.lens.long()][:, None])[:, 0])
            cache.lens += 1
        at = cache.lens.long()[:, None] + torch.arange(7, device="cuda")
        out.append(gen.extend(model, cache, tok.gather(1, at)).flatten(0, 1))
        return out, at

    got, at = run()
    monkeypatch.setattr(gen, "paged_tree_attention", _read_then_attend(gen))
    want, _ = run()
    for x, y in zip(got, want):
        assert (x.float() - y.float()).abs().max() < 0.1 and y.float().abs().max() > 3
    with torch.no_grad():
        full = model(tok)[b[:, None], at].flatten(0, 1).float()
    assert (got[-1].float() - full).norm() < 0.3 * full.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_tree_step_over_a_cache_in_8_bits(rotary_dim):
    """Accepted tokens move with the values that they were verified with, behind a context that stays."""
    import co_alibi_attn
    from co_alibi_gpt import generate as gen
    model = _model(_cfg(rotary_dim=rotary_dim))
    prompt = torch.randint(0, 331, (2, 21), generator=torch.Generator().manual_seed(7)).cuda()

    def start():
        cache = gen.PagedCache(model, 2, 60, page_size=16, kv_dtype=E4M3)
        return cache, gen.prefill(model, cache, prompt).argmax(-1)

    cache, last = start()
    greedy = [last]
    for _ in range(5):
        greedy.append(gen.extend(model, cache, greedy[-1][:, None])[:, 0].argmax(-1))
        cache.lens += 1
    plain = torch.stack(greedy, 1)
    wrong = (plain + 1) % 331
    # request 0: the right chain of 3 behind wrong siblings; request 1: wrong at once
    drafts = torch.stack((torch.stack((wrong[0, 1], wrong[0, 2], plain[0, 1], plain[0, 2], plain[0, 3])), wrong[1, 1].expand(5)))
    parents = torch.tensor([[0, 0, 0, 3, 4], [0, 1, 2, 3, 4]]).cuda()
    cache, last = start()
    rows = torch.cat((last[:, None], drafts), 1)
    words, depths = gen.tree_words(parents)
    logits = gen.extend(model, cache, rows, words, depths, cache.capacity - cache.lens)
    sampled = logits.argmax(-1)
    path = [0]  # by the samples, from row 0
    while any(int(parents[0, t]) == path[-1] and drafts[0, t] == sampled[0, path[-1]] for t in range(5)):
        path.append(next(t + 1 for t in range(5) if int(parents[0, t]) == path[-1] and drafts[0, t] == sampled[0, path[-1]]))
    at = torch.cat((torch.arange(21), 21 + torch.tensor(path)))[None].int().cuda()
    want = [gen.read_paged_kv(k[:], v, cache.table[:1], at, s, dtype=torch.float16) for k, v, s in zip(cache.k, cache.v, cache.scales)]
    tokens, n = gen.tree_step(model, cache, last, drafts, parents, temperature=0.0)
    assert n.tolist() == [len(path), 1] and len(path) >= 2 and cache.lens.tolist() == [21 + len(path), 22]
    assert torch.equal(tokens[0, :len(path)], sampled[0, torch.tensor(path).cuda()])
    now = torch.arange(21 + len(path), dtype=torch.int32)[None].cuda()
    for (k, v, s), expect in zip(zip(cache.k, cache.v, cache.scales), want):
        got = gen.read_paged_kv(k, v, cache.table[:1], now, s, dtype=torch.float16)
        assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])
    assert co_alibi_attn.device_status(reset=True) == 0


@pytest.mark.gpu
def test_generate_over_a_cache_in_8_bits():
    from co_alibi_gpt.generate import PagedCache, generate
    model = _model(_cfg(rotary_dim=32))
    prompt = torch.randint(0, 331, (4, 33), generator=torch.Generator().manual_seed(8)).cuda()
    counts = torch.tensor([33, 5, 20, 1], dtype=torch.int32).cuda()
    run = lambda seed: generate(model, prompt, 9, counts=counts, top_k=20, top_p=0.9, kv_dtype=E4M3,  # noqa: E731
                                temperature=torch.tensor([1.0, 0.7, 0.0, 1.3], device="cuda"),
                                generator=torch.Generator(device="cuda").manual_seed(seed))
    a, b, c = run(1), run(1), run(2)
    assert a.shape == (4, 9) and (a >= 0).all() and (a < 331).all()
    assert torch.equal(a, b) and not torch.equal(a, c) and torch.equal(a[2], c[2])
    with pytest.raises(ValueError):
        PagedCache(model, 1, 16, kv_dtype=torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,dt,rot,interleaved", [(8, 2, 128, torch.bfloat16, 64, False), (4, 4, 64, torch.float16, 64, True)])
def test_the_operators_in_a_row(Hq, Hkv, D, dt, rot, interleaved):
    """Heads out of a projection, into the cache, attended over, prompt and then tree, against the definitions
    applied to the same heads."""
    import co_alibi_attn
    from co_alibi_attn.co_alibi_attn import _api_slopes
    from co_alibi_attn.serving import rotary_tables
    B, page = 2, 32
    g = torch.Generator().manual_seed(12)
    kc, vc, ks, vs, table = qr.pool([70, 50], Hkv, D, page, 13)
    rotary = rotary_tables(rot, 200)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2)]
    dev = [qr.e4m3(kc.cuda()), qr.e4m3(vc.cuda()), table.cuda()]
    scales = ks.cuda(), vs.cuda()
    lens = torch.zeros(B, dtype=torch.int32)
    for S, count in ((40, [40, 23]), (1, [1, 1]), (9, [9, 9])):
        qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g).to(dt)
        with torch.no_grad():
            q, k, v = co_alibi_attn.norm_rotate_qkv(qkv.cuda(), Hq, Hkv, *(t.cuda() for t in w), rotary=tuple(t.cuda() for t in rotary),
                                                    start=lens.cuda(), interleaved=interleaved)
            co_alibi_attn.append_paged_kv(k, v, *dev, lens.cuda(), count=torch.tensor(count, dtype=torch.int32).cuda(), scales=scales)
        at = lens[:, None].long() + torch.arange(S)
        q64, k64, v64 = qr.heads(qkv.double(), Hq, Hkv, *(t.double() for t in w), 1e-6, *rotary, at, interleaved)
        for a, b in ((q, q64), (k, k64)):  # the bound of test_heads.py, the pair's |a| + |b| at most twice the row's largest
            assert ((a.cpu().double() - b).abs() <= ref.U[dt] * b.abs() + 2.0 ** -19 * b.abs().amax(-1, keepdim=True)).all()
        qr.append(k.cpu(), kc, ks, table, lens, count)
        qr.append(v.cpu(), vc, vs, table, lens, count)
        assert _same(dev[0].view(torch.uint8), kc) and _same(dev[1].view(torch.uint8), vc)
        assert torch.equal(scales[0].cpu(), ks) and torch.equal(scales[1].cpu(), vs)
        if S < 16:
            words = [ref.tree(S, 30 + b) for b in range(B)]
            mask = torch.tensor([ref.as_int64(x) for x in words], dtype=torch.int64).cuda()
            o = co_alibi_attn.paged_tree_attention(q, *dev, lens.cuda(), tree_mask=mask, scales=scales)
            slopes = _api_slopes(Hq, 8.0, dt, torch.device("cpu"))
            want, bound = qr.attention(q.cpu(), kc, vc, ks, vs, table, lens.tolist(), words, slopes, 1 / math.sqrt(D))
            assert ((o.cpu().double() - want).abs() <= bound).all()
        lens += torch.tensor(count, dtype=torch.int32)
    assert co_alibi_attn.device_status(reset=True) == 0
