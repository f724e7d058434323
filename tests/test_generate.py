"""Generation with the Co-ALiBi GPT over the paged cache: the serving operators run
together, against the model's own causal forward on the same weights."""
import pytest
import torch

from tests.test_gpt import oracle_attention


def _cfg(**kw):
    from co_alibi_gpt import GPTConfig
    return GPTConfig(**{**dict(n_layer=2, d_model=128, n_head=2, vocab=331, seq_len=96, init_std=0.15), **kw})


def _model(cfg):
    from co_alibi_gpt import build
    return build(cfg, "cuda", seed=5, dtype=torch.float16)[0].eval()


def test_rotary_model_is_causal_and_differs_on_cpu():
    from co_alibi_gpt import build, make_tokens
    cfg = _cfg(rotary_dim=32, seq_len=24)
    model, _ = build(cfg, "cpu", seed=1, dtype=torch.float32, attn_fn=oracle_attention)
    plain, _ = build(_cfg(seq_len=24), "cpu", seed=1, dtype=torch.float32, attn_fn=oracle_attention)
    tok = make_tokens(cfg, 2, seed=2)
    tok2 = tok.clone()
    tok2[:, 20] = (tok2[:, 20] + 1) % cfg.vocab
    with torch.no_grad():
        a, b, c = model(tok[:, :-1]), model(tok2[:, :-1]), plain(tok[:, :-1])
    assert torch.allclose(a[:, :20], b[:, :20], atol=1e-5) and not torch.allclose(a, c, atol=1e-2)
    model(tok[:, :-1], targets=tok[:, 1:]).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


def test_tree_words():
    pytest.importorskip("co_alibi_attn")
    from co_alibi_gpt.generate import tree_words
    parents = torch.tensor([[0, 1, 0, 3, -1], [0, 0, 0, 0, 4]])
    words, depths = tree_words(parents)
    assert words.tolist() == [[1, 0b11, 0b111, 0b1001, 0b11001, 0], [1, 0b11, 0b101, 0b1001, 0b10001, 0b110001]]
    assert depths.tolist() == [[0, 1, 2, 1, 2, 0], [0, 1, 1, 1, 1, 2]]
    chain = tree_words(torch.arange(63)[None])[0]
    assert chain[0, 63].item() == -1 and chain[0, 62].item() == (1 << 63) - 1
    with pytest.raises(ValueError):
        tree_words(torch.zeros(1, 64, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_cached_logits_match_the_causal_forward(rotary_dim):
    """Ragged prompts, then single tokens, then a chunk: float16 activations and two attention
    paths with a 2e-3 error each through two layers; logits of magnitude ~10 agree to 0.1."""
    from co_alibi_gpt.generate import PagedCache, extend, prefill
    model = _model(_cfg(rotary_dim=rotary_dim))
    tok = torch.randint(0, 331, (3, 90), generator=torch.Generator().manual_seed(6)).cuda()
    counts = torch.tensor([40, 17, 1], dtype=torch.int32).cuda()
    with torch.no_grad():
        full = model(tok)
    b = torch.arange(3, device="cuda")
    cache = PagedCache(model, 3, 90, page_size=16)
    got = prefill(model, cache, tok[:, :40], counts)
    want = [full[b, counts.long() - 1]]
    got = [got]
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


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_tree_step_accepts_what_the_samples_confirm(rotary_dim):
    from co_alibi_gpt.generate import PagedCache, extend, generate, prefill, tree_step
    model = _model(_cfg(rotary_dim=rotary_dim))
    prompt = torch.randint(0, 331, (2, 20), generator=torch.Generator().manual_seed(7)).cuda()
    plain = generate(model, prompt, 12, temperature=0.0, page_size=16)
    cache = PagedCache(model, 2, 60, page_size=16)
    logits = prefill(model, cache, prompt)
    last = logits.argmax(-1)
    assert torch.equal(last, plain[:, 0])
    # request 0: the right chain of 4 behind a wrong branch; request 1: right once, then wrong
    wrong = (plain + 1) % 331
    drafts = torch.stack((torch.stack((wrong[0, 1], plain[0, 1], plain[0, 2], plain[0, 3], plain[0, 4])),
                          torch.stack((plain[1, 1], wrong[1, 2], wrong[1, 1], wrong[1, 2], wrong[1, 2]))))
    parents = torch.tensor([[0, 0, 2, 3, 4], [0, 1, 0, 1, -1]]).cuda()
    tokens, n = tree_step(model, cache, last, drafts, parents, temperature=0.0)
    assert n.tolist() == [5, 2]
    assert torch.equal(tokens[0, :5], plain[0, 1:6]) and torch.equal(tokens[1, :2], plain[1, 1:3])
    assert cache.lens.tolist() == [25, 22]
    # the cache goes on as if the accepted tokens had come one by one
    last = torch.stack((tokens[0, 4], tokens[1, 1]))
    logits = extend(model, cache, last[:, None])[:, 0]
    for r, m in ((0, 6), (1, 3)):
        with torch.no_grad():
            full = model(torch.cat((prompt[r], plain[r, :m]))[None])[0, -1]
        assert (logits[r].float() - full.float()).abs().max() < 0.1


@pytest.mark.gpu
def test_generate_samples_with_a_seed():
    from co_alibi_gpt.generate import generate
    model = _model(_cfg())
    prompt = torch.randint(0, 331, (4, 33), generator=torch.Generator().manual_seed(8)).cuda()
    counts = torch.tensor([33, 5, 20, 1], dtype=torch.int32).cuda()
    run = lambda seed: generate(model, prompt, 9, counts=counts, top_k=20, top_p=0.9,  # noqa: E731
                                temperature=torch.tensor([1.0, 0.7, 0.0, 1.3], device="cuda"),
                                generator=torch.Generator(device="cuda").manual_seed(seed))
    a, b, c = run(1), run(1), run(2)
    assert a.shape == (4, 9) and (a >= 0).all() and (a < 331).all()
    assert torch.equal(a, b) and not torch.equal(a, c) and torch.equal(a[2], c[2])
