"""Generation at the edges of its cache and of its arguments.  On the CPU with plain forms of
the operators (the path's own indexing and bookkeeping), on the GPU with the kernels."""
import pytest
import torch

from tests import _serving_cpu
from tests.test_gpt import oracle_attention

VOCAB = 331


def _model(device, rotary_dim=0):
    from co_alibi_gpt import GPTConfig, build
    cfg = GPTConfig(n_layer=2, d_model=128, n_head=2, vocab=VOCAB, seq_len=96, init_std=0.15, rotary_dim=rotary_dim)
    if device == "cpu":
        return build(cfg, "cpu", seed=5, dtype=torch.float32, attn_fn=oracle_attention)[0].eval()
    return build(cfg, "cuda", seed=5, dtype=torch.float16)[0].eval()


def _tokens(B, S, device, seed=6):
    return torch.randint(0, VOCAB, (B, S), generator=torch.Generator().manual_seed(seed)).to(device)


@torch.no_grad()
def _greedy(model, tokens, n):
    """n greedy tokens after each row of tokens [B, S], by the causal forward; and the logits."""
    out = []
    for _ in range(n):
        logits = model(tokens)[:, -1]
        out.append(logits.argmax(-1))
        tokens = torch.cat((tokens, out[-1][:, None]), 1)
    return torch.stack(out, 1), logits


def _status(device):
    if device == "cpu":
        n = len(_serving_cpu.reports)
        _serving_cpu.reports.clear()
        return n
    import co_alibi_attn
    return co_alibi_attn.device_status(reset=True)


def _generate(device, monkeypatch):
    if device == "cpu":
        return _serving_cpu.stand_in(monkeypatch)
    from co_alibi_gpt import generate
    return generate


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("rotary_dim", [0, 32])
@pytest.mark.parametrize("device", DEVICES)
def test_a_tree_of_siblings_two_tokens_before_the_end(device, rotary_dim, monkeypatch):
    """Siblings take a slot each: with ``lens`` at max_len - 2 the right one, the last of seven,
    lies behind max_len.  It is verified and accepted, and the cache goes on from it.  Logits
    agree as in the test of the cached path, float16 through two layers."""
    gen = _generate(device, monkeypatch)
    model = _model(device, rotary_dim)
    S = 46
    prompt = _tokens(2, S, device)
    plain, after = _greedy(model, prompt, 3)
    cache = gen.PagedCache(model, 2, S + 2, page_size=16)
    last = gen.prefill(model, cache, prompt).argmax(-1)
    assert torch.equal(last, plain[:, 0])
    wrong = (plain[:, 1:2] + 1 + torch.arange(6, device=device)) % VOCAB
    drafts = torch.cat((wrong, plain[:, 1:2]), 1)
    tokens, n = gen.tree_step(model, cache, last, drafts, torch.zeros_like(drafts), temperature=0.0)
    assert n.tolist() == [2, 2] and torch.equal(tokens[:, :2], plain[:, 1:])
    assert cache.lens.tolist() == [S + 2, S + 2] and _status(device) == 0
    logits = gen.extend(model, cache, tokens[:, 1:2])[:, 0]
    full, _ = _greedy(model, torch.cat((prompt, plain), 1), 1)
    assert torch.equal(logits.argmax(-1), full[:, 0]) and _status(device) == 0


@pytest.mark.parametrize("rotary_dim", [0, 32])
@pytest.mark.parametrize("device", DEVICES)
def test_drafts_without_a_slot_are_not_accepted(device, rotary_dim, monkeypatch):
    """A chain of right drafts over a cache with room for some of them: what fits is accepted and
    the sample after it is right; a request without any room gets nothing, and is reported."""
    gen = _generate(device, monkeypatch)
    model = _model(device, rotary_dim)
    counts = torch.tensor([28, 31, 20], dtype=torch.int32, device=device)
    prompt = _tokens(3, 31, device)
    cache = gen.PagedCache(model, 3, 32, page_size=16, spare=0)
    assert cache.capacity == 32
    last = gen.prefill(model, cache, prompt, counts).argmax(-1)
    plain = torch.stack([_greedy(model, prompt[b:b + 1, :counts[b]], 8)[0][0] for b in range(3)])
    assert torch.equal(last, plain[:, 0])
    drafts, parents = plain[:, 1:7], torch.arange(6, device=device).expand(3, 6)
    tokens, n = gen.tree_step(model, cache, last, drafts, parents, temperature=0.0)
    assert n.tolist() == [4, 1, 7] and cache.lens.tolist() == [32, 32, 27] and _status(device) == 0
    for b, m in enumerate(n.tolist()):
        assert torch.equal(tokens[b, :m], plain[b, 1:m + 1])
    # the first two are full now
    before = [x.clone() for x in cache.k + cache.v]
    last = tokens.gather(1, n.long()[:, None] - 1)[:, 0]
    one = (tokens[:, :1] * 0, torch.zeros_like(parents[:, :1]))
    tokens, n = gen.tree_step(model, cache, last, *one, temperature=0.0)
    assert n.tolist()[:2] == [0, 0] and n[2] >= 1 and cache.lens.tolist()[:2] == [32, 32]
    assert (tokens[:2] == -1).all() and torch.equal(tokens[2, :1], _greedy(model, torch.cat((prompt[2, :20], plain[2]))[None], 1)[0][0])
    assert _status(device) != 0
    for x, y in zip(before, cache.k + cache.v):
        assert torch.equal(x[cache.table[:2].long()], y[cache.table[:2].long()])


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_a_chunk_past_the_end_have_no_logits(device, monkeypatch):
    gen = _generate(device, monkeypatch)
    model = _model(device, 32)
    tok = _tokens(2, 36, device)
    cache = gen.PagedCache(model, 2, 32, page_size=16, spare=0)
    gen.prefill(model, cache, tok[:, :30], torch.tensor([30, 25], dtype=torch.int32, device=device))
    chunk = torch.stack((tok[0, 30:35], tok[1, 25:30]))
    logits = gen.extend(model, cache, chunk)
    with torch.no_grad():
        full = model(tok)
    assert logits[0, 2:].isnan().all() and _status(device) != 0
    for got, want in ((logits[0, :2], full[0, 30:32]), (logits[1], full[1, 25:30])):
        assert (got.float() - want.float()).abs().max() < 0.1


@pytest.mark.parametrize("max_len,spare,page", [(48, None, 16), (50, None, 16), (33, 0, 32), (96, 8, 16)])
def test_every_slot_of_a_cache_has_an_angle(max_len, spare, page):
    from co_alibi_attn.serving import TREE_MAX_SQ
    from co_alibi_gpt.generate import PagedCache
    cache = PagedCache(_model("cpu", 32), 2, max_len, page, **({} if spare is None else {"spare": spare}))
    slots = cache.table.shape[1] * page
    assert cache.capacity == slots == cache.rotary[0].shape[0]
    assert slots >= max_len + (TREE_MAX_SQ if spare is None else spare)
    assert cache.k[0].shape[0] == cache.table.numel()


def test_a_prompt_longer_than_the_cache_is_refused(monkeypatch):
    gen = _generate("cpu", monkeypatch)
    for rotary_dim in (0, 32):
        model = _model("cpu", rotary_dim)
        with pytest.raises(ValueError):
            gen.prefill(model, gen.PagedCache(model, 1, 16, page_size=16, spare=0), _tokens(1, 17, "cpu"))


def test_more_drafts_than_a_word_has_bits_are_refused(monkeypatch):
    gen = _generate("cpu", monkeypatch)
    model = _model("cpu")
    cache = gen.PagedCache(model, 1, 16, page_size=16)
    with pytest.raises(ValueError):
        gen.tree_step(model, cache, _tokens(1, 1, "cpu")[:, 0], _tokens(1, 64, "cpu"), torch.arange(64)[None])


@pytest.mark.parametrize("device", DEVICES)
def test_padding_of_minus_one_is_not_looked_up(device, monkeypatch):
    """Prompts and drafts padded with -1, which no embedding has a row for."""
    gen = _generate(device, monkeypatch)
    model = _model(device)
    counts = torch.tensor([11, 4], dtype=torch.int32, device=device)
    prompt = _tokens(2, 11, device)
    prompt[1, 4:] = -1
    plain = torch.stack([_greedy(model, prompt[b:b + 1, :counts[b]], 4)[0][0] for b in range(2)])
    cache = gen.PagedCache(model, 2, 32, page_size=16)
    last = gen.prefill(model, cache, prompt, counts).argmax(-1)
    drafts = torch.cat((plain[:, 1:3], torch.full_like(plain[:, :2], -1)), 1)
    parents = torch.tensor([[0, 1, -1, -1]] * 2, device=device)
    tokens, n = gen.tree_step(model, cache, last, drafts, parents, temperature=0.0)
    assert n.tolist() == [3, 3] and torch.equal(tokens[:, :3], plain[:, 1:]) and _status(device) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_a_model_without_a_token_to_draw_ends_in_minus_one(device, monkeypatch):
    gen = _generate(device, monkeypatch)
    model = _model(device)
    with torch.no_grad():
        model.ln_f.weight.fill_(float("nan"))
    assert (gen.generate(model, _tokens(2, 5, device), 3, page_size=16) == -1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_counts_outside_the_prompt(device, monkeypatch):
    """A count past the prompt's width means all of it; a request without tokens has no logits."""
    gen = _generate(device, monkeypatch)
    model = _model(device)
    prompt = _tokens(4, 9, device)
    counts = torch.tensor([9, 12, 0, -3], dtype=torch.int32, device=device)
    cache = gen.PagedCache(model, 4, 16, page_size=16)
    logits = gen.prefill(model, cache, prompt, counts)
    assert cache.lens.tolist() == [9, 9, 0, 0] and logits[2:].isnan().all() and _status(device) == 0
    assert torch.equal(logits[:2].argmax(-1), _greedy(model, prompt[:2], 1)[0][:, 0])
    # with fewer slots than prompt: what entered counts, the rest leaves no logits
    cache = gen.PagedCache(model, 4, 5, page_size=16, spare=0)
    wide = _tokens(4, 20, device)
    logits = gen.prefill(model, cache, wide, torch.tensor([16, 17, 3, 20], dtype=torch.int32, device=device))
    assert cache.lens.tolist() == [16, 16, 3, 16]
    assert logits.isnan().any(1).tolist() == [False, True, False, True] and _status(device) != 0


@pytest.mark.parametrize("device", DEVICES)
def test_no_new_tokens(device, monkeypatch):
    out = _generate(device, monkeypatch).generate(_model(device), _tokens(3, 5, device), 0)
    assert out.shape == (3, 0) and out.dtype == torch.int64


@pytest.mark.parametrize("device", DEVICES)
def test_a_parent_that_does_not_come_before_its_draft_is_none(device, monkeypatch):
    """Row numbers of parents past the draft's own, past the tree, or of an absent draft: such a
    draft sees nothing and is not accepted, and no index leaves the tree."""
    gen = _generate(device, monkeypatch)
    words, depths = gen.tree_words(torch.tensor([[1, 0, 99, 2, -7]]))
    assert words.tolist() == [[1, 0, 0b101, 0, 0b10101, 0]] and depths.tolist() == [[0, 0, 1, 0, 2, 0]]
    model = _model(device)
    prompt = _tokens(1, 12, device)
    plain, _ = _greedy(model, prompt, 5)
    cache = gen.PagedCache(model, 1, 32, page_size=16)
    last = gen.prefill(model, cache, prompt).argmax(-1)
    drafts = plain[:, [1, 1, 2, 2, 3]]
    for parents, accepted in (([2, 0, 99, 2, 4], 3), ([2, 99, 0, 3, 1], 0), ([5, 1, 1, 1, 1], 0)):
        cache.lens.fill_(12)
        tokens, n = gen.tree_step(model, cache, last, drafts, torch.tensor([parents], device=device), temperature=0.0)
        assert n.tolist() == [accepted + 1] and torch.equal(tokens[0, :accepted + 1], plain[0, 1:accepted + 2])


@pytest.mark.parametrize("device", DEVICES)
def test_an_absent_token_confirms_nothing(device, monkeypatch):
    """Where nothing can be drawn the step ends, also before drafts of -1 that name a parent."""
    gen = _generate(device, monkeypatch)
    model = _model(device)
    cache = gen.PagedCache(model, 2, 32, page_size=16)
    last = gen.prefill(model, cache, _tokens(2, 5, device)).argmax(-1)
    with torch.no_grad():
        model.ln_f.weight.fill_(float("nan"))
    drafts = torch.full((2, 3), -1, device=device)
    tokens, n = gen.tree_step(model, cache, last, drafts, torch.arange(3, device=device).expand(2, 3))
    assert (tokens == -1).all() and n.tolist() == [1, 1] and cache.lens.tolist() == [6, 6]
