"""Generation with normed heads and over a cache in 8 bits: the edges of the cache and of the arguments."""
import pytest
import torch

from tests import _serving_cpu
from tests import test_generate_limits as limits
from tests.test_generate_quant import E4M3, _cfg, _model, plain_heads
from tests.test_gpt import oracle_attention
from tests.test_quant_append import _tables


@pytest.mark.gpu
def test_small_values_of_a_float16_model_move_whole():
    """Accepted tokens keep their values where float16 has none for their codes."""
    from co_alibi_attn import append_paged_kv, read_paged_kv
    from co_alibi_gpt import generate as gen
    model = _model(_cfg())
    cache = gen.PagedCache(model, 2, 60, page_size=16, kv_dtype=E4M3)
    H, D, n = 2, 64, 40
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, H, n, D, generator=g).clamp(-1, 1) * 2.0 ** torch.randint(-9, 1, (2, H, n, D), generator=g)
    x[..., -1] = 2.0  # the same scale in every block (rotated elements are at most 2^0.5)
    x = (x * 2.0 ** -15).half().cuda()
    rotary = tuple(t.cuda() for t in _tables(n, 32))  # rotated keys enter the cache from float32
    for layer, (k, v) in enumerate(zip(cache.k, cache.v)):
        append_paged_kv(x, x, k, v, cache.table, cache.lens, rotary=rotary, **cache.of(layer))
    cache.lens += 22
    path = torch.tensor([[23, 26, 31, 39], [24, 25, 38, 22]], dtype=torch.int32).cuda()
    read = lambda layer, at: read_paged_kv(cache.k[layer], cache.v[layer], cache.table, at, cache.scales[layer])  # noqa: E731
    want = [read(layer, path) for layer in range(2)]
    assert float(want[0][0].abs().max()) == 2.0 ** -14 and (want[0][0].float() != want[0][0].half().float()).any()
    cache.move(path, torch.tensor([4, 2], dtype=torch.int32).cuda())
    at = cache.lens[:, None] + torch.arange(4, dtype=torch.int32).cuda()
    for layer in range(2):
        for got, expect in zip(read(layer, at), want[layer]):
            assert torch.equal(got[0], expect[0]) and torch.equal(got[1, :, :2], expect[1, :, :2])


def reporting_heads(qkv, Hq, Hkv, q_weight, k_weight, eps=1e-6, rotary=None, start=None, positions=None):
    """norm_rotate_qkv in torch operations; a position outside the tables leaves the row as it is and is noted, as the
    kernel reports it."""
    plain = plain_heads(qkv, Hq, Hkv, q_weight, k_weight, eps)
    if rotary is None:
        return plain
    at = positions if positions is not None else torch.arange(qkv.shape[1]).expand(qkv.shape[:2]) + (0 if start is None else start[:, None])
    out = (at < 0) | (at >= rotary[0].shape[0])
    _serving_cpu.reports.extend(("angle", *w) for w in out.nonzero().tolist())
    turned = plain_heads(qkv, Hq, Hkv, q_weight, k_weight, eps, rotary, positions=at.masked_fill(out, 0))
    return tuple(torch.where(out[:, None, :, None], a, b) for a, b in zip(plain[:2], turned[:2])) + (plain[2],)


def _normed(device, rotary_dim=0):
    """Weights by which its first greedy tokens differ from one another, as the tests of drafts take them to."""
    from co_alibi_gpt import build
    cfg, kw = _cfg(rotary_dim=rotary_dim, init_std=0.3), dict(dtype=torch.float16)
    if device == "cpu":
        kw = dict(dtype=torch.float32, attn_fn=oracle_attention, heads_fn=reporting_heads)
    model = build(cfg, device, seed=4, **kw)[0].eval()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith(("q_norm", "k_norm")):
                p.fill_(2.0)
    return model


@pytest.mark.parametrize("rotary_dim", [0, 32])
@pytest.mark.parametrize("device", limits.DEVICES)
@pytest.mark.parametrize("name", ["test_a_tree_of_siblings_two_tokens_before_the_end", "test_drafts_without_a_slot_are_not_accepted",
                                  "test_rows_of_a_chunk_past_the_end_have_no_logits", "test_padding_of_minus_one_is_not_looked_up",
                                  "test_a_model_without_a_token_to_draw_ends_in_minus_one", "test_counts_outside_the_prompt", "test_no_new_tokens",
                                  "test_a_parent_that_does_not_come_before_its_draft_is_none", "test_an_absent_token_confirms_nothing"])
def test_limits_of_a_normed_model(name, device, rotary_dim, monkeypatch):
    test = getattr(limits, name)
    own = "rotary_dim" in test.__code__.co_varnames[:test.__code__.co_argcount]
    if name == "test_counts_outside_the_prompt":
        rotary_dim = 0  # (prompts wider than a cache of rotated keys are refused)
    monkeypatch.setattr(limits, "_model", lambda device, rotary=None: _normed(device, rotary_dim if rotary is None else rotary))
    test(device, *((rotary_dim,) if own else ()), monkeypatch)


@pytest.mark.parametrize("deep", [False, True])
@pytest.mark.parametrize("device", limits.DEVICES)
def test_tokens_that_counts_leaves_out_are_not_reported(device, deep, monkeypatch):
    """Their positions run past the end of the cache and of the tables; those that enter have their logits."""
    gen = limits._generate(device, monkeypatch)
    model = _normed(device, 32)
    tok = limits._tokens(2, 36, device)
    cache = gen.PagedCache(model, 2, 32, page_size=16, spare=0)
    lens = torch.tensor([29, 24], dtype=torch.int32, device=device)
    gen.prefill(model, cache, tok[:, :30], lens)
    chunk = torch.stack((tok[0, 29:34], tok[1, 24:29]))
    steps = torch.arange(5, dtype=torch.int32, device=device)
    counts = torch.tensor([3, 5], dtype=torch.int32, device=device)
    words = torch.where(steps < counts[:, None], (2 << steps.long()) - 1, 0)
    depths = (steps + torch.where(steps < counts[:, None], 0, 1000)).int() if deep else None
    logits = gen.extend(model, cache, chunk, words, depths, counts)
    assert limits._status(device) == 0
    with torch.no_grad():
        full = model(tok)
    for got, want in ((logits[0, :3], full[0, 29:32]), (logits[1], full[1, 24:29])):
        assert (got.float() - want.float()).abs().max() < 0.1
    # what enters the cache past the tables is reported
    gen.extend(model, cache, chunk, words, steps.expand(2, 5) + 1000, counts)
    assert limits._status(device) != 0


def test_rows_of_codes_are_refused():
    from co_alibi_gpt.generate import PagedCache
    model, at = limits._model("cpu"), torch.zeros(2, 3, dtype=torch.int32)
    cache = PagedCache(model, 2, 20, 16)
    assert cache.rows(cache.k[0], at).shape == (2, 2, 3, 64)
    cache = PagedCache(model, 2, 20, 16, kv_dtype=E4M3)
    with pytest.raises(ValueError):
        cache.rows(cache.k[0], at)


def _sampled_path(sampled, drafts, parents, slots):
    """How many tokens a tree step of greedy samples accepts: the walk from row 0 along drafts with a slot."""
    n, at = 1, 0
    while True:
        next_ = [t for t in range(drafts.shape[0]) if int(parents[t]) == at and t + 1 < slots and int(drafts[t]) == int(sampled[at])]
        if not next_:
            return n
        n, at = n + 1, next_[0] + 1


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm", [False, True])
def test_drafts_at_the_end_of_a_cache_in_8_bits(qk_norm):
    """A chain of drafts over caches with room for some of them.  What is accepted follows the cache's own samples (the same
    rows give the same logits again: their scales are there already); a full cache keeps its codes and is reported."""
    from co_alibi_gpt import generate as gen
    model = _normed("cuda", 32) if qk_norm else limits._model("cuda", 32)
    counts = torch.tensor([28, 31, 20], dtype=torch.int32, device="cuda")
    prompt = limits._tokens(3, 31, "cuda")

    def start():
        cache = gen.PagedCache(model, 3, 32, page_size=16, spare=0, kv_dtype=E4M3)
        return cache, gen.prefill(model, cache, prompt, counts).argmax(-1)

    cache, last = start()
    chain = [last]
    room = cache.capacity - cache.lens
    for _ in range(6):  # greedy tokens, one at a time, where there is room
        chain.append(gen.extend(model, cache, chain[-1][:, None])[:, 0].nan_to_num(nan=-1.0).argmax(-1))
        cache.lens += 1
    limits._status("cuda")
    drafts, parents = torch.stack(chain[1:], 1), torch.arange(6, device="cuda").expand(3, 6)
    cache, last = start()
    words, depths = gen.tree_words(torch.where(torch.arange(1, 7, device="cuda") < room[:, None], parents, -1))
    sampled = gen.extend(model, cache, torch.cat((last[:, None], drafts), 1), words, depths, room).nan_to_num(nan=-1.0).argmax(-1)
    assert limits._status("cuda") == 0
    want = [_sampled_path(sampled[b], drafts[b], parents[b], int(room[b])) for b in range(3)]
    tokens, n = gen.tree_step(model, cache, last, drafts, parents, temperature=0.0)
    assert limits._status("cuda") == 0 and n.tolist() == want and want[1] == 1 and want[0] >= 2 and want[2] >= 4
    assert cache.lens.tolist() == [int(c) + m for c, m in zip(counts, want)]
    for b, m in enumerate(want):
        assert torch.equal(tokens[b, :m], sampled[b, :m])
    # full now
    cache.lens[0] = cache.capacity
    before = [x.view(torch.uint8)[cache.table[:2].long()].clone() for x in cache.k + cache.v]
    scales = [s[cache.table[:2].long()].clone() for pair in cache.scales for s in pair]
    tokens, n = gen.tree_step(model, cache, tokens[:, 0], drafts[:, :1], parents[:, :1], temperature=0.0)
    assert n.tolist()[:2] == [0, 0] and n[2] >= 1 and (tokens[:2] == -1).all() and limits._status("cuda") != 0
    assert all(torch.equal(a, x.view(torch.uint8)[cache.table[:2].long()]) for a, x in zip(before, cache.k + cache.v))
    assert all(torch.equal(a, s[cache.table[:2].long()]) for a, s in zip(scales, (s for pair in cache.scales for s in pair)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["test_a_model_without_a_token_to_draw_ends_in_minus_one", "test_counts_outside_the_prompt", "test_no_new_tokens",
                                  "test_an_absent_token_confirms_nothing"])
def test_limits_of_a_cache_in_8_bits(name, monkeypatch):
    """Those that ask for no more bits than e4m3 has: statuses, lengths, absent tokens, a prompt's own logits."""
    from co_alibi_gpt import generate as gen
    real = gen.PagedCache
    monkeypatch.setattr(gen, "PagedCache", lambda *a, **kw: real(*a, **{**kw, "kv_dtype": E4M3}))
    getattr(limits, name)("cuda", monkeypatch)


@pytest.mark.gpu
def test_rows_of_a_chunk_past_the_end_of_a_cache_in_8_bits():
    """Without logits, and reported; the rows that fit have those of a chunk of them alone (two forms of the attention over
    the same codes: 0.1, as in the other tests of logits)."""
    from co_alibi_gpt import generate as gen
    model = limits._model("cuda", 32)
    tok = limits._tokens(2, 36, "cuda")
    cache = gen.PagedCache(model, 2, 32, page_size=16, spare=0, kv_dtype=E4M3)
    gen.prefill(model, cache, tok[:, :30], torch.tensor([30, 25], dtype=torch.int32, device="cuda"))
    chunk = torch.stack((tok[0, 30:35], tok[1, 25:30]))
    logits = gen.extend(model, cache, chunk)
    assert logits[0, 2:].isnan().all() and torch.isfinite(logits[1]).all() and limits._status("cuda") != 0
    fits = gen.extend(model, cache, chunk[:, :2])
    assert limits._status("cuda") == 0 and (logits[:, :2].float() - fits.float()).abs().max() < 0.1 and fits.float().abs().max() > 3
