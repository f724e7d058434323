"""Generation with the Co-ALiBi GPT: the serving operators of ``co_alibi_attn`` in use.

Prompts run through the model's causal attention once and enter a paged key/value
cache; every further step appends its tokens, attends over the cache and samples
(``generate``), or verifies a tree of drafted tokens at once and keeps the path that
the samples confirm (``tree_step``).  The reference has no counterpart.
"""
import math

import torch
import torch.nn.functional as F

from co_alibi_attn import append_paged_kv, paged_tree_attention, sample_tokens
from co_alibi_attn.serving import TREE_MAX_SQ, rotary_tables

from .model import rotate_heads

__all__ = ["PagedCache", "extend", "generate", "prefill", "tree_step", "tree_words"]


class PagedCache:
    """Keys and values of every layer for ``batch`` requests of up to ``max_len`` tokens:
    pools [n_pages, H, page_size, D], one page table for all layers, and the lengths.
    ``spare`` further slots take the drafts of a step that starts near the end: a tree's
    slots run ahead of its depths, so they may be needed though few are accepted.  In all a
    request has ``capacity`` slots, every one with its row of the rotary tables."""

    def __init__(self, model, batch, max_len, page_size=64, spare=TREE_MAX_SQ):
        cfg, weight = model.cfg, model.emb.weight
        per = -(-(max_len + spare) // page_size)
        self.capacity = per * page_size
        shape = (batch * per, cfg.n_head, page_size, cfg.d_model // cfg.n_head)
        self.k = [torch.empty(shape, dtype=weight.dtype, device=weight.device) for _ in range(cfg.n_layer)]
        self.v = [torch.empty_like(k) for k in self.k]
        self.table = torch.arange(batch * per, dtype=torch.int32, device=weight.device).view(batch, per)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=weight.device)
        self.rotary = rotary_tables(cfg.rotary_dim, self.capacity, device=weight.device) if cfg.rotary_dim else None
        self.steps = torch.arange(TREE_MAX_SQ, dtype=torch.int32, device=weight.device)
        self.limits = self.capacity - self.steps

    def missing(self, S):
        """Which of S tokens behind each request's end have no slot: bool [B, S]."""
        if S > TREE_MAX_SQ:
            raise ValueError(f"at most {TREE_MAX_SQ} tokens of a request at once, got {S}")
        return self.lens[:, None] >= self.limits[:S]

    def where(self, at):
        """Page and slot of the tokens at [B, n] of each request; past the capacity, of its last one
        (an index outside the table would be a fault on the device)."""
        size, at = self.k[0].shape[2], at.clamp(max=self.capacity - 1)
        return self.table.gather(1, (at // size).long()).long(), (at % size).long()

    def rows(self, pages, at):
        """The cached rows of tokens at [B, n] of each request: [B, H, n, D]."""
        page, slot = self.where(at)
        return pages[page, :, slot].transpose(1, 2)


def _mlp(blk, x):
    return x + blk.out(F.gelu(blk.fc(blk.ln2(x)), approximate="tanh"))


def _embed(model, tokens):
    """Embeddings; a token below 0 (padding, an absent draft, nothing drawn) takes those of token
    0, since looking it up would be a fault on the device."""
    return model.emb(tokens.clamp(min=0))


def _logits(model, x):
    return F.linear(model.ln_f(x), model.emb.weight)


@torch.no_grad()
def prefill(model, cache, tokens, counts=None):
    """Run prompts [B, S] (``counts`` [B] int32 real tokens each; the rest is padding, which
    causality keeps away from them) and fill the empty cache.  Returns the logits after
    each prompt's last token, [B, V]: NaN for a request of no tokens, or of more than the
    cache holds (of which ``lens`` then counts those that entered)."""
    x = _embed(model, tokens)
    B, S, C = x.shape
    if S > cache.capacity and (counts is None or cache.rotary is not None):
        raise ValueError(f"prompts of {S} tokens, but the cache holds {cache.capacity} of each request")
    for layer, blk in enumerate(model.blocks):
        q, k, v = blk.attn.heads(blk.ln1(x))
        if cache.rotary is not None:
            cos, sin = (t[:S] for t in cache.rotary)
            q, k = rotate_heads(q, cos, sin), rotate_heads(k, cos, sin)
        append_paged_kv(k, v, cache.k[layer], cache.v[layer], cache.table, cache.lens, count=counts)
        y = blk.attn.attn_fn(q.contiguous(), k.contiguous(), v.contiguous(), causal=True, bias_max=model.cfg.bias_max)
        x = _mlp(blk, x + blk.attn.proj(y.transpose(1, 2).reshape(B, S, C)))
    if counts is None:
        cache.lens += S
        return _logits(model, x[:, -1])
    counts = counts.clamp(0, S)
    none = (counts == 0) | (counts > cache.capacity)
    cache.lens += counts.clamp(max=cache.capacity)
    x = x[torch.arange(B, device=x.device), (counts - 1).clamp(min=0).long()]
    return _logits(model, x.masked_fill(none[:, None], math.nan))


@torch.no_grad()
def extend(model, cache, tokens, words=None, depths=None, counts=None, missing=None):
    """Logits [B, S, V] of S <= 64 further tokens of each request, appended behind the cache
    (whose lengths stay: the caller says how many of them count).  ``words`` [B, S] int64:
    which of the new tokens each sees (default: those before it and itself);
    ``depths`` [B, S] int32: their distance from the cache's end, for the rotation; ``counts``
    [B] int32: how many enter the cache (default: all).  A token behind the cache's capacity
    has no key to see itself by: its logits are NaN (``sample_tokens`` draws -1 from them),
    and the operators report it by ``device_status()`` unless ``counts`` left it out.  The
    logits after a token below 0 are NaN too.  ``missing``: ``cache.missing(S)`` where the
    caller has it."""
    if missing is None:
        missing = cache.missing(tokens.shape[1])
    x = _extend(model, cache, tokens, words, depths, counts)
    return _logits(model, x.masked_fill((missing | (tokens < 0))[..., None], math.nan))


def _extend(model, cache, tokens, words=None, depths=None, counts=None):
    """The last layer's output of ``extend``."""
    x = _embed(model, tokens)
    B, S, C = x.shape
    positions = None if depths is None else cache.lens[:, None] + depths
    for layer, blk in enumerate(model.blocks):
        q, k, v = blk.attn.heads(blk.ln1(x))
        where = (cache.k[layer], cache.v[layer], cache.table, cache.lens)
        if cache.rotary is None:
            append_paged_kv(k, v, *where, count=counts)
        else:
            q = append_paged_kv(k, v, *where, count=counts, q=q, rotary=cache.rotary, positions=positions)
        y = paged_tree_attention(q, *where, tree_mask=words, bias_max=model.cfg.bias_max)
        x = _mlp(blk, x + blk.attn.proj(y.transpose(1, 2).reshape(B, S, C)))
    return x


def _noise(logits, generator):
    return torch.empty(logits.shape, device=logits.device).exponential_(generator=generator)


@torch.no_grad()
def generate(model, prompts, max_new_tokens, counts=None, generator=None, page_size=64, **sampling):
    """``max_new_tokens`` tokens for each prompt [B, S], [B, max_new_tokens].  ``sampling``:
    temperature, top_k, top_p and min_p of ``sample_tokens``."""
    if max_new_tokens <= 0:
        return torch.empty(prompts.shape[0], 0, dtype=torch.int64, device=prompts.device)
    cache = PagedCache(model, prompts.shape[0], prompts.shape[1] + max_new_tokens, page_size, spare=0)
    logits = prefill(model, cache, prompts, counts)
    out = []
    for _ in range(max_new_tokens):
        token, _ = sample_tokens(logits, _noise(logits, generator), **sampling)
        out.append(token)
        if len(out) < max_new_tokens:
            logits = _logits(model, _extend(model, cache, token[:, None])[:, 0])  # (the cache has room for all)
            cache.lens += 1
    out = torch.stack(out, 1)
    return out.masked_fill((out < 0).cummax(1)[0], -1)  # nothing follows where nothing could be drawn


def tree_words(parents):
    """Visibility words [B, T + 1] and depths [B, T + 1] of drafted trees: row 0 is the last
    accepted token, row 1 + t draft t, hung below row ``parents[b, t]`` of 0 .. t (else, -1
    say: no draft, its word is 0 and nothing of it is read)."""
    B, T = parents.shape
    if T + 1 > TREE_MAX_SQ:
        raise ValueError(f"at most {TREE_MAX_SQ - 1} drafted tokens, got {T}")
    words = torch.zeros(B, T + 1, dtype=torch.int64, device=parents.device)
    depths = torch.zeros(B, T + 1, dtype=torch.int32, device=parents.device)
    words[:, 0] = 1
    for t in range(T):
        up = parents[:, t:t + 1].long()
        bit = (1 << (t + 1)) if t + 1 < 63 else -(1 << 63)
        here, up = (up >= 0) & (up <= t), up.clamp(0, t)
        words[:, t + 1:t + 2] = torch.where(here, words.gather(1, up) | bit, 0)
        depths[:, t + 1:t + 2] = torch.where(here, depths.gather(1, up) + 1, 0)
    return words, depths


@torch.no_grad()
def tree_step(model, cache, last, drafts, parents, generator=None, **sampling):
    """Verify drafted trees: ``last`` [B] the newest token of each request (sampled, not yet in
    the cache), ``drafts`` [B, T] and ``parents`` [B, T] as in ``tree_words``.  A token is
    sampled after every row; from row 0 on, a draft that equals its parent's sample is
    accepted, and the first sample that no draft matches ends the step.  That draws from the
    model's own distribution whatever the drafts are.  Drafts behind the cache's capacity, and
    tokens below 0, count as none: the step ends before them.

    Returns (tokens [B, T + 1], n [B] int32): the first n[b] of tokens[b] are new, the last of
    them becomes ``last``.  The cache then holds every token before it.  A request whose cache is
    full already gets n = 0 and tokens of -1, and ``device_status()`` reports it."""
    B, T = drafts.shape
    missing = cache.missing(T + 1)
    parents = parents.masked_fill(missing[:, 1:] | (parents > cache.steps[:T]) | (drafts < 0), -1)
    words, depths = tree_words(parents)
    rows = torch.cat((last[:, None], drafts), 1)
    logits = extend(model, cache, rows, words, depths, cache.capacity - cache.lens, missing)
    flat = logits.flatten(0, 1)
    per_row = {k: v.repeat_interleave(T + 1) if isinstance(v, torch.Tensor) else v for k, v in sampling.items()}
    sampled = sample_tokens(flat, _noise(flat, generator), **per_row)[0].view(B, T + 1)
    # walk down: path[b, j] is the row of the j-th accepted token (row 0 first)
    path = torch.zeros(B, T + 1, dtype=torch.int64, device=drafts.device)
    tokens = sampled[:, :1].expand(B, T + 1).clone()
    n = torch.ones(B, dtype=torch.int32, device=drafts.device)
    at, alive = torch.zeros(B, 1, dtype=torch.int64, device=drafts.device), torch.ones(B, 1, dtype=torch.bool, device=drafts.device)
    for j in range(1, T + 1):
        match = (parents == at) & (drafts == sampled.gather(1, at))
        alive = alive & match.any(1, keepdim=True)
        at = torch.where(alive, match.int().argmax(1, keepdim=True) + 1, at)
        path[:, j:j + 1] = at
        tokens[:, j:j + 1] = sampled.gather(1, at)
        n += alive[:, 0].int()
    n.masked_fill_(missing[:, 0], 0)
    # the accepted rows move together behind the context; they are rotated already, by their depth
    page, slot = cache.where(cache.lens[:, None] + path.int())
    for k, v in zip(cache.k, cache.v):
        append_paged_kv(*(x[page, :, slot].transpose(1, 2) for x in (k, v)), k, v, cache.table, cache.lens, count=n)
    cache.lens += n
    return tokens, n
