"""Serving a Co-ALiBi model: the operators of a decoding step over a paged key/value
cache.  The reference ships the attention operator alone
(``co_alibi_attn/co_alibi_attn.py:137-148``) and has no counterpart of these.

* ``append_paged_kv``: write new keys and values into the cache, rotating keys and
  queries on the way for models that add rotary positions to the Co-ALiBi bias.
* ``paged_tree_attention``: Co-ALiBi attention of one token, or of a tree of drafted
  tokens, per request over that cache.
* ``read_paged_kv``: tokens of a cache that is held in 8 bits, in 16 bits again.
* ``sample_tokens``: temperature, top-k, top-p and min-p, and a draw by given random
  numbers.

A cache is a pair of pools ``k_pages``, ``v_pages`` [n_pages, Hkv, page_size, D]
(float16 or bfloat16, any strides with contiguous rows, so a permuted token-major
pool works too; page_size a multiple of 16) and an int32 ``page_table``
[B, max_pages]: token t of request b is slot ``t % page_size`` of page
``page_table[b, t // page_size]``.  Lengths and tables live on the device and are read
there: calls launch on the current stream, never synchronise, and can be captured in a
CUDA graph, after one call outside (the first on a device, or of a number of heads, builds
what is kept, and a capture refuses it).  A token whose page is outside the pool, or past the table, is skipped and
reported by ``device_status()`` as code 11; one whose position has no row in the rotary
tables is stored unrotated and reported too.

A cache may be held in 8 bits: pools of ``torch.float8_e4m3fn`` (D a multiple of 16, strides
too) with ``scales`` = (k_scales, v_scales), float32 [n_pages, Hkv, page_size / 16], one for each
block of 16 tokens of a page and head.  A value is its code times the scale of its block.
``append_paged_kv`` writes scales that are powers of two, the least by which a block's largest
value is at most 448 (and at least 2^-100): a code's relative error is at most 2^-4 then, or 2^-10 of the scale, that is
less than 2^-17 of the block's largest, for what is smaller.  A block that already holds tokens keeps its scale unless
a new one is too large for it, and if so the old codes move to the new scale, which changes none but
those that fall below 2^-6 of it.  Reading and attention take scales that another program wrote as well: any finite ones, 0
and negative ones among them (attention's weights of values in blocks below 2^-100 are rounded as those of 2^-100).  Slots behind a request's tokens hold nothing, and those before ``start`` in
its block hold tokens; as the block's codes may move, no other request writes or reads the block in the same call.

There is no backward: where gradients are enabled, keys, values, queries and pools that
require one are refused (call under ``torch.no_grad()``), forward-mode tangents of theirs too, and log-probabilities of sampled
tokens carry none.  Appending counts as an in-place write of the pools for autograd.
"""
import torch

from .co_alibi_attn import _api_slopes, _status_word

__all__ = ["append_paged_kv", "paged_tree_attention", "read_paged_kv", "sample_tokens", "rotary_tables", "TREE_MAX_SQ",
           "QUANT_BLOCK"]

TREE_MAX_SQ = 64  # COALIBI_TREE_MAX_SQ in coalibi.h
QUANT_BLOCK = 16  # COALIBI_QUANT_BLOCK: tokens that share a scale in a cache of 8 bits

_binding = None


def _native():
    """The compiled binding (csrc/binding.cpp): argument checks, allocation and launch."""
    global _binding
    if _binding is None:
        try:
            from . import _serving
        except ImportError as e:
            raise RuntimeError("co_alibi_attn: the serving binding is not built (or PyTorch changed since); build it with "
                               f"`python co-alibi_b200/build.py` (no CPU fallback exists): {e}") from e
        _binding = _serving
    return _binding


def rotary_tables(rotary_dim, max_pos, base=10000.0, scale=1.0, device=None):
    """(cos, sin), float32 [max_pos, rotary_dim / 2]: angle(p, i) = p / scale *
    base ** (-2 i / rotary_dim), computed in float64.  ``scale`` > 1 squeezes long
    contexts into the trained range (linear interpolation)."""
    if rotary_dim <= 0 or rotary_dim % 2 or max_pos <= 0 or scale <= 0:
        raise ValueError("co_alibi_attn: rotary_tables: rotary_dim must be even and positive, max_pos and scale positive")
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] / scale * f
    return a.cos().float().to(device), a.sin().float().to(device)


def append_paged_kv(k, v, k_pages, v_pages, page_table, start, count=None, q=None, rotary=None, interleaved=False,
                    positions=None, scales=None):
    """Write the new tokens' keys and values into the cache, in place.

    k, v: [B, Hkv, S, D] (any strides with contiguous rows, e.g. views of a fused
    projection).  Token i of request b goes to position ``start[b] + i`` (``start``
    int32 [B]) for i < ``count[b]`` (int32 [B]; default S); the rest of a ragged batch is
    padding and is not read.

    ``rotary``: (cos, sin) tables, float32 [n_pos, R / 2], R a multiple of 16 up to D:
    the first R elements of each key are rotated before they are stored, in halves
    (x[i], x[i + R/2]) or ``interleaved`` pairs (x[2i], x[2i + 1]), by the row of the
    tables at the token's position, or at ``positions`` (int32 [B, S]; a drafted tree's
    tokens sit at their depth, not at their slot).  With ``q`` [B, Hq, S, D] the queries
    are rotated in the same launch and returned (rows past ``count`` are zero); without,
    None is returned.  Rotations are float32, rounded once; all else is moved as it is.

    ``scales``: those of a cache in 8 bits, written with it.  Keys (rotated in float32) and values
    are rounded once, to the nearest code of their block, ties to the even one; infinities become NaN."""
    assert k.is_cuda, "Inputs must be CUDA tensors"
    return _native().append_paged_kv(k, v, k_pages, v_pages, page_table, start, count, q, rotary, interleaved,
                                     positions, _status_word(k.device), scales)


def paged_tree_attention(q, k_pages, v_pages, page_table, ctx_lens, tree_mask=None, sm_scale=None, bias_max=8.0,
                         slopes=None, scales=None):
    """Co-ALiBi attention of each request's Sq query rows over its cache (forward only).

    q: [B, Hq, Sq, D], Sq <= 64, Hq a multiple of the cache's Hkv.  Every row sees the
    ``ctx_lens[b]`` (int32 [B]) first tokens of the request; the Sq drafted tokens, already
    appended behind them, are seen by the bits of ``tree_mask`` (int64 [B, Sq], or
    [Sq] for all requests): row i sees drafted token t where bit t of its word is set, so
    a row's word holds its ancestors and itself.  Default: a chain (bits 0 .. i), which
    for Sq = 1 is one decoding step.  A request with fewer drafts leaves its last rows'
    words 0, and drafts that no word names are not read.

    Per row: p = sm_scale * q.k, z_j = the sum of sigmoid(p) over the keys the row sees at
    j and after it in cache order, o = softmax(p - slope * z) V; scale, slopes and
    ``bias_max`` as in ``co_alibi_attention`` (``slopes`` [Hq] replaces its table, e.g. for
    a head shard).  Returns [B, Hq, Sq, D]; a row that sees nothing is zero.

    Scores, sigmoid sums, softmax statistics and the result's sums are float32 (with the
    hardware's approximate exponential and reciprocal); the weights are rounded to the
    inputs' type for the product with V, as in ``co_alibi_attention``.

    ``scales``: those of a cache in 8 bits.  Its products take the codes as float16, which holds them
    whole (bfloat16 queries too, each row by a power of two), and the weights as float16."""
    assert q.is_cuda, "Inputs must be CUDA tensors"
    if slopes is None:
        slopes = _api_slopes(q.shape[1], bias_max, q.dtype, q.device)
    return _native().paged_tree_attention(q, k_pages, v_pages, page_table, ctx_lens, tree_mask, sm_scale, slopes,
                                          _status_word(q.device), scales)


_READ_DTYPES = {torch.float16: False, torch.bfloat16: True}


def read_paged_kv(k_pages, v_pages, page_table, positions, scales, dtype=torch.bfloat16):
    """Tokens of a cache in 8 bits, as (k, v) [B, Hkv, S, D] of ``dtype`` (float16 or bfloat16).

    ``positions`` int32 [B, S]: which tokens of each request, in any order, the same one as often
    as asked for; a negative one gives a row of zeros, and so does one without a page, which is
    reported.  Values are rounded once; one past the type's largest is that.  What the append wrote is
    whole in bfloat16 (up to its largest), and in float16 under scales from 2^-15 to 2^7.  A token that is read whole and
    appended again has the same values, and under a scale as large as its old one the same codes; a larger scale rounds
    it like any other."""
    assert k_pages.is_cuda, "Inputs must be CUDA tensors"
    if dtype not in _READ_DTYPES:
        raise TypeError(f"co_alibi_attn: read_paged_kv: dtype must be float16 or bfloat16, got {dtype}")
    return _native().read_paged_kv(k_pages, v_pages, page_table, positions, scales, _READ_DTYPES[dtype],
                                   _status_word(k_pages.device))


def sample_tokens(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draw a token for each row of ``logits`` [B, V] (float16, bfloat16 or float32).

    Tokens are ranked by logit, equal ones by index, and weighted
    w = exp((logit - max) / temperature).  Kept are the first ``top_k`` (0: all), of those
    the shortest prefix whose weights reach ``top_p`` of their sum (1: all; at least one
    stays), of those the ones with w >= ``min_p``.  The token drawn is the kept one with
    the largest w / noise: with ``noise`` [B, V] float32 drawn from Exp(1)
    (``torch.empty(B, V, device="cuda").exponential_()``) that samples the renormalised
    distribution, and equal inputs always give equal tokens.  ``temperature`` 0 takes the
    first of the ranking.  Each parameter is a number or a tensor [B] (float32; ``top_k``
    int32).  Logits of -inf or NaN are never drawn; a row of nothing else gives token -1.

    Returns (tokens int64 [B], logprobs float32 [B]: the drawn token's log-probability
    among the kept).  Weights are float32 with a relative error of up to 2e-5: a token whose
    weight, or the mass before it, lies that close to a limit may fall on either side of it."""
    assert logits.is_cuda, "Inputs must be CUDA tensors"
    return _native().sample_tokens(logits, noise, temperature, top_k, top_p, min_p)
