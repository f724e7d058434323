"""Serving a Co-ALiBi model: the operators of a decoding step over a paged key/value
cache.  The reference ships the attention operator alone
(``co_alibi_attn/co_alibi_attn.py:137-148``) and has no counterpart of these.

* ``append_paged_kv``: write new keys and values into the cache, rotating keys and
  queries on the way for models that add rotary positions to the Co-ALiBi bias.
* ``paged_tree_attention``: Co-ALiBi attention of one token, or of a tree of drafted
  tokens, per request over that cache.
* ``sample_tokens``: temperature, top-k, top-p and min-p, and a draw by given random
  numbers.

A cache is a pair of pools ``k_pages``, ``v_pages`` [n_pages, Hkv, page_size, D]
(float16 or bfloat16, any strides with contiguous rows, so a permuted token-major
pool works too; page_size a multiple of 16) and an int32 ``page_table``
[B, max_pages]: token t of request b is slot ``t % page_size`` of page
``page_table[b, t // page_size]``.  Lengths and tables live on the device and are read
there: calls launch on the current stream, never synchronise, and can be captured in a
CUDA graph.  A token whose page is outside the pool, or past the table, is skipped and
reported by ``device_status()`` as code 11.
"""
import struct

import torch

from . import _lib
from .co_alibi_attn import _DTYPES, _SLOPE_DTYPES, _api_slopes, _status_word

__all__ = ["append_paged_kv", "paged_tree_attention", "sample_tokens", "rotary_tables", "TREE_MAX_SQ"]

TREE_MAX_SQ = 64  # COALIBI_TREE_MAX_SQ in coalibi.h

# The argument structs of coalibi.h, packed straight from Python integers (the layout
# of the ctypes structures in _lib, without their per-field cost on every call).
_APPEND = struct.Struct("@13P 18q q 12i 0q")
_ATTN = struct.Struct("@9P 12q 2q 10i f 0q")
_SAMPLE = struct.Struct("@8P 2q 3i f i 2f 0q")


def _check_cache(what, k_pages, v_pages, page_table, B, D, dtype, device):
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError(f"co_alibi_attn: {what}: k_pages and v_pages must both be [n_pages, Hkv, page_size, D], got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise TypeError(f"co_alibi_attn: {what}: the cache holds {k_pages.dtype}/{v_pages.dtype}, the inputs {dtype}")
    if k_pages.shape[3] != D:
        raise ValueError(f"co_alibi_attn: {what}: the cache has head_dim {k_pages.shape[3]}, the inputs {D}")
    if k_pages.shape[2] % 16 != 0 or k_pages.numel() == 0:
        raise ValueError(f"co_alibi_attn: {what}: page_size must be a positive multiple of 16 and the pool not empty, "
                         f"got {tuple(k_pages.shape)}")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if not _rows16(t):
            raise ValueError(f"co_alibi_attn: {what}: {name} must have contiguous, 16-byte aligned rows")
        if 0 in (s for s, n in zip(t.stride(), t.shape) if n > 1):
            raise ValueError(f"co_alibi_attn: {what}: {name} must not be an expanded tensor")
    if page_table.dtype != torch.int32:
        raise TypeError(f"co_alibi_attn: {what}: page_table must be int32, got {page_table.dtype}")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.shape[1] == 0 or page_table.stride(1) != 1:
        raise ValueError(f"co_alibi_attn: {what}: page_table must be [{B}, max_pages] with contiguous rows, got "
                         f"{tuple(page_table.shape)}")
    if page_table.shape[1] * k_pages.shape[2] > 0x7fffff00:
        raise ValueError(f"co_alibi_attn: {what}: a page table row must hold fewer than 2**31 tokens")
    _on(what, device, k_pages, v_pages, page_table)


def _on(what, device, *tensors):
    for t in tensors:
        if t.device != device:
            raise ValueError(f"co_alibi_attn: {what}: tensors on {t.device} and {device}")


def _rows16(t):
    """Whether every row of t [., ., ., D] is contiguous and 16-byte aligned."""
    s = _strides(t)
    return t.stride(3) == 1 and not (s[0] | s[1] | s[2]) & 7 and t.data_ptr() % 16 == 0


def _strides(t):
    """The first three strides of t, 0 for a dimension of one entry (PyTorch may report any there)."""
    n, s = t.shape, t.stride()
    return s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0


def _aligned_rows(t):
    return t if _rows16(t) else t.clone(memory_format=torch.contiguous_format)


def _ints(what, name, t, shape, dtype, device):
    if t.dtype != dtype:
        raise TypeError(f"co_alibi_attn: {what}: {name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"co_alibi_attn: {what}: {name} must have shape {shape}, got {tuple(t.shape)}")
    _on(what, device, t)
    return t.contiguous()


def _call(device, fn, what, *args):
    """Launch on the device's current stream; the library binds the device itself."""
    _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream), what)


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
                    positions=None):
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
    None is returned."""
    what = "append_paged_kv"
    assert k.is_cuda, "Inputs must be CUDA tensors"
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"co_alibi_attn: {what}: k and v must both be [B, Hkv, S, D], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    B, Hkv, S, D = k.shape
    dtype, device = k.dtype, k.device
    if dtype not in _DTYPES or v.dtype != dtype or (q is not None and q.dtype != dtype):
        raise TypeError(f"co_alibi_attn: {what}: k, v and q must all be float16 or bfloat16, got {k.dtype}/{v.dtype}")
    if D not in (64, 128):
        raise ValueError(f"co_alibi_attn: {what}: head_dim must be 64 or 128, got {D}")
    _check_cache(what, k_pages, v_pages, page_table, B, D, dtype, device)
    if k_pages.shape[1] != Hkv:
        raise ValueError(f"co_alibi_attn: {what}: the cache has {k_pages.shape[1]} kv heads, k {Hkv}")
    _on(what, device, v)
    if B == 0 or S == 0:
        return None if q is None else torch.empty_like(q)
    start = _ints(what, "start", start, (B,), torch.int32, device)
    if count is not None:
        count = _ints(what, "count", count, (B,), torch.int32, device)
    if positions is not None:
        positions = _ints(what, "positions", positions, (B, S), torch.int32, device)
    k = _aligned_rows(k)
    v = _aligned_rows(v)
    Hq, q_out, qs, qos = 0, None, (0, 0, 0), (0, 0, 0)
    if q is not None:
        if q.dim() != 4 or q.shape[0] != B or q.shape[2] != S or q.shape[3] != D:
            raise ValueError(f"co_alibi_attn: {what}: q must be [{B}, Hq, {S}, {D}], got {tuple(q.shape)}")
        _on(what, device, q)
        q = _aligned_rows(q)
        Hq, q_out = q.shape[1], torch.empty_like(q)
        qs, qos = _strides(q), _strides(q_out)
    cos = sin = None
    rot = n_pos = 0
    if rotary is not None:
        cos, sin = rotary
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise TypeError(f"co_alibi_attn: {what}: the rotary tables must be float32")
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] == 0 or cos.shape[1] % 8 or \
                not 0 < 2 * cos.shape[1] <= D:
            raise ValueError(f"co_alibi_attn: {what}: the rotary tables must be [n_pos, R / 2] with R a multiple of 16 "
                             f"up to {D}, got {tuple(cos.shape)} and {tuple(sin.shape)}")
        _on(what, device, cos, sin)
        cos, sin = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                    for t in (cos, sin))
        n_pos, rot = cos.shape[0], 2 * cos.shape[1]
    args = _APPEND.pack(
        k.data_ptr(), v.data_ptr(), q.data_ptr() if q is not None else 0, q_out.data_ptr() if q is not None else 0,
        k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), start.data_ptr(),
        count.data_ptr() if count is not None else 0, positions.data_ptr() if positions is not None else 0,
        cos.data_ptr() if rot else 0, sin.data_ptr() if rot else 0, _status_word(device).data_ptr(),
        *_strides(k), *_strides(v), *qs, *qos, *_strides(k_pages), *_strides(v_pages),
        page_table.stride(0), B, Hq, Hkv, S, D, k_pages.shape[2], page_table.shape[1], k_pages.shape[0],
        rot, n_pos, 1 if interleaved else 0, _DTYPES[dtype])
    _call(device, _lib.load().coalibi_paged_append, "coalibi_paged_append", args)
    return q_out


def paged_tree_attention(q, k_pages, v_pages, page_table, ctx_lens, tree_mask=None, sm_scale=None, bias_max=8.0,
                         slopes=None):
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
    a head shard).  Returns [B, Hq, Sq, D]; a row that sees nothing is zero."""
    what = "paged_tree_attention"
    assert q.is_cuda, "Inputs must be CUDA tensors"
    if q.dim() != 4:
        raise ValueError(f"co_alibi_attn: {what}: q must be [B, Hq, Sq, D], got {tuple(q.shape)}")
    B, Hq, Sq, D = q.shape
    dtype, device = q.dtype, q.device
    if dtype not in _DTYPES:
        raise TypeError(f"co_alibi_attn: {what}: q must be float16 or bfloat16, got {dtype}")
    if D not in (64, 128):
        raise ValueError(f"co_alibi_attn: {what}: head_dim must be 64 or 128, got {D}")
    if Sq > TREE_MAX_SQ:
        raise ValueError(f"co_alibi_attn: {what}: at most {TREE_MAX_SQ} rows per request, got {Sq}")
    _check_cache(what, k_pages, v_pages, page_table, B, D, dtype, device)
    Hkv = k_pages.shape[1]
    if Hq % Hkv != 0:
        raise ValueError(f"co_alibi_attn: {what}: num_heads {Hq} must be a multiple of num_kv_heads {Hkv}")
    if q.numel() == 0:
        return torch.empty_like(q)
    ctx_lens = _ints(what, "ctx_lens", ctx_lens, (B,), torch.int32, device)
    mask_stride = 0
    if tree_mask is not None:
        shape = (Sq,) if tree_mask.dim() == 1 else (B, Sq)
        tree_mask = _ints(what, "tree_mask", tree_mask, shape, torch.int64, device)
        mask_stride = Sq if tree_mask.dim() == 2 else 0
    if slopes is None:
        slopes = _api_slopes(Hq, bias_max, dtype, device)
    else:
        if slopes.dtype not in _SLOPE_DTYPES:
            raise TypeError(f"co_alibi_attn: {what}: slopes must be float16/bfloat16/float32, got {slopes.dtype}")
        if tuple(slopes.shape) != (Hq,):
            raise ValueError(f"co_alibi_attn: {what}: slopes must have shape ({Hq},), got {tuple(slopes.shape)}")
        _on(what, device, slopes)
        slopes = slopes.contiguous()
    q = _aligned_rows(q)
    o = torch.empty_like(q)
    lib = _lib.load()
    nbytes = lib.coalibi_paged_attention_workspace_bytes(B, Hq, Hkv, Sq, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    args = _ATTN.pack(
        q.data_ptr(), o.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), slopes.data_ptr(), page_table.data_ptr(),
        ctx_lens.data_ptr(), tree_mask.data_ptr() if tree_mask is not None else 0, _status_word(device).data_ptr(),
        *_strides(q), *_strides(o), *_strides(k_pages), *_strides(v_pages), page_table.stride(0),
        mask_stride, B, Hq, Hkv, Sq, D, k_pages.shape[2], page_table.shape[1], k_pages.shape[0], _DTYPES[dtype],
        _SLOPE_DTYPES[slopes.dtype], sm_scale if sm_scale is not None else D ** -0.5)
    _call(device, lib.coalibi_paged_attention, "coalibi_paged_attention", args, ws.data_ptr(), nbytes)
    return o


def _per_row(name, value, B, dtype, device):
    """(pointer, scalar) of a sampling parameter given as a number or a tensor [B]."""
    if isinstance(value, torch.Tensor):
        t = _ints("sample_tokens", name, value, (B,), dtype, device)
        return t, t.data_ptr(), 0
    return None, 0, value


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
    among the kept)."""
    what = "sample_tokens"
    assert logits.is_cuda, "Inputs must be CUDA tensors"
    if logits.dim() != 2 or noise.shape != logits.shape:
        raise ValueError(f"co_alibi_attn: {what}: logits and noise must both be [B, V], got {tuple(logits.shape)} and "
                         f"{tuple(noise.shape)}")
    if logits.dtype not in _SLOPE_DTYPES or noise.dtype != torch.float32:
        raise TypeError(f"co_alibi_attn: {what}: logits must be float16/bfloat16/float32 and noise float32, got "
                        f"{logits.dtype} and {noise.dtype}")
    B, V = logits.shape
    device = logits.device
    _on(what, device, noise)
    if V == 0 or V > 1 << 21:
        raise ValueError(f"co_alibi_attn: {what}: the vocabulary must have 1 to 2**21 tokens, got {V}")
    logits = logits if logits.stride(1) == 1 else logits.contiguous()
    noise = noise if noise.stride(1) == 1 else noise.contiguous()
    tokens = torch.empty(B, dtype=torch.int64, device=device)
    logprobs = torch.empty(B, dtype=torch.float32, device=device)
    if B == 0:
        return tokens, logprobs
    t0, tp, ts = _per_row("temperature", temperature, B, torch.float32, device)
    k0, kp, ks = _per_row("top_k", top_k, B, torch.int32, device)
    p0, pp, ps = _per_row("top_p", top_p, B, torch.float32, device)
    m0, mp, ms = _per_row("min_p", min_p, B, torch.float32, device)
    args = _SAMPLE.pack(logits.data_ptr(), noise.data_ptr(), tp, kp, pp, mp, tokens.data_ptr(), logprobs.data_ptr(),
                        logits.stride(0), noise.stride(0), B, V, _SLOPE_DTYPES[logits.dtype], ts, ks, ps, ms)
    _call(device, _lib.load().coalibi_sample, "coalibi_sample", args)
    return tokens, logprobs
