"""Query, key and value heads out of a fused projection, queries and keys normed per head and
rotated by their position in the same pass, with its gradient.  The reference ships the
attention operator alone (``co_alibi_attn/co_alibi_attn.py:137-148``) and has no counterpart.
"""
from .co_alibi_attn import _status_word
from .serving import _native

__all__ = ["norm_rotate_qkv"]


def norm_rotate_qkv(qkv, num_heads, num_kv_heads, q_weight=None, k_weight=None, eps=1e-6, rotary=None, start=None,
                    positions=None, interleaved=False):
    """(q [B, num_heads, S, D], k, v [B, num_kv_heads, S, D]), contiguous, out of ``qkv``
    [B, S, num_heads + 2 num_kv_heads, D] (float16 or bfloat16, D 64 or 128, any strides with contiguous
    rows): the heads of each token as a fused projection leaves them, queries, keys, values.

    A row x of a query or key head becomes x / sqrt(mean(x^2) + eps) * weight, ``q_weight`` and
    ``k_weight`` [D] (of qkv's type, or float32; None: ones), and its first R elements are rotated
    by ``rotary``: (cos, sin) tables, float32 [n_pos, R / 2], R a multiple of 16 up to D, in halves
    (x[i], x[i + R/2]) or ``interleaved`` pairs, by the row of the tables at the token's position:
    ``positions`` (int32 [B, S]), else ``start`` (int32 [B]) + i, else i.  A position outside the
    tables leaves the row unrotated and is reported by ``device_status()`` as code 11.  Values are
    moved as they are.  Arithmetic is float32, rounded once.

    Gradients reach ``qkv`` and the weights (the weights' sums are float32, added in a fixed order: results
    repeat bit for bit); tables that require one are refused, and there is neither a second
    derivative nor a forward-mode one (tangents are refused).  A
    backward that is captured in a CUDA graph takes leaves (or detached copies) of which no eager graph lives: the leaf's
    accumulation belongs to the stream of the first."""
    assert qkv.is_cuda, "Inputs must be CUDA tensors"
    return _native().norm_rotate_qkv(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps, rotary, start, positions,
                                     interleaved, _status_word(qkv.device))
