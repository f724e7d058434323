"""Query, key and value heads out of a fused projection, queries and keys normed per head and
rotated by their position in the same pass, with its gradient.  The reference ships the
attention operator alone (``co_alibi_attn/co_alibi_attn.py:137-148``) and has no counterpart.
"""
import torch
from torch.autograd.function import once_differentiable

from .co_alibi_attn import _status_word
from .serving import _native

__all__ = ["norm_rotate_qkv"]


def _requires_grad(t):
    return isinstance(t, torch.Tensor) and t.requires_grad


class _NormRotateQKV(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, num_heads, num_kv_heads, eps, rotary, start, positions, interleaved):
        status = _status_word(qkv.device)
        q, k, v = _native().heads_fwd(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps, rotary, start, positions,
                                      interleaved, status)
        cos, sin = rotary if rotary is not None else (None, None)
        ctx.save_for_backward(qkv, q_weight, k_weight, cos, sin, start, positions)
        ctx.args = num_heads, num_kv_heads, eps, interleaved
        return q, k, v

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        qkv, q_weight, k_weight, cos, sin, start, positions = ctx.saved_tensors
        num_heads, num_kv_heads, eps, interleaved = ctx.args
        d, dqw, dkw = _native().heads_bwd(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps,
                                          None if cos is None else (cos, sin), start, positions, interleaved,
                                          _status_word(qkv.device), dq, dk, dv)
        return d, dqw, dkw, None, None, None, None, None, None, None


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
    repeat bit for bit); tables that require one are refused, and there is no second derivative."""
    assert qkv.is_cuda, "Inputs must be CUDA tensors"
    if not torch.is_grad_enabled() or not (qkv.requires_grad or _requires_grad(q_weight) or _requires_grad(k_weight)):
        return _native().heads_fwd(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps, rotary, start, positions,
                                   interleaved, _status_word(qkv.device))
    if rotary is not None and any(_requires_grad(t) for t in rotary):
        raise RuntimeError("co_alibi_attn: norm_rotate_qkv: the rotary tables require grad, but get none")
    return _NormRotateQKV.apply(qkv, q_weight, k_weight, num_heads, num_kv_heads, eps, rotary, start, positions,
                                interleaved)
