"""Plain torch forms of the serving operators for CPU tensors: they stand in for the kernels
where a test is about the generation path's own bookkeeping.  A token without a slot or an
angle is skipped and noted in ``reports``, as the kernels skip and report it."""
import math

import torch

from tests import _serving_ref as ref

reports = []


def append_paged_kv(k, v, k_pages, v_pages, page_table, start, count=None, q=None, rotary=None, interleaved=False,
                    positions=None):
    B, _, S, _ = k.shape
    page = k_pages.shape[2]
    q_out = None if q is None else torch.zeros_like(q)
    for b in range(B):
        for i in range(S if count is None else min(S, int(count[b]))):
            t = int(start[b]) + i
            at = int(positions[b, i]) if positions is not None else t
            kk, qq = k[b, :, i], None if q is None else q[b, :, i]
            if rotary is not None:
                if at < rotary[0].shape[0]:
                    turn = lambda x: ref.rotated(x.double(), rotary[0][at].double(), rotary[1][at].double(),  # noqa: E731
                                                 interleaved).to(x.dtype)
                    kk, qq = turn(kk), None if q is None else turn(qq)
                else:
                    reports.append(("angle", b, i))
            if q is not None:
                q_out[b, :, i] = qq
            if t >= page_table.shape[1] * page:
                reports.append(("append", b, i))
                continue
            k_pages[page_table[b, t // page], :, t % page] = kk
            v_pages[page_table[b, t // page], :, t % page] = v[b, :, i]
    return q_out


def paged_tree_attention(q, k_pages, v_pages, page_table, ctx_lens, tree_mask=None, sm_scale=None, bias_max=8.0,
                         slopes=None):
    from co_alibi_attn.co_alibi_attn import _api_slopes
    B, Hq, Sq, D = q.shape
    room = page_table.shape[1] * k_pages.shape[2]
    words = [[(2 << i) - 1 for i in range(Sq)]] * B if tree_mask is None else tree_mask.tolist()
    inside = []
    for b in range(B):
        fit = (1 << max(0, min(Sq, room - int(ctx_lens[b])))) - 1
        if any(w & ((1 << Sq) - 1) & ~fit for w in words[b]) or int(ctx_lens[b]) > room:
            reports.append(("attend", b))
        inside.append([w & fit for w in words[b]])
    o, _ = ref.attention(q, k_pages, v_pages, page_table, ctx_lens.clamp(max=room), inside,
                         _api_slopes(Hq, bias_max, q.dtype, q.device) if slopes is None else slopes,
                         sm_scale or 1 / math.sqrt(D))
    return o.to(q.dtype)


def sample_tokens(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = lambda x: x.tolist() if isinstance(x, torch.Tensor) else [x] * logits.shape[0]  # noqa: E731
    tokens, logprobs, _ = ref.sample(logits, noise, rows(temperature), rows(top_k), rows(top_p), rows(min_p))
    return torch.tensor(tokens), torch.tensor(logprobs)


def stand_in(monkeypatch):
    """Replaces the operators that ``co_alibi_gpt.generate`` calls; returns that module."""
    from co_alibi_gpt import generate
    reports.clear()
    for f in (append_paged_kv, paged_tree_attention, sample_tokens):
        monkeypatch.setattr(generate, f.__name__, f)
    return generate
