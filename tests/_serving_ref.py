"""The serving operators from their definitions in 64 bits, request by request, and the
inputs their tests share.  CPU only, no code of the package."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half an ulp, relative


def pool(lens, Hkv, D, page, dtype, seed, token_major=False, spare=2):
    """Random pages, dealt out in random order, and the page table (-1 past a request's end)."""
    g = torch.Generator().manual_seed(seed)
    n_of = [-(-t // page) for t in lens]
    n, width = sum(n_of) + spare, max(1, max(n_of))
    order = torch.randperm(n, generator=g, dtype=torch.int32)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, m in enumerate(n_of):
        table[b, :m] = order[at:at + m]
        at += m
    shape = (n, page, Hkv, D) if token_major else (n, Hkv, page, D)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    return (k.transpose(1, 2), v.transpose(1, 2), table) if token_major else (k, v, table)


def gather(pages, table, b, n):
    """The first n tokens of request b: [Hkv, n, D]."""
    page = pages.shape[2]
    t = torch.arange(n, device=pages.device)
    return pages[table[b].long()[t // page], :, t % page].transpose(0, 1)


def tree(Sq, seed):
    """Ancestor words of a random tree, node t below one of the four nodes before it or below the context."""
    g, words = torch.Generator().manual_seed(seed), []
    for t in range(Sq):
        up = t - 1 - int(torch.randint(0, 4, (1,), generator=g))
        words.append((words[up] if up >= 0 else 0) | 1 << t)
    return words


def as_int64(words):
    return [w - (1 << 64) if w >> 63 else w for w in words]


def attention(q, k_pages, v_pages, table, ctx_lens, words, slopes, scale):
    """(o, P @ |V|), float64; words[b][i] is row i's visibility of the drafted tokens."""
    B, Hq, Sq, D = q.shape
    Hkv = k_pages.shape[1]
    o, pav = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        ctx = int(ctx_lens[b])
        for i in range(Sq):
            keys = list(range(ctx)) + [ctx + t for t in range(Sq) if words[b][i] >> t & 1]
            if not keys:
                continue
            at = torch.tensor(keys)
            k, v = (gather(x, table, b, keys[-1] + 1)[:, at].double() for x in (k_pages, v_pages))
            for h in range(Hq):
                kh, vh = k[h * Hkv // Hq], v[h * Hkv // Hq]
                p = scale * (kh @ q[b, h, i].double())
                z = torch.sigmoid(p).flip(0).cumsum(0).flip(0)
                w = torch.softmax(p - float(slopes[h]) * z, 0)
                o[b, h, i], pav[b, h, i] = w @ vh, w @ vh.abs()
    return o, pav


def rotated(x, angle_cos, angle_sin, interleaved):
    """x [..., D] float64 rotated by the angles [..., R / 2] of its rows."""
    r = angle_cos.shape[-1]
    y = x.clone()
    first = torch.arange(r) * 2 if interleaved else torch.arange(r)
    second = first + 1 if interleaved else first + r
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * angle_cos - b * angle_sin, b * angle_cos + a * angle_sin
    return y


def sample(logits, noise, temperature, top_k, top_p, min_p):
    """(tokens, logprobs, kept sets) in Python lists, row by row."""
    tokens, logprobs, kepts = [], [], []
    for b in range(logits.shape[0]):
        x = logits[b].double()
        x = torch.where(x.isnan(), -math.inf, x)
        t, k, p, least = temperature[b], top_k[b], top_p[b], min_p[b]
        m = x.max()
        if m == -math.inf:
            tokens.append(-1), logprobs.append(-math.inf), kepts.append([])
            continue
        order = torch.argsort(x, descending=True, stable=True)
        if not t > 0:
            tokens.append(int(order[0])), logprobs.append(0.0), kepts.append([int(order[0])])
            continue
        d = torch.where(x == m, torch.zeros_like(x), (x - m) / t)
        order = order[d[order] > -100]  # exp of less is 0 in float32
        if 0 < k < len(order):
            order = order[:k]
        w = d[order].exp()
        if p < 1:
            n = max(1, int((w.cumsum(0) - w < p * w.sum()).sum()))
            order, w = order[:n], w[:n]
        n = max(1, int((w >= least).sum()))
        order, w = order[:n], w[:n]
        score = w / noise[b][order].double()
        best = max(range(n), key=lambda r: (float(score[r]), -int(order[r])))
        tokens.append(int(order[best]))
        logprobs.append(float(d[order[best]] - w.sum().log()))
        kepts.append(order.tolist())
    return tokens, logprobs, kepts
