"""The serving operators of a Co-ALiBi model: what a decoding step runs beside its matrix products.

  append     new keys and values into a paged cache, queries and keys rotated on the way
  attention  Co-ALiBi attention of one token, or of a tree of drafted tokens, over that cache
  sample     the next tokens from the logits: temperature, top-k, top-p, min-p, a race of given random numbers

``run`` computes them in their plain form (torch, 32 bits), or with ``own`` set through the package's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}

# ---------------------------------------------------------------------------------------------------------------------
# Cases.  Head counts, widths and the vocabulary are those of the repository's own configurations (H16 D128; Hq32 Hkv8
# D128; 12 heads of 64 and 50304 tokens); 131072 and 32001 stand for a large and an odd vocabulary.
# ---------------------------------------------------------------------------------------------------------------------


def _append(name, B, Hq, Hkv, D, S, lo, hi, page, dtype, rot, interleaved, full):
    return {"name": name, "op": "append", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "S": S, "lo": lo, "hi": hi, "page": page, "dtype": dtype, "rot": rot,
            "interleaved": interleaved, "full": full}


def _attention(name, B, Hq, Hkv, D, Sq, lo, hi, page, dtype):
    return {"name": name, "op": "attention", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "Sq": Sq, "lo": lo, "hi": hi, "page": page, "dtype": dtype}


def _sample(name, B, V, dtype, temperature, top_k, top_p, min_p, mixed):
    return {"name": name, "op": "sample", "B": B, "V": V, "dtype": dtype, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed}


def listed():
    return [
        # one token of each of a few requests of the small GPT, no rotation: the call's latency is all there is
        _append("append gpt token", 4, 12, 12, 64, 1, 1, 900, 16, "bf16", 0, False, True),
        # a decoding step of a large batch with grouped heads, the whole head rotated, lengths all different
        _append("append decode batch", 256, 32, 8, 128, 1, 0, 500, 16, "bf16", 128, False, True),
        # prompts of ragged lengths entering the cache, half of each head rotated in interleaved pairs
        _append("append ragged prompts", 8, 32, 8, 128, 2000, 3, 0, 64, "f16", 64, True, False),
        # one token of one short chat of the small GPT
        _attention("attend one short", 1, 12, 12, 64, 1, 36, 36, 16, "f16"),
        # a decoding step of a batch of grouped heads, from empty caches to 8192 tokens
        _attention("attend decode batch", 16, 32, 8, 128, 1, 0, 8191, 64, "bf16"),
        # a few long documents, one token each: the largest reads
        _attention("attend long", 4, 32, 8, 128, 1, 65537, 131071, 64, "bf16"),
        # verifying trees of 16 drafted tokens over grouped heads: 64 rows share each key
        _attention("attend tree 16", 8, 32, 8, 128, 16, 127, 16383, 32, "bf16"),
        # the widest trees over ungrouped heads
        _attention("attend tree 64", 2, 16, 16, 128, 64, 1000, 4096, 16, "f16"),
        # one row, the usual top-k of a chat
        _sample("sample one", 1, 50304, "bf16", 0.8, 50, 1.0, 0.0, False),
        # a batch whose requests each ask for something else: greedy ones, top-k, top-p and min-p together
        _sample("sample mixed batch", 64, 50304, "f32", 0.9, 64, 0.9, 0.02, True),
        # nucleus sampling alone over an odd vocabulary: thousands of tokens stay
        _sample("sample nucleus", 300, 32001, "f16", 1.3, 0, 0.95, 0.0, False),
        # no filter at all, a large batch over a large vocabulary: two long reads
        _sample("sample unfiltered", 256, 131072, "f32", 1.0, 0, 1.0, 0.0, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "sample"])
    Hq, Hkv, D = rng.choice([(12, 12, 64), (16, 16, 128), (32, 8, 128), (8, 1, 128), (12, 4, 64)])
    page, dtype = rng.choice([16, 32, 48, 64, 128]), rng.choice(["f16", "bf16"])
    if op == "append":
        if rng.random() < 0.5:
            B, S = _log(rng, 1, 256), rng.choice([1, 1, 2, 5])
            lo, hi = 0, _log(rng, 8, 500)
        else:
            B, S = _log(rng, 1, 8), _log(rng, 7, 2000)
            lo, hi = rng.randrange(0, 50), 0
        rot = rng.choice([0, D // 4, D // 2, D])
        c = _append("", B, Hq, Hkv, D, S, lo, hi or lo, page, dtype, rot, rng.random() < 0.5, S <= 5)
    elif op == "attention":
        Sq = rng.choice([1, 1, _log(rng, 2, 64)])
        hi = _log(rng, 1, 65536 if Sq == 1 else 16384)
        most = max(1, min(64, (1 << 26) // (Hq * Sq * hi), 1_600_000_000 // (4 * Hkv * D * hi)))
        c = _attention("", _log(rng, 1, most), Hq, Hkv, D, Sq, rng.randrange(0, hi + 1), hi, page, dtype)
    else:
        V = rng.choice([50304, 32001, _log(rng, 100, 131072)])
        B = _log(rng, 1, 256)
        k = rng.choice([0, 0, 1, _log(rng, 2, 1000)])
        c = _sample("", B, V, rng.choice(["f16", "bf16", "f32"]), round(rng.uniform(0.3, 1.5), 2), min(k, V), rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
                    rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]), rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths from lo to hi; with n = 1 the larger end."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(c):
    """Tokens in each request's cache before the call (append: also how many tokens enter), by the case alone; the seed only deals them out."""
    if c["op"] == "attention":
        return _spread(c["lo"], c["hi"], c["B"]), [c["Sq"]] * c["B"]
    start = _spread(c["lo"], max(c["hi"], c["lo"]), c["B"])
    return start, [c["S"]] * c["B"] if c["full"] else _spread(1, c["S"], c["B"])


def _paged(c, total, g, cg):
    """An empty-table pool that holds `total` tokens of each request, its pages dealt out in random order; entries past a request's end are -1."""
    pages = [-(-t // c["page"]) for t in total]
    width, n = max(1, max(pages)), sum(pages) + 3
    order = torch.randperm(n, generator=cg, dtype=torch.int32)
    table = torch.full((c["B"], width), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    shape = (n, c["Hkv"], c["page"], c["D"])
    dt = DTYPES[c["dtype"]]
    return table.cuda(), torch.randn(shape, generator=g, device="cuda", dtype=dt), torch.randn(shape, generator=g, device="cuda", dtype=dt)


def _slopes(H, dtype):
    """The table of co_alibi_attention: 2 * 2^(-8 (h + 1) / n) for the n = 2^floor(log2 H) first heads, odd half steps for the others, in the inputs' type."""
    n = 2 ** int(math.log2(H))
    s = [2.0 ** (-8.0 * (h + 1) / n) for h in range(n)] + [2.0 ** (-4.0 * (2 * h + 1) / n) for h in range(H - n)]
    return (2.0 * torch.tensor(s)).cuda().to(dtype)


def _tree(Sq, cg):
    """Ancestor bits of a random draft tree: node t hangs below one of the four nodes before it, or below the context."""
    bits = []
    for t in range(Sq):
        p = t - 1 - int(torch.randint(0, 4, (1,), generator=cg))
        bits.append((bits[p] if p >= 0 else 0) | 1 << t)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def prepare(case, seed):
    c = case
    g, cg = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["op"] == "sample":
        B, V = c["B"], c["V"]
        # a language model's logits: a few tokens stand out of a wide bulk
        x = torch.randn(B, V, generator=g, device="cuda") * 2.0 + torch.randn(V, generator=g, device="cuda")
        x += 1.5 * torch.empty(B, V, device="cuda").exponential_(generator=g).sub_(6).clamp_(min=0)
        state = {"logits": x.to(dt), "noise": torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_(min=1e-10)}
        for k in ("temperature", "top_k", "top_p", "min_p"):
            state[k] = c[k]
        if c["mixed"]:  # each request asks for its own
            row = torch.arange(B, device="cuda")
            state["temperature"] = torch.where(row % 5 == 3, 0.0, c["temperature"] * (0.5 + row % 3 * 0.5)).float()
            state["top_k"] = torch.where(row % 4 == 1, 0, c["top_k"] * (1 + row % 7)).to(torch.int32)
            state["top_p"] = torch.where(row % 3 == 2, 1.0, c["top_p"]).float()
            state["min_p"] = torch.where(row % 2 == 0, 0.0, c["min_p"]).float()
        return {"case": c, **state}
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    before, new = _lens(c)
    deal = torch.randperm(B, generator=cg).tolist()
    before, new = [before[i] for i in deal], [new[i] for i in deal]
    table, kp, vp = _paged(c, [a + b for a, b in zip(before, new)], g, cg)
    lens = torch.tensor(before, dtype=torch.int32).cuda()
    state = {"case": c, "page_table": table, "k_pages": kp, "v_pages": vp, "lens": lens}
    if c["op"] == "append":
        S, R = c["S"], c["rot"]
        # what a fused projection leaves: one row of query, key and value heads for each token
        qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=dt).transpose(1, 2)
        state["q"], state["k"], state["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        state["count"] = None if c["full"] else torch.tensor(new, dtype=torch.int32).cuda()
        if R:
            a = torch.arange(max(x + y for x, y in zip(before, new)), dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
            state["cos"], state["sin"] = a.cos().float().cuda(), a.sin().float().cuda()
        return state
    # Queries and keys lean apart, as trained ones do: most scores are negative, so the sigmoid sums grow slowly and far keys still count
    lean = torch.randn(D, generator=g, device="cuda")
    q = torch.randn(B, c["Sq"], Hq, D, generator=g, device="cuda") - 0.6 * lean
    state["k_pages"] = kp + (0.6 * lean).to(dt)
    state["q"] = q.to(dt).transpose(1, 2)
    state["slopes"] = _slopes(Hq, dt)
    state["tree_mask"] = torch.tensor([_tree(c["Sq"], cg) for _ in range(B)], dtype=torch.int64).cuda() if c["Sq"] > 1 else None
    return state


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """x [B, H, S, D] in 32 bits; cos, sin [B, 1, S, R / 2] of each token's position."""
    r = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        rotated = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        rotated = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rotated, x[..., 2 * r:]), -1)


def _plain_append(s):
    c = s["case"]
    q, k, v, kp, vp = s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"]
    i = torch.arange(c["S"], device="cuda")
    pos = s["lens"][:, None].long() + i
    fresh = i < (torch.full_like(s["lens"], c["S"]) if s["count"] is None else s["count"])[:, None]
    q_out = None
    if c["rot"]:
        at = pos.clamp(max=s["cos"].shape[0] - 1)
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q_out = (_rotate(q.float(), cos, sin, c["interleaved"]) * fresh[:, None, :, None]).to(q.dtype)
        k = _rotate(k.float(), cos, sin, c["interleaved"]).to(k.dtype)
    b, t = torch.nonzero(fresh, as_tuple=True)
    pos = pos[b, t]
    page = s["page_table"][b, pos // c["page"]].long()
    kp[page, :, pos % c["page"]] = k[b, :, t]
    vp[page, :, pos % c["page"]] = v[b, :, t]
    return {"k_pages": kp, "v_pages": vp, "q": q_out}


def _plain_attention(s):
    c = s["case"]
    Sq, G, q = c["Sq"], c["Hq"] // c["Hkv"], s["q"].float()
    pos = torch.arange(c["hi"] + Sq, device="cuda")
    page = s["page_table"].clamp(min=0).long()[:, pos // c["page"]]
    k = s["k_pages"][page, :, pos % c["page"]].float().permute(0, 2, 3, 1)  # [B, Hkv, D, L]
    v = s["v_pages"][page, :, pos % c["page"]].float().transpose(1, 2)  # [B, Hkv, L, D]
    bits = torch.ones(c["B"], 1, dtype=torch.int64, device="cuda") if s["tree_mask"] is None else s["tree_mask"]
    draft = pos - s["lens"][:, None].long()  # [B, L]: which drafted token a slot holds; negative for the context
    seen = (bits[:, :, None] >> draft.clamp(0, 63)[:, None] & 1).bool() & (draft < Sq)[:, None] | (draft < 0)[:, None]
    seen = seen[:, None, None]  # [B, 1, 1, Sq, L]
    p = torch.matmul(q.reshape(c["B"], c["Hkv"], G * Sq, -1), k).view(c["B"], c["Hkv"], G, Sq, -1) / math.sqrt(c["D"])
    z = torch.where(seen, torch.sigmoid(p), 0.0).flip(-1).cumsum(-1).flip(-1)
    x = torch.where(seen, p - s["slopes"].float().view(1, c["Hkv"], G, 1, 1) * z, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(w.flatten(2, 3), v) / w.sum(-1).clamp(min=1e-30).flatten(2, 3)[..., None]
    return o.view(c["B"], c["Hq"], Sq, -1).to(s["q"].dtype)


def _rows(v, B, dtype):
    return v[:, None] if isinstance(v, torch.Tensor) else torch.full((B, 1), v, dtype=dtype, device="cuda")


def _plain_sample(s):
    B, V = s["logits"].shape
    top_k, top_p = _rows(s["top_k"], B, torch.int32), _rows(s["top_p"], B, torch.float32)
    t, min_p = _rows(s["temperature"], B, torch.float32), _rows(s["min_p"], B, torch.float32)
    x, order = s["logits"].float().sort(stable=True, dim=-1, descending=True)
    d = (x - x[:, :1]) * torch.where(t > 0, 1 / t, 0.0)
    rank = torch.arange(V, device="cuda")
    w = torch.exp(d) * ((top_k <= 0) | (rank < top_k))
    before = w.cumsum(-1) - w
    kept = (w > 0) & ((top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True)) | (rank == 0))
    kept &= (w >= min_p) & ((t > 0) | (rank == 0))
    w = w * kept
    best = torch.where(kept, w / s["noise"].gather(1, order), -1.0).argmax(-1, keepdim=True)
    # the first weight is exactly 1: the others' sum keeps a log-probability near zero exact
    return {"tokens": order.gather(1, best)[:, 0], "logprobs": (d.gather(1, best) - w[:, 1:].sum(-1, keepdim=True).log1p())[:, 0]}


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[c["op"]](s)
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "co-alibi_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from co_alibi_attn import append_paged_kv, paged_tree_attention, sample_tokens
    if c["op"] == "append":
        rotary = (s["cos"], s["sin"]) if c["rot"] else None
        q = append_paged_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lens"], count=s["count"], q=s["q"] if c["rot"] else None, rotary=rotary,
                            interleaved=c["interleaved"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": q}
    if c["op"] == "attention":
        return paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lens"], tree_mask=s["tree_mask"], slopes=s["slopes"])
    tokens, logprobs = sample_tokens(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"tokens": tokens, "logprobs": logprobs}


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "sample":
        # every logit once; a filtered row needs the random numbers of its few survivors only
        whole = not c["mixed"] and c["top_k"] == 0 and c["top_p"] >= 1 and c["min_p"] <= 0
        return {"bytes": c["B"] * (c["V"] * (size + (4 if whole else 0)) + 12), "flops": 4 * c["B"] * c["V"]}
    before, new = _lens(c)
    D, Hq, Hkv = c["D"], c["Hq"], c["Hkv"]
    if c["op"] == "append":
        n = sum(new)
        moved = 2 * n * 2 * Hkv * D * size + (c["B"] * c["S"] * Hq * D * size + n * (Hq * D * size + c["rot"] * 4) if c["rot"] else 0)
        return {"bytes": moved + 12 * c["B"], "flops": 3 * n * (Hq + Hkv) * c["rot"]}
    keys = sum(before) + sum(new)
    return {"bytes": 2 * keys * Hkv * D * size + 2 * c["B"] * Hq * c["Sq"] * D * size + 4 * keys // c["page"], "flops": (4 * D + 10) * Hq * c["Sq"] * keys}


# ---------------------------------------------------------------------------------------------------------------------
# The same answers in 64 bits, request by request
# ---------------------------------------------------------------------------------------------------------------------


def _exact_append(s):
    c = s["case"]
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    half = c["rot"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)

    def turned(x, p):  # [H, n, D] at positions p [n]
        y = x.double().clone()
        if half:
            z = torch.complex(x[..., first].double(), x[..., second].double()) * torch.complex(s["cos"][p].double(), s["sin"][p].double())
            y[..., first], y[..., second] = z.real, z.imag
        return y

    q_out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") if half else None
    for b, start in enumerate(s["lens"].tolist()):
        n = c["S"] if s["count"] is None else int(s["count"][b])
        p = start + torch.arange(n, device="cuda")
        page, slot = s["page_table"][b].long()[p // c["page"]], p % c["page"]
        kp[page, :, slot] = turned(s["k"][b, :, :n], p).transpose(0, 1)
        vp[page, :, slot] = s["v"][b, :, :n].double().transpose(0, 1)
        if half:
            q_out[b, :, :n] = turned(s["q"][b, :, :n], p)
    return {"k_pages": kp, "v_pages": vp, "q": q_out}


def _exact_attention(s):
    c = s["case"]
    G, Sq, out = c["Hq"] // c["Hkv"], c["Sq"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, ctx in enumerate(s["lens"].tolist()):
        n = ctx + Sq
        pages = s["page_table"][b, : -(-n // c["page"])].long()
        k, v = (x[pages].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (s["k_pages"], s["v_pages"]))
        words = [1] if s["tree_mask"] is None else s["tree_mask"][b].tolist()
        hidden = torch.zeros(Sq, n, dtype=torch.bool, device="cuda")
        hidden[:, ctx:] = torch.tensor([[not w >> t & 1 for t in range(Sq)] for w in words], device="cuda")
        for h in range(c["Hq"]):
            p = s["q"][b, h].double() @ k[h // G].T / math.sqrt(c["D"])
            g = (1 / (1 + torch.exp(-p))).masked_fill(hidden, 0)
            z = g.sum(-1, keepdim=True) - (g.cumsum(-1) - g)  # all of the row less what lies left of the key
            x = (p - s["slopes"][h].double() * z).masked_fill(hidden, -math.inf)
            out[b, h] = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)) @ v[h // G]
    return out


def _exact_sample(s):
    B = s["logits"].shape[0]
    tokens, logprobs = [], []
    of = lambda k, b: s[k][b].item() if isinstance(s[k], torch.Tensor) else s[k]  # noqa: E731
    for b in range(B):
        t, k, p, least = of("temperature", b), of("top_k", b), of("top_p", b), of("min_p", b)
        x = s["logits"][b].double()
        if t <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        x = (x - x.max()) / t
        order = torch.argsort(x, descending=True, stable=True)[: k or None]
        w = torch.exp(x[order])
        if p < 1:
            n = max(1, int((torch.cumsum(w, 0) - w < p * w.sum()).sum()))
            order, w = order[:n], w[:n]
        order, w = order[w >= least], w[w >= least]
        i = int(torch.argmax(torch.log(w) - torch.log(s["noise"][b][order].double())))
        tokens.append(int(order[i]))
        logprobs.append(float(x[order[i]] - torch.log(w.sum())))
    return {"tokens": torch.tensor(tokens, device="cuda"), "logprobs": torch.tensor(logprobs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](s)
