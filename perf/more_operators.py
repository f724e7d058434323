"""More operators of a Co-ALiBi model: a key/value cache held in 8 bits with the attention over it, and the normed heads that feed it.

  write   new keys and values into a paged cache of e4m3 codes with a scale for each block of 16 tokens and head, rotated on the way
  read    tokens of that cache back in 16 bits
  attend  Co-ALiBi attention of one token, or of a tree of drafted tokens, over that cache
  heads   a fused projection split into query, key and value heads, queries and keys normed per head and rotated; with its gradient

``run`` computes them in their plain form (torch, 32 bits), or with ``own`` set through the package's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16  # tokens that share a scale
EPS = 1e-6

# ---------------------------------------------------------------------------------------------------------------------
# Cases.  Head counts and widths are those of the repository's own configurations (H16 D128; Hq32 Hkv8 D128; 12 heads of
# 64), the training ones with the batch of its GPT and the batch of its grouped-head benchmark (one token short of it).
# ---------------------------------------------------------------------------------------------------------------------


def _write(name, B, Hq, Hkv, D, S, lo, hi, page, dtype, rot, interleaved, full):
    return {"name": name, "op": "write", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "S": S, "lo": lo, "hi": hi, "page": page, "dtype": dtype, "rot": rot,
            "interleaved": interleaved, "full": full}


def _read(name, B, Hkv, D, S, lo, hi, page, dtype):
    return {"name": name, "op": "read", "B": B, "Hkv": Hkv, "D": D, "S": S, "lo": lo, "hi": hi, "page": page, "dtype": dtype}


def _attend(name, B, Hq, Hkv, D, Sq, lo, hi, page, dtype):
    return {"name": name, "op": "attend", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "Sq": Sq, "lo": lo, "hi": hi, "page": page, "dtype": dtype}


def _heads(name, B, S, Hq, Hkv, D, dtype, rot, interleaved, train):
    return {"name": name, "op": "heads", "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "rot": rot, "interleaved": interleaved, "train": train}


def listed():
    return [
        # one token of each of a few requests of the small GPT, no rotation: the call's latency is all there is
        _write("write gpt token", 4, 12, 12, 64, 1, 1, 900, 16, "bf16", 0, False, True),
        # a decoding step of a large batch with grouped heads, the whole head rotated, lengths all different
        _write("write decode batch", 256, 32, 8, 128, 1, 0, 500, 16, "bf16", 128, False, True),
        # prompts of ragged lengths entering the cache, half of each head rotated in interleaved pairs
        _write("write ragged prompts", 8, 32, 8, 128, 2000, 3, 3, 64, "f16", 64, True, False),
        # the accepted paths of drafted trees, taken from their slots before they move together
        _read("read draft paths", 16, 8, 128, 9, 100, 4000, 32, "bf16"),
        # long prefixes in 16 bits again, for a prompt's next chunk
        _read("read prefixes", 4, 8, 128, 16384, 0, 0, 64, "f16"),
        # one token of one short chat of the small GPT
        _attend("attend one short", 1, 12, 12, 64, 1, 36, 36, 16, "f16"),
        # a decoding step of a batch of grouped heads, from empty caches to 8192 tokens
        _attend("attend decode batch", 16, 32, 8, 128, 1, 0, 8191, 64, "bf16"),
        # a few long documents, one token each: the largest reads
        _attend("attend long", 4, 32, 8, 128, 1, 65537, 131071, 64, "bf16"),
        # verifying trees of 16 drafted tokens over grouped heads: 64 rows share each key
        _attend("attend tree 16", 8, 32, 8, 128, 16, 127, 16383, 32, "f16"),
        # one token of each of a batch: the call's latency
        _heads("heads one token", 64, 1, 12, 12, 64, "bf16", 64, False, False),
        # a training step's layer of the small GPT
        _heads("heads train gpt", 32, 1024, 12, 12, 64, "bf16", 64, False, True),
        # a training step's layer with grouped heads and long odd sequences, half of each head rotated in interleaved pairs
        _heads("heads train grouped", 4, 8191, 32, 8, 128, "f16", 64, True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "heads"])
    Hq, Hkv, D = rng.choice([(12, 12, 64), (16, 16, 128), (32, 8, 128), (8, 1, 128), (12, 4, 64)])
    page, dtype = rng.choice([16, 32, 48, 64, 128]), rng.choice(["f16", "bf16"])
    rot, interleaved = rng.choice([0, D // 4, D // 2, D]), rng.random() < 0.5
    if op == "write":
        if rng.random() < 0.5:
            B, S, lo, hi = _log(rng, 1, 256), rng.choice([1, 1, 2, 5]), 0, _log(rng, 8, 500)
        else:
            B, S, lo = _log(rng, 1, 8), _log(rng, 7, 2000), rng.randrange(0, 50)
            hi = lo
        c = _write("", B, Hq, Hkv, D, S, lo, hi, page, dtype, rot, interleaved, S <= 5)
    elif op == "read":
        if rng.random() < 0.5:
            c = _read("", _log(rng, 1, 64), Hkv, D, _log(rng, 1, 64), _log(rng, 1, 100), _log(rng, 100, 4000), page, dtype)
        else:
            B = _log(rng, 1, 8)
            c = _read("", B, Hkv, D, _log(rng, 64, max(64, min(32768, 65536 * 8 * 128 // (B * Hkv * D)))), 0, 0, page, dtype)
    elif op == "attend":
        Sq = rng.choice([1, 1, _log(rng, 2, 64)])
        hi = _log(rng, 1, 65536 if Sq == 1 else 16384)
        most = max(1, min(64, (1 << 26) // (Hq * Sq * hi), 800_000_000 // (2 * Hkv * D * hi)))
        c = _attend("", _log(rng, 1, most), Hq, Hkv, D, Sq, rng.randrange(0, hi + 1), hi, page, dtype)
    else:
        train = rng.random() < 0.6
        B = _log(rng, 1, 64)
        S = rng.choice([1, _log(rng, 2, 64)]) if not train else _log(rng, 16, max(16, min(8192, 32768 * 48 * 128 // (B * (Hq + 2 * Hkv) * D))))
        c = _heads("", B, S, Hq, Hkv, D, dtype, rot, interleaved, train)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths from lo to hi; with n = 1 the larger end."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(c):
    """Tokens in each request's cache before the call, and how many of the call's it holds behind them, by the case alone; the seed only deals them out."""
    if c["op"] == "attend":
        return _spread(c["lo"], c["hi"], c["B"]), [c["Sq"]] * c["B"]
    start = _spread(c["lo"], max(c["hi"], c["lo"]), c["B"])
    if c["op"] == "read":  # drafts: a few of twice as many slots
        return start, [2 * c["S"] if c["hi"] else c["S"]] * c["B"]
    return start, [c["S"]] * c["B"] if c["full"] else _spread(1, c["S"], c["B"])


def _scale_of(most):
    """The least power of two, and at least 2^-100, under which `most` (float32, not negative) is at most 448, e4m3's largest value."""
    m, e = torch.frexp(most)
    k = torch.where(most > 0, e - 9 + (m > 0.875).int(), -100).clamp(min=-100)
    return torch.exp2(k.double()).float()


def _pool(shape, add, dt, g):
    """Codes and scales of a pool of random values."""
    n, H, page, D = shape
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(n, H, page // BLOCK, device="cuda")
    for i in range(0, n, 1024):
        x = torch.randn((min(1024, n - i), H, page, D), generator=g, device="cuda", dtype=dt)
        # tokens differ in size, as in earnest
        x = (x + add if add is not None else x) * torch.empty((x.shape[0], H, page, 1), device="cuda", dtype=dt).uniform_(0.25, 1.75, generator=g)
        x = x.float().view(x.shape[0], H, page // BLOCK, BLOCK, D)
        s = _scale_of(x.abs().amax((-1, -2)))
        scales[i:i + 1024] = s
        codes[i:i + 1024] = (x / s[..., None, None]).view(x.shape[0], H, page, D).to(torch.float8_e4m3fn)
    return codes, scales


def _paged(c, total, g, cg, lean=None):
    """A pool that holds `total` tokens of each request, its pages dealt out in random order; entries past a request's end are -1."""
    pages = [-(-t // c["page"]) for t in total]
    width, n = max(1, max(pages)), sum(pages) + 3
    order = torch.randperm(n, generator=cg, dtype=torch.int32)
    table = torch.full((c["B"], width), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    shape, dt = (n, c["Hkv"], c["page"], c["D"]), DTYPES[c["dtype"]]
    kp, ks = _pool(shape, lean, dt, g)
    vp, vs = _pool(shape, None, dt, g)
    return {"page_table": table.cuda(), "k_pages": kp, "v_pages": vp, "k_scales": ks, "v_scales": vs}


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


def _tables(n, R):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float().cuda(), a.sin().float().cuda()


def prepare(case, seed):
    c = case
    g, cg = torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, D, Hkv = c["B"], c["D"], c["Hkv"]
    if c["op"] == "heads":
        S, Hq = c["S"], c["Hq"]
        state = {"case": c, "qkv": torch.randn(B, S, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=dt)}
        state["q_weight"], state["k_weight"] = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt) for _ in range(2))
        # serving: each request's token at a position of its own
        state["start"] = None if c["train"] else torch.randint(0, 2000, (B,), generator=cg, dtype=torch.int32).cuda()
        if c["rot"]:
            state["cos"], state["sin"] = _tables(S if c["train"] else 2000 + S, c["rot"])
        if c["train"]:
            for name in ("qkv", "q_weight", "k_weight"):
                state[name].requires_grad_()
            state["grads"] = [torch.randn(B, H, S, D, generator=g, device="cuda", dtype=dt) for H in (Hq, Hkv, Hkv)]
        return state
    before, new = _lens(c)
    deal = torch.randperm(B, generator=cg).tolist()
    before, new = [before[i] for i in deal], [new[i] for i in deal]
    # Queries and keys lean apart, as trained ones do: most scores are negative, so the sigmoid sums grow slowly and far keys still count
    lean = torch.randn(D, generator=g, device="cuda")
    state = {"case": c, **_paged(c, [a + b for a, b in zip(before, new)], g, cg, (0.6 * lean).to(dt) if c["op"] == "attend" else None)}
    lens = torch.tensor(before, dtype=torch.int32).cuda()
    state["lens"] = lens
    if c["op"] == "write":
        S, R, Hq = c["S"], c["rot"], c["Hq"]
        # what a fused projection leaves: one row of query, key and value heads for each token
        qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=dt).transpose(1, 2)
        state["q"], state["k"], state["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        state["count"] = None if c["full"] else torch.tensor(new, dtype=torch.int32).cuda()
        if R:
            state["cos"], state["sin"] = _tables(max(x + y for x, y in zip(before, new)), R)
    elif c["op"] == "read":
        if c["hi"]:  # some of the drafts' slots, in order
            path = torch.stack([torch.randperm(2 * c["S"], generator=cg)[:c["S"]].sort()[0] for _ in range(B)])
        else:
            path = torch.arange(c["S"]).expand(B, -1)
        state["positions"] = (lens[:, None] + path.cuda()).int()
    else:
        q = torch.randn(B, c["Sq"], c["Hq"], D, generator=g, device="cuda") - 0.6 * lean
        state["q"] = q.to(dt).transpose(1, 2)
        state["slopes"] = _slopes(c["Hq"], dt)
        state["tree_mask"] = torch.tensor([_tree(c["Sq"], cg) for _ in range(B)], dtype=torch.int64).cuda() if c["Sq"] > 1 else None
    return state


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """x [..., D] in 32 bits, its first 2 r elements turned by cos, sin [..., r]."""
    r = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        rotated = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        rotated = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rotated, x[..., 2 * r:]), -1)


def _write_blocks(s, x, pages, scales, fresh):
    """x [B, S, H, D] in 32 bits into the blocks that it touches: a block's scale grows with its new tokens, and its old ones' codes with it; a block of new tokens alone
    takes theirs."""
    c = s["case"]
    B, S, H, D = x.shape
    nb = (S + BLOCK - 2) // BLOCK + 1
    first = s["lens"].long() // BLOCK  # each request's first block
    block = first[:, None] + torch.arange(nb, device="cuda")  # [B, nb]
    pos = block[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")  # [B, nb, 16]
    i = pos - s["lens"].long()[:, None, None]  # which new token a slot takes
    new = (i >= 0) & (i < fresh[:, None, None])
    touched = new.any(-1)
    row = (torch.arange(B, device="cuda")[:, None, None], i.clamp(0, S - 1))
    x = torch.where(new[..., None, None], x[row], 0.0)  # [B, nb, 16, H, D]
    at = (block * BLOCK // c["page"]).clamp(max=s["page_table"].shape[1] - 1)
    page = s["page_table"].long().gather(1, at).clamp(min=0)
    sub = block % (c["page"] // BLOCK)
    was = scales[page, :, sub]  # [B, nb, H]
    most = torch.where(torch.isfinite(x), x, 0.0).abs().amax((2, 4))
    scale = _scale_of(most)
    old = (i < 0) & touched[..., None]
    scale = torch.where(old.any(-1)[..., None], torch.maximum(scale, was), scale)
    slot = sub[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    codes = pages.view(torch.uint8)[page[..., None], :, slot].view(torch.float8_e4m3fn)  # [B, nb, 16, H, D]
    codes = torch.where(old[..., None, None], codes.float() * (was / scale)[:, :, None, :, None], x / scale[:, :, None, :, None]).to(torch.float8_e4m3fn)
    b, j, t = torch.nonzero(new | old, as_tuple=True)
    pages.view(torch.uint8)[page[b, j], :, slot[b, j, t]] = codes.view(torch.uint8)[b, j, t]
    b, j = torch.nonzero(touched, as_tuple=True)
    scales[page[b, j], :, sub[b, j]] = scale[b, j]


def _plain_write(s):
    c = s["case"]
    q, k, v = s["q"], s["k"].float(), s["v"].float()
    i = torch.arange(c["S"], device="cuda")
    fresh = torch.full_like(s["lens"], c["S"]) if s["count"] is None else s["count"]
    q_out = None
    if c["rot"]:
        at = (s["lens"][:, None].long() + i).clamp(max=s["cos"].shape[0] - 1)
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q_out = (_rotate(q.float(), cos, sin, c["interleaved"]) * (i < fresh[:, None])[:, None, :, None]).to(q.dtype)
        k = _rotate(k, cos, sin, c["interleaved"])
    _write_blocks(s, k.transpose(1, 2), s["k_pages"], s["k_scales"], fresh)
    _write_blocks(s, v.transpose(1, 2), s["v_pages"], s["v_scales"], fresh)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scales": s["k_scales"], "v_scales": s["v_scales"], "q": q_out}


def _gathered(s, pages, scales, pos):
    """The values of the tokens at pos [B, n], or [n] for all requests: [B, n, H, D]."""
    page = s["case"]["page"]
    pos = pos.long().expand(s["page_table"].shape[0], -1)
    at, slot = s["page_table"].clamp(min=0).long().gather(1, pos // page), pos % page
    codes = pages.view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn)
    return codes.float() * scales[at, :, slot // BLOCK][..., None]


def _plain_read(s):
    dt = DTYPES[s["case"]["dtype"]]
    most = torch.finfo(dt).max
    k, v = (_gathered(s, s[n + "_pages"], s[n + "_scales"], s["positions"]).clamp(-most, most).to(dt).transpose(1, 2).contiguous() for n in "kv")
    return {"k": k, "v": v}


def _plain_attend(s):
    c = s["case"]
    Sq, G, q = c["Sq"], c["Hq"] // c["Hkv"], s["q"].float()
    pos = torch.arange(c["hi"] + Sq, device="cuda")
    k = _gathered(s, s["k_pages"], s["k_scales"], pos).permute(0, 2, 3, 1)  # [B, Hkv, D, L]
    v = _gathered(s, s["v_pages"], s["v_scales"], pos).transpose(1, 2)  # [B, Hkv, L, D]
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


def _angles(s):
    """cos and sin [B or 1, S, 1, R / 2] of each token."""
    at = torch.arange(s["case"]["S"], device="cuda")[None]
    if s["start"] is not None:
        at = at + s["start"][:, None].long()
    return s["cos"][at][:, :, None], s["sin"][at][:, :, None]


def _plain_heads(s):
    c = s["case"]
    Hq, Hkv, dt = c["Hq"], c["Hkv"], s["qkv"].dtype
    x = s["qkv"].detach().float()
    w = torch.cat([s[n].detach().float().expand(H, -1) for n, H in (("q_weight", Hq), ("k_weight", Hkv))])  # [Hq + Hkv, D]
    x, v = x[:, :, :Hq + Hkv], s["qkv"].detach()[:, :, Hq + Hkv:]
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    y = x * r * w
    if c["rot"]:
        cos, sin = _angles(s)
        y = _rotate(y, cos, sin, c["interleaved"])
    q, k = (t.to(dt).transpose(1, 2).contiguous() for t in (y[:, :, :Hq], y[:, :, Hq:]))
    out = {"q": q, "k": k, "v": v.transpose(1, 2).contiguous()}
    if not c["train"]:
        return out
    d = torch.cat([t.float().transpose(1, 2) for t in s["grads"][:2]], 2)
    if c["rot"]:
        d = _rotate(d, cos, -sin, c["interleaved"])
    n = x * r
    dw = d * n
    d = d * w
    dx = r * (d - n * (d * n).mean(-1, keepdim=True))
    out["qkv"] = torch.cat([dx.to(dt), s["grads"][2].transpose(1, 2)], 2)
    out["q_weight"], out["k_weight"] = (t.sum((0, 1, 2), dtype=torch.float64).to(dt) for t in (dw[:, :, :Hq], dw[:, :, Hq:]))
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "heads": _plain_heads}[c["op"]](s)
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "co-alibi_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from co_alibi_attn import append_paged_kv, norm_rotate_qkv, paged_tree_attention, read_paged_kv
    rotary = (s["cos"], s["sin"]) if c.get("rot") else None
    if c["op"] == "heads":
        q, k, v = norm_rotate_qkv(s["qkv"], c["Hq"], c["Hkv"], s["q_weight"], s["k_weight"], eps=EPS, rotary=rotary, start=s["start"], interleaved=c["interleaved"])
        out = {"q": q, "k": k, "v": v}
        if c["train"]:
            names = ("qkv", "q_weight", "k_weight")
            out.update(zip(names, torch.autograd.grad((q, k, v), [s[n] for n in names], s["grads"])))
        return out
    cache, scales = (s["k_pages"], s["v_pages"], s["page_table"]), (s["k_scales"], s["v_scales"])
    if c["op"] == "write":
        q = append_paged_kv(s["k"], s["v"], *cache, s["lens"], count=s["count"], q=s["q"] if c["rot"] else None, rotary=rotary, interleaved=c["interleaved"], scales=scales)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scales": s["k_scales"], "v_scales": s["v_scales"], "q": q}
    if c["op"] == "read":
        k, v = read_paged_kv(*cache, s["positions"], scales=scales, dtype=DTYPES[c["dtype"]])
        return {"k": k, "v": v}
    return paged_tree_attention(s["q"], *cache, s["lens"], tree_mask=s["tree_mask"], slopes=s["slopes"], scales=scales)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    B, D, Hkv = c["B"], c["D"], c["Hkv"]
    if c["op"] == "heads":
        n = B * c["S"] * (c["Hq"] + 2 * Hkv) * D
        angles = 4 * c["rot"] * c["S"] * (1 if c["train"] else B)
        return {"bytes": 2 * n * (5 if c["train"] else 2) + angles * (2 if c["train"] else 1), "flops": n * (20 if c["train"] else 7)}
    before, new = _lens(c)
    if c["op"] == "write":
        n = sum(new)
        blocks = sum((a + b - 1) // BLOCK - a // BLOCK + 1 for a, b in zip(before, new))
        moved = n * 2 * Hkv * D * 3 + blocks * 2 * Hkv * 4
        if c["rot"]:
            moved += B * c["S"] * c["Hq"] * D * 2 + n * (c["Hq"] * D * 2 + c["rot"] * 4)
        return {"bytes": moved + 12 * B, "flops": n * (3 * (c["Hq"] + Hkv) * c["rot"] + 4 * Hkv * D)}
    if c["op"] == "read":
        n = B * c["S"]
        blocks = n if c["hi"] else -(-n // BLOCK)
        return {"bytes": n * 2 * Hkv * D * 3 + blocks * 2 * Hkv * 4 + 4 * n, "flops": n * 2 * Hkv * D}
    keys = sum(before) + sum(new)
    return {"bytes": 2 * keys * Hkv * D + 8 * keys * Hkv // BLOCK + 4 * B * c["Hq"] * c["Sq"] * D + 4 * keys // c["page"], "flops": (4 * D + 10) * c["Hq"] * c["Sq"] * keys}


# ---------------------------------------------------------------------------------------------------------------------
# The same answers in 64 bits, request by request
# ---------------------------------------------------------------------------------------------------------------------

#: every e4m3 value from 0 to 448, by its code
E4M3 = [(c & 7) / 512 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)]


def _nearest(x):
    """The e4m3 values nearest to x (at most 448 in size), of two equally near ones that with the even code."""
    grid = torch.tensor(E4M3, dtype=torch.float64, device="cuda")
    border = (grid[1:] + grid[:-1]) / 2
    a = x.abs()
    i = torch.bucketize(a, border)  # the code below or at the nearer side of its border
    tie = (i < 126) & (a == border[i.clamp(max=125)]) & (i % 2 == 1)
    return torch.copysign(grid[i + tie], x)


def _turned(x, cos, sin, interleaved):
    """x [..., n, D] turned by cos, sin [n, r], as complex numbers."""
    r = cos.shape[-1]
    first = torch.arange(r, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else r)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sin)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_write(s):
    c = s["case"]
    out = {n: s[n].double() for n in ("k_pages", "v_pages", "k_scales", "v_scales")}
    out["q"] = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") if c["rot"] else None
    for b, start in enumerate(s["lens"].tolist()):
        n = c["S"] if s["count"] is None else int(s["count"][b])
        k, v, q = (s[x][b, :, :n].double() for x in ("k", "v", "q"))
        if c["rot"]:
            cos, sin = (s[x][start:start + n].double() for x in ("cos", "sin"))
            k = _turned(k, cos, sin, c["interleaved"])
            out["q"][b, :, :n] = _turned(q, cos, sin, c["interleaved"])
        # old tokens of the first block stand before the new ones, empty slots behind the last
        head, tail = start % BLOCK, -(start + n) % BLOCK
        where = torch.arange(start - head, start + n + tail, BLOCK, device="cuda")  # each block's first slot
        page, sub = s["page_table"][b].long()[where // c["page"]], where % c["page"] // BLOCK
        for name, x in (("k", k), ("v", v)):
            codes = out[name + "_pages"].view(-1, c["Hkv"], c["page"] // BLOCK, BLOCK, c["D"])
            x = torch.nn.functional.pad(x, (0, 0, head, tail)).unflatten(1, (-1, BLOCK))  # [H, blocks, 16, D]
            most = x.abs().amax((2, 3))
            size = torch.pow(2.0, torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)).clamp(min=-100))
            size = torch.where(most > 448 * size, 2 * size, torch.where((most <= 224 * size) & (size > 2.0 ** -100), size / 2, size))
            if head:
                was = out[name + "_scales"][page[0], :, sub[0]]
                size[:, 0] = torch.maximum(size[:, 0], was)
                x[:, 0, :head] = codes[page[0], :, sub[0], :head] * was[:, None, None]
            y = _nearest(x / size[..., None, None])
            y[:, -1, BLOCK - tail:] = codes[page[-1], :, sub[-1], BLOCK - tail:]
            codes[page, :, sub] = y.transpose(0, 1)
            out[name + "_scales"][page, :, sub] = size.T
    return out


def _exact_read(s):
    c = s["case"]
    out = {}
    for n in "kv":
        whole = (s[n + "_pages"].double().unflatten(2, (-1, BLOCK)) * s[n + "_scales"].double()[..., None, None]).flatten(2, 3)
        out[n] = torch.stack([whole[s["page_table"][b].long()[p // c["page"]], :, p % c["page"]].transpose(0, 1) for b, p in enumerate(s["positions"].long())])
    return out


def _exact_attend(s):
    c = s["case"]
    G, Sq, out = c["Hq"] // c["Hkv"], c["Sq"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, ctx in enumerate(s["lens"].tolist()):
        n = ctx + Sq
        pages = s["page_table"][b, : -(-n // c["page"])].long()
        k, v = ((s[x + "_pages"][pages].double().unflatten(2, (-1, BLOCK)) * s[x + "_scales"][pages].double()[..., None, None]).flatten(2, 3).transpose(0, 1).flatten(1, 2)[:, :n]
                for x in "kv")
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


def _exact_heads(s):
    c = s["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    leaves = [s[n].detach().double().requires_grad_(c["train"]) for n in ("qkv", "q_weight", "k_weight")]
    q, k, v = (t.transpose(1, 2) for t in leaves[0].split([Hq, Hkv, Hkv], 2))
    out = []
    for x, w in ((q, leaves[1]), (k, leaves[2])):
        y = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / c["D"] + EPS).sqrt() * w
        if c["rot"]:
            half, B, S = c["rot"] // 2, c["B"], c["S"]
            at = torch.arange(S, device="cuda") + (0 if s["start"] is None else s["start"].view(B, 1, 1))
            turn = torch.complex(s["cos"].double(), s["sin"].double())[at]  # [S, half], or [B, 1, S, half]
            pairs = y[..., :c["rot"]].unflatten(-1, (half, 2) if c["interleaved"] else (2, half))
            a, b = pairs.unbind(-1 if c["interleaved"] else -2)
            z = torch.complex(a, b) * turn
            z = torch.stack((z.real, z.imag), -1 if c["interleaved"] else -2).flatten(-2)
            y = torch.cat((z, y[..., c["rot"]:]), -1)
        out.append(y)
    got = {"q": out[0].detach(), "k": out[1].detach(), "v": v.detach()}
    if c["train"]:
        got.update(zip(("qkv", "q_weight", "k_weight"), torch.autograd.grad((*out, v), leaves, [t.double() for t in s["grads"]])))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "heads": _exact_heads}[case["op"]](s)
