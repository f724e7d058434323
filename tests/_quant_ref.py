"""The paged cache in 8 bits and the normed heads from their definitions in 64 bits, and the
inputs their tests share.  CPU only, no code of the package."""
import math

import torch

from tests import _serving_ref as ref

BLOCK = 16
#: every e4m3 value from 0 to 448, by its code
GRID = torch.tensor([(c & 7) / 512 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)], dtype=torch.float64)
NAN = 0x7f


def codes_of(x):
    """uint8 codes of the e4m3 values nearest to x (float64, at most 448 in size), ties to the even code; NaN's for NaN."""
    a = x.abs()
    border = (GRID[1:] + GRID[:-1]) / 2
    i = torch.bucketize(a, border)
    i = i + ((i < 126) & (a == border[i.clamp(max=125)]) & (i % 2 == 1))
    c = torch.where(torch.signbit(x), i + 128, i)
    return torch.where(x.isnan(), NAN, c).to(torch.uint8)


def values_of(codes):
    """float64 values of uint8 codes."""
    c = codes.long()
    v = torch.cat([GRID, torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    return torch.where(c >= 128, -v, v)


def scale_of(most):
    """The least power of two, and at least 2^-100, by which the float `most` is at most 448."""
    if most == 0:
        return 2.0 ** -100
    k = math.ceil(math.log2(most / 448)) - 1
    while most > 448 * 2.0 ** k:
        k += 1
    return 2.0 ** max(k, -100)


def quantised(x):
    """(codes uint8, scales float32) of a pool [n, H, page, D]."""
    n, H, page, D = x.shape
    y = x.double().view(n, H, page // BLOCK, BLOCK, D)
    most = y.abs().amax((3, 4))
    scales = torch.tensor([scale_of(float(m)) for m in most.flatten()], dtype=torch.float64).view(most.shape)
    return codes_of(y / scales[..., None, None]).view(n, H, page, D), scales.float()


def dequantised(codes, scales):
    """float64 values of a pool."""
    return (values_of(codes).unflatten(2, (-1, BLOCK)) * scales.double()[..., None, None]).flatten(2, 3)


def pool(lens, Hkv, D, page, seed, spread=0.0, **kw):
    """Codes and scales (k, v, k_scales, v_scales, table) of random pools; `spread`: the blocks' sizes differ by 2^+-spread."""
    k, v, table = ref.pool(lens, Hkv, D, page, torch.float32, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1000)
    out = []
    for x in (k, v):
        f = 2.0 ** (spread * (2 * torch.rand((*x.shape[:2], x.shape[2] // BLOCK), generator=g) - 1))
        x = (x.unflatten(2, (-1, BLOCK)) * f[..., None, None]).flatten(2, 3)
        out.append(quantised(x))
    return out[0][0], out[1][0], out[0][1], out[1][1], table


def e4m3(codes):
    return codes.view(torch.float8_e4m3fn)


def append(x, pages, scales, table, start, count):
    """x [B, H, S, D] (the values that enter, float32 or float64) into codes `pages` and `scales`, in place, block by block."""
    page = pages.shape[2]
    for b in range(x.shape[0]):
        s, n = int(start[b]), int(count[b])
        for t0 in range(s // BLOCK * BLOCK, s + n, BLOCK):
            lo, hi = max(s - t0, 0), min(s + n - t0, BLOCK)
            at = int(table[b, t0 // page]) if t0 // page < table.shape[1] else -1
            if hi <= lo or not 0 <= at < pages.shape[0]:
                continue
            slot = t0 % page
            for h in range(x.shape[1]):
                new = x[b, h, t0 + lo - s:t0 + hi - s].double()
                new = torch.where(new.isinf(), math.nan, new)
                scale = scale_of(float(torch.nan_to_num(new, nan=0.0).abs().max()))
                if lo:
                    was = float(scales[at, h, slot // BLOCK])
                    scale = max(scale, was)
                    old = pages[at, h, slot:slot + lo]
                    pages[at, h, slot:slot + lo] = codes_of(values_of(old) * (was / scale))
                pages[at, h, slot + lo:slot + hi] = codes_of(new / scale)
                scales[at, h, slot // BLOCK] = scale


def rotated32(x, cos, sin, interleaved):
    """x [..., D] turned in float32, products and their sum rounded one by one."""
    return ref.rotated(x.float(), cos, sin, interleaved)


def attention(q, k_codes, v_codes, k_scales, v_scales, table, ctx_lens, words, slopes, scale):
    """(o, bound), float64: the result, and how far the operator's may be off, element by element.

    The output's rounding, u |o|.  Each weight goes through float32 scores, sigmoid sums and exponentials
    (2^-12 of it, as in test_serving_attention.py) and is rounded to float16 times its block's scale c, by half a step:
    2^-11 of it, or 2^-25 of the unit, which is at most the row's largest w c, times a code of at most 448 for each
    key; and 2^-20."""
    B, Hq, Sq, D = q.shape
    Hkv = k_codes.shape[1]
    kd, vd = dequantised(k_codes, k_scales), dequantised(v_codes, v_scales)
    c_of = v_scales.double().repeat_interleave(BLOCK, 2)[..., None]
    o, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        ctx = int(ctx_lens[b])
        safe = table[b:b + 1].clamp(0, kd.shape[0] - 1)
        k, v, c = (ref.gather(x, safe, 0, ctx + Sq).repeat_interleave(Hq // Hkv, 0) for x in (kd, vd, c_of))
        see = torch.ones(Sq, ctx + Sq, dtype=torch.bool)
        see[:, ctx:] = torch.tensor([[bool(w >> t & 1) for t in range(Sq)] for w in words[b]])
        used = see.any(0)
        k, v, c = (torch.where(used[:, None], x, 0.0) for x in (k, v, c))
        p = scale * (q[b].double() @ k.transpose(1, 2))
        z = torch.where(see, torch.sigmoid(p), 0.0).flip(-1).cumsum(-1).flip(-1)
        x = (p - slopes.double()[:, None, None] * z).masked_fill(~see, -math.inf)
        w = torch.softmax(x, -1).masked_fill(~see.any(1)[:, None], 0.0)
        o[b] = w @ v
        unit = (w * c.transpose(1, 2)).amax(-1, keepdim=True)
        bound[b] = ref.U[q.dtype] * o[b].abs() + (2.0 ** -11 + 2.0 ** -12) * (w @ v.abs()) + int(used.sum()) * 448 * 2.0 ** -25 * unit + 2.0 ** -20
    return o, bound


def heads(qkv, Hq, Hkv, q_weight, k_weight, eps, cos, sin, at, interleaved):
    """(q, k, v) float64 of qkv [B, S, H, D] float64; `at` [B, S]: rows of the angles, -1 for none.  Differentiable."""
    out = []
    D = qkv.shape[-1]
    for x, w in ((qkv[:, :, :Hq], q_weight), (qkv[:, :, Hq:Hq + Hkv], k_weight)):
        y = x / ((x * x).sum(-1, keepdim=True) / D + eps).sqrt() * w
        if cos is not None:
            r = cos.shape[-1]
            c, s = cos.double()[at.clamp(min=0)][:, :, None], sin.double()[at.clamp(min=0)][:, :, None]
            first = torch.arange(r) * 2 if interleaved else torch.arange(r)
            second = first + 1 if interleaved else first + r
            a, b = y[..., first], y[..., second]
            z = y.clone()
            z[..., first], z[..., second] = a * c - b * s, b * c + a * s
            y = torch.where((at >= 0)[:, :, None, None], z, y)
        out.append(y.transpose(1, 2))
    return out[0], out[1], qkv[:, :, Hq + Hkv:].transpose(1, 2)
