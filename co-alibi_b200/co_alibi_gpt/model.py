"""A small GPT whose self-attention is Co-ALiBi: the caller side of the kernels.

The reference repository ships the attention operator only (no model code), so
this module is new.  Every block runs ``co_alibi_attention`` (the sm_100a
kernels behind the reference's Python API) with causal masking; positions come
from the Co-ALiBi bias alone, so there is no position embedding.  Layer layout:
token embedding -> n_layer x [LayerNorm -> QKV -> Co-ALiBi attention -> output
projection -> residual, LayerNorm -> MLP (4x, GELU) -> residual] -> LayerNorm ->
LM head tied to the embedding -> cross-entropy.
"""
import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F


@dataclass
class GPTConfig:
    n_layer: int = 12
    d_model: int = 768
    n_head: int = 12
    vocab: int = 50304
    seq_len: int = 1024
    mlp_ratio: int = 4
    bias_max: float = 8.0
    init_std: float = 0.02
    rotary_dim: int = 0  # first elements of each query and key head rotated by position (0: none); a multiple of 16


def rotate_heads(x, cos, sin):
    """x [B, H, S, D] with its first R elements rotated in halves by tables [S, R / 2]
    (``co_alibi_attn.serving.rotary_tables``), in float32; differentiable."""
    r = cos.shape[-1]
    a, b = x[..., :r].float(), x[..., r:2 * r].float()
    return torch.cat(((a * cos - b * sin).to(x.dtype), (b * cos + a * sin).to(x.dtype), x[..., 2 * r:]), -1)


_rotary_cache = {}


def _rotary(rotary_dim, seq_len, S, device):
    """cos and sin of the first S positions, of tables that are built once per device for
    ``seq_len`` positions and again when a longer input comes: building them copies from
    the host, which stalls the stream and cannot be captured in a CUDA graph."""
    key = (rotary_dim, device)
    tables = _rotary_cache.get(key)
    if tables is None or tables[0].shape[0] < S:
        from co_alibi_attn import serving
        from co_alibi_attn.co_alibi_attn import _not_capturing
        _not_capturing(device, f"the rotary table of {S} positions")
        with torch.inference_mode(False):  # kept for training too
            tables = serving.rotary_tables(rotary_dim, max(S, seq_len), device=device)
        _rotary_cache[key] = tables
    return tables[0][:S], tables[1][:S]


class CoALiBiSelfAttention(nn.Module):
    """QKV projection, Co-ALiBi causal attention over [B, H, S, D] heads, output projection."""

    def __init__(self, cfg: GPTConfig, attn_fn):
        super().__init__()
        assert cfg.d_model % cfg.n_head == 0
        self.n_head = cfg.n_head
        self.head_dim = cfg.d_model // cfg.n_head
        if not 0 <= cfg.rotary_dim <= self.head_dim or cfg.rotary_dim % 16:  # as append_paged_kv takes it
            raise ValueError(f"rotary_dim must be a multiple of 16 up to the head width {self.head_dim}, got {cfg.rotary_dim}")
        self.qkv = nn.Linear(cfg.d_model, 3 * cfg.d_model)
        self.proj = nn.Linear(cfg.d_model, cfg.d_model)
        self.attn_fn = attn_fn
        self.bias_max = cfg.bias_max
        self.rotary_dim = cfg.rotary_dim
        self.seq_len = cfg.seq_len

    def heads(self, x):
        """Queries, keys and values of x [B, S, C] as [B, H, S, D] views of the fused projection."""
        B, S, _ = x.shape
        qkv = self.qkv(x).view(B, S, 3, self.n_head, self.head_dim)
        return [t.transpose(1, 2) for t in qkv.unbind(dim=2)]

    def forward(self, x):
        B, S, C = x.shape
        # contiguous: the kernels take row-major heads
        q, k, v = (t.contiguous() for t in self.heads(x))
        if self.rotary_dim:
            cos, sin = _rotary(self.rotary_dim, self.seq_len, S, x.device)
            q, k = rotate_heads(q, cos, sin), rotate_heads(k, cos, sin)
        y = self.attn_fn(q, k, v, causal=True, bias_max=self.bias_max)
        return self.proj(y.transpose(1, 2).reshape(B, S, C))


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig, attn_fn):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.d_model)
        self.attn = CoALiBiSelfAttention(cfg, attn_fn)
        self.ln2 = nn.LayerNorm(cfg.d_model)
        self.fc = nn.Linear(cfg.d_model, cfg.mlp_ratio * cfg.d_model)
        self.out = nn.Linear(cfg.mlp_ratio * cfg.d_model, cfg.d_model)

    def forward(self, x):
        x = x + self.attn(self.ln1(x))
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))


class CoALiBiGPT(nn.Module):
    """``forward(tokens, targets=None)`` -> logits, or the mean cross-entropy when
    targets are given.  ``attn_fn(q, k, v, causal, bias_max)`` defaults to the
    package's ``co_alibi_attention`` (CUDA only; no other attention is used)."""

    def __init__(self, cfg: GPTConfig, attn_fn=None):
        super().__init__()
        if attn_fn is None:
            from co_alibi_attn import co_alibi_attention
            attn_fn = co_alibi_attention
        self.cfg = cfg
        self.emb = nn.Embedding(cfg.vocab, cfg.d_model)
        self.blocks = nn.ModuleList(Block(cfg, attn_fn) for _ in range(cfg.n_layer))
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.reset_parameters()

    def reset_parameters(self, generator=None):
        """Weights ~ N(0, init_std) (residual output projections scaled by
        1/sqrt(2 n_layer)), biases 0, LayerNorm affine 1 / 0."""
        std = self.cfg.init_std
        with torch.no_grad():
            for name, p in self.named_parameters():
                if name.endswith("bias"):
                    p.zero_()
                elif ".ln" in name or name.startswith("ln_f"):
                    p.fill_(1.0)
                else:
                    s = std / math.sqrt(2 * self.cfg.n_layer) if name.endswith(("proj.weight", "out.weight")) else std
                    p.copy_(torch.randn(p.shape, generator=generator) * s)

    def forward(self, tokens, targets=None):
        x = self.emb(tokens)
        for blk in self.blocks:
            x = blk(x)
        logits = F.linear(self.ln_f(x), self.emb.weight)
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.shape[-1]), targets.reshape(-1))

    def flops_per_token(self):
        """Training FLOPs per token: 6 x (matmul parameters) for the dense layers and
        the tied LM head, plus the causal attention GEMMs (QK^T and PV forward, five
        GEMMs backward, on the visible half of the score matrix)."""
        c = self.cfg
        dense = c.n_layer * (4 * c.d_model * c.d_model + 2 * c.mlp_ratio * c.d_model * c.d_model)
        head = c.vocab * c.d_model
        attn = c.n_layer * 14 * c.d_model * (c.seq_len + 1) / 2
        return 6 * (dense + head) + attn
