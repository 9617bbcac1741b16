"""Llama-shaped decoder-only LM with rotated weights: RMSNorm, rotary position embedding, SwiGLU FFN, no biases.

Rotation plan per block: packed QKV projection = column-rotated ``D -> 3D`` whose shard rows are
``[q_r; k_r; v_r]`` (heads/N heads per shard), attention over all heads locally (each rank holds the full
projection of its own batch once the N column blocks are assembled), optionally over a window of recent tokens and the
first few, output projection = row-rotated ``D -> D``;
SwiGLU = column-rotated packed gate/up ``D -> 2F`` (shard rows ``[gate_r; up_r]``) and row-rotated ``F -> D``.
Embedding ``[V, D/N]`` and LM head ``[V/N, D]`` rotate as well.  Activations are ``[batch, seq, dim]``."""
from dataclasses import dataclass

import torch
import torch.nn as nn

from ..module.embedding import ParallelEmbedding
from ..module.linear import ColumnParallelLinear, RowParallelLinear
from ..parallel.context import get_context
from ..parallel import fused
from ..ops import functional as FO
from ..ops.rotary import LAYOUTS, SCALINGS, rotary_frequencies, rotary_magnitude


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    d_model: int = 5120
    n_layers: int = 40
    n_heads: int = 40
    d_ff: int = 13824
    max_seq_len: int = 2048
    rope_theta: float = 10000.0
    norm_eps: float = 1e-5
    init_std: float = 0.02
    loss_chunk_rows: int = 0     # > 0: LM head + cross-entropy this many tokens at a time (no full logits)
    # attention over the last `window` tokens and the first `sinks` (0: over all earlier ones)
    window: int = 0
    sinks: int = 0
    # rotary positions: layout of the pairs, rotated part of a head (0: all of it), stretched frequencies (ops.rotary.rotary_frequencies)
    rope_layout: str = "interleaved"
    rotary_dim: int = 0
    rope_scaling: str = "none"
    rope_factor: float = 1.0
    rope_original_length: int = 4096

    def __post_init__(self):
        if self.window < 0 or self.sinks < 0 or (self.sinks and not self.window):
            raise ValueError(f"window and sinks must not be negative, and sinks go with a window: got {self.window} and {self.sinks}")
        if self.rope_layout not in LAYOUTS or self.rope_scaling not in SCALINGS:
            raise ValueError(f"rope_layout must be one of {LAYOUTS} and rope_scaling one of {SCALINGS}, got {self.rope_layout!r} and {self.rope_scaling!r}")
        if self.rotary_dim < 0 or self.rotary_dim % 2 or self.rotary_dim > self.d_model // self.n_heads:
            raise ValueError(f"rotary_dim must be even and lie inside the head, got {self.rotary_dim}")

    @property
    def table_rope(self):
        """Whole heads in the interleaved layout with plain frequencies under full causal attention: the packed kernels' case."""
        return not self.window and self.rope_layout == "interleaved" and self.rotary_dim in (0, self.d_model // self.n_heads) and \
            self.rope_scaling == "none"

    @staticmethod
    def llama_13b():
        return LlamaConfig()


class RMSNorm(nn.Module):
    def __init__(self, dim, eps=1e-5, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, x):
        if FO.use_kernels(x):
            return FO.rms_norm(x, self.weight, self.eps)
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)).to(x.dtype) * self.weight


def rope_tables(seq_len, head_dim, theta, device, dtype=torch.float32):
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    t = torch.arange(seq_len, device=device, dtype=torch.float32)
    fr = torch.outer(t, inv)
    return fr.cos().to(dtype), fr.sin().to(dtype)


def apply_rope(x, cos, sin):
    """x: [B, S, H, hd]; rotates pairs (x[2i], x[2i+1])."""
    if FO.use_kernels(x) and x.shape[-1] % 16 == 0:
        from ..ops import kernels as K
        return K.rope(x, cos, sin, inner=1)
    x1, x2 = x[..., 0::2], x[..., 1::2]
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    out = torch.stack([x1 * c - x2 * s, x1 * s + x2 * c], dim=-1)
    return out.flatten(-2).to(x.dtype)


class LlamaBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig, device=None, dtype=None, group=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype, group=group, bias=False)
        ctx = get_context(group)
        self.cfg, self.N = cfg, ctx.world
        self.norm1 = RMSNorm(cfg.d_model, cfg.norm_eps, device, dtype)
        self.qkv = ColumnParallelLinear(cfg.d_model, 3 * cfg.d_model, packed_parts=3, **kw)
        self.proj = RowParallelLinear(cfg.d_model, cfg.d_model, **kw)
        self.norm2 = RMSNorm(cfg.d_model, cfg.norm_eps, device, dtype)
        self.gate_up = ColumnParallelLinear(cfg.d_model, 2 * cfg.d_ff, packed_parts=2, **kw)
        self.down = RowParallelLinear(cfg.d_ff, cfg.d_model, **kw)

    def _table_attention(self, qkv, cos, sin):
        cfg = self.cfg
        B, S, W = qkv.shape
        a = FO.rope_attention_packed(qkv, cos, sin, cfg.n_heads, self.N)
        if a is None:
            heads = (B, S, cfg.n_heads, W // (3 * cfg.n_heads))
            q, k, v = FO._split_packed(qkv, 3, self.N)
            q = apply_rope(q.view(heads), cos, sin)
            k = apply_rope(k.view(heads), cos, sin)
            a = FO.causal_attention(q, k, v.view(heads)).reshape(B, S, W // 3)      # [B, S, H, hd]
        return a

    def _window_attention(self, qkv, positions, freqs):
        cfg = self.cfg
        if self.N > 1:                                             # the shards' column groups side by side -> q | k | v
            qkv = torch.cat(FO._split_packed(qkv, 3, self.N), dim=-1)
        return FO.rotary_window_attention(qkv, positions, freqs, cfg.n_heads, layout=cfg.rope_layout,
                                          magnitude=rotary_magnitude(cfg.rope_scaling, cfg.rope_factor),
                                          window=cfg.window or None, sinks=cfg.sinks)

    def forward(self, x, cos, sin):
        """``cos`` and ``sin``: the tables, or positions and frequencies in their place (see ``LlamaConfig.table_rope``)."""
        qkv = self.qkv(self.norm1(x))
        x = x + self.proj((self._table_attention if self.cfg.table_rope else self._window_attention)(qkv, cos, sin))
        h = self.norm2(x)
        y = fused.gated_mlp(self.gate_up, self.down, h)
        return x + (self.down(FO.swiglu_packed(self.gate_up(h), self.N)) if y is None else y)


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig, device=None, dtype=None, group=None):
        super().__init__()
        self.cfg = cfg
        self.tok = ParallelEmbedding(cfg.vocab_size, cfg.d_model, device=device, dtype=dtype, group=group)
        self.blocks = nn.ModuleList([LlamaBlock(cfg, device, dtype, group) for _ in range(cfg.n_layers)])
        self.norm = RMSNorm(cfg.d_model, cfg.norm_eps, device, dtype)
        self.head = ColumnParallelLinear(cfg.d_model, cfg.vocab_size, bias=False, device=device, dtype=dtype, group=group)
        with torch.no_grad():
            for p in self.parameters():
                if p.dim() > 1:
                    p.normal_(0.0, cfg.init_std)

    def forward(self, ids, targets=None):
        B, S = ids.shape
        cfg = self.cfg
        hd = cfg.d_model // cfg.n_heads
        if cfg.table_rope:
            rope = rope_tables(S, hd, cfg.rope_theta, ids.device)
        else:
            rope = (torch.arange(S, device=ids.device),
                    rotary_frequencies(cfg.rotary_dim or hd, cfg.rope_theta, cfg.rope_scaling, cfg.rope_factor, cfg.rope_original_length,
                                       device=ids.device))
        x = self.tok(ids)
        for blk in self.blocks:
            x = blk(x, *rope)
        if targets is not None and self.cfg.loss_chunk_rows > 0:
            # head and loss chunk by chunk: the [tokens, vocab] logits never exist as a whole
            return FO.chunked_head_loss(self.norm(x), targets, self.head, self.cfg.loss_chunk_rows)
        logits = self.head(self.norm(x))
        if targets is None:
            return logits
        return FO.cross_entropy(logits, targets)
