"""Autograd front-ends of the sm_100a kernels for models written against the module API.

``use_kernels(x)`` is true for bf16 CUDA tensors unless the functional backend was requested; every function
below has a plain PyTorch evaluation for CPU / fp32 tensors so that the same model code runs on gloo."""
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from ..parallel.context import get_backend


def use_kernels(x: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype == torch.bfloat16 and get_backend() != "functional"


# ---------------------------------------------------------------------------------------------------------------------
# Recomputed activations.  The output of a cheap elementwise / normalisation op is usually consumed by a rotated linear,
# which would save it for its weight gradient although the op's own backward already keeps the op's INPUT.  Such outputs
# are tagged with how to rebuild them; a fused linear that receives a tagged tensor saves the (already saved) sources
# instead and rebuilds its input in backward, so the output lives only between the two forward launches.  For a GPT
# block this removes the [tokens, 4 d_model] GELU output and both LayerNorm outputs from the saved set (6 of 17
# d_model-sized rows per token and layer) for one extra elementwise pass each in backward.
# ---------------------------------------------------------------------------------------------------------------------
_RECOMPUTE = True


def set_activation_recompute(on: bool) -> bool:
    """Turns the tagging on or off (default on); returns the previous setting."""
    global _RECOMPUTE
    old, _RECOMPUTE = _RECOMPUTE, bool(on)
    return old


def activation_recompute() -> bool:
    """Whether outputs are tagged."""
    return _RECOMPUTE


def _learned(*values) -> bool:
    """Whether one of these constants of the kernels wants a gradient or carries a forward-mode derivative: only the evaluation in PyTorch
    operations has them."""
    for v in values:
        if torch.is_tensor(v):
            if v.requires_grad and torch.is_grad_enabled():
                return True
            if forward_ad._current_level >= 0 and forward_ad.unpack_dual(v).tangent is not None:
                return True
    return False


def _versions(out, srcs):
    return [t._version for t in (out, *srcs) if torch.is_tensor(t)]


def _tag(out: torch.Tensor, kind: str, *srcs):
    # a trace would keep the sources of the call that it was made from; an inference tensor cannot be kept for a backward
    if _RECOMPUTE and torch.is_grad_enabled() and torch._C._get_tracing_state() is None and \
            not any(torch.is_tensor(t) and t.is_inference() for t in srcs):
        out._rtp_recompute, out._rtp_versions = (kind, srcs), _versions(out, srcs)
    return out


def recompute_tag(x: torch.Tensor):
    """The (kind, sources) tag of a tensor produced by one of the ops below, or None: also where the tensor or one of its sources has been
    changed in place since (rebuilt from them it would be another one)."""
    tag = getattr(x, "_rtp_recompute", None)
    if tag is None or torch._C._get_tracing_state() is not None or x._rtp_versions != _versions(x, tag[1]):
        return None
    return tag


def recompute(kind: str, srcs):
    """Rebuilds a tagged tensor from its sources."""
    from . import kernels as K
    if kind == "gelu":
        return K.gelu_fwd(srcs[0])
    if kind == "swiglu":
        g, u = srcs
        return K.swiglu_fwd(g.reshape(-1, g.shape[-1]), u.reshape(-1, u.shape[-1])).view(g.shape)
    if kind == "swiglu_packed":
        y, nshard = srcs
        return K.swiglu_packed(y.reshape(-1, y.shape[-1]), nshard).view(*y.shape[:-1], y.shape[-1] // 2)
    if kind == "norm":
        x, weight, bias, eps, rms = srcs
        y = K.norm_fwd(x.reshape(-1, x.shape[-1]), None, weight, bias, eps=eps, rms=rms, save_h=False)[0]
        return y.view(x.shape)
    raise ValueError(f"unknown recompute kind {kind!r}")


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms):
        from . import kernels as K
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        y, h, mean, rstd = K.norm_fwd(x2, None, weight, bias, eps=eps, rms=rms, save_h=False)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.rms, ctx.has_bias, ctx.shape = rms, bias is not None, x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        from . import kernels as K
        x2, weight, mean, rstd = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        if weight.dtype == torch.bfloat16 and x2.shape[0] > 0:
            dx, dg, db = K.norm_bwd_params(dy2, x2, weight, mean, rstd, rms=ctx.rms, has_beta=ctx.has_bias)
            return dx.view(ctx.shape), dg, db, None, None
        dx, _, dg, db = K.norm_bwd(dy2, x2, weight, mean, rstd, rms=ctx.rms, has_beta=ctx.has_bias, want_dsub=False)
        return dx.view(ctx.shape), dg.to(weight.dtype), (db.to(weight.dtype) if ctx.has_bias else None), None, None


def layer_norm(x, weight, bias, eps=1e-5):
    if use_kernels(x) and x.shape[-1] % 8 == 0:
        y = _NormFn.apply(x, weight, bias, eps, False)
        return _tag(y, "norm", x, weight, bias, eps, False) if x.is_contiguous() else y
    return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)


def rms_norm(x, weight, eps=1e-5):
    if use_kernels(x) and x.shape[-1] % 8 == 0:
        y = _NormFn.apply(x, weight, None, eps, True)
        return _tag(y, "norm", x, weight, None, eps, True) if x.is_contiguous() else y
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * weight


class _CrossEntropyFn(torch.autograd.Function):
    """Mean (or, with ``mean=False``, summed) token cross-entropy of bf16 logits.  The input is never modified: the softmax
    gradient, produced in the same pass over the logits and already divided by the number of tokens, goes to a buffer of
    its own, and only when the logits need a gradient.  ``backward`` multiplies it by the incoming gradient, which for a
    loss that is differentiated itself is one and costs nothing."""

    @staticmethod
    def forward(ctx, logits, target, ignore_index, mean):
        from . import kernels as K
        lg = logits.reshape(-1, logits.shape[-1])
        if lg.stride(1) != 1 or lg.stride(0) % 8:
            lg = lg.contiguous()
        t = target.reshape(-1)
        grad = torch.empty(lg.shape, dtype=lg.dtype, device=lg.device) if ctx.needs_input_grad[0] else None
        if K.cross_entropy_one_read(lg):
            t = t.contiguous()
            cnt = K.ce_count(t, ignore_index) if mean else None
            rows = K.cross_entropy_to(lg, t, grad, scale=cnt[1:] if mean else None, ignore_index=ignore_index)
            loss = K.sum_f32(rows, torch.empty((), dtype=torch.float32, device=lg.device), divisor=cnt)
            ctx.save_for_backward(grad, None)
        else:
            rows = K.cross_entropy_to(lg, t, grad, grad_scale=1.0, ignore_index=ignore_index)
            n = (t != ignore_index).sum().clamp(min=1) if mean else torch.ones((), device=lg.device)
            loss = rows.sum() / n
            ctx.save_for_backward(grad, n)
        ctx.shape = logits.shape
        return loss

    @staticmethod
    def backward(ctx, g):
        from . import kernels as K
        grad, n = ctx.saved_tensors
        if n is None:
            grad = K.scale_unless_one_(grad, g.float().contiguous())
        else:
            grad = grad.mul_((g / n).to(grad.dtype))
        return grad.view(ctx.shape), None, None, None


def cross_entropy(logits, target, ignore_index=-100):
    """Mean token cross-entropy; the softmax gradient is produced in the same pass over the logits."""
    if use_kernels(logits) and logits.shape[-1] % 8 == 0:
        return _CrossEntropyFn.apply(logits, target, ignore_index, True)
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), target.reshape(-1), ignore_index=ignore_index)


class _SmallAttnFn(torch.autograd.Function):
    """q, k, v: [B, S, H, 64] -> [B, S, H, 64]; runs the short-sequence kernel on a packed [S*B, 3*H*64] buffer."""

    @staticmethod
    def forward(ctx, q, k, v):
        from . import kernels as K
        B, S, H, hd = q.shape
        packed = torch.cat([t.permute(1, 0, 2, 3).reshape(S * B, H * hd) for t in (q, k, v)], dim=1).contiguous()
        out = K.attn_small_fwd(packed, S, B, H, nshard=1, causal=True)
        ctx.save_for_backward(packed)
        ctx.dims = (B, S, H, hd)
        return out.view(S, B, H, hd).permute(1, 0, 2, 3)

    @staticmethod
    def backward(ctx, do):
        from . import kernels as K
        (packed,) = ctx.saved_tensors
        B, S, H, hd = ctx.dims
        do2 = do.permute(1, 0, 2, 3).reshape(S * B, H * hd).contiguous()
        dqkv = K.attn_small_bwd(packed, do2, S, B, H, nshard=1, causal=True)
        D = H * hd
        parts = [dqkv[:, i * D:(i + 1) * D].view(S, B, H, hd).permute(1, 0, 2, 3) for i in range(3)]
        return tuple(parts)


def causal_attention(q, k, v):
    """Causal self-attention on [B, S, H, hd] tensors (views are fine: the flash kernels take strides)."""
    B, S, H, hd = q.shape
    if use_kernels(q) and hd == 64 and S <= 96:
        return _SmallAttnFn.apply(q, k, v)
    if use_kernels(q) and hd in (64, 128):
        from .flash import flash_attention
        return flash_attention(q, k, v, causal=True)
    o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
    return o.transpose(1, 2)


def window_attention(q, k, v, window, sinks=0, sm_scale=None):
    """Causal attention over a sliding window with sinks: ``q`` [B, Sq, H, hd], ``k`` / ``v`` [B, Sk, Hk, hd] -> [B, Sq, H, hd] (views
    are fine; ``H`` a multiple of ``Hk``, whose heads serve ``H / Hk`` neighbouring query heads each).

    The queries are the last ``Sq <= Sk`` positions: query i stands at ``p = i + Sk - Sq`` and sees key j if ``j <= p`` and
    (``j > p - window`` or ``j < sinks``).  ``sm_scale``: factor on the scores, ``hd ** -0.5`` by default (one that
    wants a gradient is evaluated in PyTorch operations).

    bf16 CUDA tensors of head_dim 64 or 128 run on the tcgen05 kernels (``csrc/flash_attn.cu``): scores in fp32, probabilities and their
    gradients rounded to bf16 for the products, sums in fp32.  They take the maximum before the scale, so ``sm_scale`` has to lie between
    1e-30 and 1e30 there (``ValueError`` otherwise).  Hidden keys have a weight of exactly 0, which a dense product multiplies with
    their rows too: values and, in backward, keys have to be finite there; keys that are not leave the output as it is.  Other tensors are
    evaluated in PyTorch operations, with any scale and with all [B, H, Sq, Sk] scores in memory."""
    if use_kernels(q) and q.dim() == 4 and q.shape[3] in (64, 128) and q.numel() and not _learned(sm_scale):
        from .flash import window_attention as run
        return run(q, k, v, window, sinks, sm_scale)
    from .flash import check_window_args
    check_window_args(q, k, v, window, sinks)
    B, Sq, H, hd = q.shape
    Sk, Hk = k.shape[1:3]
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    qq = q.to(acc).transpose(1, 2).reshape(B, Hk, (H // Hk) * Sq, hd)
    s = (qq @ k.to(acc).permute(0, 2, 3, 1) * (hd ** -0.5 if sm_scale is None else sm_scale)).view(B, H, Sq, Sk)
    p, j = torch.arange(Sk - Sq, Sk, device=q.device)[:, None], torch.arange(Sk, device=q.device)
    s = s.masked_fill((j > p) | ((j <= p - window) & (j >= sinks)), float("-inf"))
    o = s.softmax(-1).view(B, Hk, (H // Hk) * Sq, Sk) @ v.to(acc).transpose(1, 2)
    return o.view(B, H, Sq, hd).transpose(1, 2).to(q.dtype)


class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        from . import kernels as K
        xc = x.contiguous()
        ctx.save_for_backward(xc)
        return K.gelu_fwd(xc)

    @staticmethod
    def backward(ctx, dy):
        from . import kernels as K
        (x,) = ctx.saved_tensors
        return K.gelu_bwd(x, dy.contiguous())


def gelu(x):
    if use_kernels(x) and x.numel() % 8 == 0:
        y = _GeluFn.apply(x)
        return _tag(y, "gelu", x) if x.is_contiguous() else y
    return F.gelu(x)


class _SwigluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, u):
        from . import kernels as K
        shape = g.shape
        g2, u2 = g.reshape(-1, shape[-1]).contiguous(), u.reshape(-1, shape[-1]).contiguous()
        ctx.save_for_backward(g2, u2)
        ctx.shape = shape
        return K.swiglu_fwd(g2, u2).view(shape)

    @staticmethod
    def backward(ctx, dy):
        from . import kernels as K
        g2, u2 = ctx.saved_tensors
        dg, du = K.swiglu_bwd(g2, u2, dy.reshape(-1, ctx.shape[-1]).contiguous())
        return dg.view(ctx.shape), du.view(ctx.shape)


def swiglu(g, u):
    """silu(g) * u."""
    if use_kernels(g) and g.shape[-1] % 8 == 0:
        # halves of a packed projection arrive as strided views: the contiguous copies made here are the tensors the
        # kernel's backward keeps, and the ones a following linear rebuilds its input from
        g, u = g.contiguous(), u.contiguous()
        return _tag(_SwigluFn.apply(g, u), "swiglu", g, u)
    return F.silu(g) * u


class _SwigluPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, nshard):
        from . import kernels as K
        y2 = y.reshape(-1, y.shape[-1]).contiguous()
        ctx.save_for_backward(y2)
        ctx.shape, ctx.nshard = y.shape, nshard
        return K.swiglu_packed(y2, nshard).view(*y.shape[:-1], y.shape[-1] // 2)

    @staticmethod
    def backward(ctx, dy):
        from . import kernels as K
        (y2,) = ctx.saved_tensors
        return K.swiglu_packed_bwd(y2, dy.reshape(y2.shape[0], -1).contiguous(), ctx.nshard).view(ctx.shape), None


def _split_packed(y, parts, nshard):
    """The ``parts`` projections of a rotated packed projection, whose columns are grouped per shard:
    [p0_j | p1_j | ...] for j = 0..nshard-1."""
    y = y.view(*y.shape[:-1], nshard, parts, y.shape[-1] // (nshard * parts))
    return [y[..., k, :].reshape(*y.shape[:-3], -1) for k in range(parts)]


def swiglu_packed(y, nshard=1):
    """silu(g) * u of a rotated packed gate / up projection [..., 2 * F], read where it lies (no split copies)."""
    if use_kernels(y) and y.shape[-1] % (16 * nshard) == 0 and y.is_contiguous() and y.data_ptr() % 16 == 0:
        return _tag(_SwigluPackedFn.apply(y, nshard), "swiglu_packed", y, nshard)
    return swiglu(*_split_packed(y, 2, nshard))


def gated_mlp(x, w_gate_up, w_down):
    """Gated feed-forward block ``(silu(x Wg^T) * (x Wu^T)) Wd^T``: ``x`` [..., D], ``w_gate_up`` [2 * F, D] (the rows of ``Wg`` before those
    of ``Wu``), ``w_down`` [O, F] -> [..., O].

    bf16 CUDA tensors whose sizes are multiples of 8 run on the tcgen05 GEMM kernel with the activation and the product in its epilogue
    (``ops/mlp.py``): sums in fp32; the product of gate and up and the gradients of both are rounded to bf16, as the operands
    of the products behind them, and gate and up where they are kept for backward."""
    from . import mlp
    if get_backend() != "functional" and x.dim() and w_gate_up.dim() == 2 and w_down.dim() == 2 and mlp.kernel_takes(x, w_gate_up, w_down):
        return mlp.gated_mlp(x, w_gate_up, w_down)
    mlp.check_args(x, w_gate_up, w_down)
    g, u = F.linear(x, w_gate_up).chunk(2, dim=-1)
    return F.linear(F.silu(g) * u, w_down)


class _RopeAttnPackedFn(torch.autograd.Function):
    """Causal self-attention of a packed projection [B * S, 3 * D] with rotary embedding of q and k.  Forward makes one rotated
    copy of the projection, which the flash kernels read in place; backward turns the q and k gradients back inside the
    packed gradient that they wrote."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, B, S, H, nshard):
        from . import flash, kernels as K
        hd = qkv.shape[1] // (3 * H)
        rot = K.rope_packed(qkv, cos, sin, hd, nshard)
        out, lse = flash.packed_fwd(rot, B, S, H, nshard, causal=True)
        ctx.save_for_backward(rot, out, lse, cos, sin)
        ctx.cfg = (B, S, H, nshard, hd)
        return out

    @staticmethod
    def backward(ctx, dout):
        from . import flash, kernels as K
        rot, out, lse, cos, sin = ctx.saved_tensors
        B, S, H, nshard, hd = ctx.cfg
        dqkv = flash.packed_bwd(rot, out, lse, dout, B, S, H, nshard, causal=True)
        return (K.rope_packed(dqkv, cos, sin, hd, nshard, out=dqkv, backward=True),) + (None,) * 6


def rope_attention_packed(qkv, cos, sin, heads, nshard=1):
    """Causal self-attention with rotary embedding on a rotated packed projection ``qkv`` [B, S, 3 * D] (its columns grouped
    per shard) -> [B, S, D].  ``cos`` / ``sin``: [S, hd / 2].  None: not a case for these kernels (also where the shards' column
    groups cut through heads)."""
    B, S, W = qkv.shape
    hd = W // (3 * heads)
    small = hd == 64 and S <= 96             # the short-sequence kernels take those
    whole = heads % nshard == 0
    if use_kernels(qkv) and hd in (64, 128) and whole and not small and qkv.is_contiguous() and qkv.data_ptr() % 16 == 0:
        c, s = cos.float().contiguous(), sin.float().contiguous()
        return _RopeAttnPackedFn.apply(qkv.view(B * S, W), c, s, B, S, heads, nshard).view(B, S, W // 3)
    return None


def rotary(q, k, positions, freqs, layout="half", magnitude=1.0):
    """Rotary positions: turns the pairs of the first ``rotary_dim`` elements of every head of ``q`` [B, S, H, hd] and ``k``
    [B, S, Hk, hd] (None: q alone; any strides) by ``positions * freqs`` radians and returns new (q, k).

    ``positions``: int64 / int32 [S] or [B, S], any values.  ``freqs``: float64 [rotary_dim / 2], see
    ``ops.rotary.rotary_frequencies``.  ``layout``: pairs ``(x[i], x[i + rotary_dim / 2])`` for ``"half"``, ``(x[2i], x[2i + 1])`` for
    ``"interleaved"``.  ``magnitude``: factor on the rotated part (``ops.rotary.rotary_magnitude``).  Frequencies or a
    magnitude that want a gradient are evaluated in PyTorch operations."""
    from . import rotary as R
    if R.kernel_takes(q) and get_backend() != "functional" and not _learned(freqs, magnitude):
        return R.rotary(q, k, positions, freqs, layout, magnitude)
    return R.rotary_plain(q, k, positions, freqs, layout, magnitude)


def rotary_window_attention(qkv, positions, freqs, heads, kv_heads=None, layout="half", magnitude=1.0, window=None, sinks=0):
    """Rotary positions and causal attention of a packed projection ``qkv`` [B, S, (heads + 2 * kv_heads) * hd], whose columns are the
    heads of q, then those of k, then those of v -> [B, S, heads * hd].  ``window`` / ``sinks`` as in :func:`window_attention` (None:
    every earlier token is seen); the other arguments as in :func:`rotary`."""
    from . import flash, rotary as R
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.dim() != 3 or heads < 1 or kv_heads < 1 or qkv.shape[2] % (heads + 2 * kv_heads):
        raise ValueError(f"rotary_window_attention: qkv must be [B, S, (heads + 2 * kv_heads) * hd], got {tuple(qkv.shape)} for {heads} and {kv_heads} heads")
    B, S, W = map(int, qkv.shape)             # tensors while a trace is made
    hd = W // (heads + 2 * kv_heads)
    window = max(S, 1) if window is None else window
    q, k, v = qkv.view(B, S, heads + 2 * kv_heads, hd).split((heads, kv_heads, kv_heads), dim=2)
    R.check_args(q, k, positions, freqs, layout)
    flash.check_window_args(q, k, v, window, sinks)
    if use_kernels(qkv) and hd in (64, 128) and qkv.numel() and qkv.is_contiguous() and qkv.data_ptr() % 16 == 0 and not _learned(freqs, magnitude):
        return flash.rotary_window_attention_packed(qkv, positions, freqs, heads, kv_heads, layout, magnitude, window, sinks)
    q, k = rotary(q, k, positions, freqs, layout, magnitude)
    return window_attention(q, k, v, window, sinks).reshape(B, S, heads * hd)


# ---------------------------------------------------------------------------------------------------------------------
# LM head + cross-entropy without the [tokens, vocab] logits
# ---------------------------------------------------------------------------------------------------------------------
class _ChunkedHeadLossFn(torch.autograd.Function):
    """Mean token cross-entropy of ``head(hidden)``, evaluated ``chunk_rows`` tokens at a time.  Forward AND backward of the
    head run chunk by chunk inside ``forward`` (the loss is the last op of a language model, so nothing is lost by doing
    the head's backward early): only one chunk of logits and of their gradient exists at any time — 0.4 GB instead of
    2 x 1.6 GB for 16 384 tokens of a 50 304-word vocabulary at 4 096 rows per chunk.  ``backward`` scales the stashed
    gradients by the incoming one.  The reference computes the full logits and hands them to ``nn.CrossEntropyLoss``
    (benchmarks/rtp_benchmark.py:182, rtp/models/transformer_lm_rtp.py:218-228).

    A rotated head pushes its shards once per chunk and direction; with N ranks that is 2 (N-1)/N of the head's bytes per
    chunk over NVLink, small against a chunk's GEMMs."""

    @staticmethod
    def forward(ctx, hidden, target, head, chunk_rows, ignore_index, *params):
        h2d = hidden.reshape(-1, hidden.shape[-1])
        t1d = target.reshape(-1)
        M = h2d.shape[0]
        n_valid = (t1d != ignore_index).sum().clamp(min=1)
        dx = torch.empty_like(h2d)
        gsum = [None] * len(params)
        total = torch.zeros((), dtype=torch.float32, device=h2d.device)
        for r0 in range(0, M, chunk_rows):
            r1 = min(r0 + chunk_rows, M)
            with torch.enable_grad():
                hc = h2d[r0:r1].detach().requires_grad_(True)
                logits = head(hc)
                # sum over the chunk's tokens; the division by the global count happens once, below
                tc = t1d[r0:r1]
                if use_kernels(logits) and logits.shape[-1] % 8 == 0:
                    loss_c = _CrossEntropyFn.apply(logits, tc, ignore_index, False)
                else:
                    loss_c = F.cross_entropy(logits.float(), tc, ignore_index=ignore_index, reduction="sum")
                grads = torch.autograd.grad(loss_c, [hc] + list(params), allow_unused=True)
            total += loss_c.detach().float()
            dx[r0:r1] = grads[0]
            for k, g in enumerate(grads[1:]):
                if g is None:
                    continue
                gsum[k] = g.detach().float() if gsum[k] is None else gsum[k].add_(g)     # fp32 across the chunks
            del logits, loss_c, grads, hc
        inv = 1.0 / n_valid.to(torch.float32)
        ctx.save_for_backward(dx, inv, *[g if g is not None else torch.zeros(0, device=h2d.device) for g in gsum])
        ctx.has = [g is not None for g in gsum]
        ctx.dtypes = [p.dtype for p in params]
        ctx.shape = hidden.shape
        return total * inv

    @staticmethod
    def backward(ctx, gout):
        dx, inv, *gs = ctx.saved_tensors
        scale = (gout.to(torch.float32) * inv)
        dh = (dx.float() * scale).to(dx.dtype).view(ctx.shape)
        gp = [(g * scale).to(dt) if has else None for g, has, dt in zip(gs, ctx.has, ctx.dtypes)]
        return (dh, None, None, None, None, *gp)


def chunked_head_loss(hidden, target, head, chunk_rows: int = 4096, ignore_index: int = -100):
    """``cross_entropy(head(hidden), target)`` without ever holding more than ``chunk_rows`` rows of logits (see
    :class:`_ChunkedHeadLossFn`).  ``head`` is any module (a rotated ``ColumnParallelLinear`` included); its parameters
    receive their gradients through autograd as usual."""
    params = [p for p in head.parameters() if p.requires_grad]
    return _ChunkedHeadLossFn.apply(hidden, target, head, int(chunk_rows), ignore_index, *params)
