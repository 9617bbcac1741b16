"""Rotary positions of queries and keys on the kernel of ``csrc/rotary.cu``: interleaved or half layout, the whole head or its first
part, any positions, stretched frequencies for long contexts, bf16 / fp16 / fp32.

The angles are made inside the kernel from positions and frequencies in 64 bits, so no table bounds the positions.  The Llama-shaped
model's own tables (``models.llama.rope_tables``, ``ops.kernels.rope``) stay for whole heads in the interleaved layout at positions
0, 1, 2, ..."""
import ctypes as C
import math
import struct

import torch

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
LAYOUTS = ("half", "interleaved")
SCALINGS = ("none", "linear", "ntk", "yarn")


_declared = False


def _L():
    global _declared
    L = _lib.lib()
    if not _declared:
        L.rtp_rotary.argtypes = [C.c_char_p, C.c_void_p]
        L.rtp_rotary_last_error.restype = C.c_char_p
        _declared = True
    return L


def rotary_frequencies(rotary_dim, theta=10000.0, scaling="none", factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device=None):
    """Angles (radians, float64 ``[rotary_dim / 2]``) by which one position turns each pair: ``theta ** (-2 i / rotary_dim)``,
    stretched for contexts ``factor`` times as long as the ``original_length`` of training:

    * ``"linear"``: every frequency divided by ``factor`` (positions squeezed);
    * ``"ntk"``: the base grows to ``theta * factor ** (d / (d - 2))``, which leaves the fastest pair alone and divides the slowest
      by ``factor``;
    * ``"yarn"`` (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", by-parts interpolation): pairs
      that turn at least ``beta_fast`` times within ``original_length`` stay, those that turn at most ``beta_slow`` times are divided
      by ``factor``, with a linear ramp between; goes with :func:`rotary_magnitude`."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}: one of {SCALINGS}")
    if not theta > 0 or not factor > 0 or not original_length > 0:
        raise ValueError("theta, factor and original_length must be positive")
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if not beta_fast > beta_slow:
            raise ValueError("beta_fast must be larger than beta_slow")
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f


def rotary_magnitude(scaling="none", factor=1.0):
    """The factor that goes with :func:`rotary_frequencies` on rotated queries and keys: ``0.1 ln(factor) + 1`` for ``"yarn"`` and
    ``factor > 1``, else 1."""
    return 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1 else 1.0


def _good_args(q, k, positions, freqs, layout):
    a, p, f = q.shape, positions.shape, freqs.shape
    if len(a) != 4 or len(f) != 1 or not 0 < 2 * f[0] <= a[3] or layout not in LAYOUTS:
        return False
    if not (p == a[1:2] or p == a[:2] or (len(p) == 2 and p[0] == 1 and p[1] == a[1])):
        return False
    if k is not None:
        b = k.shape
        if len(b) != 4 or b[0] != a[0] or b[1] != a[1] or b[3] != a[3] or k.dtype != q.dtype or k.device != q.device:
            return False
    on = q.device
    return q.dtype in _TYPES and positions.dtype in (torch.int64, torch.int32) and freqs.dtype == torch.float64 and positions.device == on and \
        freqs.device == on


def check_args(q, k, positions, freqs, layout):
    if _good_args(q, k, positions, freqs, layout):
        return
    if layout not in LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}: one of {LAYOUTS}")
    if q.dim() != 4:
        raise ValueError(f"q must be [B, S, heads, head_dim], got shape {tuple(q.shape)}")
    if not q.dtype.is_floating_point:
        raise ValueError(f"q must be a floating-point tensor, got {q.dtype}")
    if k is not None:
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise ValueError(f"k must be [B, S, heads, head_dim] with q's batch, length and head_dim: got {tuple(k.shape)} beside {tuple(q.shape)}")
        if k.dtype != q.dtype or k.device != q.device:
            raise ValueError("q and k must have the same type and device")
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"positions must be int64 or int32, got {positions.dtype}")
    if positions.dim() not in (1, 2) or positions.shape[-1] != q.shape[1] or (positions.dim() == 2 and positions.shape[0] not in (1, q.shape[0])):
        raise ValueError(f"positions must be [S] or [B, S] for q {tuple(q.shape)}, got {tuple(positions.shape)}")
    if freqs.dim() != 1 or freqs.dtype != torch.float64 or not 0 < 2 * freqs.shape[0] <= q.shape[3]:
        raise ValueError(f"freqs must be float64 [rotary_dim / 2] with rotary_dim <= head_dim, got {freqs.dtype} {tuple(freqs.shape)}")
    if positions.device != q.device or freqs.device != q.device:
        raise ValueError("q, positions and freqs must be on the same device")


def kernel_takes(q):
    """CUDA tensors of one of the kernel's types and an even head_dim up to 256."""
    return q.is_cuda and q.dtype in _TYPES and q.dim() == 4 and q.shape[3] <= 256 and q.shape[3] % 2 == 0


# RtpRotary (csrc/kernels.h) as it lies in memory: packing the numbers takes a quarter of the time that filling a ctypes structure does
_PACK = struct.Struct("@4P16qP2qPf10i0P").pack
_NO_STRIDES = (0, 0, 0, 0)


def _rotate(q, k, positions, freqs, half, magnitude, backward, qo=None, ko=None):
    """One launch for q and / or k (either may be None), into new tensors or qo and ko (which may be q and k)."""
    one = q if q is not None else k
    if one.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(one.device):
            return _rotate(q, k, positions, freqs, half, magnitude, backward, qo, ko)
    qp = kp = qop = kop = H = Hk = 0
    qs = ks = qos = kos = _NO_STRIDES
    if q is not None:
        qs = q.stride()
        if qs[3] != 1:
            q = q.contiguous()                        # lives until the launch, as k's below
            qs = q.stride()
        if qo is None:
            qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        B, S, H, hd = q.shape
        qp, qop, qos = q.data_ptr(), qo.data_ptr(), qo.stride()
    if k is not None:
        ks = k.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        if ko is None:
            ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        B, S, Hk, hd = k.shape
        kp, kop, kos = k.data_ptr(), ko.data_ptr(), ko.stride()
    freqs = freqs.contiguous()
    st = positions.stride()
    a = _PACK(qp, kp, qop, kop, *qs, *ks, *qos, *kos, positions.data_ptr(), st[0] if len(st) == 2 and positions.shape[0] > 1 else 0, st[-1],
              freqs.data_ptr(), magnitude, positions.dtype == torch.int64, B, S, H, Hk, hd, 2 * freqs.shape[0], half, _TYPES[one.dtype],
              backward)
    L = _L()
    if L.rtp_rotary(a, _lib.stream_ptr()) != 0:
        raise RuntimeError("rotary: " + L.rtp_rotary_last_error().decode())
    _lib.launches += 1
    return qo, ko


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, half, magnitude, backward):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        ctx.cfg = (half, magnitude, backward)
        return _rotate(q, k, positions, freqs, half, magnitude, backward)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, freqs = ctx.saved_tensors
        half, magnitude, backward = ctx.cfg
        needs = ctx.needs_input_grad
        dq = dq if needs[0] else None
        dk = dk if needs[1] else None
        if dq is None and dk is None:
            return (None,) * 7
        # the transposed map is the same one with the angles negated
        step = _RotaryFn.apply if torch.is_grad_enabled() else _rotate
        gq, gk = step(dq, dk, positions, freqs, half, magnitude, not backward)
        return (gq, gk) + (None,) * 5


def rotary(q, k, positions, freqs, layout="half", magnitude=1.0):
    """Kernel front-end of ``ops.functional.rotary`` (same arguments); raises for what the kernel does not take."""
    check_args(q, k, positions, freqs, layout)
    if not kernel_takes(q):
        raise ValueError(f"rotary: the kernel takes bf16, fp16 and fp32 CUDA tensors with an even head_dim up to 256, got {q.dtype} {tuple(q.shape)}")
    if torch.is_grad_enabled() and (freqs.requires_grad or (torch.is_tensor(magnitude) and magnitude.requires_grad)):
        raise ValueError("rotary: the kernel has no gradient for freqs and magnitude")
    half, magnitude = layout == "half", float(magnitude)
    if _lib.through_autograd(q, k):
        return _RotaryFn.apply(q, k, positions, freqs, half, magnitude, False)
    return _rotate(q, k, positions, freqs, half, magnitude, False)


def rotary_plain(q, k, positions, freqs, layout="half", magnitude=1.0):
    """The same in PyTorch operations: angles in 64 bits, the rest in 32 (64 for float64 tensors)."""
    check_args(q, k, positions, freqs, layout)
    rot, n = 2 * freqs.shape[0], freqs.shape[0]
    angle = (positions.double()[..., None] * freqs)
    angle = angle[None] if angle.dim() == 2 else angle

    def turn(x):
        acc = torch.float64 if x.dtype == torch.float64 else torch.float32
        cos, sin = ((f * magnitude).to(acc)[:, :, None] for f in (angle.cos(), angle.sin()))
        y = x.to(acc)
        a, b = (y[..., :n], y[..., n:rot]) if layout == "half" else (y[..., 0:rot:2], y[..., 1:rot:2])
        c, d = a * cos - b * sin, a * sin + b * cos
        t = torch.cat([c, d], dim=-1) if layout == "half" else torch.stack([c, d], dim=-1).flatten(-2)
        return torch.cat([t, y[..., rot:]], dim=-1).to(x.dtype)

    return turn(q), None if k is None else turn(k)
