"""Gated feed-forward block on the one-GPU GEMM kernel (``csrc/gemm_local.cu``): ``y = (silu(x Wg^T) * (x Wu^T)) Wd^T``.

Forward is two launches: both projections with the activation and the product in their epilogue, then the down projection.  Backward is
two as well: ``dy Wd``, whose epilogue turns the product's gradient into those of gate and up and makes the product again, then both
weight gradients and the input gradient side by side.  Products of few rows, and small weight gradients over many, fall into slices
of their contraction, which one more launch each adds up."""
import ctypes as C

import torch

from . import _lib


class GatedFwd(C.Structure):
    _fields_ = [
        ("T", C.c_int), ("D", C.c_int), ("F", C.c_int), ("O", C.c_int),
        ("x", C.c_void_p), ("ldx", C.c_longlong), ("w_gu", C.c_void_p), ("ld_gu", C.c_longlong),
        ("w_d", C.c_void_p), ("ld_d", C.c_longlong), ("gu", C.c_void_p), ("h", C.c_void_p), ("y", C.c_void_p), ("whole", C.c_int),
        ("status", C.c_void_p), ("scratch", C.c_void_p), ("scratch_bytes", C.c_ulonglong),
        ("launches", C.c_int),
    ]


class GatedBwd(C.Structure):
    _fields_ = [
        ("T", C.c_int), ("D", C.c_int), ("F", C.c_int), ("O", C.c_int),
        ("x", C.c_void_p), ("ldx", C.c_longlong), ("dy", C.c_void_p), ("ldy", C.c_longlong),
        ("w_gu", C.c_void_p), ("ld_gu", C.c_longlong), ("w_d", C.c_void_p), ("ld_d", C.c_longlong),
        ("gu", C.c_void_p), ("dgu", C.c_void_p), ("h", C.c_void_p), ("h_kept", C.c_int), ("dx", C.c_void_p), ("dw_gu", C.c_void_p), ("dw_d", C.c_void_p),
        ("whole", C.c_int), ("status", C.c_void_p), ("scratch", C.c_void_p), ("scratch_bytes", C.c_ulonglong),
        ("launches", C.c_int),
    ]


_declared = False


def _L():
    global _declared
    L = _lib.lib()
    if not _declared:
        for kind, args in (("fwd", GatedFwd), ("bwd", GatedBwd)):
            getattr(L, f"rtp_gated_{kind}").argtypes = [C.POINTER(args), C.c_void_p]
            f = getattr(L, f"rtp_gated_{kind}_scratch")
            f.argtypes, f.restype = [C.POINTER(args)], C.c_ulonglong
        _declared = True
    return L


def check_args(x, w_gate_up, w_down):
    if x.dim() < 1 or w_gate_up.dim() != 2 or w_down.dim() != 2:
        raise ValueError(f"gated_mlp: x must be [..., D], w_gate_up [2 * F, D], w_down [O, F], got {tuple(x.shape)}, {tuple(w_gate_up.shape)} and "
                         f"{tuple(w_down.shape)}")
    if w_gate_up.shape[1] != x.shape[-1] or w_gate_up.shape[0] != 2 * w_down.shape[1]:
        raise ValueError(f"gated_mlp: sizes do not fit: x {tuple(x.shape)}, w_gate_up {tuple(w_gate_up.shape)} (2 * F, D), w_down "
                         f"{tuple(w_down.shape)} (O, F)")
    if not (x.dtype == w_gate_up.dtype == w_down.dtype) or not x.dtype.is_floating_point:
        raise ValueError(f"gated_mlp: x and the weights must have one floating-point type, got {x.dtype}, {w_gate_up.dtype} and {w_down.dtype}")
    if not (x.device == w_gate_up.device == w_down.device):
        raise ValueError("gated_mlp: x and the weights must be on one device")


def kernel_takes(x, w_gate_up, w_down):
    """bf16 CUDA tensors, at least one row, sizes that are multiples of 8 (rows of 16 bytes)."""
    return (x.is_cuda and x.dtype == torch.bfloat16 and x.numel() > 0 and w_down.numel() > 0
            and not (x.shape[-1] % 8 or w_down.shape[0] % 8 or w_down.shape[1] % 8))


def _rows(t):
    """A 2-D view or copy with unit inner stride, 16-byte aligned rows that do not overlap."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _scratch(L, kind, a, device):
    need = getattr(L, f"rtp_gated_{kind}_scratch")(C.byref(a))
    if not need:
        return None
    s = torch.empty(need, dtype=torch.uint8, device=device)
    a.scratch, a.scratch_bytes = s.data_ptr(), need
    return s


def _check(rc, what, args):
    _lib.check(rc, what)
    _lib.launches += args.launches - 1


def gated_fwd(x, w_gu, w_d, keep, whole=False):
    """(y, gate | up or None, their product) of [T, D] rows.  ``whole``: the bits of separate layers."""
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return gated_fwd(x, w_gu, w_d, keep, whole)
    T, D = x.shape
    O, F = w_d.shape
    h, y = x.new_empty(T, F), x.new_empty(T, O)
    gu = x.new_empty(T, 2 * F) if keep else None
    a = GatedFwd(T, D, F, O, x.data_ptr(), x.stride(0), w_gu.data_ptr(), w_gu.stride(0), w_d.data_ptr(), w_d.stride(0),
                 gu.data_ptr() if keep else None, h.data_ptr(), y.data_ptr(), whole, _lib.status_word(x.device).data_ptr(), None, 0)
    L = _L()
    scratch = _scratch(L, "fwd", a, x.device)           # noqa: F841 (lives until the launch)
    _check(L.rtp_gated_fwd(C.byref(a), _lib.stream_ptr()), "rtp_gated_fwd", a)
    return y, gu, h


def gated_bwd(x, dy, w_gu, w_d, gu, h, dx, dw_gu, dw_d, whole=False):
    """Fills those of dx [T, D], dw_gu [2 * F, D] and dw_d [O, F] (dense) that are not None.  ``h``: the product of gate and up as the
    forward left it (None: made again for dw_d)."""
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return gated_bwd(x, dy, w_gu, w_d, gu, h, dx, dw_gu, dw_d, whole)
    T, D = x.shape
    O, F = w_d.shape
    dgu = torch.empty_like(gu)
    kept = h is not None
    if not kept and dw_d is not None:
        h = x.new_empty(T, F)
    ph, *p = [t.data_ptr() if t is not None else None for t in (h, dx, dw_gu, dw_d)]
    a = GatedBwd(T, D, F, O, x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), w_gu.data_ptr(), w_gu.stride(0), w_d.data_ptr(),
                 w_d.stride(0), gu.data_ptr(), dgu.data_ptr(), ph, kept, *p, whole, _lib.status_word(x.device).data_ptr(), None, 0)
    L = _L()
    scratch = _scratch(L, "bwd", a, x.device)           # noqa: F841 (lives until the launch)
    _check(L.rtp_gated_bwd(C.byref(a), _lib.stream_ptr()), "rtp_gated_bwd", a)


class _GatedMlpFn(torch.autograd.Function):
    """``owners``: None, or the two rotated modules of one rank whose flat shards the weights are; backward then reads the weights where
    they are, as that of a rotated layer does, and their gradients come as flat buffers.  ``rebuild``: (kind, sources) of an
    input that can be made again (see ``ops.functional``), which is then not kept."""

    @staticmethod
    def forward(ctx, x, w_gu, w_d, owners, rebuild):
        x2, wg, wd = _rows(x.reshape(-1, x.shape[-1])), _rows(w_gu), _rows(w_d)
        y, gu, h = gated_fwd(x2, wg, wd, True, owners is not None)
        kind, srcs = rebuild if rebuild is not None else (None, (x2,))
        ctx.kind, ctx.tensors = kind, [torch.is_tensor(s) for s in srcs]
        ctx.consts = [s for s in srcs if not torch.is_tensor(s)]
        # h is kept for the down projection's gradient: made again of the rounded gate and up it would have another error than the
        # forward's.  Layers of a model make it again, as they do one by one.
        ctx.save_for_backward(gu, *(() if owners else (wg, wd, h if ctx.needs_input_grad[2] else None)), *[s for s in srcs if torch.is_tensor(s)])
        ctx.owners, ctx.shape = owners, x.shape
        return y.view(*x.shape[:-1], w_d.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        gu, *kept = ctx.saved_tensors
        wg, wd, h = (*[_rows(o.linear.weight) for o in ctx.owners], None) if ctx.owners else [kept.pop(0) for _ in range(3)]
        if ctx.kind is None:
            x2 = kept[0]
        else:
            from . import functional as FO
            consts = list(ctx.consts)
            x = FO.recompute(ctx.kind, [kept.pop(0) if t else consts.pop(0) for t in ctx.tensors])
            x2 = _rows(x.reshape(-1, x.shape[-1]))
        dy2 = _rows(dy.reshape(-1, dy.shape[-1]))
        flats = [torch.empty_like(o._full_param) if o is not None and n else None
                 for o, n in zip(ctx.owners or (None, None), ctx.needs_input_grad[1:3])]
        grads = [None if not n else w.new_empty(w.shape) if f is None else f[:w.numel()].view(w.shape)
                 for w, f, n in zip((wg, wd), flats, ctx.needs_input_grad[1:3])]
        dx = x2.new_empty(x2.shape) if ctx.needs_input_grad[0] else None
        gated_bwd(x2, dy2, wg, wd, gu, h, dx, *grads, ctx.owners is not None)
        for o, f in zip(ctx.owners or (), flats):
            o._last_flat_grad = f                         # None: no gradient was asked for, and an earlier one is not this pass's
        return (dx.view(ctx.shape) if dx is not None else None, *grads, None, None)


def gated_mlp(x, w_gate_up, w_down, owners=None):
    """Kernel front-end of ``ops.functional.gated_mlp`` (same arguments)."""
    check_args(x, w_gate_up, w_down)
    if not kernel_takes(x, w_gate_up, w_down):
        raise ValueError(f"gated_mlp: the kernels take bf16 CUDA tensors with sizes that are multiples of 8, got {x.dtype} {tuple(x.shape)} on {x.device}")
    if not _lib.through_autograd(x, w_gate_up, w_down):
        x2 = _rows(x.reshape(-1, x.shape[-1]))
        return gated_fwd(x2, _rows(w_gate_up), _rows(w_down), False, owners is not None)[0].view(*x.shape[:-1], w_down.shape[0])
    from . import functional as FO
    return _GatedMlpFn.apply(x, w_gate_up, w_down, owners, FO.recompute_tag(x))
