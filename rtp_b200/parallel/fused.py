"""Dispatch of rotated layers onto the fused sm_100a kernels (filled in by rtp_b200.parallel.engine)."""
import torch

from .context import get_backend


def use_fused(x: torch.Tensor, flat: torch.Tensor) -> bool:
    """Fused path: bf16 CUDA tensors, unless the functional backend was requested explicitly."""
    be = get_backend()
    if be == "functional":
        return False
    ok = x.is_cuda and flat.is_cuda and flat.dtype == torch.bfloat16 and x.dtype == torch.bfloat16
    if be == "fused" and not ok:
        raise RuntimeError("backend 'fused' needs bf16 CUDA tensors")
    return ok


def linear(module, x, row=False):
    from .engine import fused_linear
    return fused_linear(module, x, row=row)


def linear_ok(row, in_f, out_f, world):
    """Shapes that the fused kernels cannot take (a feature count that is not a multiple of 8, e.g. a 10-class head)
    run on the functional engine instead."""
    from .engine import fused_linear_ok
    return fused_linear_ok(row, in_f, out_f, world)


def gated_mlp(gate_up, down, x):
    """``down(silu(g) * u)`` of a packed column-parallel gate / up projection and a row-parallel down projection in the fused kernels of
    one rank (``ops.mlp``); None: not a case for them (layers of another kind, with a forward or hooks of their own, a ring of several
    ranks, biases, the in-place mode, a backward pass that is not to make activations again)."""
    from ..module.linear import ColumnParallelLinear, RowParallelLinear, runs_plain_forward
    from ..ops import functional as FO, mlp
    if torch.is_grad_enabled() and not FO.activation_recompute():
        return None
    if not runs_plain_forward(gate_up, ColumnParallelLinear) or not runs_plain_forward(down, RowParallelLinear):
        return None
    if gate_up.world_size != 1 or not use_fused(x, gate_up._full_param) or not use_fused(x, down._full_param):
        return None
    wg, wd = gate_up.linear.weight, down.linear.weight
    if gate_up.linear.bias is not None or down.linear.bias is not None or gate_up.packed_parts != 2:
        return None
    if not mlp.kernel_takes(x, wg, wd):
        return None
    return mlp.gated_mlp(x, wg, wd, owners=(gate_up, down))
