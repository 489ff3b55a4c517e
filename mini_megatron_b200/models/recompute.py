"""Activation recomputation (reference model/recompute.py:4-6).

On CPU this is torch.utils.checkpoint around the layer body; on CUDA the
native DecoderLayer Function re-runs its own forward inside backward when
``layer.recompute`` is set (only the layer input is kept).
"""
import torch
import torch.utils.checkpoint


def checkpoint(layer, x, plan=None):
    """``layer(x, plan=plan)`` that keeps only ``x`` (and the plan of packed rows) for the backward pass."""
    if x.is_cuda and hasattr(layer, "native_forward"):
        return layer.native_forward(x, recompute=True, plan=plan)
    args = (x,) if plan is None else (x, plan)
    return torch.utils.checkpoint.checkpoint(layer._forward, *args, use_reentrant=False)
