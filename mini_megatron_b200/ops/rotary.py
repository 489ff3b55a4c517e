"""Rotary positions on the packed QKV activation (csrc/rotary.cu).

The last dimension of ``x [B, S, heads * head_dim]`` is cut into heads; the first
``num_heads`` of them (the Q and K heads of a packed QKV activation) are rotated, the
others are copied (or left alone in place).  A pair ``(a, b)`` at position ``p`` becomes
``m (a cos t - b sin t, b cos t + a sin t)`` with ``t = p w_i``; the gradient is the
rotation by ``-t``.  Angles are formed in 64 bits, values are rotated in 32 and rounded
once to their type.  bf16 and fp32.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import check_capture, native

SCALINGS = (None, "linear", "ntk", "yarn")


class Rotary:
    """Frequencies of a rotary embedding.

    ``rotary_dim`` (default ``head_dim``): how much of each head is rotated.  ``interleaved``: pairs are
    neighbours ``(2i, 2i + 1)``; otherwise halves ``(i, i + rotary_dim / 2)``.  ``scaling`` stretches the
    ``original_max_positions`` a model was trained on by ``factor``:

    * ``"linear"``  positions divided by ``factor`` (position interpolation);
    * ``"ntk"``     ``base`` raised to ``base * factor ** (r / (r - 2))``, so the lowest frequency is divided by
      ``factor`` and the highest kept;
    * ``"yarn"``    frequencies that turn more than ``beta_fast`` times over the original window are kept, those that
      turn less than ``beta_slow`` times are divided by ``factor``, with a linear ramp over the index between, and the
      rotated values are multiplied by ``0.1 ln(factor) + 1``.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None, factor=1.0,
                 original_max_positions=None, beta_fast=32.0, beta_slow=1.0, device=None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim must be even and at most head_dim ({head_dim}), got {rotary_dim}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
        if not base > 1 or not math.isfinite(base):
            raise ValueError("base must be finite and above 1")
        if not factor >= 1 or not math.isfinite(factor):
            raise ValueError("factor must be finite and at least 1")
        if scaling == "ntk" and rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        if scaling == "yarn" and (not original_max_positions or not beta_fast > beta_slow > 0):
            raise ValueError("yarn scaling needs original_max_positions and beta_fast > beta_slow > 0")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        # what the rotation is a function of, for checkpoints
        self.description = dict(rotary_dim=rotary_dim, base=float(base), interleaved=bool(interleaved), scaling=scaling)
        if scaling is not None:
            self.description["factor"] = float(factor)
        if scaling == "yarn":
            self.description.update(original_max_positions=original_max_positions, beta_fast=float(beta_fast),
                                    beta_slow=float(beta_slow))
        self.magnitude = 1.0
        if scaling == "ntk":
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        i = torch.arange(rotary_dim // 2, dtype=torch.float64)
        w = torch.pow(torch.tensor(base, dtype=torch.float64), -2 * i / rotary_dim)
        if scaling == "linear":
            w = w / factor
        elif scaling == "yarn":
            def index(turns):  # the (fractional) pair that turns this often over the original window
                return rotary_dim * math.log(original_max_positions / (turns * 2 * math.pi)) / (2 * math.log(base))
            lo = max(math.floor(index(beta_fast)), 0)
            hi = min(math.ceil(index(beta_slow)), rotary_dim - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            w = w / factor * ramp + w * (1 - ramp)
            self.magnitude = 0.1 * math.log(factor) + 1.0
        self.radians = w                                   # per position, on the host
        self._turns = {}
        if device is not None:
            self.turns(torch.device(device))

    def turns(self, device):
        """``[rotary_dim / 2]`` fp64 turns per position on ``device`` (kept: they are this object's weights)."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        t = self._turns.get(device)
        if t is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Rotary: pass device=... when it is made, its frequencies cannot be copied to the "
                                   "device while a CUDA graph is being captured")
            t = self._turns[device] = (self.radians / (2 * math.pi)).to(device)
            if device.type == "cuda":
                torch.cuda.current_stream(device).synchronize()  # complete for every stream that reads it later
        return t


def _run(x, rotary, num_heads, positions, out, inverse):
    if x.dim() != 3:
        raise ValueError(f"rotary needs [B, S, heads * head_dim], got {tuple(x.shape)}")
    if not x.is_cuda:
        y = _rotary_cpu(x, rotary, num_heads, positions, inverse)
        return y if out is None else out.copy_(y)
    if out is not None and torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise RuntimeError("rotary: autograd does not record what is written to out= on CUDA; use apply_rotary for tensors "
                           "that require a gradient, or torch.no_grad()")
    freqs = rotary._turns.get(x.device)
    if freqs is None:
        freqs = rotary.turns(x.device)
    return native().rotary(x, out, positions, freqs, rotary.magnitude, rotary.interleaved, rotary.head_dim,
                           rotary.rotary_dim, num_heads, inverse)


def rotary_fwd(x, rotary, num_heads, positions=None, out=None):
    """The first ``num_heads`` heads of ``x`` rotated to ``positions`` (``[B, S]`` or ``[S]`` int32 / int64;
    default: the index in the row).  ``out=x`` works in place; another ``out`` must not overlap ``x``.

    On CUDA autograd does not see this call: the result carries no gradient (:func:`apply_rotary` is the differentiable
    form), and ``out`` is refused for tensors that require one.  A write to ``out`` counts as an in-place operation, so
    a graph that saved it earlier refuses its backward pass."""
    return _run(x, rotary, num_heads, positions, out, False)


def rotary_bwd(dy, rotary, num_heads, positions=None, out=None):
    """Gradient of :func:`rotary_fwd`: the rotation by the negative angle (``out=dy`` works in place; autograd: as there)."""
    return _run(dy, rotary, num_heads, positions, out, True)


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rotary, num_heads, positions):
        ctx.rotary, ctx.num_heads = rotary, num_heads
        ctx.save_for_backward(positions)
        return rotary_fwd(x, rotary, num_heads, positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        return rotary_bwd(dy.contiguous(), ctx.rotary, ctx.num_heads, positions), None, None, None


def apply_rotary(x, rotary, num_heads, positions=None):
    """:func:`rotary_fwd` as a differentiable operation (out of place)."""
    check_capture(x)
    return _RotaryFn.apply(x, rotary, num_heads, positions)


def _rotary_cpu(x, rotary, num_heads, positions, inverse):
    B, S, W = x.shape
    d, r = rotary.head_dim, rotary.rotary_dim
    if W % d or not 1 <= num_heads <= W // d:
        raise ValueError(f"rotary: {W} columns are not heads of {d}, or num_heads is not 1 to their number")
    if positions is None:
        positions = torch.arange(S)
    elif tuple(positions.shape) not in ((S,), (B, S)) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("rotary: positions must be [S] or [B, S] int32 or int64")
    angle = positions.double()[..., None] * rotary.radians
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos = (angle.cos() * rotary.magnitude).to(acc).unsqueeze(-2)
    sin = (angle.sin() * (-rotary.magnitude if inverse else rotary.magnitude)).to(acc).unsqueeze(-2)
    y = x.reshape(B, S, W // d, d).to(acc)
    part = y[:, :, :num_heads, :r]
    if rotary.interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    head = torch.cat([turned, y[:, :, :num_heads, r:]], -1)
    return torch.cat([head, y[:, :, num_heads:]], 2).reshape(B, S, W).to(x.dtype)
