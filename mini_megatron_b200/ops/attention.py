"""Self-attention on the fused QKV activation.

:func:`flash_attn_fwd` / :func:`flash_attn_bwd`: plain causal attention (tcgen05 kernels in csrc/flash_*.cu).
:func:`attention_fwd` / :func:`attention_bwd` / :func:`attention`: documents, prefixes, padding, capped scores,
a bias linear in the distance, shared K/V heads and any sequence length (csrc/masked_attn_*.cu).

``qkv`` is the ``[B*S, 3*Hl]`` bf16 output of the QKV GEMM whose columns are
``[Q heads | K heads | V heads]`` (each ``nh*d`` wide) -- exactly the layout
the reference reshapes to ``[B, S, 3, nh, d]`` (model/transformer.py:27-33).
Outputs are ``ctx [B*S, nh*d]`` bf16 (token-major, ready for the O GEMM) and
``lse [B, nh, S]`` fp32 for the backward.  ``flash_attn_bwd`` returns
``dqkv`` in the same packed layout as ``qkv``.  There is no library fallback:
without the built extension :func:`native` raises.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import check_capture, native


def flash_attn_fwd(qkv, B, S, nh, d):
    return native().flash_attn_fwd(qkv, B, S, nh, d)


def flash_attn_bwd(dctx, qkv, ctx, lse, B, S, nh, d):
    return native().flash_attn_bwd(dctx, qkv, ctx, lse, B, S, nh, d)


# ---------------------------------------------------------------------------
# masked attention (csrc/masked_attn_*.cu)
# ---------------------------------------------------------------------------
# qkv is [B, S, (nh + 2 nkv) * d] with heads [Q | K | V]; query head h reads K/V head h // (nh / nkv).
#
#   x_ij = scale q_i.k_j, capped to softcap * tanh(x_ij / softcap), minus alibi_slopes[h] * |i - j|
#   ctx_i = sum_j softmax_j(x_ij) v_j over start_i <= j < end_i of the plan (no plan: j <= i)
#
# Rows that see nothing give ctx = 0, lse = -inf and no gradients.


def alibi_slopes(num_heads):
    """``[num_heads]`` fp32: ``2 ** (-8 (h + 1) / num_heads)``, the geometric slopes of linear distance biases.

    The series is the same for every head count; models whose slopes for a count that is no power of two were taken
    from the series of neighbouring powers pass their own."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / num_heads) for h in range(num_heads)], dtype=torch.float32)


def _options(qkv, num_heads, head_dim, num_kv_heads, plan, softcap, alibi_slopes, softmax_scale):
    if qkv.dim() != 3:
        raise ValueError(f"attention needs qkv [B, S, (num_heads + 2 num_kv_heads) * head_dim], got {tuple(qkv.shape)}")
    nkv = num_heads if num_kv_heads is None else num_kv_heads
    if plan is not None and (plan.shape != qkv.shape[:2] or (plan.tables is None) == qkv.is_cuda):
        raise ValueError(f"the plan was made for rows of {plan.shape} on {plan.device}, qkv has "
                         f"{tuple(qkv.shape[:2])} on {qkv.device}")
    if softcap is not None and not softcap > 0:
        raise ValueError("softcap must be positive (None: scores are not capped)")
    if alibi_slopes is not None and alibi_slopes.requires_grad:
        raise ValueError("alibi_slopes are constants: no gradient is computed for them")
    return nkv, softcap or 0.0, head_dim ** -0.5 if softmax_scale is None else float(softmax_scale)


def attention_fwd(qkv, num_heads, head_dim, *, num_kv_heads=None, plan=None, softcap=None, alibi_slopes=None,
                  softmax_scale=None):
    """``(ctx [B, S, num_heads * head_dim], lse [B, num_heads, S] fp32)`` of masked attention.

    ``plan``: a :class:`~mini_megatron_b200.ops.documents.DocumentPlan` (default: causal).  ``softcap`` 0.001 to 1000,
    ``alibi_slopes`` ``[num_heads]`` fp32, ``softmax_scale`` (default ``head_dim ** -0.5``).  On CUDA: bf16, head_dim
    64 or 128, up to 4096 heads, rows of up to 32 Mi tokens (2 Mi with a plan) on 16-byte boundaries.

    Everything in ``qkv`` must be finite, padding too: what a token does not see counts with weight 0, and 0 times an
    infinity or NaN is NaN.  Scores are 32-bit: one of size x is known to x / 2^24.  The gradients take the weights from
    ``lse``, so x / 2^22 is their relative error as well, below bf16's for scores up to 10^4; ctx and lse are right up to
    10^8, and from 2^31 on nothing is.  Statistics and sums are 32-bit; the weights, and in the backward pass the scores'
    gradients, are rounded to bf16 once, as operands of the tensor cores.  On CUDA autograd does not see this call:
    :func:`attention` is the differentiable form.
    """
    nkv, cap, scale = _options(qkv, num_heads, head_dim, num_kv_heads, plan, softcap, alibi_slopes, softmax_scale)
    if not qkv.is_cuda:
        return _attention_cpu(qkv, num_heads, head_dim, nkv, plan, cap, alibi_slopes, scale)
    return tuple(native().masked_attn_fwd(qkv, num_heads, nkv, head_dim, None if plan is None else plan.tables,
                                          alibi_slopes, cap, scale))


def attention_bwd(dctx, qkv, ctx, lse, num_heads, head_dim, *, num_kv_heads=None, plan=None, softcap=None,
                  alibi_slopes=None, softmax_scale=None):
    """``dqkv`` (layout of ``qkv``, contiguous) from the gradient of ``ctx`` and what :func:`attention_fwd` returned.
    CUDA only.  The same inputs give the same bits: no atomics.  ``dctx`` has to be finite in padding too, like ``qkv``."""
    nkv, cap, scale = _options(qkv, num_heads, head_dim, num_kv_heads, plan, softcap, alibi_slopes, softmax_scale)
    return native().masked_attn_bwd(dctx, qkv, ctx, lse, num_heads, nkv, head_dim, None if plan is None else plan.tables,
                                    alibi_slopes, cap, scale)


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, num_heads, head_dim, opts):
        out, lse = attention_fwd(qkv, num_heads, head_dim, **opts)
        ctx.save_for_backward(qkv, out, lse)
        ctx.args, ctx.opts = (num_heads, head_dim), opts
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, out, lse = ctx.saved_tensors
        return attention_bwd(dout.contiguous(), qkv, out, lse, *ctx.args, **ctx.opts), None, None, None


def attention(qkv, num_heads, head_dim, *, num_kv_heads=None, plan=None, softcap=None, alibi_slopes=None,
              softmax_scale=None):
    """Differentiable masked attention: :func:`attention_fwd`'s ``ctx``.

    While a CUDA graph is captured, a leaf whose autograd graph from outside of the capture is still alive is refused.
    """
    opts = dict(num_kv_heads=num_kv_heads, plan=plan, softcap=softcap, alibi_slopes=alibi_slopes,
                softmax_scale=softmax_scale)
    if not qkv.is_cuda:
        return attention_fwd(qkv, num_heads, head_dim, **opts)[0]
    check_capture(qkv)
    return _AttentionFn.apply(qkv, num_heads, head_dim, opts)


def _attention_cpu(qkv, nh, d, nkv, plan, cap, slopes, scale):
    """Plain PyTorch (the CPU path, differentiable by autograd)."""
    B, S, W = qkv.shape
    if nkv < 1 or nh % nkv or W != (nh + 2 * nkv) * d:
        raise ValueError(f"attention: {W} columns are not {nh} + 2 * {nkv} heads of {d}")
    acc = torch.float64 if qkv.dtype == torch.float64 else torch.float32
    t = qkv.reshape(B, S, nh + 2 * nkv, d).transpose(1, 2).to(acc)
    q, k, v = t[:, :nh], t[:, nh:nh + nkv], t[:, nh + nkv:]
    k, v = (z.repeat_interleave(nh // nkv, 1) for z in (k, v))
    x = q @ k.transpose(-1, -2) * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    i = torch.arange(S)
    if slopes is not None:
        x = x - slopes.to(acc).view(nh, 1, 1) * (i[:, None] - i).abs()
    sees = (i <= i[:, None]) if plan is None else plan.visible()[:, None]
    x = x.masked_fill(~sees, float("-inf"))
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    return (p @ v).transpose(1, 2).reshape(B, S, nh * d).to(qkv.dtype), lse
