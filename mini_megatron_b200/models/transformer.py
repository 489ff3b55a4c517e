"""GPT decoder: Attention, MLP, DecoderLayer, Decoder, GPT.

Module tree and parameter names match the reference (model/transformer.py:8-109)
so its ``state_dict`` keys are unchanged:
``decoder.layers.{i}.{ln1,attn.qkv,attn.o,ln2,mlp.fc1,mlp.fc2}``,
``embedding.{token,position}_embedding``, ``ln_f``, ``lm_head``.

Two execution paths share these modules:

* CUDA tensors -> :class:`DecoderLayer` runs as ONE native autograd Function
  (``native_layers.DecoderLayerFn``) over the sm_100a kernels; ``GPT`` fuses
  ``ln_f -> lm_head -> vocab-parallel CE`` likewise.
* CPU tensors -> the same math in plain PyTorch ops (pre-LN, fused QKV with
  the stride-3 TP layout, causal SDPA, exact GELU, no biases), which is the
  oracle the native path is tested against.

Beyond the reference's model (:class:`AttentionSpec`): rotary positions, a bias linear
in the distance, capped scores, shared K/V heads, and a
:class:`~mini_megatron_b200.ops.documents.DocumentPlan` of packed rows passed down with
the activations.  Plain causal attention over rows of a multiple of 128 tokens runs on the
causal kernels; everything else on the masked ones.
"""
from __future__ import annotations

import dataclasses

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..parallel import process_groups as pg
from ..parallel.tensor_parallel import ColumnParallelLinear, RowParallelLinear


@dataclasses.dataclass
class AttentionSpec:
    """What an :class:`Attention` does beyond plain causal attention (the defaults are plain)."""

    num_kv_heads: int | None = None
    rotary: object = None             # ops.rotary.Rotary
    alibi: bool = False
    softcap: float | None = None


class Attention(nn.Module):
    """Multi-head self-attention with a fused, TP-sharded QKV projection, causal unless a plan says otherwise."""

    def __init__(self, hidden_size, num_heads, sequence_parallel=None, spec=None):
        super().__init__()
        spec = spec or AttentionSpec()
        tp = pg.tp_size()
        if num_heads % tp:
            raise ValueError("num_heads must divide evenly by TP size")
        kv_heads = num_heads if spec.num_kv_heads is None else spec.num_kv_heads
        if kv_heads < 1 or num_heads % kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        if kv_heads != num_heads and tp > 1:
            raise ValueError("shared K/V heads need TP size 1: the QKV weight is sharded in equal Q, K and V parts")
        self.all_heads, self.all_kv_heads = num_heads, kv_heads  # of every tensor-parallel rank together
        self.num_heads = num_heads // tp
        self.num_kv_heads = kv_heads // tp
        self.head_dim = hidden_size // num_heads
        self.hidden_size_per_partition = hidden_size // tp
        self.spec = spec
        if spec.alibi:
            from ..ops.attention import alibi_slopes
            first = pg.tp_rank() * self.num_heads
            self._slopes = alibi_slopes(num_heads)[first:first + self.num_heads].clone()
            self.register_buffer("alibi_slopes", self._slopes.clone(), persistent=False)
        else:
            self.alibi_slopes = None
        # stride 3: each TP rank holds an equal subset of Q, K and V heads
        self.qkv = ColumnParallelLinear(hidden_size, (num_heads + 2 * kv_heads) * self.head_dim, bias=False,
                                        stride=3 if kv_heads == num_heads else 1,
                                        sequence_parallel=sequence_parallel)
        self.o = RowParallelLinear(hidden_size, hidden_size, bias=False, sequence_parallel=sequence_parallel)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.alibi_slopes is not None:  # constants of 32 bits, whatever type the parameters are turned into
            self.alibi_slopes = self._slopes.to(self.alibi_slopes.device)
        return self

    def plain(self, plan):
        """Whether this is causal attention without anything else."""
        return (plan is None and self.spec.rotary is None and not self.spec.alibi and self.spec.softcap is None
                and self.num_kv_heads == self.num_heads)

    def description(self):
        """What the weights' shapes do not say about this attention, as plain values (tensor-parallel ranks agree)."""
        rotary = self.spec.rotary
        return dict(num_heads=self.all_heads, num_kv_heads=self.all_kv_heads, alibi=bool(self.spec.alibi),
                    softcap=self.spec.softcap, rotary=None if rotary is None else rotary.description)

    def options(self, plan):
        """Arguments of the masked attention operators."""
        return dict(num_kv_heads=self.num_kv_heads, plan=plan, softcap=self.spec.softcap,
                    alibi_slopes=self.alibi_slopes)

    def native_core_fwd(self, qkv, B, S, plan):
        """(ctx, lse, qkv as the backward needs it) of the [B*S, W] bf16 activation; rotates ``qkv`` in place."""
        from ..ops import attention as A
        if self.plain(plan) and S % 128 == 0:
            return (*A.flash_attn_fwd(qkv, B, S, self.num_heads, self.head_dim), qkv)
        q3 = qkv.view(B, S, -1)
        if self.spec.rotary is not None:
            from ..ops.rotary import rotary_fwd
            rotary_fwd(q3, self.spec.rotary, self.num_heads + self.num_kv_heads, plan.positions if plan else None,
                       out=q3)
        ctx, lse = A.attention_fwd(q3, self.num_heads, self.head_dim, **self.options(plan))
        return ctx.view(B * S, -1), lse, qkv

    def native_core_bwd(self, dctx, qkv, ctx, lse, B, S, plan):
        """dqkv [B*S, W] of :meth:`native_core_fwd`."""
        from ..ops import attention as A
        if self.plain(plan) and S % 128 == 0:
            return A.flash_attn_bwd(dctx, qkv, ctx, lse, B, S, self.num_heads, self.head_dim)
        dqkv = A.attention_bwd(dctx.view(B, S, -1), qkv.view(B, S, -1), ctx.view(B, S, -1), lse, self.num_heads,
                               self.head_dim, **self.options(plan))
        if self.spec.rotary is not None:
            from ..ops.rotary import rotary_bwd
            rotary_bwd(dqkv, self.spec.rotary, self.num_heads + self.num_kv_heads, plan.positions if plan else None,
                       out=dqkv)
        return dqkv.view(B * S, -1)

    def core_attention(self, qkv, plan=None):
        B, S, _ = qkv.shape
        if not self.plain(plan):
            from ..ops.attention import attention
            if self.spec.rotary is not None:
                from ..ops.rotary import apply_rotary
                qkv = apply_rotary(qkv, self.spec.rotary, self.num_heads + self.num_kv_heads,
                                   plan.positions if plan else None)
            return attention(qkv, self.num_heads, self.head_dim, **self.options(plan))
        qkv = qkv.reshape(B, S, 3, self.num_heads, self.head_dim)
        q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
        out = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return out.transpose(1, 2).reshape(B, S, self.hidden_size_per_partition)

    def forward(self, x, plan=None):
        qkv = self.qkv(x)
        if qkv.is_cuda:
            return self.o(_AttnFn.apply(qkv, self, plan))
        return self.o(self.core_attention(qkv, plan))


class _AttnFn(torch.autograd.Function):
    """Native attention on a packed [B, S, W] qkv tensor (standalone module use)."""

    @staticmethod
    def forward(ctx, qkv, attn, plan):
        B, S, W = qkv.shape
        q2 = qkv.reshape(B * S, W).to(torch.bfloat16).contiguous()
        if attn.spec.rotary is not None and q2.data_ptr() == qkv.data_ptr():
            q2 = q2.clone()  # rotated in place below
        out, lse, q2 = attn.native_core_fwd(q2, B, S, plan)
        ctx.save_for_backward(q2, out, lse)
        ctx.shape, ctx.attn, ctx.plan, ctx.dtype = (B, S, W), attn, plan, qkv.dtype
        return out.view(B, S, -1)

    @staticmethod
    def backward(ctx, dout):
        q2, out, lse = ctx.saved_tensors
        B, S, W = ctx.shape
        d2 = dout.reshape(B * S, -1).to(torch.bfloat16).contiguous()
        dqkv = ctx.attn.native_core_bwd(d2, q2, out, lse, B, S, ctx.plan)
        return dqkv.view(B, S, W).to(ctx.dtype), None, None


class MLP(nn.Module):
    def __init__(self, hidden_size, ffn_hidden_size, sequence_parallel=None):
        super().__init__()
        self.fc1 = ColumnParallelLinear(hidden_size, ffn_hidden_size, bias=False, sequence_parallel=sequence_parallel)
        self.fc2 = RowParallelLinear(ffn_hidden_size, hidden_size, bias=False, sequence_parallel=sequence_parallel)

    def forward(self, x):
        return self.fc2(F.gelu(self.fc1(x)))


class DecoderLayer(nn.Module):
    """Pre-LN block: x + attn(ln1(x)), then + mlp(ln2(.))."""

    def __init__(self, hidden_size, num_heads, ffn_hidden_size, sequence_parallel=None, recompute=False, spec=None):
        super().__init__()
        self.ln1 = nn.LayerNorm(hidden_size)
        self.attn = Attention(hidden_size, num_heads, sequence_parallel, spec)
        self.ln2 = nn.LayerNorm(hidden_size)
        self.mlp = MLP(hidden_size, ffn_hidden_size, sequence_parallel)
        self.sequence_parallel = pg.sequence_parallel_enabled() if sequence_parallel is None else sequence_parallel
        self.recompute = recompute
        # LayerNorm parameters see only the local sequence shard under SP:
        # their gradients need a TP all-reduce before the optimizer step.
        for p in list(self.ln1.parameters()) + list(self.ln2.parameters()):
            p.sequence_parallel_grad = bool(self.sequence_parallel)

    def _forward(self, x, plan=None):
        x = x + self.attn(self.ln1(x), plan)
        x = x + self.mlp(self.ln2(x))
        return x

    def native_forward(self, x, recompute=None, plan=None):
        from .native_layers import DecoderLayerFn
        group = pg.tp_group()
        sp = bool(self.sequence_parallel and group is not None)
        rc = self.recompute if recompute is None else recompute
        return DecoderLayerFn.apply(x.float().contiguous(), self, group, sp, rc, plan, *self.parameters())

    def forward(self, x, use_checkpoint=False, plan=None):
        if x.is_cuda:
            return self.native_forward(x, recompute=use_checkpoint or self.recompute, plan=plan)
        if use_checkpoint or self.recompute:
            return torch.utils.checkpoint.checkpoint(self._forward, x, plan, use_reentrant=False)
        return self._forward(x, plan)


class Decoder(nn.Module):
    """Stack of DecoderLayer blocks (``layer_ids`` is metadata for pipeline stages)."""

    def __init__(self, hidden_size, num_heads, ffn_hidden_size, num_layers, layer_ids=None, sequence_parallel=None,
                 recompute=False, spec=None):
        super().__init__()
        self.layer_ids = list(range(num_layers)) if layer_ids is None else list(layer_ids)
        self.layers = nn.ModuleList([
            DecoderLayer(hidden_size, num_heads, ffn_hidden_size, sequence_parallel, recompute, spec)
            for _ in self.layer_ids
        ])

    def forward(self, x, plan=None):
        for layer in self.layers:
            x = layer(x, plan=plan)
        return x


class GPT(nn.Module):
    """embedding -> decoder -> ln_f -> lm_head [-> loss].

    Returns ``logits`` or ``(logits, loss)`` when labels, loss_mask and a loss
    function are given (reference model/transformer.py:90-109).  Logits are
    this rank's vocabulary shard when TP > 1 (use
    ``gather_from_model_parallel_region`` for the full vocabulary).  On CUDA
    with the package's CrossEntropyLoss the head runs fused
    (``native_layers.HeadLossFn``) and the returned logits buffer is
    overwritten by its gradient during backward.

    With ``eod_token`` rows are packed documents: attention stays inside a document
    and rotary positions restart with it.  A learned position table does not: its rows
    are those of the index in the row, so a document's logits depend on where it lies
    (with rotary positions or a distance bias they are the ones it has alone).  ``forward(..., plan=...)`` takes another
    :class:`~mini_megatron_b200.ops.documents.DocumentPlan` instead (prefixes, padding).
    """

    def __init__(self, embedding, decoder, ln_f, lm_head, loss_fn=None, eod_token=None):
        super().__init__()
        self.embedding = embedding
        self.decoder = decoder
        self.ln_f = ln_f
        self.lm_head = lm_head
        self.loss_fn = loss_fn
        self.eod_token = eod_token

    def forward(self, input_ids, labels=None, loss_mask=None, plan=None):
        if plan is None and self.eod_token is not None:
            from ..ops.documents import document_plan
            plan = document_plan(input_ids, eod=self.eod_token)
        x = self.embedding(input_ids)
        x = self.decoder(x, plan=plan)
        return head_forward(self.ln_f, self.lm_head, self.loss_fn, x, labels, loss_mask)


def head_forward(ln_f, lm_head, loss_fn, x, labels=None, loss_mask=None):
    """ln_f -> lm_head [-> loss], fused on CUDA when the loss is the package's CE."""
    from .loss import CrossEntropyLoss
    want_loss = labels is not None and loss_mask is not None and loss_fn is not None
    if (want_loss and x.is_cuda and isinstance(loss_fn, CrossEntropyLoss) and lm_head.bias is None
            and not lm_head.gather_output):
        from .native_layers import HeadLossFn
        group = pg.tp_group()
        sp = bool(lm_head.sequence_parallel and group is not None)
        n_vocab = loss_fn.vocab_size if loss_fn.vocab_size is not None else lm_head.out_features
        loss, logits = HeadLossFn.apply(x.float().contiguous(), ln_f, lm_head, labels, loss_mask, n_vocab, group,
                                        sp, ln_f.weight, ln_f.bias, lm_head.weight)
        B = labels.shape[0]
        return logits.view(B, -1, logits.shape[-1]), loss
    h = ln_f(x)
    logits = lm_head(h)
    if want_loss:
        return logits, loss_fn(logits, labels, loss_mask)
    return logits
