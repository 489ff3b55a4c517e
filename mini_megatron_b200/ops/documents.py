"""Packed rows: positions inside each document and the keys each token may see.

A row of ``S`` tokens holds documents one after another.  :func:`document_plan`
reads the rows once (one kernel, csrc/document_plan.cu) and returns a
:class:`DocumentPlan`; rotary positions take its ``positions`` and
:func:`~mini_megatron_b200.ops.attention.attention_fwd` the plan itself.  One plan
serves every layer of a step, forward and backward.

Token ``i`` sees the keys ``start[i] <= j < end[i]`` of its row:

* its own document only (``start``), up to itself (``end = i + 1``);
* with ``prefix_mask``, the tokens at the beginning of a document that are marked
  (a prompt) see each other both ways: while every token from the document's start to
  ``i`` is marked, ``end`` is the end of that run;
* tokens at ``lengths[row]`` and behind are padding: they see nothing (attention output
  and gradients are 0) and nothing sees them.

Everything stays on the device (no synchronisation), so a captured CUDA graph can
rebuild the plan from new tokens.
"""
from __future__ import annotations

import torch

from . import native


class DocumentPlan:
    """``positions``, ``start``, ``end``: ``[B, S]`` int32.  ``tables`` holds the same intervals as the attention
    kernels read them: writing to ``start`` or ``end`` does not change what they compute."""

    __slots__ = ("positions", "start", "end", "tables", "shape")

    def __init__(self, positions, start, end, tables=None):
        self.positions, self.start, self.end, self.tables = positions, start, end, tables
        self.shape = tuple(positions.shape)

    @property
    def device(self):
        return self.positions.device

    def visible(self):
        """The mask as a dense ``[B, S, S]`` bool tensor (row: query, column: key)."""
        j = torch.arange(self.positions.shape[1], device=self.device)
        return (j >= self.start[..., None]) & (j < self.end[..., None])


def document_plan(tokens=None, eod=None, *, document_ids=None, prefix_mask=None, lengths=None) -> DocumentPlan:
    """Plan of packed rows.  Exactly one of

    * ``tokens`` ``[B, S]`` int64 with ``eod``, the token that ends a document (it belongs to the document), or
    * ``document_ids`` ``[B, S]`` int64: a document starts where the id changes.

    ``prefix_mask`` ``[B, S]`` bool and ``lengths`` ``[B]`` integers are optional; lengths are clamped to
    ``[0, S]``.  Rows of up to 2 Mi tokens on CUDA.
    """
    if (tokens is None) == (document_ids is None):
        raise ValueError("document_plan needs either tokens with eod, or document_ids")
    if tokens is not None and eod is None:
        raise ValueError("document_plan needs the eod token to split tokens into documents")
    if document_ids is not None and eod is not None:
        raise ValueError("eod splits tokens; document_ids are split where they change")
    ids = tokens if tokens is not None else document_ids
    if ids.dim() != 2 or ids.dtype != torch.int64:
        raise ValueError(f"document_plan needs [B, S] int64 rows, got {tuple(ids.shape)} {ids.dtype}")
    B, S = ids.shape
    if B < 1 or S < 1:
        raise ValueError("document_plan needs at least one token")
    if prefix_mask is not None:
        if prefix_mask.shape != ids.shape or prefix_mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError("prefix_mask must be a bool tensor of the rows' shape")
        if prefix_mask.device != ids.device:
            raise ValueError("prefix_mask must be on the rows' device")
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError("lengths must be [B] int32 or int64")
        if lengths.device != ids.device:
            raise ValueError("lengths must be on the rows' device")
        lengths = lengths.clamp(0, S).to(torch.int32) if lengths.dtype == torch.int64 else lengths.contiguous()
    if not ids.is_cuda:
        return _plan_cpu(ids, eod, prefix_mask, lengths)
    ids = ids if ids.stride(1) == 1 else ids.contiguous()
    if prefix_mask is not None and prefix_mask.stride(1) != 1:
        prefix_mask = prefix_mask.contiguous()
    return DocumentPlan(*native().document_plan(ids, 0 if eod is None else eod, document_ids is not None, prefix_mask,
                                                lengths))


def _plan_cpu(ids, eod, prefix_mask, lengths):
    B, S = ids.shape
    at = torch.arange(S)
    first = torch.ones(B, S, dtype=torch.bool)
    first[:, 1:] = ids[:, :-1] == eod if eod is not None else ids[:, 1:] != ids[:, :-1]
    real = torch.ones(B, S, dtype=torch.bool) if lengths is None else at < lengths[:, None]
    start = torch.where(first, at, 0).cummax(1).values
    end = (at + 1).expand(B, S)
    if prefix_mask is not None:
        plain = (prefix_mask == 0) | ~real
        last_plain = torch.where(plain, at, -1).cummax(1).values
        stops = torch.cat([torch.where(plain | first, at, S), torch.full((B, 1), S)], 1)
        following = stops.flip(1).cummin(1).values.flip(1)[:, 1:]
        end = torch.where(last_plain < start, following, end)
    positions, start, end = (torch.where(real, t, 0).to(torch.int32) for t in (at - start, start, end))
    return DocumentPlan(positions, start, end)
