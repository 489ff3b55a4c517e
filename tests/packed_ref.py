"""64-bit plain forms of the packed-document operators, and bounds on what their kernels may be off by.

Written from the definitions, one document at a time; nothing here uses the package.
"""
import math
import random

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def split_rows(B, S, mean_doc, prefix, pad, seed, empty_row=False):
    """[(documents [(length, prefix)], tokens that are not padding)] per row."""
    rng = random.Random(seed)
    rows = []
    for b in range(B):
        length = S - rng.randrange(S // 2 + 1) if pad else S
        if empty_row and b == B - 1:
            length = 0
        docs, left = [], length
        while left:
            n = left if not mean_doc else max(1, min(left, int(rng.expovariate(1.0 / mean_doc)) + 1))
            docs.append((n, rng.randrange(n + 1) if prefix else 0))
            left -= n
        rows.append((docs, length))
    return rows


def row_tensors(rows, S, seed, eod=0, vocab=1000):
    """tokens (a document ends with eod), document ids, prefix marks, lengths."""
    g = torch.Generator().manual_seed(seed)
    B = len(rows)
    tokens = torch.randint(1, vocab, (B, S), generator=g)
    ids = torch.full((B, S), 7, dtype=torch.int64)
    marks = torch.rand(B, S, generator=g) < 0.3      # marks behind an unmarked token mean nothing
    for b, (docs, length) in enumerate(rows):
        at = 0
        for k, (n, p) in enumerate(docs):
            tokens[b, at + n - 1] = eod
            ids[b, at:at + n] = 5 * k - 3
            marks[b, at:at + p] = True
            if p < n:
                marks[b, at + p] = False
            at += n
    return tokens, ids, marks, torch.tensor([r[1] for r in rows])


def plan_ref(rows, S, prefix):
    """positions, start, end by the definition, token by token."""
    B = len(rows)
    out = torch.zeros(3, B, S, dtype=torch.int32)
    for b, (docs, _) in enumerate(rows):
        at = 0
        for n, p in docs:
            for i in range(n):
                out[0, b, at + i] = i
                out[1, b, at + i] = at
                out[2, b, at + i] = at + (p if prefix and i < p else i + 1)
            at += n
    return out[0], out[1], out[2]


def attention_ref(qkv, dctx, nh, nkv, d, start=None, end=None, cap=0.0, slopes=None, scale=None):
    """ctx, lse, dqkv in 64 bits and elementwise bounds (ctx, lse, dqkv) on a kernel that keeps scores, statistics
    and sums in 32 bits and rounds P, dS, ctx and dqkv to bf16 once each.

    Bounds (u = 2^-8, half a bf16 step): a score is off by at most ex (its fp32 sum of d products, the scaling, the
    tanh), so P by a factor within 1 +- 2 ex (numerator and row sum); rounding P adds u P.
      ctx:  sum_j (u + 2 ex) P |v| + u |ctx|
      dP:   a fp32 sum of d products;  Delta: the ctx that the kernel kept is off by its bound, so Delta by |dO|.bound
      dS:   (u + 4 ex) |dS| + P f (eDelta + edP)
      dQ:   s sum_j e(dS) |k| + u |dQ|;  dK likewise over i;  dV: sum_i (u + 2 ex) P |dO| + u |dV|
    """
    B, S, _ = qkv.shape
    scale = d ** -0.5 if scale is None else scale
    t = qkv.double().view(B, S, nh + 2 * nkv, d).transpose(1, 2)
    rep = nh // nkv
    q, k, v = t[:, :nh], t[:, nh:nh + nkv].repeat_interleave(rep, 1), t[:, nh + nkv:].repeat_interleave(rep, 1)
    i = torch.arange(S, device=qkv.device)
    if start is None:
        sees = (i <= i[:, None]).expand(B, 1, S, S)
    else:
        sees = ((i >= start[:, :, None]) & (i < end[:, :, None]))[:, None]
    raw = q @ k.transpose(-1, -2) * scale
    mag = q.abs() @ k.abs().transpose(-1, -2) * scale
    f = torch.ones_like(raw)
    x = raw
    if cap:
        f = 1 - torch.tanh(raw / cap) ** 2
        x = cap * torch.tanh(raw / cap)
    if slopes is not None:
        x = x - slopes.double().view(nh, 1, 1) * (i[:, None] - i).abs()
    biggest = max(1.0, x.abs().amax().item(), cap)
    ex = 2.0 ** -24 * d * mag.amax().item() + 2.0 ** -20 * biggest
    x = x.masked_fill(~sees, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    ctx = p @ v
    u = HALF_STEP[torch.bfloat16]
    b_ctx = (u + 2 * ex) * (p @ v.abs()) + u * ctx.abs() + 1e-30
    b_lse = ex + 2.0 ** -21 * (1 + torch.where(torch.isinf(lse), torch.zeros_like(lse), lse).abs())
    out = ctx.transpose(1, 2).reshape(B, S, nh * d)
    b_out = b_ctx.transpose(1, 2).reshape(B, S, nh * d)
    if dctx is None:
        return (out, lse, None), (b_out, b_lse, None)
    do = dctx.double().view(B, S, nh, d).transpose(1, 2)
    dp = do @ v.transpose(-1, -2)
    delta = (do * ctx).sum(-1, keepdim=True)
    ds = p * f * (dp - delta)
    e_dp = 2.0 ** -24 * d * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = (do.abs() * (b_ctx + 2.0 ** -24 * d * ctx.abs())).sum(-1, keepdim=True)
    e_f = 2.0 ** -20 if cap else 0.0    # 1 - tanh^2, absolute
    e_ds = (u + 4 * ex) * ds.abs() + p * f * (e_delta + e_dp) + p * (dp - delta).abs() * e_f
    dq = ds @ k * scale
    b_dq = e_ds @ k.abs() * scale + u * dq.abs()
    dk = (ds.transpose(-1, -2) @ q * scale).view(B, nkv, rep, S, d)
    b_dk = (e_ds.transpose(-1, -2) @ q.abs() * scale).view(B, nkv, rep, S, d).sum(2)
    dv = (p.transpose(-1, -2) @ do).view(B, nkv, rep, S, d)
    b_dv = ((u + 2 * ex) * (p.transpose(-1, -2) @ do.abs())).view(B, nkv, rep, S, d).sum(2)
    dk, dv = dk.sum(2), dv.sum(2)
    grad = torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B, S, -1)
    # fp32 sums over S terms
    slack = 1 + 2.0 ** -10
    bound = torch.cat([b_dq, b_dk + u * dk.abs(), b_dv + u * dv.abs()], 1).transpose(1, 2).reshape(B, S, -1)
    return (out, lse, grad), (b_out * slack, b_lse, bound * slack + 1e-30)


def rotary_ref(x, d, rot, num_heads, interleaved, radians, magnitude, positions, inverse=False):
    """Complex rotation in 64 bits."""
    B, S, W = x.shape
    angle = positions.double().expand(B, S)[..., None] * radians.to(x.device)
    z = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)[:, :, None]
    y = x.double().reshape(B, S, W // d, d).clone()
    part = y[:, :, :num_heads, :rot]
    pairs = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    done = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    y[:, :, :num_heads, :rot] = (done if interleaved else done.transpose(-1, -2)).flatten(-2)
    return y.view(B, S, W)
