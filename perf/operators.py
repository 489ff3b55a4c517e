"""The packed-document attention operators, as measured work.

Three operators that a GPT trained on packed rows needs next to each other:

* ``plan``       tokens of packed rows -> positions inside each document and the interval of keys each token sees
                 (documents, bidirectional prefixes, padding);
* ``rotary``     rotary positions on the Q and K heads of the packed QKV activation, forward and backward;
* ``attention``  attention over the packed QKV activation under such a plan, with scores capped by a tanh and/or
                 lowered in proportion to the distance, forward and backward, heads of K and V shared or not.

Every case is a dict of plain values.  ``run`` computes the plain form (elementary torch operations in 32 bits, angles
in 64) unless ``own`` is set, in which case it calls the package.
"""
import math
import random

import torch

own = False

EOD = 0
VOCAB = 50257


# ---------------------------------------------------------------- cases
def listed():
    return [
        # two short ragged rows: what a smoke test or a small evaluation batch pays, latency only
        {"name": "plan_two_short_rows", "op": "plan", "B": 2, "S": 257, "doc": 60, "prefix": False, "pad": True},
        # a long-context batch whose prompts are seen both ways
        {"name": "plan_long_rows", "op": "plan", "B": 8, "S": 32768, "doc": 900, "prefix": True, "pad": True},
        # a handful of tokens: latency
        {"name": "rotary_seven_tokens", "op": "rotary", "B": 1, "S": 7, "nh": 4, "nkv": 4, "d": 64, "rot": 64,
         "interleaved": False, "scaling": "none", "factor": 1.0, "far": 0, "dtype": "bf16"},
        # the GPT-125M microbatch (16 x 1024 tokens, 12 heads of 64), half layout
        {"name": "rotary_gpt125m", "op": "rotary", "B": 16, "S": 1024, "nh": 12, "nkv": 12, "d": 64, "rot": 64,
         "interleaved": False, "scaling": "none", "factor": 1.0, "far": 0, "dtype": "bf16"},
        # one long sequence at far positions, shared K/V heads, half of each head rotated, scaled frequencies
        {"name": "rotary_long_scaled", "op": "rotary", "B": 1, "S": 16384, "nh": 32, "nkv": 8, "d": 128, "rot": 64,
         "interleaved": True, "scaling": "yarn", "factor": 16.0, "far": 100003, "dtype": "bf16"},
        # short ragged rows, one partial tile: latency of a forward and a backward pass
        {"name": "attn_short_rows", "op": "attention", "B": 2, "S": 77, "nh": 4, "nkv": 4, "d": 64, "doc": 0,
         "prefix": False, "pad": False, "cap": 0.0, "alibi": False, "amp": 1.0, "train": True, "layout": 1},
        # the GPT-125M microbatch with packed documents, a training step's attention
        {"name": "attn_gpt125m_documents", "op": "attention", "B": 16, "S": 1024, "nh": 12, "nkv": 12, "d": 64,
         "doc": 300, "prefix": False, "pad": True, "cap": 0.0, "alibi": False, "amp": 1.0, "train": True, "layout": 2},
        # GPT-1.3B heads, scores capped, evaluation (forward only)
        {"name": "attn_gpt1.3b_capped_fwd", "op": "attention", "B": 4, "S": 2048, "nh": 16, "nkv": 16, "d": 128,
         "doc": 0, "prefix": False, "pad": False, "cap": 30.0, "alibi": False, "amp": 4.0, "train": False, "layout": 3},
        # GPT-6.7B heads, distance bias, a training step's attention
        {"name": "attn_gpt6.7b_distance", "op": "attention", "B": 2, "S": 2048, "nh": 32, "nkv": 32, "d": 128,
         "doc": 0, "prefix": False, "pad": False, "cap": 0.0, "alibi": True, "amp": 1.0, "train": True, "layout": 4},
        # prompts seen both ways, shared K/V heads, an odd length with padding
        {"name": "attn_prefix_shared_heads", "op": "attention", "B": 3, "S": 1999, "nh": 16, "nkv": 4, "d": 64,
         "doc": 700, "prefix": True, "pad": True, "cap": 0.0, "alibi": False, "amp": 2.0, "train": True, "layout": 5},
        # one long row of documents, everything on
        {"name": "attn_long_all", "op": "attention", "B": 1, "S": 16384, "nh": 4, "nkv": 1, "d": 128,
         "doc": 6000, "prefix": True, "pad": True, "cap": 50.0, "alibi": True, "amp": 3.0, "train": True, "layout": 6},
        # one long causal row
        {"name": "attn_long_causal", "op": "attention", "B": 1, "S": 16384, "nh": 4, "nkv": 4, "d": 64,
         "doc": 0, "prefix": False, "pad": False, "cap": 0.0, "alibi": False, "amp": 1.0, "train": True, "layout": 7},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["plan", "rotary", "attention", "attention", "attention"])
    if kind == "plan":
        S = _log(rng, 1, 32768)
        B = _log(rng, 1, max(1, min(32, 8 * 32768 // S)))
        return {"op": "plan", "B": B, "S": S, "doc": _log(rng, 1, 4096), "prefix": rng.random() < 0.5,
                "pad": rng.random() < 0.5}
    d = rng.choice([64, 128])
    nkv = rng.choice([1, 2, 3, 4, 8])
    if kind == "rotary":
        nh = nkv * rng.choice([1, 1, 2, 4])
        width = (nh + 2 * nkv) * d
        S = _log(rng, 1, min(16384, 16384 * 6144 // width))
        B = _log(rng, 1, max(1, min(16, 16384 * 6144 // width // S)))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": "rotary", "B": B, "S": S, "nh": nh, "nkv": nkv, "d": d, "rot": rng.choice([d, d, d // 2, d // 4]),
                "interleaved": rng.random() < 0.5, "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 10.0, 32.0]),
                "far": rng.choice([0, 0, _log(rng, 1000, 1000000)]), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    nh = nkv * rng.choice([1, 1, 2, 4])
    S = _log(rng, 1, 12000)
    while nh * S * S > 4 * 16384 * 16384:
        S = S * 2 // 3
    B = _log(rng, 1, max(1, min(16, 4 * 16384 * 16384 // 2 // (nh * S * S), 16384 * 4 // S)))
    docs = rng.random() < 0.6
    return {"op": "attention", "B": B, "S": S, "nh": nh, "nkv": nkv, "d": d, "doc": _log(rng, 8, 4096) if docs else 0,
            "prefix": docs and rng.random() < 0.5, "pad": docs and rng.random() < 0.5,
            "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "alibi": rng.random() < 0.4, "amp": rng.choice([0.5, 1.0, 2.0, 4.0]),
            "train": rng.random() < 0.7, "layout": rng.randrange(1 << 20)}


# ---------------------------------------------------------------- layouts of packed rows
def _layout(B, S, doc, prefix, pad, seed):
    """For each row: ([(document length, prefix length)], tokens that are not padding)."""
    rng = random.Random(seed)
    rows = []
    for _ in range(B):
        length = S - rng.randrange(S // 4 + 1) if pad else S
        docs, left = [], length
        while left > 0:
            n = left if doc == 0 else max(1, min(left, int(round(doc * math.exp(rng.gauss(-0.3, 0.8))))))
            docs.append((n, rng.randrange(n // 2 + 1) if prefix else 0))
            left -= n
        rows.append((docs, length))
    return rows


def _row_tensors(rows, S, seed):
    """Tokens (a document's last one is EOD), prefix marks and lengths of the rows, on the host."""
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(1, VOCAB, (len(rows), S), generator=g)
    marks = torch.zeros(len(rows), S, dtype=torch.bool)
    for b, (docs, _) in enumerate(rows):
        n = torch.tensor([x[0] for x in docs])
        p = torch.tensor([x[1] for x in docs])
        ends = n.cumsum(0)
        tokens[b, ends - 1] = EOD
        of = torch.repeat_interleave(torch.arange(len(docs)), n)
        at = torch.arange(int(ends[-1]))
        marks[b, :int(ends[-1])] = at - (ends - n)[of] < p[of]
    return tokens, marks, torch.tensor([r[1] for r in rows], dtype=torch.int32)


def _slopes(nh):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], dtype=torch.float32, device="cuda")


# ---------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, S = case["B"], case["S"]
    st = {"case": case}
    if case["op"] == "plan":
        tokens, marks, lengths = _row_tensors(_layout(B, S, case["doc"], case["prefix"], case["pad"], seed), S, seed)
        st["tokens"] = tokens.cuda()
        st["marks"] = marks.cuda() if case["prefix"] else None
        st["lengths"] = lengths.cuda() if case["pad"] else None
        return st
    nh, nkv, d = case["nh"], case["nkv"], case["d"]
    if case["op"] == "rotary":
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        st["x"] = torch.randn(B, S, (nh + 2 * nkv) * d, device="cuda", generator=g).to(dtype)
        st["dy"] = torch.randn(B, S, (nh + 2 * nkv) * d, device="cuda", generator=g).to(dtype)
        pos = torch.arange(S, device="cuda", dtype=torch.int32) + case["far"]
        st["positions"] = pos.expand(B, S).contiguous() if case["far"] else None
        if own:
            from mini_megatron_b200.ops.rotary import Rotary
            st["rotary"] = Rotary(d, rotary_dim=case["rot"], interleaved=case["interleaved"],
                                  scaling=None if case["scaling"] == "none" else case["scaling"],
                                  factor=case["factor"], original_max_positions=4096, device="cuda")
        else:
            st["freqs"], st["magnitude"] = _frequencies(case)
        return st
    qkv = torch.randn(B, S, (nh + 2 * nkv) * d, device="cuda", generator=g)
    qkv[..., :nh * d] *= case["amp"]
    st["qkv"] = qkv.bfloat16()
    st["dctx"] = torch.randn(B, S, nh * d, device="cuda", generator=g).bfloat16()
    st["slopes"] = _slopes(nh) if case["alibi"] else None
    st["plan"] = st["start"] = st["end"] = None
    if case["doc"]:
        tokens, marks, lengths = _row_tensors(_layout(B, S, case["doc"], case["prefix"], case["pad"], case["layout"]),
                                              S, case["layout"])
        tokens, marks, lengths = tokens.cuda(), marks.cuda() if case["prefix"] else None, lengths.cuda()
        if own:
            from mini_megatron_b200.ops.documents import document_plan
            st["plan"] = document_plan(tokens, eod=EOD, prefix_mask=marks, lengths=lengths)
        else:
            _, st["start"], st["end"] = _plain_plan(tokens, marks, lengths)
    return st


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if case["op"] == "plan":
        if own:
            from mini_megatron_b200.ops.documents import document_plan
            plan = document_plan(st["tokens"], eod=EOD, prefix_mask=st["marks"], lengths=st["lengths"])
            return plan.positions, plan.start, plan.end
        return _plain_plan(st["tokens"], st["marks"], st["lengths"])
    nh, nkv, d = case["nh"], case["nkv"], case["d"]
    if case["op"] == "rotary":
        if own:
            from mini_megatron_b200.ops.rotary import rotary_bwd, rotary_fwd
            return (rotary_fwd(st["x"], st["rotary"], nh + nkv, st["positions"]),
                    rotary_bwd(st["dy"], st["rotary"], nh + nkv, st["positions"]))
        return (_plain_rotary(st["x"], case, st["freqs"], st["magnitude"], st["positions"], 1.0),
                _plain_rotary(st["dy"], case, st["freqs"], st["magnitude"], st["positions"], -1.0))
    if own:
        from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
        opts = dict(num_kv_heads=nkv, plan=st["plan"], softcap=case["cap"] or None, alibi_slopes=st["slopes"])
        ctx, lse = attention_fwd(st["qkv"], nh, d, **opts)
        if not case["train"]:
            return ctx, lse
        return ctx, attention_bwd(st["dctx"], st["qkv"], ctx, lse, nh, d, **opts)
    return _plain_attention(st, case)


# ---------------------------------------------------------------- plain forms
def _plain_plan(tokens, marks, lengths):
    """Positions, first and one past the last visible key of every token (padding: 0, 0 and 0)."""
    B, S = tokens.shape
    at = torch.arange(S, device=tokens.device)
    first = torch.ones_like(tokens, dtype=torch.bool)
    first[:, 1:] = tokens[:, :-1] == EOD
    real = torch.ones_like(first) if lengths is None else at < lengths[:, None]
    start = torch.where(first, at, 0).cummax(1).values
    end = (at + 1).expand(B, S)
    if marks is not None:
        # the next token at or after this one that ends a run of marks: an unmarked one, a document's first, padding
        plain = ~marks | ~real
        last_plain = torch.where(plain, at, -1).cummax(1).values
        stop = torch.where(plain | first, at, S)
        nxt = torch.full((B, S + 1), S, device=tokens.device, dtype=stop.dtype)
        nxt[:, :S] = stop.flip(1).cummin(1).values.flip(1)
        end = torch.where(last_plain < start, nxt[:, 1:], end)
    zero = torch.zeros((), dtype=torch.int64, device=tokens.device)
    return tuple(torch.where(real, t, zero).int() for t in (at - start, start, end))


def _frequencies(case):
    """Radians per position of each rotated pair (64 bits) and the factor on the rotated values."""
    rot, base, f, window = case["rot"], 10000.0, case["factor"], 4096
    if case["scaling"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    w = base ** (-2 * i / rot)
    if case["scaling"] == "linear":
        w = w / f
    if case["scaling"] == "yarn":
        # turns over the trained window: above 32 the frequency stays, below 1 it is divided, linear in the index between
        def index(turns):
            return rot * math.log(window / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        w = w / f * ramp + w * (1 - ramp)
        return w, 0.1 * math.log(f) + 1.0
    return w, 1.0


def _plain_rotary(x, case, freqs, magnitude, positions, sign):
    B, S, W = x.shape
    d, rot, n = case["d"], case["rot"], case["nh"] + case["nkv"]
    pos = torch.arange(S, device=x.device) if positions is None else positions
    angle = pos.double()[..., None] * freqs
    c, s = (angle.cos() * magnitude).float(), (angle.sin() * (magnitude * sign)).float()
    c, s = c.expand(B, S, rot // 2)[:, :, None], s.expand(B, S, rot // 2)[:, :, None]
    y = x.float().view(B, S, W // d, d).clone()
    part = y[:, :, :n, :rot]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        part.copy_(torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2))
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part.copy_(torch.cat([a * c - b * s, b * c + a * s], -1))
    return y.view(B, S, W).to(x.dtype)


def _heads(t, nh, nkv, d):
    """[B, nh, S, d] queries and [B, nkv, 1, S, d] keys and values of the packed activation, in 32 bits."""
    B, S, _ = t.shape
    t = t.float().view(B, S, nh + 2 * nkv, d).transpose(1, 2)
    return t[:, :nh].reshape(B, nkv, nh // nkv, S, d), t[:, nh:nh + nkv, None], t[:, nh + nkv:, None]


def _plain_attention(st, case):
    nh, nkv, d, cap = case["nh"], case["nkv"], case["d"], case["cap"]
    qkv = st["qkv"]
    B, S, _ = qkv.shape
    q, k, v = _heads(qkv, nh, nkv, d)
    at = torch.arange(S, device=qkv.device)
    if st["start"] is None:
        sees = at[None, :] <= at[:, None]
    else:
        sees = ((at >= st["start"][:, :, None]) & (at < st["end"][:, :, None]))[:, None, None]
    x = (q @ k.transpose(-1, -2)) * d ** -0.5
    if cap:
        t = torch.tanh(x / cap)
        x = cap * t
    if st["slopes"] is not None:
        x = x - st["slopes"].view(nkv, nh // nkv, 1, 1) * (at[:, None] - at[None, :]).abs()
    x = x.masked_fill(~sees, float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(x - top)
    del x
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).reshape(B, nh, S)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    ctx = p @ v
    out = ctx.reshape(B, nh, S, d).transpose(1, 2).reshape(B, S, nh * d).to(qkv.dtype)
    if not case["train"]:
        return out, lse
    do = st["dctx"].float().view(B, S, nkv, nh // nkv, d).permute(0, 2, 3, 1, 4)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v.transpose(-1, -2) - (do * ctx).sum(-1, keepdim=True))
    del p
    if cap:
        ds = ds * (1 - t * t)
    ds = ds * d ** -0.5
    dq = (ds @ k).reshape(B, nh, S, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return out, torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B, S, -1).to(qkv.dtype)


# ---------------------------------------------------------------- what one pass cannot do without
def work(case):
    B, S = case["B"], case["S"]
    if case["op"] == "plan":
        return {"bytes": B * S * (8 + (1 if case["prefix"] else 0) + 3 * 4), "flops": 0}
    nh, nkv, d = case["nh"], case["nkv"], case["d"]
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        n = B * S * (nh + 2 * nkv) * d
        return {"bytes": 2 * 2 * n * size + (B * S * 4 if case["far"] else 0), "flops": 2 * 3 * B * S * (nh + nkv) * case["rot"]}
    rows = _layout(B, S, case["doc"], case["prefix"], case["pad"], case["layout"])
    pairs = sum(n * (n + 1) // 2 + p * (p - 1) // 2 for docs, _ in rows for n, p in docs)
    tokens, lse = B * S, 4 * B * nh * S
    plan = 8 * tokens if case["doc"] else 0
    fwd = 2 * tokens * (2 * nh + 2 * nkv) * d + lse + plan
    if not case["train"]:
        return {"bytes": fwd, "flops": 4 * d * nh * pairs}
    # backward: qkv, the output, its gradient and the sums are read, the gradient of qkv is written
    bwd = 2 * tokens * (2 * (nh + 2 * nkv) + 2 * nh) * d + lse + plan
    return {"bytes": fwd + bwd, "flops": 14 * d * nh * pairs}


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    B, S = case["B"], case["S"]
    st = prepare(case, seed)
    if case["op"] == "plan":
        return None
    nh, nkv, d = case["nh"], case["nkv"], case["d"]
    if case["op"] == "rotary":
        w, m = _frequencies(case)
        pos = (torch.arange(S, device="cuda").expand(B, S) if st["positions"] is None else st["positions"]).double()
        turn = torch.polar(torch.full((), m, dtype=torch.float64, device="cuda"), pos[..., None] * w)[:, :, None]
        outs = []
        for x, z in ((st["x"], turn), (st["dy"], turn.conj())):
            y = x.double().view(B, S, -1, d).clone()
            part = y[:, :, :nh + nkv, :case["rot"]]
            if case["interleaved"]:
                part = part.unflatten(-1, (-1, 2))
            else:
                part = part.unflatten(-1, (2, -1)).transpose(-1, -2)
            done = torch.view_as_real(torch.view_as_complex(part.contiguous()) * z)
            y[:, :, :nh + nkv, :case["rot"]] = (done if case["interleaved"] else done.transpose(-1, -2)).flatten(-2)
            outs.append(y.view(B, S, -1))
        return tuple(outs)
    qkv = st["qkv"].double().view(B, S, nh + 2 * nkv, d)
    grad = torch.zeros_like(qkv)
    out = torch.empty(B, S, nh, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(B, nh, S, dtype=torch.float64, device="cuda")
    at = torch.arange(S, device="cuda")
    rows = _layout(B, S, case["doc"], case["prefix"], case["pad"], case["layout"])
    for b in range(B):
        # a block of the mask for each document
        blocks, begin = [], 0
        for n, p in rows[b][0]:
            blocks.append((begin, begin + n, p))
            begin += n
        out[b, begin:], lse[b, :, begin:] = 0.0, float("-inf")
        for h in range(nh):
            g = nh + h // (nh // nkv)
            for lo, hi, p in blocks:
                i, j = at[lo:hi, None], at[None, lo:hi]
                hidden = (j > i) & (j >= lo + p)
                q, k, v = qkv[b, lo:hi, h], qkv[b, lo:hi, g], qkv[b, lo:hi, g + nkv]
                raw = (q @ k.T) / math.sqrt(d)
                x = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
                slope = 1.0 if case["cap"] == 0 else 1 - (x / case["cap"]) ** 2
                if case["alibi"]:
                    x = x - st["slopes"][h].double() * (i - j).abs()
                x = torch.where(hidden, -torch.inf, x)
                total = torch.logsumexp(x, 1)
                lse[b, h, lo:hi] = total
                p_ = torch.exp(x - total[:, None])
                out[b, lo:hi, h] = p_ @ v
                if case["train"]:
                    do = st["dctx"].view(B, S, nh, d)[b, lo:hi, h].double()
                    dp = do @ v.T
                    ds = p_ * (dp - (p_ * dp).sum(1, keepdim=True)) * slope / math.sqrt(d)
                    grad[b, lo:hi, h] = ds @ k
                    grad[b, lo:hi, g] += ds.T @ q
                    grad[b, lo:hi, g + nkv] += p_.T @ do
    out = out.view(B, S, nh * d)
    return (out, grad.view(B, S, -1)) if case["train"] else (out, lse)
