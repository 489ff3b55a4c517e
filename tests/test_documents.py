"""Packed rows -> positions and visible intervals, against the definition token by token."""
import pytest
import torch

from packed_ref import plan_ref, row_tensors, split_rows

CASES = [  # B, S, mean document, prefix, pad, empty last row
    (1, 1, 0, False, False, False),
    (1, 1, 0, True, False, False),
    (2, 7, 2, True, True, False),
    (3, 128, 20, False, False, False),
    (2, 129, 1, True, False, False),
    (3, 257, 60, True, True, True),
    (2, 1000, 300, True, True, False),
    (1, 4096, 100, True, False, False),
    (2, 4097, 1500, True, True, False),
    (2, 9001, 4000, True, True, True),
]


def _check(device, B, S, doc, prefix, pad, empty, by_ids):
    from mini_megatron_b200.ops.documents import document_plan
    rows = split_rows(B, S, doc, prefix, pad, seed=S + B, empty_row=empty)
    tokens, ids, marks, lengths = row_tensors(rows, S, seed=1)
    kw = dict(prefix_mask=marks.to(device) if prefix else None,
              lengths=lengths.to(device) if pad or empty else None)
    if by_ids:
        plan = document_plan(document_ids=ids.to(device), **kw)
    else:
        plan = document_plan(tokens.to(device), eod=0, **kw)
    for got, want in zip((plan.positions, plan.start, plan.end), plan_ref(rows, S, prefix)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)
    assert plan.shape == (B, S)
    return plan


@pytest.mark.parametrize("by_ids", [False, True])
@pytest.mark.parametrize("B,S,doc,prefix,pad,empty", CASES)
def test_plan_cpu(B, S, doc, prefix, pad, empty, by_ids):
    _check("cpu", B, S, doc, prefix, pad, empty, by_ids)


def _tile_tables(plan):
    """What the attention kernels read, by its definition from the dense mask: intervals of both sides, their bounds."""
    B, S = plan.shape
    n_t = (S + 127) // 128
    dense = plan.visible().cpu()

    def side(mask):
        lo = torch.zeros(B, n_t * 128, dtype=torch.int32)
        hi = torch.zeros(B, n_t * 128, dtype=torch.int32)
        some = mask.any(2)
        at = torch.arange(S)
        lo[:, :S] = torch.where(some, torch.where(mask, at, S).amin(2), 0)
        hi[:, :S] = torch.where(some, torch.where(mask, at, -1).amax(2) + 1, 0)
        assert torch.equal(mask.sum(2), (hi - lo)[:, :S].long())      # intervals without holes
        stat = torch.empty(B, n_t, 4, dtype=torch.int32)
        for t in range(n_t):
            cut = slice(t * 128, min(S, t * 128 + 128))
            l, h = lo[:, cut], hi[:, cut]
            seen = h > l
            stat[:, t, 0] = torch.where(seen, l, 2 ** 31 - 1).amin(1)
            stat[:, t, 1] = torch.where(seen, h, 0).amax(1)
            stat[:, t, 2], stat[:, t, 3] = l.amax(1), h.amin(1)
        return lo.view(B, n_t, 1, 128), hi.view(B, n_t, 1, 128), stat

    qlo, qhi, qstat = side(dense)
    klo, khi, kstat = side(dense.transpose(1, 2))
    return torch.cat([qlo, qhi, klo, khi], 2), qstat, kstat


@pytest.mark.gpu
@pytest.mark.parametrize("by_ids", [False, True])
@pytest.mark.parametrize("B,S,doc,prefix,pad,empty", CASES + [
    (2, 40000, 9000, True, True, False), (1, 70001, 300, True, True, False), (1, 140000, 50000, True, False, False)])
def test_plan_gpu(B, S, doc, prefix, pad, empty, by_ids):
    plan = _check("cuda", B, S, doc, prefix, pad, empty, by_ids)
    if S > 10000:
        return
    rows, qstat, kstat = _tile_tables(plan)
    n_t = qstat.shape[1]
    n_p = (n_t + 1) // 2
    parts = [rows.numel(), qstat.numel(), kstat.numel()] + ([B * n_p, B * n_t, B * n_t] if n_t > 4 else [])
    got_rows, got_q, got_k, *orders = plan.tables.cpu().split(parts)
    assert torch.equal(got_rows.view_as(rows), rows)
    assert torch.equal(got_q.view_as(qstat), qstat) and torch.equal(got_k.view_as(kstat), kstat)
    # every tile once, heaviest first
    keys, queries = (torch.where(s[..., 1] == 0, 0, (s[..., 1] + 127) // 128 - s[..., 0] // 128) for s in (qstat, kstat))
    pairs = torch.zeros(B, n_p, dtype=torch.int64)
    for t in range(n_t):
        pairs[:, (t + 1) // 2 if n_t % 2 else t // 2] += keys[:, t]
    for order, weight in zip(orders, (pairs, keys, queries)):
        assert torch.equal(order.sort().values, torch.arange(len(order), dtype=torch.int32))
        along = weight.flatten()[order.long()]
        assert (along[1:] <= along[:-1]).all()


@pytest.mark.gpu
def test_plan_strided_rows_other_stream_and_graph():
    from mini_megatron_b200.ops.documents import document_plan
    rows = split_rows(3, 500, 90, True, True, seed=3)
    tokens, _, marks, lengths = row_tensors(rows, 500, seed=2)
    wide = torch.zeros(3, 777, dtype=torch.int64)
    wide[:, 5:505] = tokens
    want = plan_ref(rows, 500, True)
    s = torch.cuda.Stream()
    d_tok, d_marks, d_len = wide.cuda()[:, 5:505], marks.cuda(), lengths.cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan = document_plan(d_tok, eod=0, prefix_mask=d_marks, lengths=d_len)
    s.synchronize()
    assert all(torch.equal(g.cpu(), w) for g, w in zip((plan.positions, plan.start, plan.end), want))
    # captured once, replayed on new tokens
    buf = torch.zeros(3, 500, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = document_plan(buf, eod=0)
    for seed in (5, 6):
        rows = split_rows(3, 500, 40, False, False, seed=seed)
        buf.copy_(row_tensors(rows, 500, seed=seed)[0])
        g.replay()
        assert all(torch.equal(x.cpu(), w) for x, w in
                   zip((plan.positions, plan.start, plan.end), plan_ref(rows, 500, False)))


def test_lengths_are_clamped_and_marks_may_be_bytes():
    from mini_megatron_b200.ops.documents import document_plan
    tok = torch.ones(2, 4, dtype=torch.int64)
    for dtype in (torch.int32, torch.int64):
        plan = document_plan(tok, eod=0, lengths=torch.tensor([-3, 9], dtype=dtype),
                             prefix_mask=torch.ones(2, 4, dtype=torch.uint8))
        assert plan.end.tolist() == [[0] * 4, [4] * 4]
    assert plan.visible()[1].all() and not plan.visible()[0].any()


def test_plan_refusals():
    from mini_megatron_b200.ops.documents import document_plan
    tok = torch.ones(2, 4, dtype=torch.int64)
    for args, kw in [((), {}), ((tok,), {}), ((tok, 0), {"document_ids": tok}), ((), {"document_ids": tok, "eod": 1}),
                     ((tok.int(), 0), {}), ((tok[0], 0), {}), ((tok[:, :0], 0), {}),
                     ((tok, 0), {"prefix_mask": tok}), ((tok, 0), {"prefix_mask": torch.ones(2, 3, dtype=torch.bool)}),
                     ((tok, 0), {"lengths": torch.ones(3, dtype=torch.int32)}),
                     ((tok, 0), {"lengths": torch.ones(2)})]:
        with pytest.raises(ValueError):
            document_plan(*args, **kw)


@pytest.mark.gpu
def test_plan_refusals_gpu():
    from mini_megatron_b200.ops.documents import document_plan
    tok = torch.ones(2, 4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        document_plan(tok, eod=0, lengths=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        document_plan(tok, eod=0, prefix_mask=torch.ones(2, 4, dtype=torch.bool))
