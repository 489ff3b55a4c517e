"""Masked attention (documents, prefixes, padding, capped scores, distance bias, shared heads) against 64 bits."""
import pytest
import torch

from packed_ref import attention_ref, plan_ref, row_tensors, split_rows


def _slopes(nh, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], device=device)


def _case(B, S, nh, nkv, d, doc, prefix, pad, amp, device, dtype, seed=0, empty_row=False):
    from mini_megatron_b200.ops.documents import document_plan
    g = torch.Generator().manual_seed(seed + S)
    qkv = torch.randn(B, S, (nh + 2 * nkv) * d, generator=g)
    qkv[..., :nh * d] *= amp
    dctx = torch.randn(B, S, nh * d, generator=g)
    plan = start = end = None
    if doc is not None:
        rows = split_rows(B, S, doc, prefix, pad, seed=seed + S, empty_row=empty_row)
        tokens, _, marks, lengths = row_tensors(rows, S, seed=seed)
        _, start, end = (t.to(device) for t in plan_ref(rows, S, prefix))
        plan = document_plan(tokens.to(device), eod=0, prefix_mask=marks.to(device) if prefix else None,
                             lengths=lengths.to(device))
    return qkv.to(device, dtype), dctx.to(device, dtype), plan, start, end


def _near(got, want, bound, what):
    got, want = got.double(), want.double()
    same = torch.isfinite(want)
    assert torch.equal(same, torch.isfinite(got)) and torch.equal(got[~same], want[~same]), what
    off = ((got - want).abs() - bound)[same]
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} over the bound"


def _rel(a, b):
    return ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()


# B, S, nh, nkv, d, mean document (None: causal, 0: one per row), prefix, pad, cap, alibi, amp
GRID = [
    (1, 1, 1, 1, 64, None, False, False, 0.0, False, 1.0),
    (1, 1, 2, 1, 128, 0, True, False, 20.0, True, 1.0),
    (3, 2, 2, 2, 64, 1, False, True, 0.0, False, 1.0),
    (2, 127, 3, 3, 64, None, False, False, 0.0, False, 2.0),
    (2, 128, 2, 1, 128, None, False, False, 0.0, True, 1.0),
    (2, 129, 4, 2, 64, 30, False, True, 30.0, False, 4.0),
    (1, 255, 2, 2, 128, 40, True, True, 0.0, True, 1.0),
    (2, 256, 4, 1, 64, 0, True, False, 0.0, False, 1.0),
    (2, 300, 6, 2, 128, 100, True, True, 50.0, True, 3.0),
    (1, 513, 2, 2, 64, None, False, False, 15.0, True, 4.0),
    (1, 640, 3, 3, 128, None, False, False, 0.0, False, 3.0),
    (3, 777, 2, 2, 64, 5, False, True, 0.0, False, 1.0),
    (2, 1000, 4, 4, 128, 350, True, True, 25.0, False, 2.0),
    (1, 1537, 2, 1, 64, 600, False, True, 0.0, True, 2.0),
    (5, 384, 12, 12, 64, 200, True, False, 0.0, False, 1.0),
    (40, 130, 5, 5, 64, 50, False, True, 0.0, False, 1.0),
    (9, 260, 10, 2, 128, 0, False, True, 0.0, False, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,nh,nkv,d,doc,prefix,pad,cap,alibi,amp", GRID)
def test_forward_and_backward(B, S, nh, nkv, d, doc, prefix, pad, cap, alibi, amp):
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    qkv, dctx, plan, start, end = _case(B, S, nh, nkv, d, doc, prefix, pad, amp, "cuda", torch.bfloat16,
                                        empty_row=pad and B > 2)
    slopes = _slopes(nh, "cuda") if alibi else None
    opts = dict(num_kv_heads=nkv, plan=plan, softcap=cap or None, alibi_slopes=slopes)
    ctx, lse = attention_fwd(qkv, nh, d, **opts)
    dqkv = attention_bwd(dctx, qkv, ctx, lse, nh, d, **opts)
    check_errors()
    (r_ctx, r_lse, r_grad), (b_ctx, b_lse, b_grad) = attention_ref(qkv, dctx, nh, nkv, d, start, end, cap, slopes)
    _near(ctx, r_ctx, b_ctx, "ctx")
    _near(lse, r_lse, b_lse, "lse")
    _near(dqkv, r_grad, b_grad, "dqkv")
    # three or four independent roundings of at most 2^-8 each (rms at most 2^-8 / sqrt 3): 2 * 2^-8 / sqrt 3 at most
    assert _rel(ctx, r_ctx) < 4.6e-3 and _rel(dqkv, r_grad) < 4.6e-3 or r_grad.norm() < 1e-6 * dctx.norm().double()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_scale_and_large_scores(d):
    """Scores spread over hundreds of log2 units: the running maximum moves and rows are nearly one-hot."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    qkv, dctx, plan, start, end = _case(2, 700, 2, 2, d, 300, True, False, 6.0, "cuda", torch.bfloat16, seed=5)
    ctx, lse = attention_fwd(qkv, 2, d, plan=plan, softmax_scale=0.3)
    grad = attention_bwd(dctx, qkv, ctx, lse, 2, d, plan=plan, softmax_scale=0.3)
    want, bound = attention_ref(qkv, dctx, 2, 2, d, start, end, scale=0.3)
    for g, w, b, n in zip((ctx, lse, grad), want, bound, ("ctx", "lse", "dqkv")):
        _near(g, w, b, n)


@pytest.mark.gpu
def test_same_bits_twice_and_on_another_stream():
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    qkv, dctx, plan, _, _ = _case(3, 900, 8, 2, 64, 250, True, True, 1.0, "cuda", torch.bfloat16)
    outs = []
    for k in range(3):
        s = torch.cuda.Stream() if k else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ctx, lse = attention_fwd(qkv, 8, 64, num_kv_heads=2, plan=plan, softcap=30.0)
            outs.append((ctx, lse, attention_bwd(dctx, qkv, ctx, lse, 8, 64, num_kv_heads=2, plan=plan, softcap=30.0)))
        torch.cuda.current_stream().wait_stream(s)
    for got in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, outs[0]))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls of different shapes on two streams at the same time give the bits that they give alone."""
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    sets = [(_case(6, 1100, 8, 2, 64, 250, True, True, 1.0, "cuda", torch.bfloat16), 8, 2, 64),
            (_case(3, 1500, 6, 6, 128, 400, False, True, 1.0, "cuda", torch.bfloat16, seed=9), 6, 6, 128)]

    def call(case, nh, nkv, d):
        qkv, dctx, plan, _, _ = case
        ctx, lse = attention_fwd(qkv, nh, d, num_kv_heads=nkv, plan=plan)
        return ctx, lse, attention_bwd(dctx, qkv, ctx, lse, nh, d, num_kv_heads=nkv, plan=plan)

    want = [call(*c) for c in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(12):
        for s, c in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(call(*c))
    torch.cuda.synchronize()
    check_errors()
    for k, one in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(one, want[k % 2])), k


@pytest.mark.gpu
def test_strides_and_neighbours():
    """Rows inside wider buffers, a token-major batch; padding gives zeros, what lies around is not read into it."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    B, S, nh, d = 3, 200, 2, 64
    qkv, dctx, plan, _, _ = _case(B, S, nh, nh, d, 70, False, True, 1.0, "cuda", torch.bfloat16)
    want = attention_fwd(qkv, nh, d, plan=plan)
    grad = attention_bwd(dctx, qkv, *want, nh, d, plan=plan)
    wide = torch.full((B, S + 9, 3 * nh * d + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    view = wide[:, 4:4 + S, 16:16 + 3 * nh * d]
    view.copy_(qkv)
    dwide = torch.full((S + 3, B, nh * d + 8), float("nan"), device="cuda", dtype=torch.bfloat16)
    dview = dwide[1:1 + S, :, 8:].transpose(0, 1)
    dview.copy_(dctx)
    got = attention_fwd(view, nh, d, plan=plan)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(attention_bwd(dview, view, *got, nh, d, plan=plan), grad)
    pad = plan.end == 0
    assert pad.any()
    assert (want[0][pad] == 0).all() and (grad[pad] == 0).all()
    assert (want[1].transpose(1, 2)[pad] == float("-inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,nh,nkv", [(64, 4, 4), (64, 4, 1), (128, 2, 1)])
@pytest.mark.parametrize("S", [200, 900])
def test_many_empty_rows(d, nh, nkv, S):
    """A batch of mostly empty rows: a CTA then has one tile of work among dozens without any."""
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    B = 400
    g = torch.Generator().manual_seed(S)
    lengths = torch.zeros(B, dtype=torch.int32)
    lengths[[3, 150, 151, 399]] = torch.tensor([S, 1, 130, S - 1], dtype=torch.int32)
    tokens = torch.randint(0, 40, (B, S), generator=g)
    qkv = torch.randn(B, S, (nh + 2 * nkv) * d, generator=g).bfloat16().cuda()
    dctx = torch.randn(B, S, nh * d, generator=g).bfloat16().cuda()
    plan = document_plan(tokens.cuda(), eod=0, lengths=lengths.cuda())
    ctx, lse = attention_fwd(qkv, nh, d, num_kv_heads=nkv, plan=plan)
    grad = attention_bwd(dctx, qkv, ctx, lse, nh, d, num_kv_heads=nkv, plan=plan)
    check_errors()
    some = lengths.nonzero().flatten().tolist()
    start, end = plan.start[some], plan.end[some]
    (r_ctx, r_lse, r_grad), (b_ctx, b_lse, b_grad) = attention_ref(qkv[some], dctx[some], nh, nkv, d, start, end)
    _near(ctx[some], r_ctx, b_ctx, "ctx")
    _near(lse[some], r_lse, b_lse, "lse")
    _near(grad[some], r_grad, b_grad, "dqkv")
    none = [b for b in range(B) if b not in some]
    assert not ctx[none].any() and not grad[none].any() and (lse[none] == float("-inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_tables_that_were_never_written(d):
    """Arbitrary numbers in a plan's tables give arbitrary numbers, inside the tensors; the next call is not affected."""
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import DocumentPlan
    qkv, dctx, plan, _, _ = _case(3, 900, 4, 2, d, 250, False, True, 1.0, "cuda", torch.bfloat16)
    want = attention_fwd(qkv, 4, d, num_kv_heads=2, plan=plan)
    want += (attention_bwd(dctx, qkv, *want, 4, d, num_kv_heads=2, plan=plan),)
    g = torch.Generator().manual_seed(3)
    for low, high in ((-2 ** 31, 2 ** 31), (-1000, 2000)):
        tables = torch.randint(low, high, plan.tables.shape, generator=g).to(torch.int32).cuda()
        other = DocumentPlan(plan.positions, plan.start, plan.end, tables)
        ctx, lse = attention_fwd(qkv, 4, d, num_kv_heads=2, plan=other)
        attention_bwd(dctx, qkv, ctx, lse, 4, d, num_kv_heads=2, plan=other)
        check_errors()
    got = attention_fwd(qkv, 4, d, num_kv_heads=2, plan=plan)
    got += (attention_bwd(dctx, qkv, *got, 4, d, num_kv_heads=2, plan=plan),)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    from mini_megatron_b200.ops.attention import attention
    from mini_megatron_b200.ops.rotary import Rotary, apply_rotary
    x = torch.randn(1, 40, 192, device="cuda").bfloat16().requires_grad_(True)
    for y in (attention(x, 1, 64), apply_rotary(x, Rotary(64), 2)):
        (grad,) = torch.autograd.grad(y.float().pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            grad.float().sum().backward()


@pytest.mark.gpu
def test_two_graphs_share_nothing():
    """Forward and backward captured twice, replayed alternately on new values, against eager calls."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    sets = [_case(2, 333, 4, 2, 64, 90, True, True, 1.0, "cuda", torch.bfloat16, seed=s) for s in (1, 2)]
    graphs = []
    for qkv, dctx, plan, _, _ in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ctx, lse = attention_fwd(qkv, 4, 64, num_kv_heads=2, plan=plan)
            grad = attention_bwd(dctx, qkv, ctx, lse, 4, 64, num_kv_heads=2, plan=plan)
        graphs.append((g, ctx, lse, grad))
    for k in range(3):
        for qkv, dctx, *_ in sets:
            qkv.copy_(torch.randn_like(qkv))
        for g, *_ in graphs:
            g.replay()
        for (qkv, dctx, plan, _, _), (_, ctx, lse, grad) in zip(sets, graphs):
            c, l = attention_fwd(qkv, 4, 64, num_kv_heads=2, plan=plan)
            assert torch.equal(c, ctx) and torch.equal(l, lse)
            assert torch.equal(attention_bwd(dctx, qkv, c, l, 4, 64, num_kv_heads=2, plan=plan), grad)


@pytest.mark.gpu
def test_autograd_and_broadcast_gradient():
    from mini_megatron_b200.ops.attention import attention, attention_bwd, attention_fwd
    qkv, _, plan, _, _ = _case(2, 150, 2, 2, 64, 60, False, True, 1.0, "cuda", torch.bfloat16)
    leaf = qkv.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(attention(leaf, 2, 64, plan=plan).sum(), leaf)   # an expanded gradient
    ctx, lse = attention_fwd(qkv, 2, 64, plan=plan)
    assert torch.equal(got, attention_bwd(torch.ones_like(ctx), qkv, ctx, lse, 2, 64, plan=plan))
    frozen = attention(qkv, 2, 64, plan=plan)
    assert not frozen.requires_grad and torch.equal(frozen, ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_matches_plain_causal_attention(d):
    """No plan, one K/V head per query head: the function of the framework's causal kernels."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd, flash_attn_bwd, flash_attn_fwd
    B, S, nh = 2, 512, 4
    qkv, dctx, _, _, _ = _case(B, S, nh, nh, d, None, False, False, 1.0, "cuda", torch.bfloat16)
    ctx, lse = attention_fwd(qkv, nh, d)
    c2, l2 = flash_attn_fwd(qkv.view(B * S, -1), B, S, nh, d)
    _, (b_ctx, b_lse, b_grad) = attention_ref(qkv, dctx, nh, nh, d)
    _near(ctx, c2.view_as(ctx), 2 * b_ctx, "ctx")
    _near(lse, l2, 2 * b_lse, "lse")
    g2 = flash_attn_bwd(dctx.view(B * S, -1), qkv.view(B * S, -1), c2, l2, B, S, nh, d)
    _near(attention_bwd(dctx, qkv, ctx, lse, nh, d), g2.view_as(qkv), 2 * b_grad, "dqkv")


@pytest.mark.gpu
def test_empty_batch():
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    for B, S in ((0, 5), (2, 0)):
        qkv = torch.zeros(B, S, 192, device="cuda", dtype=torch.bfloat16)
        ctx, lse = attention_fwd(qkv, 1, 64)
        assert ctx.shape == (B, S, 64) and lse.shape == (B, 1, S)
        assert attention_bwd(ctx, qkv, ctx, lse, 1, 64).shape == qkv.shape


@pytest.mark.parametrize("B,S,nh,nkv,d,doc,prefix,pad,cap,alibi,amp", GRID[:10])
def test_cpu_path(B, S, nh, nkv, d, doc, prefix, pad, cap, alibi, amp):
    from mini_megatron_b200.ops.attention import attention, attention_fwd
    qkv, dctx, plan, start, end = _case(B, S, nh, nkv, d, doc, prefix, pad, amp, "cpu", torch.float64)
    slopes = _slopes(nh, "cpu") if alibi else None
    opts = dict(num_kv_heads=nkv, plan=plan, softcap=cap or None, alibi_slopes=slopes)
    (r_ctx, r_lse, r_grad), _ = attention_ref(qkv, dctx, nh, nkv, d, start, end, cap, slopes)
    ctx, lse = attention_fwd(qkv, nh, d, **opts)
    torch.testing.assert_close(ctx, r_ctx, rtol=1e-9, atol=1e-9)
    torch.testing.assert_close(lse, r_lse, rtol=1e-9, atol=1e-9)
    leaf = qkv.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(attention(leaf, nh, d, **opts), leaf, dctx)
    torch.testing.assert_close(grad, r_grad, rtol=1e-7, atol=1e-7)


def test_reference_gradient_against_differences():
    """The formula behind every gradient test, by central differences along random directions."""
    g = torch.Generator().manual_seed(0)
    B, S, nh, nkv, d = 2, 23, 4, 2, 8
    rows = split_rows(B, S, 9, True, True, seed=4)
    _, start, end = plan_ref(rows, S, True)
    qkv = torch.randn(B, S, (nh + 2 * nkv) * d, generator=g, dtype=torch.float64)
    dctx = torch.randn(B, S, nh * d, generator=g, dtype=torch.float64)
    slopes = _slopes(nh, "cpu")

    def value(x):
        return (attention_ref(x, None, nh, nkv, d, start, end, 3.0, slopes)[0][0] * dctx).sum().item()

    grad = attention_ref(qkv, dctx, nh, nkv, d, start, end, 3.0, slopes)[0][2]
    for _ in range(3):
        z = torch.randn(qkv.shape, generator=g, dtype=torch.float64)
        slope = (value(qkv + 1e-5 * z) - value(qkv - 1e-5 * z)) / 2e-5
        assert abs(slope - (grad * z).sum().item()) < 1e-6 * max(1.0, abs(slope))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(device):
    from mini_megatron_b200.ops.attention import attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    x = torch.zeros(2, 4, 384, device=device, dtype=torch.bfloat16)
    plan = document_plan(torch.ones(2, 5, dtype=torch.int64, device=device), eod=0)
    for args, kw in [((x[0], 2, 64), {}), ((x, 2, 64), {"plan": plan}), ((x, 2, 64), {"softcap": 0.0}),
                     ((x, 2, 64), {"softcap": -1.0}),
                     ((x, 2, 64), {"alibi_slopes": torch.ones(2, device=device, requires_grad=True)})]:
        with pytest.raises(ValueError):
            attention_fwd(*args, **kw)
    for args, kw in [((x, 3, 64), {}), ((x, 4, 64), {"num_kv_heads": 3}), ((x, 4, 64), {"num_kv_heads": 0})]:
        with pytest.raises((ValueError, RuntimeError)):
            attention_fwd(*args, **kw)


@pytest.mark.gpu
def test_refusals_gpu():
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    x = torch.zeros(2, 4, 384, device="cuda", dtype=torch.bfloat16)
    wide = torch.zeros(2, 4, 400, device="cuda", dtype=torch.bfloat16)
    bad = [((x.float(), 2, 64), {}), ((x, 4, 32), {}), ((x, 2, 64), {"softcap": 1e6}),
           ((x, 2, 64), {"softcap": 1e-9}), ((x, 2, 64), {"softmax_scale": 1e30}),
           ((x.new_zeros(1, 1, 3 * 4097 * 64), 4097, 64), {}),
           ((x, 2, 64), {"softmax_scale": 0.0}), ((x, 2, 64), {"softmax_scale": float("nan")}),
           ((x, 2, 64), {"alibi_slopes": torch.ones(3, device="cuda")}),
           ((x, 2, 64), {"alibi_slopes": torch.ones(2)}),
           ((x, 2, 64), {"alibi_slopes": torch.ones(2, device="cuda", dtype=torch.float64)}),
           ((wide[..., 4:388], 2, 64), {}),                                    # rows off the 16-byte boundary
           ((x.transpose(1, 2).contiguous().transpose(1, 2), 2, 64), {}),       # not dense
           ((x[:1].expand(2, 4, 384), 2, 64), {})]                             # one row for the whole batch
    for args, kw in bad:
        with pytest.raises(RuntimeError):
            attention_fwd(*args, **kw)
    with pytest.raises(ValueError):
        attention_fwd(x, 2, 64, plan=document_plan(torch.ones(2, 4, dtype=torch.int64), eod=0))
    ctx, lse = attention_fwd(x, 2, 64)
    for args in [(ctx.float(), x, ctx, lse), (ctx[:, :3], x, ctx, lse), (ctx, x, ctx[:, :, :64], lse),
                 (ctx, x, ctx, lse[:, :1]), (ctx, x, ctx, lse.double()), (ctx, x, ctx.transpose(0, 1), lse),
                 (ctx.cpu(), x, ctx, lse), (ctx, x, ctx, lse.cpu())]:
        with pytest.raises(RuntimeError):
            attention_bwd(*args, 2, 64)


@pytest.mark.gpu
def test_tensors_off_the_16_byte_boundary_are_refused():
    """Views that are contiguous but start inside a 16-byte unit: the kernels read whole units."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import DocumentPlan, document_plan
    B, S, nh, d = 2, 700, 2, 64
    qkv = torch.randn(B, S, 3 * nh * d, device="cuda").bfloat16()
    dctx = torch.randn(B, S, nh * d, device="cuda").bfloat16()
    ctx, lse = attention_fwd(qkv, nh, d)
    for off in (1, 2, 4, 7):
        moved = torch.zeros(ctx.numel() + 8, device="cuda", dtype=ctx.dtype)[off:off + ctx.numel()].view_as(ctx)
        moved.copy_(ctx)
        assert moved.is_contiguous()
        with pytest.raises(RuntimeError, match="16-byte"):
            attention_bwd(dctx, qkv, moved, lse, nh, d)
        with pytest.raises(RuntimeError, match="16-byte"):
            attention_bwd(moved, qkv, ctx, lse, nh, d)
    plan = document_plan(torch.ones(B, S, dtype=torch.int64, device="cuda"), eod=0)
    for off in (1, 2, 3):
        tables = torch.zeros(plan.tables.numel() + 4, device="cuda", dtype=torch.int32)[off:off + plan.tables.numel()]
        with pytest.raises(RuntimeError, match="16-byte"):
            attention_fwd(qkv, nh, d, plan=DocumentPlan(plan.positions, plan.start, plan.end, tables))


@pytest.mark.gpu
def test_rows_whose_items_outlast_the_waits_are_refused():
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    qkv = torch.empty(1, 2 ** 25 + 1, 192, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="tokens"):
        attention_fwd(qkv, 1, 64)
    ctx = qkv[..., :64]
    with pytest.raises(RuntimeError, match="tokens"):
        attention_bwd(ctx, qkv, ctx, torch.empty(1, 1, 8, device="cuda"), 1, 64)


def test_shares_of_query_heads():
    """The cut of a K/V head's query heads: whole heads, items that end well before a wait gives up, work for every SM."""
    native = pytest.importorskip("mini_megatron_b200._C", reason="extension not built")
    for S in (1, 128, 129, 1999, 4096, 16384, 2 ** 17, 2 ** 21, 2 ** 25):
        for nkv in (1, 2, 3, 8, 64):
            for group in (1, 2, 3, 4, 6, 8, 16, 32, 60, 64, 4096 // nkv):
                for B in (1, 3, 40):
                    n_t = (S + 127) // 128
                    parts = native.masked_attn_dkv_parts(B, S, nkv * group, nkv, 148)
                    assert 1 <= parts <= group and group % parts == 0
                    assert group // parts * n_t <= 2 ** 18
                    smaller = [p for p in range(1, parts) if group % p == 0]
                    assert all(B * nkv * n_t * p < 2 * 148 or group // p * n_t > 2 ** 18 for p in smaller)


# B, S, nh, nkv, d, mean document, prefix, pad, cap, alibi, shares (148 SMs)
SHARED = [
    (3, 1999, 16, 4, 64, 700, True, True, 0.0, True, 2),
    (3, 1999, 16, 4, 128, 700, False, True, 30.0, False, 2),
    (2, 2000, 24, 2, 64, None, False, False, 20.0, True, 6),
    (2, 2000, 48, 4, 64, 400, False, True, 0.0, False, 3),
    (1, 1999, 48, 8, 128, 500, True, False, 0.0, True, 3),
    (1, 1200, 64, 8, 128, None, False, False, 0.0, True, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,nh,nkv,d,doc,prefix,pad,cap,alibi,shares", SHARED)
def test_some_of_a_group_in_every_share(B, S, nh, nkv, d, doc, prefix, pad, cap, alibi, shares):
    """Items that walk several query heads and leave their sums to be joined."""
    from mini_megatron_b200.ops import check_errors, native
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    assert native().masked_attn_dkv_parts(B, S, nh, nkv, native().num_sms()) == shares and 1 < shares < nh // nkv
    qkv, dctx, plan, start, end = _case(B, S, nh, nkv, d, doc, prefix, pad, 1.5, "cuda", torch.bfloat16, seed=11)
    slopes = _slopes(nh, "cuda") if alibi else None
    opts = dict(num_kv_heads=nkv, plan=plan, softcap=cap or None, alibi_slopes=slopes)
    ctx, lse = attention_fwd(qkv, nh, d, **opts)
    dqkv = attention_bwd(dctx, qkv, ctx, lse, nh, d, **opts)
    check_errors()
    for b in range(B):   # a row at a time: the 64-bit form holds several [S, S] tensors a head
        s, e = (None, None) if start is None else (start[b:b + 1], end[b:b + 1])
        (r_ctx, r_lse, r_grad), (b_ctx, b_lse, b_grad) = attention_ref(qkv[b:b + 1], dctx[b:b + 1], nh, nkv, d, s, e,
                                                                      cap, slopes)
        _near(ctx[b:b + 1], r_ctx, b_ctx, "ctx")
        _near(lse[b:b + 1], r_lse, b_lse, "lse")
        _near(dqkv[b:b + 1], r_grad, b_grad, "dqkv")


FIRST_CALL_CAPTURED = """
import torch
from mini_megatron_b200.ops import check_errors, native
from mini_megatron_b200.ops.attention import attention_fwd
x = torch.randn(1, 300, 192, device="cuda").bfloat16()
junk = [torch.full((4,), 77, device="cuda", dtype=torch.int32) for _ in range(8)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ctx, lse = attention_fwd(x, 1, 64)
check_errors()                       # nothing has run yet
native().set_error(7)
g.replay()
torch.cuda.synchronize()
assert native().get_error() == 7     # a replay does not clear what was recorded before it
native().clear_error()
g.replay()
check_errors()
want = attention_fwd(x, 1, 64)
assert torch.equal(ctx, want[0]) and torch.equal(lse, want[1])
del g, ctx, lse
torch.cuda.empty_cache()
attention_fwd(x, 1, 64)
check_errors()
print("fine")
"""


@pytest.mark.gpu
def test_first_call_inside_a_capture_keeps_the_error_word():
    """In a process of its own: the word that kernels report to does not belong to the graph."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=300,
                         cwd=root, env=dict(os.environ, PYTHONPATH=root))
    assert run.returncode == 0 and run.stdout.strip() == "fine", run.stdout + run.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e8])
@pytest.mark.parametrize("alibi", [False, True])
def test_very_large_scores(d, size, alibi):
    """Rows whose scores lie far apart see one key: ctx is its value and lse its score, however large the scores."""
    from mini_megatron_b200.ops.attention import attention_fwd
    qkv, _, plan, start, end = _case(2, 500, 2, 1, d, 200, True, True, 1.0, "cuda", torch.bfloat16, seed=21)
    slopes = _slopes(2, "cuda") if alibi else None
    scale = size / 4 / d ** 0.5          # q.k is a normal number times sqrt(d): the largest of a row about 4
    ctx, lse = attention_fwd(qkv, 2, d, num_kv_heads=1, plan=plan, alibi_slopes=slopes, softmax_scale=scale)
    q, k, v = (t.double() for t in qkv.view(2, 500, 4, d).transpose(1, 2).split([2, 1, 1], 1))
    at = torch.arange(500, device="cuda")
    x = q @ k.transpose(-1, -2) * scale
    if alibi:
        x = x - slopes.double().view(2, 1, 1) * (at[:, None] - at).abs()
    x = x.masked_fill(~((at >= start[..., None]) & (at < end[..., None]))[:, None], float("-inf"))
    top = x.topk(2, -1)
    # a 32-bit sum of d products and the scaling: off by at most 2^-23 (d + 4) of the products' size, which is below 64 d^0.5
    off = 2.0 ** -23 * (d + 4) * scale * 64 * d ** 0.5
    clear = top.values[..., 0] - top.values[..., 1] > 2 * off + 20   # the second key weighs less than e^-20
    assert clear.sum() > 0.8 * 2 * (end > start).sum()
    want = v.expand(2, 2, 500, d).gather(2, top.indices[..., :1].expand(-1, -1, -1, d))
    got = ctx.view(2, 500, 2, d).transpose(1, 2).double()
    err = (got - want).abs()
    # the key's weight and ctx are rounded once each
    assert (err <= 2.02 * 2.0 ** -8 * want.abs() + 2.0 ** -20)[clear].all()
    assert ((lse.double() - top.values[..., 0]).abs() <= off + 2.0 ** -21 * top.values[..., 0].abs() + 1e-6)[clear].all()
