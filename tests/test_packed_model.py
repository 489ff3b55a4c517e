"""Plan, rotary positions and masked attention together: as a chain, and inside the GPT and its trainer."""
import copy

import pytest
import torch
import torch.distributed as dist

from packed_ref import attention_ref, plan_ref, rotary_ref, row_tensors, split_rows


@pytest.fixture(scope="module", autouse=True)
def _pg():
    if not dist.is_initialized():
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)  # no port: workers run side by side
    yield


def _rel(a, b):
    return ((a.double() - b.double()).norm() / (b.double().norm() + 1e-12)).item()


def _cfg(**kw):
    from mini_megatron_b200.config import GPTConfig
    base = dict(num_layers=2, hidden_size=256, num_attention_heads=4, ffn_hidden_size=512, max_seq_len=256,
                vocab_size=500)
    return GPTConfig(**{**base, **kw})


VARIANTS = {
    "rotary_documents": (dict(position_embedding="rotary", eod_token=3), 200),
    "rotary_part_interleaved_shared_heads": (dict(position_embedding="rotary", rotary_percent=0.5,
                                                  rotary_interleaved=True, rotary_scaling="yarn", rotary_factor=4.0,
                                                  rotary_original_max_positions=64, num_kv_heads=2), 129),
    "distance_bias_capped": (dict(position_embedding="alibi", attn_softcap=20.0, eod_token=3), 256),
    "learned_capped_head128": (dict(attn_softcap=30.0, hidden_size=256, num_attention_heads=2, num_kv_heads=1), 77),
    "plain_odd_length": (dict(), 100),
}


def _build(cfg, seed=0):
    from mini_megatron_b200.models import build_gpt
    torch.manual_seed(seed)
    return build_gpt(cfg)


def _batch(cfg, B, S, seed=1):
    g = torch.Generator().manual_seed(seed)
    toks = torch.randint(0, cfg.vocab_size, (B, S + 1), generator=g)
    toks[torch.rand(B, S + 1, generator=g) < 0.03] = 3
    return toks[:, :-1].contiguous(), toks[:, 1:].contiguous(), torch.ones(B, S)


def test_packed_documents_equal_separate_documents():
    """A row of documents gives each of them the logits it has alone (CPU path)."""
    for pos in ("rotary", "alibi"):
        model = _build(_cfg(position_embedding=pos, eod_token=3, num_kv_heads=2)).double()
        g = torch.Generator().manual_seed(5)
        docs = [torch.cat([torch.randint(4, 500, (n - 1,), generator=g), torch.tensor([3])]) for n in (9, 1, 30, 14)]
        logits = model(torch.cat(docs)[None])[0]
        at = 0
        for doc in docs:
            torch.testing.assert_close(logits[at:at + len(doc)], model(doc[None])[0], rtol=1e-9, atol=1e-9)
            at += len(doc)


def test_prefix_plan_reaches_the_layers():
    """With a prefix both ways the first token sees the second; padding changes nothing else (CPU path)."""
    from mini_megatron_b200.ops.documents import document_plan
    model = _build(_cfg(position_embedding="rotary")).double()
    ids = torch.randint(4, 500, (1, 12), generator=torch.Generator().manual_seed(0))
    marks = torch.arange(12)[None] < 5
    plan = document_plan(ids, eod=3, prefix_mask=marks, lengths=torch.tensor([9]))
    base = model(ids, plan=plan)[0]
    other = ids.clone()
    other[0, 4] = 77
    assert not torch.allclose(model(other, plan=plan)[0, 0], base[0])
    other = ids.clone()
    other[0, 7] = 77
    changed = model(other, plan=plan)[0]
    torch.testing.assert_close(changed[:7], base[:7], rtol=0, atol=0)
    other = ids.clone()
    other[0, 10] = 77
    torch.testing.assert_close(model(other, plan=plan)[0][:9], base[:9], rtol=0, atol=0)


def test_model_refusals():
    from mini_megatron_b200.models import GPTStage
    from mini_megatron_b200.training import TrainConfig, Trainer
    for kw in [dict(position_embedding="other"), dict(num_kv_heads=3), dict(num_kv_heads=0), dict(attn_softcap=0.0),
               dict(position_embedding="rotary", rotary_percent=0.01), dict(position_embedding="rotary",
                                                                           rotary_scaling="yarn", rotary_factor=2.0)]:
        with pytest.raises(ValueError):
            _build(_cfg(**kw))
    with pytest.raises(ValueError):
        GPTStage(_cfg(eod_token=3), 0, 2)
    with pytest.raises(ValueError):
        Trainer(TrainConfig(model=_cfg(eod_token=3), pp=2), device="cpu", mpu=None)


def test_command_line_reaches_the_config():
    import main
    args = main.parse_args("--position-embedding rotary --rotary-percent 0.5 --rotary-interleaved --rotary-scaling ntk "
                           "--rotary-factor 2 --num-kv-heads 4 --attn-softcap 30 --eod-token 0".split())
    cfg = main.model_config(args)
    assert (cfg.position_embedding, cfg.rotary_percent, cfg.rotary_interleaved, cfg.rotary_scaling, cfg.rotary_factor,
            cfg.num_kv_heads, cfg.attn_softcap, cfg.eod_token) == ("rotary", 0.5, True, "ntk", 2.0, 4, 30.0, 0)
    assert main.model_config(main.parse_args([])) == main.model_config(main.parse_args(["--seq-len", "16"]))


@pytest.mark.parametrize("name", sorted(VARIANTS))
def test_parameter_count(name):
    cfg = _cfg(**VARIANTS[name][0])
    model = _build(cfg)
    assert sum(p.numel() for p in model.parameters()) == cfg.num_params(padded_vocab=512)


@pytest.mark.gpu
@pytest.mark.parametrize("d,nh,nkv", [(64, 4, 2), (128, 2, 2)])
def test_chain_against_64_bits(d, nh, nkv):
    """plan -> rotary -> attention and back, each step against the 64-bit form of that step on the same inputs."""
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    B, S = 3, 411
    rows = split_rows(B, S, 120, True, True, seed=9)
    tokens, _, marks, lengths = row_tensors(rows, S, seed=9)
    plan = document_plan(tokens.cuda(), eod=0, prefix_mask=marks.cuda(), lengths=lengths.cuda())
    pos, start, end = (t.cuda() for t in plan_ref(rows, S, True))
    assert torch.equal(plan.positions, pos) and torch.equal(plan.start, start) and torch.equal(plan.end, end)
    r = Rotary(d, rotary_dim=d // 2, scaling="linear", factor=2.0, device="cuda")
    qkv = torch.randn(B, S, (nh + 2 * nkv) * d, device="cuda").bfloat16()
    dctx = torch.randn(B, S, nh * d, device="cuda").bfloat16()
    want = rotary_ref(qkv, d, d // 2, nh + nkv, False, r.radians, 1.0, pos)
    rotary_fwd(qkv, r, nh + nkv, plan.positions, out=qkv)
    # a bf16 rounding (2^-8) of values that a 32-bit rotation leaves within 2^-20 of their pair
    assert ((qkv.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().max()).all()
    opts = dict(num_kv_heads=nkv, plan=plan, softcap=40.0)
    ctx, lse = attention_fwd(qkv, nh, d, **opts)
    dqkv = attention_bwd(dctx, qkv, ctx, lse, nh, d, **opts)
    (r_ctx, _, r_grad), (b_ctx, _, b_grad) = attention_ref(qkv, dctx, nh, nkv, d, start, end, 40.0)
    assert ((ctx.double() - r_ctx).abs() <= b_ctx).all() and ((dqkv.double() - r_grad).abs() <= b_grad).all()
    want = rotary_ref(dqkv, d, d // 2, nh + nkv, False, r.radians, 1.0, pos, inverse=True)
    rotary_bwd(dqkv, r, nh + nkv, plan.positions, out=dqkv)
    assert ((dqkv.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().max()).all()
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("S", [300, 1100])
def test_chain_without_pauses(S):
    """Buffers rewritten and used over and over without a pause give the bits of calls that are waited for each time:
    every kernel may be set up before its predecessor has finished, and reads nothing before."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    B, nh, nkv, d = 2, 4, 2, 64
    g = torch.Generator().manual_seed(S)
    rot = Rotary(d, device="cuda")
    data = [(torch.randint(0, 60, (B, S), generator=g).cuda(),
             torch.randn(B, S, (nh + 2 * nkv) * d, generator=g).bfloat16().cuda(),
             torch.randn(B, S, nh * d, generator=g).bfloat16().cuda()) for _ in range(3)]
    tokens, qkv, dctx = (torch.empty_like(t) for t in data[0])

    def step(k, pause):
        def wait():
            if pause:
                torch.cuda.synchronize()
        for t, new in zip((tokens, qkv, dctx), data[k % 3]):
            t.copy_(new)
        wait()
        plan = document_plan(tokens, eod=0)
        wait()
        rotary_fwd(qkv, rot, nh + nkv, plan.positions, out=qkv)
        wait()
        ctx, lse = attention_fwd(qkv, nh, d, num_kv_heads=nkv, plan=plan)
        wait()
        grad = attention_bwd(dctx, qkv, ctx, lse, nh, d, num_kv_heads=nkv, plan=plan)
        wait()
        return ctx, lse, rotary_bwd(grad, rot, nh + nkv, plan.positions, out=grad)

    want = [step(k, True) for k in range(3)]
    got = [step(k, False) for k in range(30)]
    torch.cuda.synchronize()
    for k, one in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(one, want[k % 3])), k


@pytest.mark.gpu
def test_activations_beyond_32_bit_offsets():
    """2.4 G elements: the last rows of the batch get the bits that they get alone."""
    from mini_megatron_b200.ops.attention import attention_bwd, attention_fwd
    from mini_megatron_b200.ops.documents import document_plan
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    B, S, nh, d = 1600, 1000, 8, 64
    torch.manual_seed(7)
    qkv = torch.randn(B, S, 3 * nh * d, device="cuda", dtype=torch.bfloat16)
    dctx = torch.randn(B, S, nh * d, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(0, 200, (B, S), device="cuda")
    rot = Rotary(d, device="cuda")
    assert qkv.numel() > 2 ** 31

    def run(qkv, dctx, tokens):
        plan = document_plan(tokens, eod=0)
        x = rotary_fwd(qkv, rot, 2 * nh, plan.positions)
        ctx, lse = attention_fwd(x, nh, d, plan=plan)
        grad = attention_bwd(dctx, x, ctx, lse, nh, d, plan=plan)
        return x[-2:].clone(), ctx[-2:].clone(), lse[-2:].clone(), rotary_bwd(grad, rot, 2 * nh, plan.positions)[-2:].clone()

    whole, alone = run(qkv, dctx, tokens), run(qkv[-2:], dctx[-2:], tokens[-2:])
    assert all(torch.equal(a, b) for a, b in zip(whole, alone))


@pytest.mark.gpu
def test_captured_backward_and_a_live_eager_graph():
    from mini_megatron_b200.ops.attention import attention
    from mini_megatron_b200.ops.rotary import Rotary, apply_rotary
    rot = Rotary(64, device="cuda")
    x = torch.randn(1, 200, 3 * 64, device="cuda").bfloat16().requires_grad_(True)
    dctx = torch.randn(1, 200, 64, device="cuda").bfloat16()

    def grad():
        return torch.autograd.grad(attention(apply_rotary(x, rot, 2), 1, 64), x, dctx)[0]

    want = grad()
    alive = attention(x, 1, 64)
    for f in (lambda: attention(x, 1, 64), lambda: apply_rotary(x, rot, 2)):
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                f()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grad()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(VARIANTS))
def test_native_model_matches_cpu(name):
    """Loss and gradients of the native model against the fp32 CPU path on the same weights.

    The gates are those of the plain model's parity test: bf16 operands in every product (2^-8 each) through two layers.
    """
    from mini_megatron_b200.ops import check_errors
    from mini_megatron_b200.optim import make_param_buffer
    kw, S = VARIANTS[name]
    cfg = _cfg(**kw)
    cpu = _build(cfg)
    gpu = copy.deepcopy(cpu).cuda()
    ids, labels, mask = _batch(cfg, 2, S)
    _, want = cpu(ids, labels, mask)
    want.backward()
    make_param_buffer(gpu)
    _, loss = gpu(ids.cuda(), labels.cuda(), mask.cuda())
    loss.backward()
    torch.cuda.synchronize()
    check_errors()
    assert abs(loss.item() - want.item()) < 2e-2 * abs(want.item())
    for (n, a), (_, b) in zip(cpu.named_parameters(), gpu.named_parameters()):
        assert _rel(b.main_grad.cpu(), a.grad) < 5e-2, n


@pytest.mark.gpu
def test_standalone_attention_module():
    from mini_megatron_b200.models import Attention, AttentionSpec
    from mini_megatron_b200.ops.rotary import Rotary
    torch.manual_seed(0)
    cpu = Attention(256, 4, spec=AttentionSpec(num_kv_heads=2, rotary=Rotary(64), softcap=20.0))
    gpu = copy.deepcopy(cpu).cuda()
    x = torch.randn(2, 90, 256)
    a, b = x.clone().requires_grad_(True), x.cuda().requires_grad_(True)
    ya, yb = cpu(a), gpu(b)
    dy = torch.randn_like(ya)
    (ga,) = torch.autograd.grad(ya, a, dy)
    (gb,) = torch.autograd.grad(yb, b, dy.cuda().to(yb.dtype))
    assert _rel(yb.cpu().detach(), ya.detach()) < 2e-2 and _rel(gb.cpu(), ga) < 5e-2


@pytest.mark.gpu
def test_trainer_graph_recompute_and_eager_agree():
    """A packed, rotary, capped model: the captured step rebuilds its plan from every batch's tokens."""
    from mini_megatron_b200.parallel import process_groups as pg
    from mini_megatron_b200.training import TrainConfig, Trainer, synthetic_batch
    mc = _cfg(position_embedding="rotary", attn_softcap=30.0, eod_token=7, vocab_size=64, num_kv_heads=2)
    runs = {}
    for mode, rc in (("off", False), ("on", False), ("off", True)):
        t = Trainer(TrainConfig(model=mc, micro_batch_size=2, seq_len=150, num_microbatches=2, lr=1e-3, warmup_steps=2,
                                num_steps=20, cuda_graph=mode, recompute=rc))
        losses = [t.train_step(*synthetic_batch(2, 2, 150, 64, seed=s, pin=True)).item() for s in range(5)]
        t.check_device_errors()
        runs[mode, rc] = losses
        t.destroy()
        pg.set_model_parallel(None)
    for other in (("on", False), ("off", True)):
        for a, b in zip(runs["off", False], runs[other]):
            assert abs(a - b) < 2e-3 * abs(a), runs


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_recomputed_layer_takes_the_plan(device):
    """A checkpointed layer attends inside the documents, like the layer itself."""
    from mini_megatron_b200.models.recompute import checkpoint
    from mini_megatron_b200.ops.documents import document_plan
    from mini_megatron_b200.optim import make_param_buffer
    layer = _build(_cfg(position_embedding="alibi", num_kv_heads=2)).decoder.layers[0].to(device)
    if device == "cuda":
        make_param_buffer(layer)
    tokens = torch.randint(0, 9, (2, 140), generator=torch.Generator().manual_seed(2)).to(device)
    plan = document_plan(tokens, eod=3)
    x = torch.randn(2, 140, 256, generator=torch.Generator().manual_seed(3)).to(device)
    outs = []
    for run in (lambda z: layer(z, plan=plan), lambda z: checkpoint(layer, z, plan)):
        leaf = x.clone().requires_grad_(True)
        y = run(leaf)
        (grad,) = torch.autograd.grad(y.square().sum(), leaf)
        outs.append((y.detach(), grad))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not torch.equal(outs[0][0], checkpoint(layer, x).detach())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_slopes_keep_their_bits(dtype):
    """Turning a model into another type does not round the distance bias: 12 slopes are no powers of two."""
    from mini_megatron_b200.ops.attention import alibi_slopes
    model = _build(_cfg(position_embedding="alibi", hidden_size=12 * 8, num_attention_heads=12))
    for turned in (model.to(dtype), copy.deepcopy(model), model.float()):
        for layer in turned.decoder.layers:
            assert layer.attn.alibi_slopes.dtype == torch.float32
            assert torch.equal(layer.attn.alibi_slopes, alibi_slopes(12))
    assert not any("alibi" in k for k in model.state_dict())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_longer_than_the_position_table_are_refused(device):
    """Any row length runs, but a learned table ends at max_seq_len; models without one have no such end."""
    ids = torch.zeros(1, 300, dtype=torch.int64, device=device)
    model = _build(_cfg(max_seq_len=256)).to(device)
    with pytest.raises((IndexError, RuntimeError)):
        model(ids)
    assert model(ids[:, :256]).shape[:2] == (1, 256)
    if device == "cuda":
        from mini_megatron_b200.ops import native
        dwte, dwpe = torch.zeros(512, 256, device=device), torch.zeros(256, 256, device=device)
        with pytest.raises(RuntimeError, match="position table"):
            native().embedding_bwd(ids.view(-1), torch.zeros(300, 256, device=device), dwte, dwpe, 1, 300, 0, 512)
    assert _build(_cfg(max_seq_len=256, position_embedding="rotary")).to(device)(ids).shape[:2] == (1, 300)


def test_trainer_row_length_without_a_position_table():
    from mini_megatron_b200.parallel import process_groups as pg
    from mini_megatron_b200.training import TrainConfig, Trainer, synthetic_batch
    small = dict(num_layers=1, hidden_size=32, num_attention_heads=2, ffn_hidden_size=64, max_seq_len=16, vocab_size=50)
    for pos in ("rotary", "alibi"):
        t = Trainer(TrainConfig(model=_cfg(**small, position_embedding=pos), micro_batch_size=2, seq_len=24), device="cpu")
        assert torch.isfinite(t.train_step(*synthetic_batch(1, 2, 24, 50)))
        t.destroy()
        pg.set_model_parallel(None)
    with pytest.raises(ValueError, match="position table"):
        Trainer(TrainConfig(model=_cfg(**small), micro_batch_size=2, seq_len=24), device="cpu")
    pg.set_model_parallel(None)


def test_learned_positions_count_along_a_packed_row():
    """A document behind others gets the logits that it has alone with the table's rows from where it begins."""
    model = _build(_cfg(eod_token=3)).double()
    g = torch.Generator().manual_seed(5)
    docs = [torch.cat([torch.randint(4, 500, (n - 1,), generator=g), torch.tensor([3])]) for n in (9, 1, 30)]
    logits = model(torch.cat(docs)[None])[0].detach()
    table = model.embedding.position_embedding.weight
    rows, at = table.detach().clone(), 0
    for doc in docs:
        with torch.no_grad():
            table.copy_(rows.roll(-at, 0))
        torch.testing.assert_close(logits[at:at + len(doc)], model(doc[None])[0].detach(), rtol=1e-9, atol=1e-9)
        at += len(doc)
