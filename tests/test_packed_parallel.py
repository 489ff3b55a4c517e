"""Attention variants under tensor and sequence parallelism (gloo, CPU).

Every rank holds its own heads: the distance bias has to be cut with them, rotary positions have to turn them as the
whole model does, and the plan of packed documents has to reach every rank.  Logits and gradients of two ranks are
those of one process, in 64 bits (from a given gradient of the logits: the sharded cross-entropy works in 32).
"""
import pytest
import torch

from dist_util import run_ranks

CFG = dict(num_layers=2, hidden_size=48, num_attention_heads=6, ffn_hidden_size=96, max_seq_len=32, vocab_size=1000)
B, S = 2, 32
VARIANTS = {
    "alibi": dict(position_embedding="alibi"),
    "alibi_documents_capped": dict(position_embedding="alibi", eod_token=3, attn_softcap=5.0),
    "rotary_documents": dict(position_embedding="rotary", eod_token=3),
    "rotary_part_interleaved": dict(position_embedding="rotary", rotary_percent=0.5, rotary_interleaved=True,
                                    rotary_scaling="ntk", rotary_factor=2.0, attn_softcap=5.0),
    "learned_documents": dict(eod_token=3),
}


def _config(name):
    from mini_megatron_b200.config import GPTConfig
    return GPTConfig(**CFG, **VARIANTS[name])


def _batch():
    g = torch.Generator().manual_seed(4)
    toks = torch.randint(0, CFG["vocab_size"], (B, S + 1), generator=g)
    toks[torch.rand(B, S + 1, generator=g) < 0.15] = 3
    return toks[:, :-1].contiguous(), torch.randn(B, S, 1024, generator=g, dtype=torch.float64)


def _shard(full, name, world, rank):
    """This rank's part of an unsharded tensor: Q, K and V in equal parts, rows, columns or all of it."""
    if name.endswith("attn.qkv.weight"):
        return torch.cat([part.chunk(world)[rank] for part in full.chunk(3)])
    if name.endswith(("mlp.fc1.weight", "lm_head.weight", "token_embedding.weight")):
        return full.chunk(world)[rank]
    if name.endswith(("attn.o.weight", "mlp.fc2.weight")):
        return full.chunk(world, 1)[rank]
    return full


def _whole(name):
    """Weights, logits and gradients of one process."""
    from mini_megatron_b200.models import build_gpt
    cfg = _config(name)
    cfg.vocab_pad_multiple = 256     # the table's size under tp = 2
    torch.manual_seed(7)
    model = build_gpt(cfg).double()
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("attn.qkv.weight"):
                p.mul_(12.0)         # scores that a cap or a bias of the wrong head would change
    tokens, dlogits = _batch()
    logits = model(tokens)
    logits.backward(dlogits)
    return model.state_dict(), logits.detach(), {n: p.grad for n, p in model.named_parameters()}


def _tp_worker(rank, world, sp, states):
    from mini_megatron_b200.models import build_gpt
    from mini_megatron_b200.parallel import process_groups as pg
    from mini_megatron_b200.parallel.data_parallel import allreduce_sequence_parallel_grads
    mpu = pg.init_model_parallel(world, 1, sp)
    pg.set_model_parallel(mpu)
    tokens, dlogits = _batch()
    out = {}
    for name, state in states.items():
        model = build_gpt(_config(name)).double()
        model.load_state_dict({n: _shard(state[n], n, world, rank) for n in model.state_dict()})
        logits = model(tokens)
        logits.backward(dlogits.chunk(world, -1)[rank])
        if sp:
            allreduce_sequence_parallel_grads([p for p in model.parameters()
                                               if getattr(p, "sequence_parallel_grad", False)], mpu["tp_group"])
        out[name] = logits.detach(), {n: p.grad for n, p in model.named_parameters()}
    pg.set_model_parallel(None)
    return out


@pytest.mark.parametrize("sp", [False, True])
def test_two_tensor_parallel_ranks(sp):
    whole = {name: _whole(name) for name in VARIANTS}
    results = run_ranks(_tp_worker, 2, sp, {name: w[0] for name, w in whole.items()})
    for rank, result in enumerate(results):
        for name, (logits, got) in result.items():
            _, want, grads = whole[name]
            # sums of about a hundred terms in 64 bits, in another order: 2^-53 * 100 a step, a dozen steps
            torch.testing.assert_close(logits, want.chunk(2, -1)[rank], rtol=1e-9, atol=1e-9, msg=name)
            assert set(got) == set(grads)
            for n, g in got.items():
                torch.testing.assert_close(g, _shard(grads[n], n, 2, rank), rtol=1e-9, atol=1e-9, msg=f"{name} {n}")
