"""Rotary positions against the complex rotation in 64 bits."""
import math

import pytest
import torch

from packed_ref import HALF_STEP, rotary_ref


def _rotary(d, rot, interleaved, scaling, device=None):
    from mini_megatron_b200.ops.rotary import Rotary
    return Rotary(d, rotary_dim=rot, interleaved=interleaved, scaling=scaling, factor=8.0 if scaling else 1.0,
                  original_max_positions=2048, device=device)


def _positions(kind, B, S):
    if kind is None:
        return None
    g = torch.Generator().manual_seed(S)
    if kind == "row":
        return torch.randint(0, 5000, (S,), generator=g, dtype=torch.int64)
    if kind == "far":
        return torch.randint(0, 2 ** 31 - 1, (B, S), generator=g, dtype=torch.int64).to(torch.int32)
    return torch.randint(-100, 2 ** 40, (B, S), generator=g, dtype=torch.int64)


def _bound(x, d, rot, heads, interleaved, m, far):
    """|error| of a rotated value: its rounding, the 32-bit rotation (products, sum, sine and cosine) and the angle.

    The turn is reduced in 64 bits and rounded to 32 (half a step of a value up to 1/2: 2^-26 turns), the 64-bit
    product itself is off by 2^-53 of the turns.
    """
    y = rotary_ref(x.abs(), d, rot, heads, interleaved, torch.zeros(rot // 2, dtype=torch.float64), 1.0,
                   torch.zeros(x.shape[1], device=x.device))
    v = y.view(*x.shape[:2], -1, d).clone()
    part = v[:, :, :heads, :rot]
    if interleaved:
        pairs = part.unflatten(-1, (-1, 2))
        part.copy_(pairs.sum(-1, keepdim=True).expand_as(pairs).flatten(-2))
    else:
        a, b = part.chunk(2, -1)
        part.copy_(torch.cat([a + b, a + b], -1))
    angle = 2 * math.pi * (2.0 ** -26 + 2.0 ** -52 * far)
    per = HALF_STEP[x.dtype] + 6 * 2.0 ** -23 + angle
    return (v.view(x.shape) * abs(m) * per * 1.01 + 1e-30)


GRID = [  # B, S, heads, rotated heads, d, rot, interleaved, scaling, positions
    (1, 1, 3, 2, 64, 64, False, None, None),
    (2, 7, 12, 8, 64, 64, False, None, "row"),
    (2, 65, 6, 4, 128, 64, True, "yarn", "any"),
    (3, 33, 5, 5, 64, 32, True, "linear", None),
    (1, 130, 4, 3, 128, 128, False, "ntk", "far"),
    (2, 19, 3, 1, 96, 48, False, None, "any"),
    (1, 1500, 3, 2, 16, 16, True, None, "far"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,n,d,rot,inter,scaling,pos", GRID)
def test_rotary_gpu(B, S, H, n, d, rot, inter, scaling, pos, dtype):
    from mini_megatron_b200.ops.rotary import rotary_bwd, rotary_fwd
    r = _rotary(d, rot, inter, scaling, "cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, S, H * d, device="cuda", generator=g).to(dtype)
    p = _positions(pos, B, S)
    p = p.cuda() if p is not None else None
    want_p = p if p is not None else torch.arange(S, device="cuda")
    far = want_p.abs().max().item() / (2 * math.pi)
    for fn, inverse in ((rotary_fwd, False), (rotary_bwd, True)):
        got = fn(x, r, n, p)
        want = rotary_ref(x, d, rot, n, inter, r.radians, r.magnitude, want_p, inverse)
        assert got.dtype == dtype and got.is_contiguous()
        assert ((got.double() - want).abs() <= _bound(x, d, rot, n, inter, r.magnitude, far)).all()
        # what is not rotated is copied bit for bit
        v, o = x.view(B, S, H, d), got.view(B, S, H, d)
        assert torch.equal(v[:, :, n:], o[:, :, n:]) and torch.equal(v[..., rot:], o[..., rot:])
        inplace = x.clone()
        assert fn(inplace, r, n, p, out=inplace) is inplace
        assert torch.equal(inplace, got)


@pytest.mark.parametrize("B,S,H,n,d,rot,inter,scaling,pos", GRID)
def test_rotary_cpu(B, S, H, n, d, rot, inter, scaling, pos):
    from mini_megatron_b200.ops.rotary import apply_rotary, rotary_bwd, rotary_fwd
    r = _rotary(d, rot, inter, scaling)
    x = torch.randn(B, S, H * d, dtype=torch.float64)
    p = _positions(pos, B, S)
    want_p = p if p is not None else torch.arange(S)
    want = rotary_ref(x, d, rot, n, inter, r.radians, r.magnitude, want_p)
    torch.testing.assert_close(rotary_fwd(x, r, n, p), want, rtol=1e-12, atol=1e-12)
    dy = torch.randn_like(x)
    leaf = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(apply_rotary(leaf, r, n, p), leaf, dy)
    torch.testing.assert_close(got, rotary_ref(dy, d, rot, n, inter, r.radians, r.magnitude, want_p, True),
                               rtol=1e-12, atol=1e-12)
    assert torch.equal(got, rotary_bwd(dy, r, n, p))
    # against differences: the map is linear, so a difference of any size is exact
    step = torch.randn_like(x)
    change = rotary_fwd(x + step, r, n, p) - rotary_fwd(x, r, n, p)
    assert math.isclose((change * dy).sum().item(), (got * step).sum().item(), rel_tol=1e-9, abs_tol=1e-9)


def test_frequencies():
    plain, lin, ntk, yarn = (_rotary(64, 64, False, s) for s in (None, "linear", "ntk", "yarn"))
    want = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    torch.testing.assert_close(plain.radians, want, rtol=1e-14, atol=0)
    torch.testing.assert_close(lin.radians, want / 8, rtol=1e-14, atol=0)
    assert ntk.radians[0] == 1 and abs(ntk.radians[-1] / want[-1] - 1 / 8) < 1e-12
    turns = want * 2048 / (2 * math.pi)
    kept, divided = turns > 40, turns < 0.8     # clear of the ramp's ends, which are rounded to whole pairs
    assert kept.any() and divided.any()
    assert torch.equal(yarn.radians[kept], want[kept])
    torch.testing.assert_close(yarn.radians[divided], want[divided] / 8, rtol=1e-14, atol=0)
    assert (yarn.radians <= want).all() and (yarn.radians >= want / 8 * (1 - 1e-12)).all()
    assert yarn.magnitude == 0.1 * math.log(8.0) + 1 and plain.magnitude == lin.magnitude == ntk.magnitude == 1.0


def test_rotary_refusals():
    from mini_megatron_b200.ops.rotary import Rotary, rotary_fwd
    for kw in [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=66), dict(scaling="other"), dict(base=1.0),
               dict(factor=0.5), dict(scaling="yarn", factor=2.0), dict(base=math.inf), dict(factor=math.nan)]:
        with pytest.raises(ValueError):
            Rotary(64, **kw)
    r = Rotary(64)
    x = torch.zeros(2, 3, 192)
    for args in [(x[0], r, 1), (x, r, 4), (x, r, 0), (x, r, 2, torch.zeros(2, dtype=torch.int64)),
                 (x, r, 2, torch.zeros(3)), (torch.zeros(2, 3, 100), r, 1)]:
        with pytest.raises(ValueError):
            rotary_fwd(*args)


@pytest.mark.gpu
def test_rotary_refusals_gpu():
    from mini_megatron_b200.ops.rotary import Rotary, rotary_fwd
    r = Rotary(64, device="cuda")
    x = torch.zeros(2, 4, 192, device="cuda", dtype=torch.bfloat16)
    bad = [(x.half(), r, 1), (x, r, 4), (x, r, 0), (x, r, 1, torch.zeros(4)), (x, r, 1, torch.zeros(3, device="cuda")),
           (x, r, 1, torch.zeros(2, 5, device="cuda", dtype=torch.int32)), (x[:, :, 1:], r, 1), (x[:, :, :100], r, 1),
           (x, Rotary(64, rotary_dim=24, device="cuda"), 1), (x.transpose(1, 2)[:, :64].transpose(1, 2)[..., ::2], r, 1)]
    for args in bad:
        with pytest.raises(RuntimeError):
            rotary_fwd(*args)
    with pytest.raises(RuntimeError):    # overlapping, but not in place
        rotary_fwd(x[:, 1:], r, 1, out=x[:, :-1])
    with pytest.raises(RuntimeError):
        rotary_fwd(x, r, 1, out=torch.empty_like(x[:, :2]))
    wide = torch.zeros(2, 4, 200, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):    # one row for the whole batch
        rotary_fwd(x, r, 1, out=wide[:1, :, :192].expand(2, 4, 192))


@pytest.mark.gpu
def test_rotary_strides_streams_graph_and_empty():
    from mini_megatron_b200.ops.rotary import Rotary, apply_rotary, rotary_fwd
    r = Rotary(64, device="cuda")
    wide = torch.randn(3, 40, 400, device="cuda").bfloat16()
    x = wide[:, 5:25, 8:200]
    want = rotary_fwd(x.contiguous(), r, 2)
    assert torch.equal(rotary_fwd(x, r, 2), want)
    dst = torch.full_like(wide, 9.0)
    rotary_fwd(x, r, 2, out=dst[:, 5:25, 8:200])
    assert torch.equal(dst[:, 5:25, 8:200], want)
    dst[:, 5:25, 8:200] = 9.0
    assert (dst == 9.0).all()                                # nothing around the target was written
    before = wide.clone()
    rotary_fwd(x, r, 2, out=x)
    assert torch.equal(x, want)
    wide[:, 5:25, 8:200] = before[:, 5:25, 8:200]
    assert torch.equal(wide, before)
    rows = torch.randn(20, 3, 192, device="cuda").bfloat16().transpose(0, 1)   # token-major batch
    assert torch.equal(rotary_fwd(rows, r, 2), rotary_fwd(rows.contiguous(), r, 2))
    assert rotary_fwd(x[:0], r, 2).shape == (0, 20, 192)
    # another stream, and a graph replayed on new values with its own output
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = rotary_fwd(x, r, 2)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, rotary_fwd(x, r, 2))
    buf = x.contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rotary_fwd(buf, r, 2)
    buf.copy_(torch.randn_like(buf))
    g.replay()
    assert torch.equal(y, rotary_fwd(buf, r, 2))
    leaf = buf.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(apply_rotary(leaf, r, 2).float().sum(), leaf)
    ones = torch.ones_like(leaf)
    from mini_megatron_b200.ops.rotary import rotary_bwd
    assert torch.equal(dx, rotary_bwd(ones, r, 2))


@pytest.mark.gpu
def test_rotary_frequencies_are_not_copied_in_a_capture():
    from mini_megatron_b200.ops.rotary import Rotary
    r = Rotary(64)
    x = torch.zeros(1, 4, 192, device="cuda", dtype=torch.bfloat16)
    real = torch.cuda.is_current_stream_capturing
    try:
        torch.cuda.is_current_stream_capturing = lambda: True
        with pytest.raises(RuntimeError, match="device="):
            r.turns(x.device)
    finally:
        torch.cuda.is_current_stream_capturing = real
    assert r.turns(x.device).is_cuda


@pytest.mark.gpu
def test_rotary_wide_heads():
    """Heads of 4096 over many tokens: the angles of four tokens would not fit a CTA's shared memory."""
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    rot = Rotary(4096)
    x = torch.randn(1, 6000, 4096, device="cuda").bfloat16()
    y = rotary_fwd(x, rot, 1)
    some = torch.tensor([0, 1, 2999, 5999])
    want = rotary_fwd(x[:, some].cpu().double(), rot, 1, positions=some)
    # a' and b' are sums of two products: angle to 2^-24 of a turn (2 pi 2^-24 relative to the pair's length), two
    # 32-bit roundings, then half a step of bf16
    size = x[:, some].cpu().double().abs().amax()
    bound = want.abs() * 2.0 ** -8 + size * 2 * 2.0 ** -20
    assert ((y[:, some].cpu().double() - want).abs() <= bound).all()
    back = rotary_bwd(y, rot, 1)
    # two roundings of bf16, each at most 2^-8 of the pair's length
    assert ((back.double() - x.double()).abs() <= 4 * 2.0 ** -8 * size.item()).all()


@pytest.mark.gpu
def test_rotary_in_place_is_seen_by_autograd():
    """Writing to ``out`` is refused where a gradient would miss it, and noticed by graphs that saved the tensor."""
    from mini_megatron_b200.ops.attention import attention
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    r = Rotary(64, device="cuda")
    leaf = torch.randn(1, 40, 192, device="cuda").bfloat16().requires_grad_(True)
    plain = leaf.detach().clone()
    inner = leaf * 1
    for x, out in ((leaf, leaf), (inner, inner), (inner, plain.clone()), (plain, inner)):
        for fn in (rotary_fwd, rotary_bwd):
            before, version = out.detach().clone(), out._version
            with pytest.raises(RuntimeError, match="apply_rotary"):
                fn(x, r, 2, out=out)
            assert torch.equal(out, before) and out._version == version
    # saved by an operator, then overwritten
    for write in (lambda t: rotary_fwd(t, r, 2, out=t), lambda t: rotary_bwd(t, r, 2, out=t),
                  lambda t: rotary_fwd(plain, r, 2, out=t)):
        x = leaf * 1
        y = attention(x, 1, 64)
        with torch.no_grad():
            write(x)
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.sum().backward()
    # a view shares its base's counter; a refused call counts nothing
    base = plain.clone()
    version = base._version
    rotary_fwd(base.view(1, 40, 192), r, 2, out=base.view(1, 40, 192))
    assert base._version == version + 1
    with pytest.raises(RuntimeError):
        rotary_fwd(base, r, 4, out=base)
    assert base._version == version + 1
    # without gradients: the values of the call that returns a new tensor
    want = rotary_fwd(plain, r, 2)
    with torch.no_grad():
        assert torch.equal(rotary_fwd(leaf, r, 2, out=leaf.detach().clone()), want)
        rotary_fwd(leaf, r, 2, out=leaf)
    assert torch.equal(leaf.detach(), want)
    with torch.inference_mode():
        x = plain * 1
        assert torch.equal(rotary_fwd(x, r, 2, out=x), want)


def test_rotary_in_place_gradients_cpu():
    """On the CPU ``out`` is an ordinary in-place operation: recorded, and refused for leaves."""
    from mini_megatron_b200.ops.rotary import Rotary, rotary_bwd, rotary_fwd
    r = Rotary(16)
    leaf = torch.randn(2, 5, 48, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(2, 5, 48, dtype=torch.float64)
    x = leaf * 1
    rotary_fwd(x, r, 2, out=x)
    (grad,) = torch.autograd.grad(x, leaf, dy)
    torch.testing.assert_close(grad, rotary_bwd(dy, r, 2), rtol=1e-12, atol=1e-12)
    with pytest.raises(RuntimeError):
        rotary_fwd(leaf, r, 2, out=leaf)
