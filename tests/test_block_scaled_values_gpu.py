"""Block-scaled 8-bit path on the device: values at the edges of their types, byte for byte where the definition gives bytes."""
import pytest
import torch

import bitblas_amd as bitblas
from test_block_scaled_gpu import T8, TO, gen, plain_quantise

pytestmark = pytest.mark.gpu


def same_bytes(q, want):
    """the bytes of two tensors of 8-bit values, whatever NaN is where one is NaN"""
    q, want = q.cpu(), want.cpu()
    nan = want.float().isnan()
    return torch.equal(q.float().isnan(), nan) and torch.equal(q.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


@pytest.mark.parametrize("dtype", list(T8))
@pytest.mark.parametrize("x", list(TO))
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape", [(1, 128), (5, 200), (130, 644)], ids=lambda s: "x".join(map(str, s)))
def test_quantise_bytes_with_signed_zeros(shape, tile, x, dtype):
    """zeros keep their sign, in blocks of nothing else too, and so do values that round to zero: the definition's bytes"""
    g = gen(sum(shape))
    t = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-24, 1, shape, generator=g).float())
    t[torch.rand(*shape, generator=g) < 0.2] = 0.0
    t[torch.rand(*shape, generator=g) < 0.2] = -0.0
    t[-1, :128] = -0.0
    t = t.to(TO[x])
    q, s = bitblas.quantize_blocks(t.cuda(), dtype, tile=tile)
    wq, ws = plain_quantise(t, dtype, tile)
    assert torch.equal(s.cpu(), ws) and same_bytes(q, wq)
    assert ((wq.view(torch.uint8) == 0x80).sum() > 0).item()


@pytest.mark.parametrize("dtype", list(T8))
@pytest.mark.parametrize("x", list(TO))
def test_gate_and_norm_keep_the_sign_of_zero(x, dtype):
    """silu(g) u and h r w are zeros of the sign that the factors' signs make"""
    sign = torch.tensor([0.0, -0.0, 1.0, -1.0]).repeat(32)
    up = torch.stack([sign, sign.flip(0), -sign, sign]).to(TO[x]).cuda()
    gate = torch.tensor([[-0.0], [0.0], [2.0], [-3.0]]).expand(4, 128).to(TO[x]).cuda()
    q, s = bitblas.quantize_blocks(up, dtype, gate=gate)
    want = torch.signbit(up) ^ torch.signbit(gate)
    assert torch.equal(q.view(torch.uint8) >= 0x80, want)
    if x == "float32":
        return
    w = torch.where(torch.arange(128) % 3 == 0, -1.0, 1.0).to(TO[x]).cuda()
    q, s = bitblas.residual_norm(up, None, w, 1e-5, quantize=dtype)[1]
    assert torch.equal(q.view(torch.uint8) >= 0x80, torch.signbit(up) ^ torch.signbit(w))


@pytest.mark.parametrize("dtype", list(T8))
@pytest.mark.parametrize("x", ["bfloat16", "float32"])
def test_gates_up_to_the_largest_of_the_type(x, dtype):
    """silu(g) is g for a large gate and 0 for a large negative one, also where g log2 e leaves float32; an infinite or NaN gate is for its own
    block only.  silu(g) u is exact here up to 2^-24 of it (u a power of two, exp(-g) beyond 24 bits), and so is the float32 quotient."""
    top = torch.finfo(TO[x]).max
    g = torch.tensor([top, top * 0.75, top * 0.69, 2.0 ** 127, 1e38, 3e5, 200.0, 40.0, -top, -top * 0.75, -2.0 ** 127, -1e38, -1e6, -200.0, 0.0, -0.0])
    gate = torch.stack([g.repeat(8).roll(i) for i in range(3)] + [g.repeat(8)] * 3).to(TO[x])
    up = torch.stack([torch.full((128,), 2.0 ** -e) for e in (0, 1, 100, 3, 0, 0)]).to(TO[x])
    gate = torch.cat([gate, gate.flip(1)], 1)
    up = torch.cat([up, -up], 1)
    gate[3, 5], gate[4, 200], gate[5, 7] = float("nan"), float("inf"), -float("inf")
    q, s = (t.cpu() for t in bitblas.quantize_blocks(up.cuda(), dtype, gate=gate.cuda()))
    bad = torch.zeros(6, 2, dtype=torch.bool)
    bad[3, 0] = bad[4, 1] = bad[5, 0] = True
    assert torch.equal(~s.isfinite(), bad)
    v = (gate.double() * torch.sigmoid(gate.double()) * up.double()).float()
    wq, ws = plain_quantise(torch.where(bad.repeat_interleave(128, 1), float("nan"), v), dtype)
    assert torch.equal(s[~bad], ws[~bad]) and same_bytes(q, wq)


@pytest.mark.parametrize("x", ["bfloat16", "float32"])
def test_gates_where_the_exponential_leaves_float32(x):
    """gates from -78 to -104: exp(-g) nears float32's largest value and leaves it, 1 / (1 + exp(-g)) its smallest normal one, 2^-126, below which
    it may be 0.  One value to a block, so that the scale is the value itself; u, 2^94, keeps it above the scale's floor.  Roundings: 8, and the
    exponential's argument's, |g| each."""
    g = torch.arange(-104.0, -78.0, 0.0625).to(TO[x])
    gate, up = (torch.zeros(g.numel(), 128, dtype=TO[x]) for _ in range(2))
    gate[:, 3], up[:, 3] = g, 2.0 ** 94
    s = bitblas.quantize_blocks(up.cuda(), gate=gate.cuda())[1][:, 0].cpu().double()
    g = g.double()
    want = (g * torch.sigmoid(g) * 2.0 ** 94).abs()
    off = (s * 448.0 - want.clamp_min(2.0 ** -40)).abs()
    assert bool((off <= want * (8 + 2 * g.abs()) * 2.0 ** -24 + g.abs() * 2.0 ** (94 - 126) + 2.0 ** -62).all())


U = 2.0 ** -24


@pytest.mark.parametrize("x", list(TO))
def test_gate_roundings(x):
    """silu(g) u, read from the scale of blocks that hold nothing else, within 2 + 3 sigmoid(-g) roundings for the gate's sigmoid (1 + exp(-g) and its
    reciprocal; exp(-g): one for its argument's lower part, two for a unit of the exponential) and three for the two products and the scale"""
    n = 1 << 14
    g = (torch.rand(n, generator=gen(21)) * 120 - 80).to(TO[x])
    if x == "float16":
        g = g * 0.125
    gate, up = (torch.zeros(n, 128, dtype=TO[x]) for _ in range(2))
    at = torch.arange(n) % 128
    gate[torch.arange(n), at] = g
    up[torch.arange(n), at] = (1 + torch.rand(n, generator=gen(22))).to(TO[x]) * (1.0 if x == "float16" else 2.0 ** 90)
    s = bitblas.quantize_blocks(up.cuda(), gate=gate.cuda())[1][:, 0].cpu().double()
    g, u = g.double(), up[torch.arange(n), at].double()
    want = (g * torch.sigmoid(g) * u).abs()
    keep = want > 2.0 ** -39
    assert keep.sum() > n // 2
    tol = want * (2 + 3 * torch.sigmoid(-g) + 3 + 0.1) * U
    off = (s * 448.0 - want).abs()
    assert bool((off <= tol)[keep].all()), f"worst {(off / tol)[keep].max().item():.3f} of the tolerance"


def _near_borders(n, seed):
    """midpoints between two neighbouring e4m3 values"""
    g = gen(seed)
    return (torch.randint(8, 16, (n,), generator=g) + 0.5).double() * torch.exp2(torch.randint(-8, 5, (n,), generator=g).double())


def _steps(t, seed):
    """float32 values moved by up to two of their own steps"""
    move = torch.randint(-2, 3, t.shape, generator=gen(seed), dtype=torch.int32)
    return (t.view(torch.int32) + move).view(torch.float32)


def _check_borders(q, s, want, roundings):
    """the bytes of `want` wherever its quotient lies further than so many roundings from a border between two 8-bit values"""
    quotient = want / s.double()
    step = torch.exp2(torch.floor(torch.log2(quotient.abs().clamp_min(2.0 ** -6))) - 3)
    part = quotient.abs() / step
    away = (part - (part.floor() + 0.5)).abs() * step / quotient.abs().clamp_min(2.0 ** -30) / U
    value = torch.round(quotient / step) * step                             # (to even, as the 8-bit values are numbered)
    sure = away > roundings
    assert (sure & (away < roundings + 2)).sum() > 1000                     # (the band that a sloppier product would lose)
    assert torch.equal(q.double()[sure], value[sure])


def test_gated_values_next_to_borders():
    """what the two products of silu(g) u round off counts: for g >= 32 the sigmoid is 1 and the only rounding left is the quotient's, so every value
    further than that from a border gets the byte of the 64-bit quotient"""
    rows = 1 << 11
    u0 = 1 + torch.rand(rows, 1, generator=gen(31))
    s = 32.0 * u0 / 448.0                                                   # (32 u0 is exact, and the largest of its block)
    border = _near_borders(rows * 128, 32).view(rows, 128)
    gate = 32 + 32 * torch.rand(rows, 128, generator=gen(33))
    up = _steps((border * s.double() / gate.double()).float(), 34)
    gate[:, 77], up[:, 77] = 32.0, u0[:, 0]
    q, got = (t.cpu() for t in bitblas.quantize_blocks(up.cuda(), gate=gate.cuda()))
    assert torch.equal(got, s)
    _check_borders(q, s, gate.double() * up.double(), 1.1)


def test_norm_values_next_to_borders():
    """the same of h r w: every h is 1.5 or -1.5 and eps 0, so the mean of squares and its root are exact and r = 2 / 3 is one rounding off; the
    quotient's is the second"""
    D = 1 << 14
    sign = torch.where(torch.rand(D, generator=gen(41)) < 0.5, -1.0, 1.0)
    w0 = 1 + torch.rand(D // 128, 1, generator=gen(42))
    s = (w0.double() / 448.0).float()
    w = _steps((_near_borders(D, 43).view(-1, 128) * s.double()).float(), 44)
    w[:, 5] = w0[:, 0]
    quotients, scales, values = [], [], []
    for i in range(16):
        wt = torch.roll(w.view(-1), 128 * i) * 2.0 ** (i - 8)
        y, got = bitblas.residual_norm((1.5 * sign).half().cuda()[None], None, wt.cuda(), 0.0, quantize="e4m3_float8")[1]
        quotients.append((sign * wt).double())
        scales.append(got.cpu().view(-1))
        values.append(y.cpu().view(-1))
    quotients, scales, values = torch.cat(quotients), torch.cat(scales), torch.cat(values)
    scales = scales.repeat_interleave(128)
    top = quotients.view(-1, 128).abs().amax(1).repeat_interleave(128)
    assert bool(((scales.double() * 448.0 - top).abs() <= top * 4.1 * U).all())    # (r, two products, the division)
    _check_borders(values, scales, quotients, 2.1)


def test_calls_that_autograd_would_record():
    """a weight that asks for gradients, and inputs with forward-mode tangents, are refused; without either the same call runs"""
    x = torch.randn(4, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    w = torch.ones(128, device="cuda").half()
    q, s = bitblas.quantize_blocks(x)
    W, sw = bitblas.quantize_blocks(x, tile=True)
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=4, K=128))
    want = op(q, W, s, sw)
    learnt = W.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        op(q, learnt, s, sw)
    with torch.no_grad():
        assert torch.equal(op(q, learnt, s, sw), want)
    ad = torch.autograd.forward_ad
    with ad.dual_level(), torch.no_grad():
        dual, scale, weight = ad.make_dual(x, torch.ones_like(x)), ad.make_dual(s, torch.ones_like(s)), ad.make_dual(w, w)
        for call in (lambda: bitblas.quantize_blocks(dual), lambda: bitblas.quantize_blocks(x, gate=dual), lambda: bitblas.residual_norm(x, dual, w),
                     lambda: bitblas.residual_norm(x, None, weight), lambda: op(q, W, scale, sw)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(op(q, W, s, sw), want)


def test_a_bias_of_another_shape_leaves_the_layer_as_it_was():
    """one value is no bias of 300 (a copy would spread it), and the weights of a refused call are not taken either"""
    lin = torch.nn.Linear(128, 300, device="cuda", dtype=torch.float16)
    layer = bitblas.BlockScaledLinear.from_linear(lin)
    held = {k: v.clone() for k, v in layer.state_dict().items()}
    for bias in (torch.ones(1), torch.ones(299), torch.ones(1, 300), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="bias"):
            layer.load_float_weight(torch.zeros(300, 128), bias)
    for name, value in layer.state_dict().items():
        assert torch.equal(value.view(torch.uint8), held[name].view(torch.uint8))
