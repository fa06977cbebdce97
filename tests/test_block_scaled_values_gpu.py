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
