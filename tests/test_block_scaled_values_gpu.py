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
