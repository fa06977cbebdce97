"""Block-scaled 8-bit path on the device, against plain forms in 64 bits.

Tolerances, from the arithmetic:
  product   a product of two 8-bit values is exact in float32.  The matrix unit adds 8 consecutive k with each product cut off at 2^-13 of
            the largest one's power of two: 7 products lose less than 2^-13 of the largest, G = sum over the groups of 8 of their
            largest |sa sw a w|, so 7 2^-13 G.  The sums of the groups and blocks are float32: 16 + KB + (slices) roundings, two for the
            scales and one for the bias, (KB + 40) 2^-23 S, S = sum |sa sw a w| + |bias|.  Then |C| eps/2.
            In the 2-norm: a cut is uniform below its bound and its sign is the product's, so the 7 of a group add up to a root mean
            square of sqrt(7 / 3) 2^-13 of the largest; twice that, and the rounding, are allowed.
  quantise  the scale is one float32 division and the value one float32 quotient rounded to 8 bits: equal bit for bit.  With a gate
            the input of both is off by the exponential, the reciprocal and two products: 8 roundings of 2^-24.
  norm      h: 8 roundings of the terms' magnitudes, then eps/2.  y: the mean of squares is a sum with at most 32 + 6 + 16 roundings in
            a chain (half of them count, under the root), the root, two products: 64 2^-24, and r w times h's error."""
import pytest
import torch

import bitblas_amd as bitblas

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
T8 = {"e4m3_float8": torch.float8_e4m3fn, "e5m2_float8": torch.float8_e5m2}
LARGEST = {"e4m3_float8": 448.0, "e5m2_float8": 57344.0}
HALF_STEP = {"e4m3_float8": (2.0 ** -4, 2.0 ** -10), "e5m2_float8": (2.0 ** -3, 2.0 ** -17)}     # relative, and next to zero
TO = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def plain_quantise(x, dtype, tile=False):
    """bytes and scales by the definition, float32 divisions, on the host"""
    x = x.detach().cpu().float()
    K = x.shape[-1]
    f = x.reshape(-1, K)
    kb, rows = -(-K // 128), 128 if tile else 1
    mb = -(-f.shape[0] // rows)
    p = torch.nn.functional.pad(f, (0, kb * 128 - K, 0, mb * rows - f.shape[0])).view(mb, rows, kb, 128)
    s = p.abs().amax((1, 3)).clamp_min(2.0 ** -40) / LARGEST[dtype]
    # (a scale that is not finite: every value of its block is NaN)
    q = torch.where(s.isfinite()[:, None, :, None], p / s[:, None, :, None], float("nan")).to(T8[dtype]).view(mb * rows, kb * 128)[:f.shape[0], :K].contiguous()
    return q.view(x.shape), s if tile else s.view(x.shape[:-1] + (kb,))


def operands(M, N, K, a="e4m3_float8", w="e4m3_float8", seed=0):
    g = gen(seed)
    A, sa = plain_quantise(torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g)), a)
    W, sw = plain_quantise(torch.randn(N, K, generator=g) * 0.05, w, tile=True)
    return A, W, sa, sw


def product64(A, W, sa, sw, bias=None):
    """(C, S) in 64 bits on the device"""
    K, N = A.shape[-1], W.shape[0]
    a = A.cuda().double() * sa.cuda().double().repeat_interleave(128, -1)[..., :K]
    w = W.cuda().double() * sw.cuda().double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    b = bias.cuda().double() if bias is not None else torch.zeros(N, dtype=torch.float64, device="cuda")
    return a @ w.t() + b, a.abs() @ w.abs().t() + b.abs()


def groups(A, W, sa, sw):
    """(sum, root of the sum of squares) over the groups of 8 k of their largest |sa sw a w|, (M, N)"""
    K, N = A.shape[-1], W.shape[0]
    a = (A.cuda().float() * sa.cuda().repeat_interleave(128, -1)[..., :K]).abs().view(-1, K // 8, 8)
    w = (W.cuda().float() * sw.cuda().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).abs().view(N, K // 8, 8)
    total, square = (torch.zeros(a.shape[0], N, dtype=torch.float64, device="cuda") for _ in range(2))
    for j in range(K // 8):
        top = a[:, j, 0, None] * w[None, :, j, 0]
        for i in range(1, 8):
            top = torch.maximum(top, a[:, j, i, None] * w[None, :, j, i])
        total += top.double()
        square += top.double().square()
    return total, square.sqrt()


def check_product(C, A, W, sa, sw, bias=None):
    want, size = product64(A, W, sa, sw, bias)
    top, root = groups(A, W, sa, sw)
    eps, tiny = torch.finfo(C.dtype).eps, torch.finfo(C.dtype).smallest_normal
    tol = 7 * 2.0 ** -13 * top + (-(-A.shape[-1] // 128) + 40) * 2.0 ** -23 * size + want.abs() * (eps / 2) + tiny * eps
    off = (C.double() - want).abs()
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.3f} of the tolerance"
    allowed = 2 * (7 / 3) ** 0.5 * 2.0 ** -13 * root.norm() + want.norm() * (eps / 2) + tiny * eps * C.numel() ** 0.5 + 2.0 ** -20 * size.norm()
    assert off.norm() <= allowed, f"{(off.norm() / allowed).item():.3f} of what the 2-norm allows"


def run_product(M, N, K, a="e4m3_float8", w="e4m3_float8", out="bfloat16", bias=False, seed=0):
    A, W, sa, sw = operands(M, N, K, a, w, seed)
    b = torch.randn(N, generator=gen(seed + 1)).to(TO[out]) if bias else None
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=K, A_dtype=a, W_dtype=w, out_dtype=out, with_bias=bias))
    C = op(A.cuda(), W.cuda(), sa.cuda(), sw.cuda(), b.cuda() if bias else None)
    assert C.shape == (M, N) and C.dtype == TO[out]
    check_product(C, A, W, sa, sw, b)


SHAPES = [(1, 1, 16), (1, 16, 128), (1, 129, 144), (2, 300, 1040), (3, 64, 2048), (7, 1000, 4112), (16, 48, 2064), (16, 1024, 8192), (17, 130, 400),
          (31, 4, 256), (33, 257, 272), (48, 640, 4096), (64, 128, 128), (65, 384, 1024), (100, 1001, 656), (128, 2048, 2048), (130, 256, 6144),
          (9, 7300, 784), (12, 10300, 656), (20, 10250, 1040), (30, 7170, 400), (60, 300, 4112), (64, 6100, 528), (50, 6200, 400),
          (200, 4099, 2064), (256, 512, 384), (300, 130, 4112), (513, 770, 1152), (1000, 1536, 512), (1025, 2050, 1168), (2050, 5000, 272), (3001, 3500, 256), (700, 6000, 272), (513, 9000, 384),
          (200, 13000, 272), (129, 12800, 384), (129, 12700, 128), (300, 4500, 1040), (190, 8000, 128), (250, 4300, 2064), (256, 4224, 2048),
          (40, 700, 6400), (33, 5000, 4112), (65, 2000, 7184), (100, 5000, 1040), (64, 300, 128), (320, 7600, 256)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product(shape):
    run_product(*shape, seed=sum(shape))


@pytest.mark.parametrize("a", list(T8))
@pytest.mark.parametrize("w", list(T8))
@pytest.mark.parametrize("out", ["float16", "bfloat16"])
@pytest.mark.parametrize("M", [4, 40, 120, 520])
def test_product_types(a, w, out, M):
    run_product(M, 272, 656, a, w, out, bias=True, seed=M)


@pytest.mark.parametrize("M", [1, 16, 24, 70, 300, 1100])
def test_product_keeps_rows_apart(M):
    """a NaN or an infinity in one row of A, and one in W, reach their own row and column and nothing else"""
    A, W, sa, sw = operands(M, 200, 400, "e5m2_float8", "e4m3_float8", seed=M)
    bad = M // 2
    A.view(torch.uint8)[bad, 390] = 0x7C                                   # +inf in the partial last block
    W.view(torch.uint8)[131, 3] = 0x7F                                     # NaN
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=200, K=400, A_dtype="e5m2_float8", out_dtype="bfloat16"))
    C = op(A.cuda(), W.cuda(), sa.cuda(), sw.cuda())
    assert not C[bad].isfinite().any() and C[:, 131].isnan().all()
    keep_m = torch.arange(M) != bad
    keep_n = torch.arange(200) != 131
    if keep_m.any():
        W.view(torch.uint8)[131, 3] = 0
        clean = op(A[keep_m].cuda(), W.cuda(), sa[keep_m].cuda(), sw.cuda())
        check_product(clean, A[keep_m], W, sa[keep_m], sw)
        keep_n = keep_n.cuda()
        got, want = C[keep_m.cuda()][:, keep_n].float(), clean[:, keep_n].float()
        # (another row count may take another member, whose sums run in another order)
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -7 + 2.0 ** -12 * want.norm() / want.numel() ** 0.5).all())


@pytest.mark.parametrize("M", [3, 50, 260])
def test_product_extreme_scales(M):
    """scales from 2^-100 to 2^60 next to each other; a block whose scale is 0 counts nothing"""
    A, W, sa, sw = operands(M, 160, 640, seed=M)
    g = gen(M + 7)
    sa = sa * torch.exp2(torch.randint(-100, 60, sa.shape, generator=g).float())
    sa[0, 1] = 0.0
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=160, K=640, out_dtype="bfloat16"))
    check_product(op(A.cuda(), W.cuda(), sa.cuda(), sw.cuda()), A, W, sa, sw)


@pytest.mark.parametrize("M", [5, 40, 300])
def test_product_layouts_and_outputs(M):
    """leading dimensions, every layout of the row scales, a caller's output: the same bits"""
    A, W, sa, sw = [t.cuda() for t in operands(M * 2, 144, 528, seed=M)]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=144, K=528, out_dtype="float16"))
    want = op(A, W, sa, sw)
    A3, sa3 = A.view(2, M, 528), sa.view(2, M, 5)
    out = torch.full((2, M, 144), 9.0, dtype=torch.float16, device="cuda")
    assert op(A3, W, sa3, sw, output=out) is out and torch.equal(out.view(2 * M, 144), want)
    side = torch.full((5, 2 * M + 3), float("nan"), device="cuda")
    side[:, :2 * M] = sa.t()
    assert torch.equal(op(A, W, side.t()[:2 * M], sw), want)
    wide = torch.zeros(2 * M, 544, dtype=torch.uint8, device="cuda").view(A.dtype)
    wide.view(torch.uint8)[:, 5:533] = A.view(torch.uint8)
    assert torch.equal(op(wide[:, 5:533], W, sa, sw), want)                 # rows apart, and off the 16-byte boundary
    odd = torch.zeros(2 * M * 528 + 1, dtype=torch.uint8, device="cuda")
    odd[1:] = A.view(torch.uint8).reshape(-1)
    assert torch.equal(op(odd[1:].view(A.dtype).view(2 * M, 528), W, sa, sw), want)
    assert op(A[:0], W, sa[:0], sw).shape == (0, 144)
    one = op(A[0], W, sa[0], sw)                                            # one row without a leading dimension
    assert one.shape == (144,) and torch.equal(one, op(A[:1], W, sa[:1], sw)[0])


@pytest.mark.parametrize("M", [9, 33, 260])
def test_product_writes_its_rows_only(M):
    """the rows around a caller's output stay as they were, and its own are the same whatever they held"""
    A, W, sa, sw = [t.cuda() for t in operands(M, 132, 272, seed=M)]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=132, K=272, out_dtype="bfloat16"))
    want = op(A, W, sa, sw)
    room = torch.full((M + 2, 132), float("nan"), dtype=torch.bfloat16, device="cuda")
    op(A, W, sa, sw, output=room[1:M + 1])
    assert torch.equal(room[1:M + 1], want) and room[0].isnan().all() and room[M + 1].isnan().all()


def test_product_refusals():
    A, W, sa, sw = [t.cuda() for t in operands(4, 128, 256)]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=128, K=256))
    with pytest.raises(ValueError):
        op(A[:, :128], W, sa, sw)
    with pytest.raises(ValueError):
        op(A.to(torch.float8_e5m2), W, sa, sw)
    with pytest.raises(ValueError):
        op(A, W.t(), sa, sw)
    with pytest.raises(ValueError):
        op(A, W, sa[:3], sw)
    with pytest.raises(ValueError):
        op(A, W, sa, sw.half())
    with pytest.raises(ValueError):
        op(A, W, sa, sw, torch.zeros(128, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        op(A, W, sa.cpu(), sw)
    with pytest.raises(ValueError):
        op(A, W, sa, sw, output=torch.empty(4, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="backward"):
        op(A, W, sa.requires_grad_(), sw)


QUANT = [(1, 1), (1, 128), (3, 130), (16, 256), (17, 1000), (5, 1024), (64, 4104), (130, 640), (300, 77), (257, 2048)]


@pytest.mark.parametrize("dtype", list(T8))
@pytest.mark.parametrize("x", list(TO))
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape", QUANT, ids=lambda s: "x".join(map(str, s)))
def test_quantise_is_the_definition_bit_for_bit(shape, tile, x, dtype):
    g = gen(shape[0] * 10007 + shape[1])
    t = (torch.randn(*shape, generator=g) * torch.exp(3 * torch.randn(shape[1], generator=g))).to(TO[x])
    if shape[0] > 2:
        t[1] = 0.0                                                          # a row of nothing
        t[2] *= 2.0 ** -14
    q, s = bitblas.quantize_blocks(t.cuda(), dtype, tile=tile)
    wq, ws = plain_quantise(t, dtype, tile)
    assert torch.equal(s.cpu().nan_to_num(-1, -2), ws.nan_to_num(-1, -2))
    assert torch.equal(q.cpu().float().nan_to_num(-1e6), wq.float().nan_to_num(-1e6)) and q.shape == t.shape


@pytest.mark.parametrize("tile", [False, True])
def test_quantise_values_that_are_not_finite(tile):
    x = torch.randn(130, 300, generator=gen(3)).to(torch.bfloat16)
    x[0, 5], x[1, 200], x[129, 299] = float("inf"), float("nan"), float("-inf")
    q, s = (t.cpu() for t in bitblas.quantize_blocks(x.cuda(), tile=tile))
    bad = torch.zeros(2 if tile else 130, 3, dtype=torch.bool)
    bad[0, 0] = bad[0 if tile else 1, 1] = bad[1 if tile else 129, 2] = True
    assert torch.equal(~s.isfinite(), bad)
    spread = bad.repeat_interleave(128, 1)[:, :300]
    spread = spread.repeat_interleave(128, 0)[:130] if tile else spread
    assert torch.equal(q.float().isnan(), spread)


@pytest.mark.parametrize("x", list(TO))
def test_quantise_extremes(x):
    """the type's largest values, its subnormals, and values under the scale's floor"""
    f = torch.finfo(TO[x])
    rows = torch.randn(6, 256, generator=gen(11))
    rows = rows / rows.abs().amax(-1, keepdim=True)
    t = torch.stack([rows[0] * f.max, rows[1] * f.smallest_normal, rows[2] * f.smallest_normal * f.eps * 16, rows[3] * 2.0 ** -41, rows[4] * 2.0 ** -20, rows[5]]).to(TO[x])
    for dtype in T8:
        q, s = bitblas.quantize_blocks(t.cuda(), dtype)
        wq, ws = plain_quantise(t, dtype)
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu().float(), wq.float())


def check_values(q, s, want, dtype, slack):
    """8-bit values and scales of `want` (64 bits), whose inputs may be off by `slack` of a value"""
    kb = s.shape[-1]
    K = want.shape[-1]
    pad = torch.nn.functional.pad(want, (0, kb * 128 - K)).view(want.shape[:-1] + (kb, 128))
    top = pad.abs().amax(-1).clamp_min(2.0 ** -40) / LARGEST[dtype]
    extra = torch.nn.functional.pad(slack, (0, kb * 128 - K)).view(pad.shape).amax(-1) / LARGEST[dtype]
    assert bool(((s.double() - top).abs() <= top * 2 * U + extra).all())
    wide = s.double().repeat_interleave(128, -1)[..., :K]
    rel, near = HALF_STEP[dtype]
    off = (q.double() * wide - want).abs()
    tol = torch.maximum(want.abs() * rel, wide * near) * (1 + 2.0 ** -20) + slack * 1.2
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.3f} of the tolerance"


@pytest.mark.parametrize("dtype", list(T8))
@pytest.mark.parametrize("x", list(TO))
@pytest.mark.parametrize("shape", [(1, 128), (3, 200), (16, 1024), (33, 1111), (70, 2816)], ids=lambda s: "x".join(map(str, s)))
def test_quantise_gated(shape, x, dtype):
    both = (torch.randn(shape[0], 2 * shape[1], generator=gen(sum(shape))) * 3).to(TO[x]).cuda()
    gate, up = both[:, :shape[1]], both[:, shape[1]:]
    q, s = bitblas.quantize_blocks(up, dtype, gate=gate)
    want = gate.double() * torch.sigmoid(gate.double()) * up.double()
    # exp(-g) is off by its argument's rounding times |g| too
    check_values(q, s, want, dtype, want.abs() * (8 + 2 * gate.double().abs()) * U)


def test_quantise_gate_extremes():
    """gates whose exponential leaves float32: silu goes to the gate itself, or to zero"""
    gate = torch.tensor([-1e4, -200.0, -89.0, 0.0, 89.0, 200.0, 1e4, 65504.0]).repeat(16).view(1, 128).to(torch.float16).cuda()
    up = torch.ones_like(gate)
    q, s = bitblas.quantize_blocks(up, gate=gate)
    assert q.float().isfinite().all() and s.isfinite().all()
    want = torch.nn.functional.silu(gate.double())
    check_values(q, s, want, "e4m3_float8", want.abs() * 8 * U + 2.0 ** -60)


def test_quantise_layouts():
    x = torch.randn(6, 4, 520, generator=gen(5)).to(torch.bfloat16).cuda()
    q, s = bitblas.quantize_blocks(x)
    f, fs = bitblas.quantize_blocks(x.view(24, 520))
    assert s.shape == (6, 4, 5) and torch.equal(q.view(24, 520).float(), f.float()) and torch.equal(s.reshape(24, 5), fs)
    for view in (x[:, 1], x[1:5, :, :300], x[:, ::2], x[..., 1:130], x.transpose(0, 1), x[0, 0]):
        a, b = bitblas.quantize_blocks(view), bitblas.quantize_blocks(view.contiguous())
        assert torch.equal(a[0].float(), b[0].float()) and torch.equal(a[1], b[1])
    kept = bitblas.quantize_blocks(x * 2)
    again = bitblas.quantize_blocks(x, output=kept)
    assert again[0] is kept[0] and torch.equal(kept[0].float(), q.float()) and torch.equal(kept[1], s)
    assert bitblas.quantize_blocks(x[:0])[1].shape == (0, 4, 5)
    wt, ws = bitblas.quantize_blocks(x.view(24, 520), tile=True)
    assert ws.shape == (1, 5)


def test_quantise_refusals():
    x = torch.randn(4, 256, device="cuda").half()
    for kw in (dict(dtype="int8"), dict(gate=x[:2]), dict(gate=x.float()), dict(tile=True, gate=x), dict(output=(x, x))):
        with pytest.raises(ValueError):
            bitblas.quantize_blocks(x, **kw)
    with pytest.raises(ValueError):
        bitblas.quantize_blocks(x.to(torch.int8))
    with pytest.raises(ValueError):
        bitblas.quantize_blocks(x.view(2, 2, 256), tile=True)
    with pytest.raises(ValueError):
        q, _ = bitblas.quantize_blocks(x)
        bitblas.quantize_blocks(x, output=(q, torch.empty(4, 2, device="cuda")))     # a row's scales side by side: another layout
    with pytest.raises(RuntimeError, match="backward"):
        bitblas.quantize_blocks(x.requires_grad_())


def norm64(x, residual, weight, eps, post, gate, scale, rscale):
    """(h, y, error allowed of h, error allowed of y) in 64 bits, before any rounding of the outputs"""
    z = x.double()
    if post is not None:
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        z = z * gate.double()
    h = scale * z + (rscale * residual.double() if residual is not None else 0.0)
    dh = (scale * z).abs() * 64 * U + ((rscale * residual.double()).abs() * 4 * U if residual is not None else 0.0)
    if weight is None:
        return h, None, dh, None
    r = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    y = h * r * weight.double()
    # the mean of squares moves by the elements' errors too
    shift = (h.abs() * dh).mean(-1, keepdim=True) * r * r
    return h, y, dh, y.abs() * (64 * U + 2 * shift) + (r * weight.double()).abs() * dh


def check_rounded(got, want, slack):
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) + slack * 1.1 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.3f} of the tolerance"


def run_norm(shape, t="bfloat16", st="bfloat16", wt=None, post=False, gate=None, q=None, scale=1.0, rscale=1.0, residual=True, eps=1e-5, seed=0):
    g = gen(seed)
    D = shape[-1]
    x = (torch.randn(*shape, generator=g) * 2).to(TO[t]).cuda()
    res = (torch.randn(*shape, generator=g) * 5).to(TO[st]).cuda() if residual else None
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(TO[wt or t]).cuda()
    p = (1 + 0.2 * torch.randn(D, generator=g)).to(TO[wt or t]).cuda() if post else None
    gt = torch.randn(*gate, generator=g).to(TO[t]).cuda() if gate is not None else None
    h, y = bitblas.residual_norm(x, res, w, eps, post_weight=p, gate=gt, scale=scale, residual_scale=rscale, quantize=q)
    wh, wy, dh, dy = norm64(x, res, w, eps, p, gt, scale, rscale)
    assert h.dtype == (TO[st] if residual else TO[t])
    check_rounded(h, wh, dh)
    if q is None:
        assert y.dtype == TO[t]
        check_rounded(y, wy, dy)
    else:
        check_values(y[0], y[1], wy, q, dy)


@pytest.mark.parametrize("D", [1, 7, 64, 100, 128, 200, 512, 1000, 1024, 2056, 4096, 5120, 8192, 9000, 16384, 20000, 32767, 32768])
@pytest.mark.parametrize("q", [None, "e4m3_float8"])
def test_norm_widths(D, q):
    run_norm((3, D), q=q, seed=D)


@pytest.mark.parametrize("t", ["float16", "bfloat16"])
@pytest.mark.parametrize("st", ["same", "float32"])
@pytest.mark.parametrize("wt", ["same", "float32"])
@pytest.mark.parametrize("q", [None, "e4m3_float8", "e5m2_float8"])
def test_norm_types(t, st, wt, q):
    run_norm((5, 3, 640), t, t if st == "same" else st, t if wt == "same" else wt, post=True, gate=(5, 1, 640), q=q, scale=0.5, rscale=0.75, seed=3)


@pytest.mark.parametrize("gate", [(328,), (4, 1, 328), (1, 3, 328), (4, 3, 328), (4, 3, 1), (1,)])
@pytest.mark.parametrize("post", [False, True])
def test_norm_gates(gate, post):
    run_norm((4, 3, 328), post=post, gate=gate, scale=0.25, seed=len(gate))


@pytest.mark.parametrize("rows", [1, 2, 17, 1000])
def test_norm_rows(rows):
    run_norm((rows, 272), "float16", "float16", q="e4m3_float8", seed=rows)


def test_norm_alone_returns_its_input():
    x = torch.randn(4, 300, generator=gen(1)).half().cuda()
    w = torch.ones(300).half().cuda()
    h, y = bitblas.residual_norm(x, None, w, 1e-6)
    assert h is x
    _, wy, _, dy = norm64(x, None, w, 1e-6, None, None, 1.0, 1.0)
    check_rounded(y, wy, dy)
    run_norm((4, 300), residual=False, post=True, seed=2)
    h, y = bitblas.residual_norm(x, x, None, post_weight=w)                 # no second norm
    assert y is None
    wh, _, dh, _ = norm64(x, x, None, 1e-6, w, None, 1.0, 1.0)
    check_rounded(h, wh, dh)


def test_norm_rows_of_zeros_and_extremes():
    """a row of zeros gives zeros whatever eps > 0; large values stay finite where the mean of squares does; NaN stays in its row"""
    x = torch.randn(6, 256, generator=gen(4)).to(torch.bfloat16)
    x[1] = 0
    x[2] *= 2.0 ** 60
    x[3] *= 2.0 ** -60
    x[4, 7] = float("nan")
    res = torch.zeros_like(x)
    w = torch.ones(256).to(torch.bfloat16)
    h, y = bitblas.residual_norm(x.cuda(), res.cuda(), w.cuda(), 1e-6)
    h, y = h.cpu(), y.cpu()
    assert (y[1] == 0).all() and y[4].isnan().all() and h[4].isnan().sum() == 1
    keep = [0, 1, 2, 3, 5]
    wh, wy, dh, dy = norm64(x[keep], res[keep], w, 1e-6, None, None, 1.0, 1.0)
    check_rounded(y[keep], wy, dy)
    q, s = bitblas.residual_norm(x.cuda(), res.cuda(), w.cuda(), 1e-6, quantize="e4m3_float8")[1]
    assert q[4].float().isnan().all() and q[keep].float().isfinite().all() and (q[1].float() == 0).all()


def test_norm_layouts_and_outputs():
    """rows apart, outputs of the caller, the stream updated in place: the same bits"""
    g = gen(9)
    x = torch.randn(3, 5, 392, generator=g).half().cuda()
    res = torch.randn(3, 5, 392, generator=g).cuda()
    w = torch.randn(392, generator=g).half().cuda()
    h, y = bitblas.residual_norm(x, res, w, 1e-5)
    wide = torch.zeros(3, 5, 800, device="cuda").half()
    wide[..., 8:400] = x
    a = bitblas.residual_norm(wide[..., 8:400], res, w, 1e-5)
    odd = torch.zeros(3, 5, 801, device="cuda").half()
    odd[..., 3:395] = x
    b = bitblas.residual_norm(odd[..., 3:395], res.transpose(0, 1).contiguous().transpose(0, 1), w, 1e-5)
    for got in (a, b):
        assert torch.equal(got[0], h) and torch.equal(got[1], y)
    stream, out = res.clone(), torch.empty_like(y)
    c = bitblas.residual_norm(x, stream, w, 1e-5, output=(stream, out))
    assert c[0] is stream and c[1] is out and torch.equal(stream, h) and torch.equal(out, y)
    q, s = bitblas.residual_norm(x, res, w, 1e-5, quantize="e4m3_float8")[1]
    h2, kept = bitblas.residual_norm(x * 2, res, w, 1e-5, quantize="e4m3_float8")
    again = bitblas.residual_norm(x, res, w, 1e-5, quantize="e4m3_float8", output=(h2,) + kept)
    assert again[0] is h2 and torch.equal(kept[0].float(), q.float()) and torch.equal(kept[1], s) and torch.equal(h2, h)
    assert bitblas.residual_norm(x[:0], res[:0], w)[1].shape == (0, 5, 392)


def test_norm_refusals():
    x = torch.randn(4, 256, device="cuda").half()
    w = torch.ones(256, device="cuda").half()
    for args, kw in (((x,), {}), ((x.float(), None, w), {}), ((x, x[:2], w), {}), ((x, x.bfloat16(), w), {}), ((x, x, w[:128]), {}),
                     ((x, x, w.bfloat16()), {}), ((x, x, w), dict(post_weight=w.float())), ((x, x, w), dict(gate=x.float())),
                     ((x, x, w), dict(gate=x[:3])), ((x, x, None), dict(quantize="e4m3_float8")), ((x, x, w), dict(quantize="int8")),
                     ((x, x, w, -1.0), {}), ((x, x.cpu(), w), {}), ((x, x, w), dict(output=(x.t(),))),
                     ((torch.zeros(1, 32776, device="cuda").half(), None, torch.ones(32776, device="cuda").half()), {})):
        with pytest.raises(ValueError):
            bitblas.residual_norm(*args, **kw)
    with pytest.raises(RuntimeError, match="backward"):
        bitblas.residual_norm(x, x, w.requires_grad_())
    with torch.no_grad():
        bitblas.residual_norm(x, x, w.requires_grad_())


def layer(x, attn, params):
    """norm -> gate and up in one product -> silu(gate) * up -> down -> norm, the way a decoder layer runs it"""
    p = params
    h, (q, s) = bitblas.residual_norm(attn, x, p["ln1"], 1e-5, quantize="e4m3_float8")
    both = p["gate_up"](q, p["wgu"], s, p["sgu"])
    inter = both.shape[-1] // 2
    q2, s2 = bitblas.quantize_blocks(both[..., inter:], gate=both[..., :inter])
    down = p["down"](q2, p["wd"], s2, p["sd"])
    return bitblas.residual_norm(down, h, p["ln2"], 1e-5)


def make_layer(D, inter, seed):
    g = gen(seed)
    p = {"ln1": torch.ones(D).bfloat16().cuda(), "ln2": torch.ones(D).bfloat16().cuda()}
    w1, w2 = torch.randn(2 * inter, D, generator=g) * D ** -0.5, torch.randn(D, inter, generator=g) * inter ** -0.5
    p["wgu"], p["sgu"] = bitblas.quantize_blocks(w1.cuda(), tile=True)
    p["wd"], p["sd"] = bitblas.quantize_blocks(w2.cuda(), tile=True)
    p["gate_up"] = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=2 * inter, K=D, out_dtype="bfloat16"))
    p["down"] = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=D, K=inter, out_dtype="bfloat16"))
    return p


@pytest.mark.parametrize("rows", [1, 13, 70, 300])
def test_a_layer_of_them(rows):
    """the operators as they run together, against the layer in 64 bits on the dequantised weights: two quantisations of relative
    error 2^-4 an element, independent, sum to about 2^-4 / sqrt(3) of the branch in the 2-norm each; twice that is allowed"""
    D, inter = 640, 1408
    p = make_layer(D, inter, 1)
    g = gen(rows)
    x, attn = (torch.randn(rows, D, generator=g).bfloat16().cuda() for _ in range(2))
    h, y = layer(x, attn, p)
    up = lambda w, s: w.double() * s.double().repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]  # noqa: E731
    h0 = x.double() + attn.double()
    n0 = h0 / torch.sqrt(h0.square().mean(-1, keepdim=True) + 1e-5)
    both = n0 @ up(p["wgu"], p["sgu"]).t()
    act = torch.nn.functional.silu(both[:, :inter]) * both[:, inter:]
    branch = act @ up(p["wd"], p["sd"]).t()
    off = (h.double() - (h0 + branch)).norm() / branch.norm()
    assert off < 2 * 2 * 2.0 ** -4 / 3 ** 0.5, off.item()


def float_tail(seed, D=512, inner=768, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    mk = lambda i, o, b=False: torch.nn.Linear(i, o, bias=b, device="cuda", dtype=dtype)  # noqa: E731
    return mk(D, D, True), mk(D, inner), mk(D, inner), mk(inner, D)


@pytest.mark.parametrize("rows", [(1,), (2, 17), (300,)])
@pytest.mark.parametrize("posts", [False, True])
def test_decoder_tail(rows, posts):
    """the modules run the operators they are made of, bit for bit, and stay near the float layers: three quantised products of relative
    error 2^-4 sqrt(2 / 3) (both operands rounded, uniformly) add up in the branches; twice their root sum of squares is allowed"""
    D, inner = 512, 768
    o, gate, up, down = float_tail(1)
    with torch.no_grad():
        mlp = bitblas.BlockScaledGatedMLP.from_linears(gate, up, down)
        o8 = bitblas.BlockScaledLinear.from_linear(o)
        g = gen(len(rows))
        w, w2, p1, p2 = ((1 + 0.1 * torch.randn(D, generator=g)).bfloat16().cuda() for _ in range(4))
        tail = bitblas.BlockScaledDecoderTail(o8, mlp, w, 1e-5, p1 if posts else None, p2 if posts else None)
        attn, x = (torch.randn(*rows, D, generator=g).bfloat16().cuda() for _ in range(2))
        out, (q, s) = tail(attn, x, next_norm=w2)
        # by hand
        y = o8.bitblas_matmul(*(lambda a: (a[0], o8.weight, a[1], o8.weight_scale))(bitblas.quantize_blocks(attn)), o8.bias)
        h, y = bitblas.residual_norm(y, x, w, 1e-5, post_weight=p1 if posts else None, quantize="e4m3_float8")
        both = mlp.gate_up.bitblas_matmul(y[0], mlp.gate_up.weight, y[1], mlp.gate_up.weight_scale)
        a = bitblas.quantize_blocks(both[..., inner:], gate=both[..., :inner])
        d = mlp.down.bitblas_matmul(a[0], mlp.down.weight, a[1], mlp.down.weight_scale)
        want, y2 = bitblas.residual_norm(d, h, w2, 1e-5, post_weight=p2 if posts else None, quantize="e4m3_float8")
        assert torch.equal(out, want) and torch.equal(q.float(), y2[0].float()) and torch.equal(s, y2[1])
        plain, none = tail(attn, x)
        assert none is None and torch.equal(plain, out)
        # the MLP alone, its norm and its residual
        full = mlp(h, residual=h, norm=(w, 1e-5))
        y3 = bitblas.residual_norm(h, None, w, 1e-5, quantize="e4m3_float8")[1]
        assert torch.equal(full, bitblas.residual_norm(mlp(y3), h)[0])
        # the float layers in 64 bits
        rms = lambda t, wt: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * wt.double()  # noqa: E731
        W = lambda l: l.weight.double().t()  # noqa: E731
        b1 = attn.double() @ W(o) + o.bias.double()
        h64 = x.double() + (rms(b1, p1) if posts else b1)
        n64 = rms(h64, w)
        act = torch.nn.functional.silu(n64 @ W(gate)) * (n64 @ W(up))
        b2 = act @ W(down)
        b2 = rms(b2, p2) if posts else b2
        allowed = 2 * 3 ** 0.5 * 2.0 ** -4 * (2 / 3) ** 0.5 * (h64 - x.double()).norm().hypot(b2.norm())
        assert (out.double() - (h64 + b2)).norm() <= allowed


def test_linear_layer():
    torch.manual_seed(3)
    lin = torch.nn.Linear(400, 300, device="cuda", dtype=torch.float16)
    layer = bitblas.BlockScaledLinear.from_linear(lin)
    assert layer.out_dtype == "float16"
    x = torch.randn(3, 7, 400, device="cuda").half()
    wq, ws = plain_quantise(lin.weight, "e4m3_float8", tile=True)
    assert torch.equal(layer.weight.cpu().float(), wq.float()) and torch.equal(layer.weight_scale.cpu(), ws)
    C = layer(x)
    q, s = plain_quantise(x, "e4m3_float8")
    assert C.shape == (3, 7, 300)
    check_product(C.view(21, 300), q.view(21, 400), wq, s.reshape(21, 4), ws, lin.bias.detach())
    assert torch.equal(layer(bitblas.quantize_blocks(x)), C)
    out = torch.empty_like(C)
    assert layer(x, output=out) is out and torch.equal(out, C)
    with pytest.raises(ValueError):
        layer.load_float_weight(torch.zeros(300, 300, device="cuda"), lin.bias)
    with pytest.raises(ValueError):
        layer.load_float_weight(lin.weight)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_captured_and_replayed(rows):
    """a captured layer replayed on new inputs, with eager work between the replays, and a second graph beside it: the eager bits"""
    p = make_layer(512, 768, 2)
    xs = [torch.randn(rows, 512, generator=gen(s)).bfloat16().cuda() for s in range(4)]
    x, attn = xs[0].clone(), xs[1].clone()
    layer(x, attn, p)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(x, attn, p)
        graphs.append((g, out))
    for i in range(4):
        a, b = xs[i % 4], xs[(i + 1) % 4]
        want = layer(a, b, p)
        x.copy_(a)
        attn.copy_(b)
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_other_streams():
    """two streams at once, each with its own partial sums"""
    p = make_layer(512, 768, 3)
    xs = [torch.randn(40, 512, generator=gen(s)).bfloat16().cuda() for s in range(2)]
    want = [layer(x, x, p) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(layer(xs[i], xs[i], p))
    torch.cuda.synchronize()
    for i in range(2):
        for h, y in got[i]:
            assert torch.equal(h, want[i][0]) and torch.equal(y, want[i][1])


@pytest.mark.parametrize("M", [1, 16, 30, 200, 600])
def test_product_repeats_bit_for_bit(M):
    A, W, sa, sw = [t.cuda() for t in operands(M, 656, 4112, seed=M)]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=656, K=4112, out_dtype="bfloat16"))
    first = op(A, W, sa, sw)
    for _ in range(5):
        assert torch.equal(op(A, W, sa, sw), first)


def _inside(room, at, shape):
    """a contiguous view into `room`, and what lies around it"""
    n = 1
    for size in shape:
        n *= size
    return room[at:at + n].view(shape), torch.cat([room[:at], room[at + n:]])


@pytest.mark.parametrize("M, N, K", [(5, 131, 272), (40, 1001, 272), (70, 6101, 144), (70, 301, 7184), (260, 9001, 144), (600, 6301, 144), (1281, 8713, 144)])
def test_product_odd_columns(M, N, K):
    """N odd, so every row starts on another boundary, and an output that starts off any: right, and nothing written beside it"""
    A, W, sa, sw = operands(M, N, K, seed=N)
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=K, out_dtype="bfloat16"))
    dev = [t.cuda() for t in (A, W, sa, sw)]
    room = torch.full((M * N + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    out, around = _inside(room, 17, (M, N))
    op(*dev, output=out)
    out, around = _inside(room, 17, (M, N))
    assert bool((around == 7.0).all())
    assert torch.equal(out, op(*dev))
    check_product(out, A, W, sa, sw)


@pytest.mark.parametrize("K", [1, 9, 127, 1041, 4095, 8193])
@pytest.mark.parametrize("x", list(TO))
def test_odd_rows_beside_others(K, x):
    """quantiser and norm over rows of an odd width, inputs and outputs on odd boundaries: the same bits as anywhere, nothing beside them"""
    m, q8 = 37, "e4m3_float8"
    wide = torch.randn(m * K + 64, generator=gen(K)).to(TO[x]).cuda()
    src, gate = wide[5:5 + m * K].view(m, K), wide[3:3 + m * K].view(m, K)
    for kw in (dict(), dict(tile=True), dict(gate=gate)):
        want = bitblas.quantize_blocks(src.clone(), q8, **{k: v.clone() if k == "gate" else v for k, v in kw.items()})
        room = torch.full((m * K + 64,), 1.0, device="cuda").to(torch.float8_e4m3fn)
        out, _ = _inside(room, 9, (m, K))
        q, s = bitblas.quantize_blocks(src, q8, output=(out, torch.empty_like(want[1])), **kw)
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
        assert bool((_inside(room, 9, (m, K))[1].float() == 1.0).all())
    if x == "float32":
        return
    w = torch.randn(K + 1, generator=gen(K + 1)).to(TO[x]).cuda()
    for st in (TO[x], torch.float32):
        res = torch.randn(m * K + 8, generator=gen(K + 2)).to(st).cuda()[3:3 + m * K].view(m, K)
        want = bitblas.residual_norm(src.clone(), res.clone(), w[1:].clone(), 1e-5, gate=gate.clone())
        h_room, y_room = torch.full((m * K + 64,), 7.0, dtype=st, device="cuda"), torch.full((m * K + 64,), 7.0, dtype=TO[x], device="cuda")
        bitblas.residual_norm(src, res, w[1:], 1e-5, gate=gate, output=(_inside(h_room, 11, (m, K))[0], _inside(y_room, 13, (m, K))[0]))
        for room, at, have in ((h_room, 11, want[0]), (y_room, 13, want[1])):
            out, around = _inside(room, at, (m, K))
            assert torch.equal(out, have) and bool((around == 7.0).all())


def test_outputs_that_autograd_tracks():
    A, W, sa, sw = [t.cuda() for t in operands(4, 32, 128)]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=32, K=128))
    with pytest.raises(RuntimeError, match="no backward"):
        op(A, W, sa, sw, output=torch.zeros(4, 32, dtype=torch.float16, device="cuda", requires_grad=True))
    x = torch.zeros(4, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="no backward"):
        bitblas.residual_norm(x, x, output=(torch.zeros_like(x, requires_grad=True),))


@pytest.mark.parametrize("M, N, K", [(257, 32900, 4112), (4300, 4001, 4096), (70, 32851, 4112)])
def test_product_last_round_in_slices(M, N, K):
    """whole tiles, and behind them some in K slices: right, the same every time, and nothing written beside the output"""
    A, W, sa, sw = operands(M, N, K, seed=N)
    bias = torch.randn(N, generator=gen(N)).bfloat16()
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=K, out_dtype="bfloat16", with_bias=True))
    plan = op.plan(M)
    tiles = -(-M // plan["block_m"]) * -(-N // plan["block_n"])
    assert plan["split_k"] > 1 and tiles < plan["grid"] < tiles * plan["split_k"]
    dev = [t.cuda() for t in (A, W, sa, sw, bias)]
    room = torch.full((M + 2, N), 7.0, dtype=torch.bfloat16, device="cuda")
    first = op(*dev, output=room[1:M + 1])
    assert bool((room[0] == 7.0).all()) and bool((room[M + 1] == 7.0).all())
    check_product(first, A, W, sa, sw, bias)
    for _ in range(3):
        assert torch.equal(op(*dev), first)


def test_offsets_beyond_32_bits():
    """operands, outputs and streams of more than 2^32 bytes: their last rows come out as they do alone"""
    m, K, tail = 524288 + 300, 8208, 300
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, K, generator=g, device="cuda", dtype=torch.bfloat16)
    last = x[-tail:].clone()
    q, s = bitblas.quantize_blocks(x)
    ql, sl = bitblas.quantize_blocks(last)
    assert torch.equal(q[-tail:].view(torch.uint8), ql.view(torch.uint8)) and torch.equal(s[-tail:], sl)
    w = torch.randn(K, generator=g, device="cuda", dtype=torch.bfloat16)
    h, y = bitblas.residual_norm(x, x, w, 1e-5)
    hl, yl = bitblas.residual_norm(last, last, w, 1e-5)
    assert torch.equal(h[-tail:], hl) and torch.equal(y[-tail:], yl)
    del h, y
    W, sw = bitblas.quantize_blocks(x[:256], tile=True)
    C = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=256, K=K, out_dtype="bfloat16"))(q, W, s, sw)
    check_product(C[-tail:].clone(), ql, W, sl, sw)
    del q, s, C
    W, sw = bitblas.quantize_blocks(x, tile=True)                         # (a tile boundary in front of the last 300 rows)
    Wl, swl = bitblas.quantize_blocks(last, tile=True)
    assert torch.equal(W[-tail:].view(torch.uint8), Wl.view(torch.uint8)) and torch.equal(sw[-3:], swl)
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=m, K=K, out_dtype="bfloat16"))
    for rows in (1, 40, 200):
        A, sa = bitblas.quantize_blocks(x[:rows])
        check_product(op(A, W, sa, sw)[:, -tail:].clone(), A, Wl, sa, swl)
    A, sa = bitblas.quantize_blocks(x[:8200, :128].contiguous())          # an output of 8.6 GB
    W, sw = bitblas.quantize_blocks(x[:, :128].contiguous(), tile=True)
    C = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=m, K=128, out_dtype="bfloat16"))(A, W, sa, sw)
    check_product(C[-40:, -tail:].clone(), A[-40:], W[-tail:], sa[-40:], sw[-3:])


@pytest.mark.parametrize("M, N, K", [(300, 8190, 28688), (512, 8192, 28672), (20, 20490, 1424), (32, 28673, 2064)])
def test_product_long_k_and_thin_batches(M, N, K):
    """long K, where tiles of 256 rows leave in K slices; up to 32 rows against a W that fills the chip with 64-row tiles"""
    g = torch.Generator(device="cuda").manual_seed(N)
    A, sa = bitblas.quantize_blocks(torch.randn(M, K, generator=g, device="cuda") * torch.exp(torch.randn(K, generator=g, device="cuda")))
    W, sw = bitblas.quantize_blocks(torch.randn(N, K, generator=g, device="cuda") * 0.05, tile=True)
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=K, out_dtype="float16"))
    plan = op.plan(M)
    assert (plan["block_m"], plan["split_k"]) == ((256, 4) if M > 32 else (64, 1))
    first = op(A, W, sa, sw)
    check_product(first, A, W, sa, sw)
    assert torch.equal(op(A, W, sa, sw), first)
