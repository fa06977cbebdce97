"""Block-scaled 8-bit path without a device: configurations, plans, refusals at the Python and the C boundary, row and gate layouts."""
import ctypes

import pytest
import torch

import bitblas_amd as bitblas
from bitblas_amd import block_scaled as bs
from bitblas_amd import lib as wlib


def test_struct_sizes_match_header():
    assert ctypes.sizeof(bs.BlockDesc) == 8 * 4
    assert ctypes.sizeof(bs.BlockQuant) == 4 * 4 + 5 * 8 + 4 * 8
    assert ctypes.sizeof(bs.ResidualNormArgs) == 8 * 4 + 7 * 8 + 8 * 8


@pytest.mark.parametrize("kw", [dict(N=0, K=128), dict(N=128, K=120), dict(N=128), dict(N=128, K=128, A_dtype="float16"),
                                dict(N=128, K=128, W_dtype="int8"), dict(N=128, K=128, out_dtype="float32"), dict(N=128.0, K=128)])
def test_config_refusals(kw):
    with pytest.raises(ValueError):
        bitblas.BlockScaledMatmulConfig(**kw)


def _desc(**kw):
    d = bs.BlockDesc()
    d.struct_size = ctypes.sizeof(bs.BlockDesc)
    d.N, d.K, d.a_dtype, d.w_dtype, d.out_dtype = 256, 256, wlib.E4M3, wlib.E4M3, wlib.F16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, code", [(dict(struct_size=4), wlib.ERR_BAD_DESC), (dict(N=0), wlib.ERR_BAD_DESC), (dict(K=-16), wlib.ERR_BAD_DESC),
                                      (dict(K=24), wlib.ERR_UNSUPPORTED), (dict(a_dtype=wlib.F16), wlib.ERR_UNSUPPORTED),
                                      (dict(w_dtype=wlib.I8), wlib.ERR_UNSUPPORTED), (dict(out_dtype=wlib.F32), wlib.ERR_UNSUPPORTED),
                                      (dict(K=(1 << 22) + 16), wlib.ERR_UNSUPPORTED)])
def test_product_descriptor_refusals(kw, code):
    L = bs._library()
    d = _desc(**kw)
    p = 4096
    assert L.wqaa_block_matmul(ctypes.byref(d), p, p, p, 8, p, None, p, 8, None, 0, None) == code
    assert L.wqaa_block_select(ctypes.byref(d), 8, None) == code
    assert L.wqaa_block_workspace_bytes(ctypes.byref(d), 8) == 0


def test_product_call_refusals():
    L = bs._library()
    p = 4096
    d = _desc()
    ok = [ctypes.byref(d), p, p, p, 8, p, None, p, 8, None, 0, None]
    for i in (1, 2, 3, 5, 7):                                             # a null operand
        assert L.wqaa_block_matmul(*(ok[:i] + [None] + ok[i + 1:])) == wlib.ERR_BAD_DESC
    assert L.wqaa_block_matmul(*(ok[:4] + [7] + ok[5:])) == wlib.ERR_BAD_DESC          # scale rows overlap
    assert L.wqaa_block_matmul(*(ok[:1] + [p + 8] + ok[2:])) == wlib.ERR_BAD_DESC      # A off its alignment
    assert L.wqaa_block_matmul(*(ok[:8] + [-1] + ok[9:])) == wlib.ERR_BAD_DESC
    assert L.wqaa_block_matmul(*(ok[:8] + [0] + ok[9:])) == wlib.OK                    # no rows: nothing to do, no device asked for
    d.with_bias = 1
    assert L.wqaa_block_matmul(*ok) == wlib.ERR_BAD_DESC


def test_plans_cover_every_row_count():
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=4096, K=4096))
    for m in (1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 333, 1024, 4096, 100000):
        plan = op.plan(m)
        assert plan["grid"] > 0 and plan["block_k"] == 128 and plan["name"].startswith("block_matmul")
        assert (op.workspace_bytes(m) > 0) == (plan["split_k"] > 1)


def _quant(**kw):
    q = bs.BlockQuant()
    q.struct_size = ctypes.sizeof(bs.BlockQuant)
    q.x_dtype, q.q_dtype, q.rows, q.K, q.x_ld, q.gate_ld, q.s_ld = wlib.F16, wlib.E4M3, 4, 256, 256, 256, 4
    q.X = q.Q = q.S = 4096
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("kw", [dict(struct_size=8), dict(rows=-1), dict(K=0), dict(X=None), dict(Q=None), dict(S=None), dict(x_ld=255),
                                dict(gate=4096, gate_ld=8), dict(s_ld=3)])
def test_quantizer_refusals(kw):
    assert bs._library().wqaa_block_quantize(ctypes.byref(_quant(**kw)), None) == wlib.ERR_BAD_DESC
    assert bs._library().wqaa_block_quantize(ctypes.byref(_quant(rows=0)), None) == wlib.OK


def _norm(**kw):
    n = bs.ResidualNormArgs()
    n.struct_size = ctypes.sizeof(bs.ResidualNormArgs)
    n.x_dtype, n.stream_dtype, n.weight_dtype, n.q_dtype = wlib.F16, wlib.F16, wlib.F16, -1
    n.rows, n.D, n.x_ld, n.residual_ld, n.gate_rows = 4, 256, 256, 256, 1
    n.x = n.weight = n.Y = 4096
    for k, v in kw.items():
        setattr(n, k, v)
    return n


@pytest.mark.parametrize("kw", [dict(struct_size=8), dict(rows=-1), dict(D=0), dict(x=None), dict(Y=None), dict(weight=None), dict(x_ld=100),
                                dict(residual=4096, residual_ld=0), dict(gate=4096, gate_rows=0), dict(gate=4096, gate_ld=-1),
                                dict(q_dtype=wlib.E4M3), dict(q_dtype=wlib.E4M3, S=4096, s_ld=3)])
def test_norm_refusals(kw):
    assert bs._library().wqaa_residual_norm(ctypes.byref(_norm(**kw)), None) == wlib.ERR_BAD_DESC
    assert bs._library().wqaa_residual_norm(ctypes.byref(_norm(rows=0)), None) == wlib.OK


def test_host_tensors_are_refused():
    x = torch.randn(2, 128, dtype=torch.float16)
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=128, K=128))
    q, s = x.to(torch.float8_e4m3fn), torch.ones(2, 1)
    for call in (lambda: bitblas.quantize_blocks(x), lambda: bitblas.residual_norm(x, x, x[0]), lambda: op(q, q, s, s)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_layers_without_a_device():
    """buffers, their state dict, and what a layer refuses"""
    lin = bitblas.BlockScaledLinear(272, 200, bias=True, out_dtype="bfloat16")
    assert lin.weight.shape == (200, 272) and lin.weight.dtype == torch.float8_e4m3fn
    assert lin.weight_scale.shape == (2, 3) and lin.bias.dtype == torch.bfloat16
    assert set(lin.state_dict()) == {"weight", "weight_scale", "bias"}
    other = bitblas.BlockScaledLinear(272, 200, bias=True, out_dtype="bfloat16")
    other.load_state_dict(lin.state_dict())
    with pytest.raises(RuntimeError, match="GPU"):
        lin.load_float_weight(torch.zeros(200, 272), torch.zeros(200))
    with pytest.raises(ValueError):
        bitblas.BlockScaledLinear(270, 200)
    with pytest.raises(ValueError):
        bitblas.BlockScaledGatedMLP(bitblas.BlockScaledLinear(256, 256), bitblas.BlockScaledLinear(256, 256))
    bitblas.BlockScaledGatedMLP(bitblas.BlockScaledLinear(256, 512), bitblas.BlockScaledLinear(256, 256))


def test_row_layouts():
    t = torch.arange(4 * 6 * 10).view(4, 6, 10)
    for view, ld in ((t, 10), (t[:, :, 2:7], 10), (t[1:3, :, :4], 10), (t.view(24, 10)[::2], 20), (t[0], 10), (t[:, 2], 60)):
        got, d = bs._rows(view)
        assert d == ld and got.data_ptr() == view.data_ptr()
        k = view.shape[-1]
        flat = torch.as_strided(got, (view.numel() // k, k), (d, 1))
        assert torch.equal(flat, view.reshape(-1, k))
    for view in (t[:, ::2], t.transpose(0, 1), t[..., ::2], t[0].t(), t[:1].expand(4, 6, 10)):
        got, d = bs._rows(view)
        k = view.shape[-1]
        assert torch.equal(torch.as_strided(got, (view.numel() // k, k), (d, 1)), view.reshape(-1, k))


@pytest.mark.parametrize("shape", [(7,), (1, 7), (4, 1, 7), (4, 3, 7), (1, 3, 7), (3, 7), (4, 3, 1), (1,), (1, 1, 7), ()])
def test_gate_layouts(shape):
    x = torch.zeros(4, 3, 7)
    gate = torch.arange(float(max(1, torch.Size(shape).numel()))).reshape(shape)
    g, ld, share = bs._gate_rows(gate, x)
    want = gate.expand(4, 3, 7).reshape(12, 7)
    flat = torch.stack([torch.as_strided(g, (7,), (1,), g.storage_offset() + r // share * ld) for r in range(12)])
    assert torch.equal(flat, want)


def test_gate_of_another_shape_is_refused():
    with pytest.raises(ValueError):
        bs._gate_rows(torch.zeros(5, 7), torch.zeros(4, 3, 7))


def test_scale_layouts():
    made = bs._new_scales((2, 3), 6, 5, "cpu")
    assert made.shape == (2, 3, 5)
    flat, ld = bs._scale_rows(made, 6, 5)
    assert flat.data_ptr() == made.data_ptr() and ld == 6 and flat.stride(0) == 1
    plain = torch.arange(30.0).view(6, 5)
    flat, ld = bs._scale_rows(plain, 6, 5)
    assert ld == 6 and torch.equal(flat, plain) and flat.stride() == (1, 6)
    one, ld = bs._scale_rows(torch.arange(5.0).view(1, 5), 1, 5)
    assert ld == 1 and one.shape == (1, 5)
    wide = torch.empty(5, 9).t()[:6]                                     # rows of a block side by side, blocks further apart
    assert bs._scale_rows(wide, 6, 5)[1] == 9


def test_more_rows_than_a_launch_holds():
    """row counts whose bytes, grid or threads leave 32 bits: refused on the host, at both boundaries"""
    L = bs._library()
    p = 4096

    def product(m, **kw):
        return L.wqaa_block_matmul(ctypes.byref(_desc(**kw)), p, p, p, m, p, None, p, m, p, 1 << 60, None)

    for m in (1 << 29, (1 << 31) - 1):
        assert product(m) == wlib.ERR_UNSUPPORTED
        assert L.wqaa_block_workspace_bytes(ctypes.byref(_desc()), m) == 0
        assert L.wqaa_block_select(ctypes.byref(_desc()), m, None) == wlib.ERR_UNSUPPORTED
    assert product(1, N=(1 << 31) - 1, K=16) == wlib.ERR_UNSUPPORTED      # 2^27 workgroups of 512 threads
    assert L.wqaa_block_select(ctypes.byref(_desc(N=1 << 20)), (1 << 29) - 1, None) == wlib.ERR_UNSUPPORTED
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=256, K=256))
    assert op.plan((1 << 29) - 1)["grid"] > 0
    for m in (1 << 29, 1 << 32, -1):                                      # (2^32: nothing of it may be cut off on the way)
        with pytest.raises(ValueError):
            op.plan(m)
        with pytest.raises(ValueError):
            op.workspace_bytes(m)

    a = bs.BlockQuant(bs._QUANT_BYTES, wlib.BF16, wlib.E4M3, 0, 1 << 28, 1, 1, 1, 1 << 28, p, None, p, p)
    a.rows = (1 << 28) + 16                                               # 2^24 + 1 workgroups of 256 threads
    a.s_ld = a.rows
    assert L.wqaa_block_quantize(ctypes.byref(a), None) == wlib.ERR_UNSUPPORTED
    a.rows = (1 << 62) + 1
    a.s_ld = a.rows
    assert L.wqaa_block_quantize(ctypes.byref(a), None) == wlib.ERR_UNSUPPORTED
    n = bs.ResidualNormArgs(bs._NORM_BYTES, wlib.BF16, wlib.BF16, wlib.BF16, -1, 1e-5, 1.0, 1.0, 1 << 26, 16, 16)
    n.x = n.weight = n.Y = p
    assert L.wqaa_residual_norm(ctypes.byref(n), None) == wlib.ERR_UNSUPPORTED


def test_outputs_that_autograd_tracks_are_refused():
    with pytest.raises(RuntimeError, match="no backward"):
        bs._refuse_grad("residual_norm", torch.zeros(2), None, torch.zeros(2, requires_grad=True))


def test_forward_mode_tangents_are_refused():
    """also where grad mode is off, which does not switch them off; a tensor without one, and a dual tensor's primal, pass"""
    x, v = torch.ones(2, 3), torch.ones(2, 3)
    bs._refuse_grad("residual_norm", x, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, v)
        for mode in (True, False):
            with torch.set_grad_enabled(mode):
                assert bs._recorded()
                bs._refuse_grad("residual_norm", x, None, torch.autograd.forward_ad.unpack_dual(dual).primal, x.to(torch.float8_e4m3fn))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    bs._refuse_grad("residual_norm", x, None, dual)
    with torch.no_grad():
        assert not bs._recorded()
        bs._refuse_grad("residual_norm", torch.zeros(2, requires_grad=True))


@pytest.mark.parametrize("tile", [0, 1])
@pytest.mark.parametrize("rows", [(1 << 63) - 1, (1 << 63) - 16, (1 << 41) + 1])
def test_quantizer_row_counts_at_the_end_of_64_bits(tile, rows):
    """a count whose rounding up to whole blocks would leave 64 bits is refused like any other that no launch holds"""
    p = 4096
    a = bs.BlockQuant(bs._QUANT_BYTES, wlib.BF16, wlib.E4M3, tile, rows, 128, 128, 128, rows, p, None, p, p)
    assert bs._library().wqaa_block_quantize(ctypes.byref(a), None) == wlib.ERR_UNSUPPORTED


def test_member_cases_are_the_members_they_name():
    """the device's tests of every member take what they say, whole K and cut"""
    import test_block_scaled_members_gpu as cases
    for name in cases.MEMBERS:
        for cut in (False, True):
            cases.operator(name, cut)
    for name, turns, extra in cases.TURNS:
        M, N, member, blocks = cases.LOOPS[name]
        plan = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=turns * blocks * 128 + extra)).plan(M)
        assert (plan["block_m"], plan["block_n"], plan["threads"]) == member, plan["name"]


@pytest.mark.parametrize("change", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float32), lambda m: m.to("meta", torch.bfloat16),
                                    lambda m: m.to(torch.zeros(1, dtype=torch.float16))], ids=["half", "bfloat16", "double", "float", "meta", "like"])
def test_a_model_cast_leaves_the_layer_its_types(change):
    """a cast of the model around it: the operator still takes the layer's buffers, and their values are whole"""
    lin = bitblas.BlockScaledLinear(256, 128, bias=True, W_dtype="e5m2_float8", out_dtype="bfloat16")
    lin.weight.view(torch.uint8).copy_(torch.arange(256, dtype=torch.uint8).expand(128, 256) & 0x3F)
    lin.weight_scale.fill_(2.0 ** -40 / 448)
    lin.bias.fill_(3.0)
    held = {k: v.clone() for k, v in lin.state_dict().items()}
    model = torch.nn.Sequential(lin, torch.nn.Linear(4, 4))
    assert change(model) is model
    for name, was in held.items():
        now = getattr(lin, name)
        assert now.dtype == was.dtype and now.shape == was.shape and now is lin.state_dict(keep_vars=True)[name]
        assert now.device.type == "meta" or torch.equal(now.view(torch.uint8), was.view(torch.uint8))


def test_rows_with_axes_of_one_between():
    """the last token of each sequence, (B, 1, K): rows as even as without the axis of one, and read where they are"""
    t = torch.arange(4 * 6 * 10).view(4, 6, 10)
    for view, ld in ((t[:, -1:], 60), (t[:, 2:3, 1:8], 60), (t[:, None, 3, :5], 60), (t.view(4, 6, 1, 10)[::2, :, :, :4][:1], 10), (t[1:3, :, None, 2:], 10)):
        assert not view.is_contiguous()
        got, d = bs._rows(view)
        k = view.shape[-1]
        assert d == ld and got.data_ptr() == view.data_ptr()
        assert torch.equal(torch.as_strided(got, (view.numel() // k, k), (d, 1), got.storage_offset()), view.reshape(-1, k))
    for view in (t[:, 1:2, ::2], t[:, :2].transpose(0, 1)[:, None], t[:1, None].expand(4, 1, 6, 10)):
        got, d = bs._rows(view)
        k = view.shape[-1]
        assert torch.equal(torch.as_strided(got, (view.numel() // k, k), (d, 1), got.storage_offset()), view.reshape(-1, k))
