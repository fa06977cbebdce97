"""Matmuls with both operands in 8-bit floating point and a float32 scale for each block of 128 - activations per row, weights
per 128 x 128 tile - with the quantiser that makes the operands and the norm launch that stands between two blocks of a layer.

The reference's fp8 matmuls (`A_dtype="e4m3_float8", W_dtype="e4m3_float8"`, bitblas/ops/general_matmul/__init__.py:372-383) multiply the
bytes as they are; a checkpoint quantised in blocks needs the scales inside the sum over k:

    C[m, n] = sum_b scale_a[m, b] scale_w[n // 128, b] sum_{k in block b} A[m, k] W[n, k]   (+ bias[n])

A decoder layer on this path (`BlockScaledLinear`, `BlockScaledGatedMLP`):

    x, y = residual_norm(attn_out, x, ln.weight, eps, quantize="e4m3_float8")   # residual add, norm, 8-bit rows: one launch
    gate_up = linear(y)                                                       # both projections, one product
    act = quantize_blocks(up, gate=gate)                                      # silu(gate) * up, 8-bit rows: one launch
    out = down(act)

Everything is float32 inside, with one rounding at the end, asynchronous on the current stream of the operands' device, and made for
inference: a call that autograd would record is refused.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch

from . import lib as _lib
from .matmul import Operator, OperatorConfig, torch_dtype

BLOCK = 128
_FP8 = ("e4m3_float8", "e5m2_float8")
_CODE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32, torch.float8_e4m3fn: _lib.E4M3,
         torch.float8_e5m2: _lib.E5M2}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class BlockDesc(ctypes.Structure):
    """struct wqaa_block_desc (include/wqaa.h)."""
    _fields_ = [("struct_size", ctypes.c_int32), ("N", ctypes.c_int32), ("K", ctypes.c_int32), ("a_dtype", ctypes.c_int32),
                ("w_dtype", ctypes.c_int32), ("out_dtype", ctypes.c_int32), ("with_bias", ctypes.c_int32), ("reserved", ctypes.c_int32 * 1)]


class BlockQuant(ctypes.Structure):
    """struct wqaa_block_quant (include/wqaa.h)."""
    _fields_ = [("struct_size", ctypes.c_int32), ("x_dtype", ctypes.c_int32), ("q_dtype", ctypes.c_int32), ("tile", ctypes.c_int32),
                ("rows", ctypes.c_int64), ("K", ctypes.c_int64), ("x_ld", ctypes.c_int64), ("gate_ld", ctypes.c_int64), ("s_ld", ctypes.c_int64),
                ("X", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("Q", ctypes.c_void_p), ("S", ctypes.c_void_p)]


class ResidualNormArgs(ctypes.Structure):
    """struct wqaa_residual_norm_args (include/wqaa.h)."""
    _fields_ = [("struct_size", ctypes.c_int32), ("x_dtype", ctypes.c_int32), ("stream_dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("q_dtype", ctypes.c_int32), ("eps", ctypes.c_float), ("scale", ctypes.c_float), ("residual_scale", ctypes.c_float),
                ("rows", ctypes.c_int64), ("D", ctypes.c_int64), ("x_ld", ctypes.c_int64), ("residual_ld", ctypes.c_int64), ("gate_ld", ctypes.c_int64),
                ("gate_rows", ctypes.c_int64), ("s_ld", ctypes.c_int64), ("x", ctypes.c_void_p), ("residual", ctypes.c_void_p),
                ("gate", ctypes.c_void_p), ("post_weight", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("stream", ctypes.c_void_p),
                ("Y", ctypes.c_void_p), ("S", ctypes.c_void_p)]


_bound = None


def _library():
    global _bound
    if _bound is None:
        lib = _lib.load_library()
        vp, ci, i64, u64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64
        dp = ctypes.POINTER(BlockDesc)
        lib.wqaa_block_matmul.restype = ci
        lib.wqaa_block_matmul.argtypes = [dp, vp, vp, vp, i64, vp, vp, vp, ci, vp, u64, vp]
        lib.wqaa_block_workspace_bytes.restype = u64
        lib.wqaa_block_workspace_bytes.argtypes = [dp, ci]
        lib.wqaa_block_select.restype = ci
        lib.wqaa_block_select.argtypes = [dp, ci, ctypes.POINTER(_lib.Plan)]
        lib.wqaa_block_quantize.restype = ci
        lib.wqaa_block_quantize.argtypes = [ctypes.POINTER(BlockQuant), vp]
        lib.wqaa_residual_norm.restype = ci
        lib.wqaa_residual_norm.argtypes = [ctypes.POINTER(ResidualNormArgs), vp]
        _bound = lib
    return _bound


def _refuse_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or detach its inputs")


def _on(what: str, device, *tensors) -> None:
    for name, t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, the call's input on {device}")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """`t` with its leading dimensions as rows a fixed distance apart: (tensor, distance in elements).  A tensor whose rows are
    not laid out like that is copied."""
    k = t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= k:
        return t, t.stride(0)
    if t.is_contiguous():
        return t, k
    if t.dim() >= 2 and t.stride(-1) == 1:
        ld = t.stride(-2)
        step = ld
        for size, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
            if size != 1 and stride != step:
                break
            step *= size
        else:
            if ld >= k:
                return t, ld
    t = t.contiguous()
    return t, k


def _scale_rows(scale: torch.Tensor, m: int, kb: int) -> Tuple[torch.Tensor, int]:
    """row scales (..., blocks) as the kernels read them: the rows of one block side by side, (tensor, distance of two blocks)"""
    if scale.dim() != 2:
        scale = scale.reshape(m, kb)                  # (a view where the layout allows one, as for what quantize_blocks returns)
    if (scale.stride(0) == 1 or m == 1) and (kb == 1 or scale.stride(1) >= m):
        return scale, scale.stride(1) if kb > 1 else m
    scale = scale.t().contiguous().t()
    return scale, m


def _new_scales(lead: Sequence[int], m: int, kb: int, device) -> torch.Tensor:
    """(*lead, kb) float32 scales over (kb, m) storage"""
    s = torch.empty((kb, m), dtype=torch.float32, device=device)
    return s.t() if len(lead) == 1 else s.view(kb, *lead).movedim(0, -1)


@dataclass(frozen=True)
class BlockScaledMatmulConfig(OperatorConfig):
    """One block-scaled product: A (M, K) x W (N, K)^T, any row count."""
    N: int = None
    K: int = None
    A_dtype: str = "e4m3_float8"
    W_dtype: str = "e4m3_float8"
    out_dtype: str = "float16"
    with_bias: bool = False

    def __post_init__(self):
        for name in ("N", "K"):
            v = getattr(self, name)
            if not isinstance(v, int) or v <= 0:
                raise ValueError(f"{name} should be a positive integer")
        if self.K % 16 != 0:
            raise ValueError("K should be a multiple of 16 (the operands are read in 16-byte pieces)")
        if self.A_dtype not in _FP8 or self.W_dtype not in _FP8:
            raise ValueError(f"A_dtype and W_dtype are one of {_FP8}")
        if self.out_dtype not in ("float16", "bfloat16"):
            raise ValueError("out_dtype is float16 or bfloat16")


class BlockScaledMatmul(Operator):
    """`op(A, W, scale_a, scale_w, bias=None, output=None)`.

    A        (..., K) in `A_dtype`; W (N, K) in `W_dtype`, contiguous
    scale_a  (..., ceil(K / 128)) float32, any layout (what `quantize_blocks` and `residual_norm` return is read as it is; another
             layout than theirs costs a small copy)
    scale_w  (ceil(N / 128), ceil(K / 128)) float32, contiguous
    bias     (N,) in `out_dtype`, added before the one rounding
    output   optional contiguous (..., N) tensor in `out_dtype`; it may not overlap the operands

    Sums are float32, but for the matrix unit's own over 8 consecutive k, which cuts every product off at 2^-13 of the largest one's power
    of two: about 2^-15 of an output of ordinary data, a few times less than a rounding to float16 (which is why there is no float32 output)."""

    def __init__(self, config: BlockScaledMatmulConfig):
        self.config = config
        self.N, self.K = config.N, config.K
        self._kb, self._nb = _blocks(self.K), _blocks(self.N)
        self._a, self._w, self._out = torch_dtype(config.A_dtype), torch_dtype(config.W_dtype), torch_dtype(config.out_dtype)
        self.torch_output_dtype = self._out
        d = BlockDesc()
        d.struct_size = ctypes.sizeof(BlockDesc)
        d.N, d.K = self.N, self.K
        d.a_dtype, d.w_dtype, d.out_dtype = _CODE[self._a], _CODE[self._w], _CODE[self._out]
        d.with_bias = int(config.with_bias)
        self.desc = d
        self._ref = ctypes.byref(d)
        self._need = {}                               # row count -> bytes of partial sums
        self._fn = _library().wqaa_block_matmul

    def plan(self, m: int) -> dict:
        """the member a call with `m` rows takes (needs no device)"""
        plan = _lib.Plan()
        _lib.check(_library().wqaa_block_select(self._ref, int(m), ctypes.byref(plan)))
        return plan.as_dict()

    def workspace_bytes(self, m: int) -> int:
        need = self._need.get(m)
        if need is None:
            need = self._need[m] = int(_library().wqaa_block_workspace_bytes(self._ref, int(m)))
        return need

    def forward(self, A, W, scale_a, scale_w, bias=None, output=None):
        N, K, kb = self.N, self.K, self._kb
        device = A.device
        if device.type != "cuda":
            raise RuntimeError("BlockScaledMatmul runs on the GPU only")
        shape = A.shape
        if A.dtype != self._a or not shape or shape[-1] != K:
            raise ValueError(f"A is (..., {K}) in {self._a}: got {tuple(shape)} in {A.dtype}")
        if W.dtype != self._w or W.shape != (N, K) or not W.is_contiguous():
            raise ValueError(f"W is a contiguous ({N}, {K}) tensor in {self._w}: got {tuple(W.shape)} in {W.dtype}")
        lead = shape[:-1]
        if scale_a.dtype != torch.float32 or scale_a.shape != lead + (kb,):
            raise ValueError(f"scale_a is {tuple(lead) + (kb,)} in float32: got {tuple(scale_a.shape)} in {scale_a.dtype}")
        if scale_w.dtype != torch.float32 or scale_w.shape != (self._nb, kb) or not scale_w.is_contiguous():
            raise ValueError(f"scale_w is a contiguous ({self._nb}, {kb}) tensor in float32: got {tuple(scale_w.shape)} in {scale_w.dtype}")
        if W.device != device or scale_a.device != device or scale_w.device != device:
            raise ValueError(f"W and the scales must be on A's device ({device})")
        if (bias is not None) != self.config.with_bias:
            raise ValueError("the bias goes with with_bias, and only with it")
        if bias is not None and (bias.dtype != self._out or bias.shape != (N,) or not bias.is_contiguous() or bias.device != device):
            raise ValueError(f"bias is a contiguous ({N},) tensor in {self._out} on A's device")
        _refuse_grad("BlockScaledMatmul", scale_a, scale_w, bias)
        m = A.numel() // K
        if not A.is_contiguous() or A.data_ptr() & 15:
            A = A.contiguous() if not A.is_contiguous() else A.clone()
        if W.data_ptr() & 15:
            raise ValueError("W must be aligned to 16 bytes")
        if output is None:
            output = torch.empty(lead + (N,), dtype=self._out, device=device)
        elif output.shape != lead + (N,) or output.dtype != self._out or not output.is_contiguous() or output.device != device:
            raise ValueError(f"output is a contiguous {tuple(lead) + (N,)} tensor in {self._out} on A's device")
        if m == 0:
            return output
        scale_a, ld = _scale_rows(scale_a, m, kb)
        need = self.workspace_bytes(m)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        status = self._fn(self._ref, A.data_ptr(), W.data_ptr(), scale_a.data_ptr(), ld, scale_w.data_ptr(), bias.data_ptr() if bias is not None else None,
                          output.data_ptr(), m, ws.data_ptr() if need else None, need, _lib.current_stream_handle(device))
        if status != _lib.OK:
            _lib.check(status)
        return output


def quantize_blocks(x: torch.Tensor, dtype: str = "e4m3_float8", *, tile: bool = False, gate: Optional[torch.Tensor] = None,
                    output: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(values, scales) of x in blocks of 128 along its last axis.

    x       (..., K) in float16, bfloat16 or float32; rows may lie apart (a slice of a wider tensor).  K is any number here; a product
            wants a multiple of 16
    tile    False: a scale per row and block, (..., ceil(K / 128)) - activations.  True: x is (N, K) and a scale stands for 128 rows
            too, (ceil(N / 128), ceil(K / 128)) - weights
    gate    as x: silu(gate) * x is quantised, computed in float32 and not rounded in between (rows only)
    output  (values, scales) of an earlier call with the same shapes, to be written again

    scale = max(max|x|, 2^-40) / L, L the largest value of `dtype` (448, 57344); value = x / scale, the float32 quotient, rounded to
    nearest even.  A block of zeros comes back as zeros, one that holds an infinity or a NaN as NaN with a scale that is not finite."""
    if dtype not in _FP8:
        raise ValueError(f"dtype is one of {_FP8}")
    device = x.device
    if device.type != "cuda":
        raise RuntimeError("quantize_blocks runs on the GPU only")
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32) or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x is (..., K) in float16, bfloat16 or float32: got {tuple(x.shape)} in {x.dtype}")
    if tile and (x.dim() != 2 or gate is not None):
        raise ValueError("tiles are taken of an (N, K) tensor, without a gate")
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype or gate.device != device):
        raise ValueError("gate has the shape, type and device of x")
    _refuse_grad("quantize_blocks", x, gate)
    shape, K = x.shape, x.shape[-1]
    lead = shape[:-1]
    m = x.numel() // K
    kb = _blocks(K)
    qt = torch_dtype(dtype)
    if output is None:
        q = torch.empty(shape, dtype=qt, device=device)
        s = torch.empty((_blocks(m), kb), dtype=torch.float32, device=device) if tile else _new_scales(lead, m, kb, device)
    else:
        q, s = output
        if q.shape != shape or q.dtype != qt or not q.is_contiguous() or q.device != device:
            raise ValueError(f"output values are a contiguous {tuple(shape)} tensor in {qt} on x's device")
        want = (_blocks(m), kb) if tile else lead + (kb,)
        if s.shape != want or s.dtype != torch.float32 or s.device != device or (tile and not s.is_contiguous()):
            raise ValueError(f"output scales are a {tuple(want)} tensor in float32 on x's device")
    if m == 0:
        return q, s
    a = BlockQuant()
    if not tile:
        flat, a.s_ld = _scale_rows(s, m, kb)
        if flat.data_ptr() != s.data_ptr():
            raise ValueError("output scales have the rows of a block side by side, as quantize_blocks returns them")
    a.struct_size = ctypes.sizeof(BlockQuant)
    a.x_dtype, a.q_dtype, a.tile = _CODE[x.dtype], _CODE[qt], int(tile)
    a.rows, a.K = m, K
    x, a.x_ld = _rows(x)
    a.X, a.Q, a.S = x.data_ptr(), q.data_ptr(), s.data_ptr()
    if gate is not None:
        gate, a.gate_ld = _rows(gate)
        a.gate = gate.data_ptr()
    status = _library().wqaa_block_quantize(ctypes.byref(a), _lib.current_stream_handle(device))
    if status != _lib.OK:
        _lib.check(status)
    return q, s


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """`gate`, broadcast against x, as (tensor, distance of two gate rows in elements, rows of x that share one)"""
    D = x.shape[-1]
    if gate.dim() == 0 or gate.shape[-1] == 1:
        gate = gate.expand(gate.shape[:-1] + (D,))
    try:
        g = gate.expand(x.shape)
    except RuntimeError:
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast against x {tuple(x.shape)}") from None
    if g.stride(-1) != 1 and D > 1:
        gate = gate.contiguous()                      # (one value for a whole row, or columns apart)
        g = gate.expand(x.shape)
    # from the last axis outwards: axes the gate does not vary along, then axes its rows lie evenly along
    share, ld, step = 1, 0, None
    for size, stride in zip(x.shape[-2::-1], g.stride()[-2::-1]):
        if size == 1:
            continue
        if stride == 0 and step is None:
            share *= size
        elif step is None:
            ld = stride
            step = stride * size
        elif stride == step:
            step *= size
        else:
            g = g.contiguous()                        # it varies along some axes in a way no pair of numbers describes
            return g, D, 1
    return g, ld, share


def residual_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0, residual_scale: float = 1.0,
                  quantize: Optional[str] = None, output: Optional[Sequence[Optional[torch.Tensor]]] = None
                  ) -> Tuple[torch.Tensor, Union[None, torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]]:
    """What stands between two blocks of a layer, in one launch: the norm behind the block, its gate, the scaled residual add, and the norm
    in front of the next block, which may leave quantised.

        z = x                    or  x rsqrt(mean x^2 + eps) post_weight
        h = residual_scale residual + scale gate z
        y = h rsqrt(mean h^2 + eps) weight

    x            (..., D) float16 or bfloat16, D <= 32768: the block's output
    residual     the stream, x's shape, in x's type or float32; None: there is none (h = scale gate z)
    weight       (D,) in x's type or float32 (post_weight the same); None: no second norm, y is None
    gate         broadcast against x, in x's type: (D,), (B, 1, D), x's shape, ...
    quantize     None: y in x's type.  An 8-bit type: y = (values, scales) as `quantize_blocks` makes them, of the unrounded y
    output       (h, y), or (h, values, scales): tensors to write; h may be `residual` itself

    Returns (h, y), h in the residual's type.  Without residual, gate, post_weight and scale, h is x and is returned as it is.  float32
    inside; y is taken of h before h is rounded, and every output is rounded once.  (The reference's norm,
    integration/BitNet/modeling_bitnet.py:89-104, rounds to the activations' type before it multiplies by the weight.)"""
    device = x.device
    if device.type != "cuda":
        raise RuntimeError("residual_norm runs on the GPU only")
    t = x.dtype
    if t not in (torch.float16, torch.bfloat16) or x.dim() < 1 or not 1 <= x.shape[-1] <= 32768:
        raise ValueError(f"x is (..., D) in float16 or bfloat16, D <= 32768: got {tuple(x.shape)} in {t}")
    shape, D = x.shape, x.shape[-1]
    st = t
    if residual is not None:
        st = residual.dtype
        if residual.shape != shape or st not in (t, torch.float32):
            raise ValueError(f"residual has x's shape, in {t} or float32: got {tuple(residual.shape)} in {st}")
    wt = None
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is None:
            continue
        if w.shape != (D,) or w.dtype not in (t, torch.float32) or not w.is_contiguous():
            raise ValueError(f"{name} is a contiguous ({D},) tensor in {t} or float32")
        if wt is not None and w.dtype != wt:
            raise ValueError("weight and post_weight have one type")
        wt = w.dtype
    if gate is not None and gate.dtype != t:
        raise ValueError(f"gate is in {t}")
    if quantize is not None and (quantize not in _FP8 or weight is None):
        raise ValueError(f"quantize is one of {_FP8}, and goes with a weight")
    if not float(eps) >= 0.0:
        raise ValueError("the norm's eps must be a non-negative number")
    _on("residual_norm", device, ("residual", residual), ("weight", weight), ("post_weight", post_weight), ("gate", gate))
    _refuse_grad("residual_norm", x, residual, weight, post_weight, gate)
    m = x.numel() // D
    kb = _blocks(D)
    passes = residual is None and gate is None and post_weight is None and scale == 1.0     # h is x
    if passes and weight is None:
        raise ValueError("nothing to do: no residual, gate, post_weight or scale, and no weight")
    out = (None,) * 3 if output is None else (tuple(output) + (None,) * 3)[:3]
    h, y, s = out
    if h is None:
        h = x if passes else torch.empty(shape, dtype=st, device=device)
        write_h = not passes
    else:
        if h.shape != shape or h.dtype != st or not h.is_contiguous() or h.device != device:
            raise ValueError(f"output h is a contiguous {tuple(shape)} tensor in {st} on x's device")
        write_h = True
    yt = t if quantize is None else torch_dtype(quantize)
    if weight is None:
        if y is not None or s is not None:
            raise ValueError("an output for y goes with a weight")
    else:
        if y is None:
            y = torch.empty(shape, dtype=yt, device=device)
        elif y.shape != shape or y.dtype != yt or not y.is_contiguous() or y.device != device:
            raise ValueError(f"output y is a contiguous {tuple(shape)} tensor in {yt} on x's device")
        if quantize is None:
            if s is not None:
                raise ValueError("an output for scales goes with quantize")
        elif s is None:
            s = _new_scales(shape[:-1], m, kb, device)
        elif s.shape != shape[:-1] + (kb,) or s.dtype != torch.float32 or s.device != device:
            raise ValueError(f"output scales are a {tuple(shape[:-1]) + (kb,)} tensor in float32 on x's device")
    result = (h, None if weight is None else y if quantize is None else (y, s))
    if m == 0:
        return result
    a = ResidualNormArgs()
    a.struct_size = ctypes.sizeof(ResidualNormArgs)
    a.x_dtype, a.stream_dtype, a.weight_dtype = _CODE[t], _CODE[st], _CODE[wt or t]
    a.q_dtype = -1 if quantize is None else _CODE[yt]
    a.eps, a.scale, a.residual_scale = float(eps), float(scale), float(residual_scale)
    a.rows, a.D = m, D
    x, a.x_ld = _rows(x)
    a.x = x.data_ptr()
    if residual is not None:
        residual, a.residual_ld = _rows(residual)
        a.residual = residual.data_ptr()
    if gate is not None:
        gate, a.gate_ld, a.gate_rows = _gate_rows(gate, result[0])
        a.gate = gate.data_ptr()
    if post_weight is not None:
        a.post_weight = post_weight.data_ptr()
    if write_h:
        a.stream = h.data_ptr()
    if weight is not None:
        a.weight, a.Y = weight.data_ptr(), y.data_ptr()
        if quantize is not None:
            flat, a.s_ld = _scale_rows(s, m, kb)
            if flat.data_ptr() != s.data_ptr():
                raise ValueError("output scales have the rows of a block side by side, as quantize_blocks returns them")
            a.S = s.data_ptr()
    status = _library().wqaa_residual_norm(ctypes.byref(a), _lib.current_stream_handle(device))
    if status != _lib.OK:
        _lib.check(status)
    return result
