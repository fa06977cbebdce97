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
inference: a call that autograd would record, backward or forward, is refused.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad as _forward_ad

from . import lib as _lib
from .matmul import Operator, OperatorConfig, torch_dtype

BLOCK = 128
_FP8 = ("e4m3_float8", "e5m2_float8")
_CODE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32, torch.float8_e4m3fn: _lib.E4M3,
         torch.float8_e5m2: _lib.E5M2}


_FP8_TYPE = {"e4m3_float8": torch.float8_e4m3fn, "e5m2_float8": torch.float8_e5m2}
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


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


_QUANT_BYTES, _NORM_BYTES = ctypes.sizeof(BlockQuant), ctypes.sizeof(ResidualNormArgs)
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


def _recorded() -> bool:
    """whether there may be anything for `_refuse_grad` to find (forward-mode tangents do not ask for grad mode)"""
    return torch.is_grad_enabled() or _forward_ad._current_level >= 0


def _refuse_grad(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or detach its inputs")
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative: unpack its inputs")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """`t` with its leading dimensions as rows a fixed distance apart: (tensor, distance in elements).  A tensor whose rows are
    not laid out like that is copied."""
    k = t.shape[-1]
    if t.is_contiguous():
        return t, k
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= k:
        return t, t.stride(0)
    if t.dim() >= 2 and t.stride(-1) == 1:
        ld = step = None
        for size, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
            if size == 1:
                continue
            if step is None:
                ld, step = stride, stride * size
            elif stride == step:
                step *= size
            else:
                break
        else:
            if ld is not None and ld >= k:
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


# (empty_like and empty_strided take about 1.3 us where empty takes 2.2, which a call of 6 notices)
def _new(like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """a contiguous tensor of `like`'s shape"""
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _new_rows(lead: Sequence[int], n: int, dtype: torch.dtype, device) -> torch.Tensor:
    """a contiguous (*lead, n) tensor"""
    if len(lead) == 1:
        return torch.empty_strided((lead[0], n), (n, 1), dtype=dtype, device=device)
    return torch.empty((*lead, n), dtype=dtype, device=device)


def _scale_strides(lead: Sequence[int], m: int) -> Tuple[int, ...]:
    """strides of (*lead, blocks) scales over (blocks, m) storage"""
    if len(lead) == 1:
        return (1, m)
    strides = [m]
    step = 1
    for size in reversed(lead):
        strides.insert(0, step)
        step *= size
    return tuple(strides)


def _new_scales(lead: Sequence[int], m: int, kb: int, device) -> torch.Tensor:
    """(*lead, kb) float32 scales over (kb, m) storage"""
    return torch.empty_strided((*lead, kb), _scale_strides(lead, m), dtype=torch.float32, device=device)


def _scale_ld(scale: torch.Tensor, lead: Sequence[int], m: int, kb: int) -> int:
    """distance of two blocks in scales the kernels write"""
    strides = scale.stride()
    if strides == _scale_strides(lead, m):
        return m
    flat, ld = _scale_rows(scale, m, kb)
    if flat.data_ptr() != scale.data_ptr():
        raise ValueError("output scales have the rows of a block side by side, as quantize_blocks returns them")
    return ld


@dataclass(frozen=True)
class BlockScaledMatmulConfig(OperatorConfig):
    """One block-scaled product: A (M, K) x W (N, K)^T, any row count; K a multiple of 16 up to 2^22."""
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
        self._w_shape, self._sw_shape, self._bias_shape = torch.Size((self.N, self.K)), torch.Size((self._nb, self._kb)), torch.Size((self.N,))
        self._with_bias = bool(config.with_bias)
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
        self.workspace_bytes(m)
        plan = _lib.Plan()
        _lib.check(_library().wqaa_block_select(self._ref, int(m), ctypes.byref(plan)))
        return plan.as_dict()

    def workspace_bytes(self, m: int) -> int:
        need = self._need.get(m)
        if need is None:
            if not 0 <= m < 1 << 29:
                raise ValueError(f"a call takes fewer than 2^29 rows: got {m}")
            need = self._need[m] = int(_library().wqaa_block_workspace_bytes(self._ref, int(m)))
        return need

    def _refuse(self, A, W, scale_a, scale_w, bias, output):
        """what `forward` found wrong, in words"""
        N, K, kb, device, lead = self.N, self.K, self._kb, A.device, tuple(A.shape[:-1])
        if device.type != "cuda":
            raise RuntimeError("BlockScaledMatmul runs on the GPU only")
        if A.dtype != self._a or A.dim() == 0 or A.shape[-1] != K:
            raise ValueError(f"A is (..., {K}) in {self._a}: got {tuple(A.shape)} in {A.dtype}")
        if W.dtype != self._w or W.shape != (N, K) or not W.is_contiguous():
            raise ValueError(f"W is a contiguous ({N}, {K}) tensor in {self._w}: got {tuple(W.shape)} in {W.dtype}")
        if scale_a.dtype != torch.float32 or scale_a.shape != lead + (kb,):
            raise ValueError(f"scale_a is {lead + (kb,)} in float32: got {tuple(scale_a.shape)} in {scale_a.dtype}")
        if scale_w.dtype != torch.float32 or scale_w.shape != (self._nb, kb) or not scale_w.is_contiguous():
            raise ValueError(f"scale_w is a contiguous ({self._nb}, {kb}) tensor in float32: got {tuple(scale_w.shape)} in {scale_w.dtype}")
        if W.device != device or scale_a.device != device or scale_w.device != device:
            raise ValueError(f"W and the scales must be on A's device ({device})")
        if W.data_ptr() & 15:
            raise ValueError("W must be aligned to 16 bytes")
        if (bias is not None) != self.config.with_bias:
            raise ValueError("the bias goes with with_bias, and only with it")
        if bias is not None and (bias.dtype != self._out or bias.shape != (N,) or not bias.is_contiguous() or bias.device != device):
            raise ValueError(f"bias is a contiguous ({N},) tensor in {self._out} on A's device")
        raise ValueError(f"output is a contiguous {lead + (N,)} tensor in {self._out} on A's device")

    def forward(self, A, W, scale_a, scale_w, bias=None, output=None):
        # (one chain of cheap tests: a decode step's call is as long as its host code)
        N, K, kb = self.N, self.K, self._kb
        dev = A.get_device()
        shape = A.shape
        lead = shape[:-1]
        if (dev < 0 or A.dtype is not self._a or not shape or shape[-1] != K or W.dtype is not self._w or W.shape != self._w_shape
                or not W.is_contiguous() or scale_a.dtype is not torch.float32 or scale_a.shape != lead + (kb,) or scale_w.dtype is not torch.float32
                or scale_w.shape != self._sw_shape or not scale_w.is_contiguous() or W.get_device() != dev or scale_a.get_device() != dev
                or scale_w.get_device() != dev):
            self._refuse(A, W, scale_a, scale_w, bias, output)
        w_ptr = W.data_ptr()
        if w_ptr & 15 or (bias is not None) is not self._with_bias:
            self._refuse(A, W, scale_a, scale_w, bias, output)
        if bias is None:
            bias_ptr = None
        else:
            if bias.dtype is not self._out or bias.shape != self._bias_shape or not bias.is_contiguous() or bias.get_device() != dev:
                self._refuse(A, W, scale_a, scale_w, bias, output)
            bias_ptr = bias.data_ptr()
        if _recorded():
            _refuse_grad("BlockScaledMatmul", A, W, scale_a, scale_w, bias, output)
        if output is None:
            output = _new_rows(lead, N, self._out, A.device)
        elif output.shape != lead + (N,) or output.dtype is not self._out or not output.is_contiguous() or output.get_device() != dev:
            self._refuse(A, W, scale_a, scale_w, bias, output)
        m = A.numel() // K
        if m == 0:
            return output
        if not A.is_contiguous():
            A = A.contiguous()
        a_ptr = A.data_ptr()
        if a_ptr & 15:
            A = A.clone()
            a_ptr = A.data_ptr()
        if len(lead) != 1 or scale_a.stride() != (1, m):
            scale_a, ld = _scale_rows(scale_a, m, kb)
        else:
            ld = m
        need = self._need.get(m)
        if need is None:
            need = self.workspace_bytes(m)
        if need:
            ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=A.device)
            status = self._fn(self._ref, a_ptr, w_ptr, scale_a.data_ptr(), ld, scale_w.data_ptr(), bias_ptr, output.data_ptr(), m, ws.data_ptr(), need,
                              _raw_stream(dev))
        else:
            status = self._fn(self._ref, a_ptr, w_ptr, scale_a.data_ptr(), ld, scale_w.data_ptr(), bias_ptr, output.data_ptr(), m, None, 0, _raw_stream(dev))
        if status != _lib.OK:
            _lib.check(status)
        return output

    __call__ = forward


def quantize_blocks(x: torch.Tensor, dtype: str = "e4m3_float8", *, tile: bool = False, gate: Optional[torch.Tensor] = None,
                    output: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(values, scales) of x in blocks of 128 along its last axis.

    x       (..., K) in float16, bfloat16 or float32; rows may lie apart (a slice of a wider tensor).  K is any number up to 2^30 here; a
            product wants a multiple of 16
    tile    False: a scale per row and block, (..., ceil(K / 128)) - activations.  True: x is (N, K) and a scale stands for 128 rows
            too, (ceil(N / 128), ceil(K / 128)) - weights
    gate    as x: silu(gate) * x is quantised, computed in float32 and not rounded in between (rows only)
    output  (values, scales) of an earlier call with the same shapes, to be written again

    scale = max(max|x|, 2^-40) / L, L the largest value of `dtype` (448, 57344); value = x / scale, the float32 quotient, rounded to
    nearest even.  A block of zeros comes back as zeros, one that holds an infinity or a NaN as NaN with a scale that is not finite."""
    qt = _FP8_TYPE.get(dtype)
    if qt is None:
        raise ValueError(f"dtype is one of {_FP8}")
    dev = x.get_device()
    shape, xt = x.shape, x.dtype
    if dev < 0:
        raise RuntimeError("quantize_blocks runs on the GPU only")
    if xt not in _FLOATS or not shape or shape[-1] == 0:
        raise ValueError(f"x is (..., K) in float16, bfloat16 or float32: got {tuple(shape)} in {xt}")
    if tile and (len(shape) != 2 or gate is not None):
        raise ValueError("tiles are taken of an (N, K) tensor, without a gate")
    if gate is not None and (gate.shape != shape or gate.dtype is not xt or gate.get_device() != dev):
        raise ValueError("gate has the shape, type and device of x")
    if _recorded():
        _refuse_grad("quantize_blocks", x, gate, *(output or ()))
    K, lead = shape[-1], shape[:-1]
    m = x.numel() // K
    kb = -(-K // BLOCK)
    if output is None:
        device = x.device
        q = _new(x, qt)
        s = torch.empty((_blocks(m), kb), dtype=torch.float32, device=device) if tile else _new_scales(lead, m, kb, device)
        ld = m
    else:
        q, s = output
        if q.shape != shape or q.dtype is not qt or not q.is_contiguous() or q.get_device() != dev:
            raise ValueError(f"output values are a contiguous {tuple(shape)} tensor in {qt} on x's device")
        want = (_blocks(m), kb) if tile else lead + (kb,)
        if s.shape != want or s.dtype is not torch.float32 or s.get_device() != dev or (tile and not s.is_contiguous()):
            raise ValueError(f"output scales are a {tuple(want)} tensor in float32 on x's device")
        ld = m if tile or m == 0 else _scale_ld(s, lead, m, kb)
    if m == 0:
        return q, s
    x, x_ld = _rows(x)
    a = BlockQuant(_QUANT_BYTES, _CODE[xt], _CODE[qt], tile, m, K, x_ld)
    a.s_ld = ld
    a.X, a.Q, a.S = x.data_ptr(), q.data_ptr(), s.data_ptr()
    if gate is not None:
        gate, a.gate_ld = _rows(gate)
        a.gate = gate.data_ptr()
    status = _library().wqaa_block_quantize(a, _raw_stream(dev))
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


def _check_norm_weight(w: torch.Tensor, name: str, D: int, t: torch.dtype, wt: torch.dtype, dev: int) -> None:
    d = w.dtype
    if w.shape != (D,) or d is not wt or (d is not t and d is not torch.float32) or not w.is_contiguous() or w.get_device() != dev:
        raise ValueError(f"{name} is a contiguous ({D},) tensor in {t} or float32 on x's device (weight and post_weight of one type): "
                         f"got {tuple(w.shape)} in {d} on {w.device}")


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
    dev = x.get_device()
    if dev < 0:
        raise RuntimeError("residual_norm runs on the GPU only")
    t, shape = x.dtype, x.shape
    if (t is not torch.float16 and t is not torch.bfloat16) or not shape or not 1 <= shape[-1] <= 32768:
        raise ValueError(f"x is (..., D) in float16 or bfloat16, D <= 32768: got {tuple(shape)} in {t}")
    D = shape[-1]
    st = wt = t
    if residual is not None:
        st = residual.dtype
        if residual.shape != shape or (st is not t and st is not torch.float32) or residual.get_device() != dev:
            raise ValueError(f"residual has x's shape and device, in {t} or float32: got {tuple(residual.shape)} in {st} on {residual.device}")
    if weight is not None:
        wt = weight.dtype
        _check_norm_weight(weight, "weight", D, t, wt, dev)
    if post_weight is not None:
        if weight is None:
            wt = post_weight.dtype
        _check_norm_weight(post_weight, "post_weight", D, t, wt, dev)
    if gate is not None and (gate.dtype is not t or gate.get_device() != dev):
        raise ValueError(f"gate is in {t}, on x's device")
    yt = t
    if quantize is not None:
        yt = _FP8_TYPE.get(quantize)
        if yt is None or weight is None:
            raise ValueError(f"quantize is one of {_FP8}, and goes with a weight")
    if not eps >= 0.0:
        raise ValueError("the norm's eps must be a non-negative number")
    if _recorded():
        _refuse_grad("residual_norm", x, residual, weight, post_weight, gate, *(output or ()))
    passes = residual is None and gate is None and post_weight is None and scale == 1.0     # h is x
    if passes and weight is None:
        raise ValueError("nothing to do: no residual, gate, post_weight or scale, and no weight")
    m = x.numel() // D
    kb = -(-D // BLOCK)
    lead = shape[:-1]
    h = y = s = None
    ld = m
    if output is not None:
        h, y, s = (tuple(output) + (None,) * 3)[:3]
        if h is not None and (h.shape != shape or h.dtype is not st or not h.is_contiguous() or h.get_device() != dev):
            raise ValueError(f"output h is a contiguous {tuple(shape)} tensor in {st} on x's device")
        if y is not None and (weight is None or y.shape != shape or y.dtype is not yt or not y.is_contiguous() or y.get_device() != dev):
            raise ValueError(f"output y goes with a weight and is a contiguous {tuple(shape)} tensor in {yt} on x's device")
        if s is not None:
            if quantize is None or s.shape != lead + (kb,) or s.dtype is not torch.float32 or s.get_device() != dev:
                raise ValueError(f"output scales go with quantize and are a {tuple(lead) + (kb,)} tensor in float32 on x's device")
            ld = _scale_ld(s, lead, m, kb) if m else m
    write_h = h is not None or not passes
    if h is None:
        h = x if passes else _new(x if residual is None else residual, st)
    if weight is None:
        result = (h, None)
    else:
        if y is None:
            y = _new(x, yt)
        if quantize is None:
            result = (h, y)
        else:
            if s is None:
                s = _new_scales(lead, m, kb, x.device)
            result = (h, (y, s))
    if m == 0:
        return result
    x, x_ld = _rows(x)
    a = ResidualNormArgs(_NORM_BYTES, _CODE[t], _CODE[st], _CODE[wt], -1 if quantize is None else _CODE[yt], eps, scale, residual_scale, m, D, x_ld)
    a.x = x.data_ptr()
    if residual is not None:
        residual, a.residual_ld = _rows(residual)
        a.residual = residual.data_ptr()
    if gate is not None:
        gate, a.gate_ld, a.gate_rows = _gate_rows(gate, h)
        a.gate = gate.data_ptr()
    if post_weight is not None:
        a.post_weight = post_weight.data_ptr()
    if write_h:
        a.stream = h.data_ptr()
    if weight is not None:
        a.weight, a.Y = weight.data_ptr(), y.data_ptr()
        if quantize is not None:
            a.S, a.s_ld = s.data_ptr(), ld
    status = _library().wqaa_residual_norm(a, _raw_stream(dev))
    if status != _lib.OK:
        _lib.check(status)
    return result


class BlockScaledLinear(torch.nn.Module):
    """A linear layer on 8-bit operands with a scale per block of 128: `BlockScaledLinear.from_linear(layer)`, or the buffers of a
    checkpoint that was quantised that way (`weight` (out, in) in `W_dtype`, `weight_scale` (ceil(out / 128), ceil(in / 128)) float32).

    forward(x): x (..., in) in float16, bfloat16 or float32 is quantised per row and block first; (values, scales), as
    `quantize_blocks` and `residual_norm(quantize=)` return them, is multiplied as it is."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, A_dtype: str = "e4m3_float8", W_dtype: str = "e4m3_float8",
                 out_dtype: str = "float16"):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.bitblas_matmul = BlockScaledMatmul(BlockScaledMatmulConfig(N=out_features, K=in_features, A_dtype=A_dtype, W_dtype=W_dtype,
                                                                        out_dtype=out_dtype, with_bias=bias))
        self.A_dtype, self.W_dtype, self.out_dtype = A_dtype, W_dtype, out_dtype
        self.register_buffer("weight", torch.zeros((out_features, in_features), dtype=torch_dtype(W_dtype)))
        self.register_buffer("weight_scale", torch.ones((_blocks(out_features), _blocks(in_features)), dtype=torch.float32))
        if bias:
            self.register_buffer("bias", torch.zeros(out_features, dtype=torch_dtype(out_dtype)))
        else:
            self.bias = None

    def _apply(self, fn, *args, **kw):
        """`.to()`, `.half()`, `.cuda()` and the like move the buffers and leave their types alone: those are the operator's, and a 16-bit scale or
        weight could not be turned back"""
        held = {name: t for name, t in self._buffers.items() if t is not None}
        super()._apply(fn, *args, **kw)
        for name, t in held.items():
            if self._buffers[name].dtype is not t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def load_float_weight(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> None:
        """Quantise a float weight into this layer's buffers, on the GPU the layer lives on."""
        if self.weight.device.type != "cuda":
            raise RuntimeError("load_float_weight quantises on the GPU: move the layer there first")
        if weight.shape != (self.out_features, self.in_features):
            raise ValueError(f"weight is ({self.out_features}, {self.in_features}): got {tuple(weight.shape)}")
        if (bias is not None) != (self.bias is not None):
            raise ValueError("the bias goes with a layer that has one, and only with it")
        if bias is not None and bias.shape != (self.out_features,):
            raise ValueError(f"bias is ({self.out_features},): got {tuple(bias.shape)}")
        w = weight.detach().to(self.weight.device)
        if w.dtype not in _FLOATS:
            w = w.float()
        quantize_blocks(w, self.W_dtype, tile=True, output=(self.weight, self.weight_scale))
        if bias is not None:
            self.bias.copy_(bias.detach())

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, A_dtype: str = "e4m3_float8", W_dtype: str = "e4m3_float8", out_dtype: Optional[str] = None):
        """a float `nn.Linear` on the GPU -> this layer; out_dtype: the linear's type where it is a 16-bit one, else float16"""
        if out_dtype is None:
            out_dtype = "bfloat16" if linear.weight.dtype is torch.bfloat16 else "float16"
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, A_dtype, W_dtype, out_dtype).to(linear.weight.device)
        layer.load_float_weight(linear.weight, linear.bias)
        return layer

    def forward(self, x, output: Optional[torch.Tensor] = None) -> torch.Tensor:
        q, s = x if isinstance(x, tuple) else quantize_blocks(x, self.A_dtype)
        return self.bitblas_matmul(q, self.weight, s, self.weight_scale, self.bias, output)


class BlockScaledGatedMLP(torch.nn.Module):
    """`down(silu(gate(x)) * up(x))` (+ residual) over block-scaled layers, gate and up as ONE product: three launches, or four with a float
    x, at any row count (`GatedMLP` is the same block over low-bit weights; integration/BitNet/modeling_bitnet.py:209-244).

    gate_up   `BlockScaledLinear(hidden, 2 * inner)`, gate's rows first; down `BlockScaledLinear(inner, hidden)`"""

    def __init__(self, gate_up: BlockScaledLinear, down: BlockScaledLinear):
        super().__init__()
        if gate_up.out_features != 2 * down.in_features:
            raise ValueError(f"gate_up gives {gate_up.out_features} features, down takes {down.in_features}: gate and up are one half each")
        self.gate_up, self.down = gate_up, down

    @classmethod
    def from_linears(cls, gate: torch.nn.Linear, up: torch.nn.Linear, down: torch.nn.Linear, **kw):
        if gate.weight.shape != up.weight.shape or (gate.bias is None) != (up.bias is None):
            raise ValueError("gate and up have one shape, and both a bias or none")
        both = torch.nn.Linear(gate.in_features, 2 * gate.out_features, bias=gate.bias is not None, device=gate.weight.device, dtype=gate.weight.dtype)
        with torch.no_grad():
            both.weight.copy_(torch.cat([gate.weight, up.weight]))
            if gate.bias is not None:
                both.bias.copy_(torch.cat([gate.bias, up.bias]))
        return cls(BlockScaledLinear.from_linear(both, **kw), BlockScaledLinear.from_linear(down, **kw))

    def forward(self, x, residual: Optional[torch.Tensor] = None, norm=None) -> torch.Tensor:
        """norm = (weight, eps): x is the hidden state in front of the MLP's norm.  residual: added to the result, as residual_norm does"""
        if norm is not None:
            x = residual_norm(x, None, norm[0], norm[1], quantize=self.gate_up.A_dtype)[1]
        both = self.gate_up(x)
        inner = self.down.in_features
        out = self.down(quantize_blocks(both[..., inner:], self.down.A_dtype, gate=both[..., :inner]))
        return out if residual is None else residual_norm(out, residual)[0]


class BlockScaledDecoderTail(torch.nn.Module):
    """The half of a decoder layer behind its attention, over block-scaled layers (`DecoderTail` is the same over low-bit weights):

        h   = x + post_attention(o_proj(attn))
        out = h + post_mlp(mlp(norm(h)))

    with the norm in front of the next block too where the caller has its weight: forward(...) -> (out, next_norm(out) or None), the latter
    quantised and ready for the next layer's projections.  post_attention / post_mlp: weights of norms behind the two blocks, or None."""

    def __init__(self, o_proj: BlockScaledLinear, mlp: BlockScaledGatedMLP, norm_weight: torch.Tensor, eps: float = 1e-6,
                 post_attention: Optional[torch.Tensor] = None, post_mlp: Optional[torch.Tensor] = None):
        super().__init__()
        self.o_proj, self.mlp = o_proj, mlp
        self.norm_weight, self.post_attention, self.post_mlp = norm_weight, post_attention, post_mlp
        self.eps = float(eps)

    def forward(self, attn, x: torch.Tensor, next_norm: Optional[torch.Tensor] = None):
        h, y = residual_norm(self.o_proj(attn), x, self.norm_weight, self.eps, post_weight=self.post_attention, quantize=self.mlp.gate_up.A_dtype)
        return residual_norm(self.mlp(y), h, next_norm, self.eps, post_weight=self.post_mlp,
                             quantize=None if next_norm is None else self.mlp.gate_up.A_dtype)


__all__ = ["BLOCK", "BlockScaledDecoderTail", "BlockScaledGatedMLP", "BlockScaledLinear", "BlockScaledMatmul", "BlockScaledMatmulConfig",
           "quantize_blocks", "residual_norm"]
