"""The operators of the block-scaled 8-bit path, as they are measured: plain forms, and the calls a user makes.

The path is the decoder layer's matmuls with both operands in 8-bit floating point, each block of 128 consecutive k with a
float32 scale of its own: activations per row, weights per 128 x 128 tile.

  product    C[m, n] = sum_b sa[m, b] sw[n // 128, b] sum_{k in block b} a[m, k] w[n, k]  (+ bias[n])
  quantise   s = max(max|x|, 2^-40) / 448 (e5m2: / 57344) over a block, q = the float32 quotient x / s rounded to the 8-bit
             type, ties to even; with a gate: x = silu(gate) * up
  norm       z = x                     or  x rsqrt(mean x^2 + eps) post_weight
             h = residual_scale residual + scale gate z                   (returned in the residual's type)
             y = h rsqrt(mean h^2 + eps) weight                           (of h before it is rounded; in x's type, or quantised in blocks)
"""
import math

import torch

own = False

FLOOR = 2.0 ** -40
EPS = 1e-5
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
NAME = {"e4m3": "e4m3_float8", "e5m2": "e5m2_float8", "f16": "float16", "bf16": "bfloat16", "f32": "float32"}
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}


def listed():
    def product(name, M, N, K, out, a="e4m3", w="e4m3", bias=False):
        return {"name": name, "op": "product", "M": M, "N": N, "K": K, "a": a, "w": w, "out": out, "bias": bias}

    def quantise(name, M, K, x, tile=False, gated=False, q="e4m3"):
        return {"name": name, "op": "quantise", "M": M, "K": K, "x": x, "q": q, "tile": tile, "gated": gated}

    def norm(name, B, S, D, x, residual, post, gate, q):
        return {"name": name, "op": "norm", "B": B, "S": S, "D": D, "x": x, "residual": residual, "post": post, "gate": gate, "q": q,
                "scale": 0.5 if post else 1.0, "residual_scale": 1.0}

    return [
        product("one token, square", 1, 4096, 4096, "f16"),                       # a decode step's attention projection: latency
        product("one token, wide", 1, 28672, 8192, "bf16"),                       # a decode step's gate or up projection: one read of W
        product("16 tokens, long k", 16, 8192, 28672, "bf16"),                    # a decode batch's down projection
        product("odd sizes", 77, 1001, 1040, "bf16", bias=True),                  # a small head: N no multiple of 4, a part of a block in K
        product("ragged batch", 333, 11008, 4096, "f16", a="e5m2", bias=True),    # sequences packed without padding; wide-range activations
        product("prefill", 4096, 28672, 8192, "bf16"),                            # a prompt through the gate or up projection
        quantise("decode gate", 16, 28672, "bf16", gated=True),                   # silu(gate) * up in front of the down projection, decode
        quantise("prefill rows", 4096, 8192, "bf16"),                             # a prompt's activations in front of a projection
        quantise("weight tiles", 28672, 8192, "bf16", tile=True),                 # a checkpoint's weight as it is loaded
        norm("one token", 1, 1, 8192, "bf16", "bf16", False, "none", "e4m3"),     # residual add and norm between two blocks, decode
        norm("ragged rows", 1, 333, 4096, "f16", "f16", False, "none", "none"),   # the same in float16 for a packed batch
        norm("prefill, both norms", 4, 1024, 8192, "bf16", "f32", True, "sequence", "e4m3"),  # norms on both sides, a gate per sequence, a float32 stream
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "quantise", "norm"])
    if op == "product":
        while True:
            M, N, K = _log(rng, 1, 4096), _log(rng, 64, 28672), 16 * _log(rng, 8, 1792)
            if M * N * K <= 4096 * 28672 * 8192 and N * K <= 28672 * 8192:
                break
        return {"op": op, "M": M, "N": N, "K": K, "a": rng.choice(["e4m3", "e4m3", "e5m2"]), "w": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "out": rng.choice(["f16", "bf16"]), "bias": rng.random() < 0.5}
    if op == "quantise":
        M, K = _log(rng, 1, 4096), _log(rng, 64, 28672)
        tile = rng.random() < 0.3
        return {"op": op, "M": M, "K": K, "x": rng.choice(["f16", "bf16", "f32"]), "q": rng.choice(["e4m3", "e4m3", "e5m2"]), "tile": tile,
                "gated": not tile and rng.random() < 0.5}
    D = _log(rng, 64, 16384)
    D = D if rng.random() < 0.4 else max(64, D // 16 * 16)
    B, S = rng.randint(1, 8), _log(rng, 1, 512)
    return {"op": op, "B": B, "S": S, "D": D, "x": rng.choice(["f16", "bf16"]), "residual": rng.choice(["same", "f32"]), "post": rng.random() < 0.5,
            "gate": rng.choice(["none", "channel", "sequence", "full"]), "q": rng.choice(["none", "e4m3", "e5m2"]), "scale": 0.5,
            "residual_scale": rng.choice([1.0, 0.25])}


def _stream(case):
    """the type of the residual stream"""
    return case["x"] if case["residual"] == "same" else case["residual"]


def _blocks(n):
    return -(-n // 128)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op, s = case["op"], {"case": case}
    if op == "product":
        M, N, K = case["M"], case["N"], case["K"]
        # activations have channels that stand out; weights do not
        channel = torch.exp(0.7 * normal(K))
        s["A"], s["sa"] = _plain_quantise(normal(M, K) * channel, case["a"], False)
        s["W"], s["sw"] = _plain_quantise(0.02 * normal(N, K), case["w"], True)
        s["sa"] = s["sa"].t().contiguous().t()       # as the quantiser stores row scales: the rows of one block side by side
        s["bias"] = normal(N).to(FLOAT[case["out"]]) if case["bias"] else None
        s["out"] = torch.empty(M, N, dtype=FLOAT[case["out"]], device="cuda")
        if own:
            import bitblas_amd as bitblas
            s["op"] = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(
                N=N, K=K, A_dtype=NAME[case["a"]], W_dtype=NAME[case["w"]], out_dtype=NAME[case["out"]], with_bias=case["bias"]))
    elif op == "quantise":
        M, K, t = case["M"], case["K"], FLOAT[case["x"]]
        if case["gated"]:
            both = normal(M, 2 * K).to(t)            # one projection's output: gate and up side by side
            s["gate"], s["x"] = both[:, :K], both[:, K:]
        else:
            s["x"] = (normal(M, K) * torch.exp(0.7 * normal(K))).to(t)
    else:
        B, S, D, t = case["B"], case["S"], case["D"], FLOAT[case["x"]]
        s["x"] = normal(B, S, D).to(t)
        s["residual"] = (4.0 * normal(B, S, D)).to(FLOAT[_stream(case)])
        s["weight"] = (1.0 + 0.1 * normal(D)).to(t)
        s["post"] = (1.0 + 0.1 * normal(D)).to(t) if case["post"] else None
        shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "full": (B, S, D)}[case["gate"]]
        s["gate"] = normal(*shape).to(t) if shape else None
    return s


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "product":
        a = s["A"].float() * s["sa"].repeat_interleave(128, 1)[:, :case["K"]]
        w = s["W"].float() * s["sw"].repeat_interleave(128, 0)[:case["N"]].repeat_interleave(128, 1)[:, :case["K"]]
        c = a @ w.t()
        if s["bias"] is not None:
            c = c + s["bias"].float()
        return c.to(FLOAT[case["out"]])
    if case["op"] == "quantise":
        x = s["x"].float()
        if case["gated"]:
            gate = s["gate"].float()
            x = gate / (1.0 + torch.exp(-gate)) * x
        return _plain_quantise(x, case["q"], case["tile"])
    z = s["x"].float()
    if s["post"] is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        z = z * s["gate"].float()
    h = case["residual_scale"] * s["residual"].float() + case["scale"] * z
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    h = h.to(FLOAT[_stream(case)])
    return (h, y.to(FLOAT[case["x"]])) if case["q"] == "none" else (h,) + _plain_quantise(y, case["q"], False)


def _run_own(s):
    import bitblas_amd as bitblas
    case = s["case"]
    if case["op"] == "product":
        return s["op"](s["A"], s["W"], s["sa"], s["sw"], s["bias"], output=s["out"])
    if case["op"] == "quantise":
        return bitblas.quantize_blocks(s["x"], NAME[case["q"]], tile=case["tile"], gate=s.get("gate"))
    h, y = bitblas.residual_norm(s["x"], s["residual"], s["weight"], EPS, post_weight=s["post"], gate=s["gate"], scale=case["scale"],
                                 residual_scale=case["residual_scale"], quantize=None if case["q"] == "none" else NAME[case["q"]])
    return (h, y) if case["q"] == "none" else (h,) + tuple(y)


def _plain_quantise(x, q, tile):
    """(values in the 8-bit type, scales) of x in float32: blocks of 128 along the last axis, of each row or of 128 rows"""
    shape, K = x.shape, x.shape[-1]
    x = x.reshape(-1, K)
    M, kb = x.shape[0], _blocks(K)
    rows = 128 if tile else 1
    mb = -(-M // rows)
    x = torch.nn.functional.pad(x, (0, kb * 128 - K, 0, mb * rows - M)).view(mb, rows, kb, 128)
    s = x.abs().amax((1, 3)).clamp_min(FLOOR) / LARGEST[q]
    v = (x / s[:, None, :, None]).to(FP8[q]).view(mb * rows, kb * 128)[:M, :K].contiguous()
    return v.view(shape), s if tile else s.view(shape[:-1] + (kb,))


def work(case):
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 4 * (M + _blocks(N)) * _blocks(K) + (M + (1 if case["bias"] else 0)) * N * SIZE[case["out"]], "flops": 2 * M * N * K}
    if case["op"] == "quantise":
        M, K = case["M"], case["K"]
        scales = (_blocks(M) if case["tile"] else M) * _blocks(K)
        return {"bytes": M * K * (SIZE[case["x"]] * (2 if case["gated"] else 1) + 1) + 4 * scales, "flops": M * K * (8 if case["gated"] else 3)}
    R, D = case["B"] * case["S"], case["D"]
    gate = {"none": 0, "channel": D, "sequence": case["B"] * D, "full": R * D}[case["gate"]]
    n = R * D * (SIZE[case["x"]] + 2 * SIZE[_stream(case)]) + SIZE[case["x"]] * (gate + D * (2 if case["post"] else 1))
    n += R * D * SIZE[case["x"]] if case["q"] == "none" else R * (D + 4 * _blocks(D))
    return {"bytes": n, "flops": R * D * (12 if case["post"] else 8)}


def _exact_round(v, q):
    """the value of the 8-bit type nearest to the float32 quotient, ties to the even one; v in 64 bits and within the type's range"""
    v = v.float().double()
    bits, least = (3, -6) if q == "e4m3" else (2, -14)
    e = (torch.frexp(v).exponent - 1).clamp_min(least).double()
    step = torch.exp2(e - bits)
    return torch.round(v / step) * step


def _exact_blocks(x, q):
    """(rounded values, scales) of rows in 64 bits, block by block; the scale is the float32 nearest to amax / largest"""
    values, scales = torch.empty_like(x), []
    for k in range(0, x.shape[-1], 128):
        part = x[..., k:k + 128]
        s = (part.abs().amax(-1).clamp_min(FLOOR) / LARGEST[q]).float().double()
        scales.append(s)
        values[..., k:k + 128] = _exact_round(part / s[..., None], q)
    return values, torch.stack(scales, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        c = torch.zeros(M, N, dtype=torch.float64, device="cuda")
        tile = torch.arange(N, device="cuda") // 128
        for b in range(_blocks(K)):
            part = s["A"][:, 128 * b:128 * b + 128].double() @ s["W"][:, 128 * b:128 * b + 128].double().t()
            part *= s["sa"][:, b, None].double()
            part *= s["sw"][tile, b].double()
            c += part
        return c if s["bias"] is None else c + s["bias"].double()
    if case["op"] == "quantise":
        x = s["x"].double()
        if case["gated"]:
            x = x * s["gate"].double() * torch.sigmoid(s["gate"].double())
        if not case["tile"]:
            return _exact_blocks(x, case["q"])
        values, scales = [], []
        for m in range(0, case["M"], 128):           # a band of 128 rows: every tile of it is one row of its blocks
            band = x[m:m + 128]
            cut = _blocks(case["K"]) * 128
            wide = torch.zeros(band.shape[0], cut, dtype=torch.float64, device="cuda")
            wide[:, :case["K"]] = band
            wide = wide.view(-1, cut // 128, 128).transpose(0, 1)
            top = (wide.abs().amax((1, 2)).clamp_min(FLOOR) / LARGEST[case["q"]]).float().double()
            v = _exact_round(wide / top[:, None, None], case["q"])
            values.append(v.transpose(0, 1).reshape(band.shape[0], cut)[:, :case["K"]])
            scales.append(top)
        return torch.cat(values), torch.stack(scales)
    z = s["x"].double()
    if s["post"] is not None:
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS) * s["post"].double()
    if s["gate"] is not None:
        z = z * s["gate"].double()
    h = case["residual_scale"] * s["residual"].double() + case["scale"] * z
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
    return (h, y) if case["q"] == "none" else (h,) + _exact_blocks(y, case["q"])
