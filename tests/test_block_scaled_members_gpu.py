"""The block-scaled product, member by member: every pair of types with K whole and cut, what padding rows, columns and scales may not do, layouts,
streams and captured graphs.  Each case names the member it is for and fails if the call takes another.

Tolerances: test_block_scaled_gpu.check_product (16-bit rounding, the matrix unit's cut, float32 sums).  Everything else is compared bit for
bit: a sum runs over its own row and column only, in an order that the member and the sizes fix."""
import pytest
import torch

import bitblas_amd as bitblas
from test_block_scaled_gpu import LARGEST, T8, TO, check_product

pytestmark = pytest.mark.gpu

# name -> (M, N, K), (rows of a tile, columns, threads, K slices).  N ends inside a weight tile, M inside a tile; "cut" calls take K + 16
MEMBERS = {
    "stream 16 x 16, 8 waves": ((3, 300, 2048), (16, 16, 512, 1)),
    "stream 16 x 16, 16 waves": ((3, 300, 8192), (16, 16, 1024, 1)),
    "stream 16 x 32": ((9, 7300, 1024), (16, 32, 1024, 1)),
    "stream 16 x 64": ((12, 10300, 640), (16, 64, 512, 1)),
    "stream 32 x 16": ((100, 400, 640), (32, 16, 512, 1)),
    "stream 32 x 32": ((30, 7170, 384), (32, 32, 512, 1)),
    "stream 32 x 64": ((20, 10250, 1024), (32, 64, 512, 1)),
    "tile 64, 4 waves": ((318, 7600, 1280), (64, 128, 256, 1)),
    "tile 64, 8 waves": ((190, 8010, 1408), (64, 128, 512, 1)),
    "tile 64, 8 waves, one block": ((190, 8010, 128), (64, 128, 512, 1)),
    "tile 64, 4 waves, slices": ((40, 700, 6400), (64, 128, 256, 8)),
    "tile 64, 8 waves, slices": ((250, 4300, 2048), (64, 128, 512, 2)),
    "tile 128, 4 waves": ((513, 9000, 1024), (128, 128, 256, 1)),
    "tile 128, 8 waves": ((129, 12810, 1152), (128, 128, 512, 1)),
    "ping-pong": ((2050, 5000, 1152), (256, 256, 512, 1)),
    "ping-pong, one round in slices": ((130, 16700, 7168), (256, 256, 512, 3)),
    "ping-pong, a last round in slices": ((500, 33100, 1920), (256, 256, 512, 4)),
}
SLICED = [name for name in MEMBERS if "slices" in name]
members = pytest.mark.parametrize("name", list(MEMBERS))
cuts = pytest.mark.parametrize("cut", [False, True], ids=["whole", "cut"])


def operator(name, cut=False, **kw):
    """(the operator, M), checked to be the member that the name says"""
    (M, N, K), (bm, bn, threads, split) = MEMBERS[name]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=K + 16 * cut, **kw))
    plan = op.plan(M)
    assert (plan["block_m"], plan["block_n"], plan["threads"], plan["split_k"]) == (bm, bn, threads, split), plan["name"]
    return op, M


def quantised(x, dtype, rows):
    """8-bit values and scales of x in blocks of `rows` x 128, on the device"""
    M, K = x.shape
    mb, kb = -(-M // rows), -(-K // 128)
    p = torch.nn.functional.pad(x, (0, kb * 128 - K, 0, mb * rows - M)).view(mb, rows, kb, 128)
    s = p.abs().amax((1, 3)).clamp_min(2.0 ** -40) / LARGEST[dtype]
    return (p / s[:, None, :, None]).to(T8[dtype]).view(mb * rows, kb * 128)[:M, :K].contiguous(), s


def operands(op, M, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    c = op.config
    A, sa = quantised(torch.randn(M, c.K, generator=g, device="cuda") * torch.exp(torch.randn(c.K, generator=g, device="cuda")), c.A_dtype, 1)
    W, sw = quantised(torch.randn(c.N, c.K, generator=g, device="cuda") * 0.05, c.W_dtype, 128)
    bias = torch.randn(c.N, generator=g, device="cuda").to(TO[c.out_dtype]) if c.with_bias else None
    return A, W, sa, sw, bias


def bits(t):
    return t.contiguous().view(torch.int16)


@members
@cuts
@pytest.mark.parametrize("a", list(T8))
@pytest.mark.parametrize("w", list(T8))
def test_types(name, cut, a, w):
    op, M = operator(name, cut, A_dtype=a, W_dtype=w, out_dtype="float16" if a == w else "bfloat16", with_bias=(a == "e4m3_float8") != cut)
    args = operands(op, M, len(name) + cut)
    C = op(*args)
    check_product(C, *args)
    assert torch.equal(bits(op(*args)), bits(C))


@members
@cuts
def test_rows_and_columns_stay_apart(name, cut):
    """values and scales that are not finite, in the first and last rows, columns and k among them, reach their own row, column or weight tile; all
    else keeps its bits"""
    op, M = operator(name, cut, A_dtype="e5m2_float8", out_dtype="bfloat16")
    A, W, sa, sw, _ = operands(op, M, 7)
    K, N, kb, nb = op.K, op.N, sa.shape[1], sw.shape[0]
    clean = op(A, W, sa, sw)
    a, w, sa, sw = A.view(torch.uint8).clone(), W.view(torch.uint8).clone(), sa.clone(), sw.clone()
    rows, columns = torch.zeros(M, dtype=torch.bool, device="cuda"), torch.zeros(N, dtype=torch.bool, device="cuda")
    a[M - 1, K - 1] = 0x7C                                                # infinity
    a[M // 2, 5] = 0x7F                                                   # NaN
    w[N - 1, K - 1] = w[1, 0] = 0x7F                                      # NaN
    sa[0, kb - 1] = float("nan")
    sw[nb // 2, kb - 1], sw[nb - 2, 0] = float("nan"), float("inf")
    rows[[0, M // 2, M - 1]] = True
    columns[[1, N - 1]] = True
    for t in (nb // 2, nb - 2):
        columns[t * 128:t * 128 + 128] = True
    C = op(a.view(A.dtype), w.view(W.dtype), sa, sw)
    assert not C[rows].isfinite().any() and not C[:, columns].isfinite().any()
    if M > 3:
        assert torch.equal(bits(C[~rows][:, ~columns]), bits(clean[~rows][:, ~columns]))
    sw = sw.clone()
    sw[nb - 1] = float("nan")                                             # the tile that N ends in, all of it
    columns[(nb - 1) * 128:] = True
    C = op(A, W, torch.where(sa.isfinite(), sa, 1.0), sw)
    assert not C[:, (nb - 1) * 128:].isfinite().any()
    assert torch.equal(bits(C[1:][:, ~columns]), bits(clean[1:][:, ~columns]))


@members
@cuts
def test_scales_of_every_size(name, cut):
    """row scales from 2^-100 to 2^59 next to each other, and scales of 0, which count nothing: a row and a tile of nothing but them are exact zeros"""
    op, M = operator(name, cut, out_dtype="bfloat16")
    A, W, sa, sw, _ = operands(op, M, 11)
    g = torch.Generator("cuda").manual_seed(5)
    sa = sa * torch.exp2(torch.randint(-100, 60, sa.shape, generator=g, device="cuda").float())
    sa[0, 0] = sw[0, -1] = 0.0
    sa[M - 1], sw[1] = 0.0, 0.0
    C = op(A, W, sa, sw)
    assert (C[M - 1] == 0).all() and (C[:, 128:256] == 0).all()
    check_product(C, A, W, sa, sw)


@members
@cuts
def test_layouts(name, cut):
    """row scales with their blocks apart and NaN between, on any 4-byte boundary, and row by row; rows of A apart and off their alignment; leading
    dimensions; an output between others': the same bits, and nothing else written"""
    op, M = operator(name, cut, out_dtype="float16", with_bias=True)
    A, W, sa, sw, bias = operands(op, M, 13)
    want = bits(op(A, W, sa, sw, bias))
    kb = sa.shape[1]
    for before, after in ((0, 3), (1, 0), (2, 5)):
        room = torch.full((kb, before + M + after), float("nan"), device="cuda")
        room[:, before:before + M] = sa.t()
        assert torch.equal(bits(op(A, W, room[:, before:before + M].t(), sw, bias)), want)
    wide = torch.zeros(M, op.K + 21, dtype=torch.uint8, device="cuda")
    wide[:, 5:5 + op.K] = A.view(torch.uint8)
    assert torch.equal(bits(op(wide[:, 5:5 + op.K].view(A.dtype), W, sa, sw, bias)), want)
    room = torch.full((M * op.N + 40,), 7.0, dtype=torch.float16, device="cuda")
    out = room[13:13 + M * op.N].view(1, M, op.N)
    assert op(A[None], W, sa[None], sw, bias, out) is out
    assert torch.equal(bits(out[0]), want) and bool((room[:13] == 7).all()) and bool((room[13 + M * op.N:] == 7).all())


@pytest.mark.parametrize("name", SLICED)
def test_slices_on_two_streams(name):
    """partial tiles of calls that run at once are each call's own"""
    op, M = operator(name, out_dtype="bfloat16")
    sets = [operands(op, M, 20 + i)[:4] for i in range(2)]
    want = [bits(op(*s)) for s in sets]
    assert op.workspace_bytes(M) > 0 and not torch.equal(want[0], want[1])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(op(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(bits(C), want[i]) for i in range(2) for C in got[i])


@pytest.mark.parametrize("name", SLICED)
def test_slices_captured(name):
    """two graphs, each of two products that leave partial tiles, replayed on inputs that change, with the same calls made eagerly between"""
    op, M = operator(name, out_dtype="bfloat16")
    A, W, sa, sw, _ = operands(op, M, 30)
    B, _, sb, _, _ = operands(op, M, 31)
    inputs = [(A, sa), (B, sb)]
    want = [bits(op(x, W, s, sw)) for x, s in inputs]
    held = [[t.clone() for t in inputs[i]] for i in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [op(held[i][0], W, held[i][1], sw), op(held[1 - i][0], W, held[1 - i][1], sw)]
        graphs.append((graph, out))
    for step in range(6):
        swap = step // 2 % 2                                              # which input the held tensors hold
        for i in range(2):
            for to, now in zip(held[i], inputs[i ^ swap]):
                to.copy_(now)
        graph, out = graphs[step % 2]
        graph.replay()
        eager = bits(op(held[0][0], W, held[0][1], sw))
        torch.cuda.synchronize()
        i = step % 2
        assert torch.equal(bits(out[0]), want[i ^ swap]) and torch.equal(bits(out[1]), want[1 - i ^ swap]) and torch.equal(eager, want[swap])


# M, N, the member, and the k-blocks that its waves take in a turn of their loop
LOOPS = {"16 x 16, 8 waves": (3, 300, (16, 16, 512), 32), "16 x 16, 16 waves": (3, 300, (16, 16, 1024), 16), "16 x 32": (9, 7300, (16, 32, 1024), 16),
         "16 x 64": (12, 10300, (16, 64, 512), 8), "32 x 16": (30, 400, (32, 16, 512), 8), "32 x 32": (30, 7170, (32, 32, 512), 8),
         "32 x 64": (20, 10250, (32, 64, 512), 8)}
# the two of 16 x 16 share their calls: 16 waves from 64 blocks on
TURNS = [(name, turns, extra) for name in LOOPS for turns in (1, 2, 3, 4, 5, 6) for extra in (-128, 0, 144)
         if "16 x 16" not in name or (turns * LOOPS[name][3] * 128 + extra > 63 * 128) == ("16 waves" in name)]


@pytest.mark.parametrize("name, turns, extra", TURNS)
def test_turns_of_the_streaming_loop(name, turns, extra):
    """K in so many turns of a wave's loop: both ways out of it, waves with a turn less, and a cut block behind"""
    M, N, member, blocks = LOOPS[name]
    op = bitblas.BlockScaledMatmul(bitblas.BlockScaledMatmulConfig(N=N, K=turns * blocks * 128 + extra, out_dtype="bfloat16"))
    plan = op.plan(M)
    assert (plan["block_m"], plan["block_n"], plan["threads"]) == member, plan["name"]
    args = operands(op, M, turns)
    check_product(op(*args), *args)
