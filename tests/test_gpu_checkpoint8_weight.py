"""The weight gradient from inputs kept in 8 bits: every form of its kernel, by what the plan of a size says, against 64 bits.

Tolerances: the tensor cores add 16 rows at a time and cut the sum off (2 U of what is added up); chains of at most 2,560 rows (fp16: 1,152) are
added rounded to nearest (U each), and so are the pieces of the rows."""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24
CHAIN = {F16: 1152, BF16: 2560}

# rows, n, k -> columns of gy per tile on 148 SMs: one CTA, a pair, a pair with two accumulators per CTA.  Remainders of the last
# stage (64 rows), of n and of k; one tile and several
FORMS = [((70001, 64, 64), 128), ((9000, 384, 640), 128), ((20000, 256, 256), 256), ((22725, 200, 671), 256), ((33646, 1985, 10), 512),
         ((20994, 1916, 432), 512), ((49844, 1197, 690), 512)]


@pytest.fixture(scope="module")
def c8(native):
    from beatsaberrl_b200 import checkpoint8
    return checkpoint8


@pytest.fixture(autouse=True)
def no_wait_ran_out(native):
    yield
    native.check(native.lib.bsrl_device_status())


def plan_of(native, rows, n, k):
    """(columns of gy per tile, columns of x per tile, 64-row stages of a piece of the rows)"""
    p = (C.c_int32 * 3)()
    native.check(native.lib.bsrl_linear8_wgrad_plan(rows, n, k, p))
    return p[0], p[1], math.ceil(rows / 64) // p[2]


def operands(c8, rows, n, k, dtype, kind):
    g = torch.Generator(device="cuda").manual_seed(rows + n + k)
    kept = c8.pack8(torch.randn(rows, k, generator=g, device="cuda").to(dtype), kind)
    return torch.randn(rows, n, generator=g, device="cuda").to(dtype), kept


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape,tile_n", FORMS)
def test_every_form(native, c8, shape, tile_n, dtype, kind):
    rows, n, k = shape
    form, _, stages = plan_of(native, rows, n, k)
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert form == tile_n
    gy, kept = operands(c8, rows, n, k, dtype, kind)
    gw, gb = c8.linear8_weight_grad(gy, kept)
    x, g = kept.expand().double(), gy.double()
    chains = math.ceil((stages + 1) * 64 / CHAIN[dtype]) + 1        # the first one of a piece is shorter
    pieces = math.ceil(rows / 64 / stages)
    most = g.abs().t() @ x.abs()
    assert ((gw.double() - g.t() @ x).abs() <= most * (CHAIN[dtype] / 16 * 2 + chains + pieces) * U).all()
    # a lane adds at most every fourth row of its piece, and there are at most 12 partial sums per piece
    assert ((gb.double() - g.sum(0)).abs() <= g.abs().sum(0) * ((stages + 1) * 16 + 12 * pieces) * U).all()
    again, none = c8.linear8_weight_grad(gy, kept, bias=False)
    assert none is None and torch.equal(again, gw)
    a, b = c8.linear8_weight_grad(torch.cat([gy[:, :1], gy], 1)[:, 1:], kept)       # rows that have to be copied
    assert torch.equal(a, gw) and torch.equal(b, gb)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", [(22725, 200, 671), (475136, 128, 128), (49844, 1197, 690), (475136, 1024, 256)])
def test_long_pieces_stay_near_the_64_bit_sums(native, c8, shape, dtype, kind):
    """What drains between chains are for.  A running sum S kept to 25 bits loses half of its last place per step on average, 0.36 x 2^-24 |S|
    (a number's last place is 0.72 x 2^-24 of it on average), always towards zero.  Over a chain of M products of 16 rows of independent
    numbers S grows with the square root of the rows, so that the losses add up to M / sqrt(3) times that of the chain's sum, and
    as much in relation of the sum of many chains: 1.24e-8 M.  fp16, M = 72: 8.9e-7, and 2e-7 of sums rounded to nearest across it: 9.1e-7.  Chains of
    26 stages (M = 104) are past the bound where a piece holds many.  bf16's products have fewer bits, of which less is cut off: its chains are longer, the bound is the same."""
    rows, n, k = shape
    assert plan_of(native, rows, n, k)[2] > 26                  # stages of a piece: well past the 18 of a chain of fp16
    gy, kept = operands(c8, rows, n, k, dtype, kind)
    want = gy.double().t() @ kept.expand().double()
    gw, _ = c8.linear8_weight_grad(gy, kept)
    assert float((gw.double() - want).norm() / want.norm()) < 1.05e-6


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("x_dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_activations_of_another_type(c8, dtype, x_dtype, kind):
    """The product is that of the checkpoint expanded to the gradient's type: exact in range; an fp16 gradient takes what lies past fp16 as infinity, in
    its own column only, and what lies below its smallest step as zero."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rows, n, k = 300, 40, 96
    x, gy = torch.randn(rows, k, generator=g, device="cuda"), torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    wide = x_dtype != F16
    if wide:
        x[7, 3] = 1e5                                   # past fp16; its neighbours in the block lose all but a step of 512 or 2
        x[:, 32:64] = 1e-9                              # below fp16's smallest step
    kept = c8.pack8(x.to(x_dtype), kind)
    gw, gb = c8.linear8_weight_grad(gy, kept)
    xv = kept.expand(dtype)
    if dtype == BF16:
        assert torch.equal(xv.double(), kept.expand(torch.float32).double())
    bad = torch.isinf(xv).any(0)
    assert bad.nonzero().flatten().tolist() == ([3] if wide and dtype == F16 else [])
    assert (gw[:, bad].isfinite() == 0).all() and gw[:, ~bad].isfinite().all()
    if wide:
        assert (gw[:, 32:64] == 0).all() == (dtype == F16)
    a, b = gy.double().t(), torch.where(bad, 0.0, xv.double())
    # truncated once per 16 rows (2 U), then at most one sum per 64-row stage and piece
    assert ((gw.double() - a @ b).abs()[:, ~bad] <= ((a.abs() @ b.abs()) * (rows / 16 * 2 + rows / 64 + 8) * U)[:, ~bad]).all()
    assert ((gb.double() - gy.double().sum(0)).abs() <= gy.double().abs().sum(0) * rows * U).all()


def test_large_forms_at_once_and_replayed(c8):
    """Calls of the form with two accumulators on two streams at the same time, and between a captured call's replays: none disturbs another."""
    shapes = [(33646, 1985, 10), (20994, 1916, 432)]
    ins = [operands(c8, *s, F16, "int8") for s in shapes]
    want = [c8.linear8_weight_grad(*i) for i in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[j] = c8.linear8_weight_grad(*ins[j])
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert all(torch.equal(p, q) for p, q in zip(out, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        held = c8.linear8_weight_grad(*ins[1])
    for _ in range(3):
        graph.replay()
        other = c8.linear8_weight_grad(*ins[0])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want[1])) and all(torch.equal(p, q) for p, q in zip(other, want[0]))
    for t in ins[1]:
        (t if torch.is_tensor(t) else t.codes).zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert not held[0].any() and not held[1].any()
