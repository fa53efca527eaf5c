"""Training operators that keep their inputs in 8 bits, against their definitions in 64 bits.

Tolerances count roundings: a result of type t is off by at most half a step, ``finfo(t).eps / 2`` of its value (half of the smallest
step near zero); fp32 arithmetic ahead of it by 2^-24 of what it adds or multiplies, per operation."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
SHAPES = [(1, 1), (1, 32), (3, 33), (2, 8), (29, 256), (7, 1001), (5, 630), (130, 40), (4, 4096), (300, 24), (1, 8192)]


@pytest.fixture(scope="module")
def c8(native):
    from beatsaberrl_b200 import checkpoint8
    return checkpoint8


@pytest.fixture(autouse=True)
def no_wait_ran_out(native):
    yield
    native.check(native.lib.bsrl_device_status())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, g, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def layouts(rows, d, dtype, g, scale=1.0):
    """The same kind of rows as they come: dense, as a slice of wider rows, from an element that no vector starts at."""
    yield "dense", randn(rows, d, g=g, dtype=dtype, scale=scale)
    yield "pitch", randn(rows, d + 24, g=g, dtype=dtype, scale=scale)[:, 8:8 + d]
    yield "odd", randn(rows, d + 5, g=g, dtype=dtype, scale=scale)[:, 1:1 + d]
    flat = randn(rows * d + 3, g=g, dtype=dtype, scale=scale)
    yield "shifted", flat[3:].view(rows, d)


def two(e):
    """2^e exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def to_e4m3(t):
    """The nearest numbers of four significant bits, down to steps of 2^-9."""
    _, e = torch.frexp(t)
    step = two((e - 4).clamp(min=-9))
    return torch.round(t / step) * step


def ref8(x, kind):
    """values, codes, exponents of x (rows, d) by the format's definition, in 64 bits."""
    rows, d = x.shape
    n = -(-d // 32)
    v = torch.zeros(rows, n * 32, dtype=torch.float64, device=x.device)
    v[:, :d] = x.double()
    v = v.view(rows, n, 32)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    v = torch.where(bad, 0.0, v)
    big = v.abs().amax(-1, keepdim=True)
    top = 15 if x.dtype == F16 else 127
    limit, up, grid = (127, 6, torch.round) if kind == "int8" else (240, 7, to_e4m3)
    _, e = torch.frexp(big)
    e = e - 1 - up
    grown = torch.where(grid(big * two(-e)) > limit, e + 1, e)
    e = torch.minimum(grown, torch.full_like(e, top - up))
    zero = (big == 0) | (e < -126)
    e = torch.where(zero, -127, e)
    q = torch.where(zero, 0.0, grid(v * two(-e)).clamp(-limit, limit))
    values = torch.where(bad, math.nan, q * two(e)).reshape(rows, n * 32)[:, :d]
    codes = q.to(torch.int8).view(torch.uint8) if kind == "int8" else q.to(torch.float8_e4m3fn).view(torch.uint8)
    return values, codes.reshape(rows, n * 32), torch.where(bad, 255, e + 127).to(torch.uint8).squeeze(-1)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=-7e300), torch.nan_to_num(b.double(), nan=-7e300))


def magnitudes(a, kind):
    """Codes without e4m3's sign of zero (minus zero has one, the reference's arithmetic may lose it)."""
    return torch.where(a == 128, 0, a) if kind == "e4m3" else a


# ---------------------------------------------------------------- the format
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_pack_and_expand(c8, rows, d, dtype, kind):
    for name, x in layouts(rows, d, dtype, gen(rows + d), 3.0):
        kept = c8.pack8(x, kind)
        values, codes, exps = ref8(x, kind)
        assert torch.equal(kept.exps, exps), name
        assert torch.equal(magnitudes(kept.codes, kind), magnitudes(codes, kind)), name
        assert same(kept.expand(), values.to(dtype)), name
        assert same(kept.expand(F32), values.float()) and same(kept.expand(BF16), values.to(BF16)), name
        assert kept.nbytes == kept.codes.numel() + kept.exps.numel() and kept.shape == (rows, d)
        again = c8.Checkpoint8(kept.codes, kept.exps, kind, x.shape, dtype)
        assert same(again.expand(), kept.expand())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_values_at_the_borders(c8, dtype, kind):
    """Ties, codes that would round past the range, the type's largest and smallest numbers, zeros, and what is not finite."""
    f = torch.finfo(dtype)
    rows = [[f.max, -f.max, 1.0], [f.max * 0.996, 1.0, -2.0], [-f.max * 0.98, f.max / 3, 0.0], [127.5, 126.5, -0.5], [-127.5, 1.5, 2.5], [127.4, -127.49, 0.5],
            [248.0, 247.0, -17.0], [-249.0, 17.0, 1.0625], [f.tiny, 0.0, -f.tiny], [f.smallest_normal / 4, 0.0, 0.0], [0.0, -0.0, 0.0],
            [math.inf, 1.0, 2.0], [1.0, math.nan, 2.0], [-math.inf, math.nan, 0.0], [2.0 ** -120, 2.0 ** -121, 0.0], [2.0 ** -119, 2.0 ** -127, 0.0]]
    x = torch.zeros(len(rows), 70, device="cuda", dtype=dtype)
    x[:, 33:36] = torch.tensor(rows, device="cuda", dtype=torch.float64).to(dtype)        # the second block; its neighbours stay zeros
    x[:, 69] = 1.0
    kept = c8.pack8(x, kind)
    values, codes, exps = ref8(x, kind)
    assert torch.equal(kept.exps, exps)
    assert torch.equal(magnitudes(kept.codes, kind), magnitudes(codes, kind))
    back = kept.expand()
    assert same(back, values.to(dtype))
    finite = torch.isfinite(x[:, 32:64].float()).all(-1)
    assert torch.isfinite(back[finite].float()).all() and torch.isnan(back[~finite][:, 32:64]).all()
    assert torch.isfinite(back[:, :32].float()).all() and (back[:, 69].float() == 1).all()


def test_ties_of_every_code(c8):
    """Every multiple of half a step of int8, every half of e4m3's range: one block each with 127 (240) beside it."""
    for kind, most, t in (("int8", 127.0, torch.arange(-254, 255) / 2), ("e4m3", 240.0, torch.arange(-0x5b80, 0x5b80, 8).abs().short().view(F16))):
        x = torch.zeros(t.numel(), 32, device="cuda", dtype=F32)
        x[:, 0] = most
        x[:, 5] = t.float().cuda()
        assert same(c8.pack8(x, kind).expand(), ref8(x, kind)[0])


def test_rows_of_more_dimensions_and_strides(c8):
    g = gen(1)
    x = randn(3, 4, 5, 48, g=g, dtype=BF16)
    for v in (x, x.transpose(0, 1), x[:, ::2], x[..., ::2], x[1, 2, 3], x.permute(0, 3, 1, 2), x[:, :, :1].expand(3, 4, 5, 48), x[:0], x[..., :1]):
        kept = c8.pack8(v, "e4m3")
        assert kept.shape == tuple(v.shape)
        assert same(kept.expand(), ref8(v.reshape(-1, v.shape[-1]), "e4m3")[0].to(BF16).view(v.shape))
        y, k2 = c8.gelu8_forward(v)
        assert y.shape == v.shape and c8.gelu8_backward(torch.ones_like(v), k2).shape == v.shape


# ---------------------------------------------------------------- GELU
def phi(a):
    return torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)


def half_step(want, dtype):
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_gelu(c8, rows, d, dtype, kind):
    g = gen(7 * rows + d)
    for name, x in layouts(rows, d, dtype, g, 2.5):
        y, kept = c8.gelu8_forward(x, kind)
        a = x.double()
        want = a * torch.special.ndtr(a)
        # the fit and its exponential: 2.4e-7 absolute; the final fma and the rounding to fp32
        assert ((y.double() - want).abs() <= half_step(want, dtype) + 2.4e-7 + 2 * U * want.abs()).all(), name
        a, gy = ref8(x, kind)[0], randn(rows, d + 2, g=g, dtype=dtype)[:, :d]
        gx = c8.gelu8_backward(gy, kept)
        slope = torch.special.ndtr(a) + a * phi(a)
        want = slope * gy.double()
        # Phi(-a): 1e-7 + 2^-22 / 2;  a phi(a) <= 0.242: 2^-22 of it from the exponential and (a^2 0.73 + 1.4) 2^-23 from its argument, together
        # below 1.7e-7;  two sums of numbers below 1.13: 1.4e-7
        assert ((gx.double() - want).abs() <= half_step(want, dtype) + gy.double().abs() * 5.5e-7 + U * want.abs()).all(), name


def test_gelu_slope_against_differences(c8):
    """The gradient is the forward's slope at what was kept: central differences in 64 bits."""
    x = torch.linspace(-9, 9, 4001, device="cuda").view(-1, 1).expand(-1, 4).contiguous()
    _, kept = c8.gelu8_forward(x, "e4m3")
    a, h = kept.expand().double(), 1e-4
    f = lambda t: t * torch.special.ndtr(t)
    want = (f(a + h) - f(a - h)) / (2 * h)
    # h^2 / 6 of a third derivative below 3, cancellation 9 * 2^-53 / h, and the slope's own 5.5e-7
    assert ((c8.gelu8_backward(torch.ones_like(x), kept).double() - want).abs() <= h * h / 2 + 2e-11 + 5.5e-7 + 2 * U).all()


def test_gelu_far_and_not_finite(c8):
    x = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, 60000.0, -60000.0, 30.0, -30.0]], device="cuda")
    y, kept = c8.gelu8_forward(x)
    assert y[0].tolist()[:2] == [math.inf, 0.0] and math.isnan(y[0, 2]) and y[0].tolist()[3:] == [0.0, 0.0, 60000.0, 0.0, 30.0, 0.0]
    assert torch.isnan(c8.gelu8_backward(torch.ones_like(x), kept)).all()              # the block is not finite
    x = torch.tensor([[60000.0, -60000.0, 3e38, -3e38]], device="cuda")
    _, kept = c8.gelu8_forward(x)
    assert c8.gelu8_backward(torch.full_like(x, 2.0), kept)[0].tolist()[2:] == [2.0, 0.0]


def test_in_place_and_nothing_beside(native):
    """y over x, gx over gy, at every alignment; elements between the rows and around them stay as they were."""
    lib, s = native.lib, torch.cuda.current_stream().cuda_stream
    for dtype, code in ((F16, 1), (BF16, 5), (F32, 0)):
        for d, ld, first in ((40, 40, 0), (41, 45, 1), (33, 33, 3), (64, 71, 5), (1001, 1001, 7), (7, 9, 2), (260, 261, 4)):
            rows, g = 37, gen(d)
            buf = randn(rows * ld + 40, g=g, dtype=dtype)
            view = lambda b: b[first:first + rows * ld].view(rows, ld)[:, :d]
            x = view(buf).clone()
            pitch = (d + 31) // 32 * 32
            codes = torch.full((rows * pitch + 64,), 77, dtype=torch.uint8, device="cuda")
            exps = torch.full((rows * pitch // 32 + 64,), 77, dtype=torch.uint8, device="cuda")
            y = torch.empty_like(x)
            native.check(lib.bsrl_gelu8(x.data_ptr(), code, d, rows, d, y.data_ptr(), d, 0, codes.data_ptr(), exps.data_ptr(), s))
            before, at = buf.clone(), buf.data_ptr() + first * buf.element_size()
            native.check(lib.bsrl_gelu8(at, code, ld, rows, d, at, ld, 0, codes.data_ptr(), exps.data_ptr(), s))
            assert torch.equal(view(buf), y)
            view(before).copy_(y)
            assert torch.equal(buf, before)
            assert (codes[rows * pitch:] == 77).all() and (exps[rows * pitch // 32:] == 77).all()
            assert (codes[:rows * pitch].view(rows, pitch)[:, d:] == 0).all()
            gx = torch.empty_like(x)
            native.check(lib.bsrl_gelu8_bwd(y.data_ptr(), code, d, codes.data_ptr(), exps.data_ptr(), 0, rows, d, gx.data_ptr(), d, s))
            native.check(lib.bsrl_gelu8_bwd(at, code, ld, codes.data_ptr(), exps.data_ptr(), 0, rows, d, at, ld, s))
            view(before).copy_(gx)
            assert torch.equal(buf, before)
            native.check(lib.bsrl_expand8(codes.data_ptr(), exps.data_ptr(), 0, rows, d, at, code, ld, s))
            view(before).copy_(ref8(x, "int8")[0].to(dtype))
            assert torch.equal(buf, before)


# ---------------------------------------------------------------- LayerNorm
def norm_reference(z, w, b, eps, kind):
    a = z.double()
    mean = a.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((a - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (a - mean) * rstd * w.double() + (b.double() if b is not None else 0)
    return y, (ref8(z, kind)[0] - mean) * rstd, mean, rstd


def check_norm(c8, x, out, residual, kind, g, bias=True, eps=1e-5, name=""):
    rows, d = x.shape
    dtype = x.dtype
    w, b = 1 + 0.3 * randn(d, g=g), (0.3 * randn(d, g=g) if bias else None)
    y, z, saved = c8.layer_norm8_forward(x, w, b, eps, residual=residual, out_dtype=out, kind=kind)
    if residual is None:
        assert z is x
    else:
        assert torch.equal(z, (x.float() + residual.float()).to(dtype)), name
    want, h, mean, rstd = norm_reference(z, w, b, eps, kind)
    a = z.double()
    # sums of d numbers, at most 8 + d / 256 of them one after the other in a lane, five to ten steps of a tree
    n = 20 + d / 256
    e_mean = n * U * a.abs().mean(-1, keepdim=True)
    assert ((saved.stats[0].double() - mean.squeeze(-1)).abs() <= e_mean.squeeze(-1)).all(), name
    # the variance: n roundings and the mean's square; rstd half of its relative error and two steps of rsqrtf
    e_rstd = (n + 8) * U + (e_mean * rstd) ** 2
    assert ((saved.stats[1].double() - rstd.squeeze(-1)).abs() <= (e_rstd * rstd).squeeze(-1)).all(), name
    hat = (a - mean).abs() * rstd
    e_y = w.double().abs() * (rstd * e_mean + hat * (e_rstd + 4 * U)) + 2 * U * want.abs()
    assert ((y.double() - want).abs() <= half_step(want, out) + e_y).all(), name
    assert torch.equal(saved.kept.exps, ref8(z, kind)[2]), name

    gy = randn(rows, d + 3, g=g, dtype=out)[:, 2:2 + d]
    g_res = randn(rows, d, g=g, dtype=dtype) if residual is not None else None
    gx, gw, gb = c8.layer_norm8_backward(gy, saved, w, g_residual=g_res)
    gyd, gh = gy.double(), gy.double() * w.double()
    gx_want = rstd * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True)) + (g_res.double() if g_res is not None else 0)
    e_h = h.abs() * (e_rstd + 4 * U) + rstd * e_mean + 2 * U * mean.abs() * rstd
    m1, m2 = gh.abs().mean(-1, keepdim=True), (gh * h).abs().mean(-1, keepdim=True)
    e_gx = rstd * ((n + 6) * U * (m1 + h.abs() * m2) + e_h * m2 + h.abs() * (gh.abs() * e_h).mean(-1, keepdim=True)
                   + (e_rstd + 6 * U) * (gh.abs() + m1 + h.abs() * m2)) + 2 * U * gx_want.abs()
    # a row whose kept values lie far from it in units of its own spread (a single element: no spread) can leave fp16: infinity from
    # half a step past the largest number on
    most = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    out_of_range = gx_want.abs() - e_gx > most
    assert (torch.isinf(gx) & (gx.sign() == gx_want.sign()) | ~out_of_range).all(), name
    assert gx.dtype == dtype and ((gx.double() - gx_want).abs() <= half_step(gx_want, dtype) + e_gx).logical_or(out_of_range).all(), name
    # over the rows: a lane's own, then at most 500 partial sums
    m = rows / 100 + 600 if rows > 100 else rows
    assert ((gw.double() - (gyd * h).sum(0)).abs() <= (gyd.abs() * (h.abs() * m * U + e_h)).sum(0) + 1e-30).all(), name
    assert ((gb.double() - gyd.sum(0)).abs() <= m * U * gyd.abs().sum(0) + 1e-30).all(), name
    again = c8.layer_norm8_backward(gy, saved, w, g_residual=g_res)
    assert all(torch.equal(p, q) for p, q in zip((gx, gw, gb), again)), name
    assert c8.layer_norm8_backward(gy, saved, w, g_residual=g_res, param_grads=False)[1:] == (None, None)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("rows,d", SHAPES + [(515, 64), (2000, 128), (33, 2048), (9, 513), (700, 300), (3, 7999)])
def test_layer_norm(c8, rows, d, dtype, out, kind):
    g = gen(rows * 3 + d)
    for name, x in layouts(rows, d, dtype, g, 2.0):
        x = x.add_(0.5) if name != "pitch" else x
        check_norm(c8, x, out, None, kind, g, bias=rows % 2 == 0, name=name)
        for rname, r in layouts(rows, d, dtype, g):
            if rname in ("dense", name):
                check_norm(c8, x, out, r, kind, g, name=name + "+" + rname)


def test_layer_norm_gradients_against_differences(c8):
    """With a checkpoint that loses nothing (whole numbers up to 127 of int8) the backward is the forward's derivative."""
    g = gen(5)
    rows, d = 3, 40
    x = torch.randint(-127, 128, (rows, d), generator=g, device="cuda").float()
    x[:, ::32] = 127
    w, b, gy = 1 + 0.3 * randn(d, g=g), randn(d, g=g), randn(rows, d, g=g)
    _, _, saved = c8.layer_norm8_forward(x, w, b)
    gx, gw, gb = c8.layer_norm8_backward(gy, saved, w)

    def loss(x, w, b):
        return (torch.nn.functional.layer_norm(x, (d,), w, b, 1e-5) * gy.double()).sum()

    h = 1e-4
    for t, got in ((x, gx), (w, gw), (b, gb)):
        args = [v.double() for v in (x, w, b)]
        k = [v.data_ptr() for v in (x, w, b)].index(t.data_ptr())
        flat, want = args[k].view(-1), []
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss(*args)
            flat[i] = keep - h
            want.append((up - loss(*args)) / (2 * h))
            flat[i] = keep
        want = torch.stack(want).view(t.shape)
        # h^2 of a third derivative of order one; fp32: some fifty roundings of sums of numbers of order ten
        assert ((got.double() - want).abs() <= 1e-7 + 50 * U * 10).all()


def test_layer_norm_special_rows(c8):
    """Equal rows (no variance), rows of zeros, a row with NaN: it keeps to itself, but for the parameters' sums."""
    w, b = torch.full((48,), 2.0, device="cuda"), torch.full((48,), 0.5, device="cuda")
    x = torch.zeros(5, 48, device="cuda")
    x[1] = 3.0
    x[2] = torch.arange(48.0)
    x[3, 7] = math.nan
    x[4, 9] = math.inf
    y, _, saved = c8.layer_norm8_forward(x, w, b)
    assert (y[:2] == 0.5).all() and torch.isfinite(y[2]).all() and torch.isnan(y[3]).all() and torch.isnan(y[4]).any()
    gx, gw, gb = c8.layer_norm8_backward(torch.ones_like(x), saved, w)
    assert torch.isfinite(gx[:3]).all() and torch.isnan(gx[3]).any() and torch.isnan(gw).all() and (gb == 5).all()
    y, z, saved = c8.layer_norm8_forward(x[:0], w, b, residual=x[:0])
    gx, gw, gb = c8.layer_norm8_backward(y, saved, w, g_residual=z)
    assert y.shape == z.shape == gx.shape == (0, 48) and not gw.any() and not gb.any()


def test_layer_norm_in_place_and_nothing_beside(native):
    """z over the residual, gx over the residual's gradient; what lies between and around the rows stays."""
    lib, s = native.lib, torch.cuda.current_stream().cuda_stream
    for dtype, code in ((F32, 0), (F16, 1)):
        for d, ld, first in ((64, 64, 0), (65, 67, 1), (31, 31, 2), (600, 603, 5), (1025, 1025, 3), (5000, 5001, 1), (1024, 1032, 8)):
            rows, g = 41, gen(d)
            bufs = [randn(rows * ld + 40, g=g, dtype=dtype) for _ in range(4)]
            view = lambda b: b[first:first + rows * ld].view(rows, ld)[:, :d]
            at = lambda b: b.data_ptr() + first * b.element_size()
            x, r, y, gr = bufs
            w = randn(d, g=g)
            pitch = (d + 31) // 32 * 32
            codes, exps = (torch.full((n + 64,), 77, dtype=torch.uint8, device="cuda") for n in (rows * pitch, rows * pitch // 32))
            stats = torch.full((2 * rows + 2,), -1.0, device="cuda")
            want = [b.clone() for b in bufs]
            z = (view(x).float() + view(r).float()).to(dtype)
            native.check(lib.bsrl_layernorm8(at(x), at(r), code, ld, ld, w.data_ptr(), None, 1e-5, rows, d, at(r), ld, at(y), code, ld, 0, codes.data_ptr(),
                                             exps.data_ptr(), stats.data_ptr(), stats.data_ptr() + 4 * rows, s))
            view(want[1]).copy_(z)
            view(want[2]).copy_(view(y))
            ref = norm_reference(z, w, None, 1e-5, "int8")[0]
            assert ((view(y).double() - ref).abs() <= half_step(ref, dtype) + 1e-4).all()
            assert all(torch.equal(b, c) for b, c in zip(bufs, want))
            assert (codes[rows * pitch:] == 77).all() and (exps[rows * pitch // 32:] == 77).all() and (stats[2 * rows:] == -1).all()
            size = lib.bsrl_layernorm8_bwd_workspace_bytes(rows, d)
            ws = torch.full((size + 64,), 77, dtype=torch.uint8, device="cuda")
            gw, gb, dense = torch.full((d + 4,), -1.0, device="cuda"), torch.full((d + 4,), -1.0, device="cuda"), torch.empty(rows, d, dtype=dtype, device="cuda")
            grads = lambda res, gx, ldx: lib.bsrl_layernorm8_bwd(
                at(y), code, ld, res, ld, codes.data_ptr(), exps.data_ptr(), 0, stats.data_ptr(), stats.data_ptr() + 4 * rows, w.data_ptr(), rows, d, gx, code,
                ldx, gw.data_ptr(), gb.data_ptr(), ws.data_ptr(), size, s)
            native.check(grads(at(gr), dense.data_ptr(), d))
            native.check(grads(at(gr), at(gr), ld))
            view(want[3]).copy_(dense)
            assert torch.equal(bufs[3], want[3]) and (gw[d:] == -1).all() and (gb[d:] == -1).all() and (ws[size:] == 77).all()


# ---------------------------------------------------------------- weight gradient
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 8, 32), (63, 16, 33), (64, 128, 64), (65, 130, 96), (29 * 64, 768, 256), (2049, 256, 513), (5000, 1000, 264),
                                      (777, 1001, 100), (130, 2048, 31), (300, 24, 2000), (20000, 256, 256), (9000, 384, 640), (70000, 64, 64)])
def test_weight_gradient(c8, rows, n, k, dtype, kind):
    g = gen(rows + n + k)
    x, gy = randn(rows, k, g=g, dtype=dtype), randn(rows, n, g=g, dtype=dtype)
    kept = c8.pack8(x, kind)
    gw, gb = c8.linear8_weight_grad(gy, kept)
    xv = ref8(x, kind)[0].to(dtype).double()           # in fp16 the smallest values are rounded on their way into the product
    want, most = gy.double().t() @ xv, gy.double().abs().t() @ xv.abs()
    # chains of at most 2,560 rows: a truncation (2 U) per 16 rows, 320 U; their sums and the splits', rounded to nearest: one per 2,560 rows, or
    # up to 300 of shorter chains.  256 and 300 here cover both
    assert ((gw.double() - want).abs() <= most * (min(rows, 2048) / 16 * 2 + rows / 2048 + 300) * U + 1e-30).all()
    # a lane's share of the rows, then at most 8 x 300 partial sums by eights
    assert ((gb.double() - gy.double().sum(0)).abs() <= gy.double().abs().sum(0) * (rows / 8 + 400) * U + 1e-30).all()
    if rows > 2048:      # far inside of that worst case: what a product with fp32 sums gives
        assert float((gw.double() - want).norm() / want.norm()) < 4e-6
    again, none = c8.linear8_weight_grad(gy, kept, bias=False)
    assert none is None and torch.equal(again, gw)
    for v in (torch.cat([gy, gy], 1)[:, :n], torch.cat([gy[:, :1], gy], 1)[:, 1:]):           # a pitch; an unaligned first element
        a, b = c8.linear8_weight_grad(v, kept)
        assert torch.equal(a, gw) and torch.equal(b, gb)


def test_weight_gradient_of_extremes(c8):
    """Scales that fp16 has no normal number for, blocks of zeros, a block that is not finite."""
    for dtype in (F16, BF16):
        g = gen(3)
        x = randn(96, 160, g=g, dtype=F32)
        x[:, 32:64] *= 2.0 ** -17
        x[:, 64:96] *= 2000.0
        x[:, 96:128] = 0
        x = x.to(dtype)
        gy = randn(96, 64, g=g, dtype=dtype)
        for kind in ("int8", "e4m3"):
            kept = c8.pack8(x, kind)
            gw, _ = c8.linear8_weight_grad(gy, kept)
            xv = kept.expand().double()
            want, most = gy.double().t() @ xv, gy.double().abs().t() @ xv.abs()
            assert ((gw.double() - want).abs() <= most * 12 * U + 1e-30).all()
            bad = x.clone()
            bad[5, 130] = math.nan
            gw2, gb2 = c8.linear8_weight_grad(gy, c8.pack8(bad, kind))
            assert torch.isnan(gw2[:, 128:]).all() and torch.equal(gw2[:, :128], gw[:, :128]) and torch.isfinite(gb2).all()
    wide = (torch.randn(64, 32, generator=gen(4), device="cuda") * 1e30).to(BF16)             # 2^23 times its scale is not finite
    one = torch.ones(64, 8, device="cuda", dtype=BF16)
    for kind in ("int8", "e4m3"):
        kept = c8.pack8(wide, kind)
        want = kept.expand().double().sum(0)
        gw, _ = c8.linear8_weight_grad(one, kept)
        assert ((gw.double() - want).abs() <= kept.expand().double().abs().sum(0) * 12 * U).all()
    gw, gb = c8.linear8_weight_grad(one[:0], c8.pack8(wide[:0]))
    assert gw.shape == (8, 32) and not gw.any() and not gb.any()


# ---------------------------------------------------------------- together
def test_ffn_block_trains_from_8_bits(c8):
    """LayerNorm, linear, GELU, linear and the residual stream, as a block of a policy has them: every gradient is the formulas' at what was
    kept."""
    g = gen(9)
    rows, d, f = 29 * 6, 64, 256
    p = {"ln_w": 1 + 0.2 * randn(d, g=g), "ln_b": 0.2 * randn(d, g=g), "w0": randn(f, d, g=g, scale=d ** -0.5), "b0": 0.1 * randn(f, g=g),
         "w2": randn(d, f, g=g, scale=f ** -0.5), "b2": 0.1 * randn(d, g=g)}
    branch, stream, g_out, g_z = (randn(rows, d, g=g) for _ in range(4))
    with torch.enable_grad():
        leaves = {k: v.clone().requires_grad_() for k, v in p.items()} | {"branch": branch.clone().requires_grad_(), "stream": stream.clone().requires_grad_()}
        y, z = c8.layer_norm8(leaves["branch"], leaves["ln_w"], leaves["ln_b"], residual=leaves["stream"], out_dtype=F16)
        a = c8.linear8(y, leaves["w0"], leaves["b0"])
        t = c8.gelu8(a)
        o = c8.linear8(t, leaves["w2"], leaves["b2"])
        (z + o.float()).mul(g_out).sum().backward()
    # the same chain by hand: each layer's gradient from what it kept of the tensors that this run made
    zv, yv, av, tv = (ref8(v.detach(), "int8")[0] for v in (z, y, a, t))
    go = g_out.half().double()
    w0, w2 = p["w0"].half().double(), p["w2"].half().double()
    want = {"w2": go.t() @ tv, "b2": go.sum(0)}
    gt = (go @ w2).half().double()
    ga = (gt * (torch.special.ndtr(av) + av * phi(av))).half().double()
    want |= {"w0": ga.t() @ yv, "b0": ga.sum(0)}
    gy = (ga @ w0).half().double()
    zd = z.detach().double()
    mean, var = zd.mean(-1, keepdim=True), zd.var(-1, unbiased=False, keepdim=True)
    rstd = 1 / torch.sqrt(var + 1e-5)
    h, gh = (zv - mean) * rstd, gy * p["ln_w"].double()
    gz = rstd * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True)) + g_out.double()
    want |= {"ln_w": (gy * h).sum(0), "ln_b": gy.sum(0), "branch": gz, "stream": gz}
    for k, v in want.items():
        got = leaves[k].grad.double()
        # three roundings to fp16 on the way (gt, ga, gy), each 2^-11 of its numbers, which may fall on the other side of a step than here
        assert got.shape == v.shape and float((got - v).norm() / v.norm()) < 3 * 2.0 ** -11, k
    # and near to the gradients of the same block that keeps everything
    with torch.enable_grad():
        q = {k: v.detach().clone().double().requires_grad_() for k, v in leaves.items()}
        zz = q["branch"] + q["stream"]
        yy = torch.nn.functional.layer_norm(zz, (d,), q["ln_w"], q["ln_b"], 1e-5)
        oo = torch.nn.functional.gelu(yy @ q["w0"].t() + q["b0"]) @ q["w2"].t() + q["b2"]
        (zz + oo).mul(g_out.double()).sum().backward()
    for k in want:
        assert float((leaves[k].grad.double() - q[k].grad).norm() / q[k].grad.norm()) < 0.03, k


def test_only_some_gradients(c8):
    g = gen(11)
    x, w, b = randn(6, 64, g=g, dtype=F16), randn(64, g=g), randn(64, g=g)
    with torch.enable_grad():
        r = x.clone().requires_grad_()
        y, z = c8.layer_norm8(x, w, b, residual=r)
        z.sum().backward()                                   # y is not used
        assert torch.equal(r.grad, torch.ones_like(r))
        r.grad = None
        y, z = c8.layer_norm8(x, w, b, residual=r)
        y.sum().backward()                                   # z is not used
        assert r.grad is not None and x.grad is None
        w1 = w.clone().requires_grad_()
        c8.layer_norm8(x, w1).sum().backward()
        assert w1.grad is not None
        m = randn(32, 64, g=g).requires_grad_()
        c8.linear8(x, m).sum().backward()
        assert m.grad.dtype == F32 and m.grad.shape == (32, 64)
        m16 = m.detach().half().requires_grad_()
        xr = x.clone().requires_grad_()
        c8.linear8(xr, m16, b[:32].clone().requires_grad_(), kind="e4m3").float().sum().backward()
        assert m16.grad.dtype == F16 and xr.grad.shape == x.shape
        e = c8.linear8(xr[:0], m16)
        assert e.shape == (0, 32)
    with pytest.raises(ValueError):
        c8.layer_norm8(x, w[:32])
    with pytest.raises(ValueError):
        c8.layer_norm8(x, w, residual=x[:3])
    with pytest.raises(ValueError):
        c8.linear8(x, m[:, :32])
    with pytest.raises(ValueError):
        c8.linear8(x, m[:31])
    with pytest.raises(TypeError):
        c8.linear8(x.bfloat16(), m)
    kept = c8.pack8(x)
    with pytest.raises(ValueError):
        c8.gelu8_backward(x[:3], kept)
    with pytest.raises(TypeError):
        c8.linear8_weight_grad(x.float(), kept)
    with pytest.raises(ValueError):
        c8.linear8_weight_grad(x[:4], kept)
    with pytest.raises(Exception, match="layernorm8"):
        c8.layer_norm8(x, w, out_dtype=F32)


def test_captured_steps(c8):
    """Two captured steps and an eager one between their replays: none disturbs another, new inputs give new results."""
    g = gen(13)
    rows, d = 500, 192

    def step(x, gy, w, b, gl):
        y, z, saved = c8.layer_norm8_forward(x, w, b, residual=gy)
        t, kept = c8.gelu8_forward(y)
        gw, gb = c8.linear8_weight_grad(gl, c8.pack8(t))
        return (y, t, *c8.layer_norm8_backward(c8.gelu8_backward(gy, kept), saved, w, g_residual=gy), gw, gb)

    ins = [[randn(rows, d, g=g, dtype=F16), randn(rows, d, g=g, dtype=F16), randn(d, g=g), randn(d, g=g), randn(rows, 80, g=g, dtype=F16)] for _ in range(3)]
    want = [step(*i) for i in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for i in (0, 1):
        with torch.cuda.stream(side):
            step(*ins[i])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(*ins[i])
            graphs.append((graph, out))
    for _ in range(2):
        for i, (graph, out) in enumerate(graphs):
            graph.replay()
            third = step(*ins[2])
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want[i]))
            assert all(torch.equal(p, q) for p, q in zip(third, want[2]))
    for a, b in zip(ins[0], ins[2]):
        a.copy_(b)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(graphs[0][1], want[2]))
    # two streams at once
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = {}
    torch.cuda.synchronize()
    for _ in range(5):
        for s, i in ((s1, 1), (s2, 2)):
            with torch.cuda.stream(s):
                outs[i] = step(*ins[i])
    torch.cuda.synchronize()
    for i in (1, 2):
        assert all(torch.equal(p, q) for p, q in zip(outs[i], want[i]))


def test_offsets_past_32_bits(c8):
    """More than 2^32 elements, codes and blocks' first elements."""
    rows, d = 2 ** 22 + 5, 1056
    x = torch.zeros(rows, d, dtype=F16, device="cuda")
    g = gen(17)
    last = randn(3, d, g=g, dtype=F16)
    x[-3:] = last
    kept = c8.pack8(x)
    assert torch.equal(kept.codes[-3:], ref8(last, "int8")[1]) and not kept.codes[-4].any() and not kept.exps[:-3].any()
    y, kept = c8.gelu8_forward(x, "e4m3")
    assert torch.equal(y[-3:], c8.gelu8_forward(last)[0]) and not y[-4].any()
    gx = c8.gelu8_backward(x, kept)
    assert torch.equal(gx[-3:], c8.gelu8_backward(last, c8.gelu8_forward(last, "e4m3")[1])) and not gx[-4].any()
    del gx, y
    w = torch.ones(d, device="cuda")
    y, _, saved = c8.layer_norm8_forward(x, w)
    want, _, alone = c8.layer_norm8_forward(last, w)
    assert torch.equal(y[-3:], want) and not y[-4].any()
    gx, gw, _ = c8.layer_norm8_backward(x, saved, w)
    gl, gwl, _ = c8.layer_norm8_backward(last, alone, w)
    assert torch.equal(gx[-3:], gl) and float((gw - gwl).abs().max()) <= 8 * U * float(gwl.abs().max())
    del gx, y
    gy = torch.zeros(rows, 8, dtype=F16, device="cuda")
    gy[-3:] = 1
    gw, gb = c8.linear8_weight_grad(gy, saved.kept)
    assert (gb == 3).all()
    want = alone.kept.expand().double().sum(0).expand(8, -1)
    assert ((gw.double() - want).abs() <= 20 * U * alone.kept.expand().double().abs().sum(0)).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,out", [(F32, F16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("rows,d", [(1, 264), (3, 511), (33, 288), (1201, 512), (4801, 264), (2403, 509)])
def test_layer_norm_of_rows_taken_by_twos(c8, rows, d, dtype, out, kind):
    """Widths of 257 to 512: odd numbers of rows, one step and several per warp."""
    g = gen(rows + 5 * d)
    for name, x in layouts(rows, d, dtype, g, 2.0):
        check_norm(c8, x, out, None, kind, g, name=name)
        check_norm(c8, x, out, randn(rows, d, g=g, dtype=dtype), kind, g, name=name + "+residual")


def test_linear_of_slices(c8):
    """Inputs, weights, biases and gradients that start between 16-byte boundaries: the same results as of copies."""
    g = gen(23)
    for n, k in ((96, 64), (64, 96)):
        flat = {"x": randn(40 * k + 3, g=g, dtype=F16), "w": randn(n * k + 5, g=g, dtype=F16), "b": randn(n + 1, g=g), "gy": randn(40 * n + 1, g=g, dtype=F16)}
        odd = [flat["x"][3:].view(40, k), flat["w"][5:].view(n, k), flat["b"][1:], flat["gy"][1:].view(40, n)]
        assert all(t.data_ptr() % 16 for t in odd)
        results = []
        for x, w, b, gy in (odd, [t.clone() for t in odd]):
            x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
            with torch.enable_grad():
                y = c8.linear8(x, w, b)
                y.backward(gy)
            results.append((y.detach(), x.grad, w.grad, b.grad))
        for p, q in zip(*results):
            assert torch.equal(p, q)
        x, w, b, gy = (t.double() for t in odd)
        # y: fp32 sums of k products (truncated: 2 U per 16 and rounding; k U covers the order), then half a step of fp16
        most = x.abs() @ w.abs().t() + b.abs()
        assert ((results[0][0].double() - (x @ w.t() + b)).abs() <= half_step(x @ w.t() + b, F16) + most * (k + 2) * U).all()
        want = gy @ w
        assert ((results[0][1].double() - want).abs() <= half_step(want, F16) + (gy.abs() @ w.abs()) * (n + 2) * U).all()


def test_copies_have_their_own_memory(c8):
    """deepcopy and pickle: the copy outlives the original; one that lands on the CPU is refused."""
    import copy
    import io
    import pickle
    x = randn(5, 3, 70, g=gen(29), dtype=F16)
    for kind in ("int8", "e4m3"):
        one = c8.pack8(x, kind)
        want, bits = one.expand(), one.codes.clone()
        for kept in (one, c8.Checkpoint8(one.codes.clone(), one.exps.clone(), kind, x.shape, F16)):
            stored = io.BytesIO()
            torch.save(kept, stored)
            copies = [copy.deepcopy(kept), pickle.loads(pickle.dumps(kept)), torch.load(io.BytesIO(stored.getvalue()), weights_only=False)]
            same = copy.copy(kept)
            assert torch.equal(same.expand(), want)
            kept.codes.zero_()
            assert not same.expand().any()
            for c in copies:
                assert c.shape == x.shape and c.dtype == F16 and c.kind == kind and torch.equal(c.expand(), want) and torch.equal(c.codes, bits)
                own = {c.codes.data_ptr(), kept.codes.data_ptr()}
                assert len(own) == 2 and c._codes_ptr == c.codes.data_ptr() and c._exps_ptr == c.exps.data_ptr()
            with pytest.raises(RuntimeError, match="CUDA"):
                torch.load(io.BytesIO(stored.getvalue()), weights_only=False, map_location="cpu")

