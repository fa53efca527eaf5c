"""LayerNorm that keeps its input in 8 bits, with parameters that start anywhere: aligned rows, weight and bias inside a flat buffer."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


@pytest.mark.parametrize("first", [(1, 0), (0, 3), (2, 5)])
@pytest.mark.parametrize("dtype,out", [(F32, F16), (F16, F16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("rows,d", [(29, 256), (500, 64), (3, 8), (130, 1024), (5, 8192), (700, 512)])
def test_parameters_inside_a_flat_buffer(native, rows, d, dtype, out, first):
    """y against its formula in 64 bits; the checkpoint and the gradients as with parameters that have memory of their own."""
    from beatsaberrl_b200 import checkpoint8 as c8
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    x, gy, res = (torch.randn(rows, d, generator=g, device="cuda").to(t) for t in (dtype, out, dtype))
    flat = torch.randn(2 * d + 16, generator=g, device="cuda")
    w, b = flat[first[0]:first[0] + d], flat[d + 8 + first[1]:2 * d + 8 + first[1]]
    assert x.data_ptr() % 32 == 0 and (w.data_ptr() % 32 or b.data_ptr() % 32)
    eps_t = torch.finfo(out).eps / 2
    for kind in ("int8", "e4m3"):
        for r in (None, res):
            y, z, saved = c8.layer_norm8_forward(x, w, b, residual=r, out_dtype=out, kind=kind)
            y2, z2, saved2 = c8.layer_norm8_forward(x, w.clone(), b.clone(), residual=r, out_dtype=out, kind=kind)
            assert torch.equal(z, z2) and torch.equal(saved.kept.codes, saved2.kept.codes) and torch.equal(saved.kept.exps, saved2.kept.exps)
            a = z.double()
            mean, rstd = a.mean(-1, keepdim=True), 1 / torch.sqrt(a.var(-1, unbiased=False, keepdim=True) + 1e-5)
            hat = (a - mean) * rstd
            want = hat * w.double() + b.double()
            # the mean by n roundings of numbers of the rows' average size, rstd by as many and two of its own; then y's fma and its type's half step
            n = 20 + d / 256
            part = w.double().abs() * (rstd * n * U * a.abs().mean(-1, keepdim=True) + hat.abs() * (n + 12) * U) + 2 * U * want.abs()
            assert ((y.double() - want).abs() <= part + want.abs() * eps_t * (1 + eps_t) + torch.finfo(out).smallest_normal * eps_t).all()
            gx, gw, gb = c8.layer_norm8_backward(gy, saved, w, g_residual=r)
            gx2, gw2, gb2 = c8.layer_norm8_backward(gy, saved, w.clone(), g_residual=r)
            # two orders of the same sums: gx within the roundings of numbers of the size of its terms, and a step of its type
            h = (saved.kept.expand(F32).double() - saved.stats[0].double().unsqueeze(1)) * saved.stats[1].double().unsqueeze(1)
            gh = gy.double() * w.double()
            m1, m2 = gh.abs().mean(-1, keepdim=True), (gh * h).abs().mean(-1, keepdim=True)
            size = rstd * (gh.abs() + m1 + h.abs() * m2) + (r.double().abs() if r is not None else 0)
            assert ((gx.double() - gx2.double()).abs() <= size * (2 * (n + 20) * U) + gx2.double().abs() * torch.finfo(dtype).eps * 1.01
                    + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()
            m = 2 * (rows + 8) * U
            assert ((gw - gw2).abs().double() <= (gy.double().abs() * h.abs()).sum(0) * m).all()
            assert ((gb - gb2).abs().double() <= gy.double().abs().sum(0) * m).all()
