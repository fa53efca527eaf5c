"""Activations kept in 8 bits: what the C entries and the Python module refuse, on a host without a GPU.  Every refusal comes
ahead of the first launch, so no device is touched."""
import ctypes as C

import pytest
import torch

NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5
A = 0x10000                       # an aligned address that nothing reads


def _pack(native, x=A, dtype=1, ldx=64, rows=4, d=64, kind=0, codes=A, exps=A):
    return native.lib.bsrl_pack8(x, dtype, ldx, rows, d, kind, codes, exps, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), NULL), (dict(codes=None), NULL), (dict(exps=None), NULL), (dict(rows=-1), SHAPE), (dict(d=0), SHAPE),
    (dict(d=2 ** 31, ldx=2 ** 31), SHAPE), (dict(ldx=63), SHAPE), (dict(ldx=2 ** 50), SHAPE), (dict(dtype=2), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED),
    (dict(kind=2), UNSUPPORTED), (dict(kind=-1), UNSUPPORTED), (dict(x=A + 1), ALIGN), (dict(x=A + 2, dtype=0), ALIGN),
    (dict(codes=A + 8), ALIGN), (dict(exps=A + 2), ALIGN)])
def test_pack8_refuses(native, bad, status):
    assert _pack(native, **bad) == status
    assert native.last_error().startswith("pack8")


def test_no_rows_is_no_work(native):
    assert _pack(native, rows=0) == 0
    assert _pack(native, rows=0, x=None, codes=None, exps=None) == 0
    assert native.lib.bsrl_expand8(A, A, 0, 0, 5, A, 0, 5, None) == 0
    assert native.lib.bsrl_gelu8(A, 1, 5, 0, 5, A, 5, 0, A, A, None) == 0
    assert native.lib.bsrl_gelu8_bwd(A, 1, 5, A, A, 0, 0, 5, A, 5, None) == 0
    assert native.lib.bsrl_layernorm8(A, None, 1, 5, 0, A, A, 1e-5, 0, 5, None, 0, A, 1, 5, 0, A, A, None, None, None) == 0
    assert native.lib.bsrl_linear8_wgrad_workspace_bytes(0, 8, 8, 1) == 0
    assert native.lib.bsrl_layernorm8_bwd_workspace_bytes(0, 8) == 0


def test_pitch(native):
    for d, want in ((1, 32), (32, 32), (33, 64), (2 ** 31 - 64, 2 ** 31 - 64), (0, -1), (-3, -1), (2 ** 31, -1)):
        assert native.lib.bsrl_pack8_pitch(d) == want


@pytest.mark.parametrize("bad,status", [(dict(out=None), NULL), (dict(ldo=4), SHAPE), (dict(out=A + 2), ALIGN), (dict(kind=3), UNSUPPORTED),
                                        (dict(dtype=4), UNSUPPORTED)])
def test_expand8_refuses(native, bad, status):
    a = dict(codes=A, exps=A, kind=1, rows=2, d=5, out=A, dtype=0, ldo=5) | bad
    assert native.lib.bsrl_expand8(*a.values(), None) == status


@pytest.mark.parametrize("bad,status", [(dict(y=None), NULL), (dict(ldy=4), SHAPE), (dict(y=A + 1), ALIGN), (dict(dtype=3), UNSUPPORTED)])
def test_gelu8_refuses(native, bad, status):
    a = dict(x=A, dtype=1, ldx=5, rows=2, d=5, y=A, ldy=5, kind=0, codes=A, exps=A) | bad
    assert native.lib.bsrl_gelu8(*a.values(), None) == status
    b = dict(gy=a["x"], dtype=a["dtype"], ldgy=a["ldx"], codes=A, exps=A, kind=0, rows=2, d=5, gx=a["y"], ldgx=a["ldy"])
    assert native.lib.bsrl_gelu8_bwd(*b.values(), None) == status


NORM = dict(x=A, residual=A, dtype=0, ldx=64, ldr=64, gamma=A, beta=A, eps=1e-5, rows=3, d=64, z=A, ldz=64, y=A, y_dtype=1, ldy=64, kind=0, codes=A,
            exps=A, mean=A, rstd=A)
NORM_BWD = dict(gy=A, gy_dtype=1, ldgy=64, g_residual=A, ldgr=64, codes=A, exps=A, kind=0, mean=A, rstd=A, gamma=A, rows=1000, d=64, gx=A, dtype=0,
                ldgx=64, g_gamma=A, g_beta=A, workspace=A, workspace_bytes=2 ** 30)


@pytest.mark.parametrize("bad,status", [
    (dict(d=8193, ldx=9000, ldr=9000, ldz=9000, ldy=9000), SHAPE), (dict(d=0), SHAPE), (dict(rows=-2), SHAPE), (dict(z=None), NULL), (dict(gamma=None), NULL),
    (dict(mean=None), NULL), (dict(rstd=None), NULL), (dict(ldr=63), SHAPE), (dict(ldz=1), SHAPE), (dict(dtype=1, y_dtype=0), UNSUPPORTED),
    (dict(dtype=5, y_dtype=1), UNSUPPORTED), (dict(y_dtype=2), UNSUPPORTED), (dict(gamma=A + 2), ALIGN), (dict(residual=A + 2), ALIGN), (dict(kind=5), UNSUPPORTED)])
def test_layernorm8_refuses(native, bad, status):
    assert native.lib.bsrl_layernorm8(*(NORM | bad).values(), None) == status
    assert native.last_error().startswith("layernorm8:")


@pytest.mark.parametrize("bad,status", [
    (dict(d=8193, ldgy=9000, ldgr=9000, ldgx=9000), SHAPE), (dict(gy=None), NULL), (dict(gx=None), NULL), (dict(gamma=None), NULL), (dict(mean=None), NULL),
    (dict(ldgy=8), SHAPE), (dict(dtype=1, gy_dtype=0), UNSUPPORTED), (dict(g_gamma=A + 1), ALIGN), (dict(workspace=None), WORKSPACE),
    (dict(workspace_bytes=16), WORKSPACE), (dict(workspace=A + 4), WORKSPACE), (dict(codes=None), NULL)])
def test_layernorm8_bwd_refuses(native, bad, status):
    assert native.lib.bsrl_layernorm8_bwd(*(NORM_BWD | bad).values(), None) == status
    assert native.last_error().startswith("layernorm8_bwd:")


WGRAD = dict(gy=A, gy_dtype=1, ldgy=64, codes=A, exps=A, kind=0, rows=100, n=64, k=32, g_weight=A, g_bias=None, workspace=A, workspace_bytes=2 ** 30)


@pytest.mark.parametrize("bad,status", [
    (dict(gy=None), NULL), (dict(g_weight=None), NULL), (dict(codes=None), NULL), (dict(rows=-1), SHAPE), (dict(rows=2 ** 31), SHAPE), (dict(n=0), SHAPE),
    (dict(k=0), SHAPE), (dict(k=2 ** 20 + 1), SHAPE), (dict(n=2 ** 20, ldgy=2 ** 20, k=2049), SHAPE), (dict(ldgy=63), SHAPE), (dict(gy_dtype=0), UNSUPPORTED), (dict(gy=A + 1), ALIGN), (dict(g_weight=A + 2), ALIGN),
    (dict(workspace=None), WORKSPACE), (dict(workspace=A + 16), WORKSPACE), (dict(workspace_bytes=64), WORKSPACE)])
def test_linear8_wgrad_refuses(native, bad, status):
    assert native.lib.bsrl_linear8_wgrad(*(WGRAD | bad).values(), None) == status
    assert native.last_error().startswith("linear8_w")


def test_workspace_sizes(native):
    """Of every size something; more where g has to be copied; never less for fewer bytes than the parts need."""
    size = native.lib.bsrl_linear8_wgrad_workspace_bytes
    for rows, n, k in ((1, 1, 1), (29, 768, 256), (1000, 1001, 33), (475136, 1024, 256), (2 ** 31 - 257, 8, 8), (100, 2 ** 20, 32)):
        a, b = size(rows, n, k, 1), size(rows, n, k, 0)
        assert 0 < a <= b and b - a >= rows * n * 2, (rows, n, k)
        assert a >= n * k * 4
    assert size(2 ** 20, 2 ** 20, 2048, 1) > 0 and size(100, 2048, 2 ** 20, 1) > 0 and size(1, 2 ** 20, 2 ** 20, 1) == -1
    assert size(-1, 8, 8, 1) == -1 and size(2 ** 31, 8, 8, 1) == -1 and size(4, 0, 8, 1) == -1
    norm = native.lib.bsrl_layernorm8_bwd_workspace_bytes
    assert norm(1, 64) == 0 and norm(475136, 256) > 0 and norm(-1, 64) == -1 and norm(4, 8193) == -1


def test_python_refusals(native):
    from beatsaberrl_b200 import checkpoint8 as c8
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        c8.pack8(x)
    with pytest.raises(TypeError):
        c8.pack8(x.double())
    with pytest.raises(ValueError, match="kind"):
        c8.pack8(x, "int4")
    with pytest.raises(ValueError, match="kind"):
        c8.gelu8_forward(x, None)
    with pytest.raises(RuntimeError, match="CUDA"):
        c8.layer_norm8(x, torch.ones(32))
    with pytest.raises(RuntimeError, match="CUDA"):
        c8.linear8(x.half(), torch.zeros(32, 32))
    codes, exps = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        c8.Checkpoint8(codes, exps, "int8", (4, 32), torch.float16)
    for bad in (dict(shape=(4, 33)), dict(shape=(5, 32)), dict(shape=()), dict(shape=(4, 0)), dict(codes=codes.char()), dict(codes=codes.t()), dict(kind="fp8")):
        a = dict(codes=codes, exps=exps, kind="int8", shape=(4, 32), dtype=torch.float16) | bad
        with pytest.raises(ValueError):
            c8.Checkpoint8(**a)
    with pytest.raises(TypeError):
        c8.Checkpoint8(codes, exps, "int8", (4, 32), torch.float64)


def test_weight_gradient_barriers_of_both_ctas_are_awaited_at_cluster_scope():
    """Barriers that the other CTA of a pair arrives at are waited for with an acquire of cluster scope, and groups that wait by
    parity divide the ring's stages."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "beatsaberrl_b200" / "csrc" / "wgrad8_tc5.cu").read_text()
    arrived = set(re.findall(r"arrive_leader\(&sh->(\w+)", text))
    assert arrived == {"full_x", "acc_empty"} and text.count("mbar_arrive_cluster(") == 1
    for bar in arrived:
        calls = re.findall(r"(mbar_wait\w*)(<[^>]*>)?\(smem_u32\(&sh->" + bar + r"\[", text)
        assert calls and all(scope == "<PAIR>" for _, scope in calls), (bar, calls)
    assert "static_assert(STAGES % GROUPS == 0 && STAGES % SUM_GROUPS == 0" in text
