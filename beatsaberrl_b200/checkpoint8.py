"""Training operators that keep what their backward needs in 8 bits: LayerNorm, exact GELU and linear layers.

A minibatch's saved activations bound its size.  These operators write an activation's 8-bit form (``Checkpoint8``) -- LayerNorm and GELU in the
pass that reads it anyway, ``linear8`` in one of its own; without grad mode too -- and their backward reads that form: 33/64 of the memory of 16-bit activations, 33/128 of fp32 ones.  Blocks of 32
neighbouring values of a row share a power of two; ``kind`` "int8" is off by at most 1/127 of a block's largest magnitude, "e4m3" by
2^-4 of every value.  ``include/bsrl.h`` ("activations kept in 8 bits") has the format, for reading it elsewhere.

* ``layer_norm8``, ``gelu8``, ``linear8``: differentiable, to write a model with;
* ``*_forward`` / ``*_backward`` / ``linear8_weight_grad``: the same halves without autograd, for hand-written steps and CUDA graphs;
* ``pack8`` / ``Checkpoint8.expand``: any activation.

Everything runs on the current stream of the tensors' device; nothing synchronises, and all memory comes from torch's allocator, so
calls can be captured (make a first call on the device outside the capture).  Gradients of parameters are fp32 sums in one order: the same inputs give the same bits.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _native as nat

KINDS = {"int8": nat.INT8, "e4m3": nat.E4M3}
_DTYPES = {torch.float32: nat.F32, torch.float16: nat.F16, torch.bfloat16: nat.BF16}
BLOCK = 32


def _kind(kind: str) -> int:
    try:
        return KINDS[kind]
    except (KeyError, TypeError):
        raise ValueError(f"kind must be one of {sorted(KINDS)}, got {kind!r}") from None


def _dtype(t, what: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}") from None


def _rows(x: torch.Tensor, what: str):
    """x (..., d) as a matrix of rows with unit stride in them (a view where its strides allow it): (matrix, rows, d, pitch)."""
    if not x.is_cuda:
        raise RuntimeError(f"{what} must live on a CUDA device (this library has no CPU path)")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} must have a last dimension of at least one element, got {tuple(x.shape)}")
    d = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, d)
    rows, pitch = x.shape[0], x.stride(0)
    if rows <= 1:
        pitch = d
    if x.stride(1) != 1 and d > 1 or pitch < d:
        x, pitch = x.contiguous(), d
    return x, rows, d, pitch


def _same(x: torch.Tensor, like: torch.Tensor, what: str, dtype=None) -> torch.Tensor:
    if x.shape != like.shape or x.device != like.device or x.dtype != (dtype or like.dtype):
        raise ValueError(f"{what} must be {tuple(like.shape)} {dtype or like.dtype} on {like.device}, got {tuple(x.shape)} {x.dtype} on {x.device}")
    return x


def _vector(v: Optional[torch.Tensor], d: int, dev, what: str) -> Optional[torch.Tensor]:
    if v is None:
        return None
    if v.shape != (d,) or v.dtype != torch.float32 or v.device != dev:
        raise ValueError(f"{what} must be ({d},) float32 on {dev}, got {tuple(v.shape)} {v.dtype} on {v.device}")
    return v.contiguous()


def _like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Room for a result of x's shape, without gaps (a shape and a device as arguments take torch four times as long to read)."""
    return torch.empty_like(x, dtype=dtype) if x.is_contiguous() else torch.empty(x.shape, dtype=dtype, device=x.device)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _call(fn, dev, *args) -> None:
    """fn(*args, stream) on the device's current stream.  The device is switched only where it is not the current one: with the context
    manager and a Stream object around every call the small ones took half as long again."""
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        nat.check(rc)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(fn: str, index: int, *args) -> int:
    with torch.cuda.device(index):           # what a kernel needs goes by the device's number of SMs
        n = getattr(nat.lib, fn)(*args)
    if n < 0:
        raise nat.BsrlError(int(n), nat.last_error())
    return n


class Checkpoint8:
    """An activation in 8 bits: ``codes`` (rows, pitch) and ``exps`` (rows, pitch / 32), uint8 without gaps, the pitch being the last dimension
    rounded up to 32; ``shape`` and ``dtype`` are those of the activation."""

    __slots__ = ("kind", "shape", "dtype", "device", "_memory", "_rows", "_blocks", "_codes_ptr", "_exps_ptr")

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor, kind: str, shape, dtype: torch.dtype):
        _kind(kind)
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        shape = tuple(shape)
        if not shape or shape[-1] < 1:
            raise ValueError(f"shape must have a last dimension of at least one element, got {shape}")
        rows = 1
        for n in shape[:-1]:
            rows *= n
        blocks = -(-shape[-1] // BLOCK)
        if (codes.shape != (rows, blocks * BLOCK) or exps.shape != (rows, blocks) or codes.dtype != torch.uint8 or exps.dtype != torch.uint8
                or not codes.is_contiguous() or not exps.is_contiguous()):
            raise ValueError(f"codes and exps must be contiguous ({rows}, {blocks * BLOCK}) and ({rows}, {blocks}) uint8, got {tuple(codes.shape)} "
                             f"{codes.dtype} and {tuple(exps.shape)} {exps.dtype}")
        if codes.device != exps.device:
            raise ValueError(f"codes and exps must be on one device, got {codes.device} and {exps.device}")
        if not codes.is_cuda:
            raise RuntimeError("a Checkpoint8 must live on a CUDA device (this library has no CPU path)")
        self.kind, self.shape, self.dtype, self.device = kind, shape, dtype, codes.device
        self._memory, self._rows, self._blocks = (codes, exps), rows, blocks
        self._codes_ptr, self._exps_ptr = codes.data_ptr(), exps.data_ptr()

    @classmethod
    def _empty(cls, rows: int, x: torch.Tensor, kind: str) -> "Checkpoint8":
        """One for x (rows, d), in one piece of memory."""
        self = cls.__new__(cls)
        blocks = -(-x.shape[-1] // BLOCK)
        memory = torch.empty(rows * blocks * (BLOCK + 1), dtype=torch.uint8, device=x.device)
        self.kind, self.shape, self.dtype, self.device = kind, tuple(x.shape), x.dtype, x.device
        self._memory, self._rows, self._blocks = memory, rows, blocks
        self._codes_ptr = memory.data_ptr()
        self._exps_ptr = self._codes_ptr + rows * blocks * BLOCK
        return self

    def __reduce__(self):
        """Copies and pickles are made anew from codes and exps, with the constructor's checks: the addresses kept here are this one's own."""
        return Checkpoint8, (self.codes, self.exps, self.kind, self.shape, self.dtype)

    @property
    def codes(self) -> torch.Tensor:
        m = self._memory
        return m[0] if type(m) is tuple else m[:self._rows * self._blocks * BLOCK].view(self._rows, self._blocks * BLOCK)

    @property
    def exps(self) -> torch.Tensor:
        m = self._memory
        return m[1] if type(m) is tuple else m[self._rows * self._blocks * BLOCK:].view(self._rows, self._blocks)

    @property
    def nbytes(self) -> int:
        return self._rows * self._blocks * (BLOCK + 1)

    def expand(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values it stands for, in ``dtype`` (default: the activation's)."""
        out = torch.empty(*self.shape, dtype=dtype or self.dtype, device=self.device)
        d = self.shape[-1]
        _call(nat.lib.bsrl_expand8, self.device, self._codes_ptr, self._exps_ptr, KINDS[self.kind], self._rows, d, out.data_ptr(),
              _dtype(out, "dtype"), d)
        return out


def pack8(x: torch.Tensor, kind: str = "int8") -> Checkpoint8:
    """x (..., d) in 8 bits.  Rows may be strided (a slice of wider rows); other strides are copied first."""
    code, k = _dtype(x, "x"), _kind(kind)
    m, rows, d, ld = _rows(x, "x")
    kept = Checkpoint8._empty(rows, x, kind)
    _call(nat.lib.bsrl_pack8, x.device, m.data_ptr(), code, ld, rows, d, k, kept._codes_ptr, kept._exps_ptr)
    return kept


# ------------------------------------------------------------------ GELU
def gelu8_forward(x: torch.Tensor, kind: str = "int8"):
    """(gelu(x), x in 8 bits); the exact (erf) GELU."""
    code, k = _dtype(x, "x"), _kind(kind)
    m, rows, d, ld = _rows(x, "x")
    y = _like(x, x.dtype)
    kept = Checkpoint8._empty(rows, x, kind)
    _call(nat.lib.bsrl_gelu8, x.device, m.data_ptr(), code, ld, rows, d, y.data_ptr(), d, k, kept._codes_ptr, kept._exps_ptr)
    return y, kept


def gelu8_backward(gy: torch.Tensor, kept: Checkpoint8) -> torch.Tensor:
    """gy gelu'(x8), in the activation's type."""
    if gy.shape != kept.shape or gy.dtype != kept.dtype or gy.device != kept.device:
        raise ValueError(f"gy must be {kept.shape} {kept.dtype} on {kept.device}, got {tuple(gy.shape)} {gy.dtype} on {gy.device}")
    m, rows, d, ld = _rows(gy, "gy")
    gx = _like(gy, gy.dtype)
    _call(nat.lib.bsrl_gelu8_bwd, gy.device, m.data_ptr(), _DTYPES[gy.dtype], ld, kept._codes_ptr, kept._exps_ptr, KINDS[kept.kind], rows, d,
          gx.data_ptr(), d)
    return gx


class _Gelu8(Function):
    @staticmethod
    def forward(ctx, x, kind):
        y, kept = gelu8_forward(x, kind)
        ctx.save_for_backward(kept.codes, kept.exps)
        ctx.kept = kind, kept.shape, kept.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        return gelu8_backward(gy, Checkpoint8(*ctx.saved_tensors, *ctx.kept)), None


def gelu8(x: torch.Tensor, kind: str = "int8") -> torch.Tensor:
    """Differentiable exact GELU that keeps its input in 8 bits."""
    return _Gelu8.apply(x, kind)


# ------------------------------------------------------------------ LayerNorm
class LayerNorm8Saved(NamedTuple):
    """What ``layer_norm8_backward`` needs: the normalised tensor in 8 bits and ``stats`` (2, rows) fp32, its rows' mean and
    1 / sqrt(var + eps)."""
    kept: Checkpoint8
    stats: torch.Tensor


def layer_norm8_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                        residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, kind: str = "int8"):
    """LayerNorm over the last dimension of z = x + residual (rounded to x's type): (y, z, saved).

    weight and bias are fp32.  y has ``out_dtype`` (default: x's type): any of the three for fp32 rows, their own for 16-bit ones.
    Without a residual z is x.  Rows are at most 8,192 wide and fastest where they start on 16 bytes (fp32 on
    32, weight and bias too).  What is kept is z: rows whose mean lies far beyond their spread keep little of the spread, and where that is less than a
    step of the 8 bits (equal values; a single one) the gradient is not small but wrong, by up to the square of (step / spread)."""
    code, k = _dtype(x, "x"), _kind(kind)
    m, rows, d, ld = _rows(x, "x")
    dev = x.device
    weight, bias = _vector(weight, d, dev, "weight"), _vector(bias, d, dev, "bias")
    y = _like(x, out_dtype or x.dtype)
    z, res, ldr = x, None, 0
    if residual is not None:
        res, _, _, ldr = _rows(_same(residual, x, "residual"), "residual")
        z = _like(x, x.dtype)
    kept = Checkpoint8._empty(rows, x, kind)
    stats = torch.empty(2, rows, dtype=torch.float32, device=dev)
    at = stats.data_ptr()
    _call(nat.lib.bsrl_layernorm8, dev, m.data_ptr(), _ptr(res), code, ld, ldr, weight.data_ptr(), _ptr(bias), eps, rows, d, z.data_ptr(), d,
          y.data_ptr(), _dtype(y, "out_dtype"), d, k, kept._codes_ptr, kept._exps_ptr, at, at + 4 * rows)
    return y, z, LayerNorm8Saved(kept, stats)


def layer_norm8_backward(gy: torch.Tensor, saved: LayerNorm8Saved, weight: torch.Tensor, g_residual: Optional[torch.Tensor] = None,
                         param_grads: bool = True):
    """(gx, g_weight, g_bias): gx is the gradient of x and of the residual, ``g_residual`` (the gradient that reaches z by other ways)
    added; the parameters' are fp32 and None without ``param_grads``."""
    kept, stats = saved
    dev = kept.device
    if gy.shape != kept.shape or gy.device != dev:
        raise ValueError(f"gy must be {kept.shape} on {dev}, got {tuple(gy.shape)} on {gy.device}")
    code = _dtype(gy, "gy")
    m, rows, d, ld = _rows(gy, "gy")
    weight = _vector(weight, d, dev, "weight")
    if stats.shape != (2, rows) or stats.dtype != torch.float32 or stats.device != dev or not stats.is_contiguous():
        raise ValueError(f"stats must be contiguous (2, {rows}) float32 on {dev}")
    gx = _like(gy, kept.dtype)
    res, ldr = None, 0
    if g_residual is not None:
        res, _, _, ldr = _rows(_same(g_residual, gx, "g_residual"), "g_residual")
    gw = torch.empty(d, dtype=torch.float32, device=dev) if param_grads else None
    gb = torch.empty(d, dtype=torch.float32, device=dev) if param_grads else None
    n = _workspace_bytes("bsrl_layernorm8_bwd_workspace_bytes", dev.index, rows, d)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    at = stats.data_ptr()
    _call(nat.lib.bsrl_layernorm8_bwd, dev, m.data_ptr(), code, ld, _ptr(res), ldr, kept._codes_ptr, kept._exps_ptr, KINDS[kept.kind], at,
          at + 4 * rows, weight.data_ptr(), rows, d, gx.data_ptr(), _DTYPES[kept.dtype], d, _ptr(gw), _ptr(gb), _ptr(ws), n)
    return gx, gw, gb


class _LayerNorm8(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, out_dtype, kind):
        ctx.set_materialize_grads(False)
        y, z, saved = layer_norm8_forward(x, weight, bias, eps, residual, out_dtype, kind)
        ctx.save_for_backward(saved.kept.codes, saved.kept.exps, saved.stats, weight)
        ctx.kept = kind, saved.kept.shape, saved.kept.dtype
        ctx.y_dtype, ctx.has = y.dtype, (bias is not None, residual is not None)
        return (y, z) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gz=None):
        codes, exps, stats, weight = ctx.saved_tensors
        kept = Checkpoint8(codes, exps, *ctx.kept)
        if gy is None:
            gy = torch.zeros(kept.shape, dtype=ctx.y_dtype, device=kept.device)
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gx, gw, gb = layer_norm8_backward(gy, LayerNorm8Saved(kept, stats), weight, gz, params)
        has_bias, has_residual = ctx.has
        return gx, gw, gb if has_bias else None, gx if has_residual else None, None, None, None


def layer_norm8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, kind: str = "int8"):
    """Differentiable LayerNorm that keeps its input in 8 bits.  Returns y, with a residual (y, z): z = x + residual is the new residual
    stream, whose own gradient is added in the same pass."""
    return _LayerNorm8.apply(x, weight, bias, residual, eps, out_dtype, kind)


# ------------------------------------------------------------------ linear
def linear8_weight_grad(gy: torch.Tensor, kept: Checkpoint8, bias: bool = True):
    """(g_weight (n, k), g_bias (n) or None) in fp32 of y = x w^T + b, from gy (..., n) float16 or bfloat16 and x (..., k) in 8 bits.

    x enters the product as ``kept.expand(gy.dtype)`` has it.  That is exact for a bfloat16 gy and for a float16 gy with a float16 activation down to
    fp16's smallest step; a float16 gy takes what a float32 or bfloat16 activation holds past 65,504 as infinity, and below 2^-25 as
    zero.  Such activations want a bfloat16 gy, or to be scaled ahead of ``pack8``."""
    if gy.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"gy must be float16 or bfloat16, got {gy.dtype}")
    if gy.shape[:-1] != kept.shape[:-1] or gy.device != kept.device:
        raise ValueError(f"gy must be {kept.shape[:-1]} x n on {kept.device}, got {tuple(gy.shape)} on {gy.device}")
    m, rows, n, ld = _rows(gy, "gy")
    k, dev = kept.shape[-1], gy.device
    gw = torch.empty(n, k, dtype=torch.float32, device=dev)
    gb = torch.empty(n, dtype=torch.float32, device=dev) if bias else None
    size = _workspace_bytes("bsrl_linear8_wgrad_workspace_bytes", dev.index, rows, n, k, int(m.data_ptr() % 16 == 0 and ld % 8 == 0))
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _call(nat.lib.bsrl_linear8_wgrad, dev, m.data_ptr(), _DTYPES[gy.dtype], ld, kept._codes_ptr, kept._exps_ptr, KINDS[kept.kind], rows, n, k,
          gw.data_ptr(), _ptr(gb), _ptr(ws), size)
    return gw, gb


def _on_16(t: torch.Tensor) -> torch.Tensor:
    """t without gaps and from a 16-byte boundary on, as the products read it: a copy where it is not (a slice of something larger)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _product(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    """a (m, k) w (n, k)^T + bias in fp16."""
    a, w, bias = _on_16(a), _on_16(w), None if bias is None else _on_16(bias)
    m, k = a.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=torch.float16, device=a.device)
    if m:
        _call(nat.lib.bsrl_linear, a.device, a.data_ptr(), w.data_ptr(), _ptr(bias), None, out.data_ptr(), 0, 0, m, n, k,
              int(k % 64 == 0 and n % 16 == 0))
    return out


class _Linear8(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kind):
        n, k = weight.shape
        w = weight.to(torch.float16)
        y = _product(x.reshape(-1, k), w, bias)
        kept = pack8(x, kind)
        ctx.save_for_backward(kept.codes, kept.exps, w)
        ctx.kept, ctx.w_dtype = (kind, kept.shape, kept.dtype), weight.dtype
        return y.view(*x.shape[:-1], n)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        codes, exps, w = ctx.saved_tensors
        n, k = w.shape
        kept = Checkpoint8(codes, exps, *ctx.kept)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        gx = gw = gb = None
        if need_x:
            gx = _product(gy.reshape(-1, n), w.t(), None).view(kept.shape)
        if need_w or need_b:
            gw, gb = linear8_weight_grad(gy, kept, need_b)
        return gx, gw.to(ctx.w_dtype) if need_w else None, gb, None


def linear8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, kind: str = "int8") -> torch.Tensor:
    """Differentiable y = x weight^T + bias that keeps x in 8 bits.

    x (..., k) and y are float16, weight (n, k) float16 or a float32 master (rounded to float16 for the products; its gradient is
    float32), bias (n) float32.  n and k multiples of 32 (the products' own limits) up to 2^20."""
    if not x.is_cuda:
        raise RuntimeError("x must live on a CUDA device (this library has no CPU path)")
    if x.dtype != torch.float16 or weight.dtype not in (torch.float16, torch.float32):
        raise TypeError(f"x must be float16 and weight float16 or float32, got {x.dtype} and {weight.dtype}")
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1] or weight.device != x.device:
        raise ValueError(f"weight must be (n, {tuple(x.shape)[-1:]}) on {x.device}, got {tuple(weight.shape)} on {weight.device}")
    if weight.shape[0] % 32 or weight.shape[1] % 32 or not weight.numel() or max(weight.shape) > 1 << 20 or weight.numel() > 1 << 31:
        raise ValueError(f"weight's sides must be multiples of 32 up to 2^20, their product at most 2^31, got {tuple(weight.shape)}")
    return _Linear8.apply(x, weight, _vector(bias, weight.shape[0], x.device, "bias"), kind)
