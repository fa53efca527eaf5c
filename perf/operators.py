"""Training operators that keep their saved activations in 8 bits, as cases that can be timed and compared.

A case names an operator (``op``), its sizes and its types:

* ``norm``    LayerNorm's training step: forward (with the residual sum in front of it where ``residual`` is set), whose input is
              kept in 8 bits, and backward (input gradient with the residual stream's own gradient added, weight and bias gradient);
* ``gelu``    the same for the exact GELU: forward keeps its input in 8 bits, backward reads it;
* ``pack``    an activation put into 8 bits and taken out again, from rows ``pitch`` elements apart;
* ``weight``  a linear layer's weight and bias gradient from an input that was kept in 8 bits.

8 bits: blocks of 32 neighbouring values of a row share a power of two, 2^e, and hold codes, int8 in [-127, 127] or e4m3 in
[-240, 240]; e is the least one for which the code of the block's largest magnitude stays in that range.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32
UPDATE_ROWS = 29 * 16384                  # token rows of a minibatch of 16,384 environments
NORM_ELEMENTS = UPDATE_ROWS * 256         # the largest listed case of each operator
GELU_ELEMENTS = UPDATE_ROWS * 1024
PACK_ELEMENTS = UPDATE_ROWS * 512
WEIGHT_PRODUCTS = UPDATE_ROWS * 1024 * 256
EPS = 1e-5


def listed():
    return [
        # one environment's 29 token rows at the headline width: what a call costs where nothing else does
        dict(name="norm_one_env", op="norm", rows=29, d=256, x="f32", y="f16", residual=False, kind="int8"),
        # the policy update's LayerNorm: fp32 residual stream in, fp16 rows out
        dict(name="norm_update", op="norm", rows=UPDATE_ROWS, d=256, x="f32", y="f16", residual=False, kind="int8"),
        # wide rows of a 16-bit residual stream, the sum in front of the norm
        dict(name="norm_stream", op="norm", rows=65536, d=1024, x="bf16", y="bf16", residual=True, kind="e4m3"),
        # a width that no vector divides
        dict(name="norm_odd", op="norm", rows=10007, d=1001, x="f16", y="f16", residual=True, kind="int8"),
        # the FFN's hidden rows of one environment
        dict(name="gelu_one_env", op="gelu", rows=29, d=1024, x="f16", kind="int8"),
        # and of an update's minibatch
        dict(name="gelu_update", op="gelu", rows=UPDATE_ROWS, d=1024, x="f16", kind="int8"),
        # rows that no vector divides
        dict(name="gelu_odd", op="gelu", rows=30011, d=1363, x="bf16", kind="e4m3"),
        # observations of a few environments
        dict(name="pack_obs", op="pack", rows=512, d=630, pitch=630, x="f32", kind="e4m3"),
        # two thirds of the packed projection's rows
        dict(name="pack_slice", op="pack", rows=UPDATE_ROWS, d=512, pitch=768, x="bf16", kind="int8"),
        # the packed projection's weight over the rows of 64 environments
        dict(name="weight_few", op="weight", rows=29 * 64, n=768, k=256, g="f16", kind="int8"),
        # the FFN-up's weight in an update
        dict(name="weight_update", op="weight", rows=UPDATE_ROWS, n=1024, k=256, g="f16", kind="int8"),
        # an odd number of rows, widths that no tile divides
        dict(name="weight_odd", op="weight", rows=100003, n=1000, k=513, g="bf16", kind="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gelu", "pack", "weight"])
    kind = rng.choice(["int8", "e4m3"])
    if op == "weight":
        n, k = _log(rng, 8, 2048), _log(rng, 8, 2048)
        if rng.random() < 0.7:
            n = -(-n // 8) * 8
        rows = _log(rng, 1, min(UPDATE_ROWS, WEIGHT_PRODUCTS // (n * k)))
        return dict(op=op, rows=rows, n=n, k=k, g=rng.choice(["f16", "bf16"]), kind=kind)
    x = rng.choice(["f32", "f16", "bf16"])
    d = _log(rng, 8, 8192)
    if rng.random() < 0.7:
        d = -(-d // 8) * 8
    most = {"norm": NORM_ELEMENTS, "gelu": GELU_ELEMENTS, "pack": PACK_ELEMENTS}[op] // (2 if x == "f32" else 1)
    rows = _log(rng, 1, min(UPDATE_ROWS, most // (2 * d)))
    if op == "norm":
        y = rng.choice(["f32", "f16", "bf16"]) if x == "f32" else x
        return dict(op=op, rows=rows, d=d, x=x, y=y, residual=rng.random() < 0.5, kind=kind)
    if op == "gelu":
        return dict(op=op, rows=rows, d=d, x=x, kind=kind)
    return dict(op=op, rows=rows, d=d, pitch=d + rng.choice([0, 0, 8, rng.randrange(1, d + 1)]), x=x, kind=kind)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    rows = case["rows"]
    if case["op"] == "weight":
        n, k = case["n"], case["k"]
        return {"bytes": rows * (2 * n + k + -(-k // BLOCK)) + 4 * n * (k + 1), "flops": 2 * rows * n * k + rows * n}
    d, x = case["d"], size[case["x"]]
    kept = rows * (d + -(-d // BLOCK))                  # the codes and exponents: written once, read once
    if case["op"] == "norm":
        y = size[case["y"]]
        stream = 3 * x if case["residual"] else 0       # the branch and the stream's gradient in, the new stream out
        return {"bytes": rows * d * (2 * x + 2 * y + stream) + 2 * kept + 2 * 8 * rows + 16 * d, "flops": 25 * rows * d}
    if case["op"] == "gelu":
        return {"bytes": rows * d * 4 * x + 2 * kept, "flops": 60 * rows * d}
    return {"bytes": rows * d * 2 * x + 2 * kept, "flops": 6 * rows * d}


# ---------------------------------------------------------------- 8 bits, in plain operations
def _blocks(x):
    """(rows, d) -> (rows, blocks, 32), zeros behind the last value."""
    rows, d = x.shape
    return torch.nn.functional.pad(x, (0, -d % BLOCK)).view(rows, -1, BLOCK)


def _power(e):
    """2^e, for e in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _exponents(blocks, kind, dtype):
    """e of every block (as int32) of values that came in `dtype`; the blocks that stand for zeros are marked by e = -127."""
    most = blocks.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(most)                            # most = m 2^e, 0.5 <= m < 1
    if kind == "int8":
        e = e - 7 + (m >= 127.5 / 128).int()
        e = e.clamp(max=math.frexp(torch.finfo(dtype).max)[1] - 7)
    else:
        e = e - 8 + (m >= 248 / 256).int()
        e = e.clamp(max=math.frexp(torch.finfo(dtype).max)[1] - 8)
    return torch.where((most == 0) | (e < -126), -127, e)


def _codes(x, kind):
    """Codes and biased exponents (uint8) of x (rows, d)."""
    b = _blocks(x.float())
    e = _exponents(b, kind, x.dtype)
    t = torch.where(e == -127, 0.0, b * _power(-e))
    if kind == "int8":
        q = torch.round(t).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        q = t.clamp(-240, 240).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.reshape(x.shape[0], -1), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, exps, kind, d):
    """What codes and exponents stand for, in 32 bits."""
    rows = codes.shape[0]
    q = codes.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn).float().view(rows, -1, BLOCK)
    scale = torch.where(exps == 0, 0.0, _power(exps.int() - 127))
    return (q * scale.unsqueeze(-1)).view(rows, -1)[:, :d]


# ---------------------------------------------------------------- what a user's program has in hand
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = case["rows"]

    def rand(*shape, dtype):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    if case["op"] == "weight":
        x = rand(rows, case["k"], dtype=DTYPES[case["g"]])
        codes, exps = _codes(x, case["kind"])
        return dict(case, codes=codes, exps=exps, gy=rand(rows, case["n"], dtype=DTYPES[case["g"]]))
    d, dt = case["d"], DTYPES[case["x"]]
    if case["op"] == "pack":
        # rows of different size, as a residual stream's are
        wide = torch.randn(rows, case["pitch"], generator=g, device="cuda")
        wide *= torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
        return dict(case, x=wide.to(dt)[:, :d])
    if case["op"] == "gelu":
        return dict(case, x=(1.5 * torch.randn(rows, d, generator=g, device="cuda")).to(dt), gy=rand(rows, d, dtype=dt))
    out = DTYPES[case["y"]]
    s = dict(case, x=(2 * torch.randn(rows, d, generator=g, device="cuda") + 0.5).to(dt), gy=rand(rows, d, dtype=out),
             weight=1 + 0.1 * rand(d, dtype=torch.float32), bias=0.1 * rand(d, dtype=torch.float32), out=out)
    if case["residual"]:
        s.update(branch=rand(rows, d, dtype=dt), g_stream=rand(rows, d, dtype=dt))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if s["op"] == "weight":
        gy = s["gy"].float()
        return gy.t() @ _values(s["codes"], s["exps"], kind, s["k"]), gy.sum(0)
    x = s["x"]
    if s["op"] == "pack":
        return _values(*_codes(x, kind), kind, s["d"]).to(x.dtype)
    if s["op"] == "gelu":
        v = x.float()
        y = 0.5 * v * torch.erfc(v * -math.sqrt(0.5))
        kept = _codes(x, kind)
        v = _values(*kept, kind, s["d"])
        slope = 0.5 * torch.erfc(v * -math.sqrt(0.5)) + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
        return y.to(x.dtype), (s["gy"].float() * slope).to(x.dtype)
    z = (x.float() + s["branch"].float()).to(x.dtype) if s["residual"] else x
    v = z.float()
    mean = v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + EPS)
    y = ((v - mean) * rstd * s["weight"] + s["bias"]).to(s["out"])
    kept = _codes(z, kind)
    h = (_values(*kept, kind, s["d"]) - mean) * rstd
    gy = s["gy"].float()
    gh = gy * s["weight"]
    gx = rstd * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True))
    if s["residual"]:
        gx = gx + s["g_stream"].float()
        return y, z, gx.to(x.dtype), (gy * h).sum(0), gy.sum(0)
    return y, gx.to(x.dtype), (gy * h).sum(0), gy.sum(0)


def _run_own(s):
    from beatsaberrl_b200 import checkpoint8 as c8
    kind = s["kind"]
    if s["op"] == "weight":
        kept = c8.Checkpoint8(s["codes"], s["exps"], kind, (s["rows"], s["k"]), s["gy"].dtype)
        return c8.linear8_weight_grad(s["gy"], kept)
    if s["op"] == "pack":
        return c8.pack8(s["x"], kind).expand()
    if s["op"] == "gelu":
        y, kept = c8.gelu8_forward(s["x"], kind)
        return y, c8.gelu8_backward(s["gy"], kept)
    y, z, saved = c8.layer_norm8_forward(s["x"], s["weight"], s["bias"], EPS, residual=s.get("branch"), out_dtype=s["out"], kind=kind)
    gx, gw, gb = c8.layer_norm8_backward(s["gy"], saved, s["weight"], g_residual=s.get("g_stream"))
    return (y, z, gx, gw, gb) if s["residual"] else (y, gx, gw, gb)


# ---------------------------------------------------------------- the definitions in 64 bits
def _kept64(x, kind):
    """What x (rows, d) stands for once it was kept in 8 bits, from the definition: the least power of two with which every code of
    a block lies in its range, found from the largest magnitude; codes to nearest, ties to even."""
    top = torch.finfo(x.dtype).max
    rows, d = x.shape
    n = -(-d // BLOCK)
    v = torch.zeros(rows, n * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :d] = x
    v = v.view(rows, n, BLOCK)
    big = v.abs().max(-1, keepdim=True).values
    limit, digits = (127.0, None) if kind == "int8" else (240.0, 4)

    def two(e):                                         # 2^e, exactly
        return ((e.long() + 1023) << 52).view(torch.float64)

    def to_grid(t):
        if digits is None:
            return torch.round(t)
        power = torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6)))
        power = torch.where(two(power + 1) <= t.abs(), power + 1, power)
        power = torch.where((two(power) > t.abs()) & (power > -6), power - 1, power)
        step = two(power - digits + 1)
        return torch.round(t / step) * step

    e = torch.floor(torch.log2(torch.where(big == 0, 1.0, big) / limit))
    e = torch.where(to_grid(big * two(-e)) > limit, e + 1, e)
    e = torch.minimum(e, torch.full_like(e, math.floor(math.log2(top)) - math.floor(math.log2(limit))))
    q = to_grid(v * two(-e)).clamp(-limit, limit)
    return torch.where((big == 0) | (e < -126), 0.0, q * two(e)).view(rows, -1)[:, :d]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "weight":
        q, w = s["codes"], s["exps"].int() - 127
        q = q.view(torch.int8).double() if case["kind"] == "int8" else q.view(torch.float8_e4m3fn).double()
        x = (q * torch.repeat_interleave(torch.where(w == -127, 0.0, _power(w).double()), BLOCK, 1))[:, :case["k"]]
        gy = s["gy"].double()
        return torch.matmul(gy.T, x), gy.sum(0)
    x = s["x"]
    if case["op"] == "pack":
        return _kept64(x, case["kind"])
    if case["op"] == "gelu":
        a = x.double()
        y = a * torch.special.ndtr(a)
        del a
        a = _kept64(x, case["kind"])
        return y, (torch.special.ndtr(a) + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)) * s["gy"].double()
    z = x
    if case["residual"]:
        z = (x.double() + s["branch"].double()).to(x.dtype)     # the sum of two such numbers, in 64 bits exact for what is drawn
    a, w, g = z.double(), s["weight"].double(), s["gy"].double()
    mu = a.sum(1, keepdim=True) / case["d"]
    sd = torch.sqrt((a * a).sum(1, keepdim=True) / case["d"] - mu * mu + EPS)
    y = (a - mu) / sd * w + s["bias"].double()
    a = (_kept64(z, case["kind"]) - mu) / sd
    gw = g * w
    gx = (gw - gw.sum(1, keepdim=True) / case["d"] - a * ((gw * a).sum(1, keepdim=True) / case["d"])) / sd
    if case["residual"]:
        return y, z.double(), gx + s["g_stream"].double(), (g * a).sum(0), g.sum(0)
    return y, gx, (g * a).sum(0), g.sum(0)
