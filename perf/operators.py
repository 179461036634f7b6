"""Measured cases of the 4-bit block floating-point operators.

Rows are held as E2M1 codes (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2,
3, 4, 6) with one scale for every `block` consecutive elements of a row:
  block 32: the scale is a power of two, 2^(floor(log2 amax) - 2), held in 8 bits (E8M0);
  block 16: the scale is amax / 6 rounded to E4M3 (4 significant bits, at most 448).
An element x * alpha is rounded to the nearest code times scale, ties to the even code,
saturating at 6 scales.  Three operators are measured:
  store    quantize_fp4 then dequantize_fp4: rows in, the values they are held as out
  read     dequantize_fp4 of rows that are held in 4 bits
  product  product_fp4 of queries (quantised within the call) with rows held in 4 bits

`own` chooses between the framework's kernels and the plain form of the same arithmetic.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # 64 new vectors of a 96-dimensional collection entering the store: latency.
        dict(name="store_64x96", op="store", n=64, dim=96, block=32, dtype="float32", out="float32", data="unit",
             alpha=1.0),
        # A whole collection of 1M x 128 vectors brought into 4 bits and read back to see what it lost.
        dict(name="store_1Mx128", op="store", n=1_000_000, dim=128, block=32, dtype="float32", out="float32",
             data="mixture", alpha=1.0),
        # Embeddings in bf16, an odd count of them, 300 wide (the last block of a row is short).
        dict(name="store_50021x300_bf16", op="store", n=50_021, dim=300, block=16, dtype="bfloat16", out="bfloat16",
             data="normal", alpha=16.0),
        # Reading a collection of 96-dimensional unit vectors back for exact re-ranking.
        dict(name="read_1Mx96", op="read", n=1_000_000, dim=96, block=32, dtype="float32", out="float16", data="unit",
             alpha=1.0),
        # A short candidate list of wide rows read back.
        dict(name="read_777x1000", op="read", n=777, dim=1000, block=16, dtype="float32", out="bfloat16",
             data="normal", alpha=16.0),
        # A few queries against 1000 cluster centroids: the smallest product, latency only.
        dict(name="product_8x1000x128", op="product", m=8, n=1000, dim=128, block=32, dtype="float32", out="float32",
             data="mixture", alpha=1.0),
        # One query scored against every one of 1M x 128 rows.
        dict(name="product_1x1Mx128", op="product", m=1, n=1_000_000, dim=128, block=32, dtype="float32",
             out="float32", data="mixture", alpha=1.0),
        # One token through a square layer whose weights are held in 4 bits.
        dict(name="product_1x8192x8192", op="product", m=1, n=8192, dim=8192, block=16, dtype="bfloat16",
             out="bfloat16", data="normal", alpha=16.0),
        # An odd batch against an odd number of rows of odd width.
        dict(name="product_333x77777x200", op="product", m=333, n=77_777, dim=200, block=16, dtype="float16",
             out="float16", data="normal", alpha=16.0),
        # 10k queries scored against 100k x 128 rows: the scores themselves are most of the traffic.
        dict(name="product_10000x100000x128", op="product", m=10_000, n=100_000, dim=128, block=32, dtype="float32",
             out="float32", data="mixture", alpha=1.0),
        # A prompt of 4096 tokens through a wide layer.
        dict(name="product_4096x16384x4096", op="product", m=4096, n=16_384, dim=4096, block=16, dtype="bfloat16",
             out="bfloat16", data="normal", alpha=16.0),
        # The largest matrix product: all arithmetic.
        dict(name="product_8192x8192x8192", op="product", m=8192, n=8192, dim=8192, block=32, dtype="bfloat16",
             out="bfloat16", data="normal", alpha=1.0),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "read", "product", "product", "product"])
    block = rng.choice([16, 32])
    c = dict(op=op, dim=_loguniform(rng, 8, 8192), block=block, dtype=rng.choice(list(_DT)), out=rng.choice(list(_DT)),
             data=rng.choice(["unit", "normal", "mixture"]), alpha=16.0 if block == 16 else 1.0)
    if c["data"] == "mixture":
        c["alpha"] = 1.0
        c["out"] = "float32" if op == "product" else c["out"]  # scores of raw byte-range vectors pass fp16's range
    if op != "product":
        c["n"] = _loguniform(rng, 1, max(1, min(1_000_000, 128_000_000 // c["dim"])))
        return c
    c["m"] = _loguniform(rng, 1, 10_000)
    # rows: at most 1M, 128M elements, 1e9 scores and 8192^3 multiplications
    most = min(1_000_000, 128_000_000 // c["dim"], 1_000_000_000 // c["m"], 8192 ** 3 // (c["m"] * c["dim"]))
    c["n"] = _loguniform(rng, 1, max(1, most))
    return c


def _data(kind, n, dim, gen):
    """Vectors as the framework's collections hold them, fp32 on the GPU."""
    if kind == "mixture":  # non-negative byte-range features around cluster centres
        centres = torch.rand(100, dim, generator=gen, device="cuda") * 255.0
        pick = torch.randint(0, 100, (n,), generator=gen, device="cuda")
        x = torch.randn(n, dim, generator=gen, device="cuda")
        return x.mul_(20.0).add_(centres[pick]).clamp_(min=0.0)
    x = torch.randn(n, dim, generator=gen, device="cuda")
    if kind == "unit":
        x.div_(x.norm(dim=1, keepdim=True).clamp_(min=1e-20))
    return x


# ------------------------------------------------------------------ plain form

def _quantise(x, alpha, block):
    """Codes as signed values (n x padded dim fp32) and scales (n x blocks fp32)."""
    n, dim = x.shape
    nb = (dim + block - 1) // block
    v = torch.zeros(n, nb * block, dtype=torch.float32, device=x.device)
    v[:, :dim] = x.float() * alpha
    v = v.view(n, nb, block)
    amax = v.abs().amax(dim=2)
    if block == 32:
        # 2^(floor(log2 amax) - 2): the float's exponent field less 2 (a block of zeros gets 0)
        scale = (((amax.view(torch.int32) >> 23) - 2).clamp(min=0) << 23).view(torch.float32)
    else:
        scale = (amax / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    y = v.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))[:, :, None]
    y = torch.where(scale[:, :, None] > 0, y, torch.zeros_like(y))
    code = (0.5 * ((y > 0.25).float() + (y >= 0.75).float() + (y > 1.25).float() + (y >= 1.75).float())
            + (y > 2.5).float() + (y >= 3.5).float() + 2.0 * (y > 5.0).float())
    return torch.copysign(code, v).view(n, nb * block), scale


def _pack(code, scale, block):
    """Plain storage of quantised rows: two codes to a byte, one byte per scale."""
    mags = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    parts = []
    for c in code.split(max(1, (1 << 26) // code.shape[1])):
        nib = torch.bucketize(c.abs(), mags).to(torch.uint8) | (torch.signbit(c).to(torch.uint8) << 3)
        parts.append(nib[:, 0::2] | (nib[:, 1::2] << 4))
    if block == 32:
        s8 = (scale.view(torch.int32) >> 23).to(torch.uint8)
    else:
        s8 = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.cat(parts), s8


def _values(codes, s8, block, dim):
    """The fp32 values of rows in the plain storage."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    n = codes.shape[0]
    v = torch.empty(n, codes.shape[1], 2, device=codes.device)
    v[:, :, 0] = table[(codes & 15).int()]
    v[:, :, 1] = table[(codes >> 4).int()]
    if block == 32:
        scale = (s8.int() << 23).view(torch.float32)
    else:
        scale = s8.view(torch.float8_e4m3fn).float()
    return (v.view(n, -1, block) * scale[:, :, None]).view(n, -1)[:, :dim]


# ------------------------------------------------------------------ the cases

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = _data(case["data"], case["n"], case["dim"], gen).to(_DT[case["dtype"]])
    state = dict(case)
    if case["op"] == "store":
        state["x"] = x
        return state
    if case["op"] == "product":
        state["q"] = _data(case["data"], case["m"], case["dim"], gen).to(_DT[case["dtype"]])
    if own:
        import garfield_b200 as gf
        state["rows"] = gf.quantize_fp4(x, alpha=case["alpha"], block=case["block"])
    else:
        parts = [_pack(*_quantise(c, case["alpha"], case["block"]), case["block"])
                 for c in x.split(max(1, (1 << 26) // case["dim"]))]
        state["rows"] = tuple(torch.cat(p) for p in zip(*parts))
    return state


def run(state):
    op, block, alpha, dim = state["op"], state["block"], state["alpha"], state["dim"]
    out = _DT[state["out"]]
    if own:
        import garfield_b200 as gf
        if op == "store":
            return gf.dequantize_fp4(gf.quantize_fp4(state["x"], alpha=alpha, block=block), dtype=out)
        if op == "read":
            return gf.dequantize_fp4(state["rows"], dtype=out)
        return gf.product_fp4(state["q"], state["rows"], dtype=out, query_alpha=alpha)
    if op == "store":
        code, scale = _quantise(state["x"], alpha, block)
        v = (code.view(code.shape[0], -1, block) * scale[:, :, None]).view(code.shape[0], -1)[:, :dim]
        return (v / alpha).to(out)
    v = _values(*state["rows"], block, dim) / alpha
    if op == "read":
        return v.to(out)
    code, scale = _quantise(state["q"], alpha, block)
    q = (code.view(code.shape[0], -1, block) * scale[:, :, None]).view(code.shape[0], -1)[:, :dim] / alpha
    return (q @ v.t()).to(out)


def work(case):
    es, os_ = torch.finfo(_DT[case["dtype"]]).bits // 8, torch.finfo(_DT[case["out"]]).bits // 8
    n, dim, block = case["n"], case["dim"], case["block"]
    held = n * ((dim + block - 1) // block) * (block // 2 + 1)
    if case["op"] == "store":  # the rows in, what is held written and read, the values out
        return {"bytes": n * dim * (es + os_) + 2 * held, "flops": 2 * n * dim}
    if case["op"] == "read":
        return {"bytes": held + n * dim * os_, "flops": n * dim}
    m = case["m"]
    return {"bytes": m * dim * es + held + m * n * os_, "flops": 2 * m * n * dim}


# ------------------------------------------------------------------ from the definition, in 64 bits

def _held(x, alpha, block):
    """The values that rows are held as, by the format's definition, in 64 bits."""
    n, dim = x.shape
    pad = -dim % block
    v = torch.nn.functional.pad((x.float() * alpha).double(), (0, pad)).unflatten(1, (-1, block))
    amax = v.abs().amax(2, keepdim=True)
    if block == 32:
        ex = torch.floor(torch.log2(torch.where(amax > 0, amax, 1.0)))
        ex = torch.where(torch.exp2(ex) > amax, ex - 1, ex)
        ex = torch.where(torch.exp2(ex + 1) <= amax, ex + 1, ex)
        s = torch.where(amax > 0, torch.exp2((ex - 2).clamp(-127, 127)), 2.0 ** -127)
    else:
        t = (amax / 6).clamp(max=448.0)
        step = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)  # E4M3: 8 steps to a binade
        s = (torch.round(t / step) * step).clamp(max=448.0)
    y = torch.where(s > 0, v.abs() / torch.where(s > 0, s, 1.0), 0.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return (torch.sign(v) * y * s).flatten(1)[:, :dim] / alpha


def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = _data(case["data"], case["n"], case["dim"], gen).to(_DT[case["dtype"]])
    parts = x.split(max(1, (1 << 26) // case["dim"]))
    if case["op"] != "product":
        return torch.cat([_held(c, case["alpha"], case["block"]) for c in parts])
    q = _held(_data(case["data"], case["m"], case["dim"], gen).to(_DT[case["dtype"]]), case["alpha"], case["block"])
    res = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
    at = 0
    for c in parts:
        res[:, at:at + c.shape[0]] = q @ _held(c, case["alpha"], case["block"]).t()
        at += c.shape[0]
    return res
