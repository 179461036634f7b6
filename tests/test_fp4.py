"""4-bit block floating point on the host: the held values against the format's definition in 64
bits, the packed byte positions, non-finite blocks and refusals."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import garfield_b200 as gf

MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """All finite non-negative E4M3 values by code."""
    v = [m / 8 * 2.0 ** -6 for m in range(8)]
    v += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return np.array(v[:127])


def nearest_even(x, table):
    """Index of the table value nearest to x (x >= 0, ascending table), ties to the even index."""
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    lo = hi - 1
    dl, dh = x - table[lo], table[hi] - x
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def held(x, alpha, block):
    """codes (signed values), scales and held values of float32 rows, from the definition in 64 bits."""
    n, dim = x.shape
    nb = -(-dim // block)
    v = np.zeros((n, nb * block))
    v[:, :dim] = (x.astype(np.float32) * np.float32(alpha)).astype(np.float64)
    v = v.reshape(n, nb, block)
    amax = np.abs(v).max(2)
    if block == 32:
        e = np.where(amax > 0, np.frexp(amax)[1] - 3, -127)
        s = 2.0 ** np.clip(e, -127, 127)
    else:
        t = e4m3_values()
        s = t[nearest_even(np.minimum(amax / 6, 448.0), t)]
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(s[:, :, None] > 0, np.abs(v) / s[:, :, None], 0.0)
    code = np.copysign(MAGS[nearest_even(np.minimum(y, 6.0), MAGS)], v)
    return code.reshape(n, -1), s, ((code * s[:, :, None]).reshape(n, -1)[:, :dim]) / alpha


def data(n, dim, seed, kind):
    rng = np.random.default_rng(seed)
    if kind == "normal":
        return rng.standard_normal((n, dim)).astype(np.float32)
    if kind == "wide":  # magnitudes over many binades, both signs, some zeros and whole zero rows
        x = rng.standard_normal((n, dim)) * 2.0 ** rng.uniform(-20, 8, (n, dim))
        x[rng.random((n, dim)) < 0.1] = 0.0
        x[rng.random((n, dim)) < 0.05] = -0.0
        x[::7] = 0.0
        return x.astype(np.float32)
    # values on and next to the borders between codes: border * scale, one ulp below and above
    b = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 4.0])
    x = (rng.choice(b, (n, dim)) * rng.choice([-1.0, 1.0], (n, dim))).astype(np.float32)
    x[:, 0] = 6.0
    y = np.nextafter(x, np.float32(0.0))
    z = np.nextafter(x, np.float32(9.0) * np.sign(x))
    pick = rng.integers(0, 3, (n, dim))
    return np.where(pick == 0, x, np.where(pick == 1, y, z)).astype(np.float32)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("alpha", [1.0, 16.0, 0.3])
@pytest.mark.parametrize("kind", ["normal", "wide", "borders"])
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 96), (130, 33), (5, 300), (129, 128)])
def test_host_values_match_definition(n, dim, kind, alpha, block):
    x = data(n, dim, n * 1000 + dim, kind)
    got = gf.dequantize_fp4_host(gf.quantize_fp4_host(x, alpha, block))
    _, _, want = held(x, alpha, block)
    if alpha == 0.3:  # alpha is rounded to fp32; 1 / alpha, times s, times the code: 3 * 2^-24
        a32 = float(np.float32(alpha))
        want = want * alpha / a32
        assert np.all(np.abs(got - want) <= 3 * 2.0 ** -24 * (1 + 2.0 ** -22) * np.abs(want) + 1e-45)
    else:
        assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("block", [16, 32])
def test_packed_positions(block):
    """Each code and scale stands where the header says."""
    n, dim = 200, 300
    x = data(n, dim, 5, "wide")
    rows = gf.quantize_fp4_host(x, 1.0, block)
    code, s, _ = held(x, 1.0, block)
    sub = 512 * (32 // block)
    panel = 3 * sub + 10 * 2048  # 300 elements: 3 groups' scales, 10 columns
    assert rows.packed.size == gf.lib().gf_fp4_bytes(n, dim, block) == 2 * panel
    t = e4m3_values()
    for i in (0, 1, 31, 32, 100, 127, 128, 199):
        for k in (0, 1, 15, 16, 31, 32, 97, 127, 128, 255, 256, 299):
            base, r = (i // 128) * panel, i % 128
            byte = rows.packed[base + 3 * sub + (k // 32) * 2048 + r * 16 + (k % 32) // 2]
            nib = (byte >> (4 * (k & 1))) & 15
            c = code[i, k]
            assert MAGS[nib & 7] == abs(c) and bool(nib & 8) == bool(np.signbit(c))
            b = k // block
            s8 = rows.packed[base + (b // 4) * 512 + (r % 32) * 16 + (r // 32) * 4 + b % 4]
            assert (t[s8] if block == 16 else 2.0 ** (int(s8) - 127)) == s[i, k // block]
    assert not rows.packed[panel + 3 * sub + (200 - 128) * 16:panel + 3 * sub + 2048].any()  # rows past n


@pytest.mark.parametrize("n,h", [(1, 16), (16, 16), (17, 32), (100, 112), (113, 128), (127, 128)])
def test_short_panel(n, h):
    """Fewer than 128 rows make one panel of their number rounded up to 16."""
    x = data(n, 70, n, "normal")
    rows = gf.quantize_fp4_host(x)
    assert rows.packed.size == 512 + 3 * h * 16
    code, _, _ = held(x, 1.0, 32)
    for k in (0, 31, 40, 69):
        byte = rows.packed[512 + (k // 32) * h * 16 + (n - 1) * 16 + (k % 32) // 2]
        nib = (byte >> (4 * (k & 1))) & 15
        assert MAGS[nib & 7] == abs(code[n - 1, k])
    assert np.array_equal(gf.dequantize_fp4_host(rows), held(x, 1.0, 32)[2].astype(np.float32))


def test_extremes():
    """The ends of fp32's range hold in blocks of 32; E4M3's range bounds blocks of 16."""
    x = np.zeros((4, 32), np.float32)
    x[0, :2] = [np.finfo(np.float32).max, -1e38]
    x[1, :2] = [2.0 ** -126, 2.0 ** -128]
    x[2, :2] = [1e-45, -1e-45]
    x[3, :2] = [1e5, 10.0]
    got = gf.dequantize_fp4_host(gf.quantize_fp4_host(x, 1.0, 32))
    assert np.array_equal(got, held(x, 1.0, 32)[2].astype(np.float32))
    got = gf.dequantize_fp4_host(gf.quantize_fp4_host(x, 1.0, 16))
    assert got[3, 0] == 6 * 448 and got[3, 1] == 0.0 and not got[1].any()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_block_reads_nan(block, bad):
    x = np.ones((3, 80), np.float32)
    x[1, 35] = bad
    got = gf.dequantize_fp4_host(gf.quantize_fp4_host(x, 1.0, block))
    want = np.ones((3, 80), bool)
    want[1, 32:32 + block] = False
    assert np.array_equal(np.isfinite(got), want)
    assert np.isnan(got[1, 32:32 + block]).all()


def test_empty():
    r = gf.quantize_fp4_host(np.zeros((0, 7), np.float32))
    assert r.packed.size == 0 and gf.dequantize_fp4_host(r).shape == (0, 7)


def test_sizes_agree():
    """The size that Python allocates is gf_fp4_bytes."""
    for n in (0, 1, 15, 16, 17, 100, 127, 128, 129, 1000, 2 ** 31):
        for dim in (1, 31, 32, 33, 128, 129, 300, 8192, 100_000):
            for block in (16, 32):
                assert gf._fp4_size(n, dim, block) == gf.lib().gf_fp4_bytes(n, dim, block)


def test_size_of_bad_shapes():
    L = gf.lib()
    assert L.gf_fp4_bytes(5, 0, 32) == 0 and L.gf_fp4_bytes(5, 8, 8) == 0
    assert L.gf_fp4_bytes(2 ** 32 - 1, 2 ** 32 - 1, 32) > 2 ** 62


@pytest.mark.parametrize("args,word", [
    (dict(dim=0), b"dim"), (dict(block=64), b"block"), (dict(alpha=0.0), b"alpha"), (dict(alpha=float("nan")), b"alpha"),
    (dict(alpha=float("inf")), b"alpha"), (dict(alpha=-1.0), b"alpha"), (dict(alpha=1e-39), b"alpha"), (dict(alpha=2e38), b"alpha"), (dict(dtype=3), b"dtype"), (dict(ld=7), b"stride"),
    (dict(data=0), b"null"), (dict(packed=0), b"null"), (dict(data=64 + 2), b"misaligned"), (dict(packed=64 + 8), b"misaligned"),
])
def test_refusals(args, word):
    """Refused before anything is launched: the pointers are never followed."""
    a = dict(data=64, dtype=0, ld=8, n=4, dim=8, alpha=1.0, block=32, packed=64)
    a.update(args)
    L, P = gf.lib(), ctypes.c_void_p
    assert L.gf_quantize_fp4(P(a["data"]), a["dtype"], a["ld"], a["n"], a["dim"], a["alpha"], a["block"], P(a["packed"]),
                             None) == 1
    assert word in L.gf_last_error()
    assert L.gf_dequantize_fp4(P(a["packed"]), a["n"], a["dim"], a["block"], a["alpha"], P(a["data"]), a["dtype"], a["ld"],
                               None) == 1
    assert word in L.gf_last_error()
    if {"dim", "block", "alpha"} & set(args):
        buf = np.zeros(4096 * 4, np.uint8)
        p = P(buf.ctypes.data)
        assert L.gf_quantize_fp4_host(p, a["n"], a["dim"], a["alpha"], a["block"], p) == 1
        assert L.gf_dequantize_fp4_host(p, a["n"], a["dim"], a["block"], a["alpha"], p) == 1


def test_python_refusals():
    import torch
    with pytest.raises(gf.GarfieldError):
        gf.quantize_fp4(torch.zeros(4, 8))  # not on a GPU
    with pytest.raises(gf.GarfieldError):
        gf.quantize_fp4_host(np.zeros((4, 8), np.float32), block=8)
    with pytest.raises(gf.GarfieldError):
        gf.dequantize_fp4(gf.quantize_fp4_host(np.zeros((4, 8), np.float32)))
    r = gf.quantize_fp4_host(np.zeros((4, 8), np.float32))
    r.n = 400
    with pytest.raises(gf.GarfieldError):
        gf.dequantize_fp4_host(r)


@pytest.mark.parametrize("args,word", [
    (dict(dim=0), b"dim"), (dict(block=8), b"block"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(dtype=7), b"dtype"), (dict(ld=4), b"stride"), (dict(q=0), b"null"),
    (dict(r=0), b"null"), (dict(out=0), b"null"), (dict(q=72), b"misaligned"), (dict(r=72), b"misaligned"),
    (dict(out=66), b"misaligned"),
])
def test_product_refusals(args, word):
    a = dict(q=64, m=3, r=64, n=5, dim=8, block=32, scale=1.0, out=64, dtype=0, ld=5)
    a.update(args)
    L, P = gf.lib(), ctypes.c_void_p
    assert L.gf_product_fp4(P(a["q"]), a["m"], P(a["r"]), a["n"], a["dim"], a["block"], a["scale"], P(a["out"]), a["dtype"],
                            a["ld"], 0, None) == 1
    assert word in L.gf_last_error()
    if args == dict(q=72):
        return  # aligned to its elements
    assert L.gf_product_fp4_raw(P(a["q"]), 0, max(a["dim"], 1), a["m"], 1.0, P(a["r"]), a["n"], a["dim"], a["block"], a["scale"],
                                P(a["out"]), a["dtype"], a["ld"], None, 0, None) == 1
    assert word in L.gf_last_error()


@pytest.mark.parametrize("args,word", [
    (dict(q_dtype=3), b"dtype"), (dict(q_ld=7), b"stride"), (dict(q_alpha=0.0), b"alpha"), (dict(q_alpha=1e39), b"alpha"),
    (dict(q=66), b"misaligned"), (dict(m=17), b"workspace"), (dict(dim=8193, q_ld=8193, m=1), b"workspace"),
    (dict(m=16, dim=2049, q_ld=2049), b"workspace"), (dict(m=17, workspace=72), b"misaligned"),
])
def test_raw_product_refusals(args, word):
    a = dict(q=64, q_dtype=0, q_ld=8, m=3, q_alpha=1.0, dim=8, workspace=0)
    a.update(args)
    L, P = gf.lib(), ctypes.c_void_p
    assert L.gf_product_fp4_raw(P(a["q"]), a["q_dtype"], a["q_ld"], a["m"], a["q_alpha"], P(64), 5, a["dim"], 32, 1.0, P(64), 0, 5,
                                P(a["workspace"]), 0, None) == 1
    assert word in L.gf_last_error()


def test_product_scale_range():
    for qa, ra in [(1.0, 1.0), (2.0 ** -64, 2.0 ** -63), (2.0 ** 63, 2.0 ** 63), (0.7, 3.0)]:
        got = np.float32(gf._fp4_scale(qa, ra, "product"))
        assert abs(float(got) * qa * ra - 1) <= 2.0 ** -24  # a normal float, rounded once
    for qa, ra in [(2.0 ** -64, 2.0 ** -64), (2.0 ** 64, 2.0 ** 63), (0.0, 1.0), (-1.0, 1.0), (float("nan"), 1.0), (float("inf"), 1.0)]:
        with pytest.raises(gf.GarfieldError):
            gf._fp4_scale(qa, ra, "product")


@pytest.mark.parametrize("test_wait", [2 ** 20 + 1, 2 ** 32 - 1])
def test_long_test_waits_are_refused(test_wait):
    """Waits that cannot succeed are bounded by those of normal use."""
    L, P = gf.lib(), ctypes.c_void_p
    assert L.gf_product_fp4(P(64), 3, P(64), 5, 8, 32, 1.0, P(64), 0, 5, test_wait, None) == 1
    assert b"test_wait" in L.gf_last_error()
    assert L.gf_product_fp4_raw(P(64), 0, 8, 3, 1.0, P(64), 5, 8, 32, 1.0, P(64), 0, 5, None, test_wait, None) == 1
    assert b"test_wait" in L.gf_last_error()


def test_streams_of_other_devices_are_refused():
    """A kernel on another device's stream would follow this device's pointers there."""
    import torch

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 64

    with pytest.raises(gf.GarfieldError, match="gf_product_fp4.*cuda:1.*cuda:0"):
        gf._fp4_run("gf_product_fp4", torch.device("cuda", 0), Stream(), pytest.fail)


def small_values(block, seed=1):
    """fp32 data near its smallest number, in blocks whose codes and scales hold them exactly with a large enough alpha."""
    rng = np.random.default_rng(seed)
    n, nb = 150, 96 // block
    e = rng.integers(-150, -120, (n, nb, 1))
    x = np.ldexp(MAGS[rng.integers(0, 8, (n, nb, block))] * rng.choice([-1.0, 1.0], (n, nb, block)), e)
    x[:, :, 0] = np.ldexp(6.0, e[:, :, 0])
    x = np.where(x == np.ldexp(np.rint(np.ldexp(x, 149)), -149), x, 0.0)  # (no parts of fp32's smallest number)
    return x.reshape(n, -1).astype(np.float32)


@pytest.mark.parametrize("block,alpha", [(32, 2.0 ** 30), (32, 2.0 ** 60), (32, 2.0 ** 100), (32, 2.0 ** 126), (16, 2.0 ** 125),
                                         (16, 2.0 ** 126), (32, 1.0), (32, 2.0)])
def test_small_values_are_rounded_once(block, alpha):
    """Scales whose quotient by a power of two is below fp32's normal numbers, or below all of them: what is read back
    is the held value, rounded only where fp32 does not have it."""
    x = small_values(block)
    want = held(x, alpha, block)[2]
    if block == 32 and alpha >= 2.0 ** 30:
        assert np.array_equal(want, x.astype(np.float64))
    assert np.array_equal(gf.dequantize_fp4_host(gf.quantize_fp4_host(x, alpha, block)), want.astype(np.float32))


@pytest.mark.parametrize("alpha", [3e35, 1.7e20, 0.3, 5.0, 8e37])
def test_small_values_read_back_within_the_bound(alpha):
    """Other alphas: three roundings of 2^-24 of the value, and half of fp32's smallest number below the normal ones."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((150, 96)) * 2.0 ** rng.integers(-145, -100, (150, 1))).astype(np.float32)
    a32 = float(np.float32(alpha))
    _, _, want = held(x, a32, 32)
    got = gf.dequantize_fp4_host(gf.quantize_fp4_host(x, alpha, 32)).astype(np.float64)
    tol = 3 * 2.0 ** -24 * (1 + 2.0 ** -22) * np.abs(want) + np.where(np.abs(want) < 2.0 ** -126, 2.0 ** -150, 0.0)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("alpha", [0.3, 1.0 + 1.9 * 2.0 ** -25, 1, 1e-30])
def test_alpha_is_one_number(alpha):
    """What the codec multiplied by is what the products are divided by: alpha in fp32."""
    assert gf.quantize_fp4_host(np.ones((3, 8), np.float32), alpha).alpha == float(np.float32(alpha))
    assert gf.Fp4Rows(None, 3, 8, 32, alpha).alpha == float(np.float32(alpha))


def test_timeout_count_refusal():
    assert gf.lib().gf_product_fp4_timeouts(None) == 1 and b"null" in gf.lib().gf_last_error()


@pytest.mark.parametrize("field", [dict(block=0), dict(block=8), dict(n=-1), dict(n=2 ** 32 + 4), dict(dim=0), dict(dim=2 ** 32 + 8),
                                   dict(dim=-8)])
def test_rows_of_bad_shapes_are_refused(field):
    """By the host call and before a GPU call (which takes both numbers in 32 bits)."""
    class Cuda(np.ndarray):
        is_cuda = True

    rows = gf.quantize_fp4_host(np.ones((4, 8), np.float32))
    for name, v in field.items():
        setattr(rows, name, v)
    with pytest.raises(gf.GarfieldError, match="block"):
        gf.dequantize_fp4_host(rows)
    rows.packed = rows.packed.view(Cuda)
    with pytest.raises(gf.GarfieldError, match="block"):
        gf._fp4_rows(rows, "gf_dequantize_fp4")


def test_host_calls_refuse_other_things():
    for bad in (np.ones(8, np.float32), np.ones((2, 2, 8), np.float32)):
        with pytest.raises(gf.GarfieldError, match="2-D"):
            gf.quantize_fp4_host(bad)
    with pytest.raises(gf.GarfieldError, match="Fp4Rows"):
        gf.dequantize_fp4_host(np.ones(8, np.uint8))
