"""4-bit block floating point on the GPU: the device quantiser's bytes against the host form's, the values
read back against the definition in 64 bits, strides, alignments, streams and graphs."""
from __future__ import annotations

import weakref

import numpy as np
import pytest

import garfield_b200 as gf
from test_fp4 import data, e4m3_values, held, small_values

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def valid_bytes(packed, n, dim, block):
    """Packed bytes of the rows that exist, as (scales, codes) lists in panel order."""
    sub = 512 * (32 // block)
    h = 128 if n >= 128 else -(-n // 16) * 16
    out = []
    at = 0
    for p in range(-(-n // 128)):
        rows = min(128, n - p * 128)
        for _ in range(0, dim, 128):
            sc = packed[at:at + sub].reshape(-1, 32, 4, 4).transpose(0, 2, 1, 3).reshape(-1, 128, 4)
            out.append(sc[:, :rows].ravel())
            at += sub
        cols = -(-dim // 32)
        out.append(packed[at:at + cols * h * 16].reshape(cols, h, 16)[:, :rows].ravel())
        at += cols * h * 16
    assert at == packed.size
    return np.concatenate(out)


def same_bytes(rows, ref):
    assert (rows.n, rows.dim, rows.block) == (ref.n, ref.dim, ref.block)
    a = valid_bytes(rows.packed.cpu().numpy(), rows.n, rows.dim, rows.block)
    b = valid_bytes(ref.packed, ref.n, ref.dim, ref.block)
    assert np.array_equal(a, b), np.flatnonzero(a != b)[:10]


SHAPES = [(1, 1), (1, 8192), (3, 96), (64, 31), (127, 32), (128, 128), (130, 33), (300, 300), (1000, 65), (513, 1000),
          (256, 8), (300, 16), (500, 24), (257, 32), (400, 5), (129, 48), (384, 64), (200, 2056)]


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_device_matches_host(n, dim, dtype, block):
    for kind, alpha in (("normal", 16.0), ("wide", 1.0), ("borders", 1.0), ("normal", 0.3), ("wide", 2.0 ** -100), ("wide", 0.7),
                        ("borders", 4.0), ("normal", 2.0 ** 20), ("normal", 1e-36)):
        x = torch.from_numpy(data(n, dim, n + dim, kind)).to(dtype)
        same_bytes(gf.quantize_fp4(x.cuda(), alpha, block), gf.quantize_fp4_host(x.float().numpy(), alpha, block))


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", SHAPES)
def test_read_back(n, dim, dtype, block):
    for kind, alpha in (("normal", 16.0), ("wide", 1.0)):
        x = data(n, dim, n + 3 * dim, kind)
        got = gf.dequantize_fp4(gf.quantize_fp4(torch.from_numpy(x).cuda(), alpha, block), dtype)
        want = torch.from_numpy(held(x, alpha, block)[2]).to(torch.float32).to(dtype)  # exact in fp32: alpha is 2^k
        assert torch.equal(got.cpu(), want)
    x = data(n, dim, 1, "normal")
    r = gf.quantize_fp4(torch.from_numpy(x).cuda(), 0.3, block)
    ref = gf.Fp4Rows(r.packed.cpu().numpy(), n, dim, block, 0.3)
    assert torch.equal(gf.dequantize_fp4(r, dtype).cpu(), torch.from_numpy(gf.dequantize_fp4_host(ref)).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [33, 96])
@pytest.mark.parametrize("offset,gap", [(0, 0), (1, 0), (4, 4), (3, 5), (0, 1)])
def test_strided_rows(dtype, dim, offset, gap):
    """Rows inside a wider matrix, at any element offset; what lies beside the output is left as it was."""
    n = 140
    x = torch.from_numpy(data(n, dim, 9, "normal")).to(dtype).cuda()
    buf = torch.full((n, offset + dim + gap), float("nan"), dtype=dtype, device="cuda")
    view = buf[:, offset:offset + dim]
    view.copy_(x)
    r = gf.quantize_fp4(view, 1.0, 32)
    same_bytes(r, gf.quantize_fp4_host(x.float().cpu().numpy(), 1.0, 32))
    out = torch.full_like(buf, 7.0)
    got = gf.dequantize_fp4(r, out=out[:, offset:offset + dim])
    assert torch.equal(got, gf.dequantize_fp4(r, dtype))
    assert (out[:, :offset] == 7.0).all() and (out[:, offset + dim:] == 7.0).all()


def test_every_e4m3_scale():
    """Blocks of 16 whose scale takes every E4M3 value, with elements on and next to every code border, and zeros of
    either sign."""
    rows = []
    for s in e4m3_values()[1:]:
        b = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float64)
        x = np.concatenate([[6.0 * s], b * s, np.zeros(8)]).astype(np.float32)
        for step in (0, 1, -1):
            y = x.copy()
            if step:
                y[1:8] = np.nextafter(y[1:8], np.float32(step * 1e9))
            y[8:] = -y[:8]
            rows.append(y)
        rows.append(np.where(np.arange(16) == 3, x[0], np.copysign(np.zeros(16), np.arange(16) % 2 - 0.5)).astype(np.float32))
    x = np.stack(rows)
    same_bytes(gf.quantize_fp4(torch.from_numpy(x).cuda(), 1.0, 16), gf.quantize_fp4_host(x, 1.0, 16))
    same_bytes(gf.quantize_fp4(torch.from_numpy(x / 8).cuda(), 8.0, 16), gf.quantize_fp4_host(x, 1.0, 16))


@pytest.mark.parametrize("alpha", [1.0, 2.0 ** -30, 2.0 ** 30, 2.0 ** -31, 2.0 ** 100, 0.3, 1e-30])
@pytest.mark.parametrize("block", [16, 32])
def test_magnitudes_from_end_to_end(block, alpha):
    """fp32 data of every binade, subnormal products among them."""
    rng = np.random.default_rng(7)
    x = (rng.standard_normal((300, 96)) * 2.0 ** rng.integers(-149, 127, (300, 1))).astype(np.float32)
    x[::3] *= (2.0 ** rng.integers(-12, 1, (100, 96))).astype(np.float32)
    x = np.clip(x, -3e38, 3e38)
    with np.errstate(over="ignore"):
        same_bytes(gf.quantize_fp4(torch.from_numpy(x).cuda(), alpha, block), gf.quantize_fp4_host(x, alpha, block))


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
def test_non_finite_block_reads_nan(block, bad):
    x = torch.ones(200, 80, device="cuda")
    x[131, 35] = bad
    r = gf.quantize_fp4(x, 1.0, block)
    same_bytes(r, gf.quantize_fp4_host(x.cpu().numpy(), 1.0, block))
    got = gf.dequantize_fp4(r)
    want = torch.ones(200, 80, dtype=torch.bool, device="cuda")
    want[131, 32:32 + block] = False
    assert torch.equal(torch.isfinite(got), want)


def test_rows_past_the_last_are_left():
    n, dim = 130, 96
    x = torch.from_numpy(data(n, dim, 2, "normal")).cuda()
    size = gf.lib().gf_fp4_bytes(n, dim, 32)
    packed = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    import ctypes
    gf._check(gf.lib().gf_quantize_fp4(ctypes.c_void_p(x.data_ptr()), 0, dim, n, dim, 1.0, 32,
                                       ctypes.c_void_p(packed.data_ptr()), gf._stream_ptr(None)), "gf_quantize_fp4")
    p = packed.cpu().numpy()
    assert (p[size:] == 0xA5).all()
    codes = p[size // 2 + 512:size].reshape(3, 128, 16)
    assert (codes[:, 2:] == 0xA5).all()


def test_empty_and_refused():
    r = gf.quantize_fp4(torch.empty(0, 16, device="cuda"))
    assert gf.dequantize_fp4(r).shape == (0, 16)
    x = torch.zeros(8, 16, device="cuda")
    for bad in (x.t(), x[0], x.double(), x.expand(8, 16)[:, ::2], x[:1].expand(8, 16)):
        with pytest.raises(gf.GarfieldError):
            gf.quantize_fp4(bad)
    with pytest.raises(gf.GarfieldError):
        gf.quantize_fp4(x, block=64)
    with pytest.raises(gf.GarfieldError):
        gf.quantize_fp4(x, alpha=0.0)
    r = gf.quantize_fp4(x)
    with pytest.raises(gf.GarfieldError):
        gf.dequantize_fp4(r, out=torch.zeros(7, 16, device="cuda"))
    with pytest.raises(gf.GarfieldError):
        gf.dequantize_fp4(r, dtype=torch.float64)
    with pytest.raises(gf.GarfieldError):
        gf.dequantize_fp4(gf.Fp4Rows(r.packed, 400, 16, 32, 1.0))


def test_streams_and_graph():
    x = torch.from_numpy(data(500, 200, 4, "normal")).cuda()
    want = gf.dequantize_fp4(gf.quantize_fp4(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = gf.dequantize_fp4(gf.quantize_fp4(x, stream=side), stream=side)
    got2 = gf.dequantize_fp4(gf.quantize_fp4(x, stream=side.cuda_stream), stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = gf.dequantize_fp4(gf.quantize_fp4(x))
    x.mul_(-3.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, gf.dequantize_fp4(gf.quantize_fp4(x)))


def test_stream_of_another_device_is_refused():
    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 64

    x = torch.ones(20, 64, device="cuda:0")
    r = gf.quantize_fp4(x)
    for call in (lambda: gf.quantize_fp4(x, stream=Stream()), lambda: gf.dequantize_fp4(r, stream=Stream()),
                 lambda: gf.product_fp4(x, r, stream=Stream())):
        with pytest.raises(gf.GarfieldError, match="cuda:1"):
            call()


def test_inputs_dropped_while_a_stream_has_to_read_them():
    """Packed rows and queries that only the call held, and memory that is handed out and written again at once."""
    x, q = torch.from_numpy(data(3000, 256, 8, "normal")).cuda(), torch.from_numpy(data(40, 256, 9, "normal")).cuda()
    want = gf.product_fp4(q, gf.quantize_fp4(x))
    back = gf.dequantize_fp4(gf.quantize_fp4(x))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def late(call, *make):
        """call's result, on a stream that is held up until the memory of what `make` makes could have been
        written again."""
        made = [m() for m in make]
        alive = [weakref.ref(t) for t in made]
        sizes = [(t.packed if isinstance(t, gf.Fp4Rows) else t) for t in made]
        sizes = [(t.data_ptr(), t.numel(), t.dtype) for t in sizes]
        room = [torch.empty(n, dtype=dt, device="cuda").fill_(1) for _, n, dt in sizes]
        del room  # the allocator has room without asking the driver, and the kernels are loaded
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(60_000_000)  # some 30 ms
        result = call(*made)
        del made
        assert not any(r() is not None for r in alive)
        new = [torch.empty(n, dtype=dt, device="cuda").fill_(3) for _, n, dt in sizes]
        assert not side.query()
        assert {t.data_ptr() for t in new}.isdisjoint(at for at, _, _ in sizes)
        side.synchronize()
        return result

    assert torch.equal(late(lambda r, y: gf.product_fp4(y, r, stream=side), lambda: gf.quantize_fp4(x), q.clone), want)
    assert torch.equal(late(lambda r: gf.dequantize_fp4(r, stream=side), lambda: gf.quantize_fp4(x)), back)
    assert torch.equal(gf.dequantize_fp4(late(lambda y: gf.quantize_fp4(y, stream=side.cuda_stream), x.clone)), back)


def test_results_dropped_while_the_current_stream_has_to_read_them():
    """Rows made on a stream, read on the current one and dropped: the stream's next rows get other memory."""
    x = torch.from_numpy(data(3000, 256, 8, "normal")).cuda()
    y, want = -x, gf.dequantize_fp4(gf.quantize_fp4(x))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    rows = gf.quantize_fp4(x, stream=side)
    at = rows.packed.data_ptr()
    room = gf.quantize_fp4(x, stream=side)
    del room  # the allocator has room on that stream without asking the driver
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    torch.cuda._sleep(60_000_000)
    got = gf.dequantize_fp4(rows)
    del rows
    again = gf.quantize_fp4(y, stream=side)
    assert not torch.cuda.current_stream().query() and again.packed.data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(gf.dequantize_fp4(again), -want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block,alpha", [(32, 1.0), (32, 2.0), (32, 2.0 ** 60), (32, 2.0 ** 126), (16, 2.0 ** 126), (32, 3e35), (32, 5.0),
                                         (16, 8e37)])
def test_small_values_as_on_the_host(block, alpha, dtype):
    """Values below fp32's normal numbers, at each width of a store."""
    x = small_values(block)
    ref = gf.quantize_fp4_host(x, alpha, block)
    want = torch.from_numpy(gf.dequantize_fp4_host(ref))
    assert want.count_nonzero() > 4000
    r = gf.Fp4Rows(gf.quantize_fp4(torch.from_numpy(x).cuda(), alpha, block).packed, *x.shape, block, alpha)
    for pad in (0, 1, 4):
        out = torch.empty(x.shape[0], x.shape[1] + pad, dtype=dtype, device="cuda")[:, :x.shape[1]]
        assert torch.equal(gf.dequantize_fp4(r, out=out).cpu(), want.to(dtype))
