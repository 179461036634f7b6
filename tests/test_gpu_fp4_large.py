"""Large products of 4-bit rows: outputs past L2 and past 32-bit offsets, checked on samples of rows."""
from __future__ import annotations

import pytest

import garfield_b200 as gf
from test_gpu_fp4_product import exact_rows

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("m,n,dim,block,dtype", [
    (5000, 99_999, 64, 32, torch.float16),    # rows that start inside sectors: pairs of CTAs
    (3000, 120_000, 96, 16, torch.float32),   # fp32: pairs of CTAs
    (20_000, 120_000, 32, 32, torch.float16),  # 2.4e9 elements
])
def test_large_outputs(m, n, dim, block, dtype):
    q = exact_rows(1000, dim, block, 1).repeat(-(-m // 1000), 1)[:m]
    r = exact_rows(n, dim, block, 2)
    got = gf.product_fp4(q, gf.quantize_fp4(r, 1.0, block), dtype)
    for i in (0, 1, 127, 128, 255, 256, 999, m // 2, m - 257, m - 1):
        assert torch.equal(got[i], (r.double() @ q[i].double()).float().to(dtype)), i
    # rows of the same query are the same
    assert torch.equal(got[:m - 1000:97], got[1000::97][:len(got[:m - 1000:97])])


@pytest.mark.parametrize("m,n,dim,block,offset", [
    (2750, 99_977, 64, 32, 0), (2701, 100_000, 96, 16, 3), (17, 16_000_001, 32, 32, 0), (40, 7_000_003, 32, 32, 5),
    (33, 8_500_005, 100, 16, 1), (129, 2_200_001, 32, 16, 7), (20_000, 14_003, 128, 32, 0),
])
def test_large_fp32_rows_inside_sectors(m, n, dim, block, offset):
    """fp32 outputs past L2 whose rows start at any element; what lies beside them is left as it was."""
    q = exact_rows(min(m, 1000), dim, block, 1).repeat(-(-m // 1000), 1)[:m]
    r = exact_rows(70_001, dim, block, 2).repeat(-(-n // 70_001), 1)[:n]
    buf = torch.full((m, n + offset + (1 if offset else 0)), 7.0, device="cuda")
    out = buf[:, offset:offset + n]
    gf.product_fp4(q, gf.quantize_fp4(r, 1.0, block), out=out)
    for j in range(0, n, 70_001):  # (fp32 holds the sums)
        e = min(n, j + 70_001)
        assert torch.equal(out[:, j:e], q @ r[:e - j].t())
    assert (buf[:, :offset] == 7.0).all() and (buf[:, offset + n:] == 7.0).all()


def test_large_store():
    """More than 2^32 bytes of rows, in and out."""
    n, dim = 9_000_000, 128
    base = exact_rows(9_000, dim, 32, 3)
    x = base.repeat(1000, 1)
    rows = gf.quantize_fp4(x)
    del x
    got = gf.dequantize_fp4(rows)
    for i in (0, 1, 499, 998, 999):
        assert torch.equal(got[i * 9000:(i + 1) * 9000], base)
    scores = gf.product_fp4(base[:3], rows)
    want = (base[:3].double() @ base.double().t()).float()
    for i in (0, 500, 999):
        assert torch.equal(scores[:, i * 9000:(i + 1) * 9000], want)
