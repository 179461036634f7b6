"""Products of rows held in 4 bits on the tensor cores, against the held values in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import garfield_b200 as gf
from test_fp4 import MAGS, data

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def exact_rows(n, dim, block, seed):
    """Rows that their 4-bit form holds exactly, with block scales 1/2, 1 and 2: products are multiples of
    2^-4 and sums of 8192 of them stay below 2^20, so fp32 adds them exactly in any order."""
    rng = np.random.default_rng(seed)
    nb = -(-dim // block)
    x = MAGS[rng.integers(0, 8, (n, nb, block))] * rng.choice([-1.0, 1.0], (n, nb, block))
    x[:, :, 0] = 6.0 * rng.choice([-1.0, 1.0], (n, nb))
    x *= 2.0 ** rng.integers(-1, 2, (n, nb, 1))
    return torch.from_numpy(x.reshape(n, -1)[:, :dim].astype(np.float32)).cuda()


def check_exact(m, n, dim, block, dtype=torch.float32):
    q, r = exact_rows(m, dim, block, m + dim), exact_rows(n, dim, block, 7 * n + dim)
    out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")  # nothing may be left unwritten
    got = gf.product_fp4(q, gf.quantize_fp4(r, 1.0, block), out=out)
    want = q.double() @ r.double().t()
    if dtype == torch.float32:
        assert torch.equal(got.double(), want)
    else:
        assert torch.equal(got, want.float().to(dtype))


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dim", [1, 16, 31, 32, 33, 64, 65, 96, 97, 128, 129, 160, 200, 256, 300, 1000, 4096, 8192])
def test_widths(dim, block):
    check_exact(5, 130, dim, block)
    check_exact(70, 257, dim, block)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 400, 520, 1000])
def test_query_counts(m, block):
    check_exact(m, 300, 200, block)
    check_exact(m, 129, 1056, block)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("n", [1, 2, 31, 127, 128, 129, 1000, 20000, 50001])
def test_row_counts(n, block):
    check_exact(1, n, 96, block)
    check_exact(40, n, 128, block)
    check_exact(300, n, 100, block)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dim", [32, 96, 128, 256])
@pytest.mark.parametrize("m,n", [(1, 80_000), (3, 200_001), (16, 100_000), (17, 90_001), (33, 120_000), (64, 81_000), (65, 80_001)])
def test_several_panels_to_a_tile(m, n, dim, block):
    check_exact(m, n, dim, block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 7, 15])
@pytest.mark.parametrize("m,n", [(2, 1), (17, 127), (40, 128), (16, 130), (130, 255), (40, 20000), (270, 19013)])
def test_rows_of_any_alignment(m, n, offset, dtype):
    """Rows of out at every offset within a sector; what lies around them is left as it was."""
    q, r = exact_rows(m, 64, 32, 1), exact_rows(n, 64, 32, 2)
    buf = torch.full((m, n + offset + 5), 7.0, dtype=dtype, device="cuda")
    got = gf.product_fp4(q, gf.quantize_fp4(r), out=buf[:, offset:offset + n])
    assert torch.equal(got, (q.double() @ r.double().t()).float().to(dtype))
    got.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [
    (129, 19001, 96), (256, 18944, 128), (257, 12801, 32), (300, 20000, 33), (1000, 4993, 200), (2000, 2500, 1000),
    (384, 9600, 520), (511, 9473, 384), (1500, 3200, 8192), (5000, 700, 640), (20000, 129, 160), (700, 20000, 416),
    (129, 19001, 1024), (257, 12801, 1000), (300, 9999, 1057), (1000, 4993, 1320), (20000, 129, 1200), (2049, 4000, 2080),
])
def test_pairs_of_ctas(m, n, dim, block):
    """Enough tiles of 256 x 256 for pairs of CTAs, with odd panel counts on either side."""
    check_exact(m, n, dim, block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [(700, 7001, 200), (1, 1000, 300), (20, 333, 128), (100, 100, 1000), (300, 501, 200)])
def test_output_types(m, n, dim, block, dtype):
    check_exact(m, n, dim, block, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [(1, 5000, 96), (9, 700, 8192), (300, 900, 777), (130, 128, 4096)])
def test_normal_data(m, n, dim, block, dtype):
    """An MMA step adds 64 products to an fp32 sum; terms aligned to the largest and cut at 2^-23 of it
    err by at most 2^-23 of the step's sum of magnitudes each way, so the whole sum errs by at most
    (dim / 64 + 2) 2^-22 sum |q r|; scale and dtype round once more each."""
    q = torch.from_numpy(data(m, dim, 3, "normal")).cuda().to(dtype)
    r = torch.from_numpy(data(n, dim, 4, "normal")).cuda().to(dtype)
    rows = gf.quantize_fp4(r, 16.0, block)
    got = gf.product_fp4(q, rows, dtype, query_alpha=16.0).double()
    qv = gf.dequantize_fp4(gf.quantize_fp4(q, 16.0, block)).double()
    rv = gf.dequantize_fp4(rows).double()
    want = qv @ rv.t()
    tol = (dim / 64 + 2) * 2.0 ** -22 * (qv.abs() @ rv.abs().t()) + (2.0 ** -23 + torch.finfo(dtype).eps / 2) * want.abs()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("block", [16, 32])
def test_scales_over_many_binades(block):
    """Block scales far apart: exact for one non-zero block per row."""
    m, n, nb = 6, 300, 8
    dim = nb * block
    q, r = torch.zeros(m, dim, device="cuda"), torch.zeros(n, dim, device="cuda")
    span = 6 if block == 16 else 40  # E4M3 scales span 2^-9 to 448
    for i in range(m):
        b = i % nb
        q[i, b * block:(b + 1) * block] = 6.0 * 2.0 ** (i % span - span // 2)
    for j in range(n):
        r[j] = -4.0 * 2.0 ** (j % span - span // 2)
        r[j, ::block] = 6.0 * 2.0 ** (j % span - span // 2)
    got = gf.product_fp4(q, gf.quantize_fp4(r, 1.0, block))
    assert torch.equal(got.double(), q.double() @ r.double().t())


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [(3, 300, 96), (70, 300, 200), (300, 19100, 168)])
def test_non_finite_blocks(m, n, dim, block):
    """A NaN or infinity reaches its own row's or column's products and no others."""
    q, r = exact_rows(m, dim, block, 1), exact_rows(n, dim, block, 2)
    want = q.double() @ r.double().t()
    r2, q2 = r.clone(), q.clone()
    r2[5, 3], r2[129, dim - 1], r2[299, 0] = float("nan"), float("inf"), -float("inf")
    q2[1, dim - 1] = float("inf")
    got = gf.product_fp4(q2, gf.quantize_fp4(r2, 1.0, block))
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[:, [5, 129, 299]] = True
    bad[1] = True
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad].double(), want[~bad])


def test_zero_rows():
    q, r = exact_rows(4, 128, 32, 1), torch.zeros(200, 128, device="cuda")
    assert not gf.product_fp4(q, gf.quantize_fp4(r)).any()
    assert not gf.product_fp4(torch.zeros(4, 128, device="cuda"), gf.quantize_fp4(exact_rows(200, 128, 32, 2))).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,gap", [(3, 129, 0), (3, 129, 1), (40, 256, 8), (300, 131, 5), (130, 64, 3), (301, 19003, 2)])
def test_strided_output(dtype, m, n, gap):
    q, r = exact_rows(m, 96, 32, 1), gf.quantize_fp4(exact_rows(n, 96, 32, 2))
    want = gf.product_fp4(q, r, dtype)
    buf = torch.full((m + 2, n + 2 * gap + 1), 7.0, dtype=dtype, device="cuda")
    view = buf[1:m + 1, gap:gap + n]
    got = gf.product_fp4(q, r, out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(got, want)
    view.fill_(7.0)
    assert (buf == 7.0).all()


def test_prepared_queries_and_alpha():
    q, r = exact_rows(9, 200, 16, 1), exact_rows(300, 200, 16, 2)
    want = q.double() @ r.double().t()
    rows = gf.quantize_fp4(r, 4.0, 16)
    assert torch.equal(gf.product_fp4(gf.quantize_fp4(q, 0.5, 16), rows).double(), want)
    assert torch.equal(gf.product_fp4(q, rows, query_alpha=2.0).double(), want)
    assert torch.equal(gf.product_fp4(rows, rows).double(), r.double() @ r.double().t())


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("qdtype", DTYPES)
@pytest.mark.parametrize("m,dim", [(1, 1), (1, 33), (3, 70), (8, 128), (16, 200), (16, 2048), (4, 8192), (1, 8192), (16, 2049),
                                   (17, 64), (1, 8193), (100, 300), (5, 1000)])
def test_raw_queries_equal_prepared_ones(m, dim, qdtype, block):
    """Queries given as they are, few (quantised in passing) or many, strided, are held as quantize_fp4 holds
    them: the products are equal bit for bit, for one panel of rows (split over a cluster) and many."""
    x = torch.from_numpy(data(m, dim + 3, dim, "normal")).to(qdtype).cuda()
    q = x[:, 3:] if dim % 2 else x[:, :dim]
    for n in (90, 3000, 40000 if dim <= 200 else 1000):
        rows = gf.quantize_fp4(torch.from_numpy(data(n, dim, 1, "normal")).cuda(), 4.0, block)
        for alpha in (1.0, 0.7):
            a = gf.product_fp4(q, rows, query_alpha=alpha)
            b = gf.product_fp4(gf.quantize_fp4(q, alpha, block), rows)
            assert torch.equal(a, b), (n, alpha)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [(1, 100, 8192), (16, 1000, 8192), (20, 500, 4096), (128, 130, 8192), (100, 129, 3000),
                                     (300, 256, 8192), (64, 4000, 2000), (1, 128, 1024), (1, 9000, 8000), (200, 128, 1100)])
def test_tiles_split_along_the_elements(m, n, dim, block):
    """Few tiles of long rows: shares of the elements in a cluster, added in its first CTA."""
    check_exact(m, n, dim, block)
    check_exact(m, n, dim, block, torch.bfloat16)


def test_repeats_are_equal():
    q = torch.from_numpy(data(70, 3000, 3, "normal")).cuda()
    rows = gf.quantize_fp4(torch.from_numpy(data(500, 3000, 4, "normal")).cuda())
    a = gf.product_fp4(q, rows)
    for _ in range(3):
        assert torch.equal(a, gf.product_fp4(q, rows))


def test_empty_and_refused():
    r = gf.quantize_fp4(torch.zeros(20, 64, device="cuda"))
    assert gf.product_fp4(torch.empty(0, 64, device="cuda"), r).shape == (0, 20)
    assert gf.product_fp4(torch.zeros(3, 64, device="cuda"), gf.quantize_fp4(torch.empty(0, 64, device="cuda"))).shape == (3, 0)
    q = torch.zeros(3, 64, device="cuda")
    for bad in (q[:, :32], q.cpu(), gf.quantize_fp4(q, block=16), q.double(), 5):
        with pytest.raises(gf.GarfieldError):
            gf.product_fp4(bad, r)
    with pytest.raises(gf.GarfieldError):
        gf.product_fp4(q, r, out=torch.zeros(3, 21, device="cuda"))
    with pytest.raises(gf.GarfieldError):
        gf.product_fp4(q, r, dtype=torch.float64)
    with pytest.raises(gf.GarfieldError):
        gf.product_fp4(q, r, out=torch.zeros(20, 3, device="cuda").t())


def test_streams_and_graphs():
    """Two streams at once, and captured calls replayed on new data."""
    rows = gf.quantize_fp4(exact_rows(3000, 300, 32, 1))
    qs = [exact_rows(30, 300, 32, 2), exact_rows(300, 300, 32, 3)]
    want = [gf.product_fp4(q, rows) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            got[i].append(gf.product_fp4(qs[i], rows, stream=streams[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gf.product_fp4(q, rows))
        graphs.append(g)
    for q in qs:
        q.neg_()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, -w)


def test_calls_from_several_threads():
    """Calls of one kernel that need different amounts of shared memory, each thread on its own stream."""
    from concurrent.futures import ThreadPoolExecutor
    shapes = [(20, 3000, 96), (20, 700, 2048), (60, 500, 300), (3, 1000, 96), (16, 1000, 1500)]
    sets = []
    for m, n, dim in shapes:
        q, r = exact_rows(m, dim, 32, m + dim), exact_rows(n, dim, 32, n + dim)
        sets.append((q, gf.quantize_fp4(r), q.double() @ r.double().t()))
    torch.cuda.synchronize()

    def work(k):
        stream = torch.cuda.Stream()
        wrong = 0
        for i in range(60):
            q, rows, want = sets[(i + k) % len(sets)]
            out = gf.product_fp4(q, rows, stream=stream)
            stream.synchronize()
            wrong += not torch.equal(out.double(), want)
        return wrong

    with ThreadPoolExecutor(4) as pool:
        assert list(pool.map(work, range(4))) == [0] * 4


def test_captured_pipeline():
    """Quantising, scoring (with and without a workspace) and reading back captured together, behind a copy and
    beside work on a second stream; two such graphs replayed at once."""
    def capture(x, y, q):
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g):
            y.copy_(x)
            rows = gf.quantize_fp4(y, 1.0, 16)
            side.wait_stream(torch.cuda.current_stream())
            few = gf.product_fp4(q[:4], rows, stream=side)
            many = gf.product_fp4(q, rows)
            torch.cuda.current_stream().wait_stream(side)
            back = gf.dequantize_fp4(rows)
            again = gf.product_fp4(gf.quantize_fp4(back, 1.0, 16), rows)
        return g, few, many, back, again

    xs = [exact_rows(700, 300, 16, 5), exact_rows(900, 300, 16, 6)]
    q = exact_rows(40, 300, 16, 7)
    made = [capture(x, torch.empty_like(x), q) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for sign in (-1.0, -1.0):
        for x in xs:
            x.mul_(sign)
        torch.cuda.synchronize()
        for s, (g, *_) in zip(streams, made):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for x, (_, few, many, back, again) in zip(xs, made):
            want = q.double() @ x.double().t()
            assert torch.equal(few.double(), want[:4]) and torch.equal(many.double(), want)
            assert torch.equal(back, x) and torch.equal(again.double(), x.double() @ x.double().t())


def test_alphas_without_a_scale():
    """Alphas whose product's inverse fp32 does not hold as a normal number are refused."""
    r = gf.quantize_fp4(torch.full((20, 64), 2.0 ** -20, device="cuda"), 2.0 ** 64)
    q = torch.ones(3, 64, device="cuda")
    for bad in (2.0 ** 63, 0.0, -1.0, float("nan")):
        with pytest.raises(gf.GarfieldError):
            gf.product_fp4(q, r, query_alpha=bad)
    with pytest.raises(gf.GarfieldError):
        gf.product_fp4(r, r)
    assert (gf.product_fp4(q, r, query_alpha=2.0 ** 62) == 2.0 ** -14).all()


def test_store_score_read_together():
    """A collection held in 4 bits, scored for candidates, read back and re-ranked by the held values."""
    x = torch.from_numpy(data(5000, 96, 11, "normal")).cuda()
    x /= x.norm(dim=1, keepdim=True)
    rows = gf.quantize_fp4(x, 64.0, 16)
    q = x[:50] + 0.01
    scores = gf.product_fp4(q, rows, query_alpha=64.0)
    top = scores.topk(20, dim=1).indices
    assert (top[:, :1] == torch.arange(50, device="cuda")[:, None]).all()
    held_rows = gf.dequantize_fp4(rows)
    held_q = gf.dequantize_fp4(gf.quantize_fp4(q, 64.0, 16)).double()
    again = torch.einsum("qd,qkd->qk", held_q, held_rows[top].double())
    ref = (held_q.abs().sum(1, keepdim=True) * held_rows.abs().max()).double()
    assert ((scores.gather(1, top).double() - again).abs() <= 2.0 ** -20 * ref).all()


@pytest.mark.parametrize("m,n,dim", [(20, 1000, 300), (300, 19000, 300), (300, 19000, 1100), (1, 500, 4096), (100, 500, 4096)])
def test_waits_that_run_out(m, n, dim):
    """The timeout path: outputs owed become NaN, and the next call is sound."""
    q, r = exact_rows(m, dim, 32, 1), exact_rows(n, dim, 32, 2)
    rows = gf.quantize_fp4(r)
    got = gf.product_fp4(q, rows, test_wait=4)
    assert torch.isnan(got).all()
    assert torch.equal(gf.product_fp4(q, rows).double(), q.double() @ r.double().t())


@pytest.mark.parametrize("m,n,dim", [(300, 19000, 1100), (40, 40000, 1024), (128, 130, 8192), (20, 1000, 300), (40, 90_000, 64)])
def test_copies_land_when_waits_run_out_at_once(m, n, dim):
    """Waits of a single poll give up with copies in flight into every SM's shared memory (pairs, rings, shares of a
    tile, resident queries, several panels to a tile); calls that follow at once use the same shared memory."""
    q, r = exact_rows(m, dim, 16, 1), exact_rows(n, dim, 16, 2)
    rows, queries = gf.quantize_fp4(r, 1.0, 16), gf.quantize_fp4(q, 1.0, 16)
    want = (q.double() @ r.double().t()).float()
    for _ in range(5):
        bad = gf.product_fp4(queries, rows, test_wait=1)
        got = [gf.product_fp4(queries, rows) for _ in range(3)]
        assert torch.isnan(bad).all()
        assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("m", [3, 40])
def test_products_use_the_alphas_of_the_codec(m):
    """An alpha that rounds to 1 in fp32 leaves the products of exactly held rows exact."""
    alpha = 1.0 + 1.9 * 2.0 ** -25
    q, r = exact_rows(m, 96, 16, 1), exact_rows(300, 96, 16, 2)
    want = q.double() @ r.double().t()
    rows = gf.quantize_fp4(r, alpha, 16)
    assert torch.equal(gf.product_fp4(q, rows, query_alpha=alpha).double(), want)
    assert torch.equal(gf.product_fp4(gf.quantize_fp4(q, alpha, 16), rows).double(), want)
    assert torch.equal(gf.dequantize_fp4(rows), r)


@pytest.mark.parametrize("m,n,dim", [(300, 19000, 1100), (1, 500, 4096), (40, 1000, 96)])
def test_waits_that_run_out_are_counted(m, n, dim):
    """NaN left by a wait that ran out is told from NaN data: pairs, shares of a tile, single CTAs."""
    q, rows = exact_rows(m, dim, 32, 1), gf.quantize_fp4(exact_rows(n, dim, 32, 2))
    before = gf.product_fp4_timeouts()
    q[0] = float("nan")
    assert torch.isnan(gf.product_fp4(q, rows)[0]).all()
    assert gf.product_fp4_timeouts() == before
    gf.product_fp4(q, rows, test_wait=4)
    after = gf.product_fp4_timeouts(torch.device("cuda", 0))
    assert before < after <= before + 148
    gf.product_fp4(q, rows)
    assert gf.product_fp4_timeouts() == after


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [
    (1, 100, 4100), (16, 100, 4480), (1, 2000, 5200), (16, 500, 6272),  # 33 to 49 groups of 128 elements: 7 CTAs
    (1, 128, 7168), (1, 100, 4096), (3, 129, 4608),  # 8
    (20, 300, 4480), (40, 128, 4225), (20, 300, 8192), (64, 1000, 2049),  # 4
    (128, 128, 1025),  # 2
])
def test_shares_of_every_number(m, n, dim, block):
    """Rows of long elements, split over clusters of 2, 4, 7 and 8 CTAs with shares that do not come out even."""
    check_exact(m, n, dim, block)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,dim", [(20_000, 100, 1024), (20_000, 1, 800), (20_000, 128, 1056), (19_201, 33, 1000), (20_000, 300, 768)])
def test_pairs_of_ctas_with_few_rows(m, n, dim, block):
    """Many queries against one row panel, short or whole, or three: the second half of some pairs' tiles is empty."""
    check_exact(m, n, dim, block)
