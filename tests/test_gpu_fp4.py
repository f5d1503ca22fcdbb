"""Microscaled 4-bit floating point on the GPU: rounding, values and products against the definition in 64 bits."""

import pytest
import torch

import plain_fp4 as P
from dryft_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
KINDS = ("mx", "nv")


def rows_of(m, k, dtype, wide=0, grow=0.5):
    x = torch.randn(m, k + wide, device="cuda") * torch.exp(grow * torch.randn(1, k + wide, device="cuda"))
    return x.to(dtype)[:, wide // 2:wide // 2 + k]


def odd_rows(k, dtype):
    """Rows with what is rare: nothing but zeros, tiny and large numbers, ties, groups of very different size, infinities and NaN."""
    x = torch.randn(12, k, device="cuda")
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 1e37
    x[3] *= 1e-30
    x[4, ::2] *= 1e-6
    x[5] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 0.3, 7.9], device="cuda").repeat(k // 12 + 1)[:k]
    x[6, k // 2] = float("nan")
    x[7, k - 1] = float("inf")
    x[8, :k // 3] = 0
    x[9] *= torch.exp(8 * torch.randn(k, device="cuda"))
    x[10] = -x[10].abs()
    x[11, 0] = torch.finfo(dtype).max
    return x.to(dtype)


def same_values(got, want, dtype):
    """Equal to the definition's values but for the factor's product (one 32-bit rounding) and the result's own."""
    assert torch.equal(got.isnan().cpu(), want.isnan())
    tiny = 2.0**-149 if dtype == F32 else 2.0**-133       # half a step of the smallest numbers, twice
    room = (torch.finfo(dtype).eps / 2 + 2.0**-24) * want.abs() + tiny
    assert bool(((got.double().cpu() - want).abs() <= room)[~want.isnan()].all())


def near(got, x, w, kind, k):
    """Sums of k terms: the tensor cores take 64 at a time and cut off what is below 2^-23 of the largest, at most, in each of 64 terms and the sum so far (2^-21 of the terms'
    magnitudes, an instruction); the factors' products and the result are rounded."""
    want, terms = P.product(x, w, kind)
    assert torch.equal(got.isnan().cpu(), want.isnan())
    room = (torch.finfo(got.dtype).eps / 2 + 2.0**-22) * want.abs() + (k / 64 + 2) * 2.0**-21 * terms
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room)[~want.isnan()].all()), float((off / room).nan_to_num().max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,wide", [(1, 16, 0), (1, 1, 0), (3, 17, 0), (130, 256, 0), (5, 2560, 0), (300, 333, 7), (2, 9728, 16), (129, 64, 8), (1, 30000, 2)])
def test_rounding_and_values(kind, dtype, m, k, wide):
    x = rows_of(m, k, dtype, wide)
    q = K.fp4_quantise(x, kind)
    want = P.values(x, kind)
    for out in (BF, F32):
        same_values(K.fp4_expand(q, out_dtype=out), want, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k", [48, 1000])
def test_rounding_of_rare_rows(kind, dtype, k):
    x = odd_rows(k, dtype)
    same_values(K.fp4_expand(K.fp4_quantise(x, kind), out_dtype=F32), P.values(x, kind), F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", [(3, 25600), (148, 13000), (149, 20000), (520, 12304)])
def test_rounding_of_wide_rows(kind, dtype, m, k):
    """Rows that more lanes hold than one block of the usual size has, and rows that no lanes hold; the largest number of a row may lie anywhere."""
    x = rows_of(m, k, dtype)
    for r in range(m):
        x[r, (r * 7919) % k] = 1000.0
    same_values(K.fp4_expand(K.fp4_quantise(x, kind), out_dtype=F32), P.values(x, kind), F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k", [(2, 25600), (150, 9728), (520, 12304)])
def test_silu_of_wide_rows(kind, m, k):
    """As of the same numbers by `silu_mul`, which has the same bits where both read 16-byte words."""
    x, q = rows_of(m, 2 * k, BF), K.fp4_quantise(rows_of(130, k, BF), kind)
    act = torch.empty(m, k, dtype=BF, device="cuda")
    K.silu_mul(x, act)
    assert torch.equal(K.linear_fp4(x, q, silu=True), K.linear_fp4(act, q))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rounding_of_signs_and_of_the_smallest_numbers(kind, dtype):
    """Infinities and NaN of either sign make their group NaN, and no other; zeros of either sign, numbers without leading bits, negative ones that are the largest of their group."""
    bits, finite = (torch.int16, 0x7f80) if dtype == BF else (torch.int32, 0x7f800000)
    x = rows_of(9, 160, dtype)
    raw = x.view(bits)
    sign = -(1 << (15 if dtype == BF else 31))
    raw[0, 40], raw[1, 40], raw[2, 40], raw[3, 40] = finite, finite + 1, finite + sign, finite + 1 + sign
    raw[4, ::2], raw[4, 1::2] = sign, 0
    raw[5] = torch.arange(160, device="cuda").to(bits)              # subnormal numbers
    raw[6] = torch.arange(160, device="cuda").to(bits) + sign
    x[7, ::16], x[8, 1::32] = -100.0, -3.0e38
    got = K.fp4_expand(K.fp4_quantise(x, kind), out_dtype=F32)
    want = P.values(x, kind)
    same_values(got, want, F32)
    assert [int(r.isnan().sum()) for r in got] == [P.GROUP[kind]] * 4 + [0] * 5


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 128, 256), (2, 256, 5120), (16, 300, 4100), (13, 129, 9728), (16, 128, 512), (5, 389, 83), (17, 200, 1000), (33, 130, 300), (100, 256, 2560), (129, 128, 256), (257, 300, 777),
                                   (700, 384, 320), (8, 40000, 320)])
def test_products(kind, m, n, k):
    x, w = rows_of(m, k, BF), rows_of(n, k, BF)
    near(K.linear_fp4(x, K.fp4_quantise(w, kind), out_dtype=F32), x, w, kind, k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,out", [(BF, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("m,n,k", [(1, 129, 1), (3, 50, 31), (20, 260, 2560), (200, 1000, 96)])
def test_products_of_other_types(kind, dtype, out, m, n, k):
    x, w = rows_of(m, k, dtype, 3), rows_of(n, k, dtype)
    near(K.linear_fp4(x, K.fp4_quantise(w, kind), out_dtype=out), x, w, kind, k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [12, 40, 150])
def test_products_of_rare_rows(kind, m):
    """Rows of zeros, tiny and huge numbers, infinities and NaN, as activations (rounded in the product and before it) and as weights; the others' results are their own."""
    k = 1000
    x = odd_rows(k, BF).repeat(-(-m // 12), 1)[:m]
    w = torch.cat([rows_of(150, k, BF) * 1e-3, odd_rows(k, BF)[:2] * 1e-3, odd_rows(k, BF)[6:11] * 1e-3])
    got, q = K.linear_fp4(x, K.fp4_quantise(w, kind), out_dtype=F32), K.fp4_quantise(x, kind)
    want, terms = P.product(x, w, kind)
    assert torch.equal(got.isnan().cpu(), want.isnan()) and bool(want.isnan().any()) and bool(want.isfinite().any())
    fits = terms < 2.0**126          # (of the rest no 32-bit sum need be a number)
    assert float(fits.double().mean()) > 0.8
    # (as `near`; numbers below the smallest normal one may be taken for zeros, an instruction's 64 at a time)
    room = 2.0**-21 * want.abs() + (k / 64 + 2) * 2.0**-21 * terms + (k / 64 + 1) * 2.0**-126
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room)[fits].all()), ((off > room) & fits).nonzero()[:8].tolist()
    assert torch.equal(K.linear_fp4(q, K.fp4_quantise(w, kind), out_dtype=F32).nan_to_num(), got.nan_to_num())
    few = torch.cat([K.linear_fp4(x[i:i + 4], K.fp4_quantise(w, kind), out_dtype=F32) for i in range(0, 12, 4)])   # (rounded by the product's blocks)
    assert torch.equal(few.isnan(), got[:12].isnan()) and bool(((few.double().cpu() - want[:12]).abs() <= room[:12])[fits[:12]].all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,apart", [(1, 200, 96, 0), (3, 130, 2560, 0), (2, 256, 9728, 0), (16, 300, 1001, 0), (48, 256, 1000, 0), (5, 128, 320, 2), (300, 256, 512, 16), (33, 129, 77, 1)])
def test_silu_in_front(kind, m, n, k, apart):
    """The operand is what `silu_mul` gives: the same bits where that reads 16-byte words.  Elsewhere it takes another exponential, some 2^-20 off: one result in 2^11 is then a
    bfloat16 neighbour, 2^-8 away, and one in 2^6 of those has another code, or another scale of its group: a row of k numbers differs with a chance of k 2^-17 + 2^-11, a tenth of
    a row of the sizes here, and by half of one of its numbers."""
    wide = rows_of(m, 2 * k + apart, BF)[:, apart // 2:apart // 2 + 2 * k]
    w = K.fp4_quantise(rows_of(n, k, BF), kind)
    act = torch.empty(m, k, dtype=BF, device="cuda")
    K.silu_mul(wide.contiguous(), act)
    want, got = K.linear_fp4(act, w), K.linear_fp4(wide, w, silu=True)
    assert float((act.cpu() != P.silu_mul(wide.cpu())).float().mean()) < 0.01
    if k % 8 == 0:
        assert torch.equal(got, want)
    else:
        assert int((got != want).any(1).sum()) <= 2 and bool(((got.float() - want.float()).norm(dim=1) <= 0.5 * want.float().norm(dim=1)).all())
    x32 = wide.float()
    act32 = torch.empty(m, k, device="cuda")
    K.silu_mul(x32.contiguous(), act32)
    assert torch.equal(K.linear_fp4(x32, w, silu=True), K.linear_fp4(act32, w))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 7, 16, 20, 64, 100, 128, 129, 200, 333, 513])
@pytest.mark.parametrize("n,k", [(300, 2100), (1000, 600)])
def test_every_way_of_cutting(monkeypatch, kind, m, n, k):
    """Whole tiles, tiles shared by clusters of every size, pairs of blocks with tiles of every width; few blocks, so that each has several tiles."""
    x, w = rows_of(m, k, BF), rows_of(n, k, BF)
    q, h = K.fp4_quantise(w, kind), K.fp4_quantise(x, kind)
    units = (k + 255) // 256
    plans = []
    for nb in (16, 32, 64, 128):
        if m <= nb or nb == 128:
            tiles = -(-n // 128) * -(-m // nb)
            plans += [(nb, min(tiles, 296), 1), (nb, min(tiles, 2), 1)] + [(nb, tiles * s, s) for s in (2, 3, 5, 8) if s <= units]
    for nb in (128, 192, 256):
        tiles = -(-n // 256) * -(-m // nb)
        plans += [(nb, 2 * min(tiles, 74), 0), (nb, 2, 0)]
    results = []
    for plan in plans:
        monkeypatch.setattr(K, "linear_fp4_plan", lambda *a: plan)
        for operand in (h, x):
            results.append(K.linear_fp4(operand, q, out_dtype=F32))
            results.append(K.linear_fp4(operand, q, out_dtype=BF))
            assert torch.equal(results[-1], results[-2].to(BF))
    near(results[0], x, w, kind, k)
    want, terms = P.product(x, w, kind)
    room = (k / 64 + 10) * 2.0**-21 * terms + 2.0**-22 * want.abs()      # (pieces of a tile: eight sums more)
    for r in results[::2]:
        assert bool(((r.double().cpu() - want).abs() <= room).all())
    K.check_error_flags()


@pytest.mark.parametrize("kind", KINDS)
def test_a_row_is_its_own(kind):
    """A row's result is the same, but for the order of 32-bit sums, whatever rows stand beside it; bit for bit in a batch of the same size."""
    k, n = 2560, 640
    x, w = rows_of(300, k, BF), rows_of(n, k, BF)
    q = K.fp4_quantise(w, kind)
    whole = K.linear_fp4(x, q, out_dtype=F32)
    _, terms = P.product(x, w, kind)
    for rows in (slice(0, 1), slice(5, 9), slice(100, 116), slice(17, 80), slice(120, 290)):
        part = K.linear_fp4(x[rows], q, out_dtype=F32)
        assert bool(((part - whole[rows]).abs().double().cpu() <= 2 * (k / 64 + 10) * 2.0**-21 * terms[rows]).all())
        other = x[rows].clone()
        other[1:] = other[1:] * 3 + 1
        assert torch.equal(K.linear_fp4(other, q, out_dtype=F32)[0], part[0])


@pytest.mark.parametrize("kind", KINDS)
def test_operands_and_results_of_other_forms(kind):
    k, n = 512, 300
    x, w = rows_of(40, k, BF), rows_of(n, k, BF)
    q = K.fp4_quantise(w, kind)
    want = K.linear_fp4(x, q)
    near(want, x, w, kind, k)
    # a result that is given, between others' numbers
    room = torch.full((44, n), 7.0, dtype=BF, device="cuda")
    assert K.linear_fp4(x, q, out=room[2:42]).data_ptr() == room[2:].data_ptr() and torch.equal(room[2:42], want)
    assert bool((room[:2] == 7).all()) and bool((room[42:] == 7).all())
    # rows apart, one row many times, rows of a range of a weight, an operand that several products read
    spread = torch.zeros(40, 3, k, dtype=BF, device="cuda")
    spread[:, 1] = x
    assert torch.equal(K.linear_fp4(spread[:, 1], q), want)
    assert torch.equal(K.linear_fp4(x[3:4].expand(40, k), q)[17], K.linear_fp4(x[3:4].repeat(40, 1), q)[17])
    assert torch.equal(K.linear_fp4(x, q[128:]), want[:, 128:]) and torch.equal(K.linear_fp4(x, q[128:200]), want[:, 128:200])
    held = K.fp4_quantise(x, kind)
    for a in (K.linear_fp4(held, q), K.linear_fp4(held, q, out_dtype=F32).to(BF), K.linear_fp4(held, q, pdl=True), K.linear_fp4(x, q, pdl=True), K.linear_fp4(x, q, pdl=False)):
        assert torch.equal(a, want)
    assert K.linear_fp4(x[:0], q).shape == (0, n)
    out = torch.empty(n, k, dtype=F32, device="cuda")
    assert K.fp4_expand(q, out) is out
    # values that begin on no word
    for dtype in (BF, F32):
        odd = torch.empty(n * k + 1, dtype=dtype, device="cuda")[1:].view(n, k)
        K.fp4_expand(q, odd)
        assert torch.equal(odd.to(F32), out.to(dtype).to(F32))


def test_refusals():
    q = K.fp4_quantise(rows_of(130, 64, BF), "nv")
    x, square = rows_of(3, 64, BF), rows_of(64, 64, BF)
    for word, call in [("64 numbers", lambda: K.linear_fp4(x[:, :60], q)), ("128 numbers", lambda: K.linear_fp4(x, q, silu=True)), ("Fp4", lambda: K.linear_fp4(x, x)),
                       ("'mx'", lambda: K.linear_fp4(K.fp4_quantise(x, "mx"), q)), ("silu", lambda: K.linear_fp4(K.fp4_quantise(x, "nv"), q, silu=True)),
                       ("float16", lambda: K.linear_fp4(x, q, out_dtype=torch.float16)), ("shape", lambda: K.linear_fp4(x, q, out=torch.empty(3, 129, device="cuda"))),
                       ("contiguous", lambda: K.linear_fp4(x, q, out=torch.empty(130, 3, device="cuda").t())), ("CUDA", lambda: K.linear_fp4(x, q, out=torch.empty(3, 130))),
                       ("overlap", lambda: K.linear_fp4(square, K.fp4_quantise(square, "nv"), out=square)), ("no numbers", lambda: K.fp4_quantise(x[:0], "nv")), ("no numbers", lambda: K.fp4_quantise(x[:, :0], "mx")), ("float16", lambda: K.fp4_expand(q, out_dtype=torch.float16)),
                       ("shape", lambda: K.fp4_expand(q, torch.empty(130, 65, device="cuda"))), ("behind one another", lambda: K.linear_fp4(rows_of(64, 3, BF).t(), q))]:
        with pytest.raises(K.KernelError) as e:
            call()
        assert word in str(e.value), str(e.value)
    # what only the launcher is asked: plans that it does not take
    lib = K.fp4_lib()
    y = torch.empty(200, 130, dtype=BF, device="cuda")
    h = K.fp4_quantise(rows_of(200, 64, BF), "nv")
    args = (1, 1, h.held.data_ptr(), h.factors.data_ptr(), q.held.data_ptr(), q.factors.data_ptr(), y.data_ptr(), 200, 130, 64)
    tail = (0, K.error_flag(y.device).data_ptr(), K._stream())
    for plan in [(64, 2, 1), (24, 2, 1), (128, 5, 1), (128, 0, 1), (128, 8, 2), (128, 4, 9), (256, 3, 0), (256, 4, 0), (160, 2, 0), (512, 2, 1)]:
        assert lib.dryft_linear_fp4(*args, *plan, *tail) == K.UNSUPPORTED, plan


@pytest.mark.parametrize("m", [1, 4, 40, 200])
def test_captured_and_replayed_on_another_stream(m):
    """Graphs that hold products of the same weight, replayed with other numbers, beside one another."""
    k, n = 2560, 640
    q = K.fp4_quantise(rows_of(n, k, BF), "nv")
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [rows_of(m, k, BF) for _ in range(2)]
    ys, graphs = [], []
    for s, x in zip(streams, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            K.linear_fp4(x, q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ys.append([K.linear_fp4(x, q, pdl=True), K.linear_fp4(K.fp4_quantise(x, "nv"), q, pdl=True)])
        graphs.append(g)
    for _ in range(5):
        new = [rows_of(m, k, BF) for _ in range(2)]
        torch.cuda.synchronize()
        for s, g, x, v in zip(streams, graphs, xs, new):
            with torch.cuda.stream(s):
                x.copy_(v)
                g.replay()
        torch.cuda.synchronize()
        for v, y in zip(new, ys):
            want = K.linear_fp4(v, q)
            assert torch.equal(y[0], want) and torch.equal(y[1], want)
    K.check_error_flags()


def test_a_weight_right_behind_its_rounding():
    """The first product of a weight may stand right behind the launch that rounds it, overlapped or not."""
    x = rows_of(1, 2560, BF)
    w = [rows_of(20000, 2560, BF) for _ in range(3)]
    want = [K.linear_fp4(x, K.fp4_quantise(v, "mx"), pdl=False) for v in w]
    torch.cuda.synchronize()
    for _ in range(5):
        for v, y in zip(w, want):
            assert torch.equal(K.linear_fp4(x, K.fp4_quantise(v, "mx"), pdl=True), y)
            assert torch.equal(K.linear_fp4(K.fp4_quantise(x, "mx"), K.fp4_quantise(v, "mx"), pdl=True), y)


def test_a_captured_product_is_not_a_weights_first_one():
    """What is captured has not run: the first product that does run still overlaps nothing."""
    x, v = rows_of(2, 512, BF), rows_of(256, 512, BF)
    K.linear_fp4(x, K.fp4_quantise(v, "nv"))     # (loads the kernels)
    q, s, g = K.fp4_quantise(v, "nv"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        y = K.linear_fp4(x, q, pdl=True)
    assert not q.read
    want = K.linear_fp4(x, q, pdl=True)
    assert q.read
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("n,k", [(300, 2560), (1000, 600)])
def test_captured_products_of_few_rows(kind, silu, n, k):
    """Rounded in the product or in a launch of its own, which a captured call chooses otherwise than an eager one, results have the same bits."""
    q = K.fp4_quantise(rows_of(n, k, BF), kind)
    xs = [rows_of(m, 2 * k if silu else k, BF) for m in (1, 2, 3, 4, 6, 8, 11, 16)]
    want = [K.linear_fp4(x, q, silu=silu) for x in xs]
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        got = [K.linear_fp4(x, q, silu=silu, pdl=True) for x in xs]
    for _ in range(3):
        for y in got:
            y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, v) for y, v in zip(got, want))
    K.check_error_flags()


def test_results_past_32_bits_of_offset():
    m, n, k = 14400, 151936, 64
    x, w = rows_of(m, k, BF), rows_of(n, k, BF)
    y = K.linear_fp4(x, K.fp4_quantise(w, "mx"))
    for rows in (slice(0, 2), slice(14130, 14140), slice(m - 3, m)):     # 14,134 rows are 2^31 numbers
        for cols in (slice(0, 300), slice(n - 300, n)):
            near(y[rows, cols], x[rows], w[cols], "mx", k)
