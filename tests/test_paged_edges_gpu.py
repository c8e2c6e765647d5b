"""Paged KV cache on the GPU: calls at the edges of what test_paged_gpu.py covers, with its cache and its bounds."""
import numpy as np
import pytest
from test_paged_gpu import Cache, attend, check_rows, scratch  # noqa: F401

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("QH,KVH,lens", [(12, 4, [500] * 63 + [40000]), (16, 4, [500] * 63 + [40000]),
                                         (16, 4, [100] * 30 + [16000] + [1000] * 33), (8, 2, [30000, 9]), (3, 1, [50, 30000])],
                         ids=["3-heads", "4-heads", "16000-among-64", "two-sequences", "two-sequences-3-heads"])
def test_a_unit_over_more_ctas_than_one_group(e4b, dev, scratch, bits, QH, KVH, lens):  # noqa: F811
    """One row a sequence, heads of 256: the parts of the long sequence's units are merged by groups of CTAs and then over
    the groups; a column is two warps' work there.  Every call gives the same bits."""
    HD, rng = 256, np.random.default_rng(QH + len(lens))
    c = Cache(e4b, dev, lens, [1] * len(lens), bits=bits, page=64, KVH=KVH, HD=HD, ragged=False)
    held = c.fill(rng)
    q = (rng.standard_normal((c.n, QH, HD)) * (3.0 / np.sqrt(HD))).astype(F32)
    first = attend(c, scratch, q, QH)
    assert dev.status() == 0
    check_rows(c, held, q, first, QH, 0, 0, 1.0)
    n = c.n * QH * HD
    bq, of = dev.upload(q), dev.alloc(n * 4)
    for _ in range(50):
        dev.memset(of, 0xff)
        e4b.ops.attn_paged(dev, c.kv, bq, None, of, None, scratch, Q_HEADS=QH, ROWS=c.n)
        assert np.array_equal(dev.read(of, np.uint32, n), first[1].ravel().view(np.uint32))
    assert dev.status() == 0
    c.kv.free()


@pytest.mark.parametrize("rows", [2, 900])
def test_norm_weights_written_by_the_call_before(e4b, dev, rows):
    """The head prep's weights come out of a GEMV that lets its successor start early: they are read after it is done."""
    QH, KVH, HD, n_in = 4, 2, 128, 16384
    rng = np.random.default_rng(rows)
    raw = dev.upload(e4b.synth.quant_q4_0(e4b.synth.normal_f32(HD * n_in, 5, "w", 0.02)))
    x = dev.upload(rng.standard_normal((rows, (QH + 2 * KVH) * HD)).astype(F32))
    vecs = [dev.upload(rng.standard_normal(n_in).astype(F32)) for _ in range(2)]
    w, bq = dev.alloc(HD * 4), dev.alloc(rows * QH * HD * 4)
    c = Cache(e4b, dev, [3], [rows], bits=16, page=64, KVH=KVH, HD=HD, ragged=True)

    def prep(vec, wait):
        e4b.ops.q40mv(dev, vec, raw, None, w, IN=n_in, OUT=HD)
        if wait:
            dev.sync()
        e4b.ops.headprep_paged(dev, c.kv, x, w, w, bq, QH=QH, ROPE_ANGLES=HD // 2, THETA=1e4, ROWS=rows)
        return [dev.read(bq, F32, rows * QH * HD)] + c.read_rows()

    want = [prep(v, True) for v in vecs]
    assert not np.array_equal(want[0][0], want[1][0])
    for i in range(20):
        for a, b in zip(prep(vecs[i % 2], False), want[i % 2]):
            assert np.array_equal(a, b)
    assert dev.status() == 0


def write(c, xs, fill=0xff):
    """The sequences' keys and values xs[s] [slots][2][KVH][HD] into the pages, `fill` in every other byte; what the pages
    then stand for."""
    pools, held = c.pools(fill), []
    for s, x in enumerate(xs):
        x, t = x.astype(np.float16), np.arange(len(x))
        pid = c.table[s, t // c.page].astype(np.int64)
        for i, pool in enumerate(pools):
            pool.write_all(pid, t % c.page, x[:, i])
        held.append([pool.read_all(pid, t % c.page) for pool in pools])
    for pool, ptr in zip(pools, (c.kv.struct.k, c.kv.struct.v)):
        c.dev.write(ptr, pool.raw)
    return held


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("HD,QH,KVH,lens,counts", [(256, 8, 2, [70, 9, 333, 0], [1] * 4), (128, 4, 1, [70, 9, 333, 0], [1] * 4),
                                                   (64, 16, 4, [70, 9, 333, 0] * 12, [1] * 48), (256, 4, 1, [70, 9], [3, 20]),
                                                   (64, 7, 1, [70, 9], [3, 20])])
def test_bits_do_not_depend_on_hidden_bytes(e4b, dev, scratch, bits, HD, QH, KVH, lens, counts):  # noqa: F811
    """The rest of a last page, a page that the table does not name, and slots between the sinks and every row's window:
    zeros, NaN, or values a thousand times the visible ones change no bit of the outputs."""
    window, sinks, rng = 37, 5, np.random.default_rng(HD + QH)
    c = Cache(e4b, dev, lens, counts, bits=bits, page=32, KVH=KVH, HD=HD, ragged=max(counts) > 1)
    xs = [rng.standard_normal((a + b, 2, KVH, HD)) for a, b in zip(lens, counts)]
    q = (rng.standard_normal((c.n, QH, HD)) * (3.0 / np.sqrt(HD))).astype(F32)
    got = []
    for fill, factor in ((0xff, 1.0), (0x00, 1.0), (0x42, 1000.0)):
        ys = [x.copy() for x in xs]
        for y, n in zip(ys, lens):
            y[sinks:max(sinks, n - window + 1)] *= factor
        held = write(c, ys, fill)
        got.append(attend(c, scratch, q, QH, window=window, sinks=sinks))
        assert dev.status() == 0
    check_rows(c, held, q, got[-1], QH, window, sinks, 1.0)
    for g in got[1:]:
        for a, b in zip(g, got[0]):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


SIZES = {  # factors of the values' blocks of 32 dims in turn, and whether they change along the sequence
    "1e-4": ([1e-4], 0), "1e-6": ([1e-6], 0), "far apart": ([1.0, 1e-4, 30.0, 1e-6], 0), "0.01 beside 20": ([0.01, 20.0], 0),
    "huge beside small": ([5000.0, 1.0, 1e-3], 0), "falling": ([1.0, 1e-3], -1), "growing": ([1e-6, 1e-4, 1.0], 1),
    "zeros, then small": ([0.0, 1e-5], 1),
}


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("QH,counts", [(4, [1, 1, 1]), (3, [9, 1, 0])])
@pytest.mark.parametrize("name", SIZES)
def test_4_bit_values_of_any_size(e4b, dev, scratch, name, HD, QH, counts):  # noqa: F811
    """Every block of 32 dims is as precise relative to its own largest value.  Scores: at most 2^-16 of the sum of
    |q| times the block's largest |k|, which moves an output by twice that of vmax.  Products p d: 2^-22 of the largest p
    times vmax each (2^-16 beside scales of 2^7 or more), so n / sum(p / max p) of it in the output.  The rest, ex2
    (2^-22), three roundings of a product (2^-20), 17 addends cut at 2^-23 in each of the two MMAs of a piece (2^-18),
    f32 sums: 2^-16 altogether."""
    factors, change = SIZES[name]
    lens, rng = [700, 45, 3], np.random.default_rng(HD)
    c = Cache(e4b, dev, lens, counts, bits=4, page=32, KVH=1, HD=HD, ragged=max(counts) > 1)
    size, xs = np.array([factors[b % len(factors)] for b in range(HD // 32)]).repeat(32), []
    for n in (a + b for a, b in zip(lens, counts)):
        x = rng.standard_normal((n, 2, 1, HD))
        x[:, 1, 0] *= size * 2.0 ** (change * np.linspace(0, 6, n))[:, None]
        xs.append(x)
    held = write(c, xs)
    q = (rng.standard_normal((c.n, QH, HD)) * 2.0 ** -10 / np.sqrt(HD)).astype(F32)
    of = attend(c, scratch, q, QH)[1]
    assert dev.status() == 0
    wide = 2.0 ** -16 if max(factors) * (64 if change > 0 else 1) > 500 else 2.0 ** -22
    for r in range(c.n):
        s, p = c.place(r)
        k, v = (a[:p + 1, 0] for a in held[s])
        sc = q[r].astype(np.float64) @ k.T                                   # [QH][slots]
        w = np.exp(sc - sc.max(1, keepdims=True))
        want = w @ v / w.sum(1, keepdims=True)
        kmax = np.abs(k).reshape(-1, HD // 32, 32).max(-1).repeat(32, -1)
        ds = 2.0 ** -16 * (np.abs(q[r]).astype(np.float64) @ kmax.T).max(1)
        vmax = np.abs(v).reshape(-1, HD // 32, 32).max((0, 2)).repeat(32)
        tol = (2 * ds + 2.0 ** -16 + wide * (p + 1) / w.sum(1))[:, None] * vmax
        assert (np.abs(of[r] - want) <= tol).all(), (r, (np.abs(of[r] - want) / np.maximum(tol, 1e-300)).max())


def test_lengths_advance_by_the_rows_that_were_written(e4b, dev):
    """A rows table that claims more rows than the call has: the refused ones do not count, nor do ones out of order."""
    lens = [5, 0, 9, 2]
    for counts, n_rows, want, bad in (([2, 3, 1, 4], 10, [7, 3, 10, 6], 0), ([2, 3, 1, 4], 12, [7, 3, 10, 6], 0),
                                      ([2, 3, 1, 4], 4, [7, 2, 9, 2], 1), ([2, 3, 1, 4], 0, lens, 1)):
        c = Cache(e4b, dev, lens, counts, bits=16, page=16, KVH=1, HD=64, ragged=True)
        e4b.ops.paged_advance(dev, c.kv, ROWS=n_rows)
        assert list(dev.read(c.kv.struct.lens, np.uint32, 4)) == want and dev.status() == bad
    e4b.ops.paged_advance(dev, c.kv)                     # all of the table's
    assert list(dev.read(c.kv.struct.lens, np.uint32, 4)) == [7, 3, 10, 6] and dev.status() == 0
    c.kv.set_tables(lens=lens, rows=dev.upload(np.array([0, 6, 2, 2, 8], np.uint32)).ptr)
    e4b.ops.paged_advance(dev, c.kv)
    assert list(dev.read(c.kv.struct.lens, np.uint32, 4)) == [11, 0, 9, 8]
    c.kv.set_tables(lens=lens, rows=0)
    e4b.ops.paged_advance(dev, c.kv, ROWS=4)
    assert list(dev.read(c.kv.struct.lens, np.uint32, 4)) == [6, 1, 10, 3] and dev.status() == 0
    with pytest.raises(e4b.E4BError, match="paged_advance: "):
        e4b.ops.paged_advance(dev, c.kv, ROWS=3)         # without a table the call has a row a sequence


def test_refused_rows_stay_out_of_sight(e4b, dev, scratch):  # noqa: F811
    """Append, attention and advance with a row count below the table's: the next call does not see what was not written."""
    c = Cache(e4b, dev, [0, 0], [3, 5], bits=4, page=16, KVH=1, HD=64, ragged=True)
    x = np.random.default_rng(1).standard_normal((6, 3 * 64)).astype(F32)
    bq = dev.alloc(6 * 64 * 4)
    e4b.ops.headprep_paged(dev, c.kv, dev.upload(x), None, None, bq, QH=1, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=6)
    e4b.ops.paged_advance(dev, c.kv, ROWS=6)
    assert list(dev.read(c.kv.struct.lens, np.uint32, 2)) == [3, 3] and dev.status() == 1
    c.kv.set_tables(lens=[2, 2], rows=0)
    of = dev.alloc(2 * 64 * 4)
    e4b.ops.attn_paged(dev, c.kv, bq, None, of, None, scratch, Q_HEADS=1, ROWS=2)
    assert np.isfinite(dev.read(of, F32, 128)).all() and dev.status() == 0


@pytest.mark.parametrize("bits,HD,QH,KVH,window,sinks", [(4, 256, 16, 4, 0, 0), (16, 256, 8, 2, 500, 7), (4, 128, 8, 1, 300, 0),
                                                         (16, 64, 12, 4, 0, 0)])
def test_prompts_of_thousands_of_rows(e4b, dev, scratch, bits, HD, QH, KVH, window, sinks):  # noqa: F811
    """Tens of thousands of units, thousands on a CTA, among them one row of a long sequence; every 61st row checked."""
    rng = np.random.default_rng(HD)
    c = Cache(e4b, dev, [0, 2000, 40, 700], [2500, 1, 0, 1803], bits=bits, page=64, KVH=KVH, HD=HD, ragged=True, rows_cap=4310)
    held = c.fill(rng)
    q = (rng.standard_normal((c.n_rows, QH, HD)) * (3.0 / np.sqrt(HD))).astype(F32)
    got = attend(c, scratch, q, QH, window=window, sinks=sinks)
    assert dev.status() == 0
    check_rows(c, held, q, got, QH, window, sinks, 1.0, rows=sorted({*range(0, c.n, 61), 2499, 2500, 2501, c.n - 1}))
    c.kv.free()


@pytest.mark.parametrize("scale", [0.0, -0.7, 1e-30, 3e5])
@pytest.mark.parametrize("counts", [[1, 1], [5, 2]])
def test_scales_of_any_sign_and_size(e4b, dev, scratch, scale, counts):  # noqa: F811
    QH, HD, rng = 4, 64, np.random.default_rng(4)
    for bits in (4, 16):
        c = Cache(e4b, dev, [90, 0], counts, bits=bits, page=16, KVH=2, HD=HD, ragged=max(counts) > 1)
        held = c.fill(rng)
        q = (rng.standard_normal((c.n, QH, HD)) * 0.4).astype(F32)
        if scale > 1:
            q *= F32(1 / scale)
        got = attend(c, scratch, q, QH, scale=scale)
        assert dev.status() == 0
        check_rows(c, held, q, got, QH, 0, 0, float(F32(scale)))


WHOLE = {  # lens, QH, KVH: about as many units as CTAs, of nearly one length
    "64 of 1000..1100": (lambda r: [int(x) for x in r.integers(1000, 1101, 64)], 16, 4),
    "falling": (lambda r: list(range(1100, 1000, -2)), 15, 5),
    "37 x 4": (lambda r: [int(x) for x in r.integers(150, 200, 37)], 16, 4),
    "74 x 4": (lambda r: [int(x) for x in r.integers(150, 200, 74)], 4, 4),
    "8 heads": (lambda r: [int(x) for x in r.integers(1000, 1101, 36)], 32, 4),
    "some empty": (lambda r: [0, 40] * 36, 6, 2),
}


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
@pytest.mark.parametrize("bits,HD", [(4, 256), (16, 256), (4, 64), (16, 128)])
def test_units_that_stay_whole(e4b, dev, scratch, bits, HD, window, sinks):  # noqa: F811
    for name, (lens, QH, KVH) in WHOLE.items():
        rng = np.random.default_rng(HD)
        lens = lens(rng)
        c = Cache(e4b, dev, lens, [1] * len(lens), bits=bits, page=32, KVH=KVH, HD=HD, ragged=False)
        held = c.fill(rng)
        q = (rng.standard_normal((c.n, QH, HD)) * (3.0 / np.sqrt(HD))).astype(F32)
        got = attend(c, scratch, q, QH, window=window, sinks=sinks)
        assert dev.status() == 0, name
        check_rows(c, held, q, got, QH, window, sinks, 1.0, rows=range(0, c.n, 3))
        c.kv.free()


BORDERS = [2.0 ** -24, 2.0 ** -14 - 2.0 ** -24, 2.0 ** -14, 2.0 ** -7 - 2.0 ** -18, 2.0 ** -7, 2 - 2.0 ** -10, 2.0, 128 - 2.0 ** -4, 128.0, 8188.0]


@pytest.mark.parametrize("first,second", [(a, b) for i, a in enumerate(BORDERS) for b in (a, BORDERS[-1 - i], BORDERS[(i + 1) % 10])])
@pytest.mark.parametrize("QH,count", [(4, 1), (8, 1), (2, 7)])
def test_scales_at_the_borders_under_growing_scores(e4b, dev, scratch, QH, count, first, second):  # noqa: F811
    """Value scales at the borders of the kernel's classes, two blocks of one size and then of another, while the scores
    grow by 2^5.5 from turn to turn of the warps, so that p is as large as it may be: nothing overflows."""
    HD, n = 64, 900
    c = Cache(e4b, dev, [n - count, n - count], [count, count], bits=4, page=32, KVH=1, HD=HD, ragged=count > 1)
    t = np.arange(n)
    xs = []
    for turn in (5, 11):
        x = np.zeros((n, 2, 1, HD))
        x[:, 0, 0, 0] = np.minimum(5.5 * (t // (16 * turn)), 22.0)
        d = np.where(t < n // 2, first, second)
        x[:, 1, 0] = d[:, None] * np.random.default_rng(turn).integers(-8, 8, (n, HD))
        x[:, 1, 0, ::32] = -8 * d[:, None]
        xs.append(x)
    held = write(c, xs)
    assert np.array_equal(held[0][0], xs[0][:, 0]) and np.array_equal(held[0][1], xs[0][:, 1])
    q = np.zeros((c.n, QH, HD), F32)
    q[..., 0] = np.log(2.0)
    _, of, lse = attend(c, scratch, q, QH)
    assert dev.status() == 0
    for r in range(c.n):
        s, p = c.place(r)
        k, v = (a[:p + 1, 0] for a in held[s])
        sc = q[r].astype(np.float64) @ k.T
        w = np.exp(sc - sc.max(1, keepdims=True))
        # scores: 2^-16 of |q k| (see test_4_bit_values_of_any_size)
        tol = (2 * 2.0 ** -16 * sc.max() + 2.0 ** -16 + 2.0 ** -16 * (p + 1) / w.sum(1))[:, None] * np.abs(v).max()
        assert (np.abs(of[r] - w @ v / w.sum(1, keepdims=True)) <= tol).all()
