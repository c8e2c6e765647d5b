"""Paged KV cache on the GPU (e4b_headprep_paged, e4b_kvread_paged,
e4b_attn_paged, e4b_paged_advance) against the 64-bit oracle (oracle/paged.py).

Tolerances.  q: f32 arithmetic of a norm over HD values, a weight and a
rotation, at most 16 roundings of 2^-24 of |a| + |b| (the rotated pair).  K and V
in the cache: one rounding to f16 (2^-11) of a value known to 2^-24.
Attention: summing HD <= 256 products in f32 in any order is off by at most
2^-16 of S1 = scale * sum |q k|, and the softmax sum over n slots by n * 2^-24;
with |v| <= vmax that moves an output by at most vmax (2^-15 S1 + 2^-16 +
n 2^-24), and the rounding to f16 by 2^-11 of it."""
import ctypes

import numpy as np
import pytest

from oracle import paged as op

pytestmark = pytest.mark.gpu
F32, F64 = np.float32, np.float64


class Cache:
    """A paged cache on the device with the page table and lengths on the host; `poison` fills what nobody writes with
    NaN scales / NaN values."""

    def __init__(self, e4b, dev, lens, counts, *, bits, page, KVH, HD, ragged, seed=0, poison=True, spare=3, rows_cap=0):
        self.e4b, self.dev, self.bits, self.page, self.KVH, self.HD = e4b, dev, bits, page, KVH, HD
        self.lens, self.counts, self.nseq = list(lens), list(counts), len(lens)
        need = [max(1, -(-(a + b) // page)) for a, b in zip(lens, counts)]
        self.max_pages, self.n_pages = max(need) + 1, sum(need) + spare
        rng = np.random.default_rng(seed)
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.nseq, self.max_pages), 0xffffffff, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
        self.n = int(self.first[-1])
        self.ragged = ragged
        self.rows = dev.upload(self.first) if ragged else None
        self.kv = e4b.PagedKV(dev, BITS=bits, PAGE=page, PAGES=self.n_pages, MAX_PAGES=self.max_pages, SEQS=self.nseq,
                              KV_HEADS=KVH, HEAD_DIM=HD, rows=self.rows.ptr if ragged else None)
        self.kv.set_tables(self.table, self.lens)
        if poison:
            for p in (self.kv.struct.k, self.kv.struct.v):
                dev.memset(p, 0xff, self.kv.pool_bytes)
        self.n_rows = max(self.n, rows_cap)

    def place(self, r):
        s = int(np.searchsorted(self.first, r, side="right")) - 1 if self.ragged else r
        return s, self.lens[s] + (r - int(self.first[s]) if self.ragged else 0)

    def pools(self, fill=0xff):
        return [op.Pool(self.bits, self.page, self.n_pages, self.KVH, self.HD, v, fill) for v in (False, True)]

    def fill(self, rng, upto=None, scale=1.0, grow=0.0):
        """Random keys and values at every position below lens + counts, through the numpy layout; returns what the
        pages stand for, per sequence [slots][KVH][HD] in 64 bits."""
        pk, pv = self.pools()
        out = []
        for s in range(self.nseq):
            n = self.lens[s] + self.counts[s] if upto is None else upto[s]
            kk, vv = np.zeros((n, self.KVH, self.HD)), np.zeros((n, self.KVH, self.HD))
            x = rng.standard_normal((n, 2, self.KVH, self.HD)) * scale
            if grow:                                     # values that grow along the sequence
                x[:, 1] *= np.linspace(1, grow, n)[:, None, None]
            x, t = x.astype(np.float16), np.arange(n)
            pid = self.table[s, t // self.page].astype(np.int64)
            pk.write_all(pid, t % self.page, x[:, 0])
            pv.write_all(pid, t % self.page, x[:, 1])
            kk[:], vv[:] = pk.read_all(pid, t % self.page), pv.read_all(pid, t % self.page)
            out.append((kk, vv))
        self.dev.write(self.kv.struct.k, pk.raw)
        self.dev.write(self.kv.struct.v, pv.raw)
        return out

    def read_rows(self, f32=1):
        """(K, V) at the rows' positions through e4b_kvread_paged; rows past the last sequence keep the fill."""
        dt = F32 if f32 else np.float16
        n = self.n_rows * self.KVH * self.HD
        bk, bv = self.dev.upload(np.full(n, 7, dt)), self.dev.upload(np.full(n, 7, dt))
        self.e4b.ops.kvread_paged(self.dev, self.kv, bk, bv, F32=f32, ROWS=self.n_rows)
        return [self.dev.read(b, dt, n).reshape(self.n_rows, self.KVH, self.HD) for b in (bk, bv)]


@pytest.fixture()
def scratch(e4b, dev):
    b = dev.alloc(int(e4b.lib().e4b_paged_scratch_bytes()))
    yield b
    dev.free(b)


def attend(c, scratch, q, QH, *, window=0, sinks=0, scale=1.0, xfo=0, dev=None):
    dev = dev or c.dev
    n = c.n_rows * QH * c.HD
    oh, of = dev.upload(np.full(n, 3, np.float16)), dev.upload(np.full(n, 3, F32))
    lse = dev.upload(np.full(c.n_rows * QH, 5, F32))
    c.e4b.ops.attn_paged(dev, c.kv, dev.upload(q.astype(F32)), oh, of, lse, scratch, Q_HEADS=QH, WINDOW=window, SINKS=sinks,
                         SCALE=scale, XFO=xfo, ROWS=c.n_rows)
    dev.sync()
    return (dev.read(oh, np.float16, n).reshape(c.n_rows, QH * c.HD), dev.read(of, F32, n).reshape(c.n_rows, QH, c.HD),
            dev.read(lse, F32, c.n_rows * QH).reshape(c.n_rows, QH))


def check_rows(c, held, q, got, QH, window, sinks, scale, rows=None, usable=None):
    oh, of, lse = got
    for r in range(c.n) if rows is None else rows:
        s, p = c.place(r)
        k, v = held[s]
        u = None if usable is None else usable[s]
        ro, rl = op.attention(q[r], p, k, v, window, sinks, scale, u)
        see = op.visible(len(k), p, window, sinks)
        if u is not None:
            see &= u
        if not see.any():
            assert (of[r] == 0).all() and (oh[r] == 0).all() and np.isneginf(lse[r]).all()
            continue
        G = QH // c.KVH
        s1 = np.array([(abs(scale) * np.abs(k[see, h // G]) @ np.abs(q[r, h].astype(F64))).max() for h in range(QH)])
        vmax = np.abs(v[see]).max()
        tol = vmax * (2.0 ** -15 * s1 + 2.0 ** -16 + see.sum() * 2.0 ** -24)
        assert (np.abs(of[r] - ro) <= tol[:, None]).all(), (r, np.abs(of[r] - ro).max(), tol.max())
        h16 = oh[r].astype(F64).reshape(QH, c.HD)
        assert (np.abs(h16 - ro) <= tol[:, None] + 2.0 ** -11 * np.abs(ro) + 2.0 ** -25).all()
        assert (np.abs(lse[r] - rl) <= 2.0 ** -16 * s1 + see.sum() * 2.0 ** -24 + 2.0 ** -22 * (1 + np.abs(rl))).all()
    for r in range(c.n, c.n_rows):                       # padding rows stay as they were
        assert (oh[r] == 3).all() and (of[r] == 3).all() and (lse[r] == 5).all()


# ------------------------------------------------------------------ append
APPEND = [  # bits, HD, QH, KVH, page, lens, counts, options
    (4, 256, 16, 4, 64, [0, 63, 64, 1000], [1, 1, 1, 1], {}),
    (16, 256, 8, 2, 16, [15, 0, 7], [1, 1, 1], dict(keqv=1, frac=0.25, theta=1e6)),
    (4, 128, 4, 1, 16, [0, 5, 31, 40], [17, 0, 33, 1], dict(pad=5)),
    (16, 64, 6, 2, 48, [100, 3], [50, 7], dict(norm=0)),
    (4, 64, 3, 3, 32, [2, 0, 30], [5, 1, 40], dict(half=1)),
    (16, 128, 5, 5, 128, [1, 127], [1, 2], dict(half=1, keqv=1, norm=0, pad=1)),
    (4, 256, 0, 2, 16, [9], [20], dict(stride=64)),
    (4, 128, 8, 8, 16, [70000, 131], [3, 2], dict(nparts=3)),
    (16, 256, 16, 4, 64, [100000], [4], dict(stride=4, theta=1e6)),
    # many rows: whole rows by bulk copies, or (partial sums, rows of 8-byte alignment or over 48 KB) by loads;
    # several turns and look-ups a CTA, sequences that begin and end within one
    (4, 64, 1, 1, 16, [0, 5, 100000, 3, 9, 31], [7000, 0, 13, 6487, 1, 7000], dict(half=1)),
    (4, 64, 1, 1, 32, [0, 5, 100000, 3, 9, 31], [7000, 0, 13, 6487, 1, 7000], dict(nparts=2)),
    (16, 256, 8, 2, 64, [0, 77, 1000], [333, 1, 400], dict(pad=9)),
    (4, 128, 16, 2, 16, [5, 0], [700, 640], dict(half=1, offset=8)),
    (4, 256, 64, 2, 64, [0, 9], [100, 90], {}),
    (4, 256, 40, 4, 16, [0], [200], {}),
    (16, 64, 14, 2, 48, [3], [801], dict(half=1, keqv=1, frac=0.3, stride=4, norm=0)),
    (16, 64, 14, 2, 48, [3], [801], dict(half=1, keqv=1, frac=0.3, stride=8, theta=1e6)),
    (4, 128, 0, 6, 16, [0] * 900, [1] * 900, {}),
]


@pytest.mark.parametrize("case", APPEND, ids=[f"{c[0]}bit-hd{c[1]}-{c[2]}q{c[3]}kv-{i}" for i, c in enumerate(APPEND)])
def test_append_and_read_back(e4b, dev, case):
    bits, HD, QH, KVH, page, lens, counts, o = case
    keqv, norm, half = o.get("keqv", 0), o.get("norm", 1), o.get("half", 0)
    nparts, theta = o.get("nparts", 1), o.get("theta", 1e4)
    angles = int(o.get("frac", 1.0) * HD // 2)
    rng = np.random.default_rng(HD + bits + QH)
    c = Cache(e4b, dev, lens, counts, bits=bits, page=page, KVH=KVH, HD=HD, ragged=any(n != 1 for n in counts),
              rows_cap=sum(counts) + o.get("pad", 0))
    width = (QH + KVH * (1 if keqv else 2)) * HD
    stride = width + o.get("stride", 0)
    x = rng.standard_normal((nparts, c.n_rows, stride)).astype(np.float16 if half else F32)
    qw, kw = (1 + 0.2 * rng.standard_normal(HD)).astype(F32), (1 + 0.2 * rng.standard_normal(HD)).astype(F32)
    bq = dev.upload(np.full(max(1, c.n_rows * QH * HD), 9, F32))
    off = o.get("offset", 0) // x.itemsize
    bx = dev.upload(np.concatenate([np.zeros(off, x.dtype), x.ravel()]))
    args = (bx.ptr + off * x.itemsize, dev.upload(qw), dev.upload(kw), bq if QH else None)
    kws = dict(QH=QH, ROPE_ANGLES=angles, THETA=theta, NORM=norm, KEQV=keqv, XF16=half, NPARTS=nparts, ROWS=c.n_rows,
               STRIDE=stride if o.get("stride") else 0)
    e4b.ops.headprep_paged(dev, c.kv, *args, **kws)
    got_k, got_v = c.read_rows()
    assert dev.status() == 0
    rows = x[0].copy()
    for part in x[1:]:
        rows = rows + part                               # in order, in the partials' type
    pos = [c.place(r)[1] for r in range(c.n)]
    rq, rk, rv = op.headprep(rows[:c.n, :width], pos, qw, kw, QH, KVH, HD, angles, theta, 1e-6, norm, keqv)
    got_q = dev.read(bq, F32, c.n_rows * QH * HD).reshape(c.n_rows, QH, HD)
    if QH:
        pair = np.abs(rq) + np.abs(np.roll(rq, HD // 2, axis=-1))
        assert (np.abs(got_q[:c.n] - rq) <= 16 * 2.0 ** -24 * np.sqrt(2) * pair).all()
        assert (got_q[c.n:] == 9).all()
    assert (got_k[c.n:] == 7).all() and (got_v[c.n:] == 7).all()
    # the f16 rows: of an f16 cache directly, of a 4-bit one from the same call on an f16 cache
    if bits == 4:
        c16 = Cache(e4b, dev, lens, counts, bits=16, page=page, KVH=KVH, HD=HD, ragged=c.ragged, rows_cap=c.n_rows)
        e4b.ops.headprep_paged(dev, c16.kv, *args, **kws)
        k16, v16 = c16.read_rows()
    else:
        k16, v16 = got_k, got_v
    for g, r in ((k16, rk), (v16, rv)):
        assert (np.abs(g[:c.n] - r) <= 2.0 ** -11 * np.abs(r) * (1 + 2.0 ** -10) + 2.0 ** -25).all()
    if bits == 4:                                        # exactly the rule's codes and scales, in the documented places
        for g, x16 in ((got_k, k16), (got_v, v16)):
            assert np.array_equal(g[:c.n].astype(F64), op.dequantise(*op.quantise(x16[:c.n].astype(np.float16))))
    pools = c.pools()
    seqs, at = np.array([c.place(r)[0] for r in range(c.n)]), np.array(pos)
    for pool, x16 in zip(pools, (k16, v16)):
        pool.write_all(c.table[seqs, at // page].astype(np.int64), at % page, x16[:c.n])
    for pool, ptr in zip(pools, (c.kv.struct.k, c.kv.struct.v)):   # every other byte is what it was
        assert np.array_equal(dev.read(ptr, np.uint8, c.kv.pool_bytes), pool.raw)
    k2, v2 = c.read_rows(f32=0)
    assert np.array_equal(k2[:c.n], got_k[:c.n].astype(np.float16)) and np.array_equal(v2[:c.n], got_v[:c.n].astype(np.float16))


def test_codes_between_two_and_of_two_largest(e4b, dev):
    """Blocks of halves and small integers (quotients exactly between two codes, largest magnitudes of both signs in
    either order, repeated), of f16's smallest and largest values, and random ones, code by code."""
    rng = np.random.default_rng(4)
    HD, n = 128, 1500                                    # (few rows and many use one quantiser; this is the staged path)
    x = rng.integers(-16, 17, (n, 2, HD)) * 0.5
    x[300:600] = rng.integers(-3, 4, (300, 2, HD))
    x[600:700] *= 2.0 ** -24 * 2
    x[700:800] = rng.choice([65504.0, -65504.0, 32752.0, 4094.0], (100, 2, HD))
    x[800:] = rng.standard_normal((700, 2, HD)) * 2.0 ** rng.integers(-20, 12, (700, 1, 1))
    x16 = x.astype(np.float16)
    c = Cache(e4b, dev, [0], [n], bits=4, page=64, KVH=1, HD=HD, ragged=True)
    e4b.ops.headprep_paged(dev, c.kv, dev.upload(x16), None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, XF16=1,
                           ROWS=n)
    assert dev.status() == 0
    for ptr, pool, i in zip((c.kv.struct.k, c.kv.struct.v), c.pools(), (0, 1)):
        t = np.arange(n)
        pool.write_all(c.table[0, t // 64].astype(np.int64), t % 64, x16[:, i:i + 1])
        assert np.array_equal(dev.read(ptr, np.uint8, c.kv.pool_bytes), pool.raw)


def test_append_of_infinities_and_zeros(e4b, dev):
    for bits in (4, 16):
        c = Cache(e4b, dev, [3, 4], [1, 1], bits=bits, page=16, KVH=1, HD=64, ragged=False)
        x = np.zeros((2, 2 * 64), F32)
        x[1, :] = 1.0
        x[1, 5], x[1, 64 + 40] = np.inf, np.nan
        e4b.ops.headprep_paged(dev, c.kv, dev.upload(x), None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=2)
        k, v = c.read_rows()
        assert dev.status() == 0 and (k[0] == 0).all() and (v[0] == 0).all()
        bad = np.zeros((2, 64), bool)
        if bits == 4:
            bad[0, :32] = bad[1, 32:] = True
            assert np.isnan(k[1, 0][bad[0]]).all() and np.isnan(v[1, 0][bad[1]]).all()
        else:
            bad[0, 5] = bad[1, 40] = True
            assert np.isinf(k[1, 0, 5]) and np.isnan(v[1, 0, 40])
        assert (k[1, 0][~bad[0]] == 1).all() and (v[1, 0][~bad[1]] == 1).all()


def test_positions_and_pages_out_of_range(e4b, dev):
    c = Cache(e4b, dev, [3, 16 * 3 - 1, 5], [2, 2, 1], bits=4, page=16, KVH=2, HD=64, ragged=True)
    full = c.max_pages * c.page
    c.lens[1] = full - 1                                 # its second row is past the table
    c.table[1, -1] = c.table[1, 0]
    c.table[2, 0] = c.n_pages                            # names no page
    c.kv.set_tables(c.table, c.lens)
    before = dev.read(c.kv.struct.k, np.uint8, c.kv.pool_bytes)
    x = np.random.default_rng(1).standard_normal((5, 4 * 64)).astype(F32)
    e4b.ops.headprep_paged(dev, c.kv, dev.upload(x), None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=5)
    assert dev.status() == 1 and dev.status() == 0
    k, v = c.read_rows()
    assert dev.status() == 1
    assert (k[3:] == 0).all() and (v[3:] == 0).all() and np.abs(k[:3]).min(axis=(1, 2)).max() < 1 and (k[:3] != 0).any()
    after = dev.read(c.kv.struct.k, np.uint8, c.kv.pool_bytes)
    touched = {int(i) // (c.page // 16 * c.KVH * 9 * 64) for i in np.flatnonzero(before != after)}
    assert touched <= {int(c.table[0, 0]), int(c.table[1, -1])}
    # a rows table that claims more rows than the buffers hold
    c2 = Cache(e4b, dev, [0, 0], [2, 6], bits=16, page=16, KVH=1, HD=64, ragged=True)
    x = np.ones((4, 128), F32)
    e4b.ops.headprep_paged(dev, c2.kv, dev.upload(x), None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=4)
    assert dev.status() == 1


# ------------------------------------------------------------------ attention
ATTN = [  # bits, HD, QH, KVH, page, lens, counts, window, sinks, scale
    (4, 256, 16, 4, 64, [0, 1, 15, 16, 17, 63, 64, 500], [1] * 8, 0, 0, 1.0),
    (16, 256, 16, 4, 64, [0, 1, 15, 16, 17, 63, 64, 500], [1] * 8, 0, 0, 1.0),
    (4, 128, 4, 1, 16, [700, 40, 0], [1, 1, 1], 100, 4, 0.7),
    (16, 128, 4, 1, 16, [700, 40, 0], [1, 1, 1], 100, 4, 0.7),
    (4, 64, 2, 2, 32, [333, 0], [1, 1], 0, 0, 1.0),
    (16, 64, 3, 1, 48, [333, 2], [1, 1], 33, 17, 1.0),
    (4, 256, 8, 1, 16, [900], [1], 0, 0, 1.0),
    (16, 256, 5, 1, 16, [300, 9], [1, 1], 0, 0, 1.0),
    (4, 128, 12, 2, 64, [200], [1], 1, 0, 1.0),
    (4, 128, 12, 2, 64, [200], [1], 1, 1, 1.0),
    (4, 256, 16, 4, 64, [0, 130, 5, 77], [33, 1, 0, 18], 0, 0, 1.0),
    (16, 256, 4, 1, 32, [0, 130], [33, 6], 20, 3, 1.0),
    (4, 64, 8, 8, 16, [50, 0], [40, 3], 16, 40, 1.0),
    (16, 64, 14, 2, 16, [250, 1], [5, 20], 0, 0, 0.5),
    (4, 128, 8, 2, 128, [3000], [3], 0, 0, 1.0),
    (16, 128, 6, 2, 16, [1500, 3], [2, 2], 512, 0, 1.0),
]


@pytest.mark.parametrize("case", ATTN, ids=[f"{c[0]}bit-hd{c[1]}-{c[2]}q{c[3]}kv-{i}" for i, c in enumerate(ATTN)])
def test_attention_matches_the_oracle(e4b, dev, scratch, case):
    bits, HD, QH, KVH, page, lens, counts, window, sinks, scale = case
    rng = np.random.default_rng(HD + bits + QH + len(lens))
    c = Cache(e4b, dev, lens, counts, bits=bits, page=page, KVH=KVH, HD=HD, ragged=any(n != 1 for n in counts),
              rows_cap=sum(counts) + (4 if any(n != 1 for n in counts) else 0))
    held = c.fill(rng)
    q = rng.standard_normal((c.n_rows, QH, HD)) * (3.0 / np.sqrt(HD))
    got = attend(c, scratch, q, QH, window=window, sinks=sinks, scale=scale)
    assert dev.status() == 0
    q = q.astype(F32)
    check_rows(c, held, q, got, QH, window, sinks, scale)
    again = attend(c, scratch, q, QH, window=window, sinks=sinks, scale=scale)
    for a, b in zip(got, again):                         # the same bits every time
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    xfo = attend(c, scratch, q, QH, window=window, sinks=sinks, scale=scale, xfo=1)[0]
    assert np.array_equal(e4b.batch.to_xfo(got[0].view(np.uint16))[:c.n], xfo.view(np.uint16)[:c.n])


@pytest.mark.parametrize("bits", [4, 16])
def test_attention_sharp_flat_and_growing_scores(e4b, dev, scratch, bits):
    """Scores that grow along the sequence (the maximum moves at every slot), far apart (one slot takes all), equal
    (zero queries), and huge or tiny queries."""
    QH, KVH, HD = 4, 1, 64
    c = Cache(e4b, dev, [600] * 5, [1] * 5, bits=bits, page=16, KVH=KVH, HD=HD, ragged=False)
    rng = np.random.default_rng(3)
    pk, pv = c.pools()
    held = []
    for s in range(5):
        kk, vv = np.zeros((601, 1, HD)), np.zeros((601, 1, HD))
        for t in range(601):
            pid = int(c.table[s, t // 16])
            row = rng.standard_normal((1, HD)).astype(np.float16)
            if s == 0:
                row = (np.sign(row) * (0.2 + 0.01 * t)).astype(np.float16) * np.sign(np.arange(HD) - 31.5).astype(np.float16) ** 2
                row = np.abs(row)
            pk.write(pid, t % 16, row)
            pv.write(pid, t % 16, rng.standard_normal((1, HD)).astype(np.float16))
            kk[t], vv[t] = pk.read(pid, t % 16), pv.read(pid, t % 16)
        held.append((kk, vv))
    dev.write(c.kv.struct.k, pk.raw)
    dev.write(c.kv.struct.v, pv.raw)
    q = rng.standard_normal((5, QH, HD))
    q[0] = 0.05
    q[1] *= 40.0
    q[2] = 0.0
    q[3] *= 1e-20
    q[4] *= 2e4
    q = q.astype(F32)
    got = attend(c, scratch, q, QH)
    assert dev.status() == 0
    check_rows(c, held, q, got, QH, 0, 0, 1.0, rows=[0, 1, 2, 3])
    # scores near 1e5: the best slot takes all unless two are closer than the scores' own rounding
    assert np.isfinite(got[1]).all() and np.abs(got[1][4]).max() <= np.abs(held[4][1]).max() * (1 + 2.0 ** -16)
    for h in range(QH):
        s = held[4][0][:, 0] @ q[4, h].astype(F64)
        top = np.sort(s)
        if top[-1] - top[-2] > 2 * 2.0 ** -16 * (np.abs(held[4][0][:, 0]) @ np.abs(q[4, h].astype(F64))).max() + 20:
            assert (np.abs(got[1][4, h] - held[4][1][s.argmax(), 0]) <= 2.0 ** -16 * 8).all()


@pytest.mark.parametrize("bits", [4, 16])
def test_hidden_slots_may_hold_anything(e4b, dev, scratch, bits):
    """Hidden middle pages need no valid id; slots behind a row's position, outside its window or in the rest of the last
    page may hold NaN, also where another row of the same call sees them."""
    QH, KVH, HD, window, sinks = 4, 1, 128, 20, 5
    c = Cache(e4b, dev, [300, 0], [6, 4], bits=bits, page=16, KVH=KVH, HD=HD, ragged=True)
    held = c.fill(np.random.default_rng(5))
    for j in range(1, 281 // 16):
        c.table[0, j] = 0xfffffffe                       # positions 16..271 are hidden from 300..305
    c.kv.set_tables(c.table, c.lens)
    q = np.random.default_rng(6).standard_normal((c.n_rows, QH, HD)).astype(F32) * 0.2
    got = attend(c, scratch, q, QH, window=window, sinks=sinks)
    assert dev.status() == 0
    check_rows(c, held, q, got, QH, window, sinks, 1.0)
    # the last two rows' own tokens become NaN: earlier rows do not see them
    x = np.full((c.n, 2 * HD), np.nan, F32)
    keep = c.lens[:]
    bad = e4b.PagedKV(dev, BITS=bits, PAGE=16, PAGES=c.n_pages, MAX_PAGES=c.max_pages, SEQS=2, KV_HEADS=KVH, HEAD_DIM=HD,
                      k=c.kv.struct.k, v=c.kv.struct.v, pages=c.kv.struct.pages)
    bad.set_tables(lens=[304, 2], rows=dev.upload(np.array([0, 2, 4], np.uint32)).ptr)
    e4b.ops.headprep_paged(dev, bad, dev.upload(x), None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=4)
    assert keep == c.lens
    got = attend(c, scratch, q, QH, window=window, sinks=sinks)
    check_rows(c, held, q, got, QH, window, sinks, 1.0, rows=[0, 1, 2, 3, 6, 7])
    for r in (4, 5, 8, 9):
        assert np.isnan(got[1][r]).all()


def test_rows_that_see_nothing_and_missing_pages(e4b, dev, scratch):
    for bits in (4, 16):
        c = Cache(e4b, dev, [40, 33, 20], [1, 1, 1], bits=bits, page=16, KVH=2, HD=64, ragged=False)
        held = c.fill(np.random.default_rng(9))
        usable = [np.ones(41, bool), np.ones(34, bool), np.zeros(21, bool)]
        c.table[0, 1] = 0xffffffff                       # slots 16..31 of the first sequence
        c.table[2, :] = c.n_pages                        # every slot of the third
        usable[0][16:32] = False
        c.kv.set_tables(c.table, c.lens)
        q = np.random.default_rng(2).standard_normal((3, 4, 64)).astype(F32) * 0.3
        got = attend(c, scratch, q, 4)
        assert dev.status() == 1
        check_rows(c, held, q, got, 4, 0, 0, 1.0, usable=usable)
        # a position past the page table
        c.kv.set_tables(lens=[c.max_pages * 16, 33, c.max_pages * 16 + 500])
        got = attend(c, scratch, q, 4, window=8)
        assert dev.status() == 1 and (got[1][2] == 0).all() and np.isneginf(got[2][2]).all()
        check_rows(c, held, q, got, 4, 8, 0, 1.0, rows=[1])


def test_many_short_sequences_and_a_long_one(e4b, dev, scratch):
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 30, 700)] + [2500] + [0] * 99
    c = Cache(e4b, dev, lens, [1] * 800, bits=4, page=16, KVH=1, HD=64, ragged=False)
    held = c.fill(rng)
    q = (rng.standard_normal((800, 2, 64)) * 0.3).astype(F32)
    got = attend(c, scratch, q, 2)
    assert dev.status() == 0
    check_rows(c, held, q, got, 2, 0, 0, 1.0)


SHAPES = {  # lens, counts, QH, KVH: which rows, heads and lengths choose the kernel's forms and how its work is cut
    "two CTAs per SM": (lambda r: [int(x) for x in r.integers(0, 260, 40)], [1] * 40, 16, 4),
    "equal units, two CTAs per SM": (lambda r: [200] * 64, [1] * 64, 8, 4),
    "equal units, one CTA per SM": (lambda r: [333] * 40, [1] * 40, 6, 3),
    "nearly equal units": (lambda r: [int(x) for x in 300 + r.integers(0, 16, 35)], [1] * 35, 16, 4),
    "long and short": (lambda r: [9000, 7], [1, 1], 3, 1),
    "long, 8 heads": (lambda r: [0, 9000], [1, 1], 8, 1),
    "long, rows": (lambda r: [8000, 3], [9, 40], 7, 1),
    "prompts": (lambda r: [0, 100, 0, 31], [130, 70, 0, 1], 4, 2),
    "equal prompts": (lambda r: [64] * 10, [16] * 10, 8, 2),
    "short rows of one head": (lambda r: [5] * 50, [3] * 50, 4, 4),
    "six heads": (lambda r: [int(x) for x in r.integers(0, 700, 9)], [2] * 9, 12, 2),
}


@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 20)])
@pytest.mark.parametrize("bits,HD", [(4, 64), (4, 128), (4, 256), (16, 64), (16, 128), (16, 256)])
def test_attention_however_the_work_is_cut(e4b, dev, scratch, bits, HD, window, sinks):
    for i, (name, (lens, counts, QH, KVH)) in enumerate(SHAPES.items()):
        rng = np.random.default_rng(100 * i + HD)
        lens = lens(rng)
        c = Cache(e4b, dev, lens, counts, bits=bits, page=(16, 48, 64)[i % 3], KVH=KVH, HD=HD, ragged=any(n != 1 for n in counts))
        held = c.fill(rng)
        q = (rng.standard_normal((c.n_rows, QH, HD)) * (3.0 / np.sqrt(HD))).astype(F32)
        got = attend(c, scratch, q, QH, window=window, sinks=sinks)
        assert dev.status() == 0, name
        check_rows(c, held, q, got, QH, window, sinks, 1.0)
        clean = dev.alloc(int(e4b.lib().e4b_paged_scratch_bytes()))    # scratch used by other shapes: no trace
        again = attend(c, clean, q, QH, window=window, sinks=sinks)
        dev.free(clean)
        for a, b in zip(got, again):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), name
        c.kv.free()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("QH,counts", [(4, [1, 1]), (8, [1, 1]), (4, [9, 4])])
def test_values_that_grow_large(e4b, dev, scratch, bits, QH, counts):
    """Value scales from far below 2 to hundreds within a sequence: p gives up its lift on the way."""
    rng = np.random.default_rng(21)
    c = Cache(e4b, dev, [900, 500], counts, bits=bits, page=32, KVH=1, HD=128, ragged=max(counts) > 1)
    held = c.fill(rng, grow=4000.0)
    q = (rng.standard_normal((c.n_rows, QH, 128)) * 0.3).astype(F32)
    got = attend(c, scratch, q, QH)
    assert dev.status() == 0
    check_rows(c, held, q, got, QH, 0, 0, 1.0)


def test_no_rows_and_only_padding(e4b, dev, scratch):
    c = Cache(e4b, dev, [20, 5, 40], [0, 0, 0], bits=4, page=16, KVH=2, HD=64, ragged=True, rows_cap=4)
    held = c.fill(np.random.default_rng(1))
    before = dev.read(c.kv.struct.k, np.uint8, c.kv.pool_bytes)
    q = np.ones((4, 4, 64), F32)
    check_rows(c, held, q, attend(c, scratch, q, 4), 4, 0, 0, 1.0)
    x = dev.upload(np.ones((4, 4 * 64), F32))
    for rows in (4, 0):
        e4b.ops.headprep_paged(dev, c.kv, x, None, None, None, QH=0, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=rows)
    c.n_rows = 0
    attend(c, scratch, np.ones((1, 4, 64), F32), 4)
    assert dev.status() == 0
    assert np.array_equal(dev.read(c.kv.struct.k, np.uint8, c.kv.pool_bytes), before)


def test_as_many_sequences_as_there_may_be(e4b, dev, scratch):
    rng = np.random.default_rng(31)
    n = 4096
    lens = [int(x) for x in rng.integers(0, 40, n)]
    c = Cache(e4b, dev, lens, [1] * n, bits=4, page=16, KVH=1, HD=64, ragged=False)
    held = c.fill(rng)
    q = (rng.standard_normal((n, 1, 64)) * 0.3).astype(F32)
    got = attend(c, scratch, q, 1)
    assert dev.status() == 0
    check_rows(c, held, q, got, 1, 0, 0, 1.0, rows=range(0, n, 7))
    # the same cache under a rows table: every row its own sequence's, some sequences without one
    counts = np.array([s % 3 for s in range(n)])
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    c.kv.set_tables(lens=np.array(lens) + 1 - np.minimum(counts, np.array(lens) + 1), rows=dev.upload(first).ptr)
    q2 = (rng.standard_normal((int(first[-1]), 1, 64)) * 0.3).astype(F32)
    c.n_rows = int(first[-1])
    got = attend(c, scratch, q2, 1)
    assert dev.status() == 0
    for s in range(0, n, 11):
        for j in range(counts[s]):
            r, p = int(first[s]) + j, lens[s] + 1 - min(counts[s], lens[s] + 1) + j
            if p > lens[s]:
                continue                                 # a slot that nobody wrote
            ro, _ = op.attention(q2[r], p, held[s][0], held[s][1], 0, 0, 1.0)
            assert np.abs(got[1][r] - ro).max() <= np.abs(held[s][1]).max() * 2.0 ** -10


def test_two_contexts_at_once(e4b, dev):
    """Calls of two contexts overlap on the device, each with its own scratch; the results are those of one at a time."""
    other = e4b.Device(0)
    try:
        sets = []
        for d, seed in ((dev, 1), (other, 2)):
            rng = np.random.default_rng(seed)
            c = Cache(e4b, d, [6000, 100, 3000], [5, 1, 2], bits=4, page=64, KVH=2, HD=128, ragged=True)
            c.fill(rng)
            s = d.alloc(int(e4b.lib().e4b_paged_scratch_bytes()))
            q = d.upload((rng.standard_normal((c.n_rows, 8, 128)) * 0.3).astype(F32))
            sets.append((d, c, s, q, [d.alloc(c.n_rows * 8 * 128 * 4) for _ in range(2)]))
        for which in range(2):
            for d, c, s, q, outs in sets:
                for _ in range(1 if which == 0 else 20):
                    e4b.ops.attn_paged(d, c.kv, q, None, outs[which], None, s, Q_HEADS=8, ROWS=c.n_rows)
                if which == 0:
                    d.sync()
            for d, *_ in sets:
                d.sync()
        for d, c, s, q, outs in sets:
            assert d.status() == 0
            a, b = (d.read(o, np.uint8, c.n_rows * 8 * 128 * 4) for o in outs)
            assert np.array_equal(a, b) and a.any()
    finally:
        other.close()


def test_offsets_past_4_gib(e4b, dev, scratch):
    """Pages at the top of pools of 4.3 GB each."""
    KVH, HD, page = 8, 256, 64
    n_pages = (1 << 32) // (KVH * page * HD * 2) + 64
    kv = e4b.PagedKV(dev, BITS=16, PAGE=page, PAGES=n_pages, MAX_PAGES=2, SEQS=1, KV_HEADS=KVH, HEAD_DIM=HD)
    assert kv.pool_bytes > 1 << 32
    try:
        kv.set_tables(np.array([[n_pages - 1, n_pages - 3]]), [0], rows=dev.upload(np.array([0, 70], np.uint32)).ptr)
        rng = np.random.default_rng(8)
        x = rng.standard_normal((70, 3 * KVH * HD)).astype(F32)
        bq = dev.alloc(70 * KVH * HD * 4)
        e4b.ops.headprep_paged(dev, kv, dev.upload(x), None, None, bq, QH=KVH, ROPE_ANGLES=0, THETA=1e4, NORM=0, ROWS=70)
        of = dev.alloc(70 * KVH * HD * 4)
        e4b.ops.attn_paged(dev, kv, bq, None, of, None, scratch, Q_HEADS=KVH, SCALE=1 / 16.0, ROWS=70)
        assert dev.status() == 0
        o = dev.read(of, F32, 70 * KVH * HD).reshape(70, KVH, HD)
        x = x.reshape(70, 3, KVH, HD)
        k, v = x[:, 1].astype(np.float16).astype(F64), x[:, 2].astype(np.float16).astype(F64)
        for r in (0, 63, 64, 69):
            ro, _ = op.attention(x[r, 0], r, k, v, 0, 0, 1 / 16.0)
            assert np.abs(o[r] - ro).max() <= np.abs(v).max() * (2.0 ** -15 * 256 * 16 / 16 + 2.0 ** -15)
    finally:
        kv.free()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
def test_prompt_then_recorded_decode_steps(e4b, dev, scratch, bits, window, sinks):
    """A ragged prompt in one call, then a recorded plan of (append, attention, advance) replayed: every step's output
    and the final cache against the oracle run over the rows that kvread gives back."""
    QH, KVH, HD, page, steps = 8, 2, 128, 16, 21
    prompt = [37, 0, 12, 1]
    c = Cache(e4b, dev, [0] * 4, prompt, bits=bits, page=page, KVH=KVH, HD=HD, ragged=True)
    c.max_pages = 5
    c.n_pages = 20
    rng = np.random.default_rng(bits + window)
    table = rng.permutation(20).reshape(4, 5).astype(np.uint32)
    kv = e4b.PagedKV(dev, BITS=bits, PAGE=page, PAGES=20, MAX_PAGES=5, SEQS=4, KV_HEADS=KVH, HEAD_DIM=HD)
    c.kv, c.table, first = kv, table, dev.upload(np.concatenate([[0], np.cumsum(prompt)]).astype(np.uint32))
    kv.set_tables(table, [0] * 4, rows=first.ptr)
    n0, width = sum(prompt), (QH + 2 * KVH) * HD
    qw, kw = (dev.upload((1 + 0.1 * rng.standard_normal(HD)).astype(F32)) for _ in range(2))
    prep = dict(QH=QH, ROPE_ANGLES=HD // 2, THETA=1e4)
    xp = rng.standard_normal((n0, width)).astype(F32)
    bq, bo = dev.alloc(n0 * QH * HD * 4), dev.alloc(n0 * QH * HD * 4)
    e4b.ops.headprep_paged(dev, kv, dev.upload(xp), qw, kw, bq, ROWS=n0, **prep)
    e4b.ops.attn_paged(dev, kv, bq, None, bo, None, scratch, Q_HEADS=QH, WINDOW=window, SINKS=sinks, SCALE=0.09, ROWS=n0)
    e4b.ops.paged_advance(dev, kv)
    op0, q0 = dev.read(bo, F32, n0 * QH * HD).reshape(n0, QH, HD), dev.read(bq, F32, n0 * QH * HD).reshape(n0, QH, HD)
    assert list(dev.read(kv.struct.lens, np.uint32, 4)) == prompt
    kv.set_tables(rows=0)
    bx, bq, bo = dev.alloc(4 * width * 4), dev.alloc(4 * QH * HD * 4), dev.alloc(4 * QH * HD * 4)
    xs = rng.standard_normal((steps, 4, width)).astype(F32)

    def step():
        e4b.ops.headprep_paged(dev, kv, bx, qw, kw, bq, ROWS=4, **prep)
        e4b.ops.attn_paged(dev, kv, bq, None, bo, None, scratch, Q_HEADS=QH, WINDOW=window, SINKS=sinks, SCALE=0.09, ROWS=4)
        e4b.ops.paged_advance(dev, kv)

    plan = ctypes.c_int()
    dev.call("e4b_plan_begin")
    step()
    dev.call("e4b_plan_end", ctypes.byref(plan))
    outs, qs = [], []
    for i in range(steps):
        dev.write(bx, xs[i])
        if i % 5 == 4:
            step()                                       # a plain call among the replays
        else:
            dev.call("e4b_plan_launch", plan.value, 1)
        outs.append(dev.read(bo, F32, 4 * QH * HD).reshape(4, QH, HD))
        qs.append(dev.read(bq, F32, 4 * QH * HD).reshape(4, QH, HD))
    dev.call("e4b_plan_destroy", plan.value)
    lens = [p + steps for p in prompt]
    assert list(dev.read(kv.struct.lens, np.uint32, 4)) == lens and dev.status() == 0
    # everything that the cache holds, read back as rows of zero-length prefixes
    full = Cache(e4b, dev, [0] * 4, lens, bits=bits, page=page, KVH=KVH, HD=HD, ragged=True)
    full.kv = e4b.PagedKV(dev, BITS=bits, PAGE=page, PAGES=20, MAX_PAGES=5, SEQS=4, KV_HEADS=KVH, HEAD_DIM=HD,
                          k=kv.struct.k, v=kv.struct.v, pages=kv.struct.pages, rows=full.rows.ptr)
    full.kv.set_tables(lens=[0] * 4)
    k, v = (a.astype(F64) for a in full.read_rows())
    vmax = np.abs(v).max()
    for s in range(4):
        ks, vs = k[full.first[s]:full.first[s + 1]], v[full.first[s]:full.first[s + 1]]

        def check(o, q, p):
            ro, _ = op.attention(q, p, ks, vs, window, sinks, float(F32(0.09)))
            s1 = 0.09 * (np.abs(q).astype(F64) @ np.abs(ks[:p + 1]).max((0, 1)))
            assert (np.abs(o - ro) <= (vmax * (2.0 ** -15 * s1 + 2.0 ** -16 + 100 * 2.0 ** -24))[:, None]).all()

        base = int(np.concatenate([[0], np.cumsum(prompt)])[s])
        for i in range(prompt[s]):
            check(op0[base + i], q0[base + i], i)
        for i in range(steps):
            check(outs[i][s], qs[i][s], prompt[s] + i)


def test_two_chains_with_their_own_scratch(e4b, dev, scratch):
    """Calls on the main and the side stream at once, each with its scratch."""
    mine = dev.alloc(int(e4b.lib().e4b_paged_scratch_bytes()))
    rng = np.random.default_rng(4)
    cs = [Cache(e4b, dev, [2000 + i, 700], [1, 1], bits=4, page=64, KVH=2, HD=128, ragged=False, seed=i) for i in range(2)]
    held = [c.fill(rng) for c in cs]
    q = (rng.standard_normal((2, 8, 128)) * 0.2).astype(F32)
    bq = dev.upload(q)
    of = [dev.alloc(2 * 8 * 128 * 4) for _ in range(2)]
    for _ in range(5):
        dev.call("e4b_side_begin")
        e4b.ops.attn_paged(dev, cs[0].kv, bq, None, of[0], None, mine, Q_HEADS=8, ROWS=2)
        dev.call("e4b_side_end")
        e4b.ops.attn_paged(dev, cs[1].kv, bq, None, of[1], None, scratch, Q_HEADS=8, ROWS=2)
        dev.call("e4b_join")
    assert dev.status() == 0
    for c, h, b in zip(cs, held, of):
        o = dev.read(b, F32, 2 * 8 * 128).reshape(2, 8, 128)
        for r in range(2):
            ro, _ = op.attention(q[r], c.lens[r], *h[r], 0, 0, 1.0)
            assert np.abs(o[r] - ro).max() <= 8 * (2.0 ** -15 * 30 + 2.0 ** -12)


def test_calls_refuse_bad_arguments(e4b, dev, scratch):
    c = Cache(e4b, dev, [3, 4], [1, 1], bits=4, page=16, KVH=2, HD=64, ragged=False)
    x = dev.alloc(4096)
    for f in (lambda: e4b.ops.attn_paged(dev, c.kv, x, x, None, None, scratch, Q_HEADS=3, ROWS=2),
              lambda: e4b.ops.attn_paged(dev, c.kv, x, x, None, None, None, Q_HEADS=4, ROWS=2),
              lambda: e4b.ops.attn_paged(dev, c.kv, x, x, None, None, scratch, Q_HEADS=4, ROWS=3),
              lambda: e4b.ops.headprep_paged(dev, c.kv, x, None, x, x, QH=2, ROPE_ANGLES=32, THETA=1e4, ROWS=2),
              lambda: e4b.ops.kvread_paged(dev, c.kv, None, None, ROWS=2)):
        with pytest.raises(e4b.E4BError, match="_paged: "):
            f()
    e = Cache(e4b, dev, [3, 4], [0, 0], bits=4, page=16, KVH=2, HD=64, ragged=True)
    e4b.ops.attn_paged(dev, e.kv, x, x, None, None, scratch, Q_HEADS=4, ROWS=0)      # no rows: nothing to do
    e4b.ops.headprep_paged(dev, e.kv, x, x, x, x, QH=2, ROPE_ANGLES=32, THETA=1e4, ROWS=0)
    e4b.ops.attn_paged(dev, e.kv, x, x, None, None, scratch, Q_HEADS=4, ROWS=1)      # one row of padding
    dev.sync()
    assert dev.status() == 0
