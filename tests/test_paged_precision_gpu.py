"""Attention over the paged cache carries the lo parts of q, p and the scaled p: f32 outputs within the bounds of
paged_precision.py, in every form of the kernel."""
import numpy as np
import pytest
from paged_precision import F32, F64, score_bound, score_case, weight_bound, weight_case
from test_paged_edges_gpu import write
from test_paged_gpu import Cache, attend, scratch  # noqa: F401

pytestmark = pytest.mark.gpu
FORMS = {"a row each": (3, 1, 4), "many sequences": (200, 1, 3), "8 heads": (3, 1, 8), "rows": (2, 9, 4), "rows of one head": (2, 40, 1)}


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("large", [0.0, 2.0 ** 14])
def test_scores(e4b, dev, scratch, large, form, bits, HD):  # noqa: F811
    """Rows that see one slot (a window of 1 where there are several rows): lse is the score, o the value."""
    nseq, rows, QH = FORMS[form]
    c = Cache(e4b, dev, [0] * nseq, [rows] * nseq, bits=bits, page=16, KVH=1, HD=HD, ragged=rows > 1)
    q, x = score_case(HD, c.n, QH, large)
    k, v = write(c, [x.repeat(rows, 0)] * nseq)[0]
    assert np.array_equal(k[0], x[0, 0])
    _, of, lse = attend(c, scratch, q, QH, window=1 if rows > 1 else 0)
    assert dev.status() == 0
    s = q.astype(F64) @ k[0, 0]
    assert (np.abs(lse - s) <= score_bound(s)).all(), np.abs(lse - s).max()
    assert (np.abs(of - v[0, 0]) <= 2.0 ** -21).all()


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("form", FORMS)
def test_weights(e4b, dev, scratch, form, bits, HD):  # noqa: F811
    nseq, rows, QH = FORMS[form]
    rng = np.random.default_rng(HD + bits)
    lens = [int(n) for n in rng.integers(0, 16, nseq)] if rows == 1 else [int(n) for n in rng.integers(0, 7, nseq)]
    c = Cache(e4b, dev, lens, [min(rows, 9)] * nseq, bits=bits, page=16, KVH=1, HD=HD, ragged=rows > 1)
    cases = [weight_case(rng, HD, min(rows, 9), QH, n + min(rows, 9)) for n in lens]
    held = write(c, [x for _, x in cases])
    q = np.concatenate([a for a, _ in cases])
    _, of, lse = attend(c, scratch, q, QH)
    assert dev.status() == 0
    for r in range(c.n):
        i, p = c.place(r)
        k, v = (a[:p + 1, 0] for a in held[i])
        s = q[r].astype(F64) @ k.T
        e = np.exp(s - s.max(-1, keepdims=True))
        assert (np.abs(of[r] - e @ v / e.sum(-1, keepdims=True)) <= weight_bound(v)).all()
        # the reference score less 2^3 (2^-21), log2 of a sum known to 2^-20 (an ulp of 8..16: 2^-20), times log(2)
        assert (np.abs(lse[r] - (s.max(-1) + np.log(e.sum(-1)))) <= 2.0 ** -18).all()


@pytest.mark.parametrize("rows", [1, 6])
def test_small_values_of_an_f16_cache(e4b, dev, scratch, rows):  # noqa: F811
    """Values of 2^-20 are f16 subnormals: the outputs are as precise as if they were 2^-14."""
    rng = np.random.default_rng(2)
    c = Cache(e4b, dev, [9, 3], [rows] * 2, bits=16, page=16, KVH=1, HD=128, ragged=rows > 1)
    cases = [weight_case(rng, 128, rows, 4, n + rows) for n in c.lens]
    for _, x in cases:
        x[:, 1] *= 2.0 ** -20
    held = write(c, [x for _, x in cases])
    q = np.concatenate([a for a, _ in cases])
    of = attend(c, scratch, q, 4)[1]
    for r in range(c.n):
        i, p = c.place(r)
        k, v = (a[:p + 1, 0] for a in held[i])
        s = q[r].astype(F64) @ k.T
        e = np.exp(s - s.max(-1, keepdims=True))
        assert (np.abs(of[r] - e @ v / e.sum(-1, keepdims=True)) <= weight_bound(np.maximum(np.abs(v), 2.0 ** -14))).all()
