"""The bounds of paged_precision.py against an oracle that loses lo parts: each loss breaks them, and the exact result
does not."""
import numpy as np
import pytest
from paged_precision import F32, F64, hi, score_bound, score_case, weight_bound, weight_case

from oracle import paged as op


def held(x, bits):
    x16 = x.astype(np.float16)
    return x16.astype(F64) if bits == 16 else op.dequantise(*op.quantise(x16))


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 16])
def test_scores_without_lo_parts_break_the_bound(HD, bits):
    q, x = score_case(HD, 5, 4)
    k = held(x, bits)[0, 0, 0]
    assert np.array_equal(k, x[0, 0, 0])
    q = q.astype(F64)
    s = q @ k
    partial = np.cumsum(q * k, -1) * 2.0 ** 14
    assert np.array_equal(partial, np.round(partial)) and partial.max() < 2.0 ** 24
    assert (np.abs(hi(q) @ k - s) > 100 * score_bound(s)).all()
    for b in range(HD // 32):                            # of one block alone
        one = q.copy()
        one[..., 32 * b:32 * b + 32] = hi(q)[..., 32 * b:32 * b + 32]
        assert (np.abs(one @ k - s) > 10 * score_bound(s)).all()


@pytest.mark.parametrize("HD", [64, 128, 256])
def test_uncentred_codes_break_the_bound(HD):
    """Codes 0..15 summed in f32 beside q of 2^14, the 8 taken off at the end; centred, every sum is exact."""
    q, x = score_case(HD, 5, 4, 2.0 ** 14)
    k = held(x, 4)[0, 0, 0]
    assert np.array_equal(k, x[0, 0, 0])
    s = q.astype(F64) @ k
    n = (k / -0.125 + 8).astype(F32)
    sums = np.cumsum((q * n).astype(F32), -1, dtype=F32)[..., -1] - 8 * np.cumsum(q, -1, dtype=F32)[..., -1]
    assert (np.abs(sums * F32(-0.125) - s) > 4 * score_bound(s)).all()
    assert np.array_equal(np.cumsum((q * (n - 8)).astype(F32), -1, dtype=F32)[..., -1] * F32(-0.125), s)


@pytest.mark.parametrize("slots", [2, 3, 7, 16])
@pytest.mark.parametrize("bits", [4, 16])
def test_weights_without_lo_parts_break_the_bound(bits, slots):
    q, x = weight_case(np.random.default_rng(slots), 64, 40, 4, slots)
    h = held(x, bits)
    k, v = h[:, 0, 0], h[:, 1, 0]
    assert np.array_equal(k, x[:, 0, 0])
    s = q.astype(F64) @ k.T
    assert np.array_equal(s * 1024, np.round(s * 1024)) and np.abs(s).max() < 4
    e = 256 * np.exp(s - s.max(-1, keepdims=True))
    total = e.sum(-1, keepdims=True)
    h16 = e.astype(np.float16).astype(F64)
    assert np.abs((h16 - e) @ v / total).max() > 2 * weight_bound(v)
    if bits == 4:                                        # the product with the scale rounded to one f16
        d = op.quantise(x[:, 1, 0].astype(np.float16))[1].astype(F64).repeat(32, -1).reshape(slots, 64)
        ed = (e[..., None] * d)
        assert np.abs(((ed.astype(np.float16).astype(F64) - ed) * (v / d)).sum(-2) / total).max() > 2 * weight_bound(v)
