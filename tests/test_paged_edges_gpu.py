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
