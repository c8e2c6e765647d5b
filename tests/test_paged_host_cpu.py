"""PagedKV's own buffers: after free(), a failed allocation, and buffers that are too small."""
import ctypes

import numpy as np
import pytest

SIZES = dict(BITS=4, PAGE=16, PAGES=5, MAX_PAGES=3, SEQS=2, KV_HEADS=1, HEAD_DIM=64)


class FakeDevice:
    def __init__(self, fail_at=99):
        self.live, self.n, self.fail_at, self.wrote = set(), 0, fail_at, 0

    def alloc(self, nbytes, name=""):
        self.n += 1
        if self.n == self.fail_at:
            raise RuntimeError("out of memory")
        b = type("B", (), {"ptr": self.n << 20, "nbytes": nbytes})()
        self.live.add(b)
        return b

    def free(self, b):
        self.live.remove(b)

    def write(self, ptr, a):
        self.wrote += 1


def test_a_freed_cache_names_no_memory(e4b):
    """Every call checks the descriptor for null pools before it launches anything."""
    d = FakeDevice()
    kv = e4b.PagedKV(d, **SIZES)
    assert kv.struct.k == 1 << 20 and kv.struct.lens == 4 << 20 and len(d.live) == 4
    kv.free()
    assert not d.live and kv.owned == []
    assert [getattr(kv.struct, f) for f in ("k", "v", "pages", "lens")] == [None] * 4
    kv.free()                                            # twice: nothing more
    with pytest.raises(ValueError):
        kv.set_tables(lens=[1, 2])
    assert d.wrote == 0


def test_free_leaves_the_callers_buffers(e4b):
    d = FakeDevice()
    kv = e4b.PagedKV(d, **SIZES, k=1 << 30, lens=1 << 31)
    kv.free()
    assert (kv.struct.k, kv.struct.v, kv.struct.pages, kv.struct.lens) == (1 << 30, None, None, 1 << 31)


@pytest.mark.parametrize("at", [1, 2, 3, 4])
def test_a_failed_allocation_leaves_none_behind(e4b, at):
    d = FakeDevice(fail_at=at)
    with pytest.raises(RuntimeError, match="memory"):
        e4b.PagedKV(d, **SIZES)
    assert not d.live


@pytest.mark.parametrize("field", ["k", "v", "pages", "lens"])
def test_small_buffers_are_refused(e4b, field):
    d = FakeDevice()
    pool = int(e4b.lib().e4b_paged_pool_bytes(4, 16, 5, 1, 64))
    need = {"k": pool, "v": pool, "pages": 24, "lens": 8}[field]
    with pytest.raises(ValueError, match="needs"):
        e4b.PagedKV(d, **SIZES, **{field: e4b.Buffer(None, 1 << 20, need - 4)})
    assert not d.live
    kv = e4b.PagedKV(d, **SIZES, **{field: e4b.Buffer(None, 1 << 20, need)})
    assert getattr(kv.struct, field) == 1 << 20 and kv.ref == ctypes.addressof(kv.struct)
    kv.set_tables(np.zeros((2, 3)), [0, 0])
