"""Host checks of the paged KV cache: the layout and visibility arithmetic of
csrc/paged.h (compiled here with the C++ compiler) against the numpy oracle,
the descriptor's checks, and the 4-bit rule."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from oracle import paged as op

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "e4b-webgpu_b200", "csrc")

SHIM = r"""
#include "paged.h"
using namespace e4b;
extern "C" {
int quad(int bits, int HD, int value, int s, int q) {
  return bits == 16 ? (value ? v16_quad(s, q) : k16_quad(s, q)) : (value ? v4_quad(s, q, HD) : k4_quad(s, q, HD));
}
int scale(int HD, int value, int s, int b) { return value ? v4_scale(s, b, HD) : k4_scale(s, b, HD); }
uint64_t piece(uint64_t page, int h, int slot, int KVH, int ps, int bytes) { return piece_offset(page, h, slot, KVH, ps, bytes); }
int bytes(int bits, int HD) { return piece_bytes(bits, HD); }
int seen(uint32_t t, uint32_t p, uint32_t w, uint32_t n) { return slot_visible(t, p, w, n); }
uint32_t range(uint32_t p0, uint32_t p1, uint32_t w, uint32_t n, uint32_t* out) {
  PieceRange r = piece_range(p0, p1, w, n);
  for (uint32_t k = 0; k < r.count; k++) out[k] = r.at(k);
  return r.count;
}
uint32_t span(uint32_t q0, uint32_t q1, uint32_t k0, uint32_t k1, uint32_t p0, uint32_t p1, uint32_t w, uint32_t n, uint32_t* out) {
  PieceSpan s = piece_span(piece_range(q0, q1, w, n), k0, k1, p0, p1, w, n);
  for (uint32_t i = 0; i < s.count; i++) out[i] = s.at(i);
  return s.count;
}
const char* f_prep(const e4b_paged_kv* kv, const void* qkv, const float* qw, const float* kw, const float* q_out, int QH,
                   int angles, float theta, float eps, int norm, int keqv, int h, int stride, int parts, int n) {
  return headprep_paged_fault(kv, qkv, qw, kw, q_out, QH, angles, theta, eps, norm, keqv, h, stride, parts, n);
}
const char* f_read(const e4b_paged_kv* kv, const void* k, const void* v, int n) { return kvread_paged_fault(kv, k, v, n); }
const char* f_attn(const e4b_paged_kv* kv, const float* q, const uint16_t* oh, const float* of, const float* lse, const void* sc,
                   int QH, int w, int s, float scale, int xfo, int n) {
  return attn_paged_fault(kv, q, oh, of, lse, sc, QH, w, s, scale, xfo, n);
}
}
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cpp").write_text(SHIM)
    so = d / "shim.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-I", CSRC, "-I",
                    os.path.join(ROOT, "include"), str(d / "shim.cpp"), "-o", str(so)], check=True)
    L = ctypes.CDLL(str(so))
    for n in ("f_prep", "f_read", "f_attn"):
        getattr(L, n).restype = ctypes.c_char_p
    L.piece.restype = ctypes.c_uint64
    L.piece.argtypes = [ctypes.c_uint64] + [ctypes.c_int] * 5
    return L


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("value", [0, 1])
def test_layout_matches_the_documented_order_and_fills_the_piece(shim, HD, bits, value):
    at, shift = op.element_place(bits, HD, bool(value))
    pb = shim.bytes(bits, HD)
    assert pb == op.piece_bytes(bits, HD)
    used = np.zeros(pb * 2, int)          # half bytes
    for s in range(16):
        for d in range(HD):
            quad = shim.quad(bits, HD, value, s, d // 4)
            if bits == 16:
                assert quad + 2 * (d % 4) == at[s, d]
                used[at[s, d] * 2:at[s, d] * 2 + 4] += 1
            else:
                assert quad == at[s, d] and shift[s, d] == 4 * (d % 4)
                used[at[s, d] * 2 + shift[s, d] // 4] += 1
        if bits == 4:
            for b in range(HD // 32):
                assert shim.scale(HD, value, s, b) == op.scale_place(HD, bool(value))[s, b]
                used[shim.scale(HD, value, s, b) * 2:shim.scale(HD, value, s, b) * 2 + 4] += 1
    assert (used == 1).all()


def test_piece_offsets_are_64_bit_and_tile_the_pool(shim):
    KVH, page, pb = 3, 48, 9 * 128
    seen = {shim.piece(p, h, s, KVH, page, pb) for p in range(4) for h in range(KVH) for s in range(0, page, 16)}
    assert seen == {i * pb for i in range(4 * KVH * 3)}
    assert shim.piece(1 << 22, 7, 4095, 8, 4096, 8192) == (((1 << 22) * 8 + 7) * 256 + 255) * 8192


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 9), (1, 0), (1, 1), (16, 4), (17, 33), (40, 16), (40, 100), (5, 1000)])
def test_piece_range_covers_exactly_the_visible_slots(shim, window, sinks):
    out = (ctypes.c_uint32 * 64)()
    for p0 in list(range(0, 70)) + [200]:
        for n in (1, 2, 5, 37):
            p1 = p0 + n - 1
            see = np.zeros(p1 + 1, bool)
            for p in range(p0, p1 + 1):
                see |= op.visible(p1 + 1, p, window, sinks)
            cnt = shim.range(p0, p1, window, sinks, out)
            got = list(out[:cnt])
            assert got == sorted(set(got)) and got[-1] == p1 // 16
            want = sorted({t // 16 for t in np.flatnonzero(see)})
            assert set(want) <= set(got)
            if n == 1:
                assert want == got
    for t in range(0, 60):
        for p in range(0, 60):
            assert bool(shim.seen(t, p, window, sinks)) == bool(op.visible(64, p, window, sinks)[t])


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (17, 33), (40, 16), (40, 100), (5, 1000)])
def test_piece_span_cuts_a_group_of_rows_out_of_a_run(shim, window, sinks):
    """Cut anywhere, the parts of a group's pieces are each needed piece once, in order."""
    out, whole = (ctypes.c_uint32 * 64)(), (ctypes.c_uint32 * 64)()
    rng = np.random.default_rng(window + sinks)
    for q0 in (0, 3, 15, 16, 100, 331):
        for rows in (1, 7, 60):
            q1 = q0 + rows - 1
            n = shim.range(q0, q1, window, sinks, whole)
            for p0 in range(q0, q1 + 1, 11):
                p1 = min(q1, p0 + int(rng.integers(0, 20)))
                m = shim.range(p0, p1, window, sinks, out)
                want = list(out[:m])
                cuts = [0] + sorted(int(x) for x in rng.integers(0, n + 1, 3)) + [n]
                got = []
                for a, b in zip(cuts, cuts[1:]):
                    c = shim.span(q0, q1, a, b, p0, p1, window, sinks, out)
                    assert all(x in list(whole[a:b]) for x in out[:c])
                    got += list(out[:c])
                assert got == want


def test_visibility_at_the_far_end(shim):
    top = (1 << 31) - 2
    assert shim.seen(top, top, 1, 0) and not shim.seen(top - 1, top, 1, 0) and shim.seen(0, top, 1, 1)
    out = (ctypes.c_uint32 * 64)()
    n = shim.range(top, top, 20, 3, out)
    assert list(out[:n]) == [0, (top - 19) // 16, top // 16] or list(out[:n]) == [0, top // 16 - 1, top // 16]


# ------------------------------------------------------------------ refusals
GOOD = dict(k=1 << 20, v=1 << 21, pages=1 << 22, lens=1 << 23, rows=None, bits=4, page=64, n_pages=8, max_pages=4, nseq=2,
            kv_heads=2, head_dim=128)


def _kv(e4b, **over):
    from importlib import import_module
    S = import_module("e4b-webgpu_b200.paged").PagedStruct
    return S(**{**GOOD, **over})


def _prep(shim, kv, **o):
    a = dict(qkv=4096, qw=4096, kw=4096, q_out=4096, QH=4, angles=64, theta=1e4, eps=1e-6, norm=1, keqv=0, h=0, stride=0,
             parts=1, n=2)
    a.update(o)
    V, F = ctypes.c_void_p, ctypes.c_float
    return shim.f_prep(kv and ctypes.byref(kv), V(a["qkv"]), V(a["qw"]), V(a["kw"]), V(a["q_out"]), a["QH"], a["angles"],
                       F(a["theta"]), F(a["eps"]), a["norm"], a["keqv"], a["h"], a["stride"], a["parts"], a["n"])


def _attn(shim, kv, **o):
    a = dict(q=4096, oh=4096, of=None, lse=None, sc=4096, QH=8, w=0, s=0, scale=1.0, xfo=0, n=2)
    a.update(o)
    V = ctypes.c_void_p
    return shim.f_attn(kv and ctypes.byref(kv), V(a["q"]), V(a["oh"]), V(a["of"]), V(a["lse"]), V(a["sc"]), a["QH"], a["w"], a["s"],
                       ctypes.c_float(a["scale"]), a["xfo"], a["n"])


def test_usable_descriptors_pass(e4b, shim):
    for hd in (64, 128, 256):
        for bits in (4, 16):
            kv = _kv(e4b, head_dim=hd, bits=bits)
            assert _prep(shim, kv, angles=hd // 2) is None and _attn(shim, kv) is None
            assert shim.f_read(ctypes.byref(kv), ctypes.c_void_p(16), None, 2) is None
    kv = _kv(e4b, rows=4096)
    assert _prep(shim, kv, n=0) is None and _attn(shim, kv, n=77, window=5) is None


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(pages=None), dict(lens=None), dict(bits=8), dict(head_dim=96),
                                 dict(head_dim=512), dict(kv_heads=0), dict(kv_heads=1025), dict(page=0), dict(page=24),
                                 dict(page=4112), dict(n_pages=0), dict(max_pages=0), dict(nseq=0), dict(nseq=4097),
                                 dict(max_pages=1 << 26), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(lens=4098),
                                 dict(pages=4098), dict(rows=4098)])
def test_bad_descriptors_are_refused_by_every_call(e4b, shim, bad):
    kv = _kv(e4b, **bad)
    assert _prep(shim, kv) and _attn(shim, kv) and shim.f_read(ctypes.byref(kv), ctypes.c_void_p(16), None, 2)


def test_bad_arguments_are_refused(e4b, shim):
    kv, ragged = _kv(e4b), _kv(e4b, rows=4096)
    assert _prep(shim, None) and _attn(shim, None)
    for bad in (dict(qkv=None), dict(qkv=4100), dict(qkv=4100, h=1), dict(qw=None), dict(kw=None), dict(q_out=None), dict(QH=-1),
                dict(angles=65), dict(angles=-1), dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")),
                dict(eps=-1.0), dict(eps=float("nan")), dict(stride=8 * 128 - 4), dict(stride=8 * 128 + 2), dict(parts=0),
                dict(parts=2, h=1), dict(n=3), dict(n=1), dict(n=-1), dict(qw=4100), dict(q_out=4104)):
        assert _prep(shim, kv, **bad), bad
    assert _prep(shim, kv, qkv=4104, h=1) is None and _prep(shim, kv, qw=None, kw=None, norm=0) is None
    assert _prep(shim, kv, QH=0, qw=None, q_out=None) is None and _prep(shim, kv, stride=8 * 128) is None
    assert _prep(shim, kv, keqv=1, stride=6 * 128) is None
    for bad in (dict(q=None), dict(q=4100), dict(oh=None), dict(sc=None), dict(sc=4104), dict(QH=0), dict(QH=3), dict(QH=18),
                dict(w=-1), dict(s=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(n=1), dict(n=-2),
                dict(oh=None, of=4096, xfo=1), dict(oh=4104), dict(of=4100), dict(lse=4098)):
        assert _attn(shim, kv, **bad), bad
    assert _attn(shim, ragged, n=-1) and _attn(shim, ragged, n=0) is None
    for call in (_prep, _attn):
        assert call(shim, ragged, n=1 << 28) is None and call(shim, ragged, n=(1 << 28) + 1) and call(shim, ragged, n=(1 << 31) - 1)
    assert shim.f_read(ctypes.byref(kv), None, None, 2) and shim.f_read(ctypes.byref(kv), ctypes.c_void_p(8), None, 2)


def test_struct_layout_matches_header(e4b, tmp_path):
    from importlib import import_module
    S = import_module("e4b-webgpu_b200.paged").PagedStruct
    names = [f for f, _ in S._fields_]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "e4b_b200.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu\\n", offsetof(e4b_paged_kv, {n}));\n' for n in names) +
        '  printf("%zu\\n", sizeof(e4b_paged_kv));\n  return 0;\n}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(S, n).offset for n in names] + [ctypes.sizeof(S)]


def test_calls_reject_a_null_context_and_size_queries(e4b):
    L = e4b.lib()
    assert L.e4b_attn_paged(None, None, None, None, None, None, None, 8, 0, 0, 1.0, 0, 1) == -1
    assert L.e4b_headprep_paged(None, None, None, None, None, None, 1, 0, 1.0, 0.0, 1, 0, 0, 0, 1, 1) == -1
    assert L.e4b_kvread_paged(None, None, None, None, 0, 1) == -1 and L.e4b_paged_advance(None, None) == -1
    assert L.e4b_paged_pool_bytes(4, 64, 10, 4, 256) == 10 * 4 * 4 * 9 * 256
    assert L.e4b_paged_pool_bytes(16, 4096, 1 << 20, 8, 256) == (1 << 20) * 8 * 4096 * 512
    for bad in ((8, 64, 1, 1, 64), (4, 24, 1, 1, 64), (4, 64, 0, 1, 64), (4, 64, 1, 1, 96)):
        assert L.e4b_paged_pool_bytes(*bad) == 0
    assert 0 < L.e4b_paged_scratch_bytes() <= 64 << 20


def test_host_class_checks_its_tables(e4b):
    class Stub:
        def __init__(self):
            self.wrote = []

        def alloc(self, n, name=""):
            return type("B", (), {"ptr": 1 << 20, "nbytes": n})()

        def write(self, ptr, a):
            self.wrote.append((ptr, a.shape))

        def free(self, b):
            pass

    d = Stub()
    kw = dict(BITS=4, PAGE=16, PAGES=5, MAX_PAGES=3, SEQS=2, KV_HEADS=1, HEAD_DIM=64)
    kv = e4b.PagedKV(d, **kw)
    kv.set_tables(np.zeros((2, 3)), [1, 2], rows=64)
    assert len(d.wrote) == 2 and kv.struct.rows == 64
    kv.set_tables(rows=0)
    assert kv.struct.rows is None
    for bad in (dict(pages=np.zeros((3, 3))), dict(lens=[1])):
        with pytest.raises(ValueError):
            kv.set_tables(**bad)
    with pytest.raises(ValueError):
        e4b.PagedKV(d, **{**kw, "BITS": 5})
    kv.free()
    assert kv.owned == []


# ------------------------------------------------------------------ the 4-bit rule
def test_quantiser_rule():
    x = np.zeros(32, np.float16)
    assert (op.quantise(x)[0] == 8).all() and op.dequantise(*op.quantise(x)).any() == False  # noqa: E712
    x = np.linspace(-1, 1, 32).astype(np.float16)       # -1 and 1: the first of the two gives the sign
    q, d = op.quantise(x)
    assert d[0] == np.float16(0.125) and q[0] == 0 and q[-1] == 15
    x = np.zeros(32, np.float16)
    x[3], x[4], x[5] = -8.0, 0.5, 1.5                   # d = 1: exactly between two codes, upwards
    q, d = op.quantise(x)
    assert d[0] == 1.0 and (q[3], q[4], q[5]) == (0, 9, 10)
    x[7] = np.inf
    assert np.isnan(op.dequantise(*op.quantise(x))).all()
    rng = np.random.default_rng(0)
    y = rng.standard_normal((50, 64)).astype(np.float16)
    err = np.abs(op.dequantise(*op.quantise(y)) - y.astype(float)).reshape(50, 2, 32)
    # half a step, or a whole one at the code that the other sign's extreme lacks; f16's rounding of the scale
    step = np.abs(y.astype(float)).reshape(50, 2, 32).max(-1, keepdims=True) / 8
    assert (err <= step * (1 + 8 * 2.0 ** -11)).all()
