// Paged KV cache: where a slot's elements sit in its page, which slots a query
// sees, and the checks of the cache descriptor.  Plain arithmetic without CUDA
// types, so the host tests compile it with the C++ compiler alone.
#pragma once

#include <stdint.h>

#include "e4b_b200.h"

#ifdef __CUDACC__
#define E4B_HD __host__ __device__ __forceinline__
#else
#define E4B_HD inline
#endif

namespace e4b {

constexpr int kPieceSlots = 16;      // slots in a piece: one m16 (keys) or k16 (values) operand tile
constexpr int kMaxSeqs = 4096;       // sequences of one paged cache
constexpr int kMaxRows = 1 << 28;    // rows of a call, padding included (row arithmetic stays in 32 bits)

// ---- layout.  A page holds its KV heads one after the other, a head's slots in
// pieces of 16.  Inside a piece the elements are in matrix-operand order, so a
// lane of m16n8k16 fetches its share with 16-byte loads that hit every bank once.
E4B_HD int piece_bytes(int bits, int HD) { return bits == 16 ? 32 * HD : 9 * HD; }
E4B_HD uint64_t piece_offset(uint64_t page, int head, int slot_in_page, int KVH, int page_slots, int bytes) {
  return ((page * KVH + head) * (uint64_t)(page_slots / kPieceSlots) + slot_in_page / kPieceSlots) * bytes;
}
// Byte of four consecutive elements (dims 4q..4q+3) of slot s (0..15) in an f16 piece.
E4B_HD int k16_quad(int s, int q) { return ((q >> 3) * 16 + s) * 64 + (q & 7) * 8; }
E4B_HD int v16_quad(int s, int q) {
  const int i = (s >> 3) * 2 + (s & 1), t = (s >> 1) & 3;
  return ((((q >> 4) * 4 + i) * 8 + ((q >> 1) & 7)) * 4 + t) * 16 + (q & 1) * 8;
}
// 4-bit piece: HD bytes of f16 block scales, then the codes.  Byte of the 16-bit
// word with the codes of dims 4q..4q+3 (lowest dim in the lowest bits).
E4B_HD int k4_quad(int s, int q, int HD) {
  const int b = q >> 3, nb = HD >= 128 ? 4 : HD / 32;
  return HD + ((((b / nb) * 16 + s) * 4 + ((q >> 1) & 3)) * nb + b % nb) * 4 + (q & 1) * 2;
}
E4B_HD int v4_quad(int s, int q, int HD) {
  const int i = (s >> 3) * 2 + (s & 1), t = (s >> 1) & 3;
  return HD + (((i * 8 + (q & 7)) * 4 + t) * (HD / 32) + (q >> 3)) * 2;
}
// Byte of the scale of block b (dims 32b..32b+31) of slot s.
E4B_HD int k4_scale(int s, int b, int HD) { return (s * (HD / 32) + b) * 2; }
E4B_HD int v4_scale(int s, int b, int HD) {
  return ((((s >> 1) & 3) * (HD / 32) + b) * 2 + (s >> 3)) * 4 + (s & 1) * 2;
}

// ---- visibility.  A query at position p sees slot t when t <= p and, with a
// window, t > p - window or t < sinks.
E4B_HD bool slot_visible(uint32_t t, uint32_t p, uint32_t window, uint32_t sinks) {
  return t <= p && (window == 0 || p - t < window || t < sinks);
}

// The pieces that hold slots visible to the queries at positions p0..p1: pieces
// 0..head-1 (the sinks) and then `tail`.., count in all (p1 < capacity).
struct PieceRange {
  uint32_t head, tail, count;
  E4B_HD uint32_t at(uint32_t k) const { return k < head ? k : tail + (k - head); }
};
E4B_HD PieceRange piece_range(uint32_t p0, uint32_t p1, uint32_t window, uint32_t sinks) {
  PieceRange r;
  const uint32_t last = p1 / kPieceSlots;
  const uint32_t from = (window == 0 || p0 < window) ? 0u : (p0 - window + 1) / kPieceSlots;
  const uint32_t sink_pieces = sinks == 0 ? 0u : (sinks - 1) / kPieceSlots + 1;
  r.head = sink_pieces < from ? sink_pieces : from;
  r.tail = from;
  r.count = r.head + (last - from + 1);
  return r;
}

// Of the pieces r.at(k0) .. r.at(k1 - 1), those that the queries at positions p0..p1
// need, p0 and p1 among the positions that r was made for: `count` of them, the
// i-th at at(i).
struct PieceSpan {
  uint32_t head, tail, first, count;
  E4B_HD uint32_t at(uint32_t i) const {
    const uint32_t n = first + i;
    return n < head ? n : tail + (n - head);
  }
};
E4B_HD PieceSpan piece_span(const PieceRange& r, uint32_t k0, uint32_t k1, uint32_t p0, uint32_t p1, uint32_t window,
                            uint32_t sinks) {
  const PieceRange u = piece_range(p0, p1, window, sinks);
  PieceSpan s;
  s.head = u.head;
  s.tail = u.tail;
  s.first = s.count = 0;
  if (k0 >= k1) return s;
  const uint32_t lo = r.at(k0), hi = r.at(k1 - 1) + 1;   // pieces lo <= p < hi
  const uint32_t a = lo < u.head ? lo : (lo <= u.tail ? u.head : u.head + (lo - u.tail));
  const uint32_t b = hi < u.head ? hi : (hi <= u.tail ? u.head : u.head + (hi - u.tail));
  s.first = a;
  s.count = (b < u.count ? b : u.count) > a ? (b < u.count ? b : u.count) - a : 0;
  return s;
}

// ---- checks of the descriptor; a message, or NULL when it is usable.
inline const char* paged_fault(const e4b_paged_kv* kv) {
  if (!kv) return "null cache descriptor";
  if (!kv->k || !kv->v || !kv->pages || !kv->lens) return "null pool, page table or lengths";
  if (kv->bits != 16 && kv->bits != 4) return "bits must be 16 or 4";
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return "head_dim must be 64, 128 or 256";
  if (kv->kv_heads < 1 || kv->kv_heads > 1024) return "kv_heads must be 1..1024";
  if (kv->page < 16 || kv->page > 4096 || kv->page % 16 != 0) return "page must be a multiple of 16 slots, 16..4096";
  if (kv->n_pages < 1 || kv->max_pages < 1) return "n_pages and max_pages must be positive";
  if (kv->nseq < 1 || kv->nseq > kMaxSeqs) return "nseq must be 1..4096";
  if ((int64_t)kv->max_pages * kv->page >= ((int64_t)1 << 31)) return "max_pages * page must be below 2^31 slots";
  if (((uintptr_t)kv->k | (uintptr_t)kv->v) % 16 != 0) return "pools must be 16-byte aligned";
  if (((uintptr_t)kv->pages | (uintptr_t)kv->lens | (uintptr_t)kv->rows) % 4 != 0) return "tables must be 4-byte aligned";
  return nullptr;
}
// Rows of the call: with no `rows` table, row s is sequence s's one row.
inline const char* paged_rows_fault(const e4b_paged_kv* kv, int n_rows) {
  if (n_rows < 0 || n_rows > kMaxRows) return "n_rows must be 0..2^28";
  if (!kv->rows && n_rows != kv->nseq) return "without a rows table the call has one row per sequence";
  return nullptr;
}
inline const char* headprep_paged_fault(const e4b_paged_kv* kv, const void* qkv, const float* qw, const float* kw,
                                        const float* q_out, int QH, int rope_angles, float theta, float eps, int norm,
                                        int keqv, int x_f16, int row_stride, int nparts, int n_rows) {
  if (const char* m = paged_fault(kv)) return m;
  if (const char* m = paged_rows_fault(kv, n_rows)) return m;
  if (!qkv) return "null qkv";
  if (QH < 0 || QH > 4096 || (QH > 0 && !q_out)) return "QH must be 0..4096, and q_out is needed for query heads";
  if (norm && (!kw || (QH > 0 && !qw))) return "norm weights are missing";
  if (rope_angles < 0 || rope_angles > kv->head_dim / 2) return "rope_angles must be 0..head_dim/2";
  if (!(theta > 0.f) || theta > 3e38f) return "theta must be positive and finite";
  if (!(eps >= 0.f)) return "eps must not be negative";
  const int64_t width = (int64_t)(QH + kv->kv_heads * (keqv ? 1 : 2)) * kv->head_dim;
  if (row_stride != 0 && (row_stride < width || row_stride % 4 != 0))
    return "row_stride must be 0 or a multiple of 4 not below the row's width";
  if (nparts < 1 || nparts > 64 || (nparts > 1 && x_f16)) return "nparts must be 1..64, and 1 for f16 rows";
  if ((uintptr_t)qkv % (x_f16 ? 8 : 16) != 0) return "qkv must be 16-byte aligned (f16: 8)";
  if (((uintptr_t)qw | (uintptr_t)kw | (uintptr_t)q_out) % 16 != 0) return "norm weights and q_out must be 16-byte aligned";
  return nullptr;
}
inline const char* kvread_paged_fault(const e4b_paged_kv* kv, const void* k_out, const void* v_out, int n_rows) {
  if (const char* m = paged_fault(kv)) return m;
  if (const char* m = paged_rows_fault(kv, n_rows)) return m;
  if (!k_out && !v_out) return "no output";
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16 != 0) return "outputs must be 16-byte aligned";
  return nullptr;
}
inline const char* attn_paged_fault(const e4b_paged_kv* kv, const float* q, const uint16_t* out_h, const float* out_f,
                                    const float* lse, const void* scratch, int QH, int window, int sinks, float scale, int xfo,
                                    int n_rows) {
  if (const char* m = paged_fault(kv)) return m;
  if (const char* m = paged_rows_fault(kv, n_rows)) return m;
  if (!q || (!out_h && !out_f) || !scratch) return "null q, output or scratch";
  if (QH < 1 || QH % kv->kv_heads != 0 || QH / kv->kv_heads > 8) return "1..8 query heads per KV head";
  if (window < 0 || sinks < 0) return "negative window or sinks";
  if (!(scale == scale) || scale > 3e38f || scale < -3e38f) return "scale must be finite";
  if (xfo && !out_h) return "fragment order is an order of out_h";
  if (((uintptr_t)q | (uintptr_t)scratch) % 16 != 0 || ((uintptr_t)out_h | (uintptr_t)out_f) % 16 != 0 ||
      (uintptr_t)lse % 4 != 0)
    return "q, outputs and scratch must be 16-byte aligned (lse: 4)";
  return nullptr;
}

}  // namespace e4b
