// Device side of the paged KV cache descriptor, shared by its kernels.
#pragma once

#include "common.cuh"
#include "paged.h"

namespace e4b {

struct PagedDev {
  uint8_t* k;
  uint8_t* v;
  const uint32_t* pages;
  const uint32_t* lens;
  const uint32_t* rows;
  uint32_t* status;
  int page, max_pages, nseq, KVH, n_rows;
  uint32_t n_pages, cap;             // cap: max_pages * page slots of a sequence
};

inline PagedDev paged_dev(const e4b_ctx* c, const e4b_paged_kv* kv, int n_rows) {
  PagedDev d;
  d.k = static_cast<uint8_t*>(kv->k);
  d.v = static_cast<uint8_t*>(kv->v);
  d.pages = kv->pages;
  d.lens = kv->lens;
  d.rows = kv->rows;
  d.status = c->status;
  d.page = kv->page;
  d.max_pages = kv->max_pages;
  d.nseq = kv->nseq;
  d.KVH = kv->kv_heads;
  d.n_rows = n_rows;
  d.n_pages = (uint32_t)kv->n_pages;
  d.cap = (uint32_t)kv->max_pages * (uint32_t)kv->page;
  return d;
}

// Rows of the call that belong to a sequence (rows past n_rows are refused).
E4B_DEV uint32_t live_rows(const PagedDev& p) {
  if (!p.rows) return (uint32_t)p.n_rows;
  const uint32_t n = p.rows[p.nseq];
  if (n > (uint32_t)p.n_rows) {
    if (threadIdx.x == 0) set_status(p.status, E4B_ST_BADINDEX);
    return (uint32_t)p.n_rows;
  }
  return n;
}

// Sequence of a live row, looked up by a warp (all 32 lanes call it): the number of
// sequences after the first that begin at or before the row.
E4B_DEV int seq_of_row(const PagedDev& p, uint32_t row) {
  if (!p.rows) return (int)row;
  int n = 0;
  for (int s0 = 1; s0 < p.nseq; s0 += 32) {
    const int s = s0 + (threadIdx.x & 31);
    n += __popc(__ballot_sync(0xffffffffu, s < p.nseq && p.rows[s] <= row));
  }
  return n;
}

// Page that holds `slot` of sequence `seq`; false (and the status bit) when the
// sequence cannot hold it or the table names no page.
E4B_DEV bool page_of(const PagedDev& p, int seq, uint64_t slot, uint32_t& page) {
  page = 0;
  if (slot < p.cap) page = p.pages[(size_t)seq * p.max_pages + (uint32_t)slot / (uint32_t)p.page];
  if (slot < p.cap && page < p.n_pages) return true;
  set_status(p.status, E4B_ST_BADINDEX);
  return false;
}

}  // namespace e4b
