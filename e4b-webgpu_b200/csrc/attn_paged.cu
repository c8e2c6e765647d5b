// Attention of ragged rows over the paged KV cache.
#include "paged.cuh"

namespace {
using namespace e4b;

constexpr int kThreads = 256;

struct AttnP {
  PagedDev d;
  const float* q;
  uint16_t* out_h;
  float* out_f;
  float* lse;
  int QH, bits, HD, xfo;
  uint32_t window, sinks;
  float scale;
};

E4B_DEV float element(const uint8_t* piece, int bits, int HD, int s, int dim, bool value) {
  const int q = dim >> 2, j = dim & 3;
  if (bits == 16)
    return h2f(*reinterpret_cast<const uint16_t*>(piece + (value ? v16_quad(s, q) : k16_quad(s, q)) + 2 * j));
  const uint32_t w = *reinterpret_cast<const uint16_t*>(piece + (value ? v4_quad(s, q, HD) : k4_quad(s, q, HD)));
  return h2f(*reinterpret_cast<const uint16_t*>(piece + (value ? v4_scale(s, q / 8, HD) : k4_scale(s, q / 8, HD)))) *
         (float)((int)((w >> (4 * j)) & 15u) - 8);
}

// A CTA per (row, query head): tiles of 256 slots, one slot's score per thread,
// then one dim's sum per thread, with a running maximum and sum.
__global__ void __launch_bounds__(kThreads) k_attn_paged(const AttnP p) {
  pdl_wait();
  __shared__ float qs[256], ps[kThreads], sh[32];
  __shared__ const uint8_t* vp[kThreads / kPieceSlots];
  const uint32_t row = blockIdx.x;
  const int h = blockIdx.y, kvh = h / (p.QH / p.d.KVH), tid = threadIdx.x, HD = p.HD, pb = piece_bytes(p.bits, HD);
  if (row >= live_rows(p.d)) return;
  const int seq = seq_of_row(p.d, row);
  const uint64_t pos64 = (uint64_t)p.d.lens[seq] + (p.d.rows ? row - p.d.rows[seq] : 0u);
  const uint32_t pos = pos64 > 0xfffffff0u ? 0xfffffff0u : (uint32_t)pos64;
  const uint32_t from = (p.window == 0 || pos < p.window) ? 0u : pos - p.window + 1;
  if (tid < HD) qs[tid] = p.q[((size_t)row * p.QH + h) * HD + tid];
  float m = -INFINITY, l = 0.f, acc = 0.f;
  if (pos64 >= p.d.cap && tid == 0) set_status(p.d.status, E4B_ST_BADINDEX);
  const uint32_t end = pos < p.d.cap ? pos + 1 : p.d.cap;
  for (uint32_t t0 = 0; t0 < end; t0 += kThreads) {
    if (t0 >= p.sinks && t0 + kThreads <= from) {
      t0 = from / kThreads * kThreads - kThreads;  // nothing visible up to the window
      continue;
    }
    const uint32_t t = t0 + tid;
    __syncthreads();
    const uint8_t* kp = nullptr;
    if (t < end && slot_visible(t, pos, p.window, p.sinks)) {
      uint32_t page;
      if (page_of(p.d, seq, t, page)) kp = p.d.k + piece_offset(page, kvh, (int)(t % p.d.page), p.d.KVH, p.d.page, pb);
    }
    float s = -INFINITY;
    if (tid % kPieceSlots == 0) vp[tid / kPieceSlots] = nullptr;
    __syncwarp();
    if (kp) {
      float dot = 0.f;
      for (int d = 0; d < HD; d++) dot = fmaf(qs[d], element(kp, p.bits, HD, t % kPieceSlots, d, false), dot);
      s = dot * p.scale;
      vp[tid / kPieceSlots] = p.d.v + (kp - p.d.k);
    }
    const float mt = fmaxf(m, block_max(s, sh));
    const float pt = kp ? expf(s - mt) : 0.f;
    ps[tid] = kp ? pt : -1.f;
    const float fix = m == -INFINITY ? 0.f : expf(m - mt);
    l = l * fix + block_sum(pt, sh);
    acc *= fix;
    m = mt;
    __syncthreads();
    if (tid < HD)
      for (int i = 0; i < kThreads; i++)
        if (ps[i] >= 0.f) acc = fmaf(ps[i], element(vp[i / kPieceSlots], p.bits, HD, i % kPieceSlots, tid, true), acc);
  }
  const size_t o = ((size_t)row * p.QH + h) * HD;
  if (tid < HD) {
    const float v = l != 0.f ? acc / l : 0.f;     // a NaN sum stays one
    if (p.out_f) p.out_f[o + tid] = v;
    if (p.out_h) p.out_h[p.xfo ? (size_t)row * p.QH * HD + xfo_pos(h * HD + tid) : o + tid] = f2h(v);
  }
  if (p.lse && tid == 0) p.lse[(size_t)row * p.QH + h] = l != 0.f ? m + logf(l) : -INFINITY;
}
}  // namespace

extern "C" {

E4B_API size_t e4b_paged_scratch_bytes(void) { return (size_t)4 << 20; }

E4B_API int e4b_attn_paged(e4b_ctx* c, const e4b_paged_kv* kv, const float* q, uint16_t* out_h, float* out_f,
                           float* lse, void* scratch, int QH, int window, int sinks, float scale, int xfo, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = attn_paged_fault(kv, q, out_h, out_f, scratch, QH, window, sinks, scale, xfo, n_rows);
  E4B_REQUIRE(c, !fault, "attn_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  AttnP p;
  p.d = paged_dev(c, kv, n_rows);
  p.q = q;
  p.out_h = out_h;
  p.out_f = out_f;
  p.lse = lse;
  p.QH = QH;
  p.bits = kv->bits;
  p.HD = kv->head_dim;
  p.xfo = xfo ? 1 : 0;
  p.window = (uint32_t)window;
  p.sinks = (uint32_t)sinks;
  p.scale = scale;
  return e4b_launch(c, "attn_paged", k_attn_paged, dim3(n_rows, QH), dim3(kThreads), 0, p);
}

}  // extern "C"
