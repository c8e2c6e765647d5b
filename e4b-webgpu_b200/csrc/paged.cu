// Paged KV cache: head prep (per-head RMSNorm, RoPE) with the append of keys and
// values in f16 or 4 bits, reading rows back, and advancing the lengths.
#include "paged.cuh"

namespace {
using namespace e4b;

constexpr int kThreads = 256;

struct PrepP {
  PagedDev d;
  const void* qkv;
  const float* qw;
  const float* kw;
  float* q_out;
  int QH, angles, norm, keqv, x_f16, nparts;
  int64_t stride;                    // elements between rows
  float eps;
  double log2_theta;
};

struct Quad {
  float x[4];
};

E4B_DEV Quad load_quad(const PrepP& p, int64_t at) {
  Quad r;
  if (p.x_f16) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.qkv) + at);
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int j = 0; j < 4; j++) r.x[j] = h2f((uint16_t)(u[j >> 1] >> (16 * (j & 1))));
    return r;
  }
  const float* x = static_cast<const float*>(p.qkv) + at;
  float4 v = *reinterpret_cast<const float4*>(x);
  for (int k = 1; k < p.nparts; k++) {
    const float4 w = *reinterpret_cast<const float4*>(x + (int64_t)k * p.d.n_rows * p.stride);
    v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
  }
  r.x[0] = v.x, r.x[1] = v.y, r.x[2] = v.z, r.x[3] = v.w;
  return r;
}

// Four consecutive f16 values of a 32-dim block held by 8 neighbouring lanes ->
// their q4_0 codes; `d16` is the block's stored scale (the same in all 8 lanes).
// The quotient x / d is a correctly rounded division, so a value that lies
// exactly between two codes goes the same way in any precision.
E4B_DEV uint32_t quantise_quad(const uint16_t (&h)[4], int lane8, uint16_t& d16) {
  // order by magnitude, then by first index; the sign rides along
  uint32_t key = 0;
#pragma unroll
  for (int j = 0; j < 4; j++)
    key = max(key, ((uint32_t)(h[j] & 0x7fffu) << 6) | ((31u - (lane8 * 4 + j)) << 1) | (h[j] >> 15));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  const uint16_t top = (uint16_t)((key >> 6) | ((key & 1u) << 15));
  if ((key >> 6) >= 0x7c00u) {       // an infinity or NaN in the block
    d16 = 0x7fffu;
    return 0x8888u;
  }
  const float d = h2f(top) * -0.125f;
  d16 = f2h(d);
  if (d == 0.f) return 0x8888u;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float c = truncf(__fadd_rn(__fdiv_rn(h2f(h[j]), d), 8.5f));
    w |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * j);
  }
  return w;
}

// One CTA takes a row at a time; HD/8 lanes take a head, each lane dims 4l..4l+3
// and HD/2 + 4l..4l+3, so a rotation pair (p, p + HD/2) and a group of four codes
// sit in one lane and a 32-dim block in 8 neighbouring lanes.  Keys and values are
// formed in 64 bits: what is stored is then the rounding of the exact value
// whatever the order of the sums, so the 4-bit codes do not depend on it.  The
// rotation's angles are formed once per row for all its heads.
template <int HD>
__global__ void __launch_bounds__(kThreads) k_headprep_paged(const PrepP p, int bits) {
  pdl_wait();
  constexpr int LPH = HD / 8, HALF = HD / 2, NS = kThreads / LPH;
  __shared__ double2 turn[HALF];     // (cos, sin) of the row's angles
  const int tid = threadIdx.x, l = tid % LPH, sub = tid / LPH, lane8 = l & 7;
  const int KVH = p.d.KVH, heads = p.QH + 2 * KVH, pb = piece_bytes(bits, HD);
  const double freq = tid < p.angles ? exp2((-2.0 * tid / HD) * p.log2_theta) * 0.3183098861837906715 : 0.0;
  const uint32_t live = live_rows(p.d);
  for (uint32_t row = blockIdx.x; row < live; row += gridDim.x) {
    const int seq = seq_of_row(p.d, row);
    const uint64_t pos = (uint64_t)p.d.lens[seq] + (p.d.rows ? row - p.d.rows[seq] : 0u);
    __syncthreads();                 // the previous row's angles have been used
    if (tid < p.angles) {
      double s, c;
      sincospi((double)pos * freq, &s, &c);
      turn[tid] = make_double2(c, s);
    }
    __syncthreads();
    // every lane of a warp makes the same number of turns (the shuffles below)
    for (int h0 = blockIdx.y * NS; h0 < heads; h0 += gridDim.y * NS) {
      const int h = h0 + sub;
      const bool on = h < heads;
      const int hh = on ? h : 0;
      const int src = p.keqv && hh >= p.QH + KVH ? hh - KVH : hh;
      const int64_t at = (int64_t)row * p.stride + (int64_t)src * HD + 4 * l;
      const Quad a = load_quad(p, at), b = load_quad(p, at + HALF);
      const bool is_q = hh < p.QH, is_v = hh >= p.QH + KVH;
      const float* w = is_q ? p.qw : p.kw;
      double inv = 1.0;
      if (p.norm) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) s += (double)a.x[j] * a.x[j] + (double)b.x[j] * b.x[j];
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        inv = rsqrt(s / HD + (double)p.eps);
      }
      double xa[4], xb[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        xa[j] = (double)a.x[j] * inv;
        xb[j] = (double)b.x[j] * inv;
        if (p.norm && !is_v) {
          xa[j] *= (double)w[4 * l + j];
          xb[j] *= (double)w[HALF + 4 * l + j];
        }
        if (!is_v && 4 * l + j < p.angles) {
          const double2 cs = turn[4 * l + j];
          const double y = xa[j] * cs.x - xb[j] * cs.y;
          xb[j] = xa[j] * cs.y + xb[j] * cs.x;
          xa[j] = y;
        }
      }
      if (is_q) {
        if (on) {
          float* qo = p.q_out + ((size_t)row * p.QH + h) * HD + 4 * l;
          *reinterpret_cast<float4*>(qo) = make_float4((float)xa[0], (float)xa[1], (float)xa[2], (float)xa[3]);
          *reinterpret_cast<float4*>(qo + HALF) = make_float4((float)xb[0], (float)xb[1], (float)xb[2], (float)xb[3]);
        }
      }
      uint16_t ha[4], hb[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        ha[j] = f2h((float)xa[j]);
        hb[j] = f2h((float)xb[j]);
      }
      const int kvh = is_v ? hh - p.QH - KVH : hh - p.QH;
      uint16_t da = 0, db = 0;
      uint32_t ca = 0, cb = 0;
      if (bits == 4) {
        ca = quantise_quad(ha, lane8, da);
        cb = quantise_quad(hb, lane8, db);
      }
      uint32_t page;
      if (!on || is_q || !page_of(p.d, seq, pos, page)) continue;
      const int in_page = (int)((uint32_t)pos % (uint32_t)p.d.page), s = in_page % kPieceSlots;
      uint8_t* piece = (is_v ? p.d.v : p.d.k) + piece_offset(page, kvh, in_page, KVH, p.d.page, pb);
      const int qa = l, qb = l + LPH;
      if (bits == 16) {
        const uint2 wa = make_uint2(ha[0] | (uint32_t)ha[1] << 16, ha[2] | (uint32_t)ha[3] << 16);
        const uint2 wb = make_uint2(hb[0] | (uint32_t)hb[1] << 16, hb[2] | (uint32_t)hb[3] << 16);
        *reinterpret_cast<uint2*>(piece + (is_v ? v16_quad(s, qa) : k16_quad(s, qa))) = wa;
        *reinterpret_cast<uint2*>(piece + (is_v ? v16_quad(s, qb) : k16_quad(s, qb))) = wb;
      } else {
        *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_quad(s, qa, HD) : k4_quad(s, qa, HD))) = (uint16_t)ca;
        *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_quad(s, qb, HD) : k4_quad(s, qb, HD))) = (uint16_t)cb;
        if (lane8 == 0) {
          *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_scale(s, qa / 8, HD) : k4_scale(s, qa / 8, HD))) = da;
          *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_scale(s, qb / 8, HD) : k4_scale(s, qb / 8, HD))) = db;
        }
      }
    }
  }
}

// Rows back out of the pages: a CTA per row, a thread per four dims.
__global__ void __launch_bounds__(kThreads) k_kvread_paged(const PagedDev d, void* k_out, void* v_out, int bits, int HD,
                                                           int out_f32) {
  pdl_wait();
  const uint32_t live = live_rows(d);
  const int quads = HD / 4, per = d.KVH * quads, pb = piece_bytes(bits, HD);
  for (uint32_t row = blockIdx.x; row < live; row += gridDim.x) {
    const int seq = seq_of_row(d, row);
    const uint64_t pos = (uint64_t)d.lens[seq] + (d.rows ? row - d.rows[seq] : 0u);
    uint32_t page;
    const bool ok = page_of(d, seq, pos, page);
    const int in_page = (int)((uint32_t)pos % (uint32_t)d.page), s = in_page % kPieceSlots;
    for (int e = threadIdx.x; e < 2 * per; e += blockDim.x) {
      const bool is_v = e >= per;
      void* out = is_v ? v_out : k_out;
      if (!out) continue;
      const int r = is_v ? e - per : e, h = r / quads, q = r % quads;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (ok) {
        const uint8_t* piece = (is_v ? d.v : d.k) + piece_offset(page, h, in_page, d.KVH, d.page, pb);
        if (bits == 16) {
          const uint2 w = *reinterpret_cast<const uint2*>(piece + (is_v ? v16_quad(s, q) : k16_quad(s, q)));
          x[0] = h2f((uint16_t)w.x), x[1] = h2f((uint16_t)(w.x >> 16));
          x[2] = h2f((uint16_t)w.y), x[3] = h2f((uint16_t)(w.y >> 16));
        } else {
          const uint32_t w = *reinterpret_cast<const uint16_t*>(piece + (is_v ? v4_quad(s, q, HD) : k4_quad(s, q, HD)));
          const float sc = h2f(*reinterpret_cast<const uint16_t*>(
              piece + (is_v ? v4_scale(s, q / 8, HD) : k4_scale(s, q / 8, HD))));
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = sc * (float)((int)((w >> (4 * j)) & 15u) - 8);
        }
      }
      const size_t at = (size_t)row * d.KVH * HD + (size_t)h * HD + 4 * q;
      if (out_f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) =
            make_uint2(f2h(x[0]) | (uint32_t)f2h(x[1]) << 16, f2h(x[2]) | (uint32_t)f2h(x[3]) << 16);
      }
    }
  }
}

__global__ void k_paged_advance(uint32_t* lens, const uint32_t* __restrict__ rows, int nseq) {
  pdl_wait();
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s < nseq) lens[s] += rows ? rows[s + 1] - rows[s] : 1u;
}
}  // namespace

extern "C" {

E4B_API size_t e4b_paged_pool_bytes(int bits, int page, int n_pages, int kv_heads, int head_dim) {
  if ((bits != 16 && bits != 4) || page < 16 || page > 4096 || page % 16 || n_pages < 1 || kv_heads < 1 ||
      kv_heads > 1024 || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  return (size_t)n_pages * kv_heads * (page / kPieceSlots) * piece_bytes(bits, head_dim);
}

E4B_API int e4b_headprep_paged(e4b_ctx* c, const e4b_paged_kv* kv, const void* qkv, const float* qw, const float* kw,
                               float* q_out, int QH, int rope_angles, float theta, float eps, int norm, int keqv,
                               int x_f16, int row_stride, int nparts, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = headprep_paged_fault(kv, qkv, qw, kw, q_out, QH, rope_angles, theta, eps, norm, keqv, x_f16,
                                           row_stride, nparts, n_rows);
  E4B_REQUIRE(c, !fault, "headprep_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  const int HD = kv->head_dim, heads = QH + 2 * kv->kv_heads;
  PrepP p;
  p.d = paged_dev(c, kv, n_rows);
  p.qkv = qkv;
  p.qw = qw;
  p.kw = kw;
  p.q_out = q_out;
  p.QH = QH;
  p.angles = rope_angles;
  p.norm = norm ? 1 : 0;
  p.keqv = keqv ? 1 : 0;
  p.x_f16 = x_f16 ? 1 : 0;
  p.nparts = nparts;
  p.stride = row_stride ? row_stride : (int64_t)(QH + kv->kv_heads * (keqv ? 1 : 2)) * HD;
  p.eps = eps;
  p.log2_theta = log2((double)theta);
  // few rows: a CTA per pass over the row's heads, so one row spreads over several SMs
  const int passes = (heads * (HD / 8) + kThreads - 1) / kThreads;
  const int most = 8 * c->sm_count;
  const dim3 grid(n_rows < most ? n_rows : most, n_rows * passes <= most ? passes : 1);
  auto kern = HD == 256 ? k_headprep_paged<256> : (HD == 128 ? k_headprep_paged<128> : k_headprep_paged<64>);
  return e4b_launch(c, "headprep_paged", kern, grid, dim3(kThreads), 0, p, kv->bits);
}

E4B_API int e4b_kvread_paged(e4b_ctx* c, const e4b_paged_kv* kv, void* k_out, void* v_out, int out_f32, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = kvread_paged_fault(kv, k_out, v_out, n_rows);
  E4B_REQUIRE(c, !fault, "kvread_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  const int most = 16 * c->sm_count;
  return e4b_launch(c, "kvread_paged", k_kvread_paged, dim3(n_rows < most ? n_rows : most), dim3(kThreads), 0,
                    paged_dev(c, kv, n_rows), k_out, v_out, kv->bits, kv->head_dim, out_f32 ? 1 : 0);
}

E4B_API int e4b_paged_advance(e4b_ctx* c, const e4b_paged_kv* kv) {
  E4B_CHECK_CTX(c);
  const char* fault = paged_fault(kv);
  E4B_REQUIRE(c, !fault, "paged_advance: %s", fault);
  return e4b_launch(c, "paged_advance", k_paged_advance, dim3((kv->nseq + 127) / 128), dim3(128), 0,
                    const_cast<uint32_t*>(kv->lens), kv->rows, kv->nseq);
}

}  // extern "C"
