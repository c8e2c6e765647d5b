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
  int QH, angles, norm, keqv, nparts;
  int64_t stride;                    // elements between rows
  uint64_t per_q, per_kv;            // ceil(2^32 / QH), ceil(2^32 / (2 KVH))
  float eps;
  double log2_theta;
};

struct Quad {
  float x[4];
};

E4B_DEV uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Dims 4q..4q+3 of a head that begins at element `at` of the input rows.
template <bool XF16>
E4B_DEV Quad load_quad(const PrepP& p, int64_t at) {
  Quad r;
  if constexpr (XF16) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.qkv) + at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    r.x[0] = a.x, r.x[1] = a.y, r.x[2] = b.x, r.x[3] = b.y;
  } else {
    const float* x = static_cast<const float*>(p.qkv) + at;
    float4 v = *reinterpret_cast<const float4*>(x);
    for (int k = 1; k < p.nparts; k++) {
      const float4 w = *reinterpret_cast<const float4*>(x + (int64_t)k * p.d.n_rows * p.stride);
      v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    r.x[0] = v.x, r.x[1] = v.y, r.x[2] = v.z, r.x[3] = v.w;
  }
  return r;
}

// Four consecutive f16 values of a 32-dim block held by 8 neighbouring lanes ->
// their q4_0 codes trunc(x / d + 8.5); `d16` is the block's stored scale (the same in
// all 8 lanes).  x and 8 d are f16, so a quotient that is not exactly between two
// codes is at least 2^-13 away from there: with 2^-15 added, the product with 1 / d
// (off by less than 2^-18) gives the exact quotient's code, ties upwards.
E4B_DEV uint32_t quantise_quad(const uint32_t (&h2)[2], int lane8, uint16_t& d16) {
  // order by magnitude, then by first index; the sign rides along
  uint32_t key = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t h = j & 1 ? h2[j >> 1] >> 16 : h2[j >> 1] & 0xffffu;
    key = max(key, ((h & 0x7fffu) << 6) | ((31u - (lane8 * 4 + j)) << 1) | (h >> 15));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  const uint32_t mag = key >> 6;
  const float d = h2f((uint16_t)(mag | (key & 1u) << 15)) * -0.125f;
  d16 = f2h(d);
  if (mag >= 0x7c00u) d16 = 0x7fffu;                     // an infinity or NaN in the block
  if (mag >= 0x7c00u || mag == 0) return 0x8888u;
  const float inv = 1.f / d;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const __half2 h = *reinterpret_cast<const __half2*>(&h2[j >> 1]);
    const float x = j & 1 ? __high2float(h) : __low2float(h);
    const float c = fminf(fmaxf(fmaf(x, inv, 8.5f + 1.f / 32768.f), 0.f), 15.f);
    // adding 2^23 towards minus infinity leaves the integer part in the low bits
    w |= (__float_as_uint(__fadd_rd(c, 8388608.f)) & 15u) << (4 * j);
  }
  return w;
}

// Where a row goes: its sequence's position, and the page that holds it.
struct RowPlace {
  uint64_t pos;
  uint32_t page;
  int in_page, ok;                   // ok: the cache has a slot for it
};
E4B_DEV RowPlace place_row(const PagedDev& d, uint32_t row) {          // a warp
  const int seq = seq_of_row(d, row);
  RowPlace r;
  r.pos = (uint64_t)d.lens[seq] + (d.rows ? row - d.rows[seq] : 0u);
  r.in_page = (int)((uint32_t)r.pos % (uint32_t)d.page);
  r.ok = page_of(d, seq, r.pos, r.page);
  return r;
}

// A CTA takes RB rows at a time; HD/8 lanes take a head, each lane dims 4l..4l+3 and
// HD/2 + 4l..4l+3, so a rotation pair (p, p + HD/2) and a group of four codes sit in
// one lane and a 32-dim block in 8 neighbouring lanes.  The rotation's angles are
// formed once per row for all its heads, in 64 bits (a position of 10^6 times a
// frequency leaves f32 no fraction).  q is computed in f32.  Keys and values are
// formed in 64 bits: what is stored is then the rounding of the exact value whatever
// the order of the sums, so the 4-bit codes do not depend on it.
// Bound by memory: per row of 16 q + 2 x 4 heads of 256, 24.6 KB read, 16.4 KB of q and
// 2.3 KB (4 bits) of cache written.
template <int HD, int RB, int BITS, bool XF16>
__global__ void __launch_bounds__(kThreads) k_headprep_paged(const PrepP p) {
  constexpr int LPH = HD / 8, HALF = HD / 2, NS = kThreads / LPH;
  __shared__ double2 turn[RB][HALF];                     // (cos, sin) of the rows' angles
  __shared__ float2 turn32[RB][HALF];
  __shared__ double kw64[HD];
  __shared__ RowPlace place[RB];
  const int tid = threadIdx.x, warp = tid >> 5, l = tid % LPH, sub = tid / LPH, lane8 = l & 7;
  const int KVH = p.d.KVH;
  constexpr int pb = BITS == 16 ? 32 * HD : 9 * HD;
  // pair tid % HALF of the angles; 1/pi: sincospi reduces its argument exactly
  const int pair = tid % HALF;
  const double freq = pair < p.angles ? exp2((-2.0 * pair / HD) * p.log2_theta) * 0.3183098861837906715 : 0.0;
  float qw[8];
#pragma unroll
  for (int j = 0; j < 8; j++) qw[j] = 1.f;
  if (p.norm) {
    if (p.QH > 0) {
      const float4 a = *reinterpret_cast<const float4*>(p.qw + 4 * l), b = *reinterpret_cast<const float4*>(p.qw + HALF + 4 * l);
      qw[0] = a.x, qw[1] = a.y, qw[2] = a.z, qw[3] = a.w, qw[4] = b.x, qw[5] = b.y, qw[6] = b.z, qw[7] = b.w;
    }
    for (int i = tid; i < HD; i += kThreads) kw64[i] = (double)p.kw[i];
  }
  pdl_wait();
  const uint32_t live = live_rows(p.d);
  for (uint32_t row0 = blockIdx.x * RB; row0 < live; row0 += gridDim.x * RB) {
    const int rows = (int)min((uint32_t)RB, live - row0);
    __syncthreads();                 // the previous rows' angles and places have been used
    if (warp < rows) {
      const RowPlace r = place_row(p.d, row0 + warp);
      if ((tid & 31) == 0) place[warp] = r;
    }
    __syncthreads();
    for (int r = tid / HALF; r < rows; r += kThreads / HALF)
      if (pair < p.angles) {
        double s, c;
        sincospi((double)place[r].pos * freq, &s, &c);
        turn[r][pair] = make_double2(c, s);
        turn32[r][pair] = make_float2((float)c, (float)s);
      }
    __syncthreads();
    // every lane of a warp makes the same number of turns (the shuffles below)
    const int nq = rows * p.QH, nkv = rows * 2 * KVH, qpasses = (nq + NS - 1) / NS;
#pragma unroll 2
    for (int ps = blockIdx.y; ps < qpasses; ps += gridDim.y) {
      const int i0 = ps * NS;
      const int i = min(i0 + sub, nq - 1), r = RB == 1 ? 0 : (int)((i * p.per_q) >> 32), h = i - r * p.QH;
      const uint32_t row = row0 + r;
      const int64_t at = (int64_t)row * p.stride + (int64_t)h * HD + 4 * l;
      Quad a = load_quad<XF16>(p, at), b = load_quad<XF16>(p, at + HALF);
      if (p.norm) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) s = fmaf(a.x[j], a.x[j], fmaf(b.x[j], b.x[j], s));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float inv = rms_scale(s, HD, p.eps);
#pragma unroll
        for (int j = 0; j < 4; j++) a.x[j] *= inv * qw[j], b.x[j] *= inv * qw[4 + j];
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (4 * l + j < p.angles) {
          const float2 cs = turn32[r][4 * l + j];
          const float y = a.x[j] * cs.x - b.x[j] * cs.y;
          b.x[j] = a.x[j] * cs.y + b.x[j] * cs.x;
          a.x[j] = y;
        }
      if (i0 + sub < nq) {
        float* qo = p.q_out + ((size_t)row * p.QH + h) * HD + 4 * l;
        *reinterpret_cast<float4*>(qo) = make_float4(a.x[0], a.x[1], a.x[2], a.x[3]);
        *reinterpret_cast<float4*>(qo + HALF) = make_float4(b.x[0], b.x[1], b.x[2], b.x[3]);
      }
    }
    for (int i0 = (int)((blockIdx.y + gridDim.y - qpasses % gridDim.y) % gridDim.y) * NS; i0 < nkv; i0 += gridDim.y * NS) {
      const int i = min(i0 + sub, nkv - 1), r = RB == 1 ? 0 : (int)((i * p.per_kv) >> 32), h = i - r * 2 * KVH;
      const bool is_v = h >= KVH;
      const int kvh = is_v ? h - KVH : h;
      const uint32_t row = row0 + r;
      const int64_t at = (int64_t)row * p.stride + (int64_t)(p.QH + (p.keqv ? kvh : h)) * HD + 4 * l;
      const Quad a = load_quad<XF16>(p, at), b = load_quad<XF16>(p, at + HALF);
      double inv = 1.0;
      if (p.norm) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) s += (double)a.x[j] * a.x[j] + (double)b.x[j] * b.x[j];
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        inv = rsqrt(s / HD + (double)p.eps);
      }
      float fa[4], fb[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        double xa = (double)a.x[j] * inv, xb = (double)b.x[j] * inv;
        if (!is_v) {
          if (p.norm) xa *= kw64[4 * l + j], xb *= kw64[HALF + 4 * l + j];
          if (4 * l + j < p.angles) {
            const double2 cs = turn[r][4 * l + j];
            const double y = xa * cs.x - xb * cs.y;
            xb = xa * cs.y + xb * cs.x;
            xa = y;
          }
        }
        fa[j] = (float)xa;
        fb[j] = (float)xb;
      }
      const uint32_t ha[2] = {pack2(fa[0], fa[1]), pack2(fa[2], fa[3])}, hb[2] = {pack2(fb[0], fb[1]), pack2(fb[2], fb[3])};
      uint16_t da = 0, db = 0;
      uint32_t ca = 0, cb = 0;
      if constexpr (BITS == 4) {
        ca = quantise_quad(ha, lane8, da);
        cb = quantise_quad(hb, lane8, db);
      }
      const RowPlace pl = place[r];
      if (i0 + sub >= nkv || !pl.ok) continue;
      const int s = pl.in_page % kPieceSlots;
      uint8_t* piece = (is_v ? p.d.v : p.d.k) + piece_offset(pl.page, kvh, pl.in_page, KVH, p.d.page, pb);
      const int qa = l, qb = l + LPH;
      if constexpr (BITS == 16) {
        *reinterpret_cast<uint2*>(piece + (is_v ? v16_quad(s, qa) : k16_quad(s, qa))) = make_uint2(ha[0], ha[1]);
        *reinterpret_cast<uint2*>(piece + (is_v ? v16_quad(s, qb) : k16_quad(s, qb))) = make_uint2(hb[0], hb[1]);
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

// Rows back out of the pages: a warp per row (several where rows are few), a lane per
// 8 elements (two quads that the layouts keep in one 16-byte or 4-byte word).
template <int HD, int BITS>
__global__ void __launch_bounds__(128) k_kvread_paged(const PagedDev d, void* k_out, void* v_out, int out_f32) {
  pdl_wait();
  const uint32_t live = live_rows(d);
  const int per = d.KVH * HD / 8;
  constexpr int pb = BITS == 16 ? 32 * HD : 9 * HD;
  for (uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5); row < live; row += gridDim.x * 4) {
    const RowPlace pl = place_row(d, row);
    const int s = pl.in_page % kPieceSlots;
#pragma unroll 4
    for (int e = blockIdx.y * 32 + (threadIdx.x & 31); e < 2 * per; e += gridDim.y * 32) {
      const bool is_v = e >= per;
      void* out = is_v ? v_out : k_out;
      if (!out) continue;
      const int r = is_v ? e - per : e, h = r / (HD / 8), w = r % (HD / 8);
      // the word's two quads: dims 8w.. (f16, and 4-bit keys); the same quad of two blocks (4-bit values)
      const bool split = BITS == 4 && is_v;
      const int q0 = split ? (w >> 3) * 16 + (w & 7) : 2 * w, q1 = split ? q0 + 8 : 2 * w + 1;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = 0.f;
      if (pl.ok) {
        const uint8_t* piece = (is_v ? d.v : d.k) + piece_offset(pl.page, h, pl.in_page, d.KVH, d.page, pb);
        if constexpr (BITS == 16) {
          const uint4 v = *reinterpret_cast<const uint4*>(piece + (is_v ? v16_quad(s, q0) : k16_quad(s, q0)));
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = h2f((uint16_t)(u[j >> 1] >> (16 * (j & 1))));
        } else {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(piece + (is_v ? v4_quad(s, q0, HD) : k4_quad(s, q0, HD)));
          const uint16_t* d0 = reinterpret_cast<const uint16_t*>(piece + (is_v ? v4_scale(s, q0 / 8, HD) : k4_scale(s, q0 / 8, HD)));
          const uint16_t* d1 = reinterpret_cast<const uint16_t*>(piece + (is_v ? v4_scale(s, q1 / 8, HD) : k4_scale(s, q1 / 8, HD)));
          const float s0 = h2f(*d0), s1 = h2f(*d1);
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = (j < 4 ? s0 : s1) * (float)((int)((v >> (4 * j)) & 15u) - 8);
        }
      }
      const size_t at = (size_t)row * d.KVH * HD + (size_t)h * HD;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const size_t o = at + 4 * (k ? q1 : q0);
        const float* y = x + 4 * k;
        if (out_f32) *reinterpret_cast<float4*>(static_cast<float*>(out) + o) = make_float4(y[0], y[1], y[2], y[3]);
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) =
              make_uint2(f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, f2h(y[2]) | (uint32_t)f2h(y[3]) << 16);
      }
    }
  }
}

__global__ void k_paged_advance(uint32_t* lens, const uint32_t* __restrict__ rows, int nseq) {
  pdl_wait();
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s < nseq) lens[s] += rows ? rows[s + 1] - rows[s] : 1u;
}
template <int HD>
int launch_prep(e4b_ctx* c, const PrepP& p, int bits, int x_f16, bool few, dim3 grid) {
  auto kern = few ? (bits == 16 ? (x_f16 ? k_headprep_paged<HD, 1, 16, true> : k_headprep_paged<HD, 1, 16, false>)
                                : (x_f16 ? k_headprep_paged<HD, 1, 4, true> : k_headprep_paged<HD, 1, 4, false>))
                  : (bits == 16 ? (x_f16 ? k_headprep_paged<HD, 4, 16, true> : k_headprep_paged<HD, 4, 16, false>)
                                : (x_f16 ? k_headprep_paged<HD, 4, 4, true> : k_headprep_paged<HD, 4, 4, false>));
  return e4b_launch(c, "headprep_paged", kern, grid, dim3(kThreads), 0, p);
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
  const int HD = kv->head_dim;
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
  p.nparts = nparts;
  p.stride = row_stride ? row_stride : (int64_t)(QH + kv->kv_heads * (keqv ? 1 : 2)) * HD;
  p.per_q = QH > 0 ? (((uint64_t)1 << 32) + QH - 1) / QH : 0;
  p.per_kv = (((uint64_t)1 << 32) + 2 * kv->kv_heads - 1) / (2 * kv->kv_heads);
  p.eps = eps;
  p.log2_theta = log2((double)theta);
  // few rows: a row per CTA, and a CTA per pass over its heads, so that a row spreads
  // over several SMs (latency); many: four rows share the barriers and the lookups
  const int ns = kThreads / (HD / 8), passes = (QH + ns - 1) / ns + (2 * kv->kv_heads + ns - 1) / ns;
  const int most = 8 * c->sm_count;
  const bool few = (int64_t)n_rows * passes <= most;
  const int groups = (n_rows + 3) / 4;
  const dim3 grid = few ? dim3(n_rows, passes) : dim3(groups < most ? groups : most);
  return HD == 256 ? launch_prep<256>(c, p, kv->bits, x_f16, few, grid)
                   : (HD == 128 ? launch_prep<128>(c, p, kv->bits, x_f16, few, grid)
                                : launch_prep<64>(c, p, kv->bits, x_f16, few, grid));
}

E4B_API int e4b_kvread_paged(e4b_ctx* c, const e4b_paged_kv* kv, void* k_out, void* v_out, int out_f32, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = kvread_paged_fault(kv, k_out, v_out, n_rows);
  E4B_REQUIRE(c, !fault, "kvread_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  const int groups = (n_rows + 3) / 4, most = 16 * c->sm_count;
  const int slices = (2 * kv->kv_heads * kv->head_dim / 8 + 63) / 64;   // of two turns a warp
  const dim3 grid = groups * slices <= most ? dim3(groups, slices) : dim3(groups < most ? groups : most);
  const int HD = kv->head_dim;
  auto kern = kv->bits == 16 ? (HD == 256 ? k_kvread_paged<256, 16> : (HD == 128 ? k_kvread_paged<128, 16> : k_kvread_paged<64, 16>))
                             : (HD == 256 ? k_kvread_paged<256, 4> : (HD == 128 ? k_kvread_paged<128, 4> : k_kvread_paged<64, 4>));
  return e4b_launch(c, "kvread_paged", kern, grid, dim3(128), 0, paged_dev(c, kv, n_rows), k_out, v_out, out_f32 ? 1 : 0);
}

E4B_API int e4b_paged_advance(e4b_ctx* c, const e4b_paged_kv* kv) {
  E4B_CHECK_CTX(c);
  const char* fault = paged_fault(kv);
  E4B_REQUIRE(c, !fault, "paged_advance: %s", fault);
  return e4b_launch(c, "paged_advance", k_paged_advance, dim3((kv->nseq + 127) / 128), dim3(128), 0,
                    const_cast<uint32_t*>(kv->lens), kv->rows, kv->nseq);
}

}  // extern "C"
