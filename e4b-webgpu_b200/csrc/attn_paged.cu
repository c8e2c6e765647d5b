// Attention of ragged rows over the paged KV cache (f16 or 4-bit pages), with an
// optional sliding window and sinks: split-KV on the tensor cores.
//
// Unit = (sequence, group of query rows, KV head).  A unit's work is the pieces
// of 16 slots that its sequence's rows can see; the pieces of all units, one
// after the other, are cut into equal runs, one per CTA, so ragged lengths and
// few long sequences alike fill the machine.  A CTA's warps take a run's pieces
// in turn; each warp streams its own (one bulk copy for the keys, one for the
// values, through a ring of its own) and keeps its own softmax state, so the
// main loop has no CTA barrier.  At a unit's end the warps' states are merged in
// shared memory; a unit cut between CTAs leaves partials in the scratch, which
// the last CTA to arrive merges in CTA order (the same bits every time).
//
// Products, per piece and 8 MMA columns (m16n8k16, f32 accumulators):
//   S[slot][col]  = K[slot][:] . q[:][col]      A = keys,   B = q
//   O[dim][col]  += V[slot][dim] p[slot][col]   A = values, B = p
// The 8 columns are 4 query heads as f16 hi and lo parts (columns 0-3, 4-7), so
// q and p carry f32 precision at the MMA cost of one f16 pass.
// 4 bits: A holds the codes n as f16 subnormals, n * 2^-24 (a code in the low
// bits of a half) or 16 n * 2^-24 (one place up; q is divided by 16 there, the
// value's sum at the end), so decoding is one AND per pair.  The -8 enters as the
// accumulator's start (keys: -8 sum q per block) and as an MMA with a constant A
// (values).  A key block's scale multiplies its block's dot product in f32; a
// value block's scale multiplies p, again as hi + lo.
#include "paged.cuh"
#include "stream.cuh"

namespace {
using namespace e4b;

constexpr int kMaxCtas = 256;
constexpr int kCols = 8;             // query heads of a unit at most (2 n-tiles of 4)
constexpr uint32_t kLowCodes = 0x000F000Fu, kHighCodes = 0x00F000F0u;
constexpr uint32_t kMinus8Low = 0x80088008u, kMinus8High = 0x80808080u;  // -8 * 2^-24, -8 * 16 * 2^-24
constexpr float kTwo24 = 16777216.f, kTwo20 = 1048576.f;

struct AttnP {
  PagedDev d;
  const float* q;
  uint16_t* out_h;
  float* out_f;
  float* lse;
  uint32_t* arrived;                 // [kMaxCtas], zero at rest
  float* parts;                      // [2 * CTAs][kCols][HD + 2]
  int QH, G, per_unit, xfo;          // per_unit: query rows of a unit
  uint32_t window, sinks;
  float scale;
};

constexpr size_t kPartFloats = (size_t)kCols * (256 + 2);

template <int BITS, int HD, int NT>
struct Shape {
  static constexpr int NB = HD / 32;
  static constexpr int PB = BITS == 16 ? 32 * HD : 9 * HD;
  static constexpr int STAGE = 2 * PB;
  // warps and ring depth: about 150-200 KB in flight per SM
  static constexpr int W = BITS == 16 && HD == 256 ? 4 : 8;
  static constexpr int ST = BITS == 16 ? (HD == 64 ? 5 : (NT == 2 ? 2 : 3)) : (HD == 256 ? (NT == 2 ? 3 : 4) : 8);
  static constexpr int THREADS = 32 * W;
  static constexpr size_t RING = (size_t)W * ST * STAGE;
  static constexpr size_t MERGE = (size_t)W * NT * 4 * HD * 4;
  static constexpr size_t QFRAG = (size_t)NT * NB * 32 * 16;
  static constexpr size_t SMEM = RING + MERGE + QFRAG + 128;
};

// One sequence's rows of the call and the pieces they see.
struct SeqWork {
  uint32_t p0, nq;                   // first row's position, rows
  uint32_t groups, np;
  PieceRange range;
};
E4B_DEV SeqWork seq_work(const AttnP& p, int s) {
  SeqWork w;
  uint32_t r0 = (uint32_t)s, r1 = r0 + 1;
  if (p.d.rows) r0 = p.d.rows[s], r1 = min(p.d.rows[s + 1], (uint32_t)p.d.n_rows);
  w.nq = r1 > r0 ? r1 - r0 : 0u;
  // positions past the table are clamped: such slots are never visible (cap)
  const uint64_t last = (uint64_t)p.d.lens[s] + w.nq;
  w.p0 = min(p.d.lens[s], 0xfffffff0u - w.nq);
  w.groups = (w.nq + p.per_unit - 1) / p.per_unit;
  w.np = 0;
  if (w.nq) {
    if (last > p.d.cap && threadIdx.x == 0) set_status(p.d.status, E4B_ST_BADINDEX);
    const uint32_t p1 = min(w.p0 + w.nq - 1, p.d.cap - 1);
    w.range = piece_range(min(w.p0, p1), p1, p.window, p.sinks);
    w.np = w.range.count;
  }
  return w;
}

// Walks a CTA's run [g, end) of pieces, unit by unit.
struct Walk {
  uint64_t g, end, base;             // base: first piece of the current sequence
  int s;
  SeqWork w;
  uint32_t kvh, group, k0, k1;       // current segment: pieces k0..k1-1 of the unit
  uint64_t unit0;                    // first piece of the unit
  uint32_t pmin, pmax;               // positions of the unit's rows
  E4B_DEV bool next(const AttnP& p) {
    if (g >= end) return false;
    const uint32_t KVH = p.d.KVH;
    uint64_t total = (uint64_t)w.np * w.groups * KVH;
    while (g >= base + total) {
      base += total;
      if (++s >= p.d.nseq) {         // the lengths changed under the call
        g = end;
        return false;
      }
      w = seq_work(p, s);
      total = (uint64_t)w.np * w.groups * KVH;
    }
    const uint64_t unit = (g - base) / w.np;
    unit0 = base + unit * w.np;
    k0 = (uint32_t)(g - unit0);
    k1 = (uint32_t)min((uint64_t)w.np, k0 + (end - g));
    kvh = (uint32_t)(unit % KVH);
    group = (uint32_t)(unit / KVH);
    pmin = w.p0 + group * p.per_unit;
    pmax = min(pmin + p.per_unit, w.p0 + w.nq) - 1;
    g += k1 - k0;
    return true;
  }
  // Does a row of the unit see a slot of the piece?
  E4B_DEV bool needs(const AttnP& p, uint32_t piece) const {
    const uint32_t t0 = piece * kPieceSlots;
    return t0 <= pmax && (p.window == 0 || t0 < p.sinks || pmin < p.window || t0 + kPieceSlots - 1 > pmin - p.window);
  }
};

E4B_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
E4B_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
E4B_DEV uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
E4B_DEV uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
E4B_DEV uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
template <int WORDS>
E4B_DEV void lds_words(uint32_t (&w)[WORDS], const uint8_t* p) {
  if constexpr (WORDS == 4) {
    const uint4 v = lds128(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <int BITS, int HD, int NT>
__global__ void __launch_bounds__(Shape<BITS, HD, NT>::THREADS, 1) k_attn_paged(const AttnP p) {
  using Sh = Shape<BITS, HD, NT>;
  constexpr int NB = Sh::NB, PB = Sh::PB, W = Sh::W, ST = Sh::ST, THREADS = Sh::THREADS, COLS = NT * 4;
  constexpr int TILES = HD / 16;     // m16 tiles of O
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem + Sh::RING);            // [W][COLS][HD]
  uint4* qfrag = reinterpret_cast<uint4*>(smem + Sh::RING + Sh::MERGE);  // [NT][NB][32]
  __shared__ uint64_t bars[W * ST];
  __shared__ int loaded[W * ST];
  __shared__ uint64_t sums[THREADS];
  __shared__ float qstart[NT * NB * 8], qfac[COLS];     // -8 sum q per block and column; score factor
  __shared__ float ml[W * COLS * 2], weight[kMaxCtas], fin[2];
  __shared__ int last_one;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  if (tid < W * ST) mbar_init(&bars[tid], 1);
  if (tid == 0) fence_barrier_init();
  pdl_wait();

  // ---- the run of this CTA: pieces of all units, cut evenly
  uint64_t mine = 0;
  const int per = (p.d.nseq + THREADS - 1) / THREADS;
  for (int s = tid * per; s < min(p.d.nseq, (tid + 1) * per); s++) {
    const SeqWork w = seq_work(p, s);
    mine += (uint64_t)w.np * w.groups * p.d.KVH;
  }
  sums[tid] = mine;
  live_rows(p.d);                    // records a row count past n_rows
  __syncthreads();
  for (int o = 1; o < THREADS; o <<= 1) {
    const uint64_t v = tid >= o ? sums[tid - o] : 0;
    __syncthreads();
    sums[tid] += v;
    __syncthreads();
  }
  const uint64_t T = sums[THREADS - 1];
  const uint64_t want = (T + W - 1) / W;                // at least a piece per warp
  const uint32_t C = want < gridDim.x ? (uint32_t)want : gridDim.x;
  const uint32_t cta = blockIdx.x;
  if (cta >= C) return;
  Walk seg;
  seg.g = T * cta / C;
  seg.end = T * (cta + 1) / C;
  {
    int lo = 0, hi = THREADS - 1;    // first thread whose sequences reach past seg.g
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (sums[mid] > seg.g) hi = mid;
      else lo = mid + 1;
    }
    seg.s = lo * per;
    seg.base = lo ? sums[lo - 1] : 0;
    seg.w = seq_work(p, seg.s);
  }

  // ---- the warp's feed: runs ST pieces ahead, into the next segments too
  Walk feed = seg;
  bool more = true;
  uint32_t fk = 0, fk1 = 0, piece_n = 0, page_n = 0;
  const auto advance = [&]() {
    for (;;) {
      while (fk < fk1) {
        piece_n = feed.w.range.at(fk);
        fk += W;
        if (feed.needs(p, piece_n)) {
          const uint32_t slot = piece_n * kPieceSlots;
          page_n = slot < p.d.cap ? p.d.pages[(size_t)feed.s * p.d.max_pages + slot / (uint32_t)p.d.page] : 0xffffffffu;
          return;
        }
      }
      if (!feed.next(p)) {
        more = false;
        return;
      }
      fk = feed.k0 + warp;
      fk1 = feed.k1;
    }
  };
  uint32_t issued = 0;
  const auto issue = [&]() {         // the pending piece into the next stage
    if (!more) return;
    if (lane == 0) {
      const uint32_t st = issued % ST;
      const bool ok = page_n < p.d.n_pages;
      loaded[warp * ST + st] = ok;
      if (ok) {
        const uint64_t off = piece_offset(page_n, feed.kvh, (int)(piece_n * kPieceSlots % (uint32_t)p.d.page), p.d.KVH,
                                          p.d.page, PB);
        uint8_t* dst = ring + (size_t)(warp * ST + st) * Sh::STAGE;
        mbar_expect_tx(&bars[warp * ST + st], 2 * PB);
        bulk_g2s(dst, p.d.k + off, PB, &bars[warp * ST + st]);
        bulk_g2s(dst + PB, p.d.v + off, PB, &bars[warp * ST + st]);
      } else {
        set_status(p.d.status, E4B_ST_BADINDEX);
        mbar_arrive(&bars[warp * ST + st]);
      }
    }
    issued++;
    advance();
  };
  advance();
  for (int i = 0; i < ST; i++) issue();

  uint32_t used = 0;                 // pieces that have landed
  bool alive = true;                 // no wait has run out
  bool first = true;                 // the CTA's first segment
  float O[NT][TILES][4];
  uint4 qreg[NT == 1 ? NB : 1];
  float creg[NT == 1 ? NB : 1][2];

  while (seg.next(p)) {
    const SeqWork& w = seg.w;
    // ---- q of the unit as B fragments: HD/8 lanes take a column, a lane the 8 dims of one (block, t)
    {
      constexpr int LPC = HD / 8;
      const int sub = tid / LPC, l = tid % LPC, blk = l >> 2, tt = l & 3;
      for (int c0 = 0; c0 < COLS; c0 += THREADS / LPC) {
        const int c = c0 + sub;
        const int nt = c >> 2, cc = c & 3;
        const int head = p.G > 4 ? c : cc;
        const uint32_t pos = seg.pmin + (p.G > 4 ? 0 : nt);
        const bool on = c < COLS && head < p.G && pos <= seg.pmax;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = 0.f;
        if (on) {
          const uint32_t row = (p.d.rows ? p.d.rows[seg.s] : (uint32_t)seg.s) + (pos - w.p0);
          const float4* src = reinterpret_cast<const float4*>(
              p.q + ((size_t)row * p.QH + seg.kvh * p.G + head) * HD + 8 * l);
          const float4 a = src[0], b = src[1];
          x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        }
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(x[j]));
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // a power of two that brings the largest |q| into [2^14, 2^15): f16 hi + lo then
        // carry every element to 2^-22 of the largest
        const int e = (int)(__float_as_uint(m) >> 23);   // biased exponent; 0: zero or subnormal, 255: inf
        const int up = e == 255 ? 0 : min(14 + 127 - e, 120);
        const float f = __uint_as_float((uint32_t)(up + 127) << 23);
        float hi[8], lo[8], sh = 0.f, sl = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float v = x[j] * f;
          hi[j] = __half2float(__float2half_rn(v));
          lo[j] = __half2float(__float2half_rn(v - hi[j]));
          sh += hi[j];
          sl += lo[j];
        }
        if constexpr (BITS == 4) {
          sh += __shfl_xor_sync(0xffffffffu, sh, 1);
          sl += __shfl_xor_sync(0xffffffffu, sl, 1);
          sh += __shfl_xor_sync(0xffffffffu, sh, 2);
          sl += __shfl_xor_sync(0xffffffffu, sl, 2);
        }
        if (c < COLS) {
          uint4 fh, fl;
          if constexpr (BITS == 4) {
            constexpr float r = 1.f / 16.f;
            fh = make_uint4(pack2(hi[0], hi[4]), pack2(hi[2], hi[6]), pack2(hi[1] * r, hi[5] * r), pack2(hi[3] * r, hi[7] * r));
            fl = make_uint4(pack2(lo[0], lo[4]), pack2(lo[2], lo[6]), pack2(lo[1] * r, lo[5] * r), pack2(lo[3] * r, lo[7] * r));
            if (tt == 0) {
              qstart[(nt * NB + blk) * 8 + cc] = sh * (-8.f / kTwo24);
              qstart[(nt * NB + blk) * 8 + cc + 4] = sl * (-8.f / kTwo24);
            }
          } else {
            fh = make_uint4(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]), pack2(hi[4], hi[5]), pack2(hi[6], hi[7]));
            fl = make_uint4(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(lo[4], lo[5]), pack2(lo[6], lo[7]));
          }
          qfrag[(nt * NB + blk) * 32 + cc * 4 + tt] = fh;
          qfrag[(nt * NB + blk) * 32 + (cc + 4) * 4 + tt] = fl;
          if (l == 0) qfac[c] = p.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - up) << 23) * (BITS == 4 ? kTwo24 : 1.f);
        }
      }
    }
    __syncthreads();
    float m[NT][2], lsum[NT][2], fac[NT][2];
    bool live[NT];
    uint32_t pos[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      pos[nt] = seg.pmin + (p.G > 4 ? 0 : nt);
      live[nt] = pos[nt] <= seg.pmax;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        m[nt][j] = -INFINITY;
        lsum[nt][j] = 0.f;
        fac[nt][j] = qfac[nt * 4 + 2 * (t & 1) + j];
      }
#pragma unroll
      for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) O[nt][i][j] = 0.f;
    }
    if constexpr (NT == 1) {
#pragma unroll
      for (int b = 0; b < NB; b++) {
        qreg[b] = qfrag[b * 32 + lane];
        if constexpr (BITS == 4) creg[b][0] = qstart[b * 8 + 2 * t], creg[b][1] = qstart[b * 8 + 2 * t + 1];
      }
    }

    for (uint32_t k = seg.k0 + warp; k < seg.k1; k += W) {
      const uint32_t piece = w.range.at(k);
      if (!seg.needs(p, piece)) continue;
      const uint32_t st = used % ST;
      if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&bars[warp * ST + st], (used / ST) & 1u, p.d.status));
      if (alive) used++;
      const bool here = alive && loaded[warp * ST + st] != 0;
      const uint8_t* kp = ring + (size_t)(warp * ST + st) * Sh::STAGE;
      const uint8_t* vp = kp + PB;
      const uint32_t t0 = piece * kPieceSlots;

      // ---- scores
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[nt][j] = 0.f;
      if constexpr (BITS == 4) {
        constexpr int RUN = NB < 4 ? NB : 4;
        uint32_t da[NB / 2], db[NB / 2];                 // scales of slots g, g + 8
        lds_words<NB / 2>(da, kp + g * NB * 2);
        lds_words<NB / 2>(db, kp + (g + 8) * NB * 2);
#pragma unroll
        for (int r = 0; r < NB / RUN; r++) {
          uint32_t wa[RUN], wb[RUN];
          lds_words<RUN>(wa, kp + HD + ((r * 16 + g) * 4 + t) * (RUN * 4));
          lds_words<RUN>(wb, kp + HD + ((r * 16 + g + 8) * 4 + t) * (RUN * 4));
#pragma unroll
          for (int i = 0; i < RUN; i++) {
            const int b = r * RUN + i;
            const uint32_t sa = wa[i] >> 8, sb = wb[i] >> 8;
            const float d0 = h2f((uint16_t)(da[b / 2] >> (16 * (b & 1)))), d1 = h2f((uint16_t)(db[b / 2] >> (16 * (b & 1))));
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              if (NT > 1 && !live[nt]) continue;
              uint4 qb;
              float acc[4];
              if constexpr (NT == 1) {
                qb = qreg[b];
                acc[0] = acc[2] = creg[b][0];
                acc[1] = acc[3] = creg[b][1];
              } else {
                qb = qfrag[(nt * NB + b) * 32 + lane];
                const float2 c2 = *reinterpret_cast<const float2*>(&qstart[(nt * NB + b) * 8 + 2 * t]);
                acc[0] = acc[2] = c2.x;
                acc[1] = acc[3] = c2.y;
              }
              mma16816(acc, wa[i] & kLowCodes, wb[i] & kLowCodes, sa & kLowCodes, sb & kLowCodes, qb.x, qb.y);
              mma16816(acc, wa[i] & kHighCodes, wb[i] & kHighCodes, sa & kHighCodes, sb & kHighCodes, qb.z, qb.w);
              s[nt][0] = fmaf(d0, acc[0], s[nt][0]);
              s[nt][1] = fmaf(d0, acc[1], s[nt][1]);
              s[nt][2] = fmaf(d1, acc[2], s[nt][2]);
              s[nt][3] = fmaf(d1, acc[3], s[nt][3]);
            }
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const uint4 wa = lds128(kp + (b * 16 + g) * 64 + t * 16), wb = lds128(kp + (b * 16 + g + 8) * 64 + t * 16);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            if (NT > 1 && !live[nt]) continue;
            uint4 qb;
            if constexpr (NT == 1) qb = qreg[b];
            else qb = qfrag[(nt * NB + b) * 32 + lane];
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(acc, wa.x, wb.x, wa.y, wb.y, qb.x, qb.y);
            mma16816(acc, wa.z, wb.z, wa.w, wb.w, qb.z, qb.w);
#pragma unroll
            for (int j = 0; j < 4; j++) s[nt][j] += acc[j];
          }
        }
      }

      // ---- softmax state and p as B fragments
      uint32_t ph[NT][2], pl[NT][2], keep[NT][2];        // slots (2t, 2t+1), (2t+8, 2t+9); keep: mask of visible halves
      bool full[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        full[nt] = here && t0 + kPieceSlots - 1 <= pos[nt] &&
                   (p.window == 0 || pos[nt] - t0 < p.window || t0 + kPieceSlots <= p.sinks);
        if (NT > 1 && !live[nt]) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[nt][j] += __shfl_xor_sync(0xffffffffu, s[nt][j], 2);     // hi + lo columns
          v[j] = s[nt][j] * fac[nt][j & 1];
        }
        bool va = true, vb = true;
        if (!full[nt]) {
          va = here && slot_visible(t0 + g, pos[nt], p.window, p.sinks);
          vb = here && slot_visible(t0 + g + 8, pos[nt], p.window, p.sinks);
          if (!va) v[0] = v[1] = -INFINITY;
          if (!vb) v[2] = v[3] = -INFINITY;
          keep[nt][0] = keep[nt][1] = 0;
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (here && slot_visible(t0 + 2 * t + (j & 1) + 8 * (j >> 1), pos[nt], p.window, p.sinks))
              keep[nt][j >> 1] |= 0xffffu << (16 * (j & 1));
        }
        const bool grow = v[0] > m[nt][0] || v[2] > m[nt][0] || v[1] > m[nt][1] || v[3] > m[nt][1];
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float n = fmaxf(v[j], v[j + 2]);
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 4));
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 8));
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 16));
            n = fmaxf(n, m[nt][j]);
            const float a = n == m[nt][j] ? 1.f : ex2(m[nt][j] - n);
            m[nt][j] = n;
            lsum[nt][j] *= a;
#pragma unroll
            for (int i = 0; i < TILES; i++) O[nt][i][j] *= a, O[nt][i][j + 2] *= a;
          }
        }
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; j++) e[j] = ex2(v[j] - m[nt][j & 1]);
        if (!full[nt]) {
          if (!va) e[0] = e[1] = 0.f;
          if (!vb) e[2] = e[3] = 0.f;
        }
        lsum[nt][0] += e[0] + e[2];
        lsum[nt][1] += e[1] + e[3];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint32_t h = pack2(e[2 * j], e[2 * j + 1]);
          const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&h));
          const uint32_t l = pack2(e[2 * j] - hf.x, e[2 * j + 1] - hf.y);
          if constexpr (BITS == 4) {
            ph[nt][j] = transpose8x8(h);
            pl[nt][j] = transpose8x8(l);
          } else {
            ph[nt][j] = transpose8x8(t < 2 ? h : l);      // columns 0-3 hi, 4-7 lo
          }
        }
      }

      // ---- O += V^T p
      if constexpr (BITS == 4) {
        uint32_t vw[4][NB / 2];
#pragma unroll
        for (int i = 0; i < 4; i++) lds_words<NB / 2>(vw[i], vp + HD + (i * 32 + lane) * (NB * 2));
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const uint2 d2 = *reinterpret_cast<const uint2*>(vp + (t * NB + b) * 8);
          const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
          const uint32_t x = __byte_perm(vw[0][b / 2], vw[1][b / 2], sel), y = __byte_perm(vw[2][b / 2], vw[3][b / 2], sel);
          const uint32_t xs = x >> 8, ys = y >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            if (NT > 1 && !live[nt]) continue;
            uint32_t bb[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
              uint32_t d = j ? d2.y : d2.x;
              if (!full[nt]) d &= keep[nt][j];
              const uint32_t hi = hmul2(ph[nt][j], d);
              const uint32_t lo = hfma2(pl[nt][j], d, hfma2(ph[nt][j], d, hi ^ 0x80008000u));
              bb[j] = g < 4 ? hi : lo;
            }
            mma16816(O[nt][2 * b], x & kLowCodes, xs & kLowCodes, y & kLowCodes, ys & kLowCodes, bb[0], bb[1]);
            mma16816(O[nt][2 * b + 1], x & kHighCodes, xs & kHighCodes, y & kHighCodes, ys & kHighCodes, bb[0], bb[1]);
            mma16816(O[nt][2 * b], kMinus8Low, kMinus8Low, kMinus8Low, kMinus8Low, bb[0], bb[1]);
            mma16816(O[nt][2 * b + 1], kMinus8High, kMinus8High, kMinus8High, kMinus8High, bb[0], bb[1]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < HD / 64; j++) {
          uint32_t vw[4][4];
#pragma unroll
          for (int i = 0; i < 4; i++) lds_words<4>(vw[i], vp + ((j * 4 + i) * 32 + lane) * 16);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t a0 = __byte_perm(vw[0][i], vw[1][i], 0x5410), a1 = __byte_perm(vw[0][i], vw[1][i], 0x7632);
            const uint32_t a2 = __byte_perm(vw[2][i], vw[3][i], 0x5410), a3 = __byte_perm(vw[2][i], vw[3][i], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              if (NT > 1 && !live[nt]) continue;
              if (full[nt]) mma16816(O[nt][4 * j + i], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
              else
                mma16816(O[nt][4 * j + i], a0 & keep[nt][0], a1 & keep[nt][0], a2 & keep[nt][1], a3 & keep[nt][1],
                         ph[nt][0], ph[nt][1]);
            }
          }
        }
      }
      __syncwarp();
      if (alive) issue();
    }

    // ---- the warps' states, merged
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float l = lsum[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (lane < 2) {
          ml[(warp * COLS + nt * 4 + 2 * t + j) * 2] = m[nt][j];
          ml[(warp * COLS + nt * 4 + 2 * t + j) * 2 + 1] = l;
        }
      }
#pragma unroll
      for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float o = O[nt][i][j];
          o += __shfl_xor_sync(0xffffffffu, o, 2);
          int dim;
          if constexpr (BITS == 4) {
            o *= i & 1 ? kTwo20 : kTwo24;
            dim = (i / 2) * 32 + 4 * g + (i & 1) + 2 * (j >> 1);
          } else {
            dim = (i / 4) * 64 + 8 * g + 2 * (i & 3) + (j >> 1);
          }
          if (t < 2) merge[(size_t)(warp * COLS + nt * 4 + 2 * t + (j & 1)) * HD + dim] = o;
        }
    }
    __syncthreads();
    const bool whole = seg.k0 == 0 && seg.k1 == w.np;
    const uint64_t unit_end = seg.unit0 + w.np;
    const uint32_t c0 = (uint32_t)(((seg.unit0 + 1) * C - 1) / T), c1 = (uint32_t)((unit_end * C - 1) / T);
    const uint32_t row0 = (p.d.rows ? p.d.rows[seg.s] : (uint32_t)seg.s) + (seg.pmin - w.p0);
    const auto finish = [&](int c, int dim, float o, float M, float L) {
      const int head = seg.kvh * p.G + (p.G > 4 ? c : c & 3);
      const size_t row = row0 + (p.G > 4 ? 0 : c >> 2);
      const float val = L != 0.f ? o / L : 0.f;          // a NaN sum stays one
      if (p.out_f) p.out_f[(row * p.QH + head) * HD + dim] = val;
      if (p.out_h)
        p.out_h[row * p.QH * HD + (p.xfo ? xfo_pos(head * HD + dim) : head * HD + dim)] = f2h(val);
      if (p.lse && dim == 0) p.lse[row * p.QH + head] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
    };
    const auto col_live = [&](int c) {
      return p.G > 4 ? c < p.G : (c & 3) < p.G && seg.pmin + (c >> 2) <= seg.pmax;
    };
    for (int e = tid; e < COLS * HD; e += THREADS) {
      const int c = e / HD, dim = e % HD;
      if (!col_live(c)) continue;
      float M = -INFINITY, o = 0.f, L = 0.f;
#pragma unroll
      for (int i = 0; i < W; i++) M = fmaxf(M, ml[(i * COLS + c) * 2]);
#pragma unroll
      for (int i = 0; i < W; i++) {
        const float mi = ml[(i * COLS + c) * 2], a = mi == M ? 1.f : ex2(mi - M);
        L = fmaf(a, ml[(i * COLS + c) * 2 + 1], L);
        o = fmaf(a, merge[(size_t)(i * COLS + c) * HD + dim], o);
      }
      if (whole) {
        finish(c, dim, o, M, L);
      } else {
        float* part = p.parts + (2 * (size_t)cta + (first ? 0 : 1)) * kPartFloats;
        part[c * HD + dim] = o;
        if (dim == 0) part[kCols * 256 + 2 * c] = M, part[kCols * 256 + 2 * c + 1] = L;
      }
    }
    if (!whole) {
      // a unit cut between CTAs c0..c1: only c0 may hold it behind other segments
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const uint32_t n = c1 - c0;
        last_one = atomicInc(&p.arrived[c0], n) == n;    // wraps to zero with the last arrival
        __threadfence();
      }
      __syncthreads();
      if (last_one) {
        const uint32_t n = c1 - c0 + 1;
        const uint64_t c0_begin = T * c0 / C;
        const auto part_of = [&](uint32_t i) {
          return p.parts + (2 * (size_t)(c0 + i) + (i == 0 && c0_begin != seg.unit0 ? 1 : 0)) * kPartFloats;
        };
        for (int c = 0; c < COLS; c++) {
          if (!col_live(c)) continue;
          if (warp == 0) {
            float M = -INFINITY, L = 0.f;
            for (uint32_t i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(&part_of(i)[kCols * 256 + 2 * c]));
            M = warp_max(M);
            for (uint32_t i = 0; i < n; i++) {
              const float mi = __ldcg(&part_of(i)[kCols * 256 + 2 * c]), li = __ldcg(&part_of(i)[kCols * 256 + 2 * c + 1]);
              const float a = mi == M ? 1.f : ex2(mi - M);
              if (lane == 0) weight[i] = a;
              L = fmaf(a, li, L);
            }
            if (lane == 0) fin[0] = M, fin[1] = L;
          }
          __syncthreads();
          for (int dim = tid; dim < HD; dim += THREADS) {
            float o = 0.f;
            for (uint32_t i = 0; i < n; i++) o = fmaf(weight[i], __ldcg(&part_of(i)[c * HD + dim]), o);
            finish(c, dim, o, fin[0], fin[1]);
          }
          __syncthreads();
        }
      }
    }
    first = false;
    __syncthreads();                 // q fragments, merge buffer and states are free again
  }
  // after a time-out: copies still in flight land (bounded) before the CTA exits
  for (; used < issued; used++) mbar_wait(&bars[warp * ST + used % ST], (used / ST) & 1u, p.d.status);
}

template <int BITS, int HD, int NT>
int launch(e4b_ctx* c, const AttnP& p) {
  using Sh = Shape<BITS, HD, NT>;
  static_assert(Sh::SMEM < 226 * 1024, "shared memory");
  E4B_CUDA(c, cudaFuncSetAttribute(k_attn_paged<BITS, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::SMEM));
  const int ctas = c->sm_count < kMaxCtas ? c->sm_count : kMaxCtas;
  return e4b_launch(c, "attn_paged", k_attn_paged<BITS, HD, NT>, dim3(ctas), dim3(Sh::THREADS), Sh::SMEM, p);
}
template <int BITS, int NT>
int launch_hd(e4b_ctx* c, const AttnP& p, int HD) {
  return HD == 256 ? launch<BITS, 256, NT>(c, p) : (HD == 128 ? launch<BITS, 128, NT>(c, p) : launch<BITS, 64, NT>(c, p));
}
}  // namespace

extern "C" {

E4B_API size_t e4b_paged_scratch_bytes(void) { return kMaxCtas * sizeof(uint32_t) + 2 * kMaxCtas * kPartFloats * sizeof(float); }

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
  p.arrived = static_cast<uint32_t*>(scratch);
  p.parts = reinterpret_cast<float*>(p.arrived + kMaxCtas);
  p.QH = QH;
  p.G = QH / kv->kv_heads;
  p.xfo = xfo ? 1 : 0;
  p.window = (uint32_t)window;
  p.sinks = (uint32_t)sinks;
  p.scale = scale;
  // n-tiles of 4 heads: one row per unit, or two rows that share the decoded keys
  // and values when a sequence may have several; more than 4 heads take both tiles
  const int NT = p.G > 4 || kv->rows ? 2 : 1;
  p.per_unit = p.G > 4 ? 1 : NT;
  if (kv->bits == 16) return NT == 1 ? launch_hd<16, 1>(c, p, kv->head_dim) : launch_hd<16, 2>(c, p, kv->head_dim);
  return NT == 1 ? launch_hd<4, 1>(c, p, kv->head_dim) : launch_hd<4, 2>(c, p, kv->head_dim);
}

}  // extern "C"
