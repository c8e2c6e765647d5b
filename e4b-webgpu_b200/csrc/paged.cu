// Paged KV cache: head prep (per-head RMSNorm, RoPE) with the append of keys and
// values in f16 or 4 bits, reading rows back, and advancing the lengths.
#include "paged.cuh"
#include "stream.cuh"

namespace {
using namespace e4b;

struct PrepP {
  PagedDev d;
  const void* qkv;
  const float* qw;
  const float* kw;
  float* q_out;
  int QH, angles, norm, keqv, nparts;
  int rows_per_turn, rows_per_cta;
  int64_t stride;                    // elements between rows
  float eps;
  double log2_theta;
};

// How the rows reach the lanes: straight from global memory, a few rows, each spread
// over CTAs (kFew); through shared memory, whole rows by bulk copies into two stages,
// so some 150 KB per SM are in flight whatever the lanes do (kStaged); or from global
// memory, some rows a turn, for what the copies cannot take (kDirect: partial sums,
// rows that are too long or not 16-byte aligned).
enum { kFew, kStaged, kDirect };
constexpr int kStageBytes = 48 * 1024;
constexpr int kBatch = 64;           // rows whose places are looked up at once
constexpr int turn_rows(int HD) { return 512 / HD; }     // rows of a turn at most
template <int MODE>
constexpr int threads_of() { return MODE == kStaged ? 512 : 256; }

struct Quad {
  float x[4];
};

E4B_DEV __half2 as_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
E4B_DEV uint32_t as_u32(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
E4B_DEV uint32_t pack2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }

// Four consecutive elements of an input row.
template <bool XF16>
E4B_DEV Quad load_quad(const uint8_t* row, int at) {
  Quad r;
  if constexpr (XF16) {
    const uint2 w = *reinterpret_cast<const uint2*>(row + 2 * at);
    const float2 a = __half22float2(as_h2(w.x)), b = __half22float2(as_h2(w.y));
    r.x[0] = a.x, r.x[1] = a.y, r.x[2] = b.x, r.x[3] = b.y;
  } else {
    const float4 v = *reinterpret_cast<const float4*>(row + 4 * at);
    r.x[0] = v.x, r.x[1] = v.y, r.x[2] = v.z, r.x[3] = v.w;
  }
  return r;
}

// With f32 partial sums (never staged), their sum in order.
template <bool XF16, int MODE>
E4B_DEV Quad load_parts(const PrepP& p, const uint8_t* row, int at) {
  Quad v = load_quad<XF16>(row, at);
  if (MODE != kStaged && !XF16)
    for (int k = 1; k < p.nparts; k++) {
      const Quad w = load_quad<XF16>(row + (uint64_t)k * p.d.n_rows * p.stride * 4, at);
#pragma unroll
      for (int j = 0; j < 4; j++) v.x[j] += w.x[j];
    }
  return v;
}

E4B_DEV float rsqrt_fast(float x) {
  float y;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
E4B_DEV float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x^-1/2 to 64-bit precision: two Newton steps from the f32 estimate.
E4B_DEV double rsqrt64(double x) {
  if (!(x > 1e-30 && x < 1e30)) return rsqrt(x);         // the estimate's range
  double y = (double)rsqrt_fast((float)x);
#pragma unroll
  for (int i = 0; i < 2; i++) y = y * fma(-0.5 * x * y, y, 1.5);
  return y;
}

// The q4_0 codes of two quads (four consecutive f16 values each, their blocks in 8
// neighbouring lanes): d = m / -8 for the first element m of the largest magnitude,
// codes trunc(x / d + 8.5).  x and 8 d are f16, so a quotient that is not exactly
// between two codes is at least 2^-13 away from there: with 2^-15 added, the product
// with 1 / d (off by less than 2^-19) gives the exact quotient's code, ties upwards.
// d16: the blocks' stored scales.
E4B_DEV void quantise(const uint32_t (&h)[2][2], int lane8, uint32_t (&codes)[2], uint32_t (&d16)[2]) {
  __half2 hi[2], lo[2];
#pragma unroll
  for (int q = 0; q < 2; q++) {
    hi[q] = __hmax2_nan(as_h2(h[q][0]), as_h2(h[q][1]));
    lo[q] = __hmin2_nan(as_h2(h[q][0]), as_h2(h[q][1]));
  }
  // both quads' largest and smallest values, then over the blocks' lanes
  __half2 top = __hmax2_nan(__lows2half2(hi[0], hi[1]), __highs2half2(hi[0], hi[1]));
  __half2 bot = __hmin2_nan(__lows2half2(lo[0], lo[1]), __highs2half2(lo[0], lo[1]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    top = __hmax2_nan(top, as_h2(__shfl_xor_sync(0xffffffffu, as_u32(top), o)));
    bot = __hmin2_nan(bot, as_h2(__shfl_xor_sync(0xffffffffu, as_u32(bot), o)));
  }
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const float t = q ? __high2float(top) : __low2float(top), b = q ? __high2float(bot) : __low2float(bot);
    float m = t > -b ? t : b;
    if (__any_sync(0xffffffffu, t == -b && t != 0.f)) {  // of both signs: the first one
      uint32_t first = 64;
#pragma unroll
      for (int j = 3; j >= 0; j--) {
        const float x = j & 1 ? __high2float(as_h2(h[q][j >> 1])) : __low2float(as_h2(h[q][j >> 1]));
        if (fabsf(x) == t) first = (uint32_t)(lane8 * 4 + j) * 2 + (x < 0.f);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      if (t == -b && t != 0.f) m = first & 1u ? b : t;
    }
    const float d = m * -0.125f;
    d16[q] = f2h(d);
    if (!(fabsf(d) < INFINITY)) d16[q] = 0x7fffu;        // an infinity or NaN in the block
    const float inv = rcp_fast(d);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = j & 1 ? __high2float(as_h2(h[q][j >> 1])) : __low2float(as_h2(h[q][j >> 1]));
      const float c = fminf(fmaxf(fmaf(x, inv, 8.5f + 1.f / 32768.f), 0.f), 15.f);
      // adding 2^23 towards minus infinity leaves the integer part in the low bits
      w |= (__float_as_uint(__fadd_rd(c, 8388608.f)) & 15u) << (4 * j);
    }
    codes[q] = d == 0.f || d16[q] == 0x7fffu ? 0x8888u : w;
  }
}

// Where a row goes: its sequence's position, and in the pools the byte of its piece of
// KV head 0 (head h is h * (page / 16) pieces further) and its slot there.
struct RowPlace {
  uint64_t pos, offset;
  int slot, ok;                      // ok: the cache has a slot for it
};
template <int PB>
E4B_DEV RowPlace place_in(const PagedDev& d, uint32_t row, int seq) {
  RowPlace r;
  r.pos = (uint64_t)d.lens[seq] + (d.rows ? row - d.rows[seq] : 0u);
  uint32_t page;
  r.ok = page_of(d, seq, r.pos, page);
  const int in_page = (int)((uint32_t)r.pos % (uint32_t)d.page);
  r.slot = in_page % kPieceSlots;
  r.offset = piece_offset(page, 0, in_page, d.KVH, d.page, PB);
  return r;
}
template <int PB>
E4B_DEV RowPlace place_row(const PagedDev& d, uint32_t row) {          // a warp
  return place_in<PB>(d, row, seq_of_row(d, row));
}
template <int PB>
E4B_DEV RowPlace place_one(const PagedDev& d, uint32_t row) {          // a thread: the last sequence that begins by the row
  int lo = 0, hi = d.rows ? d.nseq - 1 : 0;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (d.rows[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return place_in<PB>(d, row, d.rows ? lo : (int)row);
}

// HD/8 lanes take a head, each lane dims 4l..4l+3 and HD/2 + 4l..4l+3, so a rotation
// pair (p, p + HD/2) and a group of four codes sit in one lane and a 32-dim block in 8
// neighbouring lanes.  The rotation's angles are formed once per row for all its heads,
// in 64 bits (a position of 10^6 times a frequency leaves f32 no fraction).  q is
// computed in f32.  Keys and values are formed in 64 bits and rounded through f32 to f16:
// what is stored is the exact value's rounding (but within 2^-24 of a border between two
// f16, where the first rounding may decide) whatever the order of the sums, so neither the
// f16 rows nor the 4-bit codes of them depend on it.  Bound by memory for many rows (per
// row of 16 q + 2 x 4 heads of 256: 24.6 KB read, 16.4 KB of q and 2.3 KB of 4-bit cache
// written): prompts of 16 x 1..1000
// such rows take 69 us and their read-back as f16 12.8 us, 4.3 TB/s together (floor 55 us).
// f16 rows whose values are their keys, 8 x 1..500 into an f16 cache, 20 and 4.1 us (floor
// 12 us together), are bound by the lanes' conversions and 64-bit products between barriers
// (issue slots 53 % busy); one row, 2.9 and 1.9 us, and 64, 3.9 and 2.1 us, by latency: a
// chain of loads each.
// A head of a turn: where its elements are, and where it goes.
struct Item {
  uint32_t src;                      // bytes from the turn's first row (rows row_bytes apart: kStaged), or of its row
  uint16_t row, head;                // row of the turn (kNoRow: none); query head, or KV head with kKey / kValue
};
enum : uint16_t { kNoRow = 0xffff, kKey = 0x4000, kValue = 0x8000, kHeadMask = 0x3fff };

template <int HD, int BITS, bool XF16, int MODE>
__global__ void __launch_bounds__(threads_of<MODE>(), MODE == kFew ? 1 : 2) k_headprep_paged(const PrepP p) {
  constexpr int LPH = HD / 8, HALF = HD / 2, PB = BITS == 16 ? 32 * HD : 9 * HD, ES = XF16 ? 2 : 4;
  constexpr int THREADS = threads_of<MODE>(), NS = THREADS / LPH, ROWS = MODE == kFew ? 1 : turn_rows(HD);
  constexpr int BUFS = MODE == kFew ? 1 : 2, BATCH = MODE == kFew ? 1 : kBatch, GROUPS = 32 / LPH;
  extern __shared__ __align__(128) uint8_t dyn[];        // kStaged: 2 x kStageBytes; then the items
  uint8_t* const stages = dyn;
  Item* const items = reinterpret_cast<Item*>(dyn + (MODE == kStaged ? 2 * kStageBytes : 0));
  __shared__ __align__(16) double2 turns[BUFS][ROWS][HALF];            // (cos, sin) of a turn's angles
  __shared__ __align__(16) float2 turns32[BUFS][ROWS][HALF];
  __shared__ double kw64[HD];
  __shared__ RowPlace places[BATCH];
  __shared__ uint64_t landed[2];
  const int tid = threadIdx.x, warp = tid >> 5, l = tid % LPH, sub = tid / LPH, lane8 = l & 7;
  const int KVH = p.d.KVH, RT = MODE == kFew ? 1 : p.rows_per_turn;
  const uint32_t head_bytes = (uint32_t)(p.d.page / kPieceSlots) * PB;
  const uint32_t row_bytes = (uint32_t)(p.QH + KVH * (p.keqv ? 1 : 2)) * HD * ES;
  const uint8_t* const qkv = static_cast<const uint8_t*>(p.qkv);
  // pair tid % HALF of the angles; 1/pi: sincospi reduces its argument exactly
  const int pair = tid % HALF;
  const double freq = pair < p.angles ? exp2((-2.0 * pair / HD) * p.log2_theta) * 0.3183098861837906715 : 0.0;
  const int turned = min(max(p.angles - 4 * l, 0), 4);   // of the lane's four pairs
  if (MODE == kStaged && tid == 0) {
    mbar_init(&landed[0], 1);
    mbar_init(&landed[1], 1);
    fence_barrier_init();
  }
  // the turn's items: its query heads (up to a whole warp's), then its key and value heads
  const int nq = (RT * p.QH + GROUPS - 1) / GROUPS * GROUPS, total = nq + (RT * 2 * KVH + GROUPS - 1) / GROUPS * GROUPS;
  const auto item_of = [&](int i) {
    Item it{0u, kNoRow, 0};
    if (i < RT * p.QH) {
      it.row = (uint16_t)(RT == 1 ? 0 : i / p.QH);
      it.head = (uint16_t)(i - it.row * p.QH);
      it.src = (uint32_t)it.head * HD * ES;
    } else if (i >= nq && i - nq < RT * 2 * KVH) {
      it.row = (uint16_t)(RT == 1 ? 0 : (i - nq) / (2 * KVH));
      const int h = i - nq - it.row * 2 * KVH, kvh = h < KVH ? h : h - KVH;
      it.head = (uint16_t)(kvh | (h < KVH ? kKey : kValue));
      it.src = (uint32_t)(p.QH + (p.keqv ? kvh : h)) * HD * ES;
    }
    if (MODE == kStaged && it.row != kNoRow) it.src += it.row * row_bytes;
    return it;
  };
  if (MODE != kFew)
    for (int i = tid; i < total; i += THREADS) items[i] = item_of(i);
  float qw[8], kw = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) qw[j] = 1.f;
  pdl_wait();
  static_assert(HD <= THREADS, "a thread per weight");
  if (p.norm) {                      // (the call before may have written the weights)
    if (p.QH > 0) {
      const float4 a = *reinterpret_cast<const float4*>(p.qw + 4 * l), b = *reinterpret_cast<const float4*>(p.qw + HALF + 4 * l);
      qw[0] = a.x, qw[1] = a.y, qw[2] = a.z, qw[3] = a.w, qw[4] = b.x, qw[5] = b.y, qw[6] = b.z, qw[7] = b.w;
    }
    if (tid < HD) kw = p.kw[tid];
  }
  // a CTA's rows are consecutive: they share sequences, pieces and (nearly) angles
  const uint32_t live = live_rows(p.d);
  const uint32_t first_row = blockIdx.x * p.rows_per_cta, end_row = min(live, first_row + p.rows_per_cta);
  const auto bring = [&](uint32_t row, uint32_t turn_no) {             // thread 0: a turn's rows into their stage
    if (row >= end_row) return;
    const int n = (int)min((uint32_t)RT, end_row - row);
    uint64_t* bar = &landed[turn_no & 1];
    mbar_expect_tx(bar, n * row_bytes);
    for (int i = 0; i < n; i++)
      bulk_g2s(stages + (turn_no & 1) * kStageBytes + i * row_bytes, qkv + (uint64_t)(row + i) * p.stride * ES, row_bytes, bar);
  };
  if (MODE == kStaged && tid == 0) {
    bring(first_row, 0);
    bring(first_row + RT, 1);
  }
  const uint32_t batch_rows = MODE == kFew ? 1 : BATCH / RT * RT;
  const auto look_up = [&](uint32_t row) {               // the places of the batch that begins with a row
    if constexpr (MODE == kFew) {
      if (warp == 0 && row < end_row) {
        const RowPlace pl = place_row<PB>(p.d, row);
        if (tid == 0) places[0] = pl;
      }
    } else if (tid < batch_rows && row + tid < end_row) {
      places[tid] = place_one<PB>(p.d, row + tid);
    }
    __syncthreads();
  };
  // The angles of a turn: thread group g of HALF threads forms row g's.  A row RT
  // positions behind the group's last one is a rotation by RT frequencies away.
  const int group = tid / HALF;
  double c = 1.0, s = 0.0, cr = 1.0, sr = 0.0;
  uint64_t last = ~0ull;
  if constexpr (MODE != kFew)
    if (group < RT && pair < p.angles) sincospi((double)RT * freq, &sr, &cr);
  const auto form_angles = [&](uint32_t row, int at, int buf, bool anew) {
    for (int g = group; g < RT; g += THREADS / HALF)
      if (row + g < end_row && pair < p.angles) {
        const uint64_t pos = places[at + g].pos;
        if (MODE != kFew && !anew && RT <= THREADS / HALF && pos == last + RT) {
          const double t = c * cr - s * sr;
          s = s * cr + c * sr;
          c = t;
        } else {
          sincospi((double)pos * freq, &s, &c);
        }
        last = pos;
        turns[buf][g][pair] = make_double2(c, s);
        turns32[buf][g][pair] = make_float2((float)c, (float)s);
      }
  };
  look_up(first_row);
  if (tid < HD) kw64[tid] = (double)kw;
  form_angles(first_row, 0, 0, true);
  __syncthreads();
  uint32_t turn_no = 0, at_row = 0;                      // at_row: the turn's place in its batch
  bool alive = true;
  for (uint32_t row0 = first_row; row0 < end_row; row0 += RT, turn_no++) {
    const int rows = (int)min((uint32_t)RT, end_row - row0);
    const auto& turn = turns[turn_no % BUFS];
    const auto& turn32 = turns32[turn_no % BUFS];
    const RowPlace* place = places + at_row;
    if constexpr (MODE == kStaged)
      alive = __all_sync(0xffffffffu, mbar_wait(&landed[turn_no & 1], (turn_no >> 1) & 1u, p.d.status));
    float* const q_rows = p.q_out + (size_t)row0 * p.QH * HD + 4 * l;
    // every lane of a warp makes the same turns (shuffles): a group without a head works on row 0
    for (int i = blockIdx.y * NS + sub; alive && i < total; i += gridDim.y * NS) {
      const Item it = MODE == kFew ? item_of(i) : items[i];
      const bool on = it.row < rows;
      const int r = on ? it.row : 0;
      Quad a, b;
      if constexpr (MODE == kStaged) {
        const uint8_t* src = stages + (turn_no & 1) * kStageBytes + it.src;
        a = load_quad<XF16>(src, 4 * l);
        b = load_quad<XF16>(src, HALF + 4 * l);
      } else {
        const uint8_t* src = qkv + (uint64_t)(row0 + r) * p.stride * ES + it.src;
        a = load_parts<XF16, MODE>(p, src, 4 * l);
        b = load_parts<XF16, MODE>(p, src, HALF + 4 * l);
      }
      if (i < nq) {
        float(&xa)[4] = a.x;
        float(&xb)[4] = b.x;
        if (p.norm) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; j++) sum = fmaf(xa[j], xa[j], fmaf(xb[j], xb[j], sum));
#pragma unroll
          for (int o = 1; o < LPH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = rsqrt_fast(sum * (1.f / HD) + p.eps);
#pragma unroll
          for (int j = 0; j < 4; j++) xa[j] *= inv * qw[j], xb[j] *= inv * qw[4 + j];
        }
        if (turned) {
          const float4 c0 = *reinterpret_cast<const float4*>(&turn32[r][4 * l]);
          const float4 c1 = *reinterpret_cast<const float4*>(&turn32[r][4 * l + 2]);
          const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float y = xa[j] * cs[2 * j] - xb[j] * cs[2 * j + 1], z = xa[j] * cs[2 * j + 1] + xb[j] * cs[2 * j];
            if (j < turned) xa[j] = y, xb[j] = z;
          }
        }
        if (on) {
          float* qo = q_rows + (uint32_t)(r * p.QH + it.head) * HD;
          *reinterpret_cast<float4*>(qo) = make_float4(xa[0], xa[1], xa[2], xa[3]);
          *reinterpret_cast<float4*>(qo + HALF) = make_float4(xb[0], xb[1], xb[2], xb[3]);
        }
        continue;
      }
      const bool is_v = (it.head & kValue) != 0;
      double inv = 1.0;
      if (p.norm) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) sum = fma((double)a.x[j], (double)a.x[j], fma((double)b.x[j], (double)b.x[j], sum));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        inv = rsqrt64(sum * (1.0 / HD) + (double)p.eps);
      }
      float fa[4], fb[4];
      if (is_v || (!p.norm && !turned)) {
#pragma unroll
        for (int j = 0; j < 4; j++) fa[j] = (float)((double)a.x[j] * inv), fb[j] = (float)((double)b.x[j] * inv);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          double xa = (double)a.x[j] * inv, xb = (double)b.x[j] * inv;
          if (p.norm) xa *= kw64[4 * l + j], xb *= kw64[HALF + 4 * l + j];
          if (j < turned) {
            const double2 cs = turn[r][4 * l + j];
            const double y = xa * cs.x - xb * cs.y;
            xb = xa * cs.y + xb * cs.x;
            xa = y;
          }
          fa[j] = (float)xa;
          fb[j] = (float)xb;
        }
      }
      const uint32_t w[2][2] = {{pack2(fa[0], fa[1]), pack2(fa[2], fa[3])}, {pack2(fb[0], fb[1]), pack2(fb[2], fb[3])}};
      uint32_t codes[2] = {0u, 0u}, d16[2] = {0u, 0u};
      if constexpr (BITS == 4) quantise(w, lane8, codes, d16);
      if (!on || !place[r].ok) continue;
      const int slot = place[r].slot;
      uint8_t* piece = (is_v ? p.d.v : p.d.k) + place[r].offset + (uint64_t)head_bytes * (it.head & kHeadMask);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int q = l + k * LPH;
        if constexpr (BITS == 16) {
          *reinterpret_cast<uint2*>(piece + (is_v ? v16_quad(slot, q) : k16_quad(slot, q))) = make_uint2(w[k][0], w[k][1]);
        } else {
          *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_quad(slot, q, HD) : k4_quad(slot, q, HD))) = (uint16_t)codes[k];
          if (lane8 == 0)
            *reinterpret_cast<uint16_t*>(piece + (is_v ? v4_scale(slot, q / 8, HD) : k4_scale(slot, q / 8, HD))) = (uint16_t)d16[k];
        }
      }
    }
    if (row0 + RT >= end_row) break;
    // the next turn's angles, beside the others' heads; then this turn's rows, angles and
    // places have been used
    at_row += RT;
    const bool anew = at_row == batch_rows;
    if (anew) {
      at_row = 0;
      __syncthreads();
      look_up(row0 + RT);
    }
    form_angles(row0 + RT, at_row, (turn_no + 1) % BUFS, anew);
    if constexpr (MODE == kStaged) {
      if (!__syncthreads_and(alive)) break;
      if (tid == 0) bring(row0 + 2 * RT, turn_no);
    } else {
      __syncthreads();
    }
  }
  if (MODE == kStaged && !alive)     // after a time-out: copies still in flight land (bounded)
    for (uint32_t i = 0; i < 2; i++)
      if (first_row + (turn_no + i) * RT < end_row)
        mbar_wait(&landed[(turn_no + i) & 1], ((turn_no + i) >> 1) & 1u, p.d.status);
}

// Rows back out of the pages: a warp per row (several where rows are few), a lane per
// 8 elements (two quads that the layouts keep in one 16-byte or 4-byte word).
template <int HD, int BITS>
__global__ void __launch_bounds__(128) k_kvread_paged(const PagedDev d, void* k_out, void* v_out, int out_f32) {
  constexpr int PB = BITS == 16 ? 32 * HD : 9 * HD;
  pdl_wait();
  const uint32_t live = live_rows(d);
  const int per = d.KVH * HD / 8;
  const uint32_t head_bytes = (uint32_t)(d.page / kPieceSlots) * PB;
  for (uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5); row < live; row += gridDim.x * 4) {
    const RowPlace pl = place_row<PB>(d, row);
    const int s = pl.slot;
#pragma unroll
    for (int is_v = 0; is_v < 2; is_v++) {
      void* out = is_v ? v_out : k_out;
      if (!out) continue;
      const uint8_t* pool = (is_v ? d.v : d.k) + pl.offset;
      const size_t at = (size_t)row * d.KVH * HD;
#pragma unroll 4
      for (int e = blockIdx.y * 32 + (threadIdx.x & 31); e < per; e += gridDim.y * 32) {
        const int h = e / (HD / 8), w = e % (HD / 8);
        // the word's two quads: dims 8w.. (f16, and 4-bit keys); the same quad of two blocks (4-bit values)
        const int q0 = BITS == 4 && is_v ? (w >> 3) * 16 + (w & 7) : 2 * w, q1 = BITS == 4 && is_v ? q0 + 8 : 2 * w + 1;
        const uint8_t* piece = pool + (uint64_t)head_bytes * h;
        uint32_t y[4] = {0u, 0u, 0u, 0u};                // the two quads as f16 pairs
        uint16_t sc[2] = {0, 0};
        uint32_t codes = 0x88888888u;
        if (pl.ok) {
          if constexpr (BITS == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(piece + (is_v ? v16_quad(s, q0) : k16_quad(s, q0)));
            y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
          } else {
            codes = *reinterpret_cast<const uint32_t*>(piece + (is_v ? v4_quad(s, q0, HD) : k4_quad(s, q0, HD)));
            sc[0] = *reinterpret_cast<const uint16_t*>(piece + (is_v ? v4_scale(s, q0 / 8, HD) : k4_scale(s, q0 / 8, HD)));
            sc[1] = is_v ? *reinterpret_cast<const uint16_t*>(piece + v4_scale(s, q1 / 8, HD)) : sc[0];
          }
        }
        const size_t o0 = at + (size_t)h * HD + 4 * q0, o1 = at + (size_t)h * HD + 4 * q1;
        if (!out_f32) {
          uint16_t* const to = static_cast<uint16_t*>(out);
          if constexpr (BITS == 16) {
            *reinterpret_cast<uint4*>(to + o0) = make_uint4(y[0], y[1], y[2], y[3]);
          } else {
            // pairs (code j of the first quad, of the second) as f16 n - 8, times (d, d): the
            // product has 15 bits, so its f16 is the value's
            const __half2 d2 = as_h2(sc[0] | (uint32_t)sc[1] << 16);
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
              x[j] = as_u32(__hmul2(__hsub2(as_h2(((codes >> (4 * j)) & 0x000F000Fu) | 0x64006400u), as_h2(0x64086408u)), d2));
            *reinterpret_cast<uint2*>(to + o0) = make_uint2(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410));
            *reinterpret_cast<uint2*>(to + o1) = make_uint2(__byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
          }
          continue;
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if constexpr (BITS == 16) x[j] = h2f((uint16_t)(y[j >> 1] >> (16 * (j & 1))));
          else x[j] = h2f(sc[j >> 2]) * (float)((int)((codes >> (4 * j)) & 15u) - 8);
        }
        *reinterpret_cast<float4*>(static_cast<float*>(out) + o0) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(static_cast<float*>(out) + o1) = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  }
}

// n_rows: of the call whose rows these are; rows of the table past them were not written.
__global__ void k_paged_advance(const PagedDev d, uint32_t* lens) {
  pdl_wait();
  const uint32_t live = live_rows(d);
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= d.nseq) return;
  uint32_t n = 1;
  if (d.rows) {
    const uint32_t r0 = min(d.rows[s], live), r1 = min(d.rows[s + 1], live);
    n = r1 > r0 ? r1 - r0 : 0u;
  }
  lens[s] += n;
}

template <int HD, int MODE>
int launch_prep(e4b_ctx* c, const PrepP& p, int bits, int x_f16, dim3 grid) {
  auto kern = bits == 16 ? (x_f16 ? k_headprep_paged<HD, 16, true, MODE> : k_headprep_paged<HD, 16, false, MODE>)
                         : (x_f16 ? k_headprep_paged<HD, 4, true, MODE> : k_headprep_paged<HD, 4, false, MODE>);
  const size_t items = (size_t)p.rows_per_turn * (p.QH + 2 * p.d.KVH) + 8;    // with the warps' padding
  const size_t smem = (MODE == kStaged ? 2 * kStageBytes : 0) + items * sizeof(Item);
  if (smem > 32 * 1024) E4B_CUDA(c, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  return e4b_launch(c, "headprep_paged", kern, grid, dim3(threads_of<MODE>()), smem, p);
}

template <int HD>
int launch_prep(e4b_ctx* c, PrepP& p, int bits, int x_f16) {
  // few rows: a row per CTA, and a CTA per pass over its heads (latency); the rest in
  // turns of several rows, which share the barriers.  16 query and 4 KV heads of 256, three
  // passes a row, 4 bits: 64 rows 4.0 us by passes and 5.7 us by turns, 128 rows 5.9 and
  // 5.7 us, 390 rows 11.4 and 7.9 us (f16 cache 5.0 and 5.3, 7.0 and 5.3, 18 and 7.4 us);
  // 4 and 1 heads of 128, two passes: 128 rows 3.3 and 4.5 us, 256 rows 4.7 and 4.6 us
  const int ns = threads_of<kFew>() / (HD / 8);
  const int passes = (p.QH + ns - 1) / ns + (2 * p.d.KVH + ns - 1) / ns;
  if ((int64_t)p.d.n_rows * passes <= 2 * c->sm_count)
    return launch_prep<HD, kFew>(c, p, bits, x_f16, dim3(p.d.n_rows, passes));
  const int es = x_f16 ? 2 : 4;
  const int64_t row_bytes = (int64_t)(p.QH + p.d.KVH * (p.keqv ? 1 : 2)) * HD * es;
  const bool staged = p.nparts == 1 && row_bytes <= kStageBytes && reinterpret_cast<uintptr_t>(p.qkv) % 16 == 0 &&
                      p.stride * es % 16 == 0;
  const int64_t fit = staged ? kStageBytes / row_bytes : 2048 / (p.QH + 2 * p.d.KVH);   // (direct: of the item table)
  p.rows_per_turn = fit < 1 ? 1 : (fit < turn_rows(HD) ? (int)fit : turn_rows(HD));
  const int turns = (p.d.n_rows + p.rows_per_turn - 1) / p.rows_per_turn, resident = 2 * c->sm_count;
  const int per_cta = (turns + resident - 1) / resident;
  p.rows_per_cta = per_cta * p.rows_per_turn;
  const dim3 grid((turns + per_cta - 1) / per_cta);
  return staged ? launch_prep<HD, kStaged>(c, p, bits, x_f16, grid) : launch_prep<HD, kDirect>(c, p, bits, x_f16, grid);
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
  p.rows_per_turn = p.rows_per_cta = 1;
  p.stride = row_stride ? row_stride : (int64_t)(QH + kv->kv_heads * (keqv ? 1 : 2)) * HD;
  p.eps = eps;
  p.log2_theta = log2((double)theta);
  return HD == 256 ? launch_prep<256>(c, p, kv->bits, x_f16)
                   : (HD == 128 ? launch_prep<128>(c, p, kv->bits, x_f16) : launch_prep<64>(c, p, kv->bits, x_f16));
}

E4B_API int e4b_kvread_paged(e4b_ctx* c, const e4b_paged_kv* kv, void* k_out, void* v_out, int out_f32, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = kvread_paged_fault(kv, k_out, v_out, n_rows);
  E4B_REQUIRE(c, !fault, "kvread_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  const int HD = kv->head_dim, groups = (n_rows + 3) / 4, most = 16 * c->sm_count;
  // few rows: several warps a row.  4 KV heads of 256, 4 bits: 551 rows 2.6 us by four and
  // 3.9 us by one, 2202 rows 4.8 us either way, 4403 rows 8.1 and 7.1 us
  const int slices = (kv->kv_heads * HD / 8 + 31) / 32;  // of one turn a warp
  const dim3 grid = (int64_t)groups * slices <= most ? dim3(groups, slices) : dim3(groups < most ? groups : most);
  auto kern = kv->bits == 16 ? (HD == 256 ? k_kvread_paged<256, 16> : (HD == 128 ? k_kvread_paged<128, 16> : k_kvread_paged<64, 16>))
                             : (HD == 256 ? k_kvread_paged<256, 4> : (HD == 128 ? k_kvread_paged<128, 4> : k_kvread_paged<64, 4>));
  return e4b_launch(c, "kvread_paged", kern, grid, dim3(128), 0, paged_dev(c, kv, n_rows), k_out, v_out, out_f32 ? 1 : 0);
}

E4B_API int e4b_paged_advance_rows(e4b_ctx* c, const e4b_paged_kv* kv, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = paged_fault(kv);
  if (!fault) fault = paged_rows_fault(kv, n_rows);
  E4B_REQUIRE(c, !fault, "paged_advance: %s", fault);
  return e4b_launch(c, "paged_advance", k_paged_advance, dim3((kv->nseq + 127) / 128), dim3(128), 0,
                    paged_dev(c, kv, n_rows), const_cast<uint32_t*>(kv->lens));
}

E4B_API int e4b_paged_advance(e4b_ctx* c, const e4b_paged_kv* kv) {
  return e4b_paged_advance_rows(c, kv, kv && !kv->rows ? kv->nseq : kMaxRows);
}

}  // extern "C"
