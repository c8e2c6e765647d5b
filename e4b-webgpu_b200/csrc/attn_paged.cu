// Attention of ragged rows over the paged KV cache (f16 or 4-bit pages), with an
// optional sliding window and sinks: split-KV on the tensor cores.
//
// Unit = (sequence, group of query rows, KV head).  A unit's work is the pieces
// of 16 slots that its rows can see; the work of all units, one after the other,
// is cut into equal runs, one per CTA, so ragged lengths and few long sequences
// alike fill the machine.  In a CTA a producer warp streams the run's pieces (one
// bulk copy for the keys, one for the values) through a ring of stages, a lane per
// stage, into the next units too, and the consumer warps take pieces in turn, each
// with its own softmax state; at a unit's end the states are merged in shared memory.
// A unit cut between CTAs leaves partials in the scratch, which the last CTA to
// arrive merges in CTA order (the same bits every time).
//
// Bounds and measurements (B200; a call's bytes at the copy rate, 6.45 TB/s, is its floor;
// replayed calls, one at a time in the stream):
// long caches in 4 bits are bound by the latency of a warp's chain (loads, products,
// shuffles, exponents, products), 717 instructions for a piece of 4.6 KB: three warps a
// scheduler issue in 56 % of the cycles, with neither memory (44 %) nor the tensor pipe
// (20 %) near its limit.  32 sequences of 8000..16000 tokens, 16 query and 4 KV heads of 256,
// 107 us = 3.8 TB/s (floor 63 us; 109 us among calls on other caches).  64 sequences of 1035
// tokens take 30.2 us (floor 12 us) and one of 131001 tokens and 2 KV heads 30.8 us (11.7
// us): set-up, first pieces, merges and the join of the parts, 6 to 8 us one after the other,
// come beside it; one token behind 551 takes 10.8 us of them alone.  f16, 64 windows of 1024:
// 29.2 us (15.3 us).  Several rows a sequence (8 x 1..64 rows behind 300..4000 tokens, windows
// of 1024): 81 us, bound by the latency of the products on 8 warps (tensor pipe 20 % busy),
// each piece decoded once for 16 columns; 16 prompts of 1..1000 rows 1440 us.
//
// Products, per piece and 8 MMA columns (m16n8k16, f32 accumulators):
//   S[slot][col]  = K[slot][:] . q[:][col]      A = keys,   B = q
//   O[dim][col]  += V[slot][dim] p[slot][col]   A = values, B = p
// The 8 columns are 4 query heads of one row as f16 hi and lo parts (columns 0-3,
// 4-7), so q and p carry f32 precision at the MMA cost of one f16 pass.
// 4-bit keys and values: A holds n - 8, two instructions per pair of codes; a key
// block's scale multiplies its dot product in f32.  (Codes n as f16 subnormals, n * 2^-24
// by one AND, with the -8 taken off by one more MMA, take 4 % less time on long caches, but
// the MMA aligns a subnormal by its exponent field and sums larger numbers: f32 outputs
// were 0.7e-6 to 1.8e-6 off in place of 0.1e-6 to 0.8e-6.)  A value block's scale
// multiplies p, again as hi + lo.  To keep the lo parts clear of f16's subnormals p is
// lifted by 2^8, and a block of 32 dims whose visible scales have all been below 2^-7
// (2^-14) is held times 2^8 (2^15): a product is off by 2^-20 of itself and 2^-22 of the
// largest p times the block's largest value at most (2^-16 of that where scales of 2^7 or
// more stand beside such a block).
#include <type_traits>

#include "paged.cuh"
#include "stream.cuh"

namespace {
using namespace e4b;

constexpr int kMaxCtas = 320;
constexpr int kGroup = 12;           // CTAs whose parts are merged first
constexpr int kMostParts = 9;        // CTAs that share a unit evenly (10 to 12: merging them costs more than equal runs, 17.3 us against 15.1 us)
constexpr uint32_t kLowCodes = 0x000F000Fu, kHighCodes = 0x00F000F0u;
// p is held as p * 2^8 relative to a maximum that may lag behind the largest score by
// 2^6, so a rescaling of O is rare and p * d stays below 2^15 for scales d below 2.
// A visible scale of 2 or more ends the lag (d below 2^7), one of 2^7 or more leaves a
// lift of 2^2 (d up to f16's largest, 2^13).
constexpr float kLift = 8.f, kSlack = 6.f, kLowLift = 2.f;
// Scale of the values of block b in O and in the products: state c of two bits a block.
constexpr uint32_t kAllTiny = 0xAAAAAAAAu;               // nothing but zeros seen yet
E4B_DEV uint32_t scale_state(uint32_t states, int b) { return (states >> (2 * b)) & 3u; }
E4B_DEV int scale_up(uint32_t c) { return c == 2 ? 15 : (c == 1 ? 8 : 0); }
E4B_DEV uint32_t scale_half2(uint32_t c) { return c == 2 ? 0x78007800u : (c == 1 ? 0x5C005C00u : 0x3C003C00u); }
E4B_DEV float scale_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

struct AttnP {
  PagedDev d;
  const float* q;
  uint16_t* out_h;
  float* out_f;
  float* lse;
  uint32_t* arrived;                 // [3][kMaxCtas], zero at rest: by a unit's first CTA, a later group's first, for the groups
  float* parts;                      // [2 * CTAs]: [columns][HD] of O, then (max, sum) per column
  int QH, G, xfo;
  uint32_t window, sinks;
  float scale;
};

// kNarrow, kWide: a row per unit of up to 4 heads, one n-tile whose 8 MMA columns are
// the heads' hi parts and lo parts.  kRows: NT tiles a warp whose 8 columns are 8 (row,
// head) pairs, hi and lo in turn: the decoded keys and values, the softmax and the
// scaled p are then shared by twice the columns, for prompts' and speculated rows.
enum { kNarrow, kWide, kRows };
constexpr int kConsumerRegs = 224, kProducerRegs = 56;

template <int BITS, int HD, int MODE>
struct Shape {
  static constexpr int NB = HD / 32;
  static constexpr int PB = BITS == 16 ? 32 * HD : 9 * HD;
  static constexpr int STAGE = 2 * PB;
  static constexpr int NT = MODE == kRows && !(BITS == 16 && HD == 256) ? 2 : 1;
  static constexpr int LC = NT * (MODE == kRows ? 8 : 4);               // columns of a warp
  // consumer warps: a one-row warp needs 168 registers, so 12 warps fit an SM: one CTA
  // of 11 + 1 (kWide), or two of 5 + 1, where one's set-up and merges pass beside the
  // other's pieces; a kRows warp needs more, which the producer's warpgroup gives up
  // (setmaxnreg): 8 * 32 * 224 + 4 * 32 * 56 = 384 * 168, what the block was launched with
  static constexpr int PER_SM = MODE == kNarrow ? 2 : 1, MAX_CTAS = PER_SM * kMaxCtas / 2;
  static constexpr int W = MODE == kRows ? 8 : (MODE == kNarrow ? 5 : (BITS == 16 && HD == 256 ? 10 : 11));
  // ring depth: a multiple of W, so a stage's uses within a unit belong to the same
  // warps (a warp then never waits for a phase before the stage's last one is done)
  static constexpr int S = W * (BITS == 16 ? (HD == 256 ? 1 : (HD == 128 ? 2 : 4)) :
                                MODE == kRows ? (HD == 256 ? 2 : (HD == 128 ? 4 : 8)) : (HD == 256 ? 3 : (HD == 128 ? 5 : 8)));
  // what a unit costs beside its pieces (q, the merge, the outputs), in pieces.  Half of it
  // and twice it (us, as is in the middle): 48 ragged sequences, 4 bits 15.3 / 13.3 / 18.8,
  // f16 21.2 / 15.6 / 12.9; 8 x 1..64 rows 91 / 81 / 80; 300 of 1..400 tokens 16.2 / 17.3 /
  // 17.2, f16 19.1 / 15.3 / 16.9; 32 of 8000..16000 tokens 108 / 107 / 105
  static constexpr int U = MODE == kRows ? 16 : (BITS == 16 ? (HD == 256 ? 6 : (HD == 128 ? 8 : 12)) : (HD == 256 ? 12 : 16));
  static constexpr int LN = S <= 32 ? S : (W == 11 ? 11 : (W == 5 ? (S == 40 ? 20 : 25) : 32));   // producer lanes; S is a multiple
  static constexpr int THREADS = MODE == kRows ? 384 : 32 * (W + 1), CT = 32 * W;
  static constexpr int COLS = LC;                                       // columns (row, head) of a unit
  static constexpr size_t PART = (size_t)COLS * (HD + 2);               // floats of a partial
  static constexpr int TILES = NT, QPARTS = MODE == kRows ? 2 : 1;  // n-tiles of a unit; fragments of a tile
  static constexpr size_t RING = (size_t)S * STAGE;
  // q fragments [TILES][NB][QPARTS][32] while a unit's pieces pass, then the warps' O [W][LC][HD]
  static constexpr size_t MERGE = (size_t)W * LC * HD * 4;
  static constexpr size_t SMEM = RING + MERGE;
  static_assert((size_t)TILES * NB * QPARTS * 32 * 16 <= MERGE, "q fragments fit the merge buffer");
};

// Rows and heads of a unit in n-tiles.
template <int NT, int MODE>
struct Rows {
  int slots;                         // columns of a row in a tile: its heads, up to a power of two (one row: 4)
  E4B_DEV explicit Rows(int G) : slots(MODE != kRows ? 4 : (G > 4 ? 8 : (G > 2 ? 4 : G))) {}
  E4B_DEV int per_tile() const { return MODE == kRows ? 8 / slots : 1; }
  E4B_DEV uint32_t per_unit() const { return NT * per_tile(); }
};

// One sequence's rows of the call, the pieces they see and what they cost.
struct SeqWork {
  uint32_t p0, nq;                   // first row's position, rows
  PieceRange range;
  uint32_t units;                    // groups of rows times KV heads
  uint32_t parts;                    // CTAs that share each unit evenly (kRows); 0: units are cut where the runs end
  uint64_t cost;                     // U + pieces (or the parts), for each unit
};
template <int NT, int U, int MODE>
E4B_DEV SeqWork seq_work(const AttnP& p, int s) {
  SeqWork w;
  uint32_t r0 = (uint32_t)s, r1 = r0 + 1;
  if (p.d.rows) r0 = p.d.rows[s], r1 = min(p.d.rows[s + 1], (uint32_t)p.d.n_rows);
  w.nq = r1 > r0 ? r1 - r0 : 0u;
  const uint32_t len = p.d.lens[s];
  w.p0 = min(len, 0xfffffff0u - w.nq);
  w.units = w.parts = 0;
  w.cost = 0;
  if (w.nq) {
    // positions past the table are clamped: no such slot is visible
    if ((uint64_t)len + w.nq > p.d.cap) set_status(p.d.status, E4B_ST_BADINDEX);
    const uint32_t p1 = min(w.p0 + w.nq - 1, p.d.cap - 1), per = Rows<NT, MODE>(p.G).per_unit();
    w.range = piece_range(min(w.p0, p1), p1, p.window, p.sinks);
    w.units = p.d.KVH * (MODE == kRows ? (w.nq + per - 1) / per : 1u);
    w.cost = (uint64_t)(U + w.range.count) * w.units;
  }
  return w;
}

E4B_DEV uint64_t udiv(uint64_t a, uint64_t b) {
  return ((a | b) >> 32) == 0 ? (uint64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Walks a CTA's run [g, end) of the work, unit by unit.
template <int NT, int U, int MODE>
struct Walk {
  uint64_t g, end, base;             // base: where the current sequence's work begins
  int s;
  SeqWork w;
  uint64_t unit0, unit1;             // the unit's work, the first U of it its set-up (or its parts)
  uint32_t kvh, nrows;               // KV head, rows
  uint32_t pmin, pmax;               // positions of the unit's rows
  PieceSpan span;                    // this CTA's pieces of it
  E4B_DEV bool next(const AttnP& p) {
    if (g >= end) return false;
    while (g >= base + w.cost) {
      base += w.cost;
      if (++s >= p.d.nseq) {         // the lengths changed under the call
        g = end;
        return false;
      }
      w = seq_work<NT, U, MODE>(p, s);
    }
    const uint32_t per = Rows<NT, MODE>(p.G).per_unit(), KVH = p.d.KVH, np = w.range.count;
    const bool even = MODE == kRows && w.parts;
    const uint32_t length = even ? w.parts : np + U;
    const uint64_t unit = udiv(g - base, length);
    const uint32_t group = MODE == kRows ? (uint32_t)udiv(unit, KVH) : 0u;
    kvh = (uint32_t)unit - group * KVH;
    unit0 = base + unit * length;
    unit1 = unit0 + length;
    nrows = min(per, w.nq - group * per);
    pmin = w.p0 + group * per;
    pmax = pmin + nrows - 1;
    const uint64_t stop = min(unit1, end);
    const uint32_t o0 = (uint32_t)(g - unit0), o1 = (uint32_t)(stop - unit0);
    const uint32_t p1 = min(pmax, p.d.cap - 1);
    const auto piece_of = [&](uint32_t o) { return even ? o * np / length : (o <= U ? 0u : o - U); };
    span = piece_span(w.range, piece_of(o0), piece_of(o1), min(pmin, p1), p1, p.window, p.sinks);
    g = stop;
    return true;
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
// a * b - c
E4B_DEV uint32_t hfms2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b),
                            __hneg2(*reinterpret_cast<__half2*>(&c)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
E4B_DEV uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// D = A B, from a zero accumulator.
E4B_DEV void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The pair of codes in bits 0..3 (4..7) of each half, as f16 n - 8: OR-ed under the
// exponent of 1024 they read 1024 + n (1024 + 16 n), from which one instruction
// takes 1032 (and divides by 16).
E4B_DEV uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {    // one instruction: (x & mask) | bits
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}
E4B_DEV uint32_t low_codes(uint32_t x) { return hsub2(and_or(x, kLowCodes, 0x64006400u), 0x64086408u); }
E4B_DEV uint32_t high_codes(uint32_t x) {
  return hfma2(and_or(x, kHighCodes, 0x64006400u), 0x2C002C00u, 0xD480D480u);   // / 16, - 72
}
E4B_DEV bool finite2(uint32_t x) { return (x & 0x7C00u) != 0x7C00u && (x & 0x7C000000u) != 0x7C000000u; }
E4B_DEV float half_of(uint32_t x, int upper) {
  const __half2 h = *reinterpret_cast<const __half2*>(&x);
  return upper ? __high2float(h) : __low2float(h);
}
E4B_DEV uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
E4B_DEV uint4 lds128_once(const uint8_t* p) {            // a load that is not kept for later uses of the address
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(p)));
  return v;
}
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
E4B_DEV uint32_t inc_acq_rel(uint32_t* at, uint32_t last) {
  uint32_t was;
  asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(was) : "l"(at), "r"(last) : "memory");
  return was;
}
__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, uint32_t* status) {
  return mbar_wait(b, parity, status);
}

template <int BITS, int HD, int MODE>
__global__ void __launch_bounds__(Shape<BITS, HD, MODE>::THREADS, Shape<BITS, HD, MODE>::PER_SM) k_attn_paged(const AttnP p) {
  using Sh = Shape<BITS, HD, MODE>;
  constexpr int NB = Sh::NB, PB = Sh::PB, W = Sh::W, S = Sh::S, LN = Sh::LN, CT = Sh::CT, NT = Sh::NT, LC = Sh::LC;
  constexpr int TC = LC / NT, QP = Sh::QPARTS;           // columns of a tile
  static_assert(S % W == 0 && S % LN == 0 && LN <= 32 && S <= Sh::THREADS, "ring");
  constexpr int OT = HD / 16;        // m16 tiles of O
  constexpr int U = Sh::U;
  using Unit = Walk<NT, U, MODE>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem + Sh::RING);            // [W][LC][HD]
  uint4* qfrag = reinterpret_cast<uint4*>(smem + Sh::RING);            // [TILES][NB][QP][32]
  __shared__ uint64_t landed[S], freed[S];
  __shared__ int usable[S];
  __shared__ uint64_t warp_sum_[Sh::THREADS / 32];
  __shared__ uint32_t warp_units[Sh::THREADS / 32], warp_longest[Sh::THREADS / 32];
  __shared__ uint2 warp_parts[Sh::THREADS / 32];
  __shared__ float qfac[Sh::TILES * TC];
  __shared__ float ml[W * LC * 2];
  __shared__ int last_one, more_units;
  __shared__ struct { uint64_t at, base; int s; SeqWork w; } start;
  __shared__ Unit unit;
  __shared__ uint32_t unit_c0, unit_c1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  if (tid < S) {
    mbar_init(&landed[tid], 1);
    mbar_init(&freed[tid], 1);
  }
  if (tid == 0) fence_barrier_init();
  pdl_wait();

  // ---- the run of this CTA: the work of all units, cut evenly
  uint64_t mine = 0;
  uint32_t units = 0, longest = 0;
  uint32_t parts1 = 0, parts2 = 0;   // CTAs where each takes W, 2 W pieces of a unit (sums past the CTAs do not matter)
  SeqWork own;                       // of the thread's first sequence
  const int per = (p.d.nseq + Sh::THREADS - 1) / Sh::THREADS;
  for (int s = tid * per; s < min(p.d.nseq, (tid + 1) * per); s++) {
    const SeqWork w = seq_work<NT, U, MODE>(p, s);
    if (s == tid * per) own = w;
    mine += w.cost;
    units += w.units;
    if (w.units) longest = max(longest, w.range.count + U);
    if (MODE == kRows && w.units) {
      parts1 += (uint32_t)min((uint64_t)w.units * ((w.range.count - 1) / W + 1), (uint64_t)0xffff);
      parts2 += (uint32_t)min((uint64_t)w.units * ((w.range.count - 1) / (2 * W) + 1), (uint64_t)0xffff);
    }
  }
  if (blockIdx.x == 0) live_rows(p.d);                   // records a row count past n_rows
  uint64_t upto = mine;                                  // inclusive sum over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  units = __reduce_add_sync(0xffffffffu, min(units, 0xffffffu));
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (MODE == kRows) parts1 = __reduce_add_sync(0xffffffffu, parts1), parts2 = __reduce_add_sync(0xffffffffu, parts2);
  if (lane == 31) {
    warp_sum_[warp] = upto, warp_units[warp] = units, warp_longest[warp] = longest;
    if (MODE == kRows) warp_parts[warp] = make_uint2(parts1, parts2);
  }
  __syncthreads();
  uint64_t before = 0, T = 0;
  units = parts1 = parts2 = 0;
#pragma unroll
  for (int i = 0; i < Sh::THREADS / 32; i++) {
    if (i < warp) before += warp_sum_[i];
    T += warp_sum_[i];
    units += warp_units[i];
    if (MODE == kRows) parts1 += warp_parts[i].x, parts2 += warp_parts[i].y;
    longest = max(longest, warp_longest[i]);
  }
  upto += before;
  // Runs of 2 U at least, or a unit's length (no two on a CTA while others idle); an end
  // that falls within U of a unit's start or end moves there, so short units stay whole
  // and no fragment is shorter than U.
  // Units are not cut at all where the longest is at most 3 U, what cutting costs, above a
  // CTA's even share (f16, bound by memory rather than by the longest CTA: a third of it).
  // 64 sequences of 1035 tokens and 4 KV heads of 256, whole and cut: 30.2 and 35.8 us, of
  // 8000 tokens 173 and 162 us, of 1000..1100 31.4 and 36.9 us; f16, 1035 tokens 46.3 and
  // 52.3 us, 4000 tokens 154 and 164 us.  Under a rows table a run's end then moves to the
  // nearer end of a unit, which is the right one while the units together are less than half
  // the longest short of it each.
  // Where the machine has a CTA for every W (or 2 W) pieces of a kRows unit, that many share
  // it evenly, a turn (or two) of their warps, and none takes from two units (3 sequences of
  // 64 query and 8 KV heads of 128, 1024-token windows: 20.0 us -> 14.7 us).  With one row a
  // unit the longer set-up takes back what it gives: one token behind 551 10.6 -> 10.2 us,
  // 64 behind 1034 28.4 -> 29.1 us, one behind 131000 28.5 -> 29.0 us.
  const uint64_t most_over = BITS == 16 ? max(3u * U, longest / 3) : 3u * U;
  const bool uncut = units <= gridDim.x && (uint64_t)longest * gridDim.x <= T + most_over * gridDim.x &&
                     (!p.d.rows || 2 * ((uint64_t)longest * units - T) < longest);
  const uint64_t want = max(udiv(T, 2 * U), min((uint64_t)units, udiv(T, U)));
  uint32_t C = T == 0 ? 0u : (uncut ? units : (want < 1 ? 1u : (want < gridDim.x ? (uint32_t)want : gridDim.x)));
  bool even = false;
  if constexpr (MODE == kRows) {
    const uint32_t most = longest - min(longest, (uint32_t)U), quota = parts1 <= gridDim.x ? W : 2 * W;
    even = min(parts1, parts2) <= gridDim.x && most > W && most <= kMostParts * quota && per == 1;
    if (even) {                      // a thread's one sequence measured in CTAs: the sums once more
      if (mine) {
        own.parts = (own.range.count - 1) / quota + 1;
        mine = own.cost = own.parts * own.units;
      }
      uint32_t sum = (uint32_t)mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      __syncthreads();
      if (lane == 31) warp_sum_[warp] = sum;
      __syncthreads();
      upto = sum;
      T = 0;
#pragma unroll
      for (int i = 0; i < Sh::THREADS / 32; i++) {
        if (i < warp) upto += warp_sum_[i];
        T += warp_sum_[i];
      }
      C = (uint32_t)T;
    }
  }
  const auto reach_of = [](uint64_t length, bool even, bool uncut) {
    return MODE == kRows && even ? 1u : (uncut ? (uint32_t)length / 2 + 1 : (uint32_t)U);
  };
  const uint32_t cta = blockIdx.x;
  if (cta >= C) return;
  __shared__ uint64_t run_end, work_all;                 // (read back where they are needed: the loops need the registers)
  __shared__ uint32_t work_ctas;
  __shared__ bool work_uncut;
  if (uncut && !even && !p.d.rows) { // every sequence has KVH units: CTA c takes unit c (work counted from its sequence)
    if (tid == 0) {
      const int s = cta / p.d.KVH;
      const SeqWork w = seq_work<NT, U, MODE>(p, s);
      const uint64_t length = w.range.count + U;
      start.at = (cta - s * p.d.KVH) * length, start.base = 0, start.s = s, start.w = w;
      run_end = start.at + length;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {      // an end of the run, formed by the thread whose sequences hold it
      const uint64_t raw = udiv(T * (cta + i), C);
      if (upto - mine <= raw && raw < upto) {
        uint64_t base = upto - mine;
        int s = tid * per;
        SeqWork w = own;
        while (raw >= base + w.cost && s + 1 < p.d.nseq) {
          base += w.cost;
          w = seq_work<NT, U, MODE>(p, ++s);
        }
        const uint64_t length = MODE == kRows && even ? w.parts : w.range.count + U, unit0 = base + udiv(raw - base, length) * length, unit1 = unit0 + length;
        const uint64_t reach = reach_of(length, even, uncut), at = raw - unit0 < reach ? unit0 : (unit1 - raw < reach ? unit1 : raw);
        if (i == 1) run_end = at;
        else start.at = at, start.base = base, start.s = s, start.w = w;
      } else if (i == 1 && raw == T && tid == 0) {
        run_end = T;
      }
    }
  }
  if (tid == 0) work_all = T, work_ctas = C, work_uncut = uncut;
  __syncthreads();
  Unit u;
  u.g = start.at;
  u.end = run_end;
  u.base = start.base;
  u.s = start.s;
  u.w = start.w;

  if (warp >= W) {
    // ---- producer: lane i brings the CTA's pieces i, i + LN, .., piece j into stage j % S
    if constexpr (MODE == kRows) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    if (warp > W || lane >= LN) return;
    constexpr uint32_t kLanes = LN == 32 ? 0xffffffffu : (1u << (LN & 31)) - 1u;
    uint32_t j = lane, seg0 = 0, seg1 = 0, page = 0, piece = 0, in_page = 0;
    bool more = true;
    const auto find = [&]() {        // piece j of the run and its page
      while (j >= seg1) {
        if (!u.next(p)) {
          more = false;
          return;
        }
        seg0 = seg1;
        seg1 += u.span.count;
      }
      piece = u.span.at(j - seg0);
      const uint32_t slot = piece * kPieceSlots, nth = slot / (uint32_t)p.d.page;
      in_page = slot - nth * (uint32_t)p.d.page;
      page = slot < p.d.cap ? p.d.pages[(size_t)u.s * p.d.max_pages + nth] : 0xffffffffu;
    };
    find();
    uint64_t since = 0;
    uint32_t idle = 0;
    while (__any_sync(kLanes, more)) {
      const uint32_t st = j % S;
      const bool ready = more && (j < (uint32_t)S || mbar_try_wait(&freed[st], ((j / S) & 1u) ^ 1u));
      if (ready) {
        const bool ok = page < p.d.n_pages;
        usable[st] = ok;
        if (ok) {
          const uint64_t off = piece_offset(page, u.kvh, (int)in_page, p.d.KVH, p.d.page, PB);
          uint8_t* dst = ring + (size_t)st * Sh::STAGE;
          mbar_expect_tx(&landed[st], 2 * PB);
          bulk_g2s(dst, p.d.k + off, PB, &landed[st]);
          bulk_g2s(dst + PB, p.d.v + off, PB, &landed[st]);
        } else {
          set_status(p.d.status, E4B_ST_BADINDEX);
          mbar_arrive(&landed[st]);
        }
        j += LN;
        find();
      }
      if (__any_sync(kLanes, ready)) {
        idle = 0;
      } else {
        __nanosleep(200);
        if (idle == 0) since = globaltimer_ns();
        if ((++idle & 255u) == 0 && __any_sync(kLanes, globaltimer_ns() - since > 2000000000ull)) {
          set_status(p.d.status, E4B_ST_TIMEOUT);        // the consumers gave up
          break;
        }
      }
    }
    // nothing of this CTA is in flight when it ends
    for (int k = 0; k < S / LN && j >= (uint32_t)(lane + LN); k++) {
      j -= LN;
      mbar_wait(&landed[j % S], (j / S) & 1u, p.d.status);
    }
    return;
  }

  if constexpr (MODE == kRows) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  const auto consumers = []() { asm volatile("bar.sync 1, %0;" ::"n"(CT) : "memory"); };
  uint32_t j0 = 0;                   // the CTA's pieces before the unit's
  bool alive = true;                 // no wait has run out
  float O[NT][OT][4];

  // the unit in hand lives in shared memory: the loop over its pieces needs the registers
  const auto next_unit = [&](Unit& v) {                  // thread 0
    more_units = v.next(p);
    unit = v;
  };
  if (tid == 0) next_unit(u);
  consumers();
  while (more_units) {
    const uint32_t row0 = (p.d.rows ? p.d.rows[unit.s] : (uint32_t)unit.s) + (unit.pmin - unit.w.p0);
    const Rows<NT, MODE> rows(p.G);
    const int slots = rows.slots, per_tile = rows.per_tile();
    // column c of the unit -> row of the unit, head
    const auto col_row = [&](int c) { return c / TC * per_tile + c % TC / slots; };
    const auto col_head = [&](int c) { return c % TC % slots; };
    const auto col_live = [&](int c) { return col_head(c) < p.G && (uint32_t)col_row(c) < unit.nrows; };
    constexpr int cols = LC;

    // ---- q as B fragments: HD/8 lanes take a column, a lane the 8 dims of one (block, t)
    {
      constexpr int LPC = HD / 8;
      const int sub = tid / LPC, l = tid % LPC, blk = l >> 2, tt = l & 3;
      constexpr int AHEAD = MODE == kRows ? (Sh::COLS * LPC + CT - 1) / CT : 1;   // columns of a lane group, loaded together
      float4 xa[AHEAD], xb[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; n++) {
        const int c = sub + n * (CT / LPC);
        const bool on = c < cols && col_live(c);
        const float4* src = reinterpret_cast<const float4*>(
            p.q + ((size_t)(row0 + (on ? col_row(c) : 0)) * p.QH + unit.kvh * p.G + (on ? col_head(c) : 0)) * HD + 8 * l);
        xa[n] = on ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f);
        xb[n] = on ? src[1] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int n = 0; n < AHEAD; n++) {
        const int c = sub + n * (CT / LPC), tile = c / TC, cc = c % TC;
        const float x[8] = {xa[n].x, xa[n].y, xa[n].z, xa[n].w, xb[n].x, xb[n].y, xb[n].z, xb[n].w};
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // a power of two that brings the largest |q| into [2^14, 2^15): f16 hi + lo then
        // carry every element to 2^-22 of the largest
        const int e = (int)(__float_as_uint(m) >> 23);   // biased exponent; 0: zero or subnormal, 255: inf
        const int up = e == 255 ? 0 : min(14 + 127 - e, 120);
        const float f = __uint_as_float((uint32_t)(up + 127) << 23);
        float hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float v = x[i] * f;
          hi[i] = __half2float(__float2half_rn(v));
          lo[i] = __half2float(__float2half_rn(v - hi[i]));
        }
        uint4 fh, fl;
        if constexpr (BITS == 4) {
          fh = make_uint4(pack2(hi[0], hi[4]), pack2(hi[2], hi[6]), pack2(hi[1], hi[5]), pack2(hi[3], hi[7]));
          fl = make_uint4(pack2(lo[0], lo[4]), pack2(lo[2], lo[6]), pack2(lo[1], lo[5]), pack2(lo[3], lo[7]));
        } else {
          fh = make_uint4(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]), pack2(hi[4], hi[5]), pack2(hi[6], hi[7]));
          fl = make_uint4(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(lo[4], lo[5]), pack2(lo[6], lo[7]));
        }
        if (c < cols) {
          // the lo part: the tile's second fragment, or its columns 4-7
          uint4* at = qfrag + ((size_t)(tile * NB + blk) * QP) * 32 + cc * 4 + tt;
          at[0] = fh;
          at[MODE == kRows ? 32 : 16] = fl;
          if (l == 0)
            qfac[c] = p.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - up) << 23);
        }
      }
    }
    consumers();
    float top[NT][2], lsum[NT][2], fac[NT][2], lift = kLift, slack = kSlack;  // reference score; sum of p; score factor
    uint32_t ups = kAllTiny & ((1ull << (2 * NB)) - 1); // the blocks' scales
    uint32_t pos0[NT], pos1[NT], pos[NT][2], posg[NT];   // of the tile's first and last row, the lane's score columns, its p column
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int tile = nt;
      const auto position = [&](int row) { return min(unit.pmin + row, unit.pmax); };
      pos0[nt] = position(tile * per_tile);
      pos1[nt] = position(tile * per_tile + per_tile - 1);
      posg[nt] = position(col_row(tile * TC + g % TC));
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int c = tile * TC + (MODE == kRows ? 2 * t : 2 * (t & 1)) + i;
        pos[nt][i] = position(col_row(c));
        top[nt][i] = -INFINITY;
        lsum[nt][i] = 0.f;
        fac[nt][i] = qfac[c];
      }
#pragma unroll
      for (int i = 0; i < OT; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) O[nt][i][k] = 0.f;
    }
    const int live_tiles = NT > 1 && (uint32_t)((NT - 1) * per_tile) < unit.nrows ? NT : 1;
    const uint4* qf = qfrag + lane;

    const PieceSpan span = unit.span;
    const uint32_t turn = j0 % W;    // warp j % W takes the CTA's piece j
    bool fresh = true;               // O is zero
    const uint32_t i0 = (uint32_t)warp >= turn ? warp - turn : warp + W - turn;
    uint32_t st = (j0 + i0) % S, phase = (j0 + i0) / S & 1u;
    // a piece's work for the warp's first N tiles (the others hold no row)
    const auto work = [&](auto tiles, const uint8_t* kp, const uint8_t* vp, uint32_t t0, bool here) {
      constexpr int N = decltype(tiles)::value;
      // ---- scores
      float s[N][4];
#pragma unroll
      for (int nt = 0; nt < N; nt++)
#pragma unroll
        for (int k = 0; k < 4; k++) s[nt][k] = 0.f;
      if (BITS == 4) {
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
          for (int q = 0; q < RUN; q++) {
            const int b = r * RUN + q;
            const uint32_t sa = wa[q] >> 8, sb = wb[q] >> 8;
            const float d0 = half_of(da[b / 2], b & 1), d1 = half_of(db[b / 2], b & 1);
            const uint32_t al[4] = {low_codes(wa[q]), low_codes(wb[q]), low_codes(sa), low_codes(sb)};
            const uint32_t ah[4] = {high_codes(wa[q]), high_codes(wb[q]), high_codes(sa), high_codes(sb)};
#pragma unroll
            for (int nt = 0; nt < N; nt++) {
              const uint4 qb = qf[(nt * NB + b) * QP * 32];
              float acc[4];
              mma16816_zero(acc, al[0], al[1], al[2], al[3], qb.x, qb.y);
              mma16816(acc, ah[0], ah[1], ah[2], ah[3], qb.z, qb.w);
              if (MODE == kRows) {
                const uint4 ql = qf[((nt * NB + b) * QP + 1) * 32];
                mma16816(acc, al[0], al[1], al[2], al[3], ql.x, ql.y);
                mma16816(acc, ah[0], ah[1], ah[2], ah[3], ql.z, ql.w);
              }
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
          for (int nt = 0; nt < N; nt++) {
            const uint4 qb = qf[(nt * NB + b) * QP * 32];
            float acc[4];
            mma16816_zero(acc, wa.x, wb.x, wa.y, wb.y, qb.x, qb.y);
            mma16816(acc, wa.z, wb.z, wa.w, wb.w, qb.z, qb.w);
            if (MODE == kRows) {
              const uint4 ql = qf[((nt * NB + b) * QP + 1) * 32];
              mma16816(acc, wa.x, wb.x, wa.y, wb.y, ql.x, ql.y);
              mma16816(acc, wa.z, wb.z, wa.w, wb.w, ql.z, ql.w);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) s[nt][k] += acc[k];
          }
        }
      }

      // ---- the slots (2t, 2t+1) and (2t+8, 2t+9) that the lane's p column sees (keep: masks of
      // halves), and that some row of the warp sees
      bool full[N], masked = false;
      uint32_t keep[N][2], seen[2] = {0u, 0u};
#pragma unroll
      for (int nt = 0; nt < N; nt++) {
        full[nt] = here && t0 + kPieceSlots - 1 <= pos0[nt] &&
                   (p.window == 0 || pos1[nt] - t0 < p.window || t0 + kPieceSlots <= p.sinks);
        keep[nt][0] = keep[nt][1] = full[nt] ? 0xffffffffu : 0u;
        if (!full[nt]) {
          masked = true;
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (here && slot_visible(t0 + 2 * t + (k & 1) + 8 * (k >> 1), posg[nt], p.window, p.sinks))
              keep[nt][k >> 1] |= 0xffffu << (16 * (k & 1));
        }
        seen[0] |= keep[nt][0], seen[1] |= keep[nt][1];
      }
      if (MODE == kRows && masked) {                     // over the columns' rows
#pragma unroll
        for (int k = 0; k < 2; k++) {
          seen[k] |= __shfl_xor_sync(0xffffffffu, seen[k], 4);
          seen[k] |= __shfl_xor_sync(0xffffffffu, seen[k], 8);
          seen[k] |= __shfl_xor_sync(0xffffffffu, seen[k], 16);
        }
      }

      // ---- the value scales that some row sees: what p's lift and the blocks' scales have to be
      if (BITS == 4) {
        uint32_t any = 0;
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
          const uint4 d4 = lds128_once(vp + (t * NB + b) * 8);
          any |= ((d4.x | d4.z) & seen[0]) | ((d4.y | d4.w) & seen[1]);
        }
        const bool big = __any_sync(0xffffffffu, (any & 0x40004000u) != 0) && lift == kLift;   // 2 or more
        if (__builtin_expect(big || ups != 0, 0)) {
          uint32_t sizes = 0;        // two bits a block: a scale >= 2^-14, one >= 2^-7; the top one: any >= 2^7
#pragma unroll
          for (int b = 0; b < NB; b++) {
            const uint2 d = *reinterpret_cast<const uint2*>(vp + (t * NB + b) * 8);
            const uint32_t w0 = d.x & seen[0], w1 = d.y & seen[1], w = w0 | w1;
            if (w & 0x7C007C00u) sizes |= 1u << (2 * b);
            if (w & 0x60006000u) sizes |= 2u << (2 * b);
            if (big && (w & 0x40004000u)) {
              const __half2 m = __hmax2(__habs2(*reinterpret_cast<const __half2*>(&w0)), __habs2(*reinterpret_cast<const __half2*>(&w1)));
              if (!(__low2float(m) < 128.f && __high2float(m) < 128.f)) sizes |= 1u << 31;
            }
          }
          sizes = __reduce_or_sync(0xffffffffu, sizes);
          int fall = 0;              // of the lift
          if (big) slack = 0.f;
          if (sizes >> 31) {
            fall = (int)(kLift - kLowLift);
            lift = kLowLift;
          }
          const uint32_t were = ups;
#pragma unroll
          for (int b = 0; b < NB; b++) {                 // a block's scale only ever falls, to 1 in the end
            const uint32_t was = scale_state(were, b), is = min(was, 2u - min(scale_state(sizes, b), 2u));
            ups ^= (was ^ is) << (2 * b);
          }
          if (!fresh && (fall || ups != were)) {
#pragma unroll
            for (int nt = 0; nt < N; nt++) {
              lsum[nt][0] *= scale_pow2(-fall), lsum[nt][1] *= scale_pow2(-fall);
#pragma unroll
              for (int b = 0; b < NB; b++) {
                const float f = scale_pow2(scale_up(scale_state(ups, b)) - scale_up(scale_state(were, b)) - fall);
#pragma unroll
                for (int k = 0; k < 4; k++) O[nt][2 * b][k] *= f, O[nt][2 * b + 1][k] *= f;
              }
            }
          }
        }
      }

      // ---- softmax state and p as B fragments
      uint32_t ph[N][2], pl[N][2];                    // slots (2t, 2t+1), (2t+8, 2t+9)
#pragma unroll
      for (int nt = 0; nt < N; nt++) {
        float v[4];
        bool see[4] = {true, true, true, true};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if (MODE != kRows) s[nt][k] += __shfl_xor_sync(0xffffffffu, s[nt][k], 2);     // hi + lo columns
          v[k] = s[nt][k] * fac[nt][k & 1];
        }
        if (!full[nt]) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            see[k] = here && slot_visible(t0 + g + 8 * (k >> 1), pos[nt][k & 1], p.window, p.sinks);
            if (!see[k]) v[k] = -INFINITY;
          }
        }
        const bool grow = fmaxf(v[0], v[2]) > top[nt][0] + slack || fmaxf(v[1], v[3]) > top[nt][1] + slack;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float n = fmaxf(v[k], v[k + 2]);
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 4));
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 8));
            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 16));
            n = fmaxf(n, top[nt][k]);
            const float a = n == top[nt][k] ? 1.f : ex2(top[nt][k] - n);
            top[nt][k] = n;
            lsum[nt][k] *= a;
            if (!fresh) {
#pragma unroll
              for (int o = 0; o < OT; o++) O[nt][o][k] *= a, O[nt][o][k + 2] *= a;
            }
          }
        }
        float e[4];
        const float ref[2] = {top[nt][0] - lift, top[nt][1] - lift};
#pragma unroll
        for (int k = 0; k < 4; k++) e[k] = ex2(v[k] - ref[k & 1]);
        if (!full[nt]) {
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (!see[k]) e[k] = 0.f;
        }
        lsum[nt][0] += e[0] + e[2];
        lsum[nt][1] += e[1] + e[3];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint32_t h = pack2(e[2 * k], e[2 * k + 1]);
          const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&h));
          const uint32_t l = pack2(e[2 * k] - hf.x, e[2 * k + 1] - hf.y);
          if (MODE == kRows) {
            ph[nt][k] = transpose8x8(h);
            pl[nt][k] = transpose8x8(l);
          } else if (BITS == 4) {
            // columns 0-3: (0, hi), columns 4-7: (hi, lo); see the product with the scales
            ph[nt][k] = transpose8x8(t < 2 ? 0u : h);
            pl[nt][k] = transpose8x8(t < 2 ? h : l);
          } else {
            ph[nt][k] = transpose8x8(t < 2 ? h : l);      // columns 0-3 hi, 4-7 lo
          }
        }
      }

      // ---- slots that no row of the warp sees may hold anything: their scales (values)
      // become zero.  strict: a row does not see a slot that another row sees and that
      // holds an infinity or NaN, so its own mask goes on every operand.
      bool strict[N];
#pragma unroll
      for (int nt = 0; nt < N; nt++) strict[nt] = false;
      uint32_t dv[NB][2];
      if (BITS == 4) {
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
          const uint4 d4 = lds128(vp + (t * NB + b) * 8);
          dv[b][0] = d4.x, dv[b][1] = d4.y, dv[b + 1][0] = d4.z, dv[b + 1][1] = d4.w;
        }
        if (__builtin_expect(masked || ups != 0, 0)) {
          bool odd = false;
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
              dv[b][k] = hmul2(dv[b][k] & seen[k], scale_half2(scale_state(ups, b)));
              odd |= !finite2(dv[b][k]);
            }
          if (MODE == kRows && __any_sync(0xffffffffu, odd)) {
#pragma unroll
            for (int nt = 0; nt < N; nt++) strict[nt] = true;
          }
        }
      }

      // ---- O += V^T p
      if (BITS == 4) {
        uint32_t vw[4][NB / 2];
#pragma unroll
        for (int k = 0; k < 4; k++) lds_words<NB / 2>(vw[k], vp + HD + (k * 32 + lane) * (NB * 2));
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
          const uint32_t x = __byte_perm(vw[0][b / 2], vw[1][b / 2], sel), y = __byte_perm(vw[2][b / 2], vw[3][b / 2], sel);
          const uint32_t xs = x >> 8, ys = y >> 8;
          const uint32_t al[4] = {low_codes(x), low_codes(xs), low_codes(y), low_codes(ys)};
          const uint32_t ah[4] = {high_codes(x), high_codes(xs), high_codes(y), high_codes(ys)};
#pragma unroll
          for (int nt = 0; nt < N; nt++) {
            uint32_t bb[2], bh[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
              // hi: f16(hi d); lo: lo d + (hi d - f16(hi d)).  With (0, hi) for (hi, lo) the
              // second is f16(hi d): the hi columns where the tile has both
              const uint32_t d = strict[nt] ? dv[b][k] & keep[nt][k] : dv[b][k];
              bh[k] = hmul2(ph[nt][k], d);
              bb[k] = hfma2(pl[nt][k], d, hfms2(ph[nt][k], d, bh[k]));
            }
            if (MODE == kRows) {
              mma16816(O[nt][2 * b], al[0], al[1], al[2], al[3], bh[0], bh[1]);
              mma16816(O[nt][2 * b + 1], ah[0], ah[1], ah[2], ah[3], bh[0], bh[1]);
            }
            mma16816(O[nt][2 * b], al[0], al[1], al[2], al[3], bb[0], bb[1]);
            mma16816(O[nt][2 * b + 1], ah[0], ah[1], ah[2], ah[3], bb[0], bb[1]);
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < HD / 64; q++) {
          uint32_t vw[4][4];
#pragma unroll
          for (int k = 0; k < 4; k++) lds_words<4>(vw[k], vp + ((q * 4 + k) * 32 + lane) * 16);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            uint32_t a[4] = {__byte_perm(vw[0][k], vw[1][k], 0x5410), __byte_perm(vw[0][k], vw[1][k], 0x7632),
                             __byte_perm(vw[2][k], vw[3][k], 0x5410), __byte_perm(vw[2][k], vw[3][k], 0x7632)};
            bool each = false;                           // every row with its own mask
            if (masked) {
#pragma unroll
              for (int i2 = 0; i2 < 4; i2++) a[i2] &= seen[i2 >> 1];
              if (MODE == kRows)
                each = __any_sync(0xffffffffu, !finite2(a[0]) || !finite2(a[1]) || !finite2(a[2]) || !finite2(a[3]));
            }
#pragma unroll
            for (int nt = 0; nt < N; nt++) {
              float(&o)[4] = O[nt][4 * q + k];
              if (!each) {
                mma16816(o, a[0], a[1], a[2], a[3], ph[nt][0], ph[nt][1]);
                if (MODE == kRows) mma16816(o, a[0], a[1], a[2], a[3], pl[nt][0], pl[nt][1]);
                continue;
              }
              if (MODE == kRows)
                for (int r = 0; r < per_tile; r++) {     // the lanes of row r's columns give their mask and their p
                  const int from = r * slots * 4 + t;
                  const uint32_t k0 = __shfl_sync(0xffffffffu, keep[nt][0], from), k1 = __shfl_sync(0xffffffffu, keep[nt][1], from);
                  const bool mine = g / slots == r;
                  mma16816(o, a[0] & k0, a[1] & k0, a[2] & k1, a[3] & k1, mine ? ph[nt][0] : 0u, mine ? ph[nt][1] : 0u);
                  mma16816(o, a[0] & k0, a[1] & k0, a[2] & k1, a[3] & k1, mine ? pl[nt][0] : 0u, mine ? pl[nt][1] : 0u);
                }
            }
          }
        }
      }
    };
    for (uint32_t i = i0; i < span.count; i += W) {
      const uint32_t t0 = span.at(i) * kPieceSlots;
      if (!__all_sync(0xffffffffu, mbar_try_wait(&landed[st], phase)) && alive)
        alive = __all_sync(0xffffffffu, wait_slow(&landed[st], phase, p.d.status));
      const bool here = alive && usable[st] != 0;
      const uint8_t* kp = ring + (size_t)st * Sh::STAGE;
      const uint8_t* vp = kp + PB;

      if (live_tiles == NT) work(std::integral_constant<int, NT>{}, kp, vp, t0, here);
      else work(std::integral_constant<int, 1>{}, kp, vp, t0, here);
      __syncwarp();
      if (lane == 0 && alive) mbar_arrive(&freed[st]);
      fresh = false;
      st += W;
      if (st >= (uint32_t)S) st -= S, phase ^= 1u;
    }
    j0 += unit.span.count;
    const bool whole = unit.unit0 >= start.at && unit.unit1 <= run_end;
    if (!whole && lane == 0 && (uint32_t)warp == j0 % W) {               // the first to be idle
      // the CTAs c0..c1 whose runs hold the unit: a run's end less than `reach` behind the
      // unit's start moved there, one less before its end there
      const auto run_of = [&](uint64_t x) { return min((uint32_t)udiv((x + 1) * work_ctas - 1, work_all), work_ctas - 1); };
      const uint32_t F = reach_of(unit.unit1 - unit.unit0, unit.w.parts, work_uncut), c0 = run_of(min(unit.unit0 + F, unit.unit1) - 1);
      unit_c0 = c0;
      unit_c1 = unit.unit1 - unit.unit0 < 2 * F ? c0 : run_of(unit.unit1 - F);
    }

    // ---- the warps' states
    if (BITS == 4 && ups) {          // the blocks' scales come off
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const float f = scale_pow2(-scale_up(scale_state(ups, b)));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int k = 0; k < 4; k++) O[nt][2 * b][k] *= f, O[nt][2 * b + 1][k] *= f;
      }
    }
    consumers();                     // the q fragments have been read
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float l = lsum[nt][k];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (lane < TC / 2) {
          ml[(warp * LC + nt * TC + 2 * t + k) * 2] = top[nt][k] - lift;
          ml[(warp * LC + nt * TC + 2 * t + k) * 2 + 1] = l;
        }
      }
      const auto dim_of = [&](int o, int k) {
        return BITS == 4 ? (o / 2) * 32 + 4 * g + (o & 1) + 2 * (k >> 1) : (o / 4) * 64 + 8 * g + 2 * (o & 3) + (k >> 1);
      };
      if constexpr (MODE == kRows) {
#pragma unroll
        for (int o = 0; o < OT; o++)
#pragma unroll
          for (int k = 0; k < 4; k++) merge[(size_t)(warp * LC + nt * TC + 2 * t + (k & 1)) * HD + dim_of(o, k)] = O[nt][o][k];
      } else {
        // hi + lo: lanes t < 2 (the hi columns) take the even tiles, their partners the odd ones
#pragma unroll
        for (int o = 0; o < OT; o += 2)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float give = t < 2 ? O[nt][o + 1][k] : O[nt][o][k], mine = t < 2 ? O[nt][o][k] : O[nt][o + 1][k];
            const float x = mine + __shfl_xor_sync(0xffffffffu, give, 2);
            merge[(size_t)(warp * LC + 2 * (t & 1) + (k & 1)) * HD + dim_of(o, k) + (t >> 1) * (dim_of(1, 0) - dim_of(0, 0))] = x;
          }
      }
    }
    consumers();
    const uint32_t c0 = unit_c0, c1 = unit_c1;             // (of a unit that is cut)
    const auto store = [&](int c, int dim, const float4& x) {
      const int head = unit.kvh * p.G + col_head(c);
      const size_t row = row0 + col_row(c);
      if (p.out_f) *reinterpret_cast<float4*>(p.out_f + (row * p.QH + head) * HD + dim) = x;
      if (p.out_h) {
        uint16_t* out = p.out_h + row * p.QH * HD;
        const int at = head * HD + dim;
        if (p.xfo) {
          out[xfo_pos(at)] = f2h(x.x), out[xfo_pos(at + 1)] = f2h(x.y);
          out[xfo_pos(at + 2)] = f2h(x.z), out[xfo_pos(at + 3)] = f2h(x.w);
        } else {
          *reinterpret_cast<uint2*>(out + at) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
        }
      }
    };
    // a column's logarithm of the sum; what its sum is divided by (a NaN sum stays one)
    const auto close_column = [&](int c, float M, float L) {
      if (p.lse)
        p.lse[(row0 + col_row(c)) * (size_t)p.QH + unit.kvh * p.G + col_head(c)] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
      return L != 0.f ? 1.f / L : 0.f;
    };
    float* part = p.parts + (2 * (size_t)cta + (cta == c0 ? 1 : 0)) * Sh::PART;  // a run ends with at most one cut unit, and begins with one
    if constexpr (MODE == kRows) {
      for (int c = tid; c < cols; c += CT) {             // the weights of the warps' states of each column
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, ml[(i * LC + c) * 2]);
#pragma unroll
        for (int i = 0; i < W; i++) {
          float* at = ml + (i * LC + c) * 2;
          const float a = at[0] == M ? 1.f : ex2(at[0] - M);
          L = fmaf(a, at[1], L);
          at[0] = a;
        }
        float r = 1.f;
        if (!col_live(c)) r = 0.f;
        else if (whole) r = close_column(c, M, L);
        else *reinterpret_cast<float2*>(part + Sh::COLS * HD + 2 * c) = make_float2(M, L);
#pragma unroll
        for (int i = 0; i < W; i++) ml[(i * LC + c) * 2] *= r;
      }
      consumers();
#pragma unroll 2
      for (int e = tid; e < cols * (HD / 4); e += CT) {
        const int c = e / (HD / 4), dim = e % (HD / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < W; i++) {
          const int at = i * LC + c;
          const float a = ml[at * 2];
          const float4 x = *reinterpret_cast<const float4*>(merge + (size_t)at * HD + dim);
          o.x = fmaf(a, x.x, o.x), o.y = fmaf(a, x.y, o.y), o.z = fmaf(a, x.z, o.z), o.w = fmaf(a, x.w, o.w);
        }
        if (!col_live(c)) continue;
        if (whole) store(c, dim, o);
        else *reinterpret_cast<float4*>(part + c * HD + dim) = o;
      }
    } else {                         // few columns: every thread forms its column's weights
      for (int e = tid; e < LC * (HD / 4); e += CT) {
        const int c = e / (HD / 4), dim = e % (HD / 4) * 4;
        if (!col_live(c)) continue;
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, ml[(i * LC + c) * 2]);
#pragma unroll
        for (int i = 0; i < W; i++) {
          const int at = i * LC + c;
          const float mi = ml[at * 2], w = mi == M ? 1.f : ex2(mi - M);
          const float4 x = *reinterpret_cast<const float4*>(merge + (size_t)at * HD + dim);
          L = fmaf(w, ml[at * 2 + 1], L);
          o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
        }
        if (whole) {
          const float r = L != 0.f ? 1.f / L : 0.f;
          store(c, dim, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
          if (dim == 0) close_column(c, M, L);
        } else {
          *reinterpret_cast<float4*>(part + c * HD + dim) = o;
          if (dim == 0) *reinterpret_cast<float2*>(part + Sh::COLS * HD + 2 * c) = make_float2(M, L);
        }
      }
    }
    if (!whole) {
      // The last CTA to arrive merges the parts; of many parts, the last of each group of
      // kGroup merges the group's into its first CTA's, and the last of those the rest.
      const auto part_of = [&](uint32_t c) { return p.parts + (2 * (size_t)c + (c == c0 ? 1 : 0)) * Sh::PART; };
      const auto arrive = [&](uint32_t* counter, uint32_t n) {
        consumers();                   // the part is written: the arrival releases it, and acquires the others'
        if (tid == 0) last_one = inc_acq_rel(counter, n - 1) == n - 1; // wraps to zero with the last arrival
        consumers();
        return last_one != 0;
      };
      // parts of CTAs a, a + step, .. (n of them): into the outputs, or into a's part
      const auto combine = [&](uint32_t a, uint32_t step, uint32_t n, bool final) {
        if constexpr (MODE != kRows) {
          for (int e = tid; e < LC * (HD / 4); e += CT) {
            const int c = e / (HD / 4), dim = e % (HD / 4) * 4;
            if (!col_live(c)) continue;
            float M = -INFINITY, L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < n; i0 += 8) {      // eight parts' loads in flight
              float4 x[8];
              float2 y[8];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float* from = part_of(a + min(i0 + i, n - 1) * step);
                y[i] = __ldcg(reinterpret_cast<const float2*>(from + Sh::COLS * HD + 2 * c));
                x[i] = __ldcg(reinterpret_cast<const float4*>(from + c * HD + dim));
              }
              float top = M;
#pragma unroll
              for (int i = 0; i < 8; i++) top = fmaxf(top, y[i].x);
              const float f0 = M == top ? 1.f : ex2(M - top);
              M = top;
              L *= f0, o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                if (i0 + i >= n) continue;
                const float f = y[i].x == M ? 1.f : ex2(y[i].x - M);
                L = fmaf(f, y[i].y, L);
                o.x = fmaf(f, x[i].x, o.x), o.y = fmaf(f, x[i].y, o.y);
                o.z = fmaf(f, x[i].z, o.z), o.w = fmaf(f, x[i].w, o.w);
              }
            }
            if (final) {
              const float r = L != 0.f ? 1.f / L : 0.f;
              store(c, dim, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
              if (dim == 0) close_column(c, M, L);
            } else {
              *reinterpret_cast<float4*>(part_of(a) + c * HD + dim) = o;
              if (dim == 0) ml[2 * c] = M, ml[2 * c + 1] = L;
            }
          }
          if (!final) {                // a column is up to two warps: its threads have read part a's (max, sum) before it changes
            consumers();
            if (tid < LC && col_live(tid))
              *reinterpret_cast<float2*>(part_of(a) + Sh::COLS * HD + 2 * tid) = make_float2(ml[2 * tid], ml[2 * tid + 1]);
          }
        } else {
          float2* part_ml = reinterpret_cast<float2*>(merge);          // [n][cols]
          for (uint32_t e = tid; e < n * cols; e += CT)
            part_ml[e] = __ldcg(reinterpret_cast<const float2*>(part_of(a + e / cols * step) + Sh::COLS * HD + 2 * (e % cols)));
          consumers();
          for (int c = tid; c < cols; c += CT) {           // the parts' weights
            float M = -INFINITY, L = 0.f;
            for (uint32_t i = 0; i < n; i++) M = fmaxf(M, part_ml[i * cols + c].x);
            for (uint32_t i = 0; i < n; i++) {
              float2& y = part_ml[i * cols + c];
              y.x = y.x == M ? 1.f : ex2(y.x - M);
              L = fmaf(y.x, y.y, L);
            }
            if (!col_live(c)) continue;
            if (final) {
              const float r = close_column(c, M, L);
              for (uint32_t i = 0; i < n; i++) part_ml[i * cols + c].x *= r;
            } else {
              *reinterpret_cast<float2*>(part_of(a) + Sh::COLS * HD + 2 * c) = make_float2(M, L);
            }
          }
          consumers();
          constexpr int kE = 4, kI = 2;    // eight loads in flight
          for (int e0 = tid; e0 < cols * (HD / 4); e0 += kE * CT) {
            float4 o[kE];
#pragma unroll
            for (int j = 0; j < kE; j++) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < n; i0 += kI) {
              float4 x[kI][kE];
#pragma unroll
              for (int i = 0; i < kI; i++)
#pragma unroll
                for (int j = 0; j < kE; j++) {
                  const int e = min(e0 + j * CT, cols * (HD / 4) - 1);
                  x[i][j] = __ldcg(reinterpret_cast<const float4*>(part_of(a + min(i0 + i, n - 1) * step)) + e);
                }
#pragma unroll
              for (int i = 0; i < kI; i++) {
                if (i0 + i >= n) continue;
#pragma unroll
                for (int j = 0; j < kE; j++) {
                  const int e = min(e0 + j * CT, cols * (HD / 4) - 1);
                  const float f = part_ml[(i0 + i) * cols + e / (HD / 4)].x;
                  o[j].x = fmaf(f, x[i][j].x, o[j].x), o[j].y = fmaf(f, x[i][j].y, o[j].y);
                  o[j].z = fmaf(f, x[i][j].z, o[j].z), o[j].w = fmaf(f, x[i][j].w, o[j].w);
                }
              }
            }
#pragma unroll
            for (int j = 0; j < kE; j++) {
              const int e = e0 + j * CT, c = e / (HD / 4);
              if (e >= cols * (HD / 4) || !col_live(c)) continue;
              if (final) store(c, e % (HD / 4) * 4, o[j]);
              else *(reinterpret_cast<float4*>(part_of(a)) + e) = o[j];
            }
          }
        }
      };
      const uint32_t n = c1 - c0 + 1, groups = (n + kGroup - 1) / kGroup;
      if (groups == 1) {
        if (arrive(p.arrived + c0, n)) combine(c0, 1, n, true);
      } else {
        const uint32_t gi = (cta - c0) / kGroup, from = c0 + gi * kGroup;
        const uint32_t size = min((uint32_t)kGroup, n - gi * kGroup);
        if (arrive(p.arrived + (gi ? kMaxCtas : 0) + from, size)) {
          combine(from, 1, size, false);
          if (arrive(p.arrived + 2 * kMaxCtas + c0, groups)) combine(c0, kGroup, groups, true);
        }
      }
    }
    consumers();                     // the merge buffer and the states are free again
    if (tid == 0) {
      Unit v = unit;
      next_unit(v);
    }
    consumers();
  }
}

template <int BITS, int HD, int MODE>
int launch(e4b_ctx* c, const AttnP& p) {
  using Sh = Shape<BITS, HD, MODE>;
  static_assert(Sh::PER_SM * (Sh::SMEM + 8 * 1024) < 228 * 1024, "shared memory");
  E4B_CUDA(c, cudaFuncSetAttribute(k_attn_paged<BITS, HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::SMEM));
  const int ctas = Sh::PER_SM * c->sm_count < Sh::MAX_CTAS ? Sh::PER_SM * c->sm_count : Sh::MAX_CTAS;
  return e4b_launch(c, "attn_paged", k_attn_paged<BITS, HD, MODE>, dim3(ctas), dim3(Sh::THREADS), Sh::SMEM, p);
}
template <int BITS, int HD>
int launch_mode(e4b_ctx* c, const AttnP& p) {
  if (p.G > 4 || p.d.rows) return launch<BITS, HD, kRows>(c, p);
  // few units: all of an SM's warps on one (kWide against kNarrow, 4 bits, heads of 256: a
  // sequence of 131001 tokens and 2 KV heads 31.0 against 38.6 us, 32 of 8000..16000 tokens
  // and 4 KV heads 107 against 116 us); more units than SMs: two CTAs per SM (kNarrow against
  // kWide, 64 of 1035 tokens and 4 KV heads 30.3 against 36.7 us; f16, windows of 1024 in
  // 1..8000 tokens 29.3 against 42.9 us)
  if (p.d.nseq * p.d.KVH <= c->sm_count) return launch<BITS, HD, kWide>(c, p);
  return launch<BITS, HD, kNarrow>(c, p);
}
template <int BITS>
int launch_hd(e4b_ctx* c, const AttnP& p, int HD) {
  return HD == 256 ? launch_mode<BITS, 256>(c, p) : (HD == 128 ? launch_mode<BITS, 128>(c, p) : launch_mode<BITS, 64>(c, p));
}
}  // namespace

extern "C" {

E4B_API size_t e4b_paged_scratch_bytes(void) {
  // two partials for each of kMaxCtas / 2 CTAs of the shape with the largest ones
  return kMaxCtas * (3 * sizeof(uint32_t) + Shape<4, 256, kRows>::PART * sizeof(float));
}

E4B_API int e4b_attn_paged(e4b_ctx* c, const e4b_paged_kv* kv, const float* q, uint16_t* out_h, float* out_f,
                           float* lse, void* scratch, int QH, int window, int sinks, float scale, int xfo, int n_rows) {
  E4B_CHECK_CTX(c);
  const char* fault = attn_paged_fault(kv, q, out_h, out_f, lse, scratch, QH, window, sinks, scale, xfo, n_rows);
  E4B_REQUIRE(c, !fault, "attn_paged: %s", fault);
  if (n_rows == 0) return E4B_OK;
  AttnP p;
  p.d = paged_dev(c, kv, n_rows);
  p.q = q;
  p.out_h = out_h;
  p.out_f = out_f;
  p.lse = lse;
  p.arrived = static_cast<uint32_t*>(scratch);
  p.parts = reinterpret_cast<float*>(p.arrived + 3 * kMaxCtas);
  p.QH = QH;
  p.G = QH / kv->kv_heads;
  p.xfo = xfo ? 1 : 0;
  p.window = (uint32_t)window;
  p.sinks = (uint32_t)sinks;
  p.scale = scale;
  return kv->bits == 16 ? launch_hd<16>(c, p, kv->head_dim) : launch_hd<4>(c, p, kv->head_dim);
}

}  // extern "C"
