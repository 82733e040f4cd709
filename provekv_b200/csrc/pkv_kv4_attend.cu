// Attention over the 4-bit KV cache.
//
// One kernel for a few query rows per kv head (a decode step, short drafts).  Work is counted in units of 64 tokens (four
// atoms, keys and values with their scales in one contiguous run).  A warp works on its own: it streams its units
// through a ring of bulk copies and keeps running softmax statistics, so warps never wait for each other.
//
//   S^T = K Q^T     mma m16n8k16: 16 keys x 8 query rows; the A operand is dequantised straight into registers
//   O^T = V^T P^T   16 channels x 8 query rows, contraction over the 16 keys of an atom
//
// With the keys on the M side eight query rows fill a tile (shared heads seldom give more) and the tile costs half the
// products and exponentials that 16 query rows on M would.  P^T is the S^T tile transposed in registers (movmatrix).
// Key row m of a tile is token tau(m) = m/2 (even m) or 7 - m/2 (odd m) of its half atom, the same in both products:
// the order in which the 16-byte pieces of K rows and the 8-byte pieces of V rows fall on distinct banks.
//
// How the units are dealt out (make_plan):
//   short rows   a CTA per (sequence, kv head, row tile); its warps take every fourth unit and join their sums in
//                shared memory: one launch
//   long rows    as many warps as the GPU holds; all units of all rows, laid end to end, are cut into equal runs, one a warp,
//                whatever the lengths.  The stream of units runs on from one row into the next.  A row that was cut is joined
//                by a second launch from the warps' sums.
//
#include <limits.h>

#include "pkv_kv4_attend.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;
constexpr int kMaxRows = 2048;           // (sequence, kv head, row tile)s that share runs
constexpr int64_t kMostScores = 1ll << 26;  // 256 MiB
constexpr int kMassTokens = 32, kMassWarps = 8;  // keys a warp of the mass kernel holds; its warps
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a chain: no accumulator to clear
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ int tau(int m) { return (m & 8) | ((m & 1) ? 7 - ((m & 7) >> 1) : (m & 7) >> 1); }

// The B operand of S^T for query row `lane / 4` from its values of channels (lane % 4) D/4 .. (this lane's), in the
// order nibbles() delivers the keys', odd channels divided by 16; negated for a negative softmax scale, so that scores
// are scaled by something positive.  hi (and for f32 queries lo) [D / 16][2]; returns the inverse power.
template <int D, int T>
__device__ __forceinline__ float query_operand(const float (&x)[D / 4], bool negate, uint32_t (&hi)[D / 16][2],
                                               uint32_t (&lo)[D / 16][2]) {
  constexpr int CH = D / 4;
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; i++) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float inv = 1.0f / row_power(amax), pw = negate ? -row_power(amax) : row_power(amax);
#pragma unroll
  for (int j = 0; j < CH / 8; j++) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float f = (u & 1) ? 0.0625f : 1.0f;
      const float a = __fmul_rn(__fmul_rn(x[8 * j + u], pw), f), b = __fmul_rn(__fmul_rn(x[8 * j + u + 4], pw), f);
      const uint32_t h = half2_of(a, b);
      hi[2 * j + (u >> 1)][u & 1] = h;
      if constexpr (T == PKV_DST_F32) {
        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h));
        lo[2 * j + (u >> 1)][u & 1] = half2_of(__fsub_rn(a, r.x), __fsub_rn(b, r.y));
      }
    }
  }
  return inv;
}
// Those values of query row `row` (of its kv head's, token by token).
template <int D, int T>
__device__ __forceinline__ void query_values(const AttendParams& p, int s, int h, int row, int rows, float (&x)[D / 4]) {
  using E = typename PkvDst<T>::type;
  const int token = row / p.group, hq = h * p.group + (row - token * p.group);
  if (row < rows) {
    load_f32<T, D / 4>(reinterpret_cast<const E*>(p.q_ptr) + s * p.q.seq + (int64_t)token * p.q.token + hq * p.q.head +
                           (threadIdx.x & 3) * (D / 4),
                       x);
  } else {
#pragma unroll
    for (int i = 0; i < D / 4; i++) x[i] = 0.0f;
  }
}

// A lane's part of an atom's keys: tokens tau(lane / 4) and 8 on, channels (lane % 4) D/4 ..
template <int D>
struct KeyCodes {
  uint32_t w0[D / 32], w1[D / 32];
  Scale sc0[D / 64], sc1[D / 64];
  __device__ __forceinline__ KeyCodes(const uint8_t* atom, int lane) {
    using A = Atom<D>;
    const int q4 = lane & 3, t0 = tau(lane >> 2), t1 = t0 + 8;
    if constexpr (D == 128) {
      const uint4 a = *reinterpret_cast<const uint4*>(atom + A::KC + t0 * A::ROW + 16 * q4);
      const uint4 b = *reinterpret_cast<const uint4*>(atom + A::KC + t1 * A::ROW + 16 * q4);
      w0[0] = a.x; w0[1] = a.y; w0[2] = a.z; w0[3] = a.w;
      w1[0] = b.x; w1[1] = b.y; w1[2] = b.z; w1[3] = b.w;
      const uint32_t u0 = *reinterpret_cast<const uint16_t*>(atom + A::KS + t0 * A::SROW + 2 * q4);
      const uint32_t u1 = *reinterpret_cast<const uint16_t*>(atom + A::KS + t1 * A::SROW + 2 * q4);
      const Scale p0 = scale_of(__byte_perm(u0, 0u, 0x4140) << 7), p1 = scale_of(__byte_perm(u1, 0u, 0x4140) << 7);
      sc0[0] = p0.low();
      sc0[1] = p0.high();
      sc1[0] = p1.low();
      sc1[1] = p1.high();
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(atom + A::KC + t0 * A::ROW + 8 * q4);
      const uint2 b = *reinterpret_cast<const uint2*>(atom + A::KC + t1 * A::ROW + 8 * q4);
      w0[0] = a.x; w0[1] = a.y;
      w1[0] = b.x; w1[1] = b.y;
      sc0[0] = scale_of((uint32_t)atom[A::KS + t0 * A::SROW + q4] * 0x00800080u);
      sc1[0] = scale_of((uint32_t)atom[A::KS + t1 * A::SROW + q4] * 0x00800080u);
    }
  }
};

// One atom's scores: S^T[16 keys][8 NT rows] from its K codes and scales in shared memory.
//
// F32 (queries of two binary16 terms): 0 one term, 1 the terms in operands of their own, 2 side by side in one operand
// (up to four rows: rows 0..3 the first terms, 4..7 the second; half the products).
template <int D, int NT, int F32>
__device__ __forceinline__ void scores_of(const uint8_t* atom, int lane, const uint32_t (&qhi)[NT][D / 16][2],
                                          const uint32_t (&qlo)[NT][D / 16][2], float (&s)[NT][4]) {
  const KeyCodes<D> k(atom, lane);
  // F32: the tensor cores cut their sums off instead of rounding them; chains of at most D / 32 products of the queries' first
  // terms, the second terms apart, keep that below the f32 error of the sum
  float part[F32 ? NT : 1][2][4];
#pragma unroll
  for (int j = 0; j < D / 32; j++) {
    uint32_t a[4], b[4];
    nibbles(k.w0[j], k.sc0[j >> 1], a);
    nibbles(k.w1[j], k.sc1[j >> 1], b);
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const uint32_t h0 = qhi[n][2 * j + u][0], h1 = qhi[n][2 * j + u][1];
        if constexpr (F32 == 2) {
          float(&hi)[4] = 2 * j < D / 32 ? s[n] : part[n][0];
          if (2 * j % (D / 32) == 0 && u == 0) mma_first(hi, a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
          else mma(hi, a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
        } else if constexpr (F32 == 1) {
          float(&hi)[4] = 2 * j < D / 32 ? s[n] : part[n][0];
          const uint32_t l0 = qlo[n][2 * j + u][0], l1 = qlo[n][2 * j + u][1];
          if (2 * j % (D / 32) == 0 && u == 0) mma_first(hi, a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
          else mma(hi, a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
          if (j == 0 && u == 0) mma_first(part[n][1], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], l0, l1);
          else mma(part[n][1], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], l0, l1);
        } else {
          if (j == 0 && u == 0) mma_first(s[n], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
          else mma(s[n], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], h0, h1);
        }
      }
  }
  if constexpr (F32 == 1) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[n][i] = __fadd_rn(__fadd_rn(s[n][i], part[n][0][i]), part[n][1][i]);
  }
  if constexpr (F32 == 2) {  // rows r and r + 4 are in lanes that differ in bit 1: both get their sum
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x = __fadd_rn(s[n][i], part[n][0][i]);
        s[n][i] = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 2));
      }
  }
}

// O^T += V^T P^T for one atom; p[n][0..1] is the B operand (f32 queries: p[n][2..3] its remainder).
template <int D, int NT, int F32, bool FIRST>
__device__ __forceinline__ void weigh(const uint8_t* atom, int lane, const uint32_t (&p)[NT][F32 == 1 ? 4 : 2], float (&o)[D / 16][NT][4]) {
  using A = Atom<D>;
  const int q4 = lane & 3, g = lane >> 2;
  uint32_t m[2][D / 16 * 2];  // [key pair][channel of this lane]: two keys' values of one channel
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int t0 = q4 + 8 * h, t1 = 7 - q4 + 8 * h;
    uint32_t w0[D / 64], w1[D / 64];
    uint32_t sb0, sb1;
    if constexpr (D == 128) {
      const uint2 a = *reinterpret_cast<const uint2*>(atom + A::VC + t0 * A::ROW + ((8 * g) ^ A::vswap(t0)));
      const uint2 b = *reinterpret_cast<const uint2*>(atom + A::VC + t1 * A::ROW + ((8 * g) ^ A::vswap(t1)));
      w0[0] = a.x; w0[1] = a.y;
      w1[0] = b.x; w1[1] = b.y;
      sb0 = atom[A::VS + t0 * A::SROW + g];
      sb1 = atom[A::VS + t1 * A::SROW + g];
    } else {
      w0[0] = *reinterpret_cast<const uint32_t*>(atom + A::VC + t0 * A::ROW + 4 * g);
      w1[0] = *reinterpret_cast<const uint32_t*>(atom + A::VC + t1 * A::ROW + 4 * g);
      sb0 = atom[A::VS + t0 * A::SROW + (g >> 1)];
      sb1 = atom[A::VS + t1 * A::SROW + (g >> 1)];
    }
    const Scale sc = scale_of((sb0 << 7) | (sb1 << 23));
#pragma unroll
    for (int j = 0; j < D / 64; j++) {
      uint32_t lo[4], hi[4];
      nibbles(__byte_perm(w0[j], w1[j], 0x5410), sc, lo);  // channels 0..3 of the word: first token, second token
      nibbles(__byte_perm(w0[j], w1[j], 0x7632), sc, hi);  // channels 4..7
#pragma unroll
      for (int i = 0; i < 4; i++) {
        m[h][8 * j + i] = lo[i];
        m[h][8 * j + 4 + i] = hi[i];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < D / 16; j++)
#pragma unroll
    for (int n = 0; n < NT; n++) {
      if constexpr (FIRST) mma_first(o[j][n], m[0][2 * j], m[0][2 * j + 1], m[1][2 * j], m[1][2 * j + 1], p[n][0], p[n][1]);
      else mma(o[j][n], m[0][2 * j], m[0][2 * j + 1], m[1][2 * j], m[1][2 * j + 1], p[n][0], p[n][1]);
      if constexpr (F32 == 1) mma(o[j][n], m[0][2 * j], m[0][2 * j + 1], m[1][2 * j], m[1][2 * j + 1], p[n][2], p[n][3]);
    }
}

// Units of one (kv head, row tile) of a sequence: what its first to last query token see, at least one (a row that sees
// nothing is written too), none without queries.
__device__ __forceinline__ int units_of(const AttendParams& p, const Sequence& q) {
  if (q.qn == 0) return 0;
  return max(1, visible_span(p, q.len, q.end - q.qn, q.end - 1).count);
}
// Row tiles of a kv head that the sequence's queries fill (row_tiles is the number for a full batch row).
__device__ __forceinline__ int row_tiles_of(const AttendParams& p, const Sequence& q) {
  return (q.qn * p.group + p.tile_rows - 1) / p.tile_rows;
}
// (below 2^31 for all sequences together, which make_plan sees to)
__device__ __forceinline__ unsigned all_units_of(const AttendParams& p, const Sequence& q) {
  return (unsigned)(units_of(p, q) * p.c.heads * row_tiles_of(p, q));
}
__device__ __forceinline__ unsigned all_units_of(const AttendParams& p, int s) {
  return s < p.c.n_seqs ? all_units_of(p, sequence_of(p, s)) : 0u;
}

// The units of all rows, cut into runs as even as they can be; no run is empty before one that is not.
struct Runs {
  unsigned total, each, more;  // the first `more` runs have each + 1 units, the others `each`
  __device__ __forceinline__ unsigned start(unsigned i) const { return min(total, i * each + min(i, more)); }
  __device__ __forceinline__ unsigned of(unsigned unit) const {
    const unsigned cut = more * (each + 1);
    return unit < cut ? unit / (each + 1) : more + (unit - cut) / each;
  }
};
// Whole warp; `mine` is all_units_of(p, lane).
__device__ __forceinline__ Runs cut_runs(const AttendParams& p, unsigned mine) {
  unsigned sum = mine;
  for (int i = 32 + (threadIdx.x & 31); i < p.c.n_seqs; i += 32) sum += all_units_of(p, i);
  Runs r;
  r.total = __reduce_add_sync(0xffffffffu, sum);
  const unsigned n = max(1u, min((unsigned)p.runs, r.total));
  r.each = r.total / n;
  r.more = r.total - r.each * n;
  return r;
}

// A row tile on the way through all rows' units: sequence, kv head, tile; the last ones' index runs fastest.
struct Cursor {
  int s, h, tile, tiles, units;  // tiles of the sequence's kv heads; units of the tile, counted as the sequence's
  Sequence seq;
  Span span;
  __device__ __forceinline__ void place(const AttendParams& p) {
    const int pos0 = seq.end - seq.qn, row0 = tile * p.tile_rows;
    span = visible_span(p, seq.len, pos0 + row0 / p.group, pos0 + min(seq.qn - 1, (row0 + p.tile_rows - 1) / p.group));
  }
  __device__ __forceinline__ void enter(const AttendParams& p, int s_) {
    s = s_;
    seq = sequence_of(p, s);
    units = units_of(p, seq);
    tiles = row_tiles_of(p, seq);
  }
  __device__ __forceinline__ void next(const AttendParams& p) {  // only called while there is one
    if (++tile == tiles) {
      tile = 0;
      if (++h == p.c.heads) {
        h = 0;
        do enter(p, s + 1);
        while (seq.qn == 0);
      }
    }
    place(p);
  }
  __device__ __forceinline__ int rows(const AttendParams& p) const { return seq.qn * p.group; }
};

template <int D, int NT>
struct Shared {
  static constexpr int UNIT = kUnitAtoms * Atom<D>::BYTES;
  static constexpr int RING = kStages * UNIT;
  static constexpr int O_BYTES = 8 * NT * (D + 4) * 4;  // a warp's sums, in the space of its ring
  static constexpr int WARP = RING > O_BYTES ? RING : O_BYTES;
  static constexpr int BYTES = kWarps * WARP;
};

// A warp's ring: the slot that the next unit goes to or comes from, and the parity of the barrier there.
struct Ring {
  uint8_t* base;
  uint64_t* bars;
  int slot;
  uint32_t phase;
};

template <int D, int NT>
struct Sums {
  float o[D / 16][NT][4];            // channels (lane / 4) D/8 + 2 j + i / 2, row 2 (lane % 4) + i % 2
  float m[NT][2], l[NT][2];          // reference (log2) and sum of rows 2 (lane % 4) + e; l is this lane's part
};

// Streams a warp's units; whole warp.  PAIRED: f32 queries, at most four rows in all, the two terms of queries and weights
// side by side in operands of eight rows.  DIRECT: units v, v + kWarps, .. of row tile `t`; the sums stay in `r`.
// Otherwise: `count` units from unit v of row tile `t` on (number `at` of all rows' units), into the next row tiles; every row tile's sums are written
// when it ends, into out if the run has all of it, else into the run's parts.
template <int D, int NT, int T, bool DIRECT, bool PAIRED>
__device__ __forceinline__ void stream_units(const AttendParams& p, Cursor t, int v, int count, Ring& ring, Sums<D, NT>& r,
                                             Runs runs = Runs(), unsigned at = 0) {
  constexpr int F32 = T != PKV_DST_F32 ? 0 : PAIRED ? 2 : 1;
  constexpr int STEP = DIRECT ? kWarps : 1;
  using A = Atom<D>;
  using S = Shared<D, NT>;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  float qx[NT][D / 4];  // the queries' values are on their way while the first page numbers and units are
#pragma unroll
  for (int n = 0; n < NT; n++) query_values<D, T>(p, t.s, t.h, t.tile * 8 * NT + 8 * n + (PAIRED ? g & 3 : g), t.rows(p), qx[n]);

  // ---- the stream.  Page numbers are fetched for up to kBatch units of a row tile at once, one atom per lane, a batch ahead
  // of their use.
  Cursor ahead = t;        // row tile of the next batch to fetch
  int ahead_v = v, left = count;  // its first unit, and the units not yet fetched
  int next_n = 0, next_page = -1, next_s = 0;
  int64_t next_at = -1;    // place of the lane's atom in its page, -1 = nothing to load
  auto fetch = [&]() {
    if (!DIRECT && ahead_v == ahead.units && left > 0) {
      ahead.next(p);
      ahead_v = 0;
    }
    next_n = min(kBatch, DIRECT ? left : min(left, ahead.units - ahead_v));
    const int uv = ahead_v + (lane / kUnitAtoms) * STEP, a = ahead.span.unit(uv) * kUnitAtoms + lane % kUnitAtoms;
    next_at = -1;
    next_s = ahead.s;
    if (lane / kUnitAtoms < next_n && uv < ahead.span.count && a * kAtomTokens < ahead.seq.len) {
      const int page = a / p.c.page_atoms;
      next_page = __ldg(p.c.table + (int64_t)ahead.s * p.c.max_pages + page);
      next_at = (int64_t)ahead.h * p.c.page_atoms + (a - page * p.c.page_atoms);
    }
    left -= next_n;
    ahead_v += next_n * STEP;
  };
  fetch();
  const uint8_t* src = nullptr;
  unsigned live = 0;       // bit l: the atom of lane l is there (batch being issued)
  int batch_n = 0, batch_i = 0;
  unsigned quads = 0;      // of each slot of the ring: which of the unit's atoms are there, 4 bits
  int slot_in = ring.slot;
  auto issue = [&]() {     // whole warp
    if (__builtin_expect(batch_i == batch_n, 0)) {
      src = nullptr;
      if (next_at >= 0) {
        if (next_page < 0 || next_page >= p.c.n_pages) pkv_report(p.err, 0, next_s, PKV_VEC_BAD_SEQUENCE);
        else src = p.c.pages + ((int64_t)next_page * p.c.heads * p.c.page_atoms + next_at) * (int64_t)A::BYTES;
      }
      live = __ballot_sync(0xffffffffu, src != nullptr);
      batch_n = next_n;
      batch_i = 0;
      fetch();
    }
    const int l = kUnitAtoms * batch_i;
    const unsigned quad = (live >> l) & 15u;
    const uint32_t bytes = (uint32_t)__popc(quad) * A::BYTES;
    quads = (quads & ~(15u << (4 * slot_in))) | (quad << (4 * slot_in));
    uint8_t* dst = ring.base + slot_in * S::UNIT;
    uint64_t* bar = ring.bars + slot_in;
    if (lane == l) {
      pkv_mbar_expect_tx(bar, bytes);
      if (p.whole_units && bytes) pkv_bulk_load(dst, src, bytes, bar);
    }
    if (!p.whole_units) {
      __syncwarp();
      if (lane / kUnitAtoms == batch_i && src) pkv_bulk_load(dst + lane % kUnitAtoms * A::BYTES, src, A::BYTES, bar);
    }
    batch_i++;
    if (++slot_in == kStages) slot_in = 0;
  };
  int issued = 0;
#pragma unroll 1
  for (; issued < min(kStages, count); issued++) issue();

  uint32_t qhi[NT][D / 16][2], qlo[NT][D / 16][2];
  float factor[NT][2];  // of the scores of rows 2 q4 and 2 q4 + 1: softmax scale, log2 e, powers of two
  int len, pos0, row0, qpos_min, qpos_max;
  bool by_position;
  const int32_t* positions;
  auto begin_tile = [&]() {
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const float inv = query_operand<D, T>(qx[n], p.negate, qhi[n], qlo[n]);
      if constexpr (PAIRED) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) qhi[n][j][e] = g < 4 ? qhi[n][j][e] : qlo[n][j][e];
      }
      const float f = __fmul_rn(__fmul_rn(p.scale, kLog2e), kScaleShift);
#pragma unroll
      for (int e = 0; e < 2; e++) factor[n][e] = __fmul_rn(f, __shfl_sync(0xffffffffu, inv, 4 * (2 * q4 + e)));
    }
    len = t.seq.len;
    pos0 = t.seq.end - t.seq.qn;  // position of query token 0
    row0 = t.tile * 8 * NT;
    qpos_min = pos0 + row0 / p.group;
    qpos_max = pos0 + min(t.seq.qn - 1, (row0 + 8 * NT - 1) / p.group);
    // positions matter only where a row can see less than everything that is held
    by_position = p.c.positions != nullptr && (p.window > 0 || t.seq.qn > 1);
    positions = by_position ? p.c.positions + p.c.stat(t.s, t.h) : nullptr;
#pragma unroll
    for (int j = 0; j < D / 16; j++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) r.o[j][n][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        r.m[n][e] = -INFINITY;
        r.l[n][e] = 0.0f;
      }
  };
  auto join_lanes = [&]() {
    if constexpr (PAIRED) {  // what the first and the second terms of the weights gave
#pragma unroll
      for (int j = 0; j < D / 16; j++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) r.o[j][n][i] = __fadd_rn(r.o[j][n][i], __shfl_xor_sync(0xffffffffu, r.o[j][n][i], 2));
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = r.l[n][e];
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 8));
        r.l[n][e] = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 16));
      }
  };
  const int run = blockIdx.x * kWarps + warp;
  auto end_tile = [&](int v0, int n_units) {  // units v0 .. v0 + n_units - 1 of tile t are in r
    join_lanes();
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = 8 * n + 2 * q4 + e;
        float x[D / 8];
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          x[2 * j] = __fmul_rn(r.o[j][n][e], kScaleShift);
          x[2 * j + 1] = __fmul_rn(r.o[j][n][2 + e], kScaleShift / 16.0f);
        }
        if (row0 + row < t.rows(p) && (!PAIRED || q4 < 2)) {
          if (n_units < t.units) {  // a row that starts here and goes on has the run's second place
            const int64_t slot = ((int64_t)run * 2 + (v0 == 0)) * (8 * NT) + row;
            store_f32<PKV_DST_F32, D / 8>(p.part_o + slot * D + g * (D / 8), x);
            if (g == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(r.m[n][e], r.l[n][e]);
          } else {
            write_row<T, D / 8>(p, t.s, t.h, row0 + row, g * (D / 8), x, r.m[n][e], r.l[n][e], g == 0);
          }
        }
      }
  };
  int left_here = count;
#pragma unroll 1
  for (;;) {
    begin_tile();
    const int v0 = v, n_here = DIRECT ? count : min(left_here, t.units - v);
    if constexpr (!DIRECT)  // (before the first wait, which may give up)
      if (v0 == 0 && lane == 0)
        p.part_of[((int64_t)t.s * p.c.heads + t.h) * p.row_tiles + t.tile] =
            make_int2(run, n_here == t.units ? 1 : (int)runs.of(at + t.units - 1) - run + 1);
#pragma unroll 1
    for (int i = 0; i < n_here; i++, v += STEP) {
      const int token0 = t.span.unit(v) * kUnitTokens;
      int kpos[2] = {0, 0};
      if (__builtin_expect(by_position, 0)) {
#pragma unroll
        for (int k = 0; k < 2; k++)
          if (token0 + 32 * k + lane < len) kpos[k] = __ldg(positions + token0 + 32 * k + lane);
      }
      if (__builtin_expect(!__all_sync(0xffffffffu, pkv_mbar_wait(ring.bars + ring.slot, ring.phase)), 0)) {
        // a copy never arrived: give the others their time, report, and leave nothing behind
        for (int k = 1; k < kStages; k++) {
          if (++ring.slot == kStages) ring.slot = 0, ring.phase ^= 1u;
          if (ring.slot != slot_in) pkv_mbar_wait(ring.bars + ring.slot, ring.phase);
        }
        if (lane == 0) pkv_report(p.err, 0, t.s, PKV_VEC_DEVICE_WAIT);
        return;
      }
      uint8_t* unit = ring.base + ring.slot * S::UNIT;
      const unsigned quad = (quads >> (4 * ring.slot)) & 15u;
      const bool whole = quad == 15u && token0 + kUnitTokens <= len;
      unsigned there[2] = {0xffffffffu, 0xffffffffu};  // tokens that are there, one bit each
      if (__builtin_expect(!whole, 0)) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int left = len - token0 - 32 * k;
          there[k] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
          if (!((quad >> (2 * k)) & 1u)) there[k] &= 0xffff0000u;
          if (!((quad >> (2 * k)) & 2u)) there[k] &= 0x0000ffffu;
          // values of absent tokens become zeros (any bytes may lie there; 0 x inf would spoil the sums)
          if (!((there[k] >> lane) & 1u)) {
            uint8_t* sc = unit + (2 * k + (lane >> 4)) * A::BYTES + A::VS + (lane & 15) * A::SROW;
#pragma unroll
            for (int b = 0; b < A::SROW; b += 4) *reinterpret_cast<uint32_t*>(sc + b) = 0u;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      const bool masked = !whole || by_position || token0 + kUnitTokens - 1 > qpos_min ||
                          (p.window > 0 && qpos_max - token0 >= p.window && token0 + kUnitTokens > p.sinks);

      // two atoms at a time, not unrolled: the loop has to stay in the instruction cache
#pragma unroll 1
      for (int k = 0; k < 2; k++, unit += 2 * A::BYTES) {
        float sc[2][NT][4];
#pragma unroll
        for (int a = 0; a < 2; a++) scores_of<D, NT, F32>(unit + a * A::BYTES, lane, qhi, qlo, sc[a]);
        float fac[NT][2];  // what the scores are still to be multiplied by
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) fac[n][e] = factor[n][e];
        if (__builtin_expect(masked, 0)) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) fac[n][e] = 1.0f;
          const unsigned here = k ? there[1] : there[0];
          const int kp0 = k ? kpos[1] : kpos[0];
#pragma unroll
          for (int a = 0; a < 2; a++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
              const int at = 16 * a + 8 * hh + tau(g);
              const int kp = by_position ? __shfl_sync(0xffffffffu, kp0, at) : token0 + 32 * k + at;
              const bool held = (here >> at) & 1u;
#pragma unroll
              for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const int d = pos0 + (row0 + 8 * n + (PAIRED ? 2 * q4 & 3 : 2 * q4) + e) / p.group - kp;
                  const bool see = held && d >= 0 && (p.window == 0 || d < p.window || kp < p.sinks);
                  float& x = sc[a][n][2 * hh + e];
                  x = see ? __fmul_rn(x, factor[n][e]) : -INFINITY;
                }
            }
        }
        if (__builtin_expect(p.scores != nullptr, 0)) {  // for the weights to accumulate, once their sums are known
          float* to = p.scores + (p.c.stat(t.s, t.h) + token0 + 32 * k) * (8 * NT) + 2 * q4;
#pragma unroll
          for (int a = 0; a < 2; a++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
              const int at = 16 * a + 8 * hh + tau(g);
#pragma unroll
              for (int n = 0; n < NT; n++)
                if (token0 + 32 * k + at < len && (!PAIRED || q4 < 2))
                  *reinterpret_cast<float2*>(to + at * (8 * NT) + 8 * n) =
                      make_float2(__fmul_rn(sc[a][n][2 * hh], fac[n][0]), __fmul_rn(sc[a][n][2 * hh + 1], fac[n][1]));
            }
        }
        float top[NT][2];
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            top[n][e] = __fmul_rn(fmaxf(fmaxf(sc[0][n][e], sc[0][n][2 + e]), fmaxf(sc[1][n][e], sc[1][n][2 + e])), fac[n][e]);
            raise = raise || top[n][e] > __fadd_rn(r.m[n][e], kLag);
          }
        if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float x = top[n][e];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              const float m = fmaxf(r.m[n][e], x);
              const float f = r.m[n][e] == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(r.m[n][e], m));
              r.m[n][e] = m;
              r.l[n][e] = __fmul_rn(r.l[n][e], f);
#pragma unroll
              for (int j = 0; j < D / 16; j++) {
                r.o[j][n][e] = __fmul_rn(r.o[j][n][e], f);
                r.o[j][n][2 + e] = __fmul_rn(r.o[j][n][2 + e], f);
              }
            }
        }
        uint32_t pb[2][NT][F32 == 1 ? 4 : 2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float base[2];
#pragma unroll
          for (int e = 0; e < 2; e++) base[e] = r.m[n][e] == -INFINITY ? 0.0f : __fsub_rn(kWeightShift, r.m[n][e]);
#pragma unroll
          for (int a = 0; a < 2; a++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
              const float w0 = exp2_fast(__fmaf_rn(sc[a][n][2 * hh], fac[n][0], base[0]));
              const float w1 = exp2_fast(__fmaf_rn(sc[a][n][2 * hh + 1], fac[n][1], base[1]));
              r.l[n][0] = __fadd_rn(r.l[n][0], w0);
              r.l[n][1] = __fadd_rn(r.l[n][1], w1);
              uint32_t hw = half2_of(w0, w1);
              if constexpr (F32 == 2) {  // lanes of rows 4..7 hold the second terms
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hw));
                const uint32_t rest = half2_of(__fsub_rn(w0, f.x), __fsub_rn(w1, f.y));
                hw = q4 < 2 ? hw : rest;
              }
              pb[a][n][hh] = transpose8(hw);
              if constexpr (F32 == 1) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hw));
                pb[a][n][2 + hh] = transpose8(half2_of(__fsub_rn(w0, f.x), __fsub_rn(w1, f.y)));
              }
            }
        }
        if constexpr (F32) {  // two atoms' sum on its own, then one rounded addition: a long chain would drift by its cut-off bits
          float two[D / 16][NT][4];
          weigh<D, NT, F32, true>(unit, lane, pb[0], two);
          weigh<D, NT, F32, false>(unit + A::BYTES, lane, pb[1], two);
#pragma unroll
          for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int e = 0; e < 4; e++) r.o[j][n][e] = __fadd_rn(r.o[j][n][e], two[j][n][e]);
        } else {
          weigh<D, NT, F32, false>(unit, lane, pb[0], r.o);
          weigh<D, NT, F32, false>(unit + A::BYTES, lane, pb[1], r.o);
        }
      }
      __syncwarp();
      if (issued < count) {  // into the slot that was just read
        issue();
        issued++;
      }
      if (++ring.slot == kStages) ring.slot = 0, ring.phase ^= 1u;
    }
    if constexpr (DIRECT) {
      join_lanes();
      return;
    } else {
      end_tile(v0, n_here);
      at += n_here;
      left_here -= n_here;
      if (left_here == 0) return;
      t.next(p);
      v = 0;
#pragma unroll
      for (int n = 0; n < NT; n++) query_values<D, T>(p, t.s, t.h, t.tile * 8 * NT + 8 * n + (PAIRED ? g & 3 : g), t.rows(p), qx[n]);
    }
  }
}

// CTAs an SM holds: as many as the registers of the sums, the queries and (f32) their second terms leave room for.
__host__ __device__ constexpr int ctas_per_sm(int dim, int nt, bool f32) { return nt == 1 && !(f32 && dim == 128) ? 3 : 2; }

template <int D, int NT, int T, bool DIRECT, bool PAIRED>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(D, NT, T == PKV_DST_F32))
kv4_attend_kernel(const __grid_constant__ AttendParams p) {
  using S = Shared<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float s_ml[DIRECT ? kWarps : 1][8 * NT][2];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int g = lane >> 2, q4 = lane & 3;
  Ring ring = {smem + warp * S::WARP, bars[warp], 0, 0u};
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < kStages; i++) pkv_mbar_init(&bars[warp][i], 1);
  __syncwarp();
  wait_for_stream();
  Sums<D, NT> r;

  if constexpr (DIRECT) {
    // ---- a CTA per row tile
    const int s = blockIdx.z, h = blockIdx.y, tile = blockIdx.x;
    Cursor t;
    t.enter(p, s);
    t.h = h;
    t.tile = tile;
    t.place(p);
    const int row0 = tile * 8 * NT, rows = t.rows(p) - row0;  // rows of this tile that exist (may be more than it holds)
    if (rows <= 0) return;
    stream_units<D, NT, T, true, PAIRED>(p, t, warp, t.span.count > warp ? (t.span.count - warp + kWarps - 1) / kWarps : 0, ring, r);
    if (g == 0)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          s_ml[warp][8 * n + 2 * q4 + e][0] = r.m[n][e];
          s_ml[warp][8 * n + 2 * q4 + e][1] = r.l[n][e];
        }
    __syncwarp();  // every lane has read the ring's last unit
    float* so = reinterpret_cast<float*>(ring.base);  // [8 NT][D + 4]
#pragma unroll
    for (int j = 0; j < D / 16; j++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          *reinterpret_cast<float2*>(so + (8 * n + 2 * q4 + e) * (D + 4) + g * (D / 8) + 2 * j) = make_float2(r.o[j][n][e], r.o[j][n][2 + e]);
    __syncthreads();
    for (int row = warp; row < min(8 * NT, rows); row += kWarps) {
      float m = -INFINITY, l = 0.0f, f[kWarps], x[D / 32];
#pragma unroll
      for (int w = 0; w < kWarps; w++) m = fmaxf(m, s_ml[w][row][0]);
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        f[w] = s_ml[w][row][0] == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(s_ml[w][row][0], m));
        l = __fmaf_rn(f[w], s_ml[w][row][1], l);
      }
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++)
          t = __fmaf_rn(f[w], reinterpret_cast<const float*>(smem + w * S::WARP)[row * (D + 4) + lane * (D / 32) + i], t);
        x[i] = __fmul_rn(t, (i & 1) ? kScaleShift / 16.0f : kScaleShift);
      }
      write_row<T, D / 32>(p, s, h, row0 + row, lane * (D / 32), x, m, l, lane == 0);
    }
  } else {
  // ---- equal runs of all units
  const unsigned run = blockIdx.x * kWarps + warp;
  unsigned units = all_units_of(p, lane);
  const Runs runs = cut_runs(p, units);
  const unsigned at = runs.start(run);
  const int count = (int)(runs.start(run + 1) - at);
  if (count == 0) return;
  // the sequence that unit `at` lies in, 32 at a time
  int s = 0;
  unsigned base = 0;  // units before sequence s
  for (;;) {
    unsigned upto = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + upto > at);
    if (past) {
      const int k = __ffs(past) - 1;
      base += __shfl_sync(0xffffffffu, upto - units, k);
      s += k;
      break;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
    s += 32;
    units = all_units_of(p, s + lane);
  }
  Cursor t;
  t.enter(p, s);
  const unsigned off = at - base, ht = off / (unsigned)t.units;
  t.h = ht / (unsigned)t.tiles;
  t.tile = ht - t.h * t.tiles;
  t.place(p);
  stream_units<D, NT, T, false, PAIRED>(p, t, (int)(off - ht * t.units), count, ring, r, runs, at);
  }
}

// Joins the parts of query rows that were cut: W warps a row (8 for a few long rows, 1 where there are many), each taking
// every W-th part.
template <int D, int NT, int T, int W>
__global__ void __launch_bounds__(kJoinWarps * 32)
kv4_combine_kernel(const __grid_constant__ AttendParams p) {
  constexpr int PER = kJoinWarps / W;  // rows per CTA
  const int s = blockIdx.z, h = blockIdx.y, grow = blockIdx.x * PER + (threadIdx.x >> 5) / W;
  const int tile = grow / (8 * NT), row = grow - tile * (8 * NT);
  wait_for_stream();
  int qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (qn < 0 || qn > p.q.n) qn = 0;
  if (grow >= qn * p.group) return;
  const int2 of = p.part_of[((int64_t)s * p.c.heads + h) * p.row_tiles + tile];
  if (of.y == 1) return;
  // A warp that gave up leaves the entries of the row tiles it never came to as they were in the workspace.  Its parts are
  // not valid, which it has reported, and only entries inside the table are followed.
  if (of.x < 0 || of.y < 1 || of.y > p.runs || of.x > p.runs - of.y) {
    if ((threadIdx.x & 31) == 0) pkv_report(p.err, 0, s, PKV_VEC_DEVICE_WAIT);
    return;
  }
  join_parts<D, T, W>(p, s, h, grow, of.y, [&](int k) { return ((int64_t)(of.x + k) * 2 + (k == 0)) * (8 * NT) + row; });
}

// A row's lse where its weights are accumulated.  A row that is not finite (reported) weighs nothing, like one that sees nothing:
// a single one would otherwise spoil the sums of every token for good.
__device__ __forceinline__ float weighing_lse(const AttendParams& p, int s, int token, int hq) {
  const int64_t at = ((int64_t)s * p.q.n + token) * p.q_heads + hq;
  const float lse = p.lse[at];
  if (pkv_finite(lse) || lse == -INFINITY) return lse;
  pkv_report(p.err, 0, at, PKV_VEC_NONFINITE_INPUT);
  return -INFINITY;
}

// mass[key] += sum over the query rows of exp(score - lse), from the scores that the attention kernel left behind; a thread
// per slot.  One row tile, so a slot's rows are 32 or 64 consecutive bytes.
template <int NT>
__global__ void __launch_bounds__(256)
kv4_mass_of_scores_kernel(const __grid_constant__ AttendParams p) {
  __shared__ float s_lse[8 * NT];
  const int s = blockIdx.z, h = blockIdx.y;
  wait_for_stream();
  const Sequence seq = sequence_of(p, s);
  const int rows = seq.qn * p.group, pos0 = seq.end - seq.qn;
  const Span span = visible_span(p, seq.len, pos0, seq.end - 1);
  if (threadIdx.x < 8 * NT) {
    const int r = threadIdx.x, token = r / p.group, hq = h * p.group + (r - token * p.group);
    s_lse[r] = r < rows ? __fmul_rn(kLog2e, weighing_lse(p, s, token, hq)) : -INFINITY;
  }
  __syncthreads();
  for (int slot = blockIdx.x * 256 + threadIdx.x; slot < seq.len; slot += gridDim.x * 256) {
    const int unit = slot / kUnitTokens;
    if (unit >= span.head && (unit < span.from || unit >= span.from + span.count - span.head)) continue;  // not visited
    const float* x = p.scores + (p.c.stat(s, h) + slot) * (8 * NT);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NT; i += 4) {
      if (i >= rows) break;
      const float4 v = *reinterpret_cast<const float4*>(x + i);
      const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++)  // (a row that sees nothing has no lse; rows behind the last one neither)
        if (s_lse[i + j] != -INFINITY) sum = __fadd_rn(sum, exp2_fast(__fsub_rn(y[j], s_lse[i + j])));
    }
    float* m = p.c.mass + p.c.stat(s, h) + slot;
    *m = __fadd_rn(*m, sum);
  }
}

// The same by a second pass over the keys, for more query rows (or where the scores would not fit the workspace).
//
// A warp keeps 32 tokens' dequantised keys in registers as the A operand of S^T = K Q^T and walks over the rows, so every sum
// has one owner and one order.  The queries come as B operands from shared memory, 64 rows at a time, eight converted by each
// warp: rows are read and converted once for 256 tokens, keys once in all.  Two exponentials, two multiply-adds and two
// additions a score pair are left besides the products.  512 rows over 8192 tokens, 8 heads of 128: 54 us (142 with the keys dequantised
// again for every eight rows); 4096 rows 353 us, 380 with one chain of products an atom and divisions for the rows' positions.
template <int D, int T>
__global__ void __launch_bounds__(kMassWarps * 32, T == PKV_DST_F32 && D == 128 ? 1 : 2)
kv4_mass_kernel(const __grid_constant__ AttendParams p) {
  constexpr bool F32 = T == PKV_DST_F32;
  constexpr int TERMS = F32 ? 2 : 1, PER = kMassWarps * kMassTokens;
  using A = Atom<D>;
  __shared__ uint4 s_q[kMassWarps][TERMS][D / 32][32];
  __shared__ __align__(16) float2 s_row[kMassWarps][8];  // what turns a product into log2 of a weight: factor, offset
  __shared__ int2 s_span[kMassWarps];                    // positions of the first and the last of eight rows
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int g = lane >> 2, q4 = lane & 3;
  const int s = blockIdx.z, h = blockIdx.y;
  wait_for_stream();
  const Sequence seq = sequence_of(p, s);
  const int len = seq.len, qn = seq.qn;
  if (qn == 0) return;
  const int pos0 = seq.end - qn, rows = qn * p.group;
  const bool by_position = p.c.positions != nullptr && (p.window > 0 || qn > 1);
  for (int cta0 = blockIdx.x * PER; cta0 < len; cta0 += gridDim.x * PER) {
    const int token0 = cta0 + warp * kMassTokens;
    unsigned there = token0 >= len ? 0u : token0 + kMassTokens <= len ? 0xffffffffu : (1u << (len - token0)) - 1u;
    uint32_t key[2][D / 32][2][4];  // [atom][16 channels of a lane's D / 4][half atom]
#pragma unroll
    for (int a = 0; a < 2; a++) {
      const uint8_t* atom = token0 + 16 * a < len ? p.c.atom(s, h, token0 / 16 + a, A::BYTES, p.err) : nullptr;
      if (atom) {
        const KeyCodes<D> k(atom, lane);
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
          nibbles(k.w0[j], k.sc0[j >> 1], key[a][j][0]);
          nibbles(k.w1[j], k.sc1[j >> 1], key[a][j][1]);
        }
      } else {
        there &= a ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
        for (int j = 0; j < D / 32; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) key[a][j][0][i] = key[a][j][1][i] = 0u;
      }
    }
    // positions of the keys, their least and greatest
    int kp[2][2], k_min = INT_MAX, k_max = INT_MIN;
    bool held[2][2];
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int hh = 0; hh < 2; hh++) {
        const int t = 16 * a + 8 * hh + tau(g);
        held[a][hh] = (there >> t) & 1u;
        kp[a][hh] = by_position && held[a][hh] ? __ldg(p.c.positions + p.c.stat(s, h) + token0 + t) : token0 + t;
        if (held[a][hh]) {
          k_min = min(k_min, kp[a][hh]);
          k_max = max(k_max, kp[a][hh]);
        }
      }
    k_min = __reduce_min_sync(0xffffffffu, k_min);
    k_max = __reduce_max_sync(0xffffffffu, k_max);
    float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    // causal rows before every key of this CTA are passed over
    int r_first = 0;
    if (!by_position && qn > 1) r_first = (int)min((long long)rows, max(0ll, (long long)cta0 - pos0) * p.group / 8 * 8);
    for (int r0 = r_first; r0 < rows; r0 += 8 * kMassWarps) {
      if (!by_position && p.window > 0 && cta0 >= p.sinks && pos0 + r0 / p.group - (cta0 + PER - 1) >= p.window) break;
      __syncthreads();  // the rows before these have been used
      if (r0 + 8 * warp < rows) {
        uint32_t hi[D / 16][2], lo[D / 16][2];
        float x[D / 4];
        const int r = r0 + 8 * warp + g, token = r / p.group, hq = h * p.group + (r - token * p.group);
        const float lse = r < rows ? weighing_lse(p, s, token, hq) : -INFINITY;
        query_values<D, T>(p, s, h, r, rows, x);
        const float inv = query_operand<D, T>(x, p.negate, hi, lo);
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          if (lse == -INFINITY) {  // a product of 0, whatever the queries are
            hi[2 * i][0] = hi[2 * i][1] = hi[2 * i + 1][0] = hi[2 * i + 1][1] = 0u;
            if constexpr (F32) lo[2 * i][0] = lo[2 * i][1] = lo[2 * i + 1][0] = lo[2 * i + 1][1] = 0u;
          }
          s_q[warp][0][i][lane] = make_uint4(hi[2 * i][0], hi[2 * i][1], hi[2 * i + 1][0], hi[2 * i + 1][1]);
          if constexpr (F32) s_q[warp][TERMS - 1][i][lane] = make_uint4(lo[2 * i][0], lo[2 * i][1], lo[2 * i + 1][0], lo[2 * i + 1][1]);
        }
        if (lane == 0) s_span[warp] = make_int2(pos0 + (r0 + 8 * warp) / p.group, pos0 + min(rows - 1, r0 + 8 * warp + 7) / p.group);
        // (a row that sees nothing, or behind the last one, weighs nothing)
        if (q4 == 0)
          s_row[warp][g] = lse == -INFINITY ? make_float2(0.0f, -INFINITY)
                                            : make_float2(__fmul_rn(__fmul_rn(__fmul_rn(p.scale, kLog2e), kScaleShift), inv),
                                                          -__fmul_rn(kLog2e, lse));
      }
      __syncthreads();
      if (!there) continue;
#pragma unroll 1
      for (int k = 0; k < kMassWarps; k++) {
        const int ra = r0 + 8 * k;
        if (ra >= rows) break;
        const int first = s_span[k].x, last = s_span[k].y;
        if (last < k_min || (p.window > 0 && first - k_max >= p.window && k_min >= p.sinks)) continue;
        // two chains of products an atom (f32 queries: the second terms a third, as in scores_of)
        float sc[2][4], part[2][2][4];
#pragma unroll
        for (int j = 0; j < D / 64; j++) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const int at = j + half * (D / 64);
            const uint4 q = s_q[k][0][at][lane];
#pragma unroll
            for (int a = 0; a < 2; a++) {
              const uint32_t(&w)[2][4] = key[a][at];
              float(&c)[4] = half ? part[a][0] : sc[a];
              if (j == 0) mma_first(c, w[0][0], w[1][0], w[0][1], w[1][1], q.x, q.y);
              else mma(c, w[0][0], w[1][0], w[0][1], w[1][1], q.x, q.y);
              mma(c, w[0][2], w[1][2], w[0][3], w[1][3], q.z, q.w);
            }
            if constexpr (F32) {
              const uint4 q2 = s_q[k][TERMS - 1][at][lane];
#pragma unroll
              for (int a = 0; a < 2; a++) {
                const uint32_t(&w)[2][4] = key[a][at];
                if (at == 0) mma_first(part[a][1], w[0][0], w[1][0], w[0][1], w[1][1], q2.x, q2.y);
                else mma(part[a][1], w[0][0], w[1][0], w[0][1], w[1][1], q2.x, q2.y);
                mma(part[a][1], w[0][2], w[1][2], w[0][3], w[1][3], q2.z, q2.w);
              }
            }
          }
        }
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            sc[a][i] = __fadd_rn(sc[a][i], part[a][0][i]);
            if constexpr (F32) sc[a][i] = __fadd_rn(sc[a][i], part[a][1][i]);
          }
        const float4 f = *reinterpret_cast<const float4*>(&s_row[k][2 * q4]);
        const bool all = there == 0xffffffffu && first >= k_max && (p.window == 0 || last - k_min < p.window) && ra + 8 <= rows;
        if (all) {
#pragma unroll
          for (int a = 0; a < 2; a++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++)
              sum[a][hh] = __fadd_rn(sum[a][hh], __fadd_rn(exp2_fast(__fmaf_rn(sc[a][2 * hh], f.x, f.y)),
                                                           exp2_fast(__fmaf_rn(sc[a][2 * hh + 1], f.z, f.w))));
        } else {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int row = ra + 2 * q4 + e, qpos = pos0 + row / p.group;
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
              for (int hh = 0; hh < 2; hh++) {
                const int d = qpos - kp[a][hh];
                const bool see = row < rows && held[a][hh] && d >= 0 && (p.window == 0 || d < p.window || kp[a][hh] < p.sinks);
                if (see) sum[a][hh] = __fadd_rn(sum[a][hh], exp2_fast(__fmaf_rn(sc[a][2 * hh + e], e ? f.z : f.x, e ? f.w : f.y)));
              }
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int hh = 0; hh < 2; hh++) {
        float t = sum[a][hh];
        t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, 2));
        if (q4 == 0 && held[a][hh]) {
          float* m = p.c.mass + p.c.stat(s, h) + token0 + 16 * a + 8 * hh + tau(g);
          *m = __fadd_rn(*m, t);
        }
      }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
struct Plan {
  int nt, row_tiles, runs;
  int64_t part_rows, tiles;  // rows of partial sums; row tiles of all
  int64_t scores;            // of kv4_mass_of_scores_kernel
  int64_t bytes(int dim) const {
    return scores * (int64_t)sizeof(float) +
           (runs ? part_rows * (dim + 2) * (int64_t)sizeof(float) + tiles * (int64_t)sizeof(int2) : 0);
  }
};

Plan make_plan(const Cache& c, int dim, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  Plan r;
  const int64_t rows = (int64_t)q->n_tokens * (a->n_q_heads / c.heads);
  r.nt = rows > 8 ? 2 : 1;
  r.row_tiles = (int)((rows + 8 * r.nt - 1) / (8 * r.nt));
  int64_t most = c.capacity, longest = a->max_len > 0 && a->max_len < c.capacity ? a->max_len : c.capacity;
  if (a->window > 0 && !c.positions) {  // slots outside the sinks and the window of the query tokens are never visited
    const int64_t seen = (int64_t)a->window + a->sinks + q->n_tokens + 3 * kUnitTokens;
    if (seen < longest) longest = seen;
    if (seen < most) most = seen;
  }
  const int64_t units = (longest + kUnitTokens - 1) / kUnitTokens, most_units = (most + kUnitTokens - 1) / kUnitTokens;
  // Rows of up to six units a warp are not worth a second launch (32 sequences with a window of 1024, 8 kv heads: 17.2 us
  // against 24.4), and with a row for every warp there is nothing to cut while lengths are even (one long sequence among 255 short ones
  // waits for its four warps).
  const int64_t tiles = (int64_t)c.heads * r.row_tiles * c.n_seqs, resident = (int64_t)sm_count() * kWarps * ctas_per_sm(dim, r.nt, q->dtype == PKV_DST_F32);
  r.runs = 0;
  // (the kernel numbers the units of all rows in 32 bits, and max_len may be below the lengths)
  if (units > 6 * kWarps && tiles < kMaxRows && most_units * tiles < (1ll << 31)) {
    const int64_t could = (units * tiles + kWarps - 1) / kWarps * kWarps;
    r.runs = (int)(could < resident ? could : resident);
  }
  r.part_rows = (int64_t)r.runs * 2 * 8 * r.nt;
  r.tiles = tiles;
  // keeping the scores costs 32 bytes a token and kv head each way (eight rows), a second pass over the keys 72 (dim 128) and
  // their dequantisation
  r.scores = a->accumulate && r.row_tiles == 1 ? (int64_t)c.n_seqs * c.heads * c.capacity * 8 * r.nt : 0;
  if (r.scores > kMostScores) r.scores = 0;
  return r;
}

template <int D, int NT, int T>
int launch_join(const AttendParams& p, cudaStream_t s) {
  const bool many = p.runs < 16ll * p.row_tiles * p.c.heads * p.c.n_seqs;  // few parts a row
  return pkv_cuda_status(launch_early(many ? kv4_combine_kernel<D, NT, T, 1> : kv4_combine_kernel<D, NT, T, kJoinWarps>,
                                      dim3(p.row_tiles * 8 * NT / (many ? kJoinWarps : 1), p.c.heads, p.c.n_seqs), kJoinWarps * 32, 0, s,
                                      p));
}

template <int D, int NT, int T>
int launch_attend(const AttendParams& p, cudaStream_t s) {
  auto kernel = p.runs ? kv4_attend_kernel<D, NT, T, false, false> : kv4_attend_kernel<D, NT, T, true, false>;
  // f32 with up to four rows a kv head: paired terms, half the matrix instructions.  8 sequences of 4096 tokens, 32 heads of 64,
  // one row: 32.5 us, 35.5 with the terms in operands of their own; 16 of 8192, 8 heads of 128, four rows: 47.6, 51.9.
  if constexpr (T == PKV_DST_F32 && NT == 1)
    if (p.q.n * p.group <= 4) kernel = p.runs ? kv4_attend_kernel<D, NT, T, false, true> : kv4_attend_kernel<D, NT, T, true, true>;
  constexpr int bytes = Shared<D, NT>::BYTES;
  if (bytes > 48 * 1024)
    if (cudaError_t ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return pkv_cuda_status(ce);
  const dim3 rows(p.row_tiles, p.c.heads, p.c.n_seqs);
  if (cudaError_t ce = launch_early(kernel, p.runs ? dim3(p.runs / kWarps) : rows, kWarps * 32, bytes, s, p)) return pkv_cuda_status(ce);
  return p.runs ? launch_join<D, NT, T>(p, s) : PKV_OK;
}

template <int D, int T>
int launch_all(const AttendParams& p, int nt, bool accumulate, int longest, cudaStream_t s) {
  if (nt == 0) {  // done by the kernel for many rows
  } else if (int st = nt == 1 ? launch_attend<D, 1, T>(p, s) : launch_attend<D, 2, T>(p, s)) {
    return st;
  }
  if (!accumulate || longest <= 0) return PKV_OK;
  if (p.scores)
    return pkv_cuda_status(launch_early(nt == 1 ? kv4_mass_of_scores_kernel<1> : kv4_mass_of_scores_kernel<2>,
                                        dim3((longest + 255) / 256, p.c.heads, p.c.n_seqs), 256, 0, s, p));
  const int per = kMassWarps * kMassTokens;
  return pkv_cuda_status(
      launch_early(kv4_mass_kernel<D, T>, dim3((longest + per - 1) / per, p.c.heads, p.c.n_seqs), kMassWarps * 32, 0, s, p));
}

int check_args(const Cache& c, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  if (!a || a->n_q_heads < 1 || a->n_q_heads % c.heads || a->window < 0 || a->sinks < 0 || a->max_len < 0 ||
      (a->accumulate != 0 && a->accumulate != 1) || !isfinite(a->scale))
    return PKV_ERR_INVALID_ARGUMENT;
  // row numbers are 32-bit
  const int64_t rows = (int64_t)q->n_tokens * (a->n_q_heads / c.heads);
  if (rows > 0x3fffffff) return PKV_ERR_UNSUPPORTED;
  return PKV_OK;
}

}  // namespace

extern "C" int64_t pkv_kv4_attend_workspace_bytes(const pkv_kv4_cache* cache, const pkv_kv4_rows* q_rows,
                                                  const pkv_kv4_attend_args* args) {
  Cache c;
  if (make_cache(cache, &c) || !q_rows || q_rows->n_tokens < 0 || check_args(c, q_rows, args)) return 0;
  if (chunk_takes(q_rows, args->n_q_heads / c.heads)) return chunk_workspace_bytes(c, cache->dim, q_rows, args);
  return make_plan(c, cache->dim, q_rows, args).bytes(cache->dim);
}

namespace {

// What the calls check and set up alike.  `nt`: of the kernel for few rows, 0 where the other takes the call.
struct Call {
  AttendParams p;
  int nt, longest;
};
int make_call(const pkv_kv4_cache* cache, const void* q_dev, const pkv_kv4_rows* q_rows, void* out_dev, const pkv_kv4_rows* out_rows,
              float* lse_dev, const int32_t* q_lens_dev, const pkv_kv4_attend_args* args, void* workspace_dev, int64_t workspace_bytes,
              uint64_t* err_dev, Call* c) {
  AttendParams& p = c->p;
  if (int st = make_cache(cache, &p.c)) return st;
  if (int st = make_rows(q_dev, q_rows, &p.q)) return st;
  if (int st = make_rows(out_dev, out_rows, &p.o)) return st;
  if (int st = check_args(p.c, q_rows, args)) return st;
  if (!err_dev || p.q.n != p.o.n || q_rows->dtype != out_rows->dtype) return PKV_ERR_INVALID_ARGUMENT;
  if (args->accumulate && (!lse_dev || !p.c.mass)) return PKV_ERR_INVALID_ARGUMENT;
  if (p.q.n == 0 || p.c.n_seqs == 0) return PKV_OK;
  // A row tile's queries are read before its outputs are written, by the same CTA or a launch earlier, so out may be q.  The weights
  // of a second pass over the keys are made from the queries after that.
  const int shared = overlap(q_dev, p.q, out_dev, p.o, p.c.n_seqs, args->n_q_heads, cache->dim, q_rows->dtype);
  if (shared == kOverlap || (shared == kSame && args->accumulate)) return PKV_ERR_INVALID_ARGUMENT;
  const bool chunk = chunk_takes(q_rows, args->n_q_heads / p.c.heads);
  Plan plan = {};
  if (!chunk) plan = make_plan(p.c, cache->dim, q_rows, args);
  const int64_t need = chunk ? chunk_workspace_bytes(p.c, cache->dim, q_rows, args) : plan.bytes(cache->dim);
  if (need > workspace_bytes) return PKV_ERR_BUFFER_TOO_SMALL;
  if (need && (!workspace_dev || ((uintptr_t)workspace_dev & 15))) return PKV_ERR_INVALID_ARGUMENT;
  p.q_ptr = q_dev;
  p.o_ptr = out_dev;
  p.lse = lse_dev;
  p.q_lens = q_lens_dev;
  p.scale = fabsf(args->scale);
  p.negate = args->scale < 0.0f;
  p.q_heads = args->n_q_heads;
  p.group = args->n_q_heads / p.c.heads;
  p.window = args->window;
  p.sinks = args->sinks;
  p.row_tiles = plan.row_tiles;
  p.runs = plan.runs;
  p.tile_rows = 8 * plan.nt;
  p.whole_units = p.c.page_atoms % kUnitAtoms == 0;
  p.scores = plan.scores ? (float*)workspace_dev : nullptr;
  p.part_o = (float*)workspace_dev + plan.scores;
  p.part_ml = p.part_o + plan.part_rows * cache->dim;
  p.part_of = (int2*)(p.part_ml + plan.part_rows * 2);
  p.err = err_dev;
  c->nt = plan.nt;
  c->longest = args->max_len > 0 && args->max_len < p.c.capacity ? args->max_len : p.c.capacity;
  return PKV_OK;
}

}  // namespace

extern "C" int pkv_kv4_attend_dev(const pkv_kv4_cache* cache, const void* q_dev, const pkv_kv4_rows* q_rows, void* out_dev,
                                  const pkv_kv4_rows* out_rows, float* lse_dev, const int32_t* q_lens_dev,
                                  const pkv_kv4_attend_args* args, void* workspace_dev, int64_t workspace_bytes,
                                  uint64_t* err_dev, void* stream) {
  Call c;
  if (int st = make_call(cache, q_dev, q_rows, out_dev, out_rows, lse_dev, q_lens_dev, args, workspace_dev, workspace_bytes, err_dev, &c))
    return st;
  const AttendParams& p = c.p;
  if (p.q.n == 0 || p.c.n_seqs == 0) return PKV_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const bool acc = args->accumulate != 0;
  if (c.nt == 0)
    if (int st = launch_chunk(p, cache->dim, q_rows->dtype, q_rows, args, workspace_dev, s)) return st;
  if (cache->dim == 64) {
    switch (q_rows->dtype) {
      case PKV_DST_F32: return launch_all<64, PKV_DST_F32>(p, c.nt, acc, c.longest, s);
      case PKV_DST_F16: return launch_all<64, PKV_DST_F16>(p, c.nt, acc, c.longest, s);
      default: return launch_all<64, PKV_DST_BF16>(p, c.nt, acc, c.longest, s);
    }
  }
  switch (q_rows->dtype) {
    case PKV_DST_F32: return launch_all<128, PKV_DST_F32>(p, c.nt, acc, c.longest, s);
    case PKV_DST_F16: return launch_all<128, PKV_DST_F16>(p, c.nt, acc, c.longest, s);
    default: return launch_all<128, PKV_DST_BF16>(p, c.nt, acc, c.longest, s);
  }
}

extern "C" int pkv_test_kv4_join_dev(const pkv_kv4_cache* cache, const void* q_dev, const pkv_kv4_rows* q_rows, void* out_dev,
                                     const pkv_kv4_rows* out_rows, float* lse_dev, const int32_t* q_lens_dev,
                                     const pkv_kv4_attend_args* args, void* workspace_dev, int64_t workspace_bytes,
                                     uint64_t* err_dev, void* stream) {
  Call c;
  if (int st = make_call(cache, q_dev, q_rows, out_dev, out_rows, lse_dev, q_lens_dev, args, workspace_dev, workspace_bytes, err_dev, &c))
    return st;
  if (c.p.q.n == 0 || c.p.c.n_seqs == 0 || c.nt != 1 || !c.p.runs || cache->dim != 64 || q_rows->dtype != PKV_DST_F32)
    return PKV_ERR_UNSUPPORTED;
  return launch_join<64, 1, PKV_DST_F32>(c.p, (cudaStream_t)stream);
}
