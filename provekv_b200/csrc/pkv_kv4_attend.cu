// Attention over the 4-bit KV cache.
//
// One kernel for a few query rows per kv head (a decode step, short drafts).  A warp works on its own: it streams
// stages of 32 tokens (two atoms: keys and values with their scales in one contiguous run each) through a ring of
// bulk copies and keeps running softmax statistics, so warps never wait for each other before the end.
//
//   S^T = K Q^T     mma m16n8k16: 16 keys x 8 query rows; the A operand is dequantised straight into registers
//   O^T = V^T P^T   16 channels x 8 query rows, contraction over the 16 keys of an atom
//
// With the keys on the M side eight query rows fill a tile (shared heads seldom give more) and the tile costs half the
// products and exponentials that 16 query rows on M would.  P^T is the S^T tile transposed in registers (movmatrix).
// Key row m of a tile is token tau(m) = m/2 (even m) or 7 - m/2 (odd m) of its half atom, the same in both products:
// the order in which the 16-byte pieces of K rows and the 8-byte pieces of V rows fall on distinct banks.
//
// The kernel is bound by HBM (9/8 dim bytes a token) and, close behind, by instruction issue: about 9 instructions
// dequantise 8 values (pkv_kv4.cuh).
#include <math.h>

#include "pkv_kv4.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kWarps = 4;
constexpr int kStageTokens = 32;
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Weights are kept times 2^7 and the running reference may lag the true maximum by 2^8: a weight in binary16 is at most
// 2^15, and one 2^21 below the largest still has all its bits.
constexpr float kWeightShift = 7.0f, kLag = 8.0f;

struct AttendParams {
  Cache c;
  Rows q, o;
  const void* q_ptr;
  void* o_ptr;
  float* lse;
  const int32_t* q_lens;
  float scale;
  int group, q_heads, window, sinks;
  int row_tiles;      // tiles of 8 NT query rows per (sequence, kv head)
  int chunk;          // stages per CTA
  int splits;         // CTAs per (sequence, kv head, row tile)
  float* part_o;      // [tile][split][8 NT][D] unnormalised sums, splits > 1
  float* part_ml;     // [tile][split][8 NT][2] reference and sum
  uint64_t* err;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ int tau(int m) { return (m & 8) | ((m & 1) ? 7 - ((m & 7) >> 1) : (m & 7) >> 1); }

// A row's power of two that brings its largest magnitude to [2^13, 2^14): binary16 then holds a bfloat16 or
// binary16 row exactly but for components below 2^-27 of the largest.
__device__ __forceinline__ float row_power(float amax) {
  if (!(amax > 0.0f) || !pkv_finite(amax)) return 1.0f;
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  int x = 13 - e;
  x = x > 120 ? 120 : x < -120 ? -120 : x;
  return __uint_as_float((uint32_t)(x + 127) << 23);
}

// The B operand of S^T for query row `lane / 4`: this lane's D / 4 channels, in the order nibbles() delivers
// the keys', odd channels divided by 16.  hi (and for f32 queries lo) [2 D / 32][2]; returns the inverse power.
template <int D, int T>
__device__ __forceinline__ float load_query(const typename PkvDst<T>::type* p, int q4, bool live, uint32_t (&hi)[D / 16][2],
                                            uint32_t (&lo)[D / 16][2]) {
  constexpr int CH = D / 4;
  float x[CH];
  if (live) {
    load_f32<T, CH>(p + q4 * CH, x);
  } else {
#pragma unroll
    for (int i = 0; i < CH; i++) x[i] = 0.0f;
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; i++) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float pw = row_power(amax);
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
  return 1.0f / pw;
}

// One atom's scores: S^T[16 keys][8 NT rows] from its K codes and scales in shared memory.
template <int D, int NT, bool F32>
__device__ __forceinline__ void scores_of(const uint8_t* atom, int lane, const uint32_t (&qhi)[NT][D / 16][2],
                                          const uint32_t (&qlo)[NT][D / 16][2], float (&s)[NT][4]) {
  using A = Atom<D>;
  const int q4 = lane & 3, t0 = tau(lane >> 2), t1 = t0 + 8;
  uint32_t w0[D / 32], w1[D / 32];
  Scale sc0[D / 64], sc1[D / 64];
  if constexpr (D == 128) {
    const uint4 a = *reinterpret_cast<const uint4*>(atom + A::KC + t0 * A::ROW + 16 * q4);
    const uint4 b = *reinterpret_cast<const uint4*>(atom + A::KC + t1 * A::ROW + 16 * q4);
    w0[0] = a.x; w0[1] = a.y; w0[2] = a.z; w0[3] = a.w;
    w1[0] = b.x; w1[1] = b.y; w1[2] = b.z; w1[3] = b.w;
    const uint32_t u0 = *reinterpret_cast<const uint16_t*>(atom + A::KS + t0 * A::SROW + 2 * q4);
    const uint32_t u1 = *reinterpret_cast<const uint16_t*>(atom + A::KS + t1 * A::SROW + 2 * q4);
    sc0[0] = scale_of((u0 & 0xffu) * 0x00800080u);
    sc0[1] = scale_of((u0 >> 8) * 0x00800080u);
    sc1[0] = scale_of((u1 & 0xffu) * 0x00800080u);
    sc1[1] = scale_of((u1 >> 8) * 0x00800080u);
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(atom + A::KC + t0 * A::ROW + 8 * q4);
    const uint2 b = *reinterpret_cast<const uint2*>(atom + A::KC + t1 * A::ROW + 8 * q4);
    w0[0] = a.x; w0[1] = a.y;
    w1[0] = b.x; w1[1] = b.y;
    sc0[0] = scale_of((uint32_t)atom[A::KS + t0 * A::SROW + q4] * 0x00800080u);
    sc1[0] = scale_of((uint32_t)atom[A::KS + t1 * A::SROW + q4] * 0x00800080u);
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) s[n][i] = 0.0f;
#pragma unroll
  for (int j = 0; j < D / 32; j++) {
    uint32_t a[4], b[4];
    nibbles(w0[j], sc0[j >> 1], a);
    nibbles(w1[j], sc1[j >> 1], b);
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int n = 0; n < NT; n++) {
        mma(s[n], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], qhi[n][2 * j + u][0], qhi[n][2 * j + u][1]);
        if constexpr (F32)
          mma(s[n], a[2 * u], b[2 * u], a[2 * u + 1], b[2 * u + 1], qlo[n][2 * j + u][0], qlo[n][2 * j + u][1]);
      }
  }
}

// O^T += V^T P^T for one atom; p[n][0..1] is the B operand (f32 queries: p[n][2..3] its remainder).
template <int D, int NT, bool F32>
__device__ __forceinline__ void weigh(const uint8_t* atom, int lane, const uint32_t (&p)[NT][F32 ? 4 : 2], float (&o)[D / 16][NT][4]) {
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
      mma(o[j][n], m[0][2 * j], m[0][2 * j + 1], m[1][2 * j], m[1][2 * j + 1], p[n][0], p[n][1]);
      if constexpr (F32) mma(o[j][n], m[0][2 * j], m[0][2 * j + 1], m[1][2 * j], m[1][2 * j + 1], p[n][2], p[n][3]);
    }
}

// Which tokens a tile of query rows can see, in stages: `head` stages from slot 0 (the sinks), then those from
// stage `from` on, `count` in all.
struct Span {
  int head, from, count;
  __device__ __forceinline__ int stage(int v) const { return v < head ? v : v - head + from; }
};
__device__ __forceinline__ Span visible_span(const AttendParams& p, int len, int end, int pos_first, int pos_last) {
  Span r;
  int stop = len, lo = 0, sink = 0;
  if (!p.c.positions) {  // slots are positions
    stop = min(len, pos_last + 1);
    if (p.window > 0) {
      lo = max(0, pos_first - p.window + 1);
      sink = min(p.sinks, max(stop, 0));
    }
  }
  const int last = (max(stop, 0) + kStageTokens - 1) / kStageTokens;
  r.head = (sink + kStageTokens - 1) / kStageTokens;
  r.from = lo / kStageTokens;
  if (r.from <= r.head) r.from = r.head;
  r.count = r.head + max(0, last - r.from);
  if (r.from == r.head) r.count = last;
  return r;
}

template <int D, int NT>
struct Shared {
  static constexpr int STAGE = 2 * Atom<D>::BYTES;
  static constexpr int RING = kStages * STAGE;
  static constexpr int O_BYTES = 8 * NT * (D + 4) * 4;  // a warp's sums, in the space of its ring
  static constexpr int WARP = RING > O_BYTES ? RING : O_BYTES;
  static constexpr int BYTES = kWarps * WARP;
};

template <int D, int NT, int T>
__global__ void __launch_bounds__(kWarps * 32, (NT == 1 ? 4 : 2))
kv4_attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr bool F32 = T == PKV_DST_F32;
  using A = Atom<D>;
  using S = Shared<D, NT>;
  using E = typename PkvDst<T>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float s_ml[kWarps][8 * NT][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  uint8_t* ring = smem + warp * S::WARP;

  const int split = blockIdx.x, s = blockIdx.z;
  const int h = blockIdx.y / p.row_tiles, tile = blockIdx.y - h * p.row_tiles;
  const int len = p.c.length(s, p.err);
  const int end = p.c.end(s, len);
  int qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (qn < 0 || qn > p.q.n) {
    if (threadIdx.x == 0) pkv_report(p.err, 0, s, PKV_VEC_BAD_SEQUENCE);
    qn = 0;
  }
  const int row0 = tile * 8 * NT, rows = qn * p.group - row0;  // rows of this tile that exist (may be more than it holds)
  if (rows <= 0) return;
  const int pos0 = end - qn;  // position of query token 0
  const int first_token = row0 / p.group, last_token = min(qn - 1, (row0 + 8 * NT - 1) / p.group);
  const Span span = visible_span(p, len, end, pos0 + first_token, pos0 + last_token);
  // the last split takes what is left, should a length be above the caller's hint
  const int v_begin = split * p.chunk, v_end = split == p.splits - 1 ? span.count : min(span.count, v_begin + p.chunk);
  // a later split without work leaves nothing to combine; the first one writes the rows that see nothing
  if (v_begin >= v_end && split > 0) return;

  if (lane == 0)
#pragma unroll
    for (int i = 0; i < kStages; i++) pkv_mbar_init(&bars[warp][i], 1);
  __syncwarp();

  // ---- the stream of stages: this warp takes v_begin + warp, + 4, ...; page numbers are fetched for 16 stages at once,
  // one atom per lane
  const int n_mine = v_end - v_begin > warp ? (v_end - v_begin - warp + kWarps - 1) / kWarps : 0;
  auto stage_of = [&](int i) { return span.stage(v_begin + warp + i * kWarps); };
  auto page_of = [&](int i0) -> const uint8_t* {  // lane l: atom l & 1 of stage i0 + l / 2; null = nothing to load
    const int i = i0 + (lane >> 1);
    if (i >= n_mine) return nullptr;
    const int a = stage_of(i) * 2 + (lane & 1);
    if (a * kAtomTokens >= len) return nullptr;
    return p.c.atom(s, h, a, A::BYTES, p.err);
  };
  const uint8_t* src = page_of(0);       // atoms of the batch being issued
  unsigned live_issue = 0;               // bit l: src of lane l is there (for the batch being issued)
  unsigned live_use = 0;                 // the same for the batch being consumed
  live_issue = __ballot_sync(0xffffffffu, src != nullptr);
  live_use = live_issue;
  auto issue = [&](int i) {  // whole warp; i < n_mine
    if (i && (i & 15) == 0) {
      src = page_of(i);
      live_issue = __ballot_sync(0xffffffffu, src != nullptr);
    }
    const int slot = i % kStages;
    const int l = 2 * (i & 15);
    uint8_t* dst = ring + slot * S::STAGE;
    const unsigned pair = (live_issue >> l) & 3u;
    if ((lane & ~1) == l) {
      if (lane == l) pkv_mbar_expect_tx(&bars[warp][slot], (uint32_t)__popc(pair) * A::BYTES);
    }
    __syncwarp();
    if ((lane & ~1) == l && src) pkv_bulk_load(dst + (lane & 1) * A::BYTES, src, A::BYTES, &bars[warp][slot]);
  };
  int issued = 0;
  for (; issued < min(kStages, n_mine); issued++) issue(issued);

  // ---- queries
  uint32_t qhi[NT][D / 16][2], qlo[NT][D / 16][2];
  float factor[NT][2];  // of the scores of rows 2 q4 and 2 q4 + 1: softmax scale, log2 e, powers of two
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const int r = row0 + 8 * n + g, token = r / p.group, hq = h * p.group + (r - token * p.group);
    const bool live = 8 * n + g < rows;
    const E* qp = reinterpret_cast<const E*>(p.q_ptr) + s * p.q.seq + (int64_t)token * p.q.token + hq * p.q.head;
    const float inv = load_query<D, T>(qp, q4, live, qhi[n], qlo[n]);
    const float f = __fmul_rn(__fmul_rn(p.scale, kLog2e), kScaleShift);
#pragma unroll
    for (int e = 0; e < 2; e++) factor[n][e] = __fmul_rn(f, __shfl_sync(0xffffffffu, inv, 4 * (2 * q4 + e)));
  }
  int qpos[NT][2];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++) qpos[n][e] = pos0 + (row0 + 8 * n + 2 * q4 + e) / p.group;
  const int qpos_min = pos0 + first_token, qpos_max = pos0 + last_token;
  // positions matter only where a row can see less than everything that is held
  const bool by_position = p.c.positions != nullptr && (p.window > 0 || qn > 1);
  const int32_t* positions = by_position ? p.c.positions + p.c.stat(s, h) : nullptr;

  float o[D / 16][NT][4];
  float m_ref[NT][2], l_sum[NT][2];
#pragma unroll
  for (int j = 0; j < D / 16; j++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[j][n][i] = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      m_ref[n][e] = -INFINITY;
      l_sum[n][e] = 0.0f;
    }

  bool fine = true;
  int done = 0;
  for (; done < n_mine; done++) {
    const int slot = done % kStages;
    if (done && (done & 15) == 0) live_use = live_issue;  // issue() of this batch's first stage has run
    const int token0 = stage_of(done) * kStageTokens;
    int kpos = 0;
    if (by_position && token0 + lane < len) kpos = __ldg(positions + token0 + lane);
    const unsigned pair = (live_use >> (2 * (done & 15))) & 3u;
    if (!__all_sync(0xffffffffu, pkv_mbar_wait(&bars[warp][slot], (uint32_t)(done / kStages) & 1u))) {
      fine = false;
      break;
    }
    uint8_t* stage = ring + slot * S::STAGE;
    // tokens that are there, one bit each
    unsigned there = token0 + kStageTokens <= len ? 0xffffffffu : (1u << (len - token0)) - 1u;
    if (!(pair & 1u)) there &= 0xffff0000u;
    if (!(pair & 2u)) there &= 0x0000ffffu;
    if (there != 0xffffffffu) {
      // values of absent tokens become zeros (any bytes may lie there; 0 x inf would spoil the sums)
      if (!((there >> lane) & 1u)) {
        uint8_t* sc = stage + (lane >> 4) * A::BYTES + A::VS + (lane & 15) * A::SROW;
#pragma unroll
        for (int i = 0; i < A::SROW; i += 4) *reinterpret_cast<uint32_t*>(sc + i) = 0u;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    const bool masked = there != 0xffffffffu || by_position || token0 + kStageTokens - 1 > qpos_min ||
                        (p.window > 0 && qpos_max - token0 >= p.window && token0 + kStageTokens > p.sinks);

    float sc[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; a++) scores_of<D, NT, F32>(stage + a * A::BYTES, lane, qhi, qlo, sc[a]);
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) top[n][e] = -INFINITY;
    if (masked) {
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
          const int t = 16 * a + 8 * hh + tau(g);
          const int kp = by_position ? __shfl_sync(0xffffffffu, kpos, t) : token0 + t;
          const bool held = (there >> t) & 1u;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int d = qpos[n][e] - kp;
              const bool see = held && d >= 0 && (p.window == 0 || d < p.window || kp < p.sinks);
              float& x = sc[a][n][2 * hh + e];
              x = see ? __fmul_rn(x, factor[n][e]) : -INFINITY;
              top[n][e] = fmaxf(top[n][e], x);
            }
        }
    } else {
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            sc[a][n][i] = __fmul_rn(sc[a][n][i], factor[n][i & 1]);
            top[n][i & 1] = fmaxf(top[n][i & 1], sc[a][n][i]);
          }
    }
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) raise = raise || top[n][e] > __fadd_rn(m_ref[n][e], kLag);
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float t = top[n][e];
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
          const float m = fmaxf(m_ref[n][e], t);
          const float f = m_ref[n][e] == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(m_ref[n][e], m));
          m_ref[n][e] = m;
          l_sum[n][e] = __fmul_rn(l_sum[n][e], f);
#pragma unroll
          for (int j = 0; j < D / 16; j++) {
            o[j][n][e] = __fmul_rn(o[j][n][e], f);
            o[j][n][2 + e] = __fmul_rn(o[j][n][2 + e], f);
          }
        }
    }
    uint32_t pb[2][NT][F32 ? 4 : 2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float base[2];
#pragma unroll
      for (int e = 0; e < 2; e++) base[e] = m_ref[n][e] == -INFINITY ? 0.0f : __fsub_rn(m_ref[n][e], kWeightShift);
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
          const float w0 = exp2_fast(__fsub_rn(sc[a][n][2 * hh], base[0]));
          const float w1 = exp2_fast(__fsub_rn(sc[a][n][2 * hh + 1], base[1]));
          l_sum[n][0] = __fadd_rn(l_sum[n][0], w0);
          l_sum[n][1] = __fadd_rn(l_sum[n][1], w1);
          const uint32_t hw = half2_of(w0, w1);
          pb[a][n][hh] = transpose8(hw);
          if constexpr (F32) {
            const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&hw));
            pb[a][n][2 + hh] = transpose8(half2_of(__fsub_rn(w0, r.x), __fsub_rn(w1, r.y)));
          }
        }
    }
#pragma unroll
    for (int a = 0; a < 2; a++) weigh<D, NT, F32>(stage + a * A::BYTES, lane, pb[a], o);
    __syncwarp();
    if (issued < n_mine) issue(issued++);
  }
  if (!fine) {  // a copy never arrived: give the others their time, report, and leave nothing behind
    for (int i = done + 1; i < issued; i++) pkv_mbar_wait(&bars[warp][i % kStages], (uint32_t)(i / kStages) & 1u);
    if (lane == 0) pkv_report(p.err, 0, s, PKV_VEC_DEVICE_WAIT);
  }

  // ---- the four warps' sums become one
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float t = l_sum[n][e];
      t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, 4));
      t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, 8));
      t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, 16));
      if (g == 0) {
        s_ml[warp][8 * n + 2 * q4 + e][0] = m_ref[n][e];
        s_ml[warp][8 * n + 2 * q4 + e][1] = t;
      }
    }
  float* so = reinterpret_cast<float*>(ring);  // [8 NT][D + 4]
#pragma unroll
  for (int j = 0; j < D / 16; j++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) so[(8 * n + 2 * q4 + (i & 1)) * (D + 4) + g * (D / 8) + 2 * j + (i >> 1)] = o[j][n][i];
  __syncthreads();
  const int held_rows = min(8 * NT, rows);
  for (int r = warp; r < held_rows; r += kWarps) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; w++) m = fmaxf(m, s_ml[w][r][0]);
    float l = 0.0f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      f[w] = s_ml[w][r][0] == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(s_ml[w][r][0], m));
      l = __fmaf_rn(f[w], s_ml[w][r][1], l);
    }
    float x[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++)
        t = __fmaf_rn(f[w], reinterpret_cast<const float*>(smem + w * S::WARP)[r * (D + 4) + lane * (D / 32) + i], t);
      // undo the scale shift and the 16 of odd channels
      x[i] = __fmul_rn(t, (i & 1) ? kScaleShift / 16.0f : kScaleShift);
    }
    if (p.splits > 1) {
      const int64_t at = (((int64_t)s * gridDim.y + blockIdx.y) * p.splits + split) * (8 * NT) + r;
      float* dst = p.part_o + at * D + lane * (D / 32);
      if constexpr (D == 128) *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
      else *reinterpret_cast<float2*>(dst) = make_float2(x[0], x[1]);
      if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
    } else {
      const int rr = row0 + r, token = rr / p.group, hq = h * p.group + (rr - token * p.group);
      const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
      E* dst = reinterpret_cast<E*>(p.o_ptr) + s * p.o.seq + (int64_t)token * p.o.token + hq * p.o.head + lane * (D / 32);
#pragma unroll
      for (int i = 0; i < D / 32; i += 2) {
        const float a = __fmul_rn(x[i], inv), b = __fmul_rn(x[i + 1], inv);
        if constexpr (F32) *reinterpret_cast<float2*>(dst + i) = make_float2(a, b);
        else *reinterpret_cast<uint32_t*>(dst + i) = pkv_pack2<T>(a, b);
      }
      if (p.lse && lane == 0)
        p.lse[((int64_t)s * p.q.n + token) * p.q_heads + hq] =
            l == 0.0f ? -INFINITY : __fmul_rn(kLn2, __fadd_rn(m, __fsub_rn(log2f(l), kWeightShift)));
    }
  }
}

// Joins the splits of a row: one CTA per query row, a warp takes every fourth split.
template <int D, int NT, int T>
__global__ void __launch_bounds__(128)
kv4_combine_kernel(const __grid_constant__ AttendParams p) {
  using E = typename PkvDst<T>::type;
  __shared__ float s_o[4][D];
  __shared__ float s_ml[4][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = blockIdx.z, r = blockIdx.x % (8 * NT), tile = blockIdx.x / (8 * NT), h = blockIdx.y;
  const int len = p.c.length(s, p.err), end = p.c.end(s, len);
  int qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (qn < 0 || qn > p.q.n) qn = 0;
  const int row0 = tile * 8 * NT;
  if (row0 + r >= qn * p.group) return;
  const int first_token = row0 / p.group, last_token = min(qn - 1, (row0 + 8 * NT - 1) / p.group);
  const Span span = visible_span(p, len, end, end - qn + first_token, end - qn + last_token);
  const int n = min(p.splits, max(1, (span.count + p.chunk - 1) / p.chunk));  // splits that had work (the first always writes)
  const int64_t base = (((int64_t)s * p.c.heads + h) * p.row_tiles + tile) * p.splits * (8 * NT) + r;
  float m = -INFINITY, l = 0.0f, x[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; i++) x[i] = 0.0f;
  for (int w = warp; w < n; w += 4) {
    const int64_t at = base + (int64_t)w * (8 * NT);
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    float y[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; i++) y[i] = p.part_o[at * D + lane * (D / 32) + i];
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;
    const float top = fmaxf(m, ml.x);
    const float fa = m == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(m, top)), fb = exp2_fast(__fsub_rn(ml.x, top));
    m = top;
    l = __fmaf_rn(l, fa, __fmul_rn(ml.y, fb));
#pragma unroll
    for (int i = 0; i < D / 32; i++) x[i] = __fmaf_rn(x[i], fa, __fmul_rn(y[i], fb));
  }
#pragma unroll
  for (int i = 0; i < D / 32; i++) s_o[warp][lane * (D / 32) + i] = x[i];
  if (lane == 0) {
    s_ml[warp][0] = m;
    s_ml[warp][1] = l;
  }
  __syncthreads();
  if (threadIdx.x * 2 >= D) return;
  float top = -INFINITY, sum = 0.0f, a = 0.0f, b = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w][0]);
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float f = s_ml[w][0] == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(s_ml[w][0], top));
    sum = __fmaf_rn(f, s_ml[w][1], sum);
    a = __fmaf_rn(f, s_o[w][2 * threadIdx.x], a);
    b = __fmaf_rn(f, s_o[w][2 * threadIdx.x + 1], b);
  }
  const int rr = row0 + r, token = rr / p.group, hq = h * p.group + (rr - token * p.group);
  const float inv = sum > 0.0f ? __fdiv_rn(1.0f, sum) : (sum == 0.0f ? 0.0f : sum);
  E* dst = reinterpret_cast<E*>(p.o_ptr) + s * p.o.seq + (int64_t)token * p.o.token + hq * p.o.head + 2 * threadIdx.x;
  if constexpr (T == PKV_DST_F32) *reinterpret_cast<float2*>(dst) = make_float2(__fmul_rn(a, inv), __fmul_rn(b, inv));
  else *reinterpret_cast<uint32_t*>(dst) = pkv_pack2<T>(__fmul_rn(a, inv), __fmul_rn(b, inv));
  if (p.lse && threadIdx.x == 0)
    p.lse[((int64_t)s * p.q.n + token) * p.q_heads + hq] =
        sum == 0.0f ? -INFINITY : __fmul_rn(kLn2, __fadd_rn(top, __fsub_rn(log2f(sum), kWeightShift)));
}

// mass[key] += sum over the query rows of exp(score - lse).  A warp keeps the dequantised keys of 32 tokens in
// registers and walks over the rows, so every sum has one owner and one order.
template <int D, int T>
__global__ void __launch_bounds__(kWarps * 32)
kv4_mass_kernel(const __grid_constant__ AttendParams p) {
  constexpr bool F32 = T == PKV_DST_F32;
  using A = Atom<D>;
  using E = typename PkvDst<T>::type;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  const int s = blockIdx.z, h = blockIdx.y;
  const int len = p.c.length(s, p.err), end = p.c.end(s, len);
  int qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (qn < 0 || qn > p.q.n) qn = 0;
  if (qn == 0) return;
  const int pos0 = end - qn, rows = qn * p.group;
  for (int token0 = (blockIdx.x * kWarps + warp) * kStageTokens; token0 < len; token0 += gridDim.x * kWarps * kStageTokens) {
  const uint8_t* atom[2];
  unsigned there = token0 + kStageTokens <= len ? 0xffffffffu : (1u << (len - token0)) - 1u;
#pragma unroll
  for (int a = 0; a < 2; a++) {
    atom[a] = token0 + 16 * a < len ? p.c.atom(s, h, token0 / 16 + a, A::BYTES, p.err) : nullptr;
    if (!atom[a]) there &= a ? 0x0000ffffu : 0xffff0000u;
  }
  if (!there) continue;
  const bool by_position = p.c.positions != nullptr && (p.window > 0 || qn > 1);
  int kp[2][2];
  bool held[2][2];
#pragma unroll
  for (int a = 0; a < 2; a++)
#pragma unroll
    for (int hh = 0; hh < 2; hh++) {
      const int t = 16 * a + 8 * hh + tau(g);
      held[a][hh] = (there >> t) & 1u;
      kp[a][hh] = by_position && held[a][hh] ? p.c.positions[p.c.stat(s, h) + token0 + t] : token0 + t;
    }
  float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
  // rows of 8 at a time; a causal row before every key of this warp is passed over
  int r_first = 0;
  if (!by_position && qn > 1) r_first = max(0, token0 - pos0) * p.group / 8 * 8;
  for (int r0 = r_first; r0 < rows; r0 += 8) {
    if (!by_position && p.window > 0 && token0 >= p.sinks && pos0 + r0 / p.group - (token0 + kStageTokens - 1) >= p.window) break;
    uint32_t qhi[1][D / 16][2], qlo[1][D / 16][2];
    const int r = r0 + g, token = r / p.group, hq = h * p.group + (r - token * p.group);
    const E* qp = reinterpret_cast<const E*>(p.q_ptr) + s * p.q.seq + (int64_t)token * p.q.token + hq * p.q.head;
    const float inv = load_query<D, T>(qp, q4, r < rows, qhi[0], qlo[0]);
    const float lse = r < rows ? p.lse[((int64_t)s * p.q.n + token) * p.q_heads + hq] : -INFINITY;
    const float f = __fmul_rn(__fmul_rn(__fmul_rn(p.scale, kLog2e), kScaleShift), inv);
    float factor[2], base[2];
    int qpos[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      factor[e] = __shfl_sync(0xffffffffu, f, 4 * (2 * q4 + e));
      base[e] = __fmul_rn(kLog2e, __shfl_sync(0xffffffffu, lse, 4 * (2 * q4 + e)));
      qpos[e] = pos0 + (r0 + 2 * q4 + e) / p.group;
    }
#pragma unroll
    for (int a = 0; a < 2; a++) {
      if (!atom[a]) continue;
      float sc[1][4];
      scores_of<D, 1, F32>(atom[a], lane, qhi, qlo, sc);
#pragma unroll
      for (int hh = 0; hh < 2; hh++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int d = qpos[e] - kp[a][hh];
          const bool see = r0 + 2 * q4 + e < rows && held[a][hh] && d >= 0 &&
                           (p.window == 0 || d < p.window || kp[a][hh] < p.sinks);
          const float w = see ? exp2_fast(__fsub_rn(__fmul_rn(sc[0][2 * hh + e], factor[e]), base[e])) : 0.0f;
          sum[a][hh] = __fadd_rn(sum[a][hh], w);
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
  int nt, row_tiles, chunk, splits;
  int64_t part_rows;  // rows of partial sums, 0 without a split
};

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

Plan make_plan(const Cache& c, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  Plan r;
  const int64_t rows = (int64_t)q->n_tokens * (a->n_q_heads / c.heads);
  r.nt = rows > 8 ? 2 : 1;
  r.row_tiles = (int)((rows + 8 * r.nt - 1) / (8 * r.nt));
  int64_t longest = a->max_len > 0 && a->max_len < c.capacity ? a->max_len : c.capacity;
  if (a->window > 0 && !c.positions) {  // slots outside the sinks and the window of a tile's tokens are never visited
    const int64_t seen = (int64_t)a->window + a->sinks + q->n_tokens + 4 * kStageTokens;
    if (seen < longest) longest = seen;
  }
  const int64_t stages = (longest + kStageTokens - 1) / kStageTokens;
  const int64_t tiles = (int64_t)c.n_seqs * c.heads * r.row_tiles;
  // enough CTAs for every SM to hold its four, and at least four stages for each of a CTA's warps
  const int64_t want = (int64_t)sm_count() * (r.nt == 1 ? 4 : 2);
  int64_t chunk = (stages * tiles + want - 1) / want;
  if (chunk < 4 * kWarps) chunk = 4 * kWarps;
  if (chunk > stages) chunk = stages > 0 ? stages : 1;
  r.chunk = (int)((chunk + kWarps - 1) / kWarps * kWarps);
  r.splits = (int)((stages + r.chunk - 1) / r.chunk);
  if (r.splits < 1) r.splits = 1;
  r.part_rows = r.splits > 1 ? tiles * r.splits * 8 * r.nt : 0;
  return r;
}

template <int D, int NT, int T>
int launch_attend(const AttendParams& p, cudaStream_t s) {
  auto kernel = kv4_attend_kernel<D, NT, T>;
  constexpr int bytes = Shared<D, NT>::BYTES;
  if (bytes > 48 * 1024)
    if (cudaError_t ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return pkv_cuda_status(ce);
  kernel<<<dim3(p.splits, p.c.heads * p.row_tiles, p.c.n_seqs), kWarps * 32, bytes, s>>>(p);
  pkv_count_launch();
  if (cudaError_t ce = cudaGetLastError()) return pkv_cuda_status(ce);
  if (p.splits > 1) {
    kv4_combine_kernel<D, NT, T><<<dim3(p.row_tiles * 8 * NT, p.c.heads, p.c.n_seqs), 128, 0, s>>>(p);
    pkv_count_launch();
  }
  return pkv_cuda_status(cudaGetLastError());
}

template <int D, int T>
int launch_all(const AttendParams& p, int nt, bool accumulate, int longest, cudaStream_t s) {
  if (int st = nt == 1 ? launch_attend<D, 1, T>(p, s) : launch_attend<D, 2, T>(p, s)) return st;
  if (accumulate && longest > 0) {
    const int per = kWarps * kStageTokens;
    kv4_mass_kernel<D, T><<<dim3((longest + per - 1) / per, p.c.heads, p.c.n_seqs), kWarps * 32, 0, s>>>(p);
    pkv_count_launch();
  }
  return pkv_cuda_status(cudaGetLastError());
}

int check_args(const Cache& c, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  if (!a || a->n_q_heads < 1 || a->n_q_heads % c.heads || a->window < 0 || a->sinks < 0 || a->max_len < 0 ||
      (a->accumulate != 0 && a->accumulate != 1) || !isfinite(a->scale))
    return PKV_ERR_INVALID_ARGUMENT;
  // row numbers are 32-bit, and heads x row tiles is a grid dimension
  const int64_t rows = (int64_t)q->n_tokens * (a->n_q_heads / c.heads);
  if (rows > 0x3fffffff || (rows / 8 + 1) * c.heads > 65535) return PKV_ERR_UNSUPPORTED;
  return PKV_OK;
}

}  // namespace

extern "C" int64_t pkv_kv4_attend_workspace_bytes(const pkv_kv4_cache* cache, const pkv_kv4_rows* q_rows,
                                                  const pkv_kv4_attend_args* args) {
  Cache c;
  if (make_cache(cache, &c) || !q_rows || q_rows->n_tokens < 0 || check_args(c, q_rows, args)) return 0;
  return make_plan(c, q_rows, args).part_rows * (cache->dim + 2) * (int64_t)sizeof(float);
}

extern "C" int pkv_kv4_attend_dev(const pkv_kv4_cache* cache, const void* q_dev, const pkv_kv4_rows* q_rows, void* out_dev,
                                  const pkv_kv4_rows* out_rows, float* lse_dev, const int32_t* q_lens_dev,
                                  const pkv_kv4_attend_args* args, void* workspace_dev, int64_t workspace_bytes,
                                  uint64_t* err_dev, void* stream) {
  AttendParams p;
  if (int st = make_cache(cache, &p.c)) return st;
  if (int st = make_rows(q_dev, q_rows, &p.q)) return st;
  if (int st = make_rows(out_dev, out_rows, &p.o)) return st;
  if (int st = check_args(p.c, q_rows, args)) return st;
  if (!err_dev || p.q.n != p.o.n || q_rows->dtype != out_rows->dtype) return PKV_ERR_INVALID_ARGUMENT;
  if (args->accumulate && (!lse_dev || !p.c.mass)) return PKV_ERR_INVALID_ARGUMENT;
  if (p.q.n == 0 || p.c.n_seqs == 0) return PKV_OK;
  const Plan plan = make_plan(p.c, q_rows, args);
  if (plan.part_rows * (cache->dim + 2) * (int64_t)sizeof(float) > workspace_bytes) return PKV_ERR_BUFFER_TOO_SMALL;
  if (plan.part_rows && (!workspace_dev || ((uintptr_t)workspace_dev & 15))) return PKV_ERR_INVALID_ARGUMENT;
  p.q_ptr = q_dev;
  p.o_ptr = out_dev;
  p.lse = lse_dev;
  p.q_lens = q_lens_dev;
  p.scale = args->scale;
  p.q_heads = args->n_q_heads;
  p.group = args->n_q_heads / p.c.heads;
  p.window = args->window;
  p.sinks = args->sinks;
  p.row_tiles = plan.row_tiles;
  p.chunk = plan.chunk;
  p.splits = plan.splits;
  p.part_o = (float*)workspace_dev;
  p.part_ml = p.part_o + plan.part_rows * cache->dim;
  p.err = err_dev;
  const int longest = args->max_len > 0 && args->max_len < p.c.capacity ? args->max_len : p.c.capacity;
  cudaStream_t s = (cudaStream_t)stream;
  const bool acc = args->accumulate != 0;
  if (cache->dim == 64) {
    switch (q_rows->dtype) {
      case PKV_DST_F32: return launch_all<64, PKV_DST_F32>(p, plan.nt, acc, longest, s);
      case PKV_DST_F16: return launch_all<64, PKV_DST_F16>(p, plan.nt, acc, longest, s);
      default: return launch_all<64, PKV_DST_BF16>(p, plan.nt, acc, longest, s);
    }
  }
  switch (q_rows->dtype) {
    case PKV_DST_F32: return launch_all<128, PKV_DST_F32>(p, plan.nt, acc, longest, s);
    case PKV_DST_F16: return launch_all<128, PKV_DST_F16>(p, plan.nt, acc, longest, s);
    default: return launch_all<128, PKV_DST_BF16>(p, plan.nt, acc, longest, s);
  }
}
