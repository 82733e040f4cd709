// What the two attention kernels over the 4-bit cache share: the arguments, what a query can see, softmax constants, the
// last step of a row.
#pragma once

#include <math.h>

#include "pkv_kv4.cuh"

namespace pkv_kv4 {

constexpr int kUnitAtoms = 4, kUnitTokens = kUnitAtoms * kAtomTokens;
constexpr int kJoinWarps = 8;
constexpr int kBatch = 32 / kUnitAtoms;  // units whose page numbers a warp fetches at once
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
  float scale;        // its magnitude
  int negate;         // its sign
  int group, q_heads, window, sinks;
  int row_tiles;      // tiles of 8 NT query rows per (sequence, kv head)
  int runs;           // warps that share the units of all rows; 0: a CTA per row tile
  int tile_rows;      // query rows of a tile, 8 NT
  int whole_units;    // 1: a unit never crosses a page, one copy brings it
  float* part_o;      // [run][2][8 NT][D] unnormalised sums of a run's first and last row, where it has only a part of it
  float* part_ml;     // [run][2][8 NT][2] reference and sum
  int2* part_of;      // [sequence][kv head][row tile] first run and number of runs that have a part of it
  float* scores;      // accumulating, one row tile: [sequence][kv head][slot][8 NT] scaled scores (log2), else null
  uint64_t* err;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// A row's power of two that brings its largest magnitude to [2^13, 2^14): binary16 then holds a bfloat16 or
// binary16 row exactly but for components below 2^-27 of the largest.
__device__ __forceinline__ float row_power(float amax) {
  if (!(amax > 0.0f) || !pkv_finite(amax)) return 1.0f;
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  int x = 13 - e;
  x = x > 120 ? 120 : x < -120 ? -120 : x;
  return __uint_as_float((uint32_t)(x + 127) << 23);
}

// Which tokens a tile of query rows can see, in units: `head` units from slot 0 (the sinks), then those from unit
// `from` on, `count` in all.
struct Span {
  int head, from, count;
  __device__ __forceinline__ int unit(int v) const { return v < head ? v : v - head + from; }
};
__device__ __forceinline__ Span visible_span(const AttendParams& p, int len, int pos_first, int pos_last) {
  Span r;
  int stop = len, lo = 0, sink = 0;
  if (!p.c.positions) {  // slots are positions
    stop = max(0, min(len, pos_last + 1));
    if (p.window > 0) {
      lo = (int)max(0ll, (long long)pos_first - p.window + 1);
      sink = min(p.sinks, stop);
    }
  }
  const int last = (stop + kUnitTokens - 1) / kUnitTokens;
  r.head = (sink + kUnitTokens - 1) / kUnitTokens;
  r.from = lo / kUnitTokens;
  if (r.from <= r.head) r.from = r.head;
  r.count = r.from == r.head ? last : r.head + max(0, last - r.from);
  return r;
}

// A sequence as the kernels see it: bad lengths are reported and count as empty.
struct Sequence {
  int len, end, qn;
};
__device__ __forceinline__ Sequence sequence_of(const AttendParams& p, int s) {
  Sequence r;
  r.len = p.c.length(s, p.err);
  r.end = p.c.end(s, r.len, p.err);
  r.qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (r.qn < 0 || r.qn > p.q.n) {
    pkv_report(p.err, 0, s, PKV_VEC_BAD_SEQUENCE);
    r.qn = 0;
  }
  return r;
}
// Writes N channels of a row, sums x (scale and the 16 of odd channels already undone) over l.
template <int T, int N>
__device__ __forceinline__ void write_row(const AttendParams& p, int s, int h, int row, int channel, const float (&x)[N], float m, float l,
                                          bool first) {
  using E = typename PkvDst<T>::type;
  const int token = row / p.group, hq = h * p.group + (row - token * p.group);
  const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
  E* dst = reinterpret_cast<E*>(p.o_ptr) + s * p.o.seq + (int64_t)token * p.o.token + hq * p.o.head + channel;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = __fmul_rn(x[i], inv);
  if constexpr (T == PKV_DST_F32 ? N % 4 == 0 : N % 8 == 0) {
    store_f32<T, N>(dst, y);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (T == PKV_DST_F32) *reinterpret_cast<float2*>(dst + i) = make_float2(y[i], y[i + 1]);
      else *reinterpret_cast<uint32_t*>(dst + i) = pkv_pack2<T>(y[i], y[i + 1]);
    }
  }
  if (p.lse && first)
    p.lse[((int64_t)s * p.q.n + token) * p.q_heads + hq] =
        l == 0.0f ? -INFINITY : __fmul_rn(kLn2, __fadd_rn(m, __fsub_rn(log2f(l), kWeightShift)));
}

// Joins the parts of query row `row` and writes it: W warps of a CTA (all of it, or one warp alone), each every W-th part.
// slot_of(k): which row of part_o and part_ml is part k's.
template <int D, int T, int W, typename SlotOf>
__device__ __forceinline__ void join_parts(const AttendParams& p, int s, int h, int row, int parts, SlotOf slot_of) {
  constexpr int N = D / 32;
  __shared__ float s_x[W > 1 ? W : 1][D], s_ml[W > 1 ? W : 1][2];
  const int lane = threadIdx.x & 31, warp = W > 1 ? threadIdx.x >> 5 : 0;
  float m = -INFINITY, l = 0.0f, x[N];
#pragma unroll
  for (int i = 0; i < N; i++) x[i] = 0.0f;
  // a warp's parts: k = warp + W j; references of 32 of them at a time, then the sums, eight loads in flight
  for (int k0 = warp; k0 < parts; k0 += 32 * W) {
    const int n = min(32, (parts - k0 + W - 1) / W);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(p.part_ml + slot_of(k0 + lane * W) * 2);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(top, m);
    const float fold = m == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(m, top));
    // (a part without a visible key, or with nothing but NaN, has no reference)
    const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : ml.y) : exp2_fast(__fsub_rn(ml.x, top));
    float sum = __fmul_rn(f, ml.y);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    l = __fmaf_rn(l, fold, sum);
    m = top;
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = __fmul_rn(x[i], fold);
#pragma unroll 8
    for (int j = 0; j < n; j++) {
      const float fj = __shfl_sync(0xffffffffu, f, j);
      const float* src = p.part_o + slot_of(k0 + j * W) * D + lane * N;
      float y[N];
      if constexpr (N == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        y[0] = v.x; y[1] = v.y;
      }
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = __fmaf_rn(fj, y[i], x[i]);
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < N; i++) s_x[warp][lane * N + i] = x[i];
    if (lane == 0) {
      s_ml[warp][0] = m;
      s_ml[warp][1] = l;
    }
    __syncthreads();
    if (warp) return;
    const int w = lane & (W - 1);
    m = s_ml[w][0];
#pragma unroll
    for (int o = W / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float f = s_ml[w][0] == -INFINITY ? (s_ml[w][1] == 0.0f ? 0.0f : s_ml[w][1]) : exp2_fast(__fsub_rn(s_ml[w][0], m));
    l = __fmul_rn(f, s_ml[w][1]);
#pragma unroll
    for (int o = W / 2; o; o >>= 1) l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, o));
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) {
      const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = __fmaf_rn(fk, s_x[k][lane * N + i], x[i]);
    }
  }
  write_row<T, N>(p, s, h, row, lane * N, x, m, l, lane == 0);
}

inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// pkv_kv4_chunk.cu: the kernel for many query rows per kv head (16-bit queries).  Whether it takes a call, its workspace,
// and the launch.
bool chunk_takes(const pkv_kv4_rows* q, int group);
int64_t chunk_workspace_bytes(const Cache& c, int dim, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a);
int launch_chunk(AttendParams p, int dim, int dtype, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a, void* workspace,
                 cudaStream_t s);

}  // namespace pkv_kv4
