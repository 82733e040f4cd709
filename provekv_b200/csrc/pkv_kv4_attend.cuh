// What the two attention kernels over the 4-bit cache share: the arguments, what a query can see, softmax constants, the
// last step of a row.
#pragma once

#include <math.h>

#include "pkv_kv4.cuh"

namespace pkv_kv4 {

constexpr int kUnitAtoms = 4, kUnitTokens = kUnitAtoms * kAtomTokens;
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
      lo = max(0, pos_first - p.window + 1);
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
  r.end = p.c.end(s, r.len);
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
