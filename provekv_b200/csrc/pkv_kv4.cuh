// The 4-bit KV cache: its layout in memory, the argument checks the calls share, and the device pieces
// that turn codes into binary16 operands.
#pragma once

#include "pkv_common.cuh"

namespace pkv_kv4 {

constexpr int kAtomTokens = 16;
constexpr int64_t kMostSlots = 0x7fff0000;  // of a sequence, and tokens of a call: 32-bit numbers with room for a tile behind the last
constexpr int kMaxScaleByte = 0xDE;  // 7168: the largest scale for which the dequantisation below stays in range

// Byte offsets inside an atom (16 tokens of one kv head).
template <int D>
struct Atom {
  static constexpr int BYTES = 18 * D;
  static constexpr int KC = 0, VC = 8 * D, KS = 16 * D, VS = 17 * D;
  static constexpr int ROW = D / 2;   // code bytes of a token
  static constexpr int SROW = D / 16; // scale bytes of a token
  // The halves of a V code row are swapped for tokens with bit 1 set (D = 128): in the attention kernels a warp reads
  // pieces of four rows 64 bytes apart at once, which would otherwise meet in the same banks.
  static __host__ __device__ constexpr int vswap(int t) { return D == 128 ? (t & 2) << 4 : 0; }
};

struct Cache {
  uint8_t* pages;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* ends;
  int32_t* positions;
  float* mass;
  int64_t n_pages;
  int heads, page_tokens, page_atoms, n_seqs, max_pages, capacity;

  // length of sequence s; a bad one is reported and counts as 0
  __device__ __forceinline__ int length(int s, uint64_t* err) const {
    const int n = lens[s];
    if (n < 0 || n > capacity) {
      pkv_report(err, 0, s, PKV_VEC_BAD_SEQUENCE);
      return 0;
    }
    return n;
  }
  // tokens the sequence has had; where positions are kept, fewer than it holds are reported (and taken as they are)
  __device__ __forceinline__ int end(int s, int length, uint64_t* err) const {
    const int n = ends ? ends[s] : length;
    if (n < length && positions) pkv_report(err, 0, s, PKV_VEC_BAD_SEQUENCE);
    return n;
  }
  // Atom `a` (tokens 16 a .. 16 a + 15) of sequence s and kv head h, or null for a bad page number (reported).
  __device__ __forceinline__ uint8_t* atom(int s, int h, int a, int atom_bytes, uint64_t* err) const {
    const int p = a / page_atoms;
    const int64_t page = table[(int64_t)s * max_pages + p];
    if (page < 0 || page >= n_pages) {
      pkv_report(err, 0, s, PKV_VEC_BAD_SEQUENCE);
      return nullptr;
    }
    return pages + ((page * heads + h) * page_atoms + (a - p * page_atoms)) * (int64_t)atom_bytes;
  }
  __device__ __forceinline__ int64_t stat(int s, int h) const { return ((int64_t)s * heads + h) * capacity; }
};

struct Rows {
  int64_t seq, token, head;
  int n;
};

inline int make_cache(const pkv_kv4_cache* c, Cache* out) {
  if (!c || !c->pages || !c->page_table || !c->lens || c->reserved != 0) return PKV_ERR_INVALID_ARGUMENT;
  if (c->n_pages < 0 || c->n_kv_heads < 1 || c->n_seqs < 0 || c->max_pages < 0 || c->page_tokens < 1)
    return PKV_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)c->pages | (uintptr_t)c->positions | (uintptr_t)c->mass) & 15) return PKV_ERR_INVALID_ARGUMENT;
  if ((c->dim != 64 && c->dim != 128) || c->page_tokens % kAtomTokens) return PKV_ERR_UNSUPPORTED;
  // sequences and heads go into grid dimensions
  if ((int64_t)c->max_pages * c->page_tokens > kMostSlots || c->n_kv_heads > 65535 || c->n_seqs > 65535)
    return PKV_ERR_UNSUPPORTED;
  out->pages = c->pages;
  out->table = c->page_table;
  out->lens = c->lens;
  out->ends = c->ends;
  out->positions = c->positions;
  out->mass = c->mass;
  out->n_pages = c->n_pages;
  out->heads = c->n_kv_heads;
  out->page_tokens = c->page_tokens;
  out->page_atoms = c->page_tokens / kAtomTokens;
  out->n_seqs = c->n_seqs;
  out->max_pages = c->max_pages;
  out->capacity = c->max_pages * c->page_tokens;
  return PKV_OK;
}

inline int make_rows(const void* base, const pkv_kv4_rows* r, Rows* out) {
  if (!r || r->n_tokens < 0 || (!base && r->n_tokens > 0)) return PKV_ERR_INVALID_ARGUMENT;
  if (r->dtype != PKV_DST_F32 && r->dtype != PKV_DST_F16 && r->dtype != PKV_DST_BF16) return PKV_ERR_INVALID_ARGUMENT;
  const int unit = r->dtype == PKV_DST_F32 ? 4 : 8;
  if (((uintptr_t)base & 15) || r->seq_stride % unit || r->token_stride % unit || r->head_stride % unit)
    return PKV_ERR_INVALID_ARGUMENT;
  if (r->n_tokens > kMostSlots) return PKV_ERR_UNSUPPORTED;
  out->seq = r->seq_stride;
  out->token = r->token_stride;
  out->head = r->head_stride;
  out->n = r->n_tokens;
  return PKV_OK;
}

// Whether two sets of vectors [n_seqs][n][heads][dim] of one type share memory.  Equal strides: looked for exactly, largest
// stride first (a slice and its neighbours in one buffer are apart); others: by their ranges, so perhaps for nothing.
enum { kApart, kSame, kOverlap };
struct Axis {
  int64_t stride, n;
};
// whether `delta` is within `row` of a difference of two of the axes' offsets
inline bool meets(int64_t delta, const Axis* axis, int axes, int64_t row) {
  if (axes == 0) return delta > -row && delta < row;
  int64_t e = axis->stride ? delta / axis->stride : 0;
  for (int64_t k = e - 1; k <= e + 1; k++)
    if (k > -axis->n && k < axis->n && meets(delta - k * axis->stride, axis + 1, axes - 1, row)) return true;
  return false;
}
inline int overlap(const void* a, const Rows& ra, const void* b, const Rows& rb, int n_seqs, int heads, int dim, int dtype) {
  const int64_t size = dtype == PKV_DST_F32 ? 4 : 2, row = dim * size, delta = (int64_t)((uintptr_t)b - (uintptr_t)a);
  Axis x[3] = {{ra.seq, n_seqs}, {ra.token, ra.n}, {ra.head, heads}}, y[3] = {{rb.seq, n_seqs}, {rb.token, rb.n}, {rb.head, heads}};
  bool equal = true;
  int64_t low = 0, high = row;  // from the first byte of a to behind its last, and of both where they meet
  int64_t low_b = delta, high_b = delta + row;
  for (int i = 0; i < 3; i++) {
    if (x[i].n <= 1) x[i].stride = y[i].stride = 0;  // says nothing
    x[i].stride *= size;
    y[i].stride *= size;
    equal = equal && x[i].stride == y[i].stride;
    const int64_t ea = x[i].stride * (x[i].n - 1), eb = y[i].stride * (y[i].n - 1);
    (ea < 0 ? low : high) += ea;
    (eb < 0 ? low_b : high_b) += eb;
  }
  if (high <= low_b || high_b <= low) return kApart;
  if (!equal) return kOverlap;
  if (delta == 0) return kSame;
  auto size_of = [](const Axis& v) { return v.stride < 0 ? -v.stride : v.stride; };
  for (int i = 0; i < 2; i++)
    for (int j = 0; j + 1 < 3 - i; j++)
      if (size_of(x[j]) < size_of(x[j + 1])) {
        const Axis t = x[j];
        x[j] = x[j + 1];
        x[j + 1] = t;
      }
  return meets(delta, x, 3, row) ? kOverlap : kApart;
}

// Every kernel over this cache is launched so that it may come up while the one before it in the stream ends, and waits
// here, before its first access to memory (saves about 1 us between two short kernels).
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = s;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  pkv_count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// N consecutive values as f32; N a multiple of 4 (f32) or 8, the address 16-byte aligned.
template <int T, int N>
__device__ __forceinline__ void load_f32(const typename PkvDst<T>::type* p, float (&x)[N]) {
  if constexpr (T == PKV_DST_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + i));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (T == PKV_DST_F16) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          x[i + 2 * j] = f.x; x[i + 2 * j + 1] = f.y;
        } else {  // a bfloat16 is the upper half of an f32
          x[i + 2 * j] = __uint_as_float(w[j] << 16);
          x[i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
  }
}

template <int T, int N>
__device__ __forceinline__ void store_f32(typename PkvDst<T>::type* p, const float (&x)[N]) {
  if constexpr (T == PKV_DST_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      *reinterpret_cast<uint4*>(p + i) = make_uint4(pkv_pack2<T>(x[i], x[i + 1]), pkv_pack2<T>(x[i + 2], x[i + 3]),
                                                    pkv_pack2<T>(x[i + 4], x[i + 5]), pkv_pack2<T>(x[i + 6], x[i + 7]));
  }
}

// ---- codes to binary16 ------------------------------------------------------------------------------------------------
// OR-ing a nibble into the low bits of 0x6400 gives 1024 + n, and into bits 7..4 gives 1024 + 16 n.  One fused
// multiply-add per pair then subtracts the offset and applies the scale s' = s / 128:
//   (1024 + n) s' - 1032 s' = (n - 8) s'          (1024 + 16 n) s' - 1152 s' = 16 (n - 8) s'
// 1032 s' and 1152 s' have at most 11 significant bits and stay below 65504 for s <= 7168, s' is exact (s is a
// multiple of 2^-17), and (n - 8) s' has at most 7: every value is exact.  Odd channels come out 16 times too
// large; who uses them divides (a power of two, on the queries or on the sums).  9 instructions for 8 values.
constexpr float kScaleShift = 128.0f;

struct Scale {
  __half2 s, lo, hi;  // s', -1032 s', -1152 s'
  // one of the two for both halves (the instructions select halves of their operands themselves)
  __device__ __forceinline__ Scale low() const { return {__low2half2(s), __low2half2(lo), __low2half2(hi)}; }
  __device__ __forceinline__ Scale high() const { return {__high2half2(s), __high2half2(lo), __high2half2(hi)}; }
};
__device__ __forceinline__ Scale scale_of(uint32_t two_halves) {  // two scales as binary16, s not yet divided
  Scale r;
  const __half2 s = *reinterpret_cast<const __half2*>(&two_halves);
  r.s = __hmul2(s, __float2half2_rn(1.0f / kScaleShift));
  r.lo = __hmul2(s, __float2half2_rn(-1032.0f / kScaleShift));
  r.hi = __hmul2(s, __float2half2_rn(-1152.0f / kScaleShift));
  return r;
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, __half2 b, __half2 c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), b, c);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// out[i] = nibbles (i, i + 4) of w, as two binary16; i = 1, 3 are 16 times too large
__device__ __forceinline__ void nibbles(uint32_t w, const Scale& sc, uint32_t (&out)[4]) {
  out[0] = fma2(and_or(w, 0x000f000fu, 0x64006400u), sc.s, sc.lo);
  out[1] = fma2(and_or(w, 0x00f000f0u, 0x64006400u), sc.s, sc.hi);
  w >>= 8;
  out[2] = fma2(and_or(w, 0x000f000fu, 0x64006400u), sc.s, sc.lo);
  out[3] = fma2(and_or(w, 0x00f000f0u, 0x64006400u), sc.s, sc.hi);
}

}  // namespace pkv_kv4
