// Writing vectors into the 4-bit KV cache and reading them back.
//
// Append: a thread owns one block of 16 channels of a token's key and of its value, so that the block's largest
// magnitude needs no other thread and both loads are in flight together.  A CTA covers 128 / (D / 16) tokens of one kv head,
// whose code and scale bytes form contiguous runs.
// Read: a thread owns 16 bytes of the output, so that a warp's stores are contiguous.
// A vector is read once and written once.  Append of f32 runs at 82 % of the copy bandwidth (2 x 4099 tokens, 32 heads of 64: 28.5 us),
// of 16-bit vectors, twice the values a byte, it is bound by issue (73 % of the slots; 4 x 8192, 8 heads of 128: 38 us, 4.5 TB/s).  Read
// (36 and 38 us) by issue (65 to 68 %) and the latency of page number and codes.
#include "pkv_kv4.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kThreads = 128, kReadThreads = 256;

// The nearest scale to amax / 7 (ties to the even code), as its byte; 256 if it is beyond kMaxScaleByte.  Decided
// on exact products: the candidate below an approximate quotient, then amax against 7 x the midpoint above it.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const float s = __fmul_rn(amax, 0.142857149f);
  if (s > 8192.0f) return 256u;
  float lo, step;
  if (s >= 6.103515625e-05f) {  // 2^-14 and up: 3 fraction bits
    lo = __uint_as_float(__float_as_uint(s) & 0xfff00000u);
    step = __uint_as_float((__float_as_uint(s) & 0x7f800000u) - (3u << 23));
  } else {
    step = 7.62939453125e-06f;  // 2^-17
    lo = __fmul_rn(floorf(__fmul_rn(s, 131072.0f)), step);
  }
  // the code of lo: multiples of 2^-17 below 2^-14, then exponent and fraction bits
  uint32_t code = lo < 6.103515625e-05f ? (uint32_t)__fmul_rn(lo, 131072.0f) : (__float_as_uint(lo) >> 20) - (112u << 3);
  const float mid7 = __fmul_rn(7.0f, __fadd_rn(lo, __fmul_rn(0.5f, step)));  // exact: 5 bits x 3 bits
  if (amax > mid7 || (amax == mid7 && (code & 1u))) code++;
  return code > (uint32_t)kMaxScaleByte ? 256u : code;
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// A block done step by step, every decision on exact values: (codes, codes, scale byte or 256).
__device__ __forceinline__ uint3 quantise_exactly(const float (&x)[16], float amax) {
  const uint32_t byte = scale_byte(amax);
  if (byte > 255u) return make_uint3(0u, 0u, 256u);
  if (byte == 0u) return make_uint3(0x88888888u, 0x88888888u, 0u);  // below half the smallest scale: zeros (code 8)
  uint32_t w[2] = {0u, 0u};
  const float s = scale_value(byte), r = __frcp_rn(s), half = __fmul_rn(0.5f, s);
#pragma unroll
  for (int i = 0; i < 16; i++) {  // (inline and unrolled: the values stay in registers on the common way too)
    // x / s to the nearest integer, ties to even, by the remainder
    const float q = rintf(fminf(fmaxf(__fmul_rn(x[i], r), -8.0f), 7.0f));
    const float rest = __fmaf_rn(-q, s, x[i]);
    const int qi = (int)q, odd = qi & 1;
    const int up = rest > half || (rest == half && odd) ? 1 : 0;
    const int down = rest < -half || (rest == -half && odd) ? 1 : 0;
    w[i >> 3] |= (uint32_t)(min(7, max(-8, qi + up - down)) + 8) << (4 * (i & 7));
  }
  return make_uint3(w[0], w[1], byte);
}

// 16 channels -> 8 code bytes and the scale byte; false if they cannot be stored.
//
// The common way takes approximate quotients; what that could spoil:
//   the scale     amax / 7 is rounded to 4 significant bits on its bits.  16-bit types: at most 11 significant bits over 7, a
//                 quotient that is no tie is at least 2^-13 (relative) away from one, so rounding it to 18 bits first
//                 restores exact ties and moves nothing across one.  f32: a quotient within 2^-21 of a tie (its error is below
//                 2^-22) has the block done exactly, as does any below the scales of full precision;
//   the codes     amax / s is below 7.44, so no quotient needs clamping.  x / s is rounded by adding 1.5 x 2^23 + 8, which
//                 leaves n in the lowest byte of the sum's bits.  16-bit types: at most 11 significant bits over 4, no
//                 quotient but a tie is within 2^-13 of one, and rounding to a multiple of 2^-15 first (the sum with 384)
//                 restores those.  f32: a block with a quotient within 2^-16 of a tie (the error is below 2^-18) is done
//                 exactly.
template <int T>
__device__ __forceinline__ bool quantise(const float (&x)[16], uint2& codes, uint32_t& byte, int& why) {
  uint32_t top = 0u;  // magnitudes order like their bits, infinities and NaN above the finite ones
#pragma unroll
  for (int i = 0; i < 16; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  if (top >= 0x7f800000u) {
    why = PKV_VEC_NONFINITE_INPUT;
    return false;
  }
  uint32_t q7 = __float_as_uint(__fmul_rn(__uint_as_float(top), 0.142857149f));
  if constexpr (T != PKV_DST_F32) q7 = (q7 + 16u) & ~31u;
  bool unsure = q7 < 0x38800000u;  // 2^-14
  if constexpr (T == PKV_DST_F32) unsure = unsure || ((q7 - 0x7fffcu) & 0xfffffu) <= 8u;
  byte = ((q7 + 0x7ffffu + ((q7 >> 20) & 1u)) >> 20) - (112u << 3);
  const float s = __uint_as_float((byte + (112u << 3)) << 20);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  constexpr float kMagic = 12582912.0f + 8.0f;
  uint32_t n[16];
  float worst = 0.0f;  // the largest distance of a quotient from its integer
#pragma unroll
  for (int i = 0; i < 16; i++) {
    if constexpr (T == PKV_DST_F32) {
      const float q = __fmul_rn(x[i], r), rounded = __fadd_rn(q, kMagic);
      n[i] = __float_as_uint(rounded);
      worst = fmaxf(worst, fabsf(__fsub_rn(q, __fsub_rn(rounded, kMagic))));
    } else {
      n[i] = __float_as_uint(__fadd_rn(__fmaf_rn(x[i], r, 384.0f), kMagic - 384.0f));
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {  // two codes a byte, four bytes a word; what is above the lowest byte falls away
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = n[8 * h + 2 * i + 1] * 16u + n[8 * h + 2 * i];
    w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  if (unsure || worst > 0.5f - 1.52587890625e-05f) {
    w[0] = w[1] = 0x88888888u;
    byte = 0u;
    if (top != 0u) {
      const uint3 e = quantise_exactly(x, __uint_as_float(top));
      w[0] = e.x;
      w[1] = e.y;
      byte = e.z;
    }
  }
  if (byte > (uint32_t)kMaxScaleByte) {
    why = PKV_VEC_NORM_RANGE;
    return false;
  }
  codes = make_uint2(w[0], w[1]);
  return true;
}

// The rows of a sequence in a call: row i < fresh goes to slot first + i, whose token has position `position` + i.
struct Fresh {
  int fresh, first, position;
};
__device__ __forceinline__ Fresh fresh_of(const Cache& c, int s, int n_tokens, const int32_t* new_lens, uint64_t* err) {
  Fresh r;
  const int n = c.length(s, err);
  r.fresh = new_lens ? new_lens[s] : n_tokens;
  if (r.fresh < 0 || r.fresh > n_tokens || r.fresh > n) {
    pkv_report(err, 0, s, PKV_VEC_BAD_SEQUENCE);
    r.fresh = 0;
  }
  r.first = n - r.fresh;
  r.position = c.end(s, n, err) - r.fresh;
  return r;
}

// 16 values as they lie in memory, and as f32.
template <int T>
struct Raw {
  static constexpr int N = T == PKV_DST_F32 ? 4 : 2;
  uint4 v[N];
  __device__ __forceinline__ void load(const typename PkvDst<T>::type* p) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void to_f32(float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (T == PKV_DST_F32) {
          x[4 * i + j] = __uint_as_float(w[j]);
        } else if constexpr (T == PKV_DST_F16) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          x[8 * i + 2 * j] = f.x;
          x[8 * i + 2 * j + 1] = f.y;
        } else {  // a bfloat16 is the upper half of an f32
          x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
  }
};

// Tokens a thread has in flight: 128 bytes of loads in either case.
template <int T>
constexpr int kAppendTurns = T == PKV_DST_F32 ? 1 : 2;

template <int D, int T>
__global__ void __launch_bounds__(kThreads)
kv4_append_kernel(Cache c, const typename PkvDst<T>::type* __restrict__ k, Rows kr,
                  const typename PkvDst<T>::type* __restrict__ v, Rows vr, const int32_t* __restrict__ new_lens, uint64_t* err) {
  using A = Atom<D>;
  constexpr int TOK = kThreads / A::SROW, TURNS = kAppendTurns<T>;
  const int b = threadIdx.x % A::SROW;  // block of 16 channels
  const int s = blockIdx.z, h = blockIdx.y;
  const int i0 = blockIdx.x * TOK * TURNS + threadIdx.x / A::SROW;
  const unsigned row_lanes = ((1u << A::SROW) - 1u) << ((threadIdx.x & 31) / A::SROW * A::SROW);
  Raw<T> raw[TURNS][2];
  uint8_t* atom[TURNS];
  wait_for_stream();
  const Fresh f = fresh_of(c, s, kr.n, new_lens, err);
  k += s * kr.seq + h * kr.head + 16 * b;
  v += s * vr.seq + h * vr.head + 16 * b;
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int i = i0 + u * TOK;
    atom[u] = nullptr;
    if (i < f.fresh) {  // (padding is not fetched)
      raw[u][0].load(k + i * kr.token);
      raw[u][1].load(v + i * vr.token);
      atom[u] = c.atom(s, h, (f.first + i) / kAtomTokens, A::BYTES, err);
    }
  }
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    if (!__any_sync(0xffffffffu, atom[u] != nullptr)) continue;
    const int slot = f.first + i0 + u * TOK, t = slot % kAtomTokens;
#pragma unroll
    for (int side = 0; side < 2; side++) {
      float x[16];
      if (!atom[u]) raw[u][side].clear();
      raw[u][side].to_f32(x);
      uint2 codes = make_uint2(0u, 0u);
      uint32_t byte = 0u;
      int why = 0;
      const bool ok = quantise<T>(x, codes, byte, why);
      // one block that cannot be stored empties the whole row; the row's threads are neighbours in a warp
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad & row_lanes) {
        codes = make_uint2(0u, 0u);
        byte = 0u;
        if (!ok) pkv_report(err, 0, (((int64_t)s * kr.n + i0 + u * TOK) * c.heads + h) * 2 + side, why);
      }
      const int at = side ? A::VC + t * A::ROW + ((8 * b) ^ A::vswap(t)) : A::KC + t * A::ROW + 8 * b;
      if (atom[u]) {
        *reinterpret_cast<uint2*>(atom[u] + at) = codes;
        atom[u][(side ? A::VS : A::KS) + t * A::SROW + b] = (uint8_t)byte;
      }
    }
    if (b == 0 && atom[u]) {
      if (c.positions) c.positions[c.stat(s, h) + slot] = f.position + i0 + u * TOK;
      if (c.mass) c.mass[c.stat(s, h) + slot] = 0.0f;
    }
  }
}

// 16 bytes of output from their codes (16 or 32 bits) and scale.
template <int T>
__device__ __forceinline__ uint4 values_of(uint32_t w, uint32_t byte) {
  if constexpr (T == PKV_DST_F32) {
    const float f = scale_value(byte);
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)  // 2^23 + n as bits, less 2^23 + 8
      x[j] = __fmul_rn(__fadd_rn(__uint_as_float(and_or(w >> (4 * j), 15u, 0x4b000000u)), -8388616.0f), f);
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  } else {
    uint32_t p[4];  // channels (j, j + 4)
    if constexpr (T == PKV_DST_F16) {
      // 1024 + n as bits, less 1032, times s: every step exact
      const uint32_t s2 = byte * 0x00800080u;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t u = and_or(w >> (4 * j), 0x000f000fu, 0x64006400u);
        const __half2 d = __hadd2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(-1032.0f));
        const __half2 r = __hmul2(d, *reinterpret_cast<const __half2*>(&s2));
        p[j] = *reinterpret_cast<const uint32_t*>(&r);
      }
    } else {
      const __nv_bfloat162 s2 = __float2bfloat162_rn(scale_value(byte));
#pragma unroll
      for (int j = 0; j < 4; j++) {  // 128 + n as bits, less 136, times s
        const uint32_t u = and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);
        const __nv_bfloat162 d = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(-136.0f));
        const __nv_bfloat162 r = __hmul2(d, s2);
        p[j] = *reinterpret_cast<const uint32_t*>(&r);
      }
    }
    return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632),
                      __byte_perm(p[2], p[3], 0x7632));
  }
}

template <int D, int T>
struct ReadShape {
  static constexpr int N = T == PKV_DST_F32 ? 4 : 8;   // channels of a 16-byte piece
  static constexpr int PIECES = D / N;                 // of a row
  static constexpr int ROWS = kReadThreads / PIECES;   // tokens a CTA covers at once
  static constexpr int TURNS = 4;                      // tokens a thread has in flight
};
template <int D, int T>
__global__ void __launch_bounds__(kReadThreads)
kv4_read_kernel(Cache c, typename PkvDst<T>::type* __restrict__ k, Rows kr, typename PkvDst<T>::type* __restrict__ v,
                Rows vr, const int32_t* __restrict__ new_lens, int clear_rest, uint64_t* err) {
  using A = Atom<D>;
  using R = ReadShape<D, T>;
  constexpr int N = R::N;
  const int piece = threadIdx.x % R::PIECES;
  const int s = blockIdx.z, h = blockIdx.y;
  const int i0 = blockIdx.x * R::ROWS * R::TURNS + threadIdx.x / R::PIECES;
  wait_for_stream();
  const Fresh f = fresh_of(c, s, kr.n, new_lens, err);
  k += s * kr.seq + h * kr.head + piece * N;
  v += s * vr.seq + h * vr.head + piece * N;
  uint32_t codes[R::TURNS][2], scale[R::TURNS][2];
  bool live[R::TURNS];
#pragma unroll
  for (int u = 0; u < R::TURNS; u++) {
    const int i = i0 + u * R::ROWS, slot = f.first + i;
    const uint8_t* atom = i < f.fresh ? c.atom(s, h, slot / kAtomTokens, A::BYTES, err) : nullptr;
    live[u] = atom != nullptr;
    if (!live[u]) continue;
    const int t = slot % kAtomTokens, at = piece * N / 2;
    const uint8_t* kc = atom + A::KC + t * A::ROW + at;
    const uint8_t* vc = atom + A::VC + t * A::ROW + (at ^ A::vswap(t));
    if constexpr (N == 8) {
      codes[u][0] = *reinterpret_cast<const uint32_t*>(kc);
      codes[u][1] = *reinterpret_cast<const uint32_t*>(vc);
    } else {
      codes[u][0] = *reinterpret_cast<const uint16_t*>(kc);
      codes[u][1] = *reinterpret_cast<const uint16_t*>(vc);
    }
    scale[u][0] = atom[A::KS + t * A::SROW + piece * N / 16];
    scale[u][1] = atom[A::VS + t * A::SROW + piece * N / 16];
  }
#pragma unroll
  for (int u = 0; u < R::TURNS; u++) {
    const int i = i0 + u * R::ROWS;
    uint4 out[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (live[u]) {
      out[0] = values_of<T>(codes[u][0], scale[u][0]);
      out[1] = values_of<T>(codes[u][1], scale[u][1]);
    } else if (!clear_rest || i >= kr.n) {
      continue;
    }
    *reinterpret_cast<uint4*>(k + i * kr.token) = out[0];
    *reinterpret_cast<uint4*>(v + i * vr.token) = out[1];
  }
}

template <int D, int T>
cudaError_t launch_rows(bool append, const Cache& c, const void* k, const Rows& kr, const void* v, const Rows& vr,
                 const int32_t* new_lens, int clear_rest, uint64_t* err, cudaStream_t s) {
  using E = typename PkvDst<T>::type;
  constexpr int TOK = kThreads / Atom<D>::SROW * kAppendTurns<T>, READ = ReadShape<D, T>::ROWS * ReadShape<D, T>::TURNS;
  const int per = append ? TOK : READ;
  const dim3 grid((unsigned)((kr.n + per - 1) / per), (unsigned)c.heads, (unsigned)c.n_seqs);
  if (append) return launch_early(kv4_append_kernel<D, T>, grid, kThreads, 0, s, c, (const E*)k, kr, (const E*)v, vr, new_lens, err);
  return launch_early(kv4_read_kernel<D, T>, grid, kReadThreads, 0, s, c, (E*)const_cast<void*>(k), kr, (E*)const_cast<void*>(v), vr,
                      new_lens, clear_rest, err);
}

int rows_call(bool append, const pkv_kv4_cache* cache, const void* k, const pkv_kv4_rows* k_rows, const void* v,
              const pkv_kv4_rows* v_rows, const int32_t* new_lens, int clear_rest, uint64_t* err, void* stream) {
  Cache c;
  Rows kr, vr;
  if (int st = make_cache(cache, &c)) return st;
  if (int st = make_rows(k, k_rows, &kr)) return st;
  if (int st = make_rows(v, v_rows, &vr)) return st;
  if (!err || kr.n != vr.n || k_rows->dtype != v_rows->dtype || (clear_rest != 0 && clear_rest != 1)) return PKV_ERR_INVALID_ARGUMENT;
  if (kr.n > c.capacity && !new_lens) return PKV_ERR_INVALID_ARGUMENT;
  if (kr.n == 0 || c.n_seqs == 0) return PKV_OK;
  // both are written; sets of vectors that are only between one another are apart
  if (!append && overlap(k, kr, v, vr, c.n_seqs, c.heads, cache->dim, k_rows->dtype) != kApart) return PKV_ERR_INVALID_ARGUMENT;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t ce;
#define PKV_KV4_ROWS(D)                                                                                                    \
  switch (k_rows->dtype) {                                                                                                 \
    case PKV_DST_F32: ce = launch_rows<D, PKV_DST_F32>(append, c, k, kr, v, vr, new_lens, clear_rest, err, s); break;                       \
    case PKV_DST_F16: ce = launch_rows<D, PKV_DST_F16>(append, c, k, kr, v, vr, new_lens, clear_rest, err, s); break;                       \
    default: ce = launch_rows<D, PKV_DST_BF16>(append, c, k, kr, v, vr, new_lens, clear_rest, err, s); break;                               \
  }
  if (cache->dim == 64) PKV_KV4_ROWS(64) else PKV_KV4_ROWS(128)
#undef PKV_KV4_ROWS
  return pkv_cuda_status(ce);
}

}  // namespace

extern "C" int pkv_kv4_append_dev(const pkv_kv4_cache* cache, const void* k_dev, const pkv_kv4_rows* k_rows,
                                  const void* v_dev, const pkv_kv4_rows* v_rows, const int32_t* new_lens_dev,
                                  uint64_t* err_dev, void* stream) {
  return rows_call(true, cache, k_dev, k_rows, v_dev, v_rows, new_lens_dev, 0, err_dev, stream);
}

extern "C" int pkv_kv4_read_dev(const pkv_kv4_cache* cache, void* k_dev, const pkv_kv4_rows* k_rows, void* v_dev,
                                const pkv_kv4_rows* v_rows, const int32_t* new_lens_dev, int32_t clear_rest, uint64_t* err_dev,
                                void* stream) {
  return rows_call(false, cache, k_dev, k_rows, v_dev, v_rows, new_lens_dev, clear_rest, err_dev, stream);
}
