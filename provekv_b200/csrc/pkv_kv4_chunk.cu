// Attention over the 4-bit KV cache for many query rows per kv head (prompt chunks), 16-bit queries.
//
// A CTA takes up to 256 query rows of one kv head (two tiles of 128) over a run of units of 64 tokens, on the fifth-
// generation tensor cores:
//
//   S = Q K^T    128 rows x 64 tokens, A = Q, B = dequantised keys, both in shared memory; two S per tile
//   O += P V     128 rows x dim, A = P in tensor memory (over S), B = dequantised values, transposed, in shared memory
//
// Warps 0-3 and 4-7: the softmax of a tile each, a thread per row.  Warps 8-11 dequantise keys, 12-15 values; warp 16 brings
// codes (bulk copies through a ring of three units), warp 17 issues the products.  The scores of the next unit are on
// their way while a tile's softmax works on the last.
//
// A unit of 64 tokens costs the tensor cores 1024 cycles for 256 rows (dim 128), and the exponentials the same at 16 a
// cycle; shared memory gives the products their operands in another 1024, and the dequantised unit goes into it in about
// 400.  Dequantising takes about 900 warp instructions, shared by 256 rows.
//
// Both operands in shared memory are K-major with the 128-byte swizzle.  Row n of a unit's keys is token sigma(n), the same
// order on the tokens' side of the values: it spreads the lanes that gather the values' codes over the banks.
#include "pkv_kv4_attend.cuh"
#include "pkv_tcgen05.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kThreads = 20 * 32;  // the last two warps only complete a warpgroup
constexpr int kTileRows = 128, kTaskRows = 2 * kTileRows;
constexpr int kCodeSlots = 3, kStagesKv = 4, kQuadSlots = 16;
constexpr int kMinUnits = 8;  // a split of the tokens has at least this many units

struct ChunkParams {
  AttendParams a;
  int tasks, splits;  // tasks of 256 rows of a kv head; splits of the tokens
};

// Token of row n of a unit's keys, of column n of its scores.
__host__ __device__ constexpr int sigma(int n) { return (n & ~3) | ((n & 3) ^ ((n >> 3) & 3)); }

// 128-byte swizzle: 16-byte piece c of row r of an operand with 128-byte rows.
__device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4)); }

// kind::f16: f32 accumulator, A and B binary16, both K-major
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= A[smem] B[smem]^T, one step of 16 along K
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]^T
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pkv_smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 64 columns of this thread's lane, one wait
__device__ __forceinline__ void tmem_load32_async(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait(uint32_t (&r)[32]) {  // no use of the registers moves above it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_load64(uint32_t addr, float (&x)[2][32]) {
  uint32_t a[32], b[32];
  tmem_load32_async(addr, a);
  tmem_load32_async(addr + 32, b);
  tmem_load_wait(a);
  tmem_load_wait(b);
#pragma unroll
  for (int i = 0; i < 32; i++) {
    x[0][i] = __uint_as_float(a[i]);
    x[1][i] = __uint_as_float(b[i]);
  }
}
// two f32 operations in one instruction
__device__ __forceinline__ float2 fma2_f32(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2_f32(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Registers move between the roles (whole warpgroups): 2 x 128 threads of 128, 2 x 128 of 80 and 128 of 64 are the 640 x 96
// that the block was launched with.
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D>
struct Layout {
  static constexpr int UNIT = kUnitAtoms * Atom<D>::BYTES;
  static constexpr int KEYS = 64 * D * 2, VALUES = D * 64 * 2;  // a unit's operands
  static constexpr int STAGE = KEYS + VALUES;
  static constexpr int QUERY = kTileRows * D * 2;                // a tile's queries
  static constexpr int QUERIES = kStagesKv * STAGE, CODES = QUERIES + 2 * QUERY;
  static constexpr int BYTES = CODES + kCodeSlots * UNIT + 1024; // room to align the operands to 1024 bytes
  // tensor memory columns of a tile: two S (P over each), O
  static constexpr int S = 0, O = 128;
};

struct Barriers {
  uint64_t codes_full[kCodeSlots], codes_empty[kCodeSlots];  // copies -> dequantising warps -> copies
  uint64_t kv_full[kStagesKv], kv_empty[kStagesKv];                          // operands -> products -> operands
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2]; // per tile (and S)
  uint64_t drain;
};

template <int D, int T>
__global__ void __launch_bounds__(kThreads, 1)
kv4_chunk_kernel(const __grid_constant__ ChunkParams cp) {
  using A = Atom<D>;
  using Y = Layout<D>;
  using E = typename PkvDst<T>::type;
  const AttendParams& p = cp.a;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) Barriers bar;
  __shared__ uint32_t s_tmem;
  __shared__ uint32_t s_quad[kQuadSlots];  // which of a unit's atoms are there
  uint8_t* smem = smem_raw + ((1024u - (pkv_smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  wait_for_stream();

  // ---- the task
  const int split = blockIdx.x / cp.tasks, task = blockIdx.x - split * cp.tasks;
  const int h = blockIdx.y, s = blockIdx.z;
  const Sequence seq = sequence_of(p, s);
  const int all_rows = seq.qn * p.group, row0 = task * kTaskRows;
  if (row0 >= all_rows) return;
  const int n_tiles = all_rows - row0 > kTileRows ? 2 : 1;
  const int len = seq.len, pos0 = seq.end - seq.qn;
  const int qpos_first = pos0 + row0 / p.group, qpos_last = pos0 + min(seq.qn - 1, (row0 + kTaskRows - 1) / p.group);
  const Span span = visible_span(p, len, qpos_first, qpos_last);
  const int first = (int)((int64_t)split * span.count / cp.splits), n = (int)((int64_t)(split + 1) * span.count / cp.splits) - first;

  if (tid == 0) {
    for (int i = 0; i < kCodeSlots; i++) {
      pkv_mbar_init(&bar.codes_full[i], 1);
      pkv_mbar_init(&bar.codes_empty[i], 8);
    }
    for (int i = 0; i < kStagesKv; i++) {
      pkv_mbar_init(&bar.kv_full[i], 8);
      pkv_mbar_init(&bar.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      pkv_mbar_init(&bar.q_full[i], kTileRows);
      for (int b = 0; b < 2; b++) {
        pkv_mbar_init(&bar.s_full[i][b], 1);
        pkv_mbar_init(&bar.p_full[i][b], kTileRows);
      }
      pkv_mbar_init(&bar.o_done[i], 1);
    }
    pkv_mbar_init(&bar.drain, 1);
  }
  if (warp == 17) pkv_tc::tmem_alloc(&s_tmem, 512);
  __syncthreads();
  pkv_tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  bool fine = true;

  if (warp >= 16) {
    fewer_registers<64>();
  } else if (warp >= 8) {
    fewer_registers<80>();
  } else {
    more_registers<128>();
  }
  if (warp == 16) {
    // ---- codes: page numbers of kBatch units at once, one atom per lane, a batch ahead of their use
    auto atom_of = [&](int i0) -> int {
      const int i = i0 + lane / kUnitAtoms;
      if (i >= n) return -1;
      const int a = span.unit(first + i) * kUnitAtoms + lane % kUnitAtoms;
      return a * kAtomTokens < len ? a : -1;
    };
    auto page_of = [&](int a) -> int { return a < 0 ? -1 : __ldg(p.c.table + (int64_t)s * p.c.max_pages + a / p.c.page_atoms); };
    int atom = atom_of(0), page = page_of(atom), issued = 0;
    const uint8_t* src = nullptr;
    unsigned live = 0;
    for (int i = 0; i < n; i++) {
      if (i % kBatch == 0) {
        src = nullptr;
        if (atom >= 0) {
          if (page < 0 || page >= p.c.n_pages) pkv_report(p.err, 0, s, PKV_VEC_BAD_SEQUENCE);
          else src = p.c.pages + (((int64_t)page * p.c.heads + h) * p.c.page_atoms + atom % p.c.page_atoms) * (int64_t)A::BYTES;
        }
        live = __ballot_sync(0xffffffffu, src != nullptr);
        atom = atom_of(i + kBatch);
        page = page_of(atom);
      }
      const int slot = i % kCodeSlots;
      if (!__all_sync(0xffffffffu, pkv_mbar_wait(&bar.codes_empty[slot], ((i / kCodeSlots) & 1) ^ 1))) {
        fine = false;
        break;
      }
      const int l = kUnitAtoms * (i % kBatch);
      const unsigned quad = (live >> l) & 15u;
      if (lane == 0) {
        s_quad[i % kQuadSlots] = quad;
        pkv_mbar_expect_tx(&bar.codes_full[slot], (uint32_t)__popc(quad) * A::BYTES);
      }
      __syncwarp();
      if (lane / kUnitAtoms == i % kBatch && src)
        pkv_bulk_load(smem + Y::CODES + slot * Y::UNIT + lane % kUnitAtoms * A::BYTES, src, A::BYTES, &bar.codes_full[slot]);
      issued = i + 1;
    }
    if (!fine)  // leave no copy behind
      for (int i = max(0, issued - kCodeSlots); i < issued; i++) pkv_mbar_wait(&bar.codes_full[i % kCodeSlots], (i / kCodeSlots) & 1);
  } else if (warp >= 17) {
    // ---- products.  The whole warp walks through the units, so that descriptors and addresses stay in uniform registers
    // (moving them there for every instruction costs a lone thread about 100 cycles a step); one lane issues.
    if (warp == 17) {
      constexpr uint32_t id_s = idesc_f16(128, 64), id_o = idesc_f16(128, D);
      const bool leader = elect_one();
      const uint32_t operands = pkv_smem_u32(smem);
      auto scores = [&](int t, int i) {
        const uint64_t a = pkv_tc::smem_desc_sw128(operands + Y::QUERIES + t * Y::QUERY);
        const uint64_t b = pkv_tc::smem_desc_sw128(operands + (i % kStagesKv) * Y::STAGE);
        const uint32_t d = tmem + 256u * t + Y::S + 64u * (i & 1);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; k++)
            mma_ss(d, a + (uint64_t)(((k >> 2) * (kTileRows * 128) + (k & 3) * 32) >> 4),
                   b + (uint64_t)(((k >> 2) * (64 * 128) + (k & 3) * 32) >> 4), id_s, k > 0);
          pkv_tc::mma_commit(&bar.s_full[t][i & 1]);
        }
        __syncwarp();
      };
      auto outputs = [&](int t, int i) {
        const uint64_t b = pkv_tc::smem_desc_sw128(operands + (i % kStagesKv) * Y::STAGE + Y::KEYS);
        const uint32_t base = tmem + 256u * t;
        if (leader) {
#pragma unroll
          for (int k = 0; k < 4; k++) mma_ts(base + Y::O, base + Y::S + 64u * (i & 1) + 8 * k, b + (uint64_t)((k * 32) >> 4), id_o, i > 0 || k > 0);
          pkv_tc::mma_commit(&bar.o_done[t]);
        }
        __syncwarp();
      };
      auto wait = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, pkv_mbar_wait(b, parity)) != 0; };
      for (int i = 0; i < n && fine; i++) {
        if (i == 0) {
          fine = wait(&bar.kv_full[0], 0);
          for (int t = 0; t < n_tiles && fine; t++) {
            fine = wait(&bar.q_full[t], 0);
            pkv_tc::fence_after_sync();
            if (fine) scores(t, 0);
          }
        }
        // the S that the next scores go into was read by the unit before's product, which is ahead of them in order
        if (fine && i + 1 < n) {
          fine = wait(&bar.kv_full[(i + 1) % kStagesKv], ((i + 1) / kStagesKv) & 1);
          for (int t = 0; t < n_tiles && fine; t++) scores(t, i + 1);
        }
        for (int t = 0; t < n_tiles && fine; t++) {
          fine = wait(&bar.p_full[t][i & 1], (i >> 1) & 1);
          pkv_tc::fence_after_sync();
          if (fine) outputs(t, i);
        }
        if (fine && leader) pkv_tc::mma_commit(&bar.kv_empty[i % kStagesKv]);
        __syncwarp();
      }
      if (leader) pkv_tc::mma_commit(&bar.drain);
      __syncwarp();
      pkv_mbar_wait(&bar.drain, 0);
    }
  } else if (warp >= 8) {
    // ---- codes to operands
    const int w4 = warp & 3;
    const bool values = warp >= 12;
    for (int i = 0; i < n; i++) {
      const int slot = i % kCodeSlots;
      const bool ok = pkv_mbar_wait(&bar.codes_full[slot], (i / kCodeSlots) & 1) && pkv_mbar_wait(&bar.kv_empty[i % kStagesKv], ((i / kStagesKv) & 1) ^ 1);
      if (!__all_sync(0xffffffffu, ok)) {
        fine = false;
        break;
      }
      const uint8_t* codes = smem + Y::CODES + slot * Y::UNIT;
      const unsigned quad = s_quad[i % kQuadSlots];
      const int held = len - span.unit(first + i) * kUnitTokens;  // tokens of the unit below the sequence's length
      const bool whole = quad == 15u && held >= kUnitTokens;
      auto there = [&](int t) { return whole || (((quad >> (t >> 4)) & 1u) && t < held); };
      if (!values) {
        // a lane: one block of 16 channels of a token; four blocks x eight tokens a warp, so that the lanes of a store cover
        // distinct banks
        uint8_t* keys = smem + (i % kStagesKv) * Y::STAGE;
        constexpr int BLOCKS = D / 16, PASSES = 64 * BLOCKS / 128;
#pragma unroll
        for (int k = 0; k < PASSES; k++) {
          const int unit = k * 4 + w4;  // (group of 8 tokens, group of 4 blocks)
          const int b = (lane & 3) + 4 * (unit % (BLOCKS / 4)), row = (lane >> 2) + 8 * (unit / (BLOCKS / 4)), t = sigma(row);
          const uint8_t* atom = codes + (t >> 4) * A::BYTES;
          uint2 w = make_uint2(0u, 0u);
          uint32_t sb = 0u;
          if (there(t)) {
            w = *reinterpret_cast<const uint2*>(atom + A::KC + (t & 15) * A::ROW + 8 * b);
            sb = atom[A::KS + (t & 15) * A::SROW + b];
          }
          const Scale sc = scale_of(sb * 0x00800080u);
          uint32_t o0[4], o1[4];
          nibbles(w.x, sc, o0);
          nibbles(w.y, sc, o1);
          uint8_t* slab = keys + (b >> 2) * (64 * 128);
          *reinterpret_cast<uint4*>(slab + piece(row, 2 * (b & 3))) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
          *reinterpret_cast<uint4*>(slab + piece(row, 2 * (b & 3) + 1)) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
        }
      } else {
        // a lane: eight channels (a word of codes) of eight tokens, which become 16 bytes of eight rows of the transpose
        uint8_t* vals = smem + (i % kStagesKv) * Y::STAGE + Y::KEYS;
        constexpr int WORDS = D / 8;
        for (int k = w4; k < WORDS / 4; k += 4) {
          const int tg = lane & 7, word = 4 * k + (lane >> 3);
          uint32_t m[4][8];  // [token pair][channel]
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t w[2], sb[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const int t = 8 * tg + ((2 * j + e) ^ (tg & 3)), ta = t & 15;  // sigma(8 tg + 2 j + e)
              const uint8_t* atom = codes + (t >> 4) * A::BYTES;
              w[e] = sb[e] = 0u;
              if (there(t)) {
                w[e] = *reinterpret_cast<const uint32_t*>(atom + A::VC + ta * A::ROW + ((4 * word) ^ A::vswap(ta)));
                sb[e] = atom[A::VS + ta * A::SROW + (word >> 1)];
              }
            }
            const Scale sc = scale_of((sb[0] << 7) | (sb[1] << 23));
            uint32_t lo[4], hi[4];
            nibbles(__byte_perm(w[0], w[1], 0x5410), sc, lo);
            nibbles(__byte_perm(w[0], w[1], 0x7632), sc, hi);
#pragma unroll
            for (int c = 0; c < 4; c++) {
              m[j][c] = lo[c];
              m[j][4 + c] = hi[c];
            }
          }
#pragma unroll
          for (int c = 0; c < 8; c++)
            *reinterpret_cast<uint4*>(vals + piece(8 * word + c, tg)) = make_uint4(m[0][c], m[1][c], m[2][c], m[3][c]);
        }
      }
      pkv_tc::fence_smem_to_async();
      __syncwarp();
      if (lane == 0) {
        arrive(&bar.kv_full[i % kStagesKv]);
        arrive(&bar.codes_empty[slot]);
      }
    }
  } else if ((warp >> 2) < n_tiles) {
    // ---- softmax of tile t, a thread per row
    const int t = warp >> 2, row = row0 + kTileRows * t + (tid & 127);
    const uint32_t base = tmem + 256u * t + ((uint32_t)(32 * (warp & 3)) << 16);
    const bool live = row < all_rows;
    const int token = row / p.group, hq = h * p.group + (row - token * p.group), qpos = pos0 + token;
    float factor;
    {  // the query, scaled by a power of two, odd channels divided by 16, in the order of the keys' channels
      const E* q = reinterpret_cast<const E*>(p.q_ptr) + s * p.q.seq + (int64_t)token * p.q.token + hq * p.q.head;
      float amax = 0.0f;
#pragma unroll 2
      for (int c = 0; c < D && live; c += 16) {
        float x[16];
        load_f32<T, 16>(q + c, x);
#pragma unroll
        for (int j = 0; j < 16; j++) amax = fmaxf(amax, fabsf(x[j]));
      }
      const float pw = p.negate ? -row_power(amax) : row_power(amax);
      factor = __fmul_rn(__fmul_rn(__fmul_rn(p.scale, kLog2e), kScaleShift), 1.0f / row_power(amax));
      uint8_t* to = smem + Y::QUERIES + t * Y::QUERY;
#pragma unroll 2
      for (int c = 0; c < D; c += 16) {
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = 0.0f;
        if (live) load_f32<T, 16>(q + c, x);
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int at = 8 * (j >> 2) + (j & 3);
          const float f = (j & 1) ? __fmul_rn(pw, 0.0625f) : pw;
          r[j] = half2_of(__fmul_rn(x[at], f), __fmul_rn(x[at + 4], f));
        }
        uint8_t* slab = to + (c >> 6) * (kTileRows * 128);
        *reinterpret_cast<uint4*>(slab + piece(tid & 127, (c >> 3) & 7)) = make_uint4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<uint4*>(slab + piece(tid & 127, ((c >> 3) & 7) + 1)) = make_uint4(r[4], r[5], r[6], r[7]);
      }
      pkv_tc::fence_smem_to_async();
      arrive(&bar.q_full[t]);
    }
    const bool by_position = p.c.positions != nullptr && (p.window > 0 || seq.qn > 1);
    const int32_t* positions = by_position ? p.c.positions + p.c.stat(s, h) : nullptr;
    const int tile_first = pos0 + (row0 + kTileRows * t) / p.group;
    const int tile_last = pos0 + min(seq.qn - 1, (row0 + kTileRows * t + kTileRows - 1) / p.group);
    // positions of a unit's tokens, two a lane, loaded a unit ahead.  Only units with a token that some row of the tile must not
    // see are masked token by token.
    int kp[2] = {0, 0};
    auto load_positions = [&](int i) {
      const int at = i < n ? span.unit(first + i) * kUnitTokens + lane : len;
#pragma unroll
      for (int e = 0; e < 2; e++) kp[e] = at + 32 * e < len ? __ldg(positions + at + 32 * e) : 0;
    };
    if (by_position) load_positions(0);
    float m = -INFINITY, l = 0.0f;
    for (int i = 0; i < n; i++) {
      int at[2] = {kp[0], kp[1]};
      if (by_position) load_positions(i + 1);
      if (!__all_sync(0xffffffffu, pkv_mbar_wait(&bar.s_full[t][i & 1], (i >> 1) & 1))) {
        fine = false;
        break;
      }
      pkv_tc::fence_after_sync();
      const uint32_t s_at = base + Y::S + 64u * (i & 1);
      float x[2][32];
      tmem_load64(s_at, x);
      const int token0 = span.unit(first + i) * kUnitTokens;
      const unsigned quad = s_quad[i % kQuadSlots];
      float fac = factor;
      int newest = token0 + kUnitTokens - 1, oldest = token0;
      if (by_position) {
        newest = __reduce_max_sync(0xffffffffu, max(at[0], at[1]));
        oldest = __reduce_min_sync(0xffffffffu, min(at[0], at[1]));
      }
      if (quad != 15u || token0 + kUnitTokens > len || newest > tile_first ||
          (p.window > 0 && tile_last - oldest >= p.window && newest >= p.sinks)) {
        fac = 1.0f;
#pragma unroll
        for (int c = 0; c < 64; c++) {
          const int k = sigma(c);
          bool see = ((quad >> (k >> 4)) & 1u) && token0 + k < len;
          const int kp = by_position ? __shfl_sync(0xffffffffu, at[k >> 5], k & 31) : token0 + k;
          const int d = qpos - kp;
          see = see && d >= 0 && (p.window == 0 || d < p.window || kp < p.sinks);
          x[c >> 5][c & 31] = see ? __fmul_rn(x[c >> 5][c & 31], factor) : -INFINITY;
        }
      }
      float tops[4];  // four chains, their latencies side by side
#pragma unroll
      for (int c = 0; c < 4; c++) tops[c] = fmaxf(x[0][c], x[0][c + 4]);
#pragma unroll
      for (int c = 8; c < 64; c += 8)
#pragma unroll
        for (int j = 0; j < 4; j++) tops[j] = fmaxf(tops[j], fmaxf(x[c >> 5][(c & 31) + j], x[c >> 5][(c & 31) + j + 4]));
      const float top = __fmul_rn(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), fac);
      const bool raise = __any_sync(0xffffffffu, top > __fadd_rn(m, kLag));
      float f = 1.0f;
      if (raise) {
        const float raised = fmaxf(m, top);
        f = m == -INFINITY ? 0.0f : exp2_fast(__fsub_rn(m, raised));
        m = raised;
        l = __fmul_rn(l, f);
      }
      const float shift = m == -INFINITY ? 0.0f : __fsub_rn(kWeightShift, m);
      float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int c = 0; c < 64; c += 16) {
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          float2 w = fma2_f32(make_float2(x[c >> 5][(c & 31) + 2 * j], x[c >> 5][(c & 31) + 2 * j + 1]), make_float2(fac, fac),
                              make_float2(shift, shift));
          w.x = exp2_fast(w.x);
          w.y = exp2_fast(w.y);
          sums[j & 1] = add2_f32(sums[j & 1], w);
          r[j] = half2_of(w.x, w.y);
        }
        tmem_store8(s_at + c / 2, r);
      }
      const float2 sum = add2_f32(sums[0], sums[1]);
      l = __fadd_rn(l, __fadd_rn(sum.x, sum.y));
      // the sums up to the unit before are complete (their product was issued a turn ago)
      if (i > 0 && !__all_sync(0xffffffffu, pkv_mbar_wait(&bar.o_done[t], (i - 1) & 1))) {
        fine = false;
        break;
      }
      if (raise && i > 0) {
        pkv_tc::fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < D; c += 8) {
          float o[8];
          pkv_tc::tmem_load<8>(base + Y::O + c, o);
          uint32_t r[8];
#pragma unroll
          for (int j = 0; j < 8; j++) r[j] = __float_as_uint(__fmul_rn(o[j], f));
          tmem_store8(base + Y::O + c, r);
        }
      }
      tmem_store_wait();
      pkv_tc::fence_before_sync();
      arrive(&bar.p_full[t][i & 1]);
    }
    if (fine && n > 0) fine = __all_sync(0xffffffffu, pkv_mbar_wait(&bar.o_done[t], (n - 1) & 1));
    pkv_tc::fence_after_sync();
    if (!fine && lane == 0) pkv_report(p.err, 0, s, PKV_VEC_DEVICE_WAIT);
    const int64_t part = (((((int64_t)s * p.c.heads + h) * cp.tasks + task) * cp.splits + split) * kTaskRows) + kTileRows * t + (tid & 127);
    if (cp.splits > 1 && live) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      float o[32];
      __syncwarp();
      if (n > 0) {
        pkv_tc::tmem_load32(base + Y::O + c, o);
      } else {
#pragma unroll
        for (int j = 0; j < 32; j++) o[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 32; j++) o[j] = __fmul_rn(o[j], (j & 1) ? kScaleShift / 16.0f : kScaleShift);
      if (!live) continue;
      if (cp.splits > 1) store_f32<PKV_DST_F32, 32>(p.part_o + part * D + c, o);
      else write_row<T, 32>(p, s, h, row, c, o, m, l, c == 0);
    }
  }
  // every product has been waited for (warp 17) and every read of tensor memory is done
  pkv_tc::fence_before_sync();
  __syncthreads();
  if (warp == 17) {
    pkv_tc::fence_after_sync();
    pkv_tc::tmem_free(tmem, 512);
  }
}

// Joins the splits of a query row; a warp per row, or (W = kJoinWarps) a CTA.
template <int D, int T, int W>
__global__ void __launch_bounds__(kJoinWarps * 32)
kv4_chunk_join_kernel(const __grid_constant__ ChunkParams cp) {
  const AttendParams& p = cp.a;
  const int h = blockIdx.y, s = blockIdx.z, row = blockIdx.x * (kJoinWarps / W) + (threadIdx.x >> 5) / W;
  wait_for_stream();
  int qn = p.q_lens ? p.q_lens[s] : p.q.n;
  if (qn < 0 || qn > p.q.n) qn = 0;
  if (row >= qn * p.group) return;
  const int task = row / kTaskRows;
  const int64_t first = ((((int64_t)s * p.c.heads + h) * cp.tasks + task) * cp.splits) * kTaskRows + (row - task * kTaskRows);
  join_parts<D, T, W>(p, s, h, row, cp.splits, [&](int k) { return first + (int64_t)k * kTaskRows; });
}

struct Plan {
  int tasks, splits;
  int64_t part_rows;
};

Plan make_plan(const Cache& c, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  Plan r;
  const int64_t rows = (int64_t)q->n_tokens * (a->n_q_heads / c.heads);
  r.tasks = (int)((rows + kTaskRows - 1) / kTaskRows);
  int64_t longest = a->max_len > 0 && a->max_len < c.capacity ? a->max_len : c.capacity;
  if (a->window > 0 && !c.positions) {
    const int64_t seen = (int64_t)a->window + a->sinks + q->n_tokens + 3 * kUnitTokens;
    if (seen < longest) longest = seen;
  }
  const int64_t units = (longest + kUnitTokens - 1) / kUnitTokens, ctas = (int64_t)r.tasks * c.heads * c.n_seqs;
  // one CTA fits an SM; where the tasks leave SMs idle the tokens are split
  int64_t splits = sm_count() / (ctas > 0 ? ctas : 1);
  if (splits > units / kMinUnits) splits = units / kMinUnits;
  r.splits = splits < 1 ? 1 : (int)splits;
  r.part_rows = r.splits > 1 ? ctas * r.splits * kTaskRows : 0;
  return r;
}

template <int D, int T>
int launch(const ChunkParams& cp, int64_t rows, cudaStream_t s) {
  auto kernel = kv4_chunk_kernel<D, T>;
  constexpr int bytes = Layout<D>::BYTES;
  if (cudaError_t ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return pkv_cuda_status(ce);
  if (cudaError_t ce = launch_early(kernel, dim3(cp.tasks * cp.splits, cp.a.c.heads, cp.a.c.n_seqs), kThreads, bytes, s, cp))
    return pkv_cuda_status(ce);
  if (cp.splits == 1) return PKV_OK;
  const bool many = cp.splits <= 16;  // few splits a row
  return pkv_cuda_status(launch_early(many ? kv4_chunk_join_kernel<D, T, 1> : kv4_chunk_join_kernel<D, T, kJoinWarps>,
                                      dim3((unsigned)(many ? (rows + kJoinWarps - 1) / kJoinWarps : rows), cp.a.c.heads, cp.a.c.n_seqs),
                                      kJoinWarps * 32, 0, s, cp));
}

}  // namespace

namespace pkv_kv4 {

// More rows than three of the other kernel's largest tiles; f32 queries stay there (their two terms do not fit the tile).
// 8 kv heads of 128, 48 rows, here and there: 32 sequences of 8192 tokens 253 and 244 us, one of 131,071 122 and 127, four of
// 1024 22.5 and 14.9; 64 rows: 254 and 320, 121 and 165, 23 and 15.
bool chunk_takes(const pkv_kv4_rows* q, int group) {
  return q->dtype != PKV_DST_F32 && (int64_t)q->n_tokens * group > 48;
}

int64_t chunk_workspace_bytes(const Cache& c, int dim, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a) {
  return make_plan(c, q, a).part_rows * (dim + 2) * (int64_t)sizeof(float);
}

int launch_chunk(AttendParams p, int dim, int dtype, const pkv_kv4_rows* q, const pkv_kv4_attend_args* a, void* workspace,
                 cudaStream_t s) {
  const Plan plan = make_plan(p.c, q, a);
  ChunkParams cp;
  p.part_o = (float*)workspace;
  p.part_ml = p.part_o + plan.part_rows * dim;
  cp.a = p;
  cp.tasks = plan.tasks;
  cp.splits = plan.splits;
  const int64_t rows = (int64_t)q->n_tokens * p.group;
  if (dim == 64) return dtype == PKV_DST_F16 ? launch<64, PKV_DST_F16>(cp, rows, s) : launch<64, PKV_DST_BF16>(cp, rows, s);
  return dtype == PKV_DST_F16 ? launch<128, PKV_DST_F16>(cp, rows, s) : launch<128, PKV_DST_BF16>(cp, rows, s);
}

}  // namespace pkv_kv4
