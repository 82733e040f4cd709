// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Two launches.  The first has one CTA per (sequence, kv head): a radix selection over the weights' bits finds the
// smallest one that stays (weights are not negative, so their bits order like they do; 8 bits at a time from the
// top, counts only, so no order of the atomics shows), then one ordered pass lists the slots freed below the budget
// and the kept slots above it.  The second launch moves the rows of the lists; sources and destinations are
// disjoint, so no order is needed, and only what has to move does.  The keys stay in shared memory between the
// passes where they fit; the first launch then reads 8 bytes a slot once.
#include "pkv_kv4.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxSharedKeys = 48 * 1024;

struct EvictParams {
  Cache c;
  int budget, sinks, recent;
  int list;         // entries of each of a list's halves
  int shared_keys;  // 1: the keys of a sequence fit in shared memory
  int32_t* lists;   // [n_seqs][heads][2][list]: destinations, sources
  int32_t* counts;  // [n_seqs][heads]
  uint64_t* err;
};

// Weights that are not above zero (NaN as well) count as 0; the tokens that stay anyway come before every weight.
__device__ __forceinline__ uint32_t key_of(int position, float mass, int sinks, int recent_from) {
  if (position < sinks || position >= recent_from) return 0xffffffffu;
  return mass > 0.0f ? __float_as_uint(mass) : 0u;
}

__global__ void __launch_bounds__(kThreads)
kv4_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_pick[2];      // digit, how many are left to take within it
  __shared__ int s_warp[32][3];
  const int h = blockIdx.x, s = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = p.c.length(s, p.err);
  const int64_t at = (int64_t)s * p.c.heads + h;
  if (n <= p.budget) {
    if (tid == 0) p.counts[at] = 0;
    return;
  }
  const int recent_from = p.c.end(s, n) - p.recent;
  const int32_t* pos = p.c.positions + p.c.stat(s, h);
  const float* mass = p.c.mass + p.c.stat(s, h);
  auto key = [&](int j) {
    return p.shared_keys ? s_keys[j] : key_of(__ldg(pos + j), __ldg(mass + j), p.sinks, recent_from);
  };
  if (p.shared_keys) {
    for (int j = tid; j < n; j += kThreads) s_keys[j] = key_of(__ldg(pos + j), __ldg(mass + j), p.sinks, recent_from);
  }
  // the budget-th largest key, digit by digit: `prefix` are the digits found, `left` how many of the keys that
  // share them are still to be taken
  uint32_t prefix = 0, left = (uint32_t)p.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kThreads) {
      const uint32_t k = key(j);
      if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {  // lane l owns digits 255 - 8 l .. 248 - 8 l
      uint32_t mine = 0, c[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        c[i] = s_hist[255 - 8 * lane - i];
        mine += c[i];
      }
      uint32_t before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += t;
      }
      before -= mine;
      if (before < left && left <= before + mine) {
        uint32_t have = before;
        int i = 0;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k == i && have + c[k] < left) {
            have += c[k];
            i = k + 1;
          }
        s_pick[0] = 255u - 8u * lane - (uint32_t)i;
        s_pick[1] = left - have;
      }
    }
    __syncthreads();
    prefix = (prefix << 8) | s_pick[0];
    left = s_pick[1];
  }
  // slots in order: of the keys equal to `prefix` the first `left` stay
  int32_t* dst = p.lists + at * 2 * p.list;
  int32_t* src = dst + p.list;
  int equal_before = 0, holes_before = 0, moves_before = 0;
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? key(j) : 0u;
    const bool equal = j < n && k == prefix;
    const unsigned eq = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) s_warp[warp][0] = __popc(eq);
    __syncthreads();
    int e = equal_before + __popc(eq & ((1u << lane) - 1u)), e_all = 0;
    {
      const int t = s_warp[lane][0];
      int before = lane < warp ? t : 0, all = t;
      before = __reduce_add_sync(0xffffffffu, before);
      e_all = __reduce_add_sync(0xffffffffu, all);
      e += before;
    }
    equal_before += e_all;
    const bool kept = j < n && (k > prefix || (equal && e < (int)left));
    const bool hole = j < n && !kept && j < p.budget, move = kept && j >= p.budget;
    const unsigned hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, move);
    if (lane == 0) {
      s_warp[warp][1] = __popc(hb);
      s_warp[warp][2] = __popc(mb);
    }
    __syncthreads();
    const int th = s_warp[lane][1], tm = s_warp[lane][2];
    const int h_at = holes_before + __reduce_add_sync(0xffffffffu, lane < warp ? th : 0) + __popc(hb & ((1u << lane) - 1u));
    const int m_at = moves_before + __reduce_add_sync(0xffffffffu, lane < warp ? tm : 0) + __popc(mb & ((1u << lane) - 1u));
    holes_before += __reduce_add_sync(0xffffffffu, th);
    moves_before += __reduce_add_sync(0xffffffffu, tm);
    if (hole && h_at < p.list) dst[h_at] = j;
    if (move && m_at < p.list) src[m_at] = j;
    __syncthreads();
  }
  if (tid == 0) p.counts[at] = min(min(holes_before, moves_before), p.list);
}

// 16 lanes move a row: K codes, V codes (their halves swap places where the two slots differ in bit 1), scales,
// position and mass.
template <int D>
__global__ void __launch_bounds__(256)
kv4_move_kernel(const __grid_constant__ EvictParams p) {
  using A = Atom<D>;
  const int h = blockIdx.y, s = blockIdx.z;
  const int64_t at = (int64_t)s * p.c.heads + h;
  const int count = p.counts[at];
  const int32_t* dst = p.lists + at * 2 * p.list;
  const int32_t* src = dst + p.list;
  const int part = threadIdx.x & 15;
  for (int i = blockIdx.x * 16 + (threadIdx.x >> 4); i < count; i += gridDim.x * 16) {
    const int a = src[i], b = dst[i];
    const uint8_t* from = p.c.atom(s, h, a / kAtomTokens, A::BYTES, p.err);
    uint8_t* to = p.c.atom(s, h, b / kAtomTokens, A::BYTES, p.err);
    if (!from || !to) continue;
    const int ta = a % kAtomTokens, tb = b % kAtomTokens;
    constexpr int PIECES = A::ROW / 16;  // 16-byte pieces of a code row: 4 or 2
    if (part < PIECES) {
      *reinterpret_cast<uint4*>(to + A::KC + tb * A::ROW + 16 * part) =
          *reinterpret_cast<const uint4*>(from + A::KC + ta * A::ROW + 16 * part);
    } else if (part < 2 * PIECES) {
      const int o = 16 * (part - PIECES);
      *reinterpret_cast<uint4*>(to + A::VC + tb * A::ROW + (o ^ A::vswap(tb))) =
          *reinterpret_cast<const uint4*>(from + A::VC + ta * A::ROW + (o ^ A::vswap(ta)));
    } else if (part < 2 * PIECES + 2 * (A::SROW / 4)) {
      const int o = part - 2 * PIECES, side = o / (A::SROW / 4), w = 4 * (o % (A::SROW / 4));
      const int base = side ? A::VS : A::KS;
      *reinterpret_cast<uint32_t*>(to + base + tb * A::SROW + w) =
          *reinterpret_cast<const uint32_t*>(from + base + ta * A::SROW + w);
    } else if (part == 14) {
      p.c.positions[p.c.stat(s, h) + b] = p.c.positions[p.c.stat(s, h) + a];
    } else if (part == 15) {
      p.c.mass[p.c.stat(s, h) + b] = p.c.mass[p.c.stat(s, h) + a];
    }
  }
}

int list_entries(const Cache& c, int budget) {
  const int above = c.capacity - budget;
  return above <= 0 ? 0 : (above < budget ? above : budget);
}

}  // namespace

extern "C" int64_t pkv_kv4_evict_workspace_bytes(const pkv_kv4_cache* cache, int32_t budget) {
  Cache c;
  if (make_cache(cache, &c) || budget < 1) return 0;
  return (int64_t)c.n_seqs * c.heads * (2 * (int64_t)list_entries(c, budget) + 1) * (int64_t)sizeof(int32_t);
}

extern "C" int pkv_kv4_evict_dev(const pkv_kv4_cache* cache, int32_t budget, int32_t sinks, int32_t recent, void* workspace_dev,
                                 int64_t workspace_bytes, uint64_t* err_dev, void* stream) {
  EvictParams p;
  if (int st = make_cache(cache, &p.c)) return st;
  if (!p.c.positions || !p.c.mass || !err_dev || budget < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return PKV_ERR_INVALID_ARGUMENT;
  p.list = list_entries(p.c, budget);
  if (p.list == 0 || p.c.n_seqs == 0) return PKV_OK;  // no sequence can be longer than the budget
  if (workspace_bytes < pkv_kv4_evict_workspace_bytes(cache, budget)) return PKV_ERR_BUFFER_TOO_SMALL;
  if (!workspace_dev || ((uintptr_t)workspace_dev & 15)) return PKV_ERR_INVALID_ARGUMENT;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  p.shared_keys = p.c.capacity <= kMaxSharedKeys;
  p.lists = (int32_t*)workspace_dev;
  p.counts = p.lists + (int64_t)p.c.n_seqs * p.c.heads * 2 * p.list;
  p.err = err_dev;
  cudaStream_t s = (cudaStream_t)stream;
  const int bytes = p.shared_keys ? p.c.capacity * 4 : 0;
  if (bytes > 48 * 1024)
    if (cudaError_t ce = cudaFuncSetAttribute(kv4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSharedKeys * 4))
      return pkv_cuda_status(ce);
  kv4_select_kernel<<<dim3(p.c.heads, p.c.n_seqs), kThreads, bytes, s>>>(p);
  pkv_count_launch();
  if (cudaError_t ce = cudaGetLastError()) return pkv_cuda_status(ce);
  const int ctas = (p.list + 63) / 64;  // up to four rows for each 16 lanes
  const dim3 grid(ctas, p.c.heads, p.c.n_seqs);
  if (cache->dim == 64) kv4_move_kernel<64><<<grid, 256, 0, s>>>(p);
  else kv4_move_kernel<128><<<grid, 256, 0, s>>>(p);
  pkv_count_launch();
  return pkv_cuda_status(cudaGetLastError());
}
