// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Two launches.  The first has one CTA per (sequence, kv head): a radix selection over the weights' bits finds the
// smallest one that stays (weights are not negative, so their bits order like they do; 11, 11 and 10 bits from the
// top, counts only, so no order of the atomics shows), then every warp walks over a contiguous part of the slots and lists the
// slots freed below the budget and the kept slots above it.  The second launch moves the rows of the lists; sources
// and destinations are disjoint, so no order is needed, and only what has to move does.  The keys stay in shared
// memory between the passes where they fit; the first launch then reads 8 bytes a slot once.
#include "pkv_kv4.cuh"

using namespace pkv_kv4;

namespace {

constexpr int kMaxSharedKeys = 48 * 1024;
constexpr int kBins = 2048;

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

// THREADS: 256 for caches of a few thousand slots (eight CTAs an SM), 1024 for long ones.
template <int THREADS>
__global__ void __launch_bounds__(THREADS)
kv4_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int WARPS = THREADS / 32, PER = kBins / THREADS;
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_warp[2][WARPS];
  __shared__ uint32_t s_pick[2];  // digit, how many are left to take within it
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
  // the sum of a value over the warps before this one; `slot` keeps two calls apart that no barrier separates
  auto before_warp = [&](int slot, uint32_t mine, uint32_t* all) -> uint32_t {
    if (lane == 0) s_warp[slot][warp] = mine;
    __syncthreads();
    const uint32_t v = lane < WARPS ? s_warp[slot][lane] : 0u;
    *all = __reduce_add_sync(0xffffffffu, v);
    return __reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
  };
  if (p.shared_keys) {
#pragma unroll 4
    for (int j = tid; j < n; j += THREADS) s_keys[j] = key_of(__ldg(pos + j), __ldg(mass + j), p.sinks, recent_from);
  }
  // the budget-th largest key, digit by digit: `prefix` are the digits found, `left` how many of the keys that
  // share them are still to be taken
  uint32_t prefix = 0, left = (uint32_t)p.budget;
#pragma unroll
  for (int turn = 0; turn < 3; turn++) {
    const int shift = turn == 0 ? 21 : turn == 1 ? 10 : 0, bits = turn == 2 ? 10 : 11;
    for (int j = tid; j < kBins; j += THREADS) s_hist[j] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += THREADS) {
      const uint32_t k = key(j);
      if (turn == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // thread t owns the PER bins below kBins - t PER, from the top
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      c[i] = s_hist[kBins - 1 - tid * PER - i];
      mine += c[i];
    }
    uint32_t upto = mine, all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const uint32_t before = before_warp(0, __shfl_sync(0xffffffffu, upto, 31), &all) + upto - mine;
    if (before < left && left <= before + mine) {
      uint32_t have = before;
      int i = 0;
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (k == i && have + c[k] < left) {
          have += c[k];
          i = k + 1;
        }
      s_pick[0] = (uint32_t)(kBins - 1 - tid * PER - i);
      s_pick[1] = left - have;
    }
    __syncthreads();
    prefix = (prefix << bits) | s_pick[0];
    left = s_pick[1];
  }
  // slots in order, a contiguous part per warp; of the keys equal to `prefix` the first `left` stay
  const int part = (n + THREADS - 1) / THREADS * 32, j0 = warp * part, j1 = min(n, j0 + part);
  const unsigned below = (1u << lane) - 1u;
  uint32_t equal = 0, all;
  for (int j = j0 + lane; j - lane < j1; j += 32) equal += __popc(__ballot_sync(0xffffffffu, j < j1 && key(j) == prefix));
  const uint32_t equal0 = before_warp(0, equal, &all);
  auto walk = [&](auto each) {  // each(slot, hole, move, lanes with a hole, lanes with a move)
    uint32_t e = equal0;
    for (int j = j0 + lane; j - lane < j1; j += 32) {
      const uint32_t k = j < j1 ? key(j) : 0u;
      const bool same = j < j1 && k == prefix;
      const unsigned eq = __ballot_sync(0xffffffffu, same);
      const bool kept = j < j1 && (k > prefix || (same && e + __popc(eq & below) < left));
      e += __popc(eq);
      const bool hole = j < j1 && !kept && j < p.budget, move = kept && j >= p.budget;
      each(j, hole, move, __ballot_sync(0xffffffffu, hole), __ballot_sync(0xffffffffu, move));
    }
  };
  uint32_t holes = 0, moves = 0, all_moves;
  walk([&](int, bool, bool, unsigned hb, unsigned mb) {
    holes += __popc(hb);
    moves += __popc(mb);
  });
  uint32_t hole_at = before_warp(1, holes, &all);
  uint32_t move_at = before_warp(0, moves, &all_moves);
  int32_t* dst = p.lists + at * 2 * p.list;
  int32_t* src = dst + p.list;
  walk([&](int j, bool hole, bool move, unsigned hb, unsigned mb) {
    const uint32_t a = hole_at + __popc(hb & below), b = move_at + __popc(mb & below);
    if (hole && a < (uint32_t)p.list) dst[a] = j;
    if (move && b < (uint32_t)p.list) src[b] = j;
    hole_at += __popc(hb);
    move_at += __popc(mb);
  });
  if (tid == 0) p.counts[at] = min(min((int)all, (int)all_moves), p.list);
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
  constexpr int PIECES = A::ROW / 16, WORDS = A::SROW / 4;  // 16-byte pieces of a code row, words of a scale row
  constexpr int TURNS = 4;                                  // rows that 16 lanes have in flight
  const int64_t stat = p.c.stat(s, h);
  for (int i0 = blockIdx.x * 16 * TURNS + (threadIdx.x >> 4); i0 < count; i0 += gridDim.x * 16 * TURNS) {
    uint8_t* to[TURNS];
    uint4 v[TURNS];
    int slot[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      to[u] = nullptr;
      const int i = i0 + 16 * u;
      if (i >= count) continue;
      const int a = src[i], b = dst[i];
      const uint8_t* from = p.c.atom(s, h, a / kAtomTokens, A::BYTES, p.err);
      uint8_t* into = p.c.atom(s, h, b / kAtomTokens, A::BYTES, p.err);
      if (!from || !into) continue;
      const int ta = a % kAtomTokens, tb = b % kAtomTokens;
      slot[u] = b;
      if (part < PIECES) {
        v[u] = *reinterpret_cast<const uint4*>(from + A::KC + ta * A::ROW + 16 * part);
        to[u] = into + A::KC + tb * A::ROW + 16 * part;
      } else if (part < 2 * PIECES) {
        const int o = 16 * (part - PIECES);
        v[u] = *reinterpret_cast<const uint4*>(from + A::VC + ta * A::ROW + (o ^ A::vswap(ta)));
        to[u] = into + A::VC + tb * A::ROW + (o ^ A::vswap(tb));
      } else if (part < 2 * PIECES + 2 * WORDS) {
        const int o = part - 2 * PIECES, base = o / WORDS ? A::VS : A::KS, w = 4 * (o % WORDS);
        v[u].x = *reinterpret_cast<const uint32_t*>(from + base + ta * A::SROW + w);
        to[u] = into + base + tb * A::SROW + w;
      } else if (part >= 14) {
        v[u].x = part == 14 ? (uint32_t)p.c.positions[stat + a] : __float_as_uint(p.c.mass[stat + a]);
        to[u] = into;
      }
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      if (!to[u]) continue;
      if (part < 2 * PIECES) *reinterpret_cast<uint4*>(to[u]) = v[u];
      else if (part < 14) *reinterpret_cast<uint32_t*>(to[u]) = v[u].x;
      else if (part == 14) p.c.positions[stat + slot[u]] = (int32_t)v[u].x;
      else p.c.mass[stat + slot[u]] = __uint_as_float(v[u].x);
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
  const dim3 select(p.c.heads, p.c.n_seqs);
  if (p.c.capacity <= 8192) {
    kv4_select_kernel<256><<<select, 256, bytes, s>>>(p);
  } else {
    if (cudaError_t ce = cudaFuncSetAttribute(kv4_select_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSharedKeys * 4))
      return pkv_cuda_status(ce);
    kv4_select_kernel<1024><<<select, 1024, bytes, s>>>(p);
  }
  pkv_count_launch();
  if (cudaError_t ce = cudaGetLastError()) return pkv_cuda_status(ce);
  const int ctas = (p.list + 63) / 64;  // every move in flight at once
  const dim3 grid(ctas, p.c.heads, p.c.n_seqs);
  if (cache->dim == 64) kv4_move_kernel<64><<<grid, 256, 0, s>>>(p);
  else kv4_move_kernel<128><<<grid, 256, 0, s>>>(p);
  pkv_count_launch();
  return pkv_cuda_status(cudaGetLastError());
}
