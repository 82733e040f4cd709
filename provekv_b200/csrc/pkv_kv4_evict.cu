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
  int fused;        // 1: the first launch moves the rows too
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

// 16 lanes move a row: K codes, V codes (their halves swap places where the two slots differ in bit 1), scales,
// position and mass.  Rows first, first + step, .. of the lists.
template <int D, int TURNS>  // TURNS: rows that 16 lanes have in flight
__device__ __forceinline__ void move_rows(const EvictParams& p, int s, int h, const int32_t* dst, const int32_t* src, int count, int first,
                                          int step) {
  using A = Atom<D>;
  const int part = threadIdx.x & 15;
  constexpr int PIECES = A::ROW / 16, WORDS = A::SROW / 4;  // 16-byte pieces of a code row, words of a scale row
  const int64_t stat = p.c.stat(s, h);
  // what this lane moves: bytes into the atom, per token, and whether the token swaps halves
  const bool wide = part < 2 * PIECES, scale = !wide && part < 2 * PIECES + 2 * WORDS, swaps = wide && part >= PIECES;
  int base, per_token;
  if (wide) {
    base = part < PIECES ? A::KC + 16 * part : A::VC;
    per_token = A::ROW;
  } else {
    const int o = part - 2 * PIECES;
    base = (o / WORDS ? A::VS : A::KS) + 4 * (o % WORDS);
    per_token = A::SROW;
  }
  const int half = swaps ? 16 * (part - PIECES) : 0;
  auto at = [&](int slot) { return base + (slot % kAtomTokens) * per_token + (swaps ? half ^ A::vswap(slot) : 0); };
  auto page_of = [&](int slot) { return __ldg(p.c.table + (int64_t)s * p.c.max_pages + slot / p.c.page_tokens); };
  auto atom_of = [&](int page, int slot) {
    return p.c.pages + (((int64_t)page * p.c.heads + h) * p.c.page_atoms + slot % p.c.page_tokens / kAtomTokens) * (int64_t)A::BYTES;
  };
#pragma unroll 1
  for (int i0 = first; i0 < count; i0 += step * TURNS) {
    int from[TURNS], to[TURNS], from_page[TURNS], to_page[TURNS];
    bool live[TURNS];
    uint4 v[TURNS];
    // step by step for all rows, so that their loads are in flight together
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      const int i = min(i0 + step * u, count - 1);
      live[u] = i0 + step * u < count;
      from[u] = src[i];
      to[u] = dst[i];
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      from_page[u] = page_of(from[u]);
      to_page[u] = page_of(to[u]);
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      if (from_page[u] < 0 || from_page[u] >= p.c.n_pages || to_page[u] < 0 || to_page[u] >= p.c.n_pages) {
        if (live[u] && part == 0) pkv_report(p.err, 0, s, PKV_VEC_BAD_SEQUENCE);
        live[u] = false;
      }
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      if (live[u] && wide) v[u] = *reinterpret_cast<const uint4*>(atom_of(from_page[u], from[u]) + at(from[u]));
      if (live[u] && scale) v[u].x = *reinterpret_cast<const uint32_t*>(atom_of(from_page[u], from[u]) + at(from[u]));
      if (live[u] && part == 14) v[u].x = (uint32_t)p.c.positions[stat + from[u]];
      if (live[u] && part == 15) v[u].x = __float_as_uint(p.c.mass[stat + from[u]]);
    }
#pragma unroll
    for (int u = 0; u < TURNS; u++) {
      if (live[u] && wide) *reinterpret_cast<uint4*>(atom_of(to_page[u], to[u]) + at(to[u])) = v[u];
      if (live[u] && scale) *reinterpret_cast<uint32_t*>(atom_of(to_page[u], to[u]) + at(to[u])) = v[u].x;
      if (live[u] && part == 14) p.c.positions[stat + to[u]] = (int32_t)v[u].x;
      if (live[u] && part == 15) p.c.mass[stat + to[u]] = __uint_as_float(v[u].x);
    }
  }
}

// THREADS: 256 for caches of a few thousand slots (several CTAs an SM), 1024 for long ones.
template <int D, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 6 : 1)
kv4_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int WARPS = THREADS / 32, PER = kBins / THREADS;
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_warp[2][WARPS];
  __shared__ uint32_t s_pick[3];  // digit, how many are left to take within it, how many there are
  const int h = blockIdx.x, s = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wait_for_stream();
  const int n = p.c.length(s, p.err);
  const int64_t at = (int64_t)s * p.c.heads + h;
  if (n <= p.budget) {
    if (tid == 0 && !p.fused) p.counts[at] = 0;
    return;
  }
  const int recent_from = p.c.end(s, n, p.err) - p.recent;
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
    // four slots a load; the last one may reach behind the sequence, never behind its capacity (a multiple of 16)
    const int4* pos4 = reinterpret_cast<const int4*>(pos);
    const float4* mass4 = reinterpret_cast<const float4*>(mass);
#pragma unroll 4
    for (int j = tid; j < (n + 3) / 4; j += THREADS) {
      const int4 q = __ldg(pos4 + j);
      const float4 m = __ldg(mass4 + j);
      reinterpret_cast<uint4*>(s_keys)[j] =
          make_uint4(key_of(q.x, m.x, p.sinks, recent_from), key_of(q.y, m.y, p.sinks, recent_from),
                     key_of(q.z, m.z, p.sinks, recent_from), key_of(q.w, m.w, p.sinks, recent_from));
    }
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
      s_pick[2] = 0u;
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (k == i) s_pick[2] = c[k];
    }
    __syncthreads();
    prefix = (prefix << bits) | s_pick[0];
    left = s_pick[1];
  }
  // Slots in order, a contiguous part per warp.  Of the keys equal to `prefix` the first `left` stay: all of them, unless the
  // budget cuts through equal weights.
  const bool cut = left < s_pick[2];
  const int part = (n + THREADS - 1) / THREADS * 32, j0 = warp * part, j1 = min(n, j0 + part);
  const unsigned below = (1u << lane) - 1u;
  uint32_t equal0 = 0, all;
  if (cut) {
    uint32_t equal = 0;
    for (int j = j0 + lane; j - lane < j1; j += 32) equal += __popc(__ballot_sync(0xffffffffu, j < j1 && key(j) == prefix));
    equal0 = before_warp(0, equal, &all);
  }
  // each(slot, whether it is in its list, the row's lanes that are, the row's lanes below the budget): a slot below the
  // budget is listed when it is freed, one above when it is kept
  auto walk = [&](auto each) {
    uint32_t e = equal0;
    for (int j = j0 + lane, row = j0; row < j1; j += 32, row += 32) {
      const uint32_t k = j < j1 ? key(j) : 0u;
      bool kept = k >= prefix;
      if (cut) {
        const unsigned eq = __ballot_sync(0xffffffffu, j < j1 && k == prefix);
        kept = k > prefix || (k == prefix && e + __popc(eq & below) < left);
        e += __popc(eq);
      }
      const bool listed = j < j1 && (j < p.budget) != kept;
      const unsigned low = row + 32 <= p.budget ? 0xffffffffu : row >= p.budget ? 0u : (1u << (p.budget - row)) - 1u;
      each(j, listed, __ballot_sync(0xffffffffu, listed), low);
    }
  };
  uint32_t holes = 0, moves = 0, all_moves;
  walk([&](int, bool, unsigned rows, unsigned low) {
    holes += __popc(rows & low);
    moves += __popc(rows & ~low);
  });
  uint32_t hole_at = before_warp(1, holes, &all);
  uint32_t move_at = before_warp(0, moves, &all_moves);
  int32_t* dst = p.lists + at * 2 * p.list;
  int32_t* src = dst + p.list;
  walk([&](int j, bool listed, unsigned rows, unsigned low) {
    if (listed) {
      const bool hole = j < p.budget;
      const uint32_t i = hole ? hole_at + __popc(rows & low & below) : move_at + __popc(rows & ~low & below);
      if (i < (uint32_t)p.list) (hole ? dst : src)[i] = j;
    }
    hole_at += __popc(rows & low);
    move_at += __popc(rows & ~low);
  });
  const int count = min(min((int)all, (int)all_moves), p.list);
  if (p.fused) {  // few rows: this CTA moves them, without a second launch
    __syncthreads();
    move_rows<D, 1>(p, s, h, dst, src, count, tid >> 4, THREADS / 16);
  } else if (tid == 0) {
    p.counts[at] = count;
  }
}

template <int D>
__global__ void __launch_bounds__(256, 5)
kv4_move_kernel(const __grid_constant__ EvictParams p) {
  const int h = blockIdx.y, s = blockIdx.z;
  wait_for_stream();
  const int64_t at = (int64_t)s * p.c.heads + h;
  const int count = min(p.counts[at], (int)blockIdx.x * 32 + 32);
  const int32_t* dst = p.lists + at * 2 * p.list;
  move_rows<D, 2>(p, s, h, dst, dst + p.list, count, blockIdx.x * 32 + (threadIdx.x >> 4), 16);
}


int list_entries(const Cache& c, int budget) {
  const int above = c.capacity - budget;
  return above <= 0 ? 0 : (above < budget ? above : budget);
}

template <int D>
int launch(const EvictParams& p, cudaStream_t s) {
  const int bytes = p.shared_keys ? p.c.capacity * 4 : 0;
  const dim3 select(p.c.heads, p.c.n_seqs);
  if (p.c.capacity > 8192)
    if (cudaError_t ce = cudaFuncSetAttribute(kv4_select_kernel<D, 1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSharedKeys * 4))
      return pkv_cuda_status(ce);
  if (cudaError_t ce = p.c.capacity <= 8192 ? launch_early(kv4_select_kernel<D, 256>, select, 256, bytes, s, p)
                                            : launch_early(kv4_select_kernel<D, 1024>, select, 1024, bytes, s, p))
    return pkv_cuda_status(ce);
  if (p.fused) return PKV_OK;
  return pkv_cuda_status(
      launch_early(kv4_move_kernel<D>, dim3((p.list + 31) / 32, p.c.heads, p.c.n_seqs), 256, 0, s, p));  // every move in flight at once
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
  p.fused = p.list <= 256;  // a few turns of a CTA's 16-lane groups
  p.lists = (int32_t*)workspace_dev;
  p.counts = p.lists + (int64_t)p.c.n_seqs * p.c.heads * 2 * p.list;
  p.err = err_dev;
  cudaStream_t s = (cudaStream_t)stream;
  return cache->dim == 64 ? launch<64>(p, s) : launch<128>(p, s);
}
