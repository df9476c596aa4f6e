// paged_evict.cu -- the tokens of least accumulated attention weight leave the
// cache.
//
// Per row and key head, of len > budget cached tokens the len - budget lowest
// by (protected, weight, index) are the victims; protected are the positions
// below `sink` and those at or above seen - recent.  A NaN weight counts as
// +inf.  The i-th victim below the budget (a hole) then takes the keys, values,
// weight and position of the i-th survivor at or above it (a mover): holes and
// movers are equally many, no slot is both read and written, and a step that
// is one token over its budget moves one token instead of the whole cache.
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {
namespace {

// The order of the victims as one unsigned number: it rises with the weight, a
// NaN is +inf, the protected come last.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sink, int first_recent) {
  if (pos < sink || pos >= first_recent) return 0xFFFFFFFFu;
  if (w != w) return 0xFF800000u;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kThreads = 512;
constexpr int kBins = 2048;  // 11 bits a pass: the key's 32 in three
constexpr int kMaxCluster = 8;

// Inclusive prefix sums over the block of two counts at once.
__device__ __forceinline__ int2 block_scan(int2 x, int2* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xFFFFFFFFu, x.x, o), b = __shfl_up_sync(0xFFFFFFFFu, x.y, o);
    if (lane >= o) {
      x.x += a;
      x.y += b;
    }
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int2 y = lane < kThreads / 32 ? sums[lane] : make_int2(0, 0);
#pragma unroll
    for (int o = 1; o < kThreads / 32; o <<= 1) {
      const int a = __shfl_up_sync(0xFFFFFFFFu, y.x, o), b = __shfl_up_sync(0xFFFFFFFFu, y.y, o);
      if (lane >= o) {
        y.x += a;
        y.y += b;
      }
    }
    if (lane < kThreads / 32) sums[lane] = y;
  }
  __syncthreads();
  if (warp > 0) {
    x.x += sums[warp - 1].x;
    x.y += sums[warp - 1].y;
  }
  return x;
}

// One cluster per (key head, row).  Each block keeps the keys of its share of
// the slots in shared memory, so weights and positions are read once.  Three
// passes over 11 bits, their histograms summed over the cluster, find the last
// victim's key; prefix sums in the order of the slots number ties, holes and
// movers; every hole and mover is written to the list of the block that will
// move it, and the blocks move their pairs in 16-byte pieces.
// Bound by latency where few tokens move (six cluster barriers), else by the
// rows moved.
__global__ void __launch_bounds__(kThreads, 2) evict_kernel(const EvictParams p, int slots) {
  extern __shared__ __align__(16) uint32_t keys[];  // [slots]; then to[slots / 2 + 1], by[slots / 2 + 1]
  __shared__ __align__(16) int hist[3][kBins];
  __shared__ int2 sums[kThreads / 32];
  __shared__ int pick[2];
  __shared__ int2 count[2];  // this block's (ties, -), (holes, movers)
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int h = blockIdx.x / C, row = blockIdx.y, tid = threadIdx.x;
  griddep_wait();
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int len = p.lens[row];
  if (len < 0 || len > cap) {
    if (tid == 0) atomicOr(p.c.status, kPagedBadIndex);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  if (h == 0 && rank == 0 && tid == 0 && p.new_lens) p.new_lens[row] = min(len, p.budget);
  if (len <= p.budget) return;
  for (int i = tid; i < 3 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
  __syncthreads();

  // This block's slots [n0, n0 + mine); thread t owns `run` of them from t * run
  // on (an odd number: its walk meets no bank conflict).
  const int share = (len + C - 1) / C, n0 = min(len, rank * share), mine = min(share, len - n0);
  const int run = (mine + kThreads - 1) / kThreads | 1, first_recent = p.seen[row] - p.recent;
  auto slot_at = [&](int n) {
    const int64_t s = slot_of(p.c, p.t, row, n);
    return s < 0 ? -1 : static_cast<int>(s) + h * p.c.page_size;
  };
#pragma unroll 4
  for (int i = tid; i < mine; i += kThreads) {
    const int s = slot_at(n0 + i);
    const uint32_t k = s < 0 ? 0xFFFFFFFFu : evict_key(p.c.weight[s], p.c.position[s], p.sink, first_recent);
    keys[i] = k;
    atomicAdd(&hist[0][k >> 21], 1);
  }
  int need = len - p.budget;  // victims among the keys that share the prefix
  uint32_t prefix = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    if (pass > 0) {
      const int above = pass == 1 ? 21 : 10;
      for (int i = tid; i < mine; i += kThreads) {
        const uint32_t k = keys[i];
        if (k >> above == prefix >> above) atomicAdd(&hist[pass][(k >> shift) & (kBins - 1)], 1);
      }
    }
    cluster.sync();
    int bin[kBins / kThreads], all = 0;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) bin[i] = 0;
    for (int c = 0; c < C; ++c) {
      const int4 x = *reinterpret_cast<const int4*>(cluster.map_shared_rank(&hist[pass][0], c) + 4 * tid);
      bin[0] += x.x;
      bin[1] += x.y;
      bin[2] += x.z;
      bin[3] += x.w;
    }
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) all += bin[i];
    int below = block_scan(make_int2(all, 0), sums).x - all;
    if (below < need && need <= below + all) {
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) {
        if (need > below && need <= below + bin[i]) {
          pick[0] = 4 * tid + i;
          pick[1] = need - below;
        }
        below += bin[i];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    need = pick[1];
  }

  // Victims are the keys below `prefix` and the first `need` equal to it.
  const int i0 = min(mine, tid * run), i1 = min(mine, i0 + run);
  int ties = 0;
  for (int i = i0; i < i1; ++i) ties += keys[i] == prefix;
  int2 upto = block_scan(make_int2(ties, 0), sums);
  if (tid == kThreads - 1) count[0] = upto;
  cluster.sync();
  int tie = upto.x - ties;
  for (int c = 0; c < rank; ++c) tie += cluster.map_shared_rank(&count[0], c)->x;
  auto victim = [&](uint32_t k, int& t) { return k < prefix || (k == prefix && t++ < need); };
  int2 own = make_int2(0, 0);  // holes, movers of this thread's run
  for (int i = i0, t = tie; i < i1; ++i) {
    const bool out = victim(keys[i], t), low = n0 + i < p.budget;
    own.x += out && low;
    own.y += !out && !low;
  }
  upto = block_scan(own, sums);
  if (tid == kThreads - 1) count[1] = upto;
  cluster.sync();
  int2 at = make_int2(upto.x - own.x, upto.y - own.y);
  int pairs = 0;
  for (int c = 0; c < C; ++c) {
    const int2 x = *cluster.map_shared_rank(&count[1], c);
    pairs += x.x;
    if (c < rank) {
      at.x += x.x;
      at.y += x.y;
    }
  }
  const int per = (pairs + C - 1) / C, room = slots / 2 + 1;  // pairs of a block's list; per <= room as holes <= len / 2
  int* to = reinterpret_cast<int*>(keys + slots);
  int* by = to + room;
  if (own.x + own.y > 0) {
    for (int i = i0, t = tie; i < i1; ++i) {
      const bool out = victim(keys[i], t), low = n0 + i < p.budget;
      if (out != low) continue;
      const int e = out ? at.x++ : at.y++, c = e / per;
      *cluster.map_shared_rank((out ? to : by) + (e - c * per), c) = slot_at(n0 + i);
    }
  }
  cluster.sync();

  const int list = min(per, pairs - rank * per), bytes = p.c.head_dim * (p.c.dtype == MXMOE_F32 ? 4 : p.c.dtype == MXMOE_BF16 ? 2 : 1);
  const int pieces = bytes / 16;
  uint4 *k16 = static_cast<uint4*>(p.c.k), *v16 = static_cast<uint4*>(p.c.v);
#pragma unroll 4
  for (int i = tid; i < list * pieces; i += kThreads) {
    const int e = i / pieces, c = i - e * pieces;
    if (to[e] < 0 || by[e] < 0) continue;
    const int64_t d = static_cast<int64_t>(to[e]) * pieces + c, f = static_cast<int64_t>(by[e]) * pieces + c;
    const uint4 a = k16[f], b = v16[f];
    k16[d] = a;
    v16[d] = b;
  }
  for (int e = tid; e < list; e += kThreads) {
    if (to[e] < 0 || by[e] < 0) continue;
    p.c.weight[to[e]] = p.c.weight[by[e]];
    p.c.position[to[e]] = p.c.position[by[e]];
  }
}

constexpr int kLongThreads = 1024;

// Exclusive prefix sum over the block of a 0 / 1 flag; `total` gets the sum.
__device__ __forceinline__ int block_rank(bool flag, int* warp_sums, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned b = __ballot_sync(0xFFFFFFFFu, flag);
  if (lane == 0) warp_sums[warp] = __popc(b);
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < kLongThreads / 32; ++i) {
    const int s = warp_sums[i];
    if (i < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + __popc(b & ((1u << lane) - 1));
}

// For tables too long for the kernel above.  One block per (key head, row): a
// radix selection of the last victim's key, the keys read anew in each pass,
// then one walk over the slots below the budget and one over those above it,
// which hand each other holes and movers through shared memory.
__global__ void __launch_bounds__(kLongThreads) evict_long_kernel(const EvictParams p) {
  griddep_wait();
  __shared__ int hist[256], sums[kLongThreads / 32], pick[2];
  __shared__ int64_t holes[kLongThreads], movers[kLongThreads];
  const int h = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int len = p.lens[row];
  if (len < 0 || len > cap) {
    if (tid == 0) atomicOr(p.c.status, kPagedBadIndex);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  if (h == 0 && tid == 0 && p.new_lens) p.new_lens[row] = min(len, p.budget);
  if (len <= p.budget) return;
  const int first_recent = p.seen[row] - p.recent;
  const int64_t head = static_cast<int64_t>(h) * p.c.page_size;
  auto key_at = [&](int n, int64_t& slot) {
    slot = slot_of(p.c, p.t, row, n);
    if (slot < 0) return 0xFFFFFFFFu;
    slot += head;
    return evict_key(p.c.weight[slot], p.c.position[slot], p.sink, first_recent);
  };
  int need = len - p.budget;  // victims among the keys that still share the prefix
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int n = tid; n < len; n += kLongThreads) {
      int64_t slot;
      const uint32_t k = key_at(n, slot);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int below = 0, d = 0;
      while (below + hist[d] < need) below += hist[d++];
      pick[0] = d;
      pick[1] = need - below;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    need = pick[1];
    __syncthreads();
  }
  // Victims: keys below `prefix`, and the first `need` of those equal to it.
  const int64_t row_bytes = static_cast<int64_t>(p.c.head_dim) * (p.c.dtype == MXMOE_F32 ? 4 : p.c.dtype == MXMOE_BF16 ? 2 : 1);
  const int words = static_cast<int>(row_bytes / 8);
  int ties = 0, lo = 0, hi = p.budget, n_holes = 0, n_movers = 0;
  int hi_ties = 0;  // ties below the budget, counted first: the walk above it goes on from there
  for (int n0 = 0; n0 < p.budget; n0 += kLongThreads) {
    int64_t slot;
    int total;
    block_rank(n0 + tid < p.budget && key_at(n0 + tid, slot) == prefix, sums, total);
    hi_ties += total;
  }
  while (true) {
    while (n_holes == 0 && lo < p.budget) {
      const int n = lo + tid;
      int64_t slot = -1;
      const uint32_t k = n < p.budget ? key_at(n, slot) : 0xFFFFFFFFu;
      int total;
      const int r = ties + block_rank(n < p.budget && k == prefix, sums, total);
      ties += total;
      const bool hole = n < p.budget && slot >= 0 && (k < prefix || (k == prefix && r < need));
      const int i = block_rank(hole, sums, n_holes);
      if (hole) holes[i] = slot;
      lo += kLongThreads;
    }
    while (n_movers == 0 && hi < len) {
      const int n = hi + tid;
      int64_t slot = -1;
      const uint32_t k = n < len ? key_at(n, slot) : 0;
      int total;
      const int r = hi_ties + block_rank(n < len && k == prefix, sums, total);
      hi_ties += total;
      const bool mover = n < len && slot >= 0 && (k > prefix || (k == prefix && r >= need));
      const int i = block_rank(mover, sums, n_movers);
      if (mover) movers[i] = slot;
      hi += kLongThreads;
    }
    __syncthreads();
    const int m = min(n_holes, n_movers);
    if (m == 0) break;
    for (int i = tid; i < m * words; i += kLongThreads) {
      const int j = i / words;
      const int64_t to = holes[j] * words + (i - j * words), by = movers[j] * words + (i - j * words);
      static_cast<uint2*>(p.c.k)[to] = static_cast<uint2*>(p.c.k)[by];
      static_cast<uint2*>(p.c.v)[to] = static_cast<uint2*>(p.c.v)[by];
    }
    int64_t keep = -1;
    const bool left_hole = tid >= m && tid < n_holes, left_mover = tid >= m && tid < n_movers;
    if (tid < m) {
      p.c.weight[holes[tid]] = p.c.weight[movers[tid]];
      p.c.position[holes[tid]] = p.c.position[movers[tid]];
    }
    if (left_hole) keep = holes[tid];
    if (left_mover) keep = movers[tid];
    __syncthreads();
    if (left_hole) holes[tid - m] = keep;
    if (left_mover) movers[tid - m] = keep;
    n_holes -= m;
    n_movers -= m;
    __syncthreads();
  }
}

// New lengths in the place of the old ones, once every block has read those.
__global__ void lens_kernel(const EvictParams p, int32_t* lens) {
  griddep_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.rows) return;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  const int64_t len = min(max(static_cast<int64_t>(p.lens[i]), static_cast<int64_t>(0)), cap);
  lens[i] = static_cast<int>(min(len, static_cast<int64_t>(p.budget)));
}

cudaError_t launch_select(const EvictParams& p, int sms, cudaStream_t st) {
  // Blocks of a (row, key head): enough for two a SM, no more than leaves each
  // a thread's slot, and at least what the longest row's keys and lists (8 bytes
  // a slot) need.
  constexpr int kSlots = 10 * 1024;  // two blocks share a SM
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int C = 1;
  while (C < kMaxCluster && ((cap + C - 1) / C > kSlots || (p.rows * p.c.kv_heads * C < 2 * sms && cap / C > 2 * kThreads))) C *= 2;
  const int64_t slots = ((cap + C - 1) / C + 3) / 4 * 4;
  if (slots > 24 * 1024) {  // past one block's shared memory
    return launch_kernel(evict_long_kernel, dim3(p.c.kv_heads, p.rows), dim3(kLongThreads), 0, st, p);
  }
  const size_t smem = (static_cast<size_t>(slots) + 2 * (slots / 2 + 1)) * 4;
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(evict_kernel), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.c.kv_heads * C, p.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = C;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_kernel, p, static_cast<int>(slots));
}

}  // namespace

cudaError_t launch_paged_evict(const EvictParams& p, int sms, cudaStream_t st) {
  EvictParams q = p;
  const bool over = p.new_lens < p.lens + p.rows && p.lens < p.new_lens + p.rows;
  if (over) q.new_lens = nullptr;
  const cudaError_t e = launch_select(q, sms, st);
  if (e != cudaSuccess || !over) return e;
  return launch_kernel(lens_kernel, dim3((p.rows + 255) / 256), dim3(256), 0, st, p, p.new_lens);
}

}  // namespace mxmoe
