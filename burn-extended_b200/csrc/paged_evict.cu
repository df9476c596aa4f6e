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

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBins = 2 * kThreads;  // 11 bits a pass: the key's 32 in three
constexpr int kFew = 256;            // candidates that are ranked one against another
constexpr int kMaxCluster = 8;

// A list's pairs, in 16-byte pieces of keys and values, several of a thread in
// flight: sources and destinations are never the same slots.
__device__ __forceinline__ void move_pairs(const EvictParams& p, const int* to, const int* by, int pairs) {
  constexpr int kAtOnce = 4;
  const int pieces = p.c.head_dim * (p.c.dtype == MXMOE_F32 ? 4 : p.c.dtype == MXMOE_BF16 ? 2 : 1) / 16;
  uint4 *k = static_cast<uint4*>(p.c.k), *v = static_cast<uint4*>(p.c.v);
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < pairs * pieces; i0 += kAtOnce * kThreads) {
    uint4 a[kAtOnce], b[kAtOnce];
    int64_t dst[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + j * kThreads, e = i / pieces, c = i - e * pieces;
      dst[j] = -1;
      if (i >= pairs * pieces || to[e] < 0 || by[e] < 0) continue;
      dst[j] = static_cast<int64_t>(to[e]) * pieces + c;
      const int64_t src = static_cast<int64_t>(by[e]) * pieces + c;
      a[j] = k[src];
      b[j] = v[src];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (dst[j] < 0) continue;
      k[dst[j]] = a[j];
      v[dst[j]] = b[j];
    }
  }
#pragma unroll 1
  for (int e = threadIdx.x; e < pairs; e += kThreads) {
    if (to[e] < 0 || by[e] < 0) continue;
    p.c.weight[to[e]] = p.c.weight[by[e]];
    p.c.position[to[e]] = p.c.position[by[e]];
  }
}

// One to a bin for every lane that calls: those of the first lane's bin are
// added together, as weights may all be alike, the others one by one.
__device__ __forceinline__ void count_bin(int* hist, uint32_t bin) {
  const uint32_t active = __activemask(), first = __ffs(active) - 1;
  const uint32_t same = __ballot_sync(active, bin == __shfl_sync(active, bin, first));
  if (!(same >> (threadIdx.x & 31) & 1))
    atomicAdd(hist + bin, 1);
  else if ((threadIdx.x & 31) == first)
    atomicAdd(hist + bin, __popc(same));
}

// The sums of the warps before this one and of all, of two counts.
__device__ __forceinline__ void over_warps(int2 x, int2* sums, int2& before, int2& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sums[warp] = x;
  __syncthreads();
  int2 y = sums[lane];  // one for each of the 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xFFFFFFFFu, y.x, o), b = __shfl_up_sync(0xFFFFFFFFu, y.y, o);
    if (lane >= o) {
      y.x += a;
      y.y += b;
    }
  }
  all = make_int2(__shfl_sync(0xFFFFFFFFu, y.x, 31), __shfl_sync(0xFFFFFFFFu, y.y, 31));
  const int from = warp == 0 ? 0 : warp - 1;
  before = make_int2(__shfl_sync(0xFFFFFFFFu, y.x, from), __shfl_sync(0xFFFFFFFFu, y.y, from));
  if (warp == 0) before = make_int2(0, 0);
  __syncthreads();
}

// One cluster per (key head, row).  Each block keeps the keys of its share of
// the slots in shared memory, so weights and positions are read once.  The
// last victim is found as a (key, index): passes over 11 bits of the key, their
// histograms summed over the cluster, until at most kFew candidates share its
// prefix, which are then ranked one against another.  Each warp numbers the
// holes and movers of a stretch of slots by ballots; every hole and mover is
// written to the list of the block that will move it, and the blocks move their
// pairs in 16-byte pieces.  Bound by the latency of these steps where few
// tokens move (one of 2049, 8 key heads: 7.5 us, the launch alone 2.5), else by
// the selection's instructions first (some 400 warp instructions to 32 keys,
// issued 46% of the time) and then by the moves.  The first eviction of 16 rows
// of 1000 to 8192 tokens to 2048, 8 key heads of 64 in bf16, reads and writes 70
// MB in 32 us, 2.2 TB/s; of 2 rows of 60001 and 65536 to 16384, 8-bit heads of
// 128, 112 MB in 50 us on 96 SMs, 2.2 TB/s.  The same calls again, on caches
// where the survivors behind the budget are copies and only 18 and 17 MB move,
// take 17 and 30 us.
__global__ void __launch_bounds__(kThreads, 1) evict_kernel(const EvictParams p, int slots, int four) {
  extern __shared__ __align__(16) uint32_t keys[];  // [slots]; then to[slots / 2 + 1], by[slots / 2 + 1]
  __shared__ __align__(16) int hist[3][kBins];
  __shared__ uint2 few[kFew];  // of block 0: the candidates' keys and indexes
  __shared__ int2 sums[kWarps], count[2];
  __shared__ int pick[3], n_few;
  __shared__ uint2 last;  // of block 0: the last victim
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int h = blockIdx.x / C, row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto sync = [&]() {
    if (C == 1)
      __syncthreads();
    else
      cluster.sync();
  };
  griddep_wait();
  griddep_launch_dependents();
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int len = p.lens[row];
  for (int i = tid; i < 3 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
  if (tid == 0) n_few = 0;
  if (len < 0 || len > cap) {
    if (tid == 0) atomicOr(p.c.status, kPagedBadIndex);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  if (h == 0 && rank == 0 && tid == 0 && p.new_lens) p.new_lens[row] = min(len, p.budget);
  if (len <= p.budget) return;
  const int first_recent = p.seen[row] - p.recent;
  __syncthreads();

  const int share = ((len + C - 1) / C + 3) / 4 * 4, n0 = min(len, rank * share), mine = min(share, len - n0);
  int bad = 0;
  auto slot_at = [&](int n) {
    const int64_t s = slot_of(p.c, p.t, row, n, bad);
    return s < 0 ? -1 : static_cast<int>(s) + h * p.c.page_size;
  };
  if (four) {
    // four slots of one page at a time: page_size and n0 are multiples of four
    constexpr int kAtOnce = 4;
#pragma unroll 1
    for (int i0 = 4 * tid; i0 < mine; i0 += 4 * kAtOnce * kThreads) {
      int at[kAtOnce];
      float4 w[kAtOnce];
      int4 q[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) at[j] = i0 + 4 * j * kThreads < mine ? slot_at(n0 + i0 + 4 * j * kThreads) : -1;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (at[j] < 0) continue;
        w[j] = *reinterpret_cast<const float4*>(p.c.weight + at[j]);
        q[j] = *reinterpret_cast<const int4*>(p.c.position + at[j]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int i = i0 + 4 * j * kThreads;
        if (i >= mine) break;
        uint4 k = make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
        if (at[j] >= 0)
          k = make_uint4(evict_key(w[j].x, q[j].x, p.sink, first_recent), evict_key(w[j].y, q[j].y, p.sink, first_recent),
                         evict_key(w[j].z, q[j].z, p.sink, first_recent), evict_key(w[j].w, q[j].w, p.sink, first_recent));
        *reinterpret_cast<uint4*>(keys + i) = k;  // `slots` is a multiple of four
      }
    }
    __syncthreads();
  } else {
    constexpr int kAtOnce = 8;  // slots of a thread whose loads are in flight together
#pragma unroll 1
    for (int i0 = tid; i0 < mine; i0 += kAtOnce * kThreads) {
      int at[kAtOnce], position[kAtOnce];
      float weight[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) at[j] = i0 + j * kThreads < mine ? slot_at(n0 + i0 + j * kThreads) : -1;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        weight[j] = at[j] < 0 ? 0.0f : p.c.weight[at[j]];
        position[j] = at[j] < 0 ? 0 : p.c.position[at[j]];
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (i0 + j * kThreads < mine)
          keys[i0 + j * kThreads] = at[j] < 0 ? 0xFFFFFFFFu : evict_key(weight[j], position[j], p.sink, first_recent);
    }
  }
  if (bad) atomicOr(p.c.status, bad);
  int need = len - p.budget, candidates = len;  // victims among the keys that share the prefix
  uint32_t prefix = 0;
  int above = 32;  // the prefix's lowest bit
#pragma unroll 1
  for (int pass = 0; pass < 3 && (pass == 0 || candidates > kFew); ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
#pragma unroll 2
    for (int i = tid; i < mine; i += kThreads) {
      const uint32_t k = keys[i];
      if (pass == 0 || k >> above == prefix >> above) count_bin(hist[pass], (k >> shift) & (kBins - 1));
    }
    sync();
    int2 bin = make_int2(0, 0);
    for (int c = 0; c < C; ++c) {
      const int2 x = *reinterpret_cast<const int2*>(cluster.map_shared_rank(&hist[pass][0], c) + 2 * tid);
      bin.x += x.x;
      bin.y += x.y;
    }
    int upto = bin.x + bin.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += a;
    }
    int2 before, all;
    over_warps(make_int2(__shfl_sync(0xFFFFFFFFu, upto, 31), 0), sums, before, all);
    const int low = before.x + upto - bin.x - bin.y;  // keys below this thread's bins
    if (need > low && need <= low + bin.x + bin.y) {
      const bool second = need > low + bin.x;
      pick[0] = 2 * tid + second;
      pick[1] = need - low - (second ? bin.x : 0);
      pick[2] = second ? bin.y : bin.x;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    need = pick[1];
    candidates = pick[2];
    above = shift;
  }

  // The last victim: candidate number `need` by (key, index).
  uint2 bound;
  const int seg = (mine + kThreads - 1) / kThreads * 32, s0 = min(mine, warp * seg), s1 = min(mine, s0 + seg);  // this warp's slots
  if (candidates <= kFew) {
    int* counter = cluster.map_shared_rank(&n_few, 0);
    uint2* list = cluster.map_shared_rank(few, 0);
    for (int i = tid; i < mine; i += kThreads)
      if (keys[i] >> above == prefix >> above) list[atomicAdd(counter, 1)] = make_uint2(keys[i], n0 + i);
    sync();
    if (rank == 0 && tid < candidates) {
      const uint2 me = few[tid];
      int less = 0;
      for (int i = 0; i < candidates; ++i) {
        const uint2 x = few[i];
        less += x.x < me.x || (x.x == me.x && x.y < me.y);
      }
      if (less == need - 1) last = me;
    }
    sync();
    bound = *cluster.map_shared_rank(&last, 0);
  } else {
    // whole keys, too many alike: the need-th of them in the order of the slots
    int ties = 0;
    for (int i = s0 + lane; i - lane < s1; i += 32) ties += __popc(__ballot_sync(0xFFFFFFFFu, i < s1 && keys[i] == prefix));
    int2 before, all;
    over_warps(make_int2(ties, 0), sums, before, all);
    if (tid == 0) count[0] = all;
    sync();
    int upto = before.x;
    for (int c = 0; c < rank; ++c) upto += cluster.map_shared_rank(&count[0], c)->x;
    if (upto < need && need <= upto + ties) {
      for (int i = s0 + lane; i - lane < s1; i += 32) {
        const uint32_t b = __ballot_sync(0xFFFFFFFFu, i < s1 && keys[i] == prefix);
        if ((b >> lane & 1) && upto + __popc(b & ((2u << lane) - 1)) == need)
          *cluster.map_shared_rank(&last, 0) = make_uint2(prefix, n0 + i);
        upto += __popc(b);
      }
    }
    sync();
    bound = *cluster.map_shared_rank(&last, 0);
  }

  auto victim = [&](int i) {
    const uint32_t k = keys[i];
    return k < bound.x || (k == bound.x && n0 + i <= static_cast<int>(bound.y));
  };
  int2 own = make_int2(0, 0), before, all;  // holes, movers of this warp's slots
  for (int i = s0 + lane; i - lane < s1; i += 32) {
    const bool in = i < s1, out = in && victim(i), low = n0 + i < p.budget;
    own.x += __popc(__ballot_sync(0xFFFFFFFFu, out && low));
    own.y += __popc(__ballot_sync(0xFFFFFFFFu, in && !out && !low));
  }
  over_warps(own, sums, before, all);
  int pairs = all.x;
  if (C > 1) {
    if (tid == 0) count[1] = all;
    cluster.sync();
    pairs = 0;
    for (int c = 0; c < C; ++c) {
      const int2 x = *cluster.map_shared_rank(&count[1], c);
      pairs += x.x;
      if (c < rank) {
        before.x += x.x;
        before.y += x.y;
      }
    }
  }
  const int per = max(1, (pairs + C - 1) / C), room = slots / 2 + 1;  // pairs of a block; holes <= len / 2, so per <= room
  int* to = reinterpret_cast<int*>(keys + slots);
  int* by = to + room;
  if (own.x + own.y > 0) {
#pragma unroll 4
    for (int i = s0 + lane; i - lane < s1; i += 32) {
      const bool in = i < s1, out = in && victim(i), low = n0 + i < p.budget;
      const uint32_t holes = __ballot_sync(0xFFFFFFFFu, out && low), movers = __ballot_sync(0xFFFFFFFFu, in && !out && !low);
      const int slot = in && out == low ? slot_at(n0 + i) : -1;
      if (in && out == low) {
        const int e = out ? before.x + __popc(holes & ((1u << lane) - 1)) : before.y + __popc(movers & ((1u << lane) - 1));
        const int c = C == 1 ? 0 : e / per;
        *cluster.map_shared_rank((out ? to : by) + (e - c * per), c) = slot;
      }
      before.x += __popc(holes);
      before.y += __popc(movers);
    }
  }
  sync();

  move_pairs(p, to, by, min(per, pairs - rank * per));
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

// For tables too wide for the kernel above (8 x 24K slots), whatever their rows
// hold.  Simple, and slow: one of 2049 tokens under 262144 slots takes 38 us, 7.5
// under a table of its size; 2 rows of 60001 and 65536 to 16384 770 us, 50 there.
// One block per (key head, row): a radix selection of the last victim's key, the
// keys read anew in each pass, then one walk over the slots below the budget and
// one over those above it, which hand each other holes and movers through shared
// memory.
__global__ void __launch_bounds__(kLongThreads) evict_long_kernel(const EvictParams p) {
  griddep_wait();
  griddep_launch_dependents();
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

// New lengths in the place of the old ones or of `seen`, once every block has
// read those.
__global__ void lens_kernel(const EvictParams p, int32_t* lens) {
  griddep_wait();
  griddep_launch_dependents();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.rows) return;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  const int64_t len = min(max(static_cast<int64_t>(p.lens[i]), static_cast<int64_t>(0)), cap);
  lens[i] = static_cast<int>(min(len, static_cast<int64_t>(p.budget)));
}

cudaError_t launch_select(const EvictParams& p, int sms, cudaStream_t st) {
  // Blocks of a (row, key head): as many as its keys and lists (8 bytes a slot)
  // need.  Rows of more than 8192 slots that leave SMs idle get up to kSpread, of
  // at least 4096 slots each.  One row of 8 heads, one token over the budget: 12000
  // slots 11.5 us with three blocks, 13.6 with one; 8000 slots 11.0 with one, 11.1
  // with two; 4500 slots 9.2 and 10.3, where a cluster's barriers cost more than
  // the shorter share saves.  First evictions of many, between two events, 5 us of
  // which are theirs: half of 12000 slots 29 and 47, of 8000 35 and 29, of 4500 27
  // and 25, so for those the limit could be lower; 2 rows of 65536 slots, 16
  // clusters, 56 with six blocks each, 66 with four, 98 with three, and with
  // eight, which do not all find room at once, 84; the 24 clusters of 3 rows do
  // not with six either: 104, with four 74.  All of this goes by the table's width,
  // as the lengths are not known here: under a table much wider than its rows a
  // call is slower (16 rows of up to 8192 tokens 32 us under a table of 8192
  // slots, 85 under one of 131072).
  constexpr int kSlots = 24 * 1024, kSpread = 6;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size, pairs = static_cast<int64_t>(p.rows) * p.c.kv_heads;
  const int64_t need = (cap + kSlots - 1) / kSlots;
  const int64_t spread = cap > 8192 ? std::min({(cap + 4095) / 4096, sms / pairs, static_cast<int64_t>(kSpread)}) : 1;
  const int C = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxCluster, std::max(need, spread))));
  const int64_t slots = ((cap + C - 1) / C + 3) / 4 * 4;
  if (slots > kSlots) {
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
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C == 1 ? 1 : 2;  // one block is a cluster by itself
  const int four = p.c.page_size % 4 == 0 && reinterpret_cast<uintptr_t>(p.c.weight) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.c.position) % 16 == 0;
  return cudaLaunchKernelEx(&cfg, evict_kernel, p, static_cast<int>(slots), four);
}

}  // namespace

cudaError_t launch_paged_evict(const EvictParams& p, int sms, cudaStream_t st) {
  EvictParams q = p;
  const bool over = !apart(p.new_lens, p.lens, p.rows) || !apart(p.new_lens, p.seen, p.rows);
  if (over) q.new_lens = nullptr;
  const cudaError_t e = launch_select(q, sms, st);
  if (e != cudaSuccess || !over) return e;
  return launch_kernel(lens_kernel, dim3((p.rows + 255) / 256), dim3(256), 0, st, p, p.new_lens);
}

}  // namespace mxmoe
