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
#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {
namespace {

constexpr int kThreads = 1024;

// The order of the victims as one unsigned number: it rises with the weight, a
// NaN is +inf, the protected come last.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sink, int first_recent) {
  if (pos < sink || pos >= first_recent) return 0xFFFFFFFFu;
  if (w != w) return 0xFF800000u;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the block of a 0 / 1 flag; `total` gets the sum.
__device__ __forceinline__ int block_rank(bool flag, int* warp_sums, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned b = __ballot_sync(0xFFFFFFFFu, flag);
  if (lane == 0) warp_sums[warp] = __popc(b);
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < kThreads / 32; ++i) {
    const int s = warp_sums[i];
    if (i < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + __popc(b & ((1u << lane) - 1));
}

// One block per (key head, row): a radix selection of the last victim's key,
// then one walk over the slots below the budget and one over those above it,
// which hand each other holes and movers through shared memory.
__global__ void __launch_bounds__(kThreads) evict_kernel(const EvictParams p) {
  __shared__ int hist[256], sums[kThreads / 32], pick[2];
  __shared__ int64_t holes[kThreads], movers[kThreads];
  const int h = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int len = p.lens[row];
  if (len < 0 || len > cap) {
    if (tid == 0) atomicOr(p.c.status, kPagedBadIndex);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  if (h == 0 && tid == 0) p.new_lens[row] = min(len, p.budget);
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
    for (int n = tid; n < len; n += kThreads) {
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
  for (int n0 = 0; n0 < p.budget; n0 += kThreads) {
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
      lo += kThreads;
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
      hi += kThreads;
    }
    __syncthreads();
    const int m = min(n_holes, n_movers);
    if (m == 0) break;
    for (int i = tid; i < m * words; i += kThreads) {
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

}  // namespace

cudaError_t launch_paged_evict(const EvictParams& p, cudaStream_t st) {
  return launch_kernel(evict_kernel, dim3(p.c.kv_heads, p.rows), dim3(kThreads), 0, st, p);
}

}  // namespace mxmoe
