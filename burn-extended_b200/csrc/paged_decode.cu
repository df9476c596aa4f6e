// paged_decode.cu -- attention of one new token per row over a paged cache.
//
// For row r, query head h and its key head g, over the keys n in
// [max(0, len - window), len):
//   s_n = scale q . k_n + bias_n,   m = max(s_n, sink_h, [quiet] 0)
//   L = sum_n e^(s_n - m) + e^(sink_h - m) + [quiet] e^(-m)
//   o = sum_n e^(s_n - m) v_n / L
// A row without keys, or whose scores are all -inf, gives zeros.  With track
// the shares e^(s_n - m) / L of the heads that read key head g are added to the
// weight of slot n.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {
namespace {

__device__ __forceinline__ float ld_any(const void* p, int dtype, int64_t i) {
  if (dtype == MXMOE_F32) return static_cast<const float*>(p)[i];
  if (dtype == MXMOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  __nv_fp8_e4m3 x;
  x.__x = static_cast<const uint8_t*>(p)[i];
  return static_cast<float>(x);
}

constexpr int kThreads = 128;
constexpr int kMaxGroup = 1024;  // query heads, checked at creation

// One block per (key head, row); it takes the head's query heads in turn: a
// pass for the maximum and the sum, a thread per key, and a pass over tiles of
// keys for the output, a thread per column.
__global__ void __launch_bounds__(kThreads) decode_kernel(const DecodeParams p) {
  __shared__ float qs[256], ps[kThreads], red[kThreads];
  __shared__ int64_t at[kThreads];
  __shared__ float top[kMaxGroup], inv[kMaxGroup];
  const int kvh = blockIdx.x, row = blockIdx.y, hd = p.c.head_dim, tid = threadIdx.x;
  const int G = p.c.n_heads / p.c.kv_heads;
  int len = p.lens[row];
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  if (len < 0 || len > cap) {
    if (tid == 0) atomicOr(p.c.status, kPagedBadIndex);
    len = len < 0 ? 0 : static_cast<int>(cap);
  }
  const int lo = p.window && p.window < len ? len - p.window : 0;
  const float ks = p.scale * (p.c.k_scale ? p.c.k_scale[kvh] : 1.0f), vs = p.c.v_scale ? p.c.v_scale[kvh] : 1.0f;
  for (int g = 0; g < G; ++g) {
    const int h = kvh * G + g;
    __syncthreads();
    for (int i = tid; i < hd; i += kThreads) qs[i] = ld_any(p.q, p.q_dtype, row * p.q_row + h * p.q_head + i);
    __syncthreads();
    const float* bias = p.bias ? p.bias + row * p.bias_row + h * p.bias_head : nullptr;
    auto score = [&](int n, int64_t slot) {
      const int64_t base = (slot + static_cast<int64_t>(kvh) * p.c.page_size) * hd;
      float s = 0.0f;
      for (int i = 0; i < hd; ++i) s = fmaf(qs[i], ld_any(p.c.k, p.c.dtype, base + i), s);
      s *= ks;
      return bias && n < p.bias_len ? s + bias[n] : s;
    };
    float m = -INFINITY, l = 0.0f;
    bool nan = false;
    for (int n = lo + tid; n < len; n += kThreads) {
      const int64_t slot = slot_of(p.c, p.t, row, n);
      const float s = slot < 0 ? -INFINITY : score(n, slot);
      nan |= s != s;
      const float mn = fmaxf(m, s);
      if (s != -INFINITY) {
        l = l * (m == -INFINITY ? 0.0f : expf(m - mn)) + expf(s - mn);
        m = mn;
      }
    }
    red[tid] = nan ? NAN : m;
    __syncthreads();
    float M = p.sinks ? p.sinks[h] : -INFINITY;
    if (p.quiet) M = M != M ? M : fmaxf(M, 0.0f);
    for (int i = 0; i < kThreads; ++i) M = (M != M || red[i] != red[i]) ? NAN : fmaxf(M, red[i]);
    __syncthreads();
    red[tid] = m == -INFINITY ? 0.0f : l * expf(m - M);
    __syncthreads();
    float L = 0.0f;
    for (int i = 0; i < kThreads; ++i) L += red[i];
    if (p.sinks && M != -INFINITY) L += expf(p.sinks[h] - M);
    if (p.quiet) L += expf(-M);
    const bool none = M == -INFINITY;
    if (tid == 0) {
      top[g] = M;
      inv[g] = none ? 0.0f : 1.0f / L;
    }
    float acc[2] = {0.0f, 0.0f};
    for (int n0 = lo; n0 < len && !none; n0 += kThreads) {
      const int n = n0 + tid;
      __syncthreads();
      if (n < len) {
        const int64_t slot = slot_of(p.c, p.t, row, n);
        const float s = slot < 0 ? -INFINITY : score(n, slot), w = s == -INFINITY ? 0.0f : expf(s - M) / L;
        ps[tid] = w;
        at[tid] = slot;
      }
      __syncthreads();
      for (int j = 0; j < min(kThreads, len - n0); ++j) {
        if (at[j] < 0) continue;
        const int64_t base = (at[j] + static_cast<int64_t>(kvh) * p.c.page_size) * hd;
        for (int e = 0; e < 2; ++e)
          if (tid + e * kThreads < hd) acc[e] = fmaf(ps[j], ld_any(p.c.v, p.c.dtype, base + tid + e * kThreads), acc[e]);
      }
    }
    for (int e = 0; e < 2; ++e) {
      const int i = tid + e * kThreads;
      if (i >= hd) continue;
      const int64_t o = row * p.out_row + h * p.out_head + i;
      if (p.out_dtype == MXMOE_F32)
        static_cast<float*>(p.out)[o] = acc[e] * vs;
      else
        static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(acc[e] * vs);
    }
    if (p.lse && tid == 0) p.lse[static_cast<int64_t>(row) * p.c.n_heads + h] = none ? -INFINITY : M + logf(L);
  }
  if (!p.track) return;
  __syncthreads();
  for (int n = lo + tid; n < len; n += kThreads) {  // the heads' shares together, then one addition
    const int64_t slot = slot_of(p.c, p.t, row, n);
    if (slot < 0) continue;
    const int64_t base = (slot + static_cast<int64_t>(kvh) * p.c.page_size) * hd;
    float w = 0.0f;
    for (int g = 0; g < G; ++g) {
      const int h = kvh * G + g;
      float s = 0.0f;
      for (int i = 0; i < hd; ++i)
        s = fmaf(ld_any(p.q, p.q_dtype, row * p.q_row + h * p.q_head + i), ld_any(p.c.k, p.c.dtype, base + i), s);
      s *= ks;
      if (p.bias && n < p.bias_len) s += p.bias[row * p.bias_row + h * p.bias_head + n];
      if (s != -INFINITY) w += expf(s - top[g]) * inv[g];
    }
    p.c.weight[slot + static_cast<int64_t>(kvh) * p.c.page_size] += w;
  }
}

}  // namespace

cudaError_t launch_paged_decode(const DecodeParams& p, cudaStream_t st) {
  return launch_kernel(decode_kernel, dim3(p.c.kv_heads, p.rows), dim3(kThreads), 0, st, p);
}

}  // namespace mxmoe
