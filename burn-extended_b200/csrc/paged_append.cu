// paged_append.cu -- rotary positions on new queries and keys, and the write
// of keys and values into the pages of their sequences.
//
// With c, s = cos, sin of (position x frequency i) from the table, i < rot / 2:
//   a' = a c - b s,   b' = b c + a s
// over the pairs (x_i, x_{i + rot/2}) (half layout) or (x_{2i}, x_{2i+1})
// (interleaved); columns from rot on pass through.  The map is linear and its
// transpose is the same with -s, so the inverse rotation (sign = -1) is also
// the gradient towards the input.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {
namespace {

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float x) { *p = x; }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One value into the cache's element type.  8 bits hold x / scale, rounded to
// nearest and held at +-448.
__device__ __forceinline__ void st_cache(void* pool, int dtype, int64_t i, float x, float inv_scale) {
  if (dtype == MXMOE_F32)
    static_cast<float*>(pool)[i] = x;
  else if (dtype == MXMOE_BF16)
    static_cast<__nv_bfloat16*>(pool)[i] = __float2bfloat16_rn(x);
  else
    static_cast<uint8_t*>(pool)[i] = __nv_cvt_float_to_fp8(x * inv_scale, __NV_SATFINITE, __NV_E4M3);
}

// One block per token: the pairs of every query and key head, the columns
// that pass, then the value rows.
template <typename T>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  const int t = blockIdx.x, hd = p.c.head_dim, half = p.rot / 2;
  const int nH = p.q ? p.c.n_heads : 0, H = p.k ? p.c.kv_heads : 0;
  const int index = p.index ? p.index[t] : -1;
  int pos = p.positions ? p.positions[t] : (index > 0 ? index : 0);
  if (p.rot && (pos < 0 || pos >= p.n_positions)) {
    if (threadIdx.x == 0 && p.c.status) atomicOr(p.c.status, kPagedBadPosition);
    pos = 0;
  }
  int64_t slot = -1;
  if (H && index >= 0) {
    const int row = p.rows ? p.rows[t] : t;
    if (row < 0 || row >= p.t.n_rows)
      atomicOr(p.c.status, kPagedBadIndex);
    else
      slot = slot_of(p.c, p.t, row, index);
  }
  const float* cs = p.cos + static_cast<int64_t>(pos) * half;  // unread without a rotation
  const float* sn = p.sin + static_cast<int64_t>(pos) * half;
  const int per = hd - half;  // pairs, then the columns that pass
  for (int i = threadIdx.x; i < (nH + H) * per; i += blockDim.x) {
    const int h = i / per, j = i - h * per;
    const bool isq = h < nH;
    const int kh = h - nH;
    const T* x = isq ? static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head
                     : static_cast<const T*>(p.k) + t * p.k_token + kh * p.k_head;
    T* y = isq ? static_cast<T*>(p.q_out) + t * p.qo_token + h * p.qo_head
               : (p.k_out ? static_cast<T*>(p.k_out) + t * p.ko_token + kh * p.ko_head : nullptr);
    const int64_t kbase = isq || slot < 0 ? -1 : (slot + static_cast<int64_t>(kh) * p.c.page_size) * hd;
    const float inv = !isq && p.c.k_scale ? 1.0f / p.c.k_scale[kh] : 1.0f;
    const int ca = j < half ? (p.interleaved ? 2 * j : j) : half + j;
    const int cb = p.interleaved ? ca + 1 : ca + half;
    const float a = ld1(x + ca);
    if (j < half) {
      const float b = ld1(x + cb), c = cs[j], s = p.sign * sn[j];
      const float u = a * c - b * s, w = b * c + a * s;
      if (y) {
        st1(y + ca, u);
        st1(y + cb, w);
      }
      if (kbase >= 0) {
        st_cache(p.c.k, p.c.dtype, kbase + ca, u, inv);
        st_cache(p.c.k, p.c.dtype, kbase + cb, w, inv);
      }
    } else {
      if (y) st1(y + ca, a);
      if (kbase >= 0) st_cache(p.c.k, p.c.dtype, kbase + ca, a, inv);
    }
  }
  if (slot < 0) return;
  for (int i = threadIdx.x; i < H * hd; i += blockDim.x) {
    const int h = i / hd, j = i - h * hd;
    const float inv = p.c.v_scale ? 1.0f / p.c.v_scale[h] : 1.0f;
    st_cache(p.c.v, p.c.dtype, (slot + static_cast<int64_t>(h) * p.c.page_size) * hd + j,
             ld1(static_cast<const T*>(p.v) + t * p.v_token + h * p.v_head + j), inv);
  }
  for (int h = threadIdx.x; h < H; h += blockDim.x) {
    const int64_t at = slot + static_cast<int64_t>(h) * p.c.page_size;
    if (p.c.weight) p.c.weight[at] = 0.0f;
    if (p.c.position) p.c.position[at] = pos;
  }
}

// cos and sin of position x frequency, the product and its cosine in 64 bits:
// at position 131072 a 32-bit product is off by up to 0.004 radians.
__global__ void rotary_table_kernel(const double* __restrict__ inv_freq, int half, int64_t first, int n, double factor,
                                    float* __restrict__ cs, float* __restrict__ sn) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= static_cast<int64_t>(n) * half) return;
  const int64_t pos = first + i / half;
  double s, c;
  sincos(static_cast<double>(pos) * inv_freq[i % half], &s, &c);
  cs[i] = static_cast<float>(c * factor);
  sn[i] = static_cast<float>(s * factor);
}

}  // namespace

cudaError_t launch_paged_append(const AppendParams& p, cudaStream_t st) {
  if (p.dtype == MXMOE_BF16) return launch_kernel(append_kernel<__nv_bfloat16>, dim3(p.tokens), dim3(256), 0, st, p);
  return launch_kernel(append_kernel<float>, dim3(p.tokens), dim3(256), 0, st, p);
}

cudaError_t launch_rotary_table(const double* inv_freq, int half, int64_t first, int n, double factor, float* cos,
                                float* sin, cudaStream_t st) {
  const int64_t total = static_cast<int64_t>(n) * half;
  return launch_kernel(rotary_table_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, st, inv_freq,
                       half, first, n, factor, cos, sin);
}

}  // namespace mxmoe
