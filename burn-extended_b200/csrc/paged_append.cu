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

#include <algorithm>

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
// nearest and held at +-448: the quotient itself, as x times the rounded 1 /
// scale goes to the other neighbour near a tie.
__device__ __forceinline__ void st_cache(void* pool, int dtype, int64_t i, float x, float scale) {
  if (dtype == MXMOE_F32)
    static_cast<float*>(pool)[i] = x;
  else if (dtype == MXMOE_BF16)
    static_cast<__nv_bfloat16*>(pool)[i] = __float2bfloat16_rn(x);
  else
    static_cast<uint8_t*>(pool)[i] = __nv_cvt_float_to_fp8(x / scale, __NV_SATFINITE, __NV_E4M3);
}

// Where a token goes, and how far it turns.
struct Token {
  int64_t slot;  // its cache slot of head 0, -1: not written
  int pos;
  const float *cs, *sn;  // its row of the table
};

// A position outside the table: the outputs turn as position 0, nothing enters
// the cache.
__device__ __forceinline__ Token token_of(const AppendParams& p, int t) {
  const int index = p.index ? __ldg(p.index + t) : -1, half = p.rot / 2;
  Token k{-1, p.positions ? __ldg(p.positions + t) : (index > 0 ? index : 0), nullptr, nullptr};
  const bool on_table = !p.rot || (k.pos >= 0 && k.pos < p.n_positions);
  if (!on_table && p.c.status) atomicOr(p.c.status, kPagedBadPosition);
  const int64_t from = on_table ? static_cast<int64_t>(k.pos) * half : 0;  // unread without a rotation
  k.cs = p.cos + from;
  k.sn = p.sin + from;
  if (p.k && index >= 0) {  // looked up while the position comes
    const int row = p.rows ? __ldg(p.rows + t) : t;
    if (row < 0 || row >= p.t.n_rows)
      atomicOr(p.c.status, kPagedBadIndex);
    else
      k.slot = slot_of(p.c, p.t, row, index);
  }
  if (!on_table) k.slot = -1;
  return k;
}

__device__ __forceinline__ void mark_slot(const AppendParams& p, const Token& k) {
  if (k.slot < 0 || !(p.c.weight || p.c.position)) return;
  for (int h = threadIdx.x; h < p.c.kv_heads; h += blockDim.x) {
    const int64_t at = k.slot + static_cast<int64_t>(h) * p.c.page_size;
    if (p.c.weight) p.c.weight[at] = 0.0f;
    if (p.c.position) p.c.position[at] = k.pos;
  }
}

// 16 bytes of activations as floats.
template <typename T>
struct Piece;
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int kN = 8;
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void open(float (&x)[8]) const {
    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Piece<float> {
  static constexpr int kN = 4;
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void open(float (&x)[4]) const { x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; }
};

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int N>
__device__ __forceinline__ void store(float* p, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int N>
__device__ __forceinline__ void store(__nv_bfloat16* p, const float (&x)[N]) {
  if (N == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4 % N], x[5 % N]),
                                              bf16_pair(x[6 % N], x[7 % N]));
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]));
}
template <int N>
__device__ __forceinline__ void store_cache(void* pool, int dtype, int64_t at, const float (&x)[N], float scale) {
  if (dtype == MXMOE_F32) {
    store(static_cast<float*>(pool) + at, x);
  } else if (dtype == MXMOE_BF16) {
    store(static_cast<__nv_bfloat16*>(pool) + at, x);
  } else {
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] / scale, x[4 * i + 1] / scale), __NV_SATFINITE, __NV_E4M3);
      const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] / scale, x[4 * i + 3] / scale), __NV_SATFINITE, __NV_E4M3);
      w[i] = a | b << 16;
    }
    uint8_t* d = static_cast<uint8_t*>(pool) + at;
    if (N == 8)
      *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[N / 4 - 1]);
    else
      *reinterpret_cast<uint32_t*>(d) = w[0];
  }
}

// A unit of a head: one piece, or the two that turn together.
template <typename T, bool kInterleaved>
struct Unit {
  static constexpr int N = Piece<T>::kN;
  Piece<T> a, b;

  __device__ __forceinline__ void load(const T* x, int apart, bool two) {
    a.load(x);
    if (two) b.load(x + apart);
  }
  __device__ __forceinline__ void turn(const float (&c)[N], const float (&s)[N], bool turns, bool two, float (&x)[N],
                                       float (&y)[N]) const {
    a.open(x);
    if (two) {
      b.open(y);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float u = x[j], w = y[j];
        x[j] = u * c[j] - w * s[j];
        y[j] = w * c[j] + u * s[j];
      }
    } else if (kInterleaved && turns) {
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float u = x[j], w = x[j + 1];
        x[j] = u * c[j / 2] - w * s[j / 2];
        x[j + 1] = w * c[j / 2] + u * s[j / 2];
      }
    }
  }
};

// Everything moves in 16-byte pieces, each read and written once: bound by
// memory, and by latency where tokens are few.  A thread keeps one unit of
// columns for every `per_pass`-th query head, so the token's cosines are read
// once per thread; then the keys' units and the values' pieces are shared out
// over the block.  The loads of up to kBatch query heads, a key unit and a value
// piece are in flight while the token's place and cosines come.
constexpr int kBatch = 2;
constexpr int kAtOnce = 16;     // tokens whose places a block of many looks up together
constexpr int kManyBlocks = 5;  // such blocks on one SM
// Token t; place_of() is its Token, asked for once the loads are on their way.
template <typename T, bool kInterleaved, class PlaceOf>
__device__ __forceinline__ void append_token(const AppendParams& p, int units, int per_pass, int t, PlaceOf place_of) {
  constexpr int N = Piece<T>::kN;
  const int hd = p.c.head_dim, half = p.rot / 2, nt = blockDim.x, tid = threadIdx.x;
  const int nH = p.q ? p.c.n_heads : 0, H = p.k ? p.c.kv_heads : 0;
  const int first = tid / units, unit = tid - first * units;
  const bool turns = unit * N < (kInterleaved ? p.rot : half), two = !kInterleaved && turns;
  const int ca = kInterleaved || turns ? unit * N : half + unit * N;
  const int64_t q_step = per_pass * p.q_head, qo_step = per_pass * p.qo_head;
  const int mine = first < per_pass && first < nH ? (nH - first + per_pass - 1) / per_pass : 0;  // query heads of this thread
  // Keys: unit e % units of head e / units; a thread's columns are the same as
  // for the queries where per_pass heads fill the block, so that the first
  // round takes the cosines that it has.
  const int v_pieces = hd / N, v_all = H * v_pieces;
  const bool has_key = first < per_pass && first < H;
  const int v0 = nt - 1 - tid;  // from the block's other end, where no keys are
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + first * p.q_head + ca;
  T* q_out = static_cast<T*>(p.q_out) + t * p.qo_token + first * p.qo_head + ca;
  Unit<T, kInterleaved> u[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (i < mine) u[i].load(q + i * q_step, half, two);
  Unit<T, kInterleaved> ku;
  if (has_key) ku.load(static_cast<const T*>(p.k) + t * p.k_token + first * p.k_head + ca, half, two);
  auto value_at = [&](int i) {
    const int h = i / v_pieces;
    return static_cast<const T*>(p.v) + t * p.v_token + h * p.v_head + (i - h * v_pieces) * N;
  };
  Piece<T> v;
  if (v0 < v_all) v.load(value_at(v0));
  const Token k = place_of();
  __align__(16) float c[N];  // interleaved: the first half of them
  __align__(16) float s[N];
  if (turns && (mine > 0 || has_key)) {
    const int from = kInterleaved ? unit * N / 2 : unit * N;
    constexpr int kCos = kInterleaved ? N / 2 : N, kStep = kCos % 4 ? 2 : 4;
#pragma unroll
    for (int i = 0; i < kCos; i += kStep) {
      if (kStep == 4) {
        *reinterpret_cast<float4*>(c + i) = __ldg(reinterpret_cast<const float4*>(k.cs + from + i));
        *reinterpret_cast<float4*>(s + i) = __ldg(reinterpret_cast<const float4*>(k.sn + from + i));
      } else {
        *reinterpret_cast<float2*>(c + i) = __ldg(reinterpret_cast<const float2*>(k.cs + from + i));
        *reinterpret_cast<float2*>(s + i) = __ldg(reinterpret_cast<const float2*>(k.sn + from + i));
      }
    }
#pragma unroll
    for (int i = 0; i < kCos; ++i) s[i] *= p.sign;
  }
  float x[N], y[N];
#pragma unroll 1
  for (int i0 = 0; i0 < mine; i0 += kBatch) {
    if (i0 > 0) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (i0 + i < mine) u[i].load(q + i * q_step, half, two);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= mine) break;
      u[i].turn(c, s, turns, two, x, y);
      store(q_out + i * qo_step, x);
      if (two) store(q_out + i * qo_step + half, y);
    }
    q += kBatch * q_step;
    q_out += kBatch * qo_step;
  }
  if (first < per_pass) {
#pragma unroll 1
    for (int h = first; h < H; h += per_pass) {
      if (h != first) ku.load(static_cast<const T*>(p.k) + t * p.k_token + h * p.k_head + ca, half, two);
      ku.turn(c, s, turns, two, x, y);
      if (p.k_out) {
        T* out = static_cast<T*>(p.k_out) + t * p.ko_token + h * p.ko_head + ca;
        store(out, x);
        if (two) store(out + half, y);
      }
      if (k.slot >= 0) {
        const int64_t at = (k.slot + static_cast<int64_t>(h) * p.c.page_size) * hd + ca;
        const float scale = p.c.k_scale ? __ldg(p.c.k_scale + h) : 1.0f;
        store_cache(p.c.k, p.c.dtype, at, x, scale);
        if (two) store_cache(p.c.k, p.c.dtype, at + half, y, scale);
      }
    }
  }
  if (k.slot >= 0) {
#pragma unroll 1
    for (int i = v0; i < v_all; i += nt) {
      if (i != v0) v.load(value_at(i));
      const int h = i / v_pieces;
      v.open(x);
      store_cache(p.c.v, p.c.dtype, (k.slot + static_cast<int64_t>(h) * p.c.page_size) * hd + (i - h * v_pieces) * N, x,
                  p.c.v_scale ? __ldg(p.c.v_scale + h) : 1.0f);
    }
  }
  mark_slot(p, k);
}

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(512, 1) append_wide_kernel(const AppendParams p, int units, int per_pass) {
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x;
  append_token<T, kInterleaved>(p, units, per_pass, t, [&]() { return token_of(p, t); });
}

// Many tokens: a block goes from one to the next, and looks the places of its
// next kAtOnce up together, so that index, page table and position cost their
// latency once for all of them.  8192 tokens of 64 + 8 heads of 64 in bf16: 32.3
// us, 5.3 TB/s; 44.1 us with a block per token.  Five blocks an SM leave enough
// registers for the pieces in flight; with four 34.6 us, six 36.1, seven 36.2,
// and with three query heads in flight 34.4.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(128, kManyBlocks) append_many_kernel(const AppendParams p, int units, int per_pass) {
  __shared__ Token places[kAtOnce];
  griddep_wait();
  griddep_launch_dependents();
  int turn = 0;
#pragma unroll 1
  for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    append_token<T, kInterleaved>(p, units, per_pass, t, [&]() {
      if (turn == 0) {
        __syncthreads();  // the places before are used up
        const int64_t mine = t + threadIdx.x * static_cast<int64_t>(gridDim.x);
        if (threadIdx.x < kAtOnce && mine < p.tokens) places[threadIdx.x] = token_of(p, static_cast<int>(mine));
        __syncthreads();
      }
      return places[turn];
    });
    if (++turn == kAtOnce) turn = 0;
  }
}

// Any layout, stride and alignment, one pair or column per thread.  One block
// per token.
template <typename T>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x, hd = p.c.head_dim, half = p.rot / 2;
  const int nH = p.q ? p.c.n_heads : 0, H = p.k ? p.c.kv_heads : 0;
  const Token k = token_of(p, t);
  const int per = hd - half;  // pairs, then the columns that pass
  for (int i = threadIdx.x; i < (nH + H) * per; i += blockDim.x) {
    const int h = i / per, j = i - h * per;
    const bool isq = h < nH;
    const int kh = h - nH;
    const T* x = isq ? static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head
                     : static_cast<const T*>(p.k) + t * p.k_token + kh * p.k_head;
    T* y = isq ? static_cast<T*>(p.q_out) + t * p.qo_token + h * p.qo_head
               : (p.k_out ? static_cast<T*>(p.k_out) + t * p.ko_token + kh * p.ko_head : nullptr);
    const int64_t kbase = isq || k.slot < 0 ? -1 : (k.slot + static_cast<int64_t>(kh) * p.c.page_size) * hd;
    const float scale = !isq && p.c.k_scale ? p.c.k_scale[kh] : 1.0f;
    const int ca = j < half ? (p.interleaved ? 2 * j : j) : half + j;
    const int cb = p.interleaved ? ca + 1 : ca + half;
    const float a = ld1(x + ca);
    if (j < half) {
      const float b = ld1(x + cb), c = k.cs[j], s = p.sign * k.sn[j];
      const float u = a * c - b * s, w = b * c + a * s;
      if (y) {
        st1(y + ca, u);
        st1(y + cb, w);
      }
      if (kbase >= 0) {
        st_cache(p.c.k, p.c.dtype, kbase + ca, u, scale);
        st_cache(p.c.k, p.c.dtype, kbase + cb, w, scale);
      }
    } else {
      if (y) st1(y + ca, a);
      if (kbase >= 0) st_cache(p.c.k, p.c.dtype, kbase + ca, a, scale);
    }
  }
  if (k.slot >= 0) {
    for (int i = threadIdx.x; i < H * hd; i += blockDim.x) {
      const int h = i / hd, j = i - h * hd;
      const float scale = p.c.v_scale ? p.c.v_scale[h] : 1.0f;
      st_cache(p.c.v, p.c.dtype, (k.slot + static_cast<int64_t>(h) * p.c.page_size) * hd + j,
               ld1(static_cast<const T*>(p.v) + t * p.v_token + h * p.v_head + j), scale);
    }
  }
  mark_slot(p, k);
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

bool wide(const void* p, int64_t a, int64_t b, int n, size_t elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a * elem) % 16 == 0 && (b * elem) % 16 == 0 && n * elem % 16 == 0;
}

template <typename T>
cudaError_t launch_append(const AppendParams& p, int sms, cudaStream_t st) {
  constexpr int N = Piece<T>::kN;
  const int hd = p.c.head_dim, half = p.rot / 2;
  const bool aligned = wide(p.q, p.q_token, p.q_head, hd, sizeof(T)) && wide(p.k, p.k_token, p.k_head, hd, sizeof(T)) &&
                       wide(p.v, p.v_token, p.v_head, hd, sizeof(T)) && wide(p.q_out, p.qo_token, p.qo_head, hd, sizeof(T)) &&
                       wide(p.k_out, p.ko_token, p.ko_head, hd, sizeof(T)) && (p.interleaved ? p.rot : half) % N == 0;
  const int units = (hd - (p.interleaved ? 0 : half)) / N;
  if (!aligned || units > 512) return launch_kernel(append_kernel<T>, dim3(p.tokens), dim3(256), 0, st, p);
  // Threads of a token: enough of them to fill the SMs (2048 a SM), up to a
  // thread per unit for the shortest chain.  1023 tokens of 32 + 8 heads of 128 in
  // 32 bits into 8: 12.9 us with 256 threads, 14.5 with 224, 16.3 with 128.
  const int heads = p.q ? p.c.n_heads : p.c.kv_heads;
  const int want = std::max(units, std::min(512, std::max(128, sms * 2048 / p.tokens / 32 * 32)));
  const int passes = (heads * units + want - 1) / want, per_pass = std::min(want / units, (heads + passes - 1) / passes);
  const int threads = (per_pass * units + 31) / 32 * 32;
  if (threads > 128)
    return launch_kernel(p.interleaved ? append_wide_kernel<T, true> : append_wide_kernel<T, false>, dim3(p.tokens), dim3(threads), 0, st,
                         p, units, per_pass);
  return launch_kernel(p.interleaved ? append_many_kernel<T, true> : append_many_kernel<T, false>,
                       dim3(std::min(p.tokens, kManyBlocks * sms)), dim3(threads), 0, st, p, units, per_pass);
}

}  // namespace

cudaError_t launch_paged_append(const AppendParams& p, int sms, cudaStream_t st) {
  return p.dtype == MXMOE_BF16 ? launch_append<__nv_bfloat16>(p, sms, st) : launch_append<float>(p, sms, st);
}

cudaError_t launch_rotary_table(const double* inv_freq, int half, int64_t first, int n, double factor, float* cos,
                                float* sin, cudaStream_t st) {
  const int64_t total = static_cast<int64_t>(n) * half;
  return launch_kernel(rotary_table_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, st, inv_freq,
                       half, first, n, factor, cos, sin);
}

}  // namespace mxmoe
