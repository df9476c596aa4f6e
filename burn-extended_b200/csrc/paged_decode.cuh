// paged_decode.cuh -- the attention kernel of paged_decode.cu, a template over
// the cache's element type.
//
// The keys of all (row, key head) pairs, cut into tiles of 16, form one list;
// its tiles are dealt out evenly in contiguous ranges, so a ragged batch loads
// every SM alike.  A worker is a group of warps; each warp streams its own
// tiles through its own shared-memory ring (cp.async, no block barrier) and
// keeps a running maximum, sum and output for 8 query heads in registers.  At
// the end of a (row, key head) the group joins its warps in shared memory; a
// pair that more than one worker holds goes through partial results in global
// memory, and the last worker to arrive joins them in the workers' order, so the
// result does not depend on timing.
//
// The products run on the warp MMA, m = 16: rows 0-7 hold the heads' queries
// (or shares) rounded to the operand type, rows 8-15 what the rounding left, so
// their sum is exact to 16 bits and more at no extra cost -- at 8 query heads
// per key head the tile would be half empty otherwise.  The kernel is bound by
// the bytes of K and V; a tensor-core tile of 128 rows would be 1/16 full.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {

constexpr int kDecodeMaxStages = 6;

// How one launch is laid out; set by decode_plan in paged_decode.cu.
struct DecodePlan {
  int warps, stages;
  int stage_bytes;  // K rows, then V rows; room for 8 x (head_dim + 8) floats
  int smem;         // of the block: the warps' rings, and 128 bytes that a read past the last row may touch
  int grid;
};

namespace decode {

// Bytes from one key to the next in a ring: an odd number of 16-byte pieces, so
// that 8 rows at one column lie in 8 different groups of banks.
constexpr int ring_row(int bytes) { return (bytes / 16 | 1) * 16; }

// Keys of a tile in 16s: two independent halves hide each other's latency where
// a row is short; longer rows have enough columns for that.
constexpr int tile_halves(int bytes) { return bytes <= 128 ? 2 : 1; }

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^(a - b) for a <= b, 0 where a is -inf; the difference first, so that two
// scores near the type's lowest value stay apart from -inf.
__device__ __forceinline__ float exp_diff(float a, float b) { return ex2((a - (b == -INFINITY ? 0.0f : b)) * kLog2e); }

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_wait_for(int newer) {
  switch (newer) {
    case 0: cp_wait<0>(); break;
    case 1: cp_wait<1>(); break;
    case 2: cp_wait<2>(); break;
    case 3: cp_wait<3>(); break;
    case 4: cp_wait<4>(); break;
    case 5: cp_wait<5>(); break;
    default: cp_wait<6>(); break;
  }
}

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void lds128(float (&r)[4], uint32_t a) {
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]) : "r"(a) : "memory");
}

#define MXMOE_MMA(name, shape)                                                                                      \
  __device__ __forceinline__ void name(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, \
                                       uint32_t b1) {                                                               \
    asm volatile("mma.sync.aligned." shape " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                 \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                   \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                           \
  }
MXMOE_MMA(mma_bf16, "m16n8k16.row.col.f32.bf16.bf16.f32")
MXMOE_MMA(mma_f16, "m16n8k16.row.col.f32.f16.f16.f32")
MXMOE_MMA(mma_tf32, "m16n8k8.row.col.f32.tf32.tf32.f32")
#undef MXMOE_MMA

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_of(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

__device__ __forceinline__ float ld_act(const void* p, int dtype, int64_t i) {
  return dtype == MXMOE_F32 ? static_cast<const float*>(p)[i]
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// ---- the cache's element types ----
//
// Each has: Q, the query operand; load(), which fills it for lane (g, t) =
// (lane / 4, lane % 4) from head g's row; scores(), s[4] of keys 2t, 2t + 1,
// 8 + 2t, 9 + 2t; and add(), o = o corr + p V over the tile's 16 keys.  HDT:
// head_dim rounded up to the register arrays' size; X: 32-bit activations, a
// third term each for queries and shares where two hold 16 bits only.

template <int HDT, bool X>
struct Bf16 {
  static constexpr int kElem = 2, rb = ring_row(HDT * 2), NT = tile_halves(HDT * 2);
  struct Q {
    uint32_t a[HDT / 16][X ? 6 : 2];
    float back;
  };
  static __device__ __forceinline__ void load(Q& q, const void* src, int dtype, int64_t base, bool on, int hd, int t) {
    q.back = 1.0f;
#pragma unroll
    for (int s = 0; s < HDT / 16; ++s) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = 16 * s + 8 * half + 2 * t;
        float x = 0.0f, y = 0.0f;
        if (on && c < hd) {
          x = ld_act(src, dtype, base + c);
          y = ld_act(src, dtype, base + c + 1);
        }
        const uint32_t h = pack_bf16(x, y);
        q.a[s][half] = h;
        if (X) {
          x -= lo_of(h);
          y -= hi_of(h);
          const uint32_t l = pack_bf16(x, y);
          q.a[s][2 + half] = l;
          q.a[s][4 + half] = pack_bf16(x - lo_of(l), y - hi_of(l));
        }
      }
    }
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    float c[2 * NT][4] = {};
    const uint32_t at = k + ((lane >> 4) * 8 + (lane & 7)) * rb + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < HDT / 16; ++i) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        uint32_t b[4];
        ldm4(b, at + 16 * u * rb + 32 * i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (X) {
            mma_bf16(c[2 * u + j], q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], b[2 * j], b[2 * j + 1]);
            mma_bf16(c[2 * u + j], q.a[i][4], 0, q.a[i][5], 0, b[2 * j], b[2 * j + 1]);
          } else {
            mma_bf16(c[2 * u + j], q.a[i][0], 0, q.a[i][1], 0, b[2 * j], b[2 * j + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      s[2 * j] = X ? c[j][0] + c[j][2] : c[j][0];
      s[2 * j + 1] = X ? c[j][1] + c[j][3] : c[j][1];
    }
  }
  static __device__ __forceinline__ void add(float (&o)[HDT / 8][2], const float (&p)[4 * NT], float corr, uint32_t v,
                                             int lane) {
    uint32_t h[2 * NT], l[2 * NT], m[2 * NT];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      h[j] = pack_bf16(p[2 * j], p[2 * j + 1]);
      const float x = p[2 * j] - lo_of(h[j]), y = p[2 * j + 1] - hi_of(h[j]);
      l[j] = pack_bf16(x, y);
      m[j] = X ? pack_bf16(x - lo_of(l[j]), y - hi_of(l[j])) : 0;
    }
    const uint32_t at = v + (((lane >> 3) & 1) * 8 + (lane & 7)) * rb + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < HDT / 8; n += 2) {
      float d[2][4] = {};
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        uint32_t b[4];
        ldm4t(b, at + 16 * u * rb + 16 * n);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mma_bf16(d[e], h[2 * u], l[2 * u], h[2 * u + 1], l[2 * u + 1], b[2 * e], b[2 * e + 1]);
          if (X) mma_bf16(d[e], m[2 * u], 0, m[2 * u + 1], 0, b[2 * e], b[2 * e + 1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        o[n + e][0] = fmaf(o[n + e][0], corr, d[e][0] + d[e][2]);
        o[n + e][1] = fmaf(o[n + e][1], corr, d[e][1] + d[e][3]);
      }
    }
  }
  // The column of o[n][e].
  static __device__ __forceinline__ int column(int n, int e, int t) { return 8 * n + 2 * t + e; }
};

// 8-bit keys and values widen to f16 without loss.  A query row is scaled by a
// power of two to a maximum of 2^8 to 2^9 (f16's range is too short for any
// row), two f16 terms then hold 22 bits of it; a share lies in [0, 1].  The
// order of the contracted columns within 16 is free as long as both operands
// agree: lane t takes bytes 4t to 4t + 3 of a key's 16, as one ldmatrix gives.
template <int HDT, bool X>
struct E4m3 {
  static constexpr int kElem = 1, rb = ring_row(HDT), NT = tile_halves(HDT);
  struct Q {
    uint32_t a[HDT / 16][4];
    float back;
  };
  static __device__ __forceinline__ void load(Q& q, const void* src, int dtype, int64_t base, bool on, int hd, int t) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < HDT / 16; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (on && 16 * s < hd) top = fmaxf(top, fabsf(ld_act(src, dtype, base + 16 * s + 4 * t + e)));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const int ex = (__float_as_uint(top) >> 23) & 255;
    const int field = ex == 0 || ex == 255 ? 127 : min(253, 262 - ex);
    const float f = __uint_as_float(static_cast<uint32_t>(field) << 23);
    q.back = __uint_as_float(static_cast<uint32_t>(254 - field) << 23);
#pragma unroll
    for (int s = 0; s < HDT / 16; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x = 0.0f, y = 0.0f;
        if (on && 16 * s < hd) {
          x = ld_act(src, dtype, base + 16 * s + 4 * t + 2 * half) * f;
          y = ld_act(src, dtype, base + 16 * s + 4 * t + 2 * half + 1) * f;
        }
        const uint32_t h = pack_f16(x, y);
        const __half2 hh = *reinterpret_cast<const __half2*>(&h);
        q.a[s][half] = h;
        q.a[s][2 + half] = X ? pack_f16(x - __low2float(hh), y - __high2float(hh)) : 0;
      }
  }
  static __device__ __forceinline__ uint32_t widen(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
    return static_cast<uint32_t>(h.x) | static_cast<uint32_t>(h.y) << 16;
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    float c[2 * NT][4] = {};
    // one ldmatrix: keys 0-7 and 8-15 of two 16-byte pieces
    const uint32_t at = k + ((lane >> 4) * 8 + (lane & 7)) * rb + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < HDT / 16; i += 2) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        uint32_t b[4];
        ldm4(b, at + 16 * u * rb + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = j & 1;
          const uint32_t w = b[j];
          mma_f16(c[2 * u + (j >> 1)], q.a[i + e][0], q.a[i + e][2], q.a[i + e][1], q.a[i + e][3], widen(w & 0xFFFF), widen(w >> 16));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      s[2 * j] = X ? c[j][0] + c[j][2] : c[j][0];
      s[2 * j + 1] = X ? c[j][1] + c[j][3] : c[j][1];
    }
  }
  static __device__ __forceinline__ void add(float (&o)[HDT / 8][2], const float (&p)[4 * NT], float corr, uint32_t v,
                                             int lane) {
    const int g = lane >> 2, t = lane & 3;
    uint32_t h[2 * NT], l[2 * NT];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      h[j] = pack_f16(p[2 * j], p[2 * j + 1]);
      const __half2 x = *reinterpret_cast<const __half2*>(&h[j]);
      l[j] = pack_f16(p[2 * j] - __low2float(x), p[2 * j + 1] - __high2float(x));
    }
    const uint32_t at = v + 2 * t * rb + 4 * g;
#pragma unroll
    for (int n = 0; n < HDT / 8; n += 4) {  // 32 columns: lane g holds 4g to 4g + 3 of four keys
      float d[4][4] = {};
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const uint32_t from = at + 16 * u * rb + 8 * n;
        const uint32_t w0 = lds32(from), w1 = lds32(from + rb), w2 = lds32(from + 8 * rb), w3 = lds32(from + 9 * rb);
        const uint32_t x[4] = {__byte_perm(w0, w1, 0x5140), __byte_perm(w0, w1, 0x7362), __byte_perm(w2, w3, 0x5140),
                               __byte_perm(w2, w3, 0x7362)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t y = x[e >> 1], z = x[2 + (e >> 1)];
          mma_f16(d[e], h[2 * u], l[2 * u], h[2 * u + 1], l[2 * u + 1], widen(e & 1 ? y >> 16 : y & 0xFFFF),
                  widen(e & 1 ? z >> 16 : z & 0xFFFF));
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[n + e][0] = fmaf(o[n + e][0], corr, d[e][0] + d[e][2]);
        o[n + e][1] = fmaf(o[n + e][1], corr, d[e][1] + d[e][3]);
      }
    }
  }
  static __device__ __forceinline__ int column(int n, int e, int t) { return 32 * (n / 4) + 8 * t + 4 * e + n % 4; }
};

// 32-bit keys and values as two tf32 terms each, cut off so that the second is
// exact: 21 bits of either operand.
template <int HDT, bool X>
struct F32 {
  static constexpr int kElem = 4, rb = ring_row(HDT * 4), NT = tile_halves(HDT * 4);
  struct Q {
    uint32_t a[HDT / 8][4];
    float back;
  };
  static __device__ __forceinline__ uint32_t top(float x) { return __float_as_uint(x) & 0xFFFFE000u; }
  static __device__ __forceinline__ uint32_t rest(float x) { return __float_as_uint(x - __uint_as_float(top(x))); }
  static __device__ __forceinline__ void load(Q& q, const void* src, int dtype, int64_t base, bool on, int hd, int t) {
    q.back = 1.0f;
#pragma unroll
    for (int s = 0; s < HDT / 8; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float x = on && 8 * s < hd ? ld_act(src, dtype, base + 8 * s + 4 * half + t) : 0.0f;
        q.a[s][half] = top(x);
        q.a[s][2 + half] = rest(x);
      }
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    float c[2 * NT][4] = {};
    const uint32_t at = k + ((lane >> 4) * 8 + (lane & 7)) * rb + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i = 0; i < HDT / 8; ++i) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        uint32_t b[4];
        ldm4(b, at + 16 * u * rb + 32 * i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = __uint_as_float(b[2 * j]), y = __uint_as_float(b[2 * j + 1]);
          mma_tf32(c[2 * u + j], q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], top(x), top(y));
          mma_tf32(c[2 * u + j], q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], rest(x), rest(y));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      s[2 * j] = c[j][0] + c[j][2];
      s[2 * j + 1] = c[j][1] + c[j][3];
    }
  }
  static __device__ __forceinline__ void add(float (&o)[HDT / 8][2], const float (&p)[4 * NT], float corr, uint32_t v,
                                             int lane) {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t at = v + 2 * t * rb + 16 * g;
#pragma unroll
    for (int n = 0; n < HDT / 8; n += 4) {
      float d[4][4] = {};
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) {  // keys 8u to 8u + 7
        float w[2][4];
        lds128(w[0], at + 8 * u * rb + 32 * n);
        lds128(w[1], at + (8 * u + 1) * rb + 32 * n);
        const float p0 = p[2 * u], p1 = p[2 * u + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mma_tf32(d[e], top(p0), rest(p0), top(p1), rest(p1), top(w[0][e]), top(w[1][e]));
          mma_tf32(d[e], top(p0), rest(p0), top(p1), rest(p1), rest(w[0][e]), rest(w[1][e]));
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[n + e][0] = fmaf(o[n + e][0], corr, d[e][0] + d[e][2]);
        o[n + e][1] = fmaf(o[n + e][1], corr, d[e][1] + d[e][3]);
      }
    }
  }
  static __device__ __forceinline__ int column(int n, int e, int t) { return 32 * (n / 4) + 8 * t + 4 * e + n % 4; }
};

// ---- the list of tiles ----

// Rows of a launch: cached length, and the tiles of the rows before.
struct Rows {
  int64_t* before;  // [rows + 1]
  int* len;         // [rows]
};

__device__ __forceinline__ int first_key(int len, int window) { return window && window < len ? len - window : 0; }

// All threads; ends with a barrier.
__device__ __forceinline__ void list_rows(const DecodeParams& p, Rows r, int tile) {
  __shared__ int64_t sums[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int64_t base = 0;
  for (int r0 = 0; r0 < p.rows; r0 += blockDim.x) {
    const int i = r0 + threadIdx.x;
    int len = 0;
    if (i < p.rows) {
      len = p.lens[i];
      if (len < 0 || len > cap) {
        atomicOr(p.c.status, kPagedBadIndex);
        len = len < 0 ? 0 : static_cast<int>(cap);
      }
      r.len[i] = len;
    }
    int64_t x = (len - first_key(len, p.window) + tile - 1) / tile;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int64_t all = base;
    for (int w = 0; w < n_warps; ++w) {
      if (w == warp) x += all;
      all += sums[w];
    }
    if (i < p.rows) r.before[i + 1] = x;
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) r.before[0] = 0;
  __syncthreads();
}

// A place in the list: segment `seg` (key head x group of 8 query heads) of row
// `row`, its tile `tile` of `tiles`.
struct Place {
  int row, seg, tile, tiles, len, lo;

  __device__ __forceinline__ void at_row(const DecodeParams& p, Rows r, int i) {
    row = i;
    tiles = static_cast<int>(r.before[i + 1] - r.before[i]);
    len = r.len[i];
    lo = first_key(len, p.window);
  }
  __device__ __forceinline__ void find(const DecodeParams& p, Rows r, int segs, int64_t x) {
    int a = 0, b = p.rows;  // before[a] segs <= x < before[b] segs
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (r.before[m] * segs <= x) a = m; else b = m;
    }
    at_row(p, r, a);
    const int64_t y = x - r.before[a] * segs;
    seg = static_cast<int>(y / tiles);
    tile = static_cast<int>(y - static_cast<int64_t>(seg) * tiles);
  }
  __device__ __forceinline__ void next_segment(const DecodeParams& p, Rows r, int segs) {
    tile = 0;
    if (++seg < segs) return;
    seg = 0;
    int i = row + 1;
    while (r.before[i + 1] == r.before[i]) ++i;
    at_row(p, r, i);
  }
};

__device__ __forceinline__ void store_out(const DecodeParams& p, int row, int h, int col, float4 x) {
  const int64_t o = row * p.out_row + h * p.out_head + col;
  if (p.out_dtype == MXMOE_F32) {
    float* y = static_cast<float*>(p.out) + o;
    if (p.out_wide) {
      *reinterpret_cast<float4*>(y) = x;
    } else {
      y[0] = x.x; y[1] = x.y; y[2] = x.z; y[3] = x.w;
    }
  } else {
    __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.out) + o;
    if (p.out_wide) {
      *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    } else {
      y[0] = __float2bfloat16_rn(x.x); y[1] = __float2bfloat16_rn(x.y);
      y[2] = __float2bfloat16_rn(x.z); y[3] = __float2bfloat16_rn(x.w);
    }
  }
}

// A head's maximum and sum so far, and four columns of its output.
struct Joined {
  float top = -INFINITY, sum = 0.0f;
  float4 acc = {0.0f, 0.0f, 0.0f, 0.0f};

  __device__ __forceinline__ void add(float m, float l, float4 o) {
    const float t = fmaxf(top, m), a = exp_diff(top, t), b = exp_diff(m, t);
    top = t;
    sum = fmaf(l, b, sum * a);
    acc.x = fmaf(o.x, b, acc.x * a);
    acc.y = fmaf(o.y, b, acc.y * a);
    acc.z = fmaf(o.z, b, acc.z * a);
    acc.w = fmaf(o.w, b, acc.w * a);
  }
};

// Joins the sink's and the quiet softmax's terms to a head's maximum and sum:
// the factor on its output, and the log of the normalizer.
__device__ __forceinline__ float finish(const DecodeParams& p, int h, float m, float l, float& lse) {
  float top = m;
  if (p.sinks) top = fmaxf(top, p.sinks[h]);
  if (p.quiet) top = fmaxf(top, 0.0f);
  if (top == -INFINITY && l == 0.0f) {  // no key, or every score -inf
    lse = -INFINITY;
    return 0.0f;
  }
  const float f = exp_diff(m, top);
  float sum = l * f;
  if (p.sinks) sum += exp_diff(p.sinks[h], top);
  if (p.quiet) sum += exp_diff(0.0f, top);
  lse = top + logf(sum);
  return f / sum;
}

// Four finished columns of a head, and with the first its normalizer.
__device__ __forceinline__ void write_head(const DecodeParams& p, const DecodeScratch& ws, int row, int h, int c, float vs,
                                           const Joined& j) {
  float lse;
  const float f = finish(p, h, j.top, j.sum, lse) * vs;
  store_out(p, row, h, c, make_float4(j.acc.x * f, j.acc.y * f, j.acc.z * f, j.acc.w * f));
  if (c != 0) return;
  if (p.lse) p.lse[static_cast<int64_t>(row) * p.c.n_heads + h] = lse;
  if (p.track) ws.lse[row * p.c.n_heads + h] = lse;
}

template <class C, int HDT>
__global__ void __launch_bounds__(32 * kDecodeWarps, 1)
    attend_kernel(const DecodeParams p, const DecodeScratch ws, const DecodePlan plan) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ int64_t before[kDecodeMaxRows + 1];
  __shared__ int len_of[kDecodeMaxRows];
  __shared__ int arrived[kDecodeWarps], join_at[kDecodeWarps];
  __shared__ float join_ml[kDecodeWarps][kDecodeHeads][2];
  __shared__ uint32_t there[kDecodeWarps][kDecodeMaxStages];  // which keys of a stage are in the cache
  const Rows rows{before, len_of};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int hd = p.c.head_dim, H = p.c.kv_heads, G = p.c.n_heads / H;
  const int hgroups = (G + kDecodeHeads - 1) / kDecodeHeads, segs = H * hgroups;
  constexpr int rb = C::rb, ldo = HDT + 8, NT = C::NT, kTile = 16 * NT;
  const int W = plan.warps;
  const uint32_t mine = smem_u32(ring) + warp * plan.stages * plan.stage_bytes;
  list_rows(p, rows, kTile);
  const int64_t total = before[p.rows] * segs;

  // Rows without keys: zeros.
  for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
    if (before[r + 1] != before[r]) continue;
    for (int i = threadIdx.x; i < p.c.n_heads * (hd / 4); i += blockDim.x)
      write_head(p, ws, r, i / (hd / 4), 4 * (i % (hd / 4)), 0.0f, Joined());
  }
  if (total == 0) return;

  // Warps of a worker: one where every warp has many tiles (no join in shared
  // memory), else up to half the tiles of a mean segment, so that short work
  // spreads.
  int wg = 1;
  if (total < 16LL * W * gridDim.x) {
    const int64_t mean = total / (static_cast<int64_t>(p.rows) * segs);
    while (wg < W && 2 * wg < mean) wg <<= 1;
  }
  const int group = warp / wg, in_group = warp - group * wg;
  // No more workers than give each of their warps a tile.
  int64_t n_workers = static_cast<int64_t>(gridDim.x) * (W / wg);
  if (n_workers > (total + wg - 1) / wg) n_workers = (total + wg - 1) / wg;
  const int64_t worker = static_cast<int64_t>(group) * gridDim.x + blockIdx.x;
  if (worker >= n_workers) return;
  const int64_t begin = total * worker / n_workers, end = total * (worker + 1) / n_workers;
  auto group_sync = [&]() {
    if (wg == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * wg) : "memory");
  };

  // What this warp loads next: its tile, and each lane's page of the tile's key
  // of that number, read one tile ahead.
  Place ld;
  ld.find(p, rows, segs, begin);
  int64_t ld_left = end - begin;
  int ld_off = in_group, ld_tile = 0, page = -1, slot = 0;
  bool ld_on = true;
  auto look_ahead = [&]() {
    while (true) {
      if (ld_left <= 0) {
        ld_on = false;
        return;
      }
      const int n = static_cast<int>(min(static_cast<int64_t>(ld.tiles - ld.tile), ld_left));
      if (ld_off < n) break;
      ld_left -= n;
      ld_off = in_group;
      if (ld_left > 0) ld.next_segment(p, rows, segs);
    }
    ld_tile = ld.tile + ld_off;
    ld_off += wg;
    const int n = ld.lo + ld_tile * kTile + lane % kTile;
    page = -1;
    if (n < ld.len) {
      const int pi = page_of(p.c, n);
      slot = n - pi * p.c.page_size;
      page = __ldg(p.t.tables + ld.row * p.t.stride + pi);
      if (page < 0 || page >= p.c.n_pages) page = -2;
    }
  };
  int ld_stage = 0;
  auto load_tile = [&]() {
    if (ld_on) {
      if (page == -2) atomicOr(p.c.status, kPagedBadPage);
      const uint32_t keys = __ballot_sync(0xFFFFFFFFu, page >= 0);
      if (lane == 0) there[warp][ld_stage] = keys;
      const int kvh = ld.seg / hgroups;
      const int64_t row = page < 0 ? -1
                                   : ((static_cast<int64_t>(page) * H + kvh) * p.c.page_size + slot) * (hd * C::kElem);
      const uint32_t ks = mine + ld_stage * plan.stage_bytes, vs = ks + kTile * rb;
      constexpr int kPieces = HDT * C::kElem / 16;  // 16 bytes each, zeros past head_dim
      constexpr int kLanes = kPieces % 8 == 0 ? 8 : 4, kKeys = 32 / kLanes;
      const int piece = lane % kLanes * 16;
#pragma unroll
      for (int i = 0; i < kTile / kKeys; ++i) {
        const int key = i * kKeys + lane / kLanes;
        const int64_t at = __shfl_sync(0xFFFFFFFFu, row, key);
        const int64_t from = at < 0 ? 0 : at;
        const uint8_t *kf = static_cast<const uint8_t*>(p.c.k) + from, *vf = static_cast<const uint8_t*>(p.c.v) + from;
#pragma unroll
        for (int j = 0; j < (kPieces + kLanes - 1) / kLanes; ++j) {
          const int c = j * kLanes * 16 + piece;
          if (kPieces % kLanes && c >= kPieces * 16) break;
          const bool in = at >= 0 && c < hd * C::kElem;
          cp16(ks + key * rb + c, kf + (in ? c : 0), in ? 16 : 0);
          cp16(vs + key * rb + c, vf + (in ? c : 0), in ? 16 : 0);
        }
      }
      look_ahead();
    }
    cp_commit();
    if (++ld_stage == plan.stages) ld_stage = 0;
  };
  look_ahead();
  for (int i = 0; i + 1 < plan.stages; ++i) load_tile();

  Place at;
  at.find(p, rows, segs, begin);
  int stage = 0;
  for (int64_t x = begin; x < end;) {
    const int n = static_cast<int>(min(static_cast<int64_t>(at.tiles - at.tile), end - x));
    const int kvh = at.seg / hgroups, h0 = kvh * G + (at.seg - kvh * hgroups) * kDecodeHeads;
    const int heads = min(kDecodeHeads, (kvh + 1) * G - h0);
    typename C::Q q;
    C::load(q, p.q, p.q_dtype, at.row * p.q_row + static_cast<int64_t>(h0 + g) * p.q_head, g < heads, hd, t);
    const float ks = p.scale * q.back * (p.c.k_scale ? p.c.k_scale[kvh] : 1.0f);
    const float* bias = p.bias && g < heads ? p.bias + at.row * p.bias_row + (h0 + g) * p.bias_head : nullptr;
    float m = -INFINITY, l = 0.0f;
    float o[HDT / 8][2];
#pragma unroll
    for (int i = 0; i < HDT / 8; ++i) o[i][0] = o[i][1] = 0.0f;

    for (int j = in_group; j < n; j += wg) {
      cp_wait_for(plan.stages - 2);
      __syncwarp();
      load_tile();  // into the stage that the tile before this one left
      const uint32_t k = mine + stage * plan.stage_bytes, v = k + kTile * rb;
      float s[4 * NT], w[4 * NT];
      C::scores(s, q, k, lane);
      const uint32_t keys = there[warp][stage] >> (2 * t);
      float top = m;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        const int e = 8 * (i >> 1) + (i & 1);
        s[i] *= ks;
        if (bias) {
          const int n = at.lo + (at.tile + j) * kTile + e + 2 * t;
          if (n < p.bias_len && n < at.len) s[i] += bias[n];
        }
        if (!(keys >> e & 1)) s[i] = -INFINITY;
        top = fmaxf(top, s[i]);
      }
      if (p.track && x + j < ws.score_tiles) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
          *reinterpret_cast<float4*>(ws.scores + (((x + j) * NT + u) * 32 + lane) * 4) =
              make_float4(s[4 * u], s[4 * u + 1], s[4 * u + 2], s[4 * u + 3]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const float corr = exp_diff(m, top);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        w[i] = exp_diff(s[i], top);
        sum += w[i];
      }
      l = fmaf(l, corr, sum);
      m = top;
      C::add(o, w, corr, v, lane);
      __syncwarp();
      if (++stage == plan.stages) stage = 0;
    }

    // The group's warps join in shared memory, each in the stage that it loads
    // next: nothing uses that until then.
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    const int at_stage = (warp * plan.stages + ld_stage) * plan.stage_bytes;
    float* jo = reinterpret_cast<float*>(ring + at_stage) + g * ldo;
#pragma unroll
    for (int i = 0; i < HDT / 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) jo[C::column(i, e, t)] = o[i][e];
    if (t == 0) {
      join_ml[warp][g][0] = m;
      join_ml[warp][g][1] = l;
    }
    if (lane == 0) join_at[warp] = at_stage;
    group_sync();
    const int w0 = group * wg, tid = threadIdx.x - w0 * 32, nt = 32 * wg;
    const bool whole = n == at.tiles;
    const int slot_floats = kDecodeHeads * (hd + 2), quads = hd / 4;
    float* part = ws.part + (2 * worker + (at.tile == 0 ? 1 : 0)) * slot_floats;
    const float vs = p.c.v_scale ? p.c.v_scale[kvh] : 1.0f;
    for (int i = tid; i < heads * quads; i += nt) {
      const int h = i / quads, c = 4 * (i - h * quads);
      Joined j;
      for (int w = w0; w < w0 + wg; ++w)
        j.add(join_ml[w][h][0], join_ml[w][h][1], *reinterpret_cast<const float4*>(ring + join_at[w] + 4 * (h * ldo + c)));
      if (whole) {
        write_head(p, ws, at.row, h0 + h, c, vs, j);
      } else {
        *reinterpret_cast<float4*>(part + 4 * i) = j.acc;
        if (c == 0) *reinterpret_cast<float2*>(part + kDecodeHeads * hd + 2 * h) = make_float2(j.top, j.sum);
      }
    }
    if (!whole) {
      // Workers first_w to last_w hold this segment; the last of them to come
      // here joins their parts in order.
      const int64_t s0 = before[at.row] * segs + static_cast<int64_t>(at.seg) * at.tiles, s1 = s0 + at.tiles;
      const int64_t first_w = ((s0 + 1) * n_workers - 1) / total, last_w = (s1 * n_workers - 1) / total;
      __threadfence();
      group_sync();
      if (tid == 0) arrived[group] = atomicAdd(ws.tickets + first_w, 1);
      group_sync();
      if (arrived[group] == static_cast<int>(last_w - first_w)) {
        __threadfence();
        if (tid == 0) ws.tickets[first_w] = 0;
        constexpr int kAtOnce = 4;  // pieces of the output whose loads are in flight together
        for (int i0 = tid; i0 < heads * quads; i0 += kAtOnce * nt) {
          Joined j[kAtOnce];
#pragma unroll 2
          for (int64_t w = first_w; w <= last_w; ++w) {
            const float* from = ws.part + (2 * w + (w == first_w ? 1 : 0)) * slot_floats;
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
              const int i = i0 + e * nt;
              if (i >= heads * quads) break;
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(from + kDecodeHeads * hd) + i / quads);
              j[e].add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(from) + i));
            }
          }
#pragma unroll
          for (int e = 0; e < kAtOnce; ++e) {
            const int i = i0 + e * nt, h = i / quads;
            if (i < heads * quads) write_head(p, ws, at.row, h0 + h, 4 * (i - h * quads), vs, j[e]);
          }
        }
      }
    }
    group_sync();  // the joining buffers are free again
    x += n;
    if (x < end) at.next_segment(p, rows, segs);
  }
  cp_wait<0>();
}

template <class C, int HDT>
cudaError_t launch(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  const auto fn = attend_kernel<C, HDT>;
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fn), plan.smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(fn, dim3(plan.grid), dim3(32 * plan.warps), plan.smem, st, p, ws, plan);
}

}  // namespace decode

cudaError_t launch_attend_bf16(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_bf16_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_e4m3(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_e4m3_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_f32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);

}  // namespace mxmoe
