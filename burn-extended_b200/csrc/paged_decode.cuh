// paged_decode.cuh -- the attention kernel of paged_decode.cu, a template over
// the cache's element type.
//
// The keys of all (row, key head) pairs, cut into tiles of 16 or 32, form one
// list; its tiles are dealt out evenly in contiguous ranges, so a ragged batch
// loads every SM alike.  A worker is a group of warps; each warp streams its own
// tiles through its own shared-memory ring (cp.async, no block barrier) and
// keeps a running maximum, sum and output for 8 query heads in registers: with
// m the maximum so far,
//   l = l e^(m_old - m) + sum e^(s - m),   o = o e^(m_old - m) + e^(s - m) v.
// At the end of a (row, key head) the group joins its warps in shared memory; a
// pair that more than one range holds goes through partial results in global
// memory, which a second kernel joins in the order of the keys, so the result
// does not depend on timing.
//
// The products run on the warp MMA, m = 16.  Scores: rows 0-7 hold the heads'
// queries rounded to the operand type, rows 8-15 what the rounding left, so
// their sum is exact to 16 bits and more at no extra cost -- at 8 query heads
// per key head the tile would be half empty otherwise.  Outputs: transposed,
// the values' columns as rows, as a lane's scores are then the other operand as
// they stand.  The tensor cores' larger tiles (tcgen05), with 64 or 128 keys as
// rows and the heads as 8 or 16 columns, are not used and have not been
// measured here: a full bf16 batch is bound by memory as it is, an 8-bit one
// might gain.
//
// Bound by the bytes of K and V in a full batch (64 rows of 8192 tokens, 8 key
// heads of 64 in bf16: 175 us for 1.07 GB, 6.1 TB/s, and 7 us to join).  Shorter
// work pays the start (4 us until the first keys are asked for, 3 until they
// come), the end of the last range (3) and the join (5): 32 rows of 0 to 4096
// tokens take 40 us where the bytes need 21.  8-bit and 32-bit caches cost more
// instructions per byte, a warp issues one in five cycles, and two warps share a
// scheduler: 43 us where 23 are needed (8 rows of 2K to 16K, head of 128, 8
// bits), 26 against 10 (50001 tokens, head of 80, 32 bits).  Heads of more than
// 128 spill registers and leave room for 4 warps (bf16) or 2 (32 bits): 32 rows
// of 2048 tokens, 4 key heads of 256 in bf16, take 80 us where the bytes need 42.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {

constexpr int kWholeTiles = 8;

// How one launch is laid out.
struct DecodePlan {
  int grid;
  int whole;  // no segment has more than kWholeTiles tiles: none is cut
};

namespace decode {

// Bytes from one key to the next in a ring: an odd number of 16-byte pieces, so
// that 8 rows at one column lie in 8 different groups of banks.
constexpr int ring_row(int bytes) { return (bytes / 16 | 1) * 16; }

// Tiles of a warp's ring: one in use, one on its way.  A third slows the memory
// (64 rows of 8192 tokens in bf16 189 us against 183, and 207 against 197 once the
// power cap holds the clocks down; a head of 80 13% slower).
constexpr int kStages = 2;

// Keys of a tile in 16s.  Two independent halves hide each other's latency, and
// keep more bytes on their way (heads of 64, 80, 96 in bf16 25%, 7% and 6% faster
// than with one); longer rows have enough columns, and no room.
constexpr int tile_halves(int bytes) { return bytes <= 192 ? 2 : 1; }

// One tile's keys and values, with room for a warp's output of 8 heads.
constexpr int stage_bytes(int hd, int elem) {
  const int kv = 32 * tile_halves(hd * elem) * ring_row(hd * elem), out = kDecodeHeads * hd * 4;
  return kv > out ? kv : out;
}

// Warps of a block: 8 where their rings fit, else 4 or 2.
// More do not pay: 16 with tiles of 16 keys and 128 registers spill (8 rows of 2K
// to 16K tokens in 8 bits 85 us against 45; bf16 full batch 2% slower), 12 take 50.
constexpr int kRingBytes = 217 * 1024;  // of an SM's 227 KB, beside the row list
constexpr int warps_for(int stage) { return 8 * 2 * stage <= kRingBytes ? 8 : 4 * 2 * stage <= kRingBytes ? 4 : 2; }

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
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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
__device__ __forceinline__ void lds64(float (&r)[4], uint32_t a) {
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r[0]), "=f"(r[1]) : "r"(a) : "memory");
}

// d += a b, and d = a b.
#define MXMOE_MMA(name, shape)                                                                                      \
  __device__ __forceinline__ void name(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, \
                                       uint32_t b1) {                                                               \
    asm("mma.sync.aligned." shape " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                 \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                   \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                           \
  }                                                                                                                 \
  __device__ __forceinline__ void name##_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,     \
                                             uint32_t b0, uint32_t b1) {                                            \
    asm("mma.sync.aligned." shape " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"             \
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                   \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));                                \
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

// The queries of up to 8 heads on their way to shared memory: lane l holds
// columns 4 (l + 32 i) of [8][HDT], zeros past `heads` and head_dim.  Loaded one
// segment ahead, since under a full memory pipe the answer takes microseconds.
template <int HDT, bool X>
struct Queries {
  using Quad = typename std::conditional<X, float4, uint2>::type;  // bf16 queries stay packed
  static constexpr int kQuads = kDecodeHeads * HDT / 128;
  Quad x[kQuads];

  __device__ __forceinline__ void load(const DecodeParams& p, int64_t base, int heads, int lane) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int e = lane + 32 * i, h = e / (HDT / 4), c = 4 * (e % (HDT / 4));
      const int64_t at = base + h * p.q_head + c;
      x[i] = Quad{};
      if (h >= heads || c >= p.c.head_dim) continue;
      if (X && p.q_dtype == MXMOE_F32) {
        const float* q = static_cast<const float*>(p.q) + at;
        set(i, p.q_wide ? *reinterpret_cast<const float4*>(q) : make_float4(q[0], q[1], q[2], q[3]));
      } else {
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + at;
        const uint2 u = p.q_wide ? *reinterpret_cast<const uint2*>(q)
                                 : make_uint2(q[0] | static_cast<uint32_t>(q[1]) << 16, q[2] | static_cast<uint32_t>(q[3]) << 16);
        set(i, u);
      }
    }
  }
  __device__ __forceinline__ void store(float* to, int lane) const {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) *reinterpret_cast<float4*>(to + 4 * (lane + 32 * i)) = wide(x[i]);
  }

 private:
  static __device__ __forceinline__ float4 wide(uint2 u) { return make_float4(lo_of(u.x), hi_of(u.x), lo_of(u.y), hi_of(u.y)); }
  static __device__ __forceinline__ float4 wide(float4 v) { return v; }
  __device__ __forceinline__ void set(int i, uint2 u) { put(x[i], u); }
  __device__ __forceinline__ void set(int i, float4 v) { put(x[i], v); }
  static __device__ __forceinline__ void put(uint2& d, uint2 u) { d = u; }
  static __device__ __forceinline__ void put(float4& d, uint2 u) { d = wide(u); }
  static __device__ __forceinline__ void put(float4& d, float4 v) { d = v; }
  static __device__ __forceinline__ void put(uint2&, float4) {}
};

// A warp's output, transposed: the MMA's rows are 16 columns of the values, its
// columns the 8 heads, so that shares need no second row half, and a lane keeps
// half as many sums as with heads as rows.  Of columns' group n, lane (g, t)
// holds the two that belong to g, for heads 2t and 2t + 1; pair 2n + e is head
// 2t + e's.  In 32 bits (X) each tile's products are summed apart and joined by
// one rounded addition: the MMA's own sums are cut off, and over a long row that
// would show.  For a bf16 output the MMA adds to the sums: 64 rows of 8192 tokens
// are as far from 64 bits as the formula in 32 bits, but 0.3% of the outputs
// round to the other bf16 neighbour (0.1% there).
template <int HDT, bool X>
struct Output {
  float x[HDT / 16][4];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < HDT / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
  }
  __device__ __forceinline__ void scale(float f, float g) {
#pragma unroll
    for (int n = 0; n < HDT / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] *= e & 1 ? g : f;
  }
  __device__ __forceinline__ void add(int n, const float (&d)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[n][e] += d[e];
  }
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(x[i / 2][i & 1], x[i / 2][2 + (i & 1)]); }
};

// Two scores of a lane from the two row halves of a product, or added to them:
// in 32 bits no more than four MMAs in a row add up, as each cuts its sum off.
template <int N>
__device__ __forceinline__ void sum_pair(float (&s)[N], int j, const float (&d)[4], bool first) {
  s[2 * j] = first ? d[0] + d[2] : s[2 * j] + (d[0] + d[2]);
  s[2 * j + 1] = first ? d[1] + d[3] : s[2 * j + 1] + (d[1] + d[3]);
}

// ---- the cache's element types ----
//
// Each has: Q, the query operand; V, values on their way; load(), which fills them for lane (g, t) =
// (lane / 4, lane % 4) from head g's row in shared memory; scores(), s[4] of keys 2t, 2t + 1,
// 8 + 2t, 9 + 2t; and add(), o = o corr + p V over the tile's 16 keys, with
// shares p (and so o and their sum l) that are 2^kShareBits too large.  HDT:
// head_dim rounded up to the register arrays' size; X: 32-bit activations, a
// third term each for queries and shares where two hold 16 bits only.

template <int HDT, bool X>
struct Bf16 {
  static constexpr bool kWide = X;
  static constexpr int kShareBits = 0;
  using Elem = __nv_bfloat16;
  static constexpr int kElem = 2, rb = ring_row(HDT * 2), NT = tile_halves(HDT * 2), kWarps = warps_for(stage_bytes(HDT, 2));
  static constexpr int kStageBytes = stage_bytes(HDT, 2);
  struct Q {
    uint32_t a[HDT / 16][X ? 6 : 2];
    float back;
  };
  static __device__ __forceinline__ void load(Q& q, const float* row, int t) {
    q.back = 1.0f;
#pragma unroll
    for (int s = 0; s < HDT / 16; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float2 x = *reinterpret_cast<const float2*>(row + 16 * s + 8 * half + 2 * t);
        const uint32_t h = pack_bf16(x.x, x.y);
        q.a[s][half] = h;
        if (X) {
          const float u = x.x - lo_of(h), v = x.y - hi_of(h);
          const uint32_t l = pack_bf16(u, v);
          q.a[s][2 + half] = l;
          q.a[s][4 + half] = pack_bf16(u - lo_of(l), v - hi_of(l));
        }
      }
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    constexpr int kAhead = HDT / 16 * NT <= 8 ? HDT / 16 : 4;  // steps whose keys are loaded together
    float c[2 * NT][4];
    const uint32_t at = k + ((lane >> 4) * 8 + (lane & 7)) * rb + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i0 = 0; i0 < HDT / 16; i0 += kAhead) {
      uint32_t b[kAhead][NT][4];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int u = 0; u < NT; ++u)
          if (i0 + i < HDT / 16) ldm4(b[i][u], at + 16 * u * rb + 32 * (i0 + i));
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int i = i0 + e;
        if (i >= HDT / 16) break;
        const uint32_t l0 = X ? q.a[i][X ? 2 : 0] : 0, l1 = X ? q.a[i][X ? 3 : 0] : 0;
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
          const uint32_t b0 = b[e][j / 2][2 * (j & 1)], b1 = b[e][j / 2][2 * (j & 1) + 1];
          if (i == 0 || X && i % 2 == 0)
            mma_bf16_new(c[j], q.a[i][0], l0, q.a[i][1], l1, b0, b1);
          else
            mma_bf16(c[j], q.a[i][0], l0, q.a[i][1], l1, b0, b1);
          if (X) mma_bf16(c[j], q.a[i][X ? 4 : 0], 0, q.a[i][X ? 5 : 0], 0, b0, b1);
          if (X && (i % 2 == 1 || i + 1 == HDT / 16)) sum_pair(s, j, c[j], i < 2);
        }
      }
    }
    if (X) return;
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      s[2 * j] = c[j][0];
      s[2 * j + 1] = c[j][1];
    }
  }
  // The values of the first kPre pairs of column groups, loaded ahead of the shares.
  static constexpr int kPre = HDT / 16 * NT <= 8 ? HDT / 16 : 4;
  struct V {
    uint32_t b[kPre][NT][4];
  };
  static __device__ __forceinline__ uint32_t value_at(uint32_t v, int lane) {
    return v + (((lane >> 3) & 1) * 8 + (lane & 7)) * rb + (lane >> 4) * 16;
  }
  static __device__ __forceinline__ void load(V& x, uint32_t v, int lane) {
#pragma unroll
    for (int n = 0; n < kPre; ++n)
#pragma unroll
      for (int u = 0; u < NT; ++u) ldm4t(x.b[n][u], value_at(v, lane) + 16 * u * rb + 32 * n);
  }
  static __device__ __forceinline__ void add(Output<HDT, X>& o, V& x, const float (&p)[4 * NT], uint32_t v, int lane) {
    uint32_t h[2 * NT], l[2 * NT], m[2 * NT];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      h[j] = pack_bf16(p[2 * j], p[2 * j + 1]);
      const float y = p[2 * j] - lo_of(h[j]), z = p[2 * j + 1] - hi_of(h[j]);
      l[j] = pack_bf16(y, z);
      m[j] = X ? pack_bf16(y - lo_of(l[j]), z - hi_of(l[j])) : 0;
    }
#pragma unroll
    for (int n0 = 0; n0 < HDT / 16; n0 += kPre) {
      if (n0 > 0) {
#pragma unroll
        for (int n = 0; n < kPre; ++n)
#pragma unroll
          for (int u = 0; u < NT; ++u)
            if (n0 + n < HDT / 16) ldm4t(x.b[n][u], value_at(v, lane) + 16 * u * rb + 32 * (n0 + n));
      }
#pragma unroll
      for (int i = 0; i < kPre; ++i) {
        const int n = n0 + i;
        if (n >= HDT / 16) break;
        float d[4];
        // the smallest terms first: what their sum cuts off is small too
        if constexpr (X) {
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            const uint32_t(&a)[4] = x.b[i][u];
            if (u == 0)
              mma_bf16_new(d, a[0], a[2], a[1], a[3], m[0], m[1]);
            else
              mma_bf16(d, a[0], a[2], a[1], a[3], m[2 * u], m[2 * u + 1]);
            mma_bf16(d, a[0], a[2], a[1], a[3], l[2 * u], l[2 * u + 1]);
          }
#pragma unroll
          for (int u = 0; u < NT; ++u)
            mma_bf16(d, x.b[i][u][0], x.b[i][u][2], x.b[i][u][1], x.b[i][u][3], h[2 * u], h[2 * u + 1]);
          o.add(n, d);
        } else {
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            const uint32_t(&a)[4] = x.b[i][u];
            mma_bf16(o.x[n], a[0], a[2], a[1], a[3], h[2 * u], h[2 * u + 1]);
            mma_bf16(o.x[n], a[0], a[2], a[1], a[3], l[2 * u], l[2 * u + 1]);
          }
        }
      }
    }
  }
  // The two columns of group n that belong to g: the first, and how far the
  // second is.
  static constexpr int kApart = 8;
  static __device__ __forceinline__ int column(int n, int g) { return 16 * n + g; }
};

// 8-bit keys and values widen to f16 without loss.  A query row is scaled by a
// power of two to a maximum of 2^8 to 2^9 (f16's range is too short for any
// row), two f16 terms then hold 22 bits of it, the first alone a bf16 query's
// eight.  A share lies in [0, 1] and is held in two terms as well, times 2^14
// until its segment is summed: f16 ends at 2^-24, so that unscaled terms would
// lose the shares below 2^-25, thousands of which may stand under one large
// one.  Scaled they are off by 2^-39 of the largest at most.  The MMA on
// 8-bit operands would save the widening, but its sums keep too few bits: scores
// were off by 6e-4.
// The order of the contracted columns within 16 is free as long as both
// operands agree: lane t takes bytes 4t to 4t + 3 of a key's 16, as one ldmatrix
// gives.
template <int HDT, bool X>
struct E4m3 {
  static constexpr bool kWide = X;
  static constexpr int kShareBits = 14;
  using Elem = __nv_fp8_e4m3;
  static constexpr int kElem = 1, rb = ring_row(HDT), NT = tile_halves(HDT), kWarps = warps_for(stage_bytes(HDT, 1));
  static constexpr int kStageBytes = stage_bytes(HDT, 1);
  struct Q {
    uint32_t a[HDT / 16][X ? 4 : 2];
    float back;
  };
  // Two and two of a word's four bytes, widened.
  static __device__ __forceinline__ void widen(uint32_t four, uint32_t& low, uint32_t& high) {
    asm("{.reg .b16 x, y;\n mov.b32 {x, y}, %2;\n cvt.rn.f16x2.e4m3x2 %0, x;\n cvt.rn.f16x2.e4m3x2 %1, y;}"
        : "=r"(low), "=r"(high) : "r"(four));
  }
  static __device__ __forceinline__ void load(Q& q, const float* row, int t) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < HDT / 16; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(row + 16 * s + 4 * t);
      top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
    }
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
        const float2 x = *reinterpret_cast<const float2*>(row + 16 * s + 4 * t + 2 * half);
        const uint32_t h = pack_f16(x.x * f, x.y * f);
        const __half2 hh = *reinterpret_cast<const __half2*>(&h);
        q.a[s][half] = h;
        if (X) q.a[s][X ? 2 + half : 0] = pack_f16(x.x * f - __low2float(hh), x.y * f - __high2float(hh));
      }
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    constexpr int kAhead = HDT / 32 * NT <= 8 ? HDT / 32 : 4;  // ldmatrixes whose keys are loaded together
    float c[2 * NT][4];
    // one ldmatrix: keys 0-7 and 8-15 of two 16-byte pieces
    const uint32_t at = k + ((lane >> 4) * 8 + (lane & 7)) * rb + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int i0 = 0; i0 < HDT / 32; i0 += kAhead) {
      uint32_t b[kAhead][NT][4];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int u = 0; u < NT; ++u)
          if (i0 + i < HDT / 32) ldm4(b[i][u], at + 16 * u * rb + 32 * (i0 + i));
#pragma unroll
      for (int e = 0; e < 2 * kAhead; ++e) {
        const int i = 2 * i0 + e;
        if (i >= HDT / 16) break;
        const uint32_t l0 = X ? q.a[i][X ? 2 : 0] : 0, l1 = X ? q.a[i][X ? 3 : 0] : 0;
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
          uint32_t b0, b1;
          widen(b[e / 2][j / 2][2 * (j & 1) + (e & 1)], b0, b1);
          if (i == 0 || X && i % 4 == 0)
            mma_f16_new(c[j], q.a[i][0], l0, q.a[i][1], l1, b0, b1);
          else
            mma_f16(c[j], q.a[i][0], l0, q.a[i][1], l1, b0, b1);
          if (X && (i % 4 == 3 || i + 1 == HDT / 16)) sum_pair(s, j, c[j], i < 4);
        }
      }
    }
    if (X) return;
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      s[2 * j] = c[j][0];
      s[2 * j + 1] = c[j][1];
    }
  }
  // All the tile's values, loaded ahead of the shares: of 32 columns and 16
  // keys, lane g holds columns 4g to 4g + 3 of four keys.
  struct V {
    uint32_t w[HDT / 32][NT][4];
  };
  static __device__ __forceinline__ void load(V& x, uint32_t v, int lane) {
    const uint32_t at = v + 2 * (lane & 3) * rb + 4 * (lane >> 2);
#pragma unroll
    for (int n = 0; n < HDT / 32; ++n)
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) x.w[n][u][e] = lds32(at + (16 * u + 8 * (e >> 1) + (e & 1)) * rb + 32 * n);
  }
  static __device__ __forceinline__ void add(Output<HDT, X>& o, V& x, const float (&p)[4 * NT], uint32_t v, int lane) {
    uint32_t h[2 * NT], l[2 * NT];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      h[j] = pack_f16(p[2 * j], p[2 * j + 1]);
      const __half2 y = *reinterpret_cast<const __half2*>(&h[j]);
      l[j] = pack_f16(p[2 * j] - __low2float(y), p[2 * j + 1] - __high2float(y));
    }
#pragma unroll
    for (int n = 0; n < HDT / 32; ++n) {
      float d[2][4];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const uint32_t* w = x.w[n][u];
        uint32_t y[2][4];  // [keys 2t, 8 + 2t][column]: a pair of keys each
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          widen(__byte_perm(w[2 * i], w[2 * i + 1], 0x5140), y[i][0], y[i][1]);
          widen(__byte_perm(w[2 * i], w[2 * i + 1], 0x7362), y[i][2], y[i][3]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (X) {
            if (u == 0)
              mma_f16_new(d[e], y[0][2 * e], y[0][2 * e + 1], y[1][2 * e], y[1][2 * e + 1], l[0], l[1]);
            else
              mma_f16(d[e], y[0][2 * e], y[0][2 * e + 1], y[1][2 * e], y[1][2 * e + 1], l[2 * u], l[2 * u + 1]);
            mma_f16(d[e], y[0][2 * e], y[0][2 * e + 1], y[1][2 * e], y[1][2 * e + 1], h[2 * u], h[2 * u + 1]);
          } else {
            mma_f16(o.x[2 * n + e], y[0][2 * e], y[0][2 * e + 1], y[1][2 * e], y[1][2 * e + 1], h[2 * u], h[2 * u + 1]);
            mma_f16(o.x[2 * n + e], y[0][2 * e], y[0][2 * e + 1], y[1][2 * e], y[1][2 * e + 1], l[2 * u], l[2 * u + 1]);
          }
        }
      }
      if constexpr (X) {
        o.add(2 * n, d[0]);
        o.add(2 * n + 1, d[1]);
      }
    }
  }
  static constexpr int kApart = 1;
  static __device__ __forceinline__ int column(int n, int g) { return 32 * (n / 2) + 4 * g + 2 * (n % 2); }
};

// 32-bit keys and values as two tf32 terms each, cut off so that the second is
// exact: 21 bits of either operand.
template <int HDT, bool X>
struct F32 {
  static_assert(X, "a 32-bit cache is read in 32 bits");
  static constexpr bool kWide = true;
  static constexpr int kShareBits = 0;
  using Elem = float;
  static constexpr int kElem = 4, rb = ring_row(HDT * 4), NT = tile_halves(HDT * 4), kWarps = warps_for(stage_bytes(HDT, 4));
  static constexpr int kStageBytes = stage_bytes(HDT, 4);
  struct Q {
    uint32_t a[HDT / 8][4];
    float back;
  };
  static __device__ __forceinline__ uint32_t top(float x) { return __float_as_uint(x) & 0xFFFFE000u; }
  static __device__ __forceinline__ uint32_t rest(float x) { return __float_as_uint(x - __uint_as_float(top(x))); }
  static __device__ __forceinline__ void load(Q& q, const float* row, int t) {
    q.back = 1.0f;
#pragma unroll
    for (int s = 0; s < HDT / 8; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float x = row[8 * s + 4 * half + t];
        q.a[s][half] = top(x);
        q.a[s][2 + half] = rest(x);
      }
  }
  static __device__ __forceinline__ void scores(float (&s)[4 * NT], const Q& q, uint32_t k, int lane) {
    float c[2 * NT][4];
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
          float(&d)[4] = c[2 * u + j];
          if (i % 2 == 0)
            mma_tf32_new(d, q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], rest(x), rest(y));
          else
            mma_tf32(d, q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], rest(x), rest(y));
          mma_tf32(d, q.a[i][0], q.a[i][2], q.a[i][1], q.a[i][3], top(x), top(y));
          if (i % 2 == 1) sum_pair(s, 2 * u + j, d, i < 2);
        }
      }
    }
  }
  struct V {};
  static __device__ __forceinline__ void load(V&, uint32_t, int) {}
  static __device__ __forceinline__ void add(Output<HDT, X>& o, V&, const float (&p)[4 * NT], uint32_t v, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t at = v + 2 * t * rb;
#pragma unroll
    for (int n = 0; n < HDT / 16; n += 2) {
      const bool both = n + 1 < HDT / 16;  // 32 columns, four a lane, or the last 16, two a lane
      float d[2][4];
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) {  // keys 8u to 8u + 7
        float w[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (both)
            lds128(w[i], at + 16 * g + (8 * u + i) * rb + 64 * n);
          else
            lds64(w[i], at + 8 * g + (8 * u + i) * rb + 64 * n);
        }
        const float p0 = p[2 * u], p1 = p[2 * u + 1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e == 1 && !both) break;
          const float a0 = w[0][2 * e], a1 = w[0][2 * e + 1], a2 = w[1][2 * e], a3 = w[1][2 * e + 1];
          if (u == 0)
            mma_tf32_new(d[e], rest(a0), rest(a1), rest(a2), rest(a3), rest(p0), rest(p1));
          else
            mma_tf32(d[e], rest(a0), rest(a1), rest(a2), rest(a3), rest(p0), rest(p1));
          mma_tf32(d[e], rest(a0), rest(a1), rest(a2), rest(a3), top(p0), top(p1));
          mma_tf32(d[e], top(a0), top(a1), top(a2), top(a3), rest(p0), rest(p1));
          mma_tf32(d[e], top(a0), top(a1), top(a2), top(a3), top(p0), top(p1));
        }
      }
      o.add(n, d[0]);
      if (both) o.add(n + 1, d[1]);
    }
  }
  static constexpr int kApart = 1;
  static __device__ __forceinline__ int column(int n, int g) {
    return 32 * (n / 2) + (n + 1 < HDT / 16 || n % 2 ? 4 * g + 2 * (n % 2) : 2 * g);
  }
};

// ---- the list of tiles ----

// Rows of a launch: cached length, and the tiles of the rows before.
struct Rows {
  int* before;  // [rows + 1]
  int* len;         // [rows]
};

__device__ __forceinline__ int first_key(int len, int window) { return window && window < len ? len - window : 0; }

// All threads; ends with a barrier.
__device__ __forceinline__ void list_rows(const DecodeParams& p, Rows r, int tile) {
  __shared__ int sums[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
  const int64_t cap = static_cast<int64_t>(p.t.max_pages) * p.c.page_size;
  int base = 0;
#pragma unroll 1
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
    int x = (len - first_key(len, p.window) + tile - 1) / tile;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int all = base;
#pragma unroll 1
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

// A place in the list: tile `tile` of the `tiles` of a segment, which is a row,
// a key head and up to 8 of the query heads that read it.
struct Place {
  int row, kvh, part, tile, tiles, len, lo;

  __device__ __forceinline__ void at_row(const DecodeParams& p, Rows r, int i) {
    row = i;
    tiles = r.before[i + 1] - r.before[i];
    len = r.len[i];
    lo = first_key(len, p.window);
  }
  // Tile x of the list, in which a row has `parts` segments per key head.
  __device__ __forceinline__ void find(const DecodeParams& p, Rows r, int parts, int x) {
    const int segs = p.c.kv_heads * parts;
    int a = 0, b = p.rows;  // before[a] segs <= x < before[b] segs
#pragma unroll 1
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (r.before[m] * segs <= x) a = m; else b = m;
    }
    at_row(p, r, a);
    const int y = x - r.before[a] * segs, seg = y / tiles;
    tile = y - seg * tiles;
    kvh = seg / parts;
    part = seg - kvh * parts;
  }
  __device__ __forceinline__ void next_segment(const DecodeParams& p, Rows r, int parts) {
    tile = 0;
    if (++part < parts) return;
    part = 0;
    if (++kvh < p.c.kv_heads) return;
    kvh = 0;
    int i = row + 1;
#pragma unroll 1
    while (r.before[i + 1] == r.before[i]) ++i;
    at_row(p, r, i);
  }
};

// Joins the sink's term (-inf: none) and the quiet softmax's to a head's maximum
// and sum: the factor on its output, and the log of the normalizer.
static __device__ __noinline__ float2 finish(float sink, int quiet, float m, float l) {
  const float top = fmaxf(fmaxf(m, sink), quiet ? 0.0f : -INFINITY);
  if (top == -INFINITY && l == 0.0f) return make_float2(0.0f, -INFINITY);  // no key, or every score -inf
  const float f = exp_diff(m, top), sum = l * f + exp_diff(sink, top) + (quiet ? exp_diff(0.0f, top) : 0.0f);
  return make_float2(f / sum, top + logf(sum));
}

__device__ __forceinline__ float element(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float element(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float element(const __nv_fp8_e4m3* p, int64_t i) { return static_cast<float>(p[i]); }

// Head i of the segment at `at` again, over this warp's tiles (`first`, first +
// step and so on of n), by the formula in 32-bit arithmetic: a key of score -inf
// does not count, whatever lies there, and an infinite value is infinite in its
// column.  The products of the tile loop give NaN for both, since they multiply
// by shares of 0 and split shares, queries and 32-bit keys into terms of either
// sign; a head whose sums came out NaN there is computed here.  A lane takes a
// key for the scores, columns for the output, which goes to `out`; the maximum
// and sum are returned.  64 rows of 8192 tokens with a NaN in one query head of
// each row take as long as without; with all queries NaN 0.5 ms against 0.2.
template <class C, int HDT>
static __device__ __noinline__ float2 plain_head(const DecodeParams& p, const DecodeScratch& ws, Place at, int x, int n,
                                                 int first, int step, int i, float* out) {
  using Elem = typename C::Elem;
  constexpr int kTile = 16 * C::NT, kColumns = (HDT + 31) / 32;
  const int lane = threadIdx.x & 31, hd = p.c.head_dim, G = p.c.n_heads / p.c.kv_heads, h = at.kvh * G + at.part * kDecodeHeads + i;
  const Elem *k = static_cast<const Elem*>(p.c.k), *v = static_cast<const Elem*>(p.c.v);
  const int64_t q0 = at.row * p.q_row + h * p.q_head;
  const float* qf = p.q_dtype == MXMOE_F32 ? static_cast<const float*>(p.q) + q0 : nullptr;
  const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(p.q) + q0;
  const float by = p.scale * (p.c.k_scale ? p.c.k_scale[at.kvh] : 1.0f);
  const float* bias = p.bias ? p.bias + at.row * p.bias_row + h * p.bias_head : nullptr;
  int slot = -1;  // of this lane's key, -1: none
  auto score = [&](int j) {
    const int key = at.lo + (at.tile + j) * kTile + lane;
    int bad = 0;  // has been reported where the tile was loaded
    const int64_t s = lane < kTile && key < at.len ? slot_of(p.c, p.t, at.row, key, bad) : -1;
    slot = s < 0 ? -1 : static_cast<int>(s) + at.kvh * p.c.page_size;
    if (slot < 0) return -INFINITY;
    float d[4] = {};
#pragma unroll 1
    for (int c = 0; c < hd; c += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        d[e] = fmaf(qf ? qf[c + e] : element(qb, c + e), element(k, static_cast<int64_t>(slot) * hd + c + e), d[e]);
    const float sum = ((d[0] + d[1]) + (d[2] + d[3])) * by;
    return bias && key < p.bias_len ? sum + bias[key] : sum;
  };
  float m = -INFINITY, l = 0.0f, o[kColumns] = {};
#pragma unroll 1
  for (int j = first; j < n; j += step) {
    const float s = score(j);
    m = fmaxf(m, s);
    if (!__any_sync(0xFFFFFFFFu, isnan(s) || s == INFINITY)) continue;
    // NaN scores, or inf - inf: nothing else can come of the head
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
      if (lane + 32 * c < HDT) out[lane + 32 * c] = NAN;
    return make_float2(0.0f, NAN);
  }
#pragma unroll
  for (int a = 1; a < 32; a <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, a));
#pragma unroll 1
  for (int j = first; j < n; j += step) {
    const float s = score(j), w = exp_diff(s, m);
    l += w;
    if (p.track && x + j < ws.score_tiles && lane < kTile)  // where the tile loop put it
      ws.scores[((static_cast<int64_t>(x + j) * C::NT + lane / 16) * 32 + 4 * i + lane % 8 / 2) * 4 + lane % 16 / 8 * 2 + lane % 2] = s;
#pragma unroll 1
    for (int e = 0; e < kTile; ++e) {
      const float share = __shfl_sync(0xFFFFFFFFu, w, e);
      const int64_t from = static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, slot, e)) * hd;
      if (share == 0.0f) continue;
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
        if (lane + 32 * c < hd) o[c] = fmaf(share, element(v, from + lane + 32 * c), o[c]);
    }
  }
#pragma unroll
  for (int a = 1; a < 32; a <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, a);
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
    if (lane + 32 * c < HDT) out[lane + 32 * c] = o[c];
  return make_float2(m, l);
}

__device__ __forceinline__ void store_lse(const DecodeParams& p, const DecodeScratch& ws, int row, int h, float lse) {
  if (p.lse) p.lse[static_cast<int64_t>(row) * p.c.n_heads + h] = lse;
  if (p.track) ws.lse[row * p.c.n_heads + h] = lse;
}

// How the tile list is cut into ranges, each of which one worker, a group of
// `wg` warps, works through.
//
// whole: rows are so short that every segment is a range of its own, and worker
// w takes the ranges w, w + n_workers and so on.
// Else the first n_workers ranges are dealt out, one to a worker (no more
// workers than give each of their warps a tile), the first `more` of them one
// tile above the others.  SMs are not served alike by the memory, though: with
// 8 tiles a warp and more, where warps work alone, a quarter of the list is kept
// back and goes in small ranges (n_big of 2 `small` tiles, then of `small`) to
// whoever is done.  A segment that several ranges hold has its parts joined by
// join_kernel.
struct Cut {
  Rows rows;
  int segs, whole, wg, n_workers, n_ranges, dealt, kept, each, more, small, n_big;

  // `total` tiles of n_rows x segs segments over `warps` warps, W to a block.
  __device__ __forceinline__ Cut(Rows r, int n_rows, int segs_of_row, int total, int warps, int W, int whole_)
      : rows(r), segs(segs_of_row), whole(whole_), wg(1) {
    const int n_segs = n_rows * segs;
    // A warp alone waits for no other; but where there are few segments, warps
    // in groups leave fewer parts to join.  No more warps than a mean segment
    // has tiles.
    const int most = whole ? warps / (2 * n_segs) : warps / (32 * n_segs);
#pragma unroll 1
    while (wg < W && wg < most + whole && wg * n_segs < total) wg <<= 1;
    if (whole) {
      n_workers = min(warps / wg, n_segs);
      n_ranges = n_segs;
      kept = 0;
      return;
    }
    n_workers = min(warps / wg, (total + wg - 1) / wg);
    kept = wg == 1 && total >= 8 * warps ? total / 4 : 0;
    dealt = total - kept;
    each = dealt / n_workers;
    more = dealt - each * n_workers;
    small = max(2, (kept + 3 * warps - 1) / (3 * warps));
    n_big = min(warps, kept / (2 * small));
    n_ranges = n_workers + n_big + (kept - 2 * small * n_big + small - 1) / small;
  }
  // The first tile of range r; whole: its segment's, which may have none.
  __device__ __forceinline__ int begin_of(int r) const {
    if (whole) {
      const int row = r / segs;
      return rows.before[row] * segs + (r - row * segs) * (rows.before[row + 1] - rows.before[row]);
    }
    if (r <= n_workers) return r * each + min(r, more);
    r -= n_workers;
    return dealt + (r <= n_big ? 2 * small * r : min(kept, 2 * small * n_big + small * (r - n_big)));
  }
  __device__ __forceinline__ int end_of(int r) const {
    if (!whole) return begin_of(r + 1);
    const int row = r / segs;
    return begin_of(r) + rows.before[row + 1] - rows.before[row];
  }
  // The range of tile x (not whole).
  __device__ __forceinline__ int range_of(int x) const {
    const int edge = more * (each + 1), big = dealt + 2 * small * n_big;
    if (x < edge) return x / (each + 1);
    if (x < dealt) return more + (x - edge) / each;
    return n_workers + (x < big ? (x - dealt) / (2 * small) : n_big + (x - big) / small);
  }
  // whole: the next of a worker's ranges from r on that has tiles.
  __device__ __forceinline__ int filled(int r) const {
#pragma unroll 1
    while (r < n_ranges && rows.before[r / segs + 1] == rows.before[r / segs]) r += n_workers;
    return r;
  }
};

// Two finished columns of a head.
template <int kApart>
__device__ __forceinline__ void store_out(const DecodeParams& p, int row, int h, int col, float x, float y) {
  const int64_t o = row * p.out_row + h * p.out_head + col;
  const int hd = p.c.head_dim;
  if (p.out_dtype == MXMOE_F32) {
    float* d = static_cast<float*>(p.out) + o;
    if (col < hd) d[0] = x;
    if (col + kApart < hd) d[kApart] = y;
  } else {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.out) + o;
    if (kApart == 1 && p.out_wide) {
      if (col < hd) *reinterpret_cast<uint32_t*>(d) = pack_bf16(x, y);
    } else {
      if (col < hd) d[0] = __float2bfloat16_rn(x);
      if (col + kApart < hd) d[kApart] = __float2bfloat16_rn(y);
    }
  }
}

template <class C, int HDT>
__global__ void __launch_bounds__(32 * C::kWarps, 1)
    attend_kernel(const __grid_constant__ DecodeParams p, const __grid_constant__ DecodeScratch ws, const DecodePlan plan) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ int before[kDecodeMaxRows + 1];
  __shared__ int len_of[kDecodeMaxRows];
  __shared__ int join_at[kDecodeWarps], queue[kDecodeWarps][8];
  __shared__ float join_ml[kDecodeWarps][kDecodeHeads][2];
  __shared__ uint32_t there[kDecodeWarps][kStages];  // which keys of a stage are in the cache
  // The tile after the loaded ones: first key, keys left, key head (-1: no tile),
  // and each lane's page number.
  __shared__ int4 ahead[C::kWarps];
  __shared__ int page_at[C::kWarps][32];
  const Rows rows{before, len_of};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int hd = p.c.head_dim, H = p.c.kv_heads, G = p.c.n_heads / H;
  const int parts = (G + kDecodeHeads - 1) / kDecodeHeads, segs = H * parts;
  constexpr int W = C::kWarps, kStageBytes = C::kStageBytes;
  constexpr uint32_t kAllKeys = 0xFFFFFFFFu;
  constexpr int rb = C::rb, NT = C::NT, kTile = 16 * NT, kPairs = HDT / 8;  // column pairs of a lane
  uint8_t* const mine = ring + warp * kStages * kStageBytes;
  griddep_wait();
  griddep_launch_dependents();
  list_rows(p, rows, kTile);
  const int total = before[p.rows] * segs, n_segs = p.rows * segs;

  auto idle_rows = [&]() {  // rows without keys: zeros
#pragma unroll 1
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
      if (before[r + 1] != before[r]) continue;
#pragma unroll 1
      for (int i = threadIdx.x; i < p.c.n_heads * hd; i += blockDim.x) {
        const int h = i / hd;
        const int64_t o = r * p.out_row + h * p.out_head + (i - h * hd);
        if (p.out_dtype == MXMOE_F32)
          static_cast<float*>(p.out)[o] = 0.0f;
        else
          static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(0.0f);
      }
#pragma unroll 1
      for (int h = threadIdx.x; h < p.c.n_heads; h += blockDim.x)
        store_lse(p, ws, r, h, finish(p.sinks ? p.sinks[h] : -INFINITY, p.quiet, -INFINITY, 0.0f).y);
    }
  };
  if (total == 0) {
    idle_rows();
#pragma unroll 1
    for (int s = blockIdx.x + gridDim.x * threadIdx.x; s < n_segs && !plan.whole; s += gridDim.x * blockDim.x)
      ws.held[s] = make_int2(0, 0);
    return;
  }

  const Cut cut(rows, p.rows, segs, total, W * gridDim.x, W, plan.whole);
  const int wg = cut.wg, group = warp / wg, in_group = warp - group * wg, w0 = group * wg, tid = threadIdx.x - w0 * 32, nt = 32 * wg;
  const int worker = group * gridDim.x + blockIdx.x;
  int range = cut.whole ? cut.filled(worker) : worker;
  const bool works = worker < cut.n_workers && range < cut.n_ranges;
  auto group_sync = [&]() {
    if (wg == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * wg) : "memory");
  };

  // The place of the next tile that this warp looks at.
  Place ld, at;
  int x = 0, end = 0, ld_left = 0, ld_off = in_group, ld_stage = 0;
  // The next segment's queries and its heads' sinks.
  Queries<HDT, C::kWide> queries;
  float sink_next = -INFINITY;
  auto fetch = [&](const Place& of) {
    const int h0 = of.kvh * G + of.part * kDecodeHeads, heads = min(kDecodeHeads, G - of.part * kDecodeHeads);
    queries.load(p, of.row * p.q_row + h0 * p.q_head, heads, lane);
    if (p.sinks && g < heads) sink_next = p.sinks[h0 + g];
  };
  // Ranges taken after the first.  One that was kept back is asked for when the
  // one before it begins to be loaded, and waits in `queue` for its use; each
  // has two tiles at least but the list's last, and the load side is two tiles
  // ahead.
  int ld_range = range, asked = 0, queued = 0, used = 0;
  bool last_piece = false, fetched = false;  // of the range in use; the next one's queries are on their way
  auto ask = [&]() {
    if (cut.kept > 0 && lane == 0) asked = cut.n_workers + atomicAdd(ws.taken, 1);
  };
  constexpr int kPieces = HDT * C::kElem / 16;  // of a key's row, 16 bytes each; zeros past head_dim
  constexpr int kLanes = kPieces % 8 == 0 ? 8 : 4, kKeys = 32 / kLanes;
  const int piece = lane % kLanes * 16;
  const uint8_t* const k_piece = static_cast<const uint8_t*>(p.c.k) + piece;
  const int64_t v_apart = static_cast<const uint8_t*>(p.c.v) - static_cast<const uint8_t*>(p.c.k);
  // Looks at the next tile: its place into `ahead`, its keys' page numbers on
  // their way to `page_at`, in the group of copies that is open.  Under a full
  // memory pipe the answer takes as long as the tiles before it in the pipe, so a
  // number that travels with one tile's keys is there when that tile is used and
  // the next is loaded.
  auto look = [&]() {
    int n = min(ld.tiles - ld.tile, ld_left);
#pragma unroll 1
    while (ld_off >= n && ld_left > 0) {
      ld_left -= n;
      ld_off = in_group;
      if (ld_left > 0) {
        ld.next_segment(p, rows, parts);
      } else if (cut.whole || cut.kept > 0) {
        ld_range = cut.whole ? cut.filled(ld_range + cut.n_workers) : __shfl_sync(0xFFFFFFFFu, asked, 0);
        if (cut.kept > 0 && lane == 0) queue[warp][queued & 7] = ld_range;
        ++queued;
        if (ld_range < cut.n_ranges) {
          const int y = cut.begin_of(ld_range);
          ld_left = cut.end_of(ld_range) - y;
          ld.find(p, rows, parts, y);
          ask();
          if (cut.kept > 0 && last_piece && !fetched && queued - 1 == used) {  // it is the next one
            fetch(ld);
            fetched = true;
          }
        }
      }
      n = min(ld.tiles - ld.tile, ld_left);
    }
    int4 a = make_int4(0, 0, -1, 0);
    if (ld_left > 0) {
      a.x = ld.lo + (ld.tile + ld_off) * kTile;
      a.y = ld.len - a.x;
      a.z = ld.kvh;
      ld_off += wg;
      if (lane % kTile < a.y)
        cp4(smem_u32(&page_at[warp][lane]), p.t.tables + ld.row * p.t.stride + page_of(p.c, a.x + lane % kTile));
    }
    if (lane == 0) ahead[warp] = a;
  };
  // Loads the tile that was looked at into the stage that is free, all its keys,
  // then all its values, and looks at another.  In one burst: values asked for
  // after the scores, or keys and values in turn, come slower (full batch at the
  // power cap 206 and 195 us against 194).
  auto load_tile = [&]() {
    const int4 a = ahead[warp];
    if (a.z >= 0) {
      const int key0 = a.x + lane % kTile;
      const bool in = lane % kTile < a.y;
      const int page = in ? page_at[warp][lane] : -1;
      const bool good = in && page >= 0 && page < p.c.n_pages;
      if (in && !good) atomicOr(p.c.status, kPagedBadPage);
      const uint32_t keys = __ballot_sync(0xFFFFFFFFu, good);
      if (lane == 0) there[warp][ld_stage] = keys;
      const int row = good ? (page * H + a.z) * p.c.page_size + key0 - page_of(p.c, key0) * p.c.page_size : -1;
      const uint32_t ks = smem_u32(mine) + ld_stage * kStageBytes, vs = ks + kTile * rb;
      if (keys == kAllKeys && kPieces * 16 == hd * C::kElem) {
        const uint8_t* kf[kTile / kKeys];
#pragma unroll
        for (int i = 0; i < kTile / kKeys; ++i) {
          const int key = i * kKeys + lane / kLanes;
          kf[i] = k_piece + static_cast<int64_t>(__shfl_sync(0xFFFFFFFFu, row, key)) * (HDT * C::kElem);
#pragma unroll
          for (int j = 0; j < (kPieces + kLanes - 1) / kLanes; ++j) {
            const int c = j * kLanes * 16;
            if (kPieces % kLanes && c + piece >= kPieces * 16) break;
            cp16(ks + key * rb + piece + c, kf[i] + c, 16);
          }
        }
#pragma unroll
        for (int i = 0; i < kTile / kKeys; ++i) {
          const int key = i * kKeys + lane / kLanes;
#pragma unroll
          for (int j = 0; j < (kPieces + kLanes - 1) / kLanes; ++j) {
            const int c = j * kLanes * 16;
            if (kPieces % kLanes && c + piece >= kPieces * 16) break;
            cp16(vs + key * rb + piece + c, kf[i] + v_apart + c, 16);
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kTile / kKeys; ++i) {
          const int key = i * kKeys + lane / kLanes;
          const int from = __shfl_sync(0xFFFFFFFFu, row, key);
          const uint8_t* kf = k_piece + static_cast<int64_t>(max(from, 0)) * (hd * C::kElem) - piece;
#pragma unroll
          for (int j = 0; j < (kPieces + kLanes - 1) / kLanes; ++j) {
            const int c = j * kLanes * 16 + piece;
            if (kPieces % kLanes && c >= kPieces * 16) break;
            const bool in = from >= 0 && c < hd * C::kElem;
            cp16(ks + key * rb + c, kf + (in ? c : 0), in ? 16 : 0);
            cp16(vs + key * rb + c, kf + v_apart + (in ? c : 0), in ? 16 : 0);
          }
        }
      }
    }
    __syncwarp();  // `ahead` has been read
    look();
    cp_commit();
    ld_stage ^= 1;
  };

  // The first tiles and queries are on their way before anything else is done.
  if (works) {
    x = cut.begin_of(range);
    end = cut.end_of(range);
    ld_left = end - x;
    ld.find(p, rows, parts, x);
    at = ld;
    ask();
    look();
    cp_commit();
    fetch(at);
    cp_wait<0>();
    __syncwarp();
    load_tile();
  }
  idle_rows();
  if (!plan.whole) {
    // For join_kernel: the first and last range of every segment.
#pragma unroll 1
    for (int s = blockIdx.x + gridDim.x * threadIdx.x; s < n_segs; s += gridDim.x * blockDim.x) {
      const int r = s / segs, tiles = before[r + 1] - before[r], y = before[r] * segs + (s - r * segs) * tiles;
      ws.held[s] = tiles == 0 ? make_int2(0, 0) : make_int2(cut.range_of(y), cut.range_of(y + tiles - 1));
    }
  }
  if (!works) return;

  constexpr int kPartPairs = 32 * kPairs + kDecodeHeads;  // [pairs][lane] of o, then (m, l) by head
  float2* const part_of = reinterpret_cast<float2*>(ws.part);
  int stage = 0;
  while (true) {
    if (x >= end) {
      if (!cut.whole && cut.kept == 0) break;
      range = cut.whole ? cut.filled(range + cut.n_workers) : queue[warp][used++ & 7];
      if (range >= cut.n_ranges) break;
      x = cut.begin_of(range);
      end = cut.end_of(range);
      at.find(p, rows, parts, x);
      if (!fetched) fetch(at);
      fetched = false;
    }
    const int row = at.row, kvh = at.kvh, part = at.part;
    float2* to = nullptr;  // where this range's part of the segment goes; null: the output
    float m = -INFINITY, l = 0.0f, unit = 1.0f;
    Output<HDT, C::kWide> o;
    o.clear();
    const float sink = sink_next;
    {
      const int n = min(at.tiles - at.tile, end - x), h0 = kvh * G + part * kDecodeHeads;
      if (n < at.tiles) {
        const int e = at.tile == 0 ? 1 : 0;
        to = part_of + (2 * range + e) * kPartPairs;
      }
      // the queries go through the stage that is free until the next load
      typename C::Q q;
      {
        float* qs = reinterpret_cast<float*>(mine + ld_stage * kStageBytes);
        queries.store(qs, lane);
        __syncwarp();
        C::load(q, qs + g * HDT, t);
        __syncwarp();
      }
      // Scores stay as the product gives them where a positive factor alone
      // stands between them and the exponent: e^(unit (s - m)) = 2^(c (s - m)).
      // With a bias they are brought to its unit first; the difference comes
      // before log2 e, so that the type's lowest values stay apart from -inf.
      const float ks = p.scale * q.back * (p.c.k_scale ? p.c.k_scale[kvh] : 1.0f);
      const bool plain = !p.bias && ks > 0.0f;
      unit = plain ? ks : 1.0f;
      const float c = unit * kLog2e;
      const float* bias = p.bias && part * kDecodeHeads + g < G ? p.bias + row * p.bias_row + (h0 + g) * p.bias_head : nullptr;
      last_piece = x + n >= end;
      if (!last_piece) {
        Place then = at;
        then.next_segment(p, rows, parts);
        fetch(then);
      } else if (cut.whole || queued > used) {
        // the next range is known (else the load side fetches, when it comes to that)
        const int r = cut.whole ? cut.filled(range + cut.n_workers) : queue[warp][used & 7];
        if (r < cut.n_ranges) {
          Place then;
          then.find(p, rows, parts, cut.begin_of(r));
          fetch(then);
          fetched = true;
        }
      }
#pragma unroll 1
      for (int j = in_group; j < n; j += wg) {
        cp_wait<0>();
        __syncwarp();
        load_tile();
        const uint32_t k = smem_u32(mine) + stage * kStageBytes, v = k + kTile * rb;
        float s[4 * NT], w[4 * NT];
        C::scores(s, q, k, lane);
        typename C::V values;
        C::load(values, v, lane);
        if (!plain) {
#pragma unroll
          for (int i = 0; i < 4 * NT; ++i) {
            s[i] *= ks;
            const int key = at.lo + (at.tile + j) * kTile + 8 * (i >> 1) + (i & 1) + 2 * t;
            if (bias && key < p.bias_len && key < at.len) s[i] += bias[key];
          }
        }
        const uint32_t keys = there[warp][stage];
        if (keys != kAllKeys) {
#pragma unroll
          for (int i = 0; i < 4 * NT; ++i)
            if (!(keys >> (2 * t + 8 * (i >> 1) + (i & 1)) & 1)) s[i] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 4 * NT; ++i) top = fmaxf(top, s[i]);
        if (p.track && x + j < ws.score_tiles) {
#pragma unroll
          for (int u = 0; u < NT; ++u)
            *reinterpret_cast<float4*>(ws.scores + ((static_cast<int64_t>(x + j) * NT + u) * 32 + lane) * 4) =
                make_float4(s[4 * u] * unit, s[4 * u + 1] * unit, s[4 * u + 2] * unit, s[4 * u + 3] * unit);
        }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        top = fmaxf(top, m);
        const float base = top == -INFINITY ? 0.0f : top, corr = ex2((m - base) * c);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i) {
          w[i] = C::kShareBits ? ex2(fmaf(s[i] - base, c, C::kShareBits)) : ex2((s[i] - base) * c);
          sum += w[i];
        }
        l = fmaf(l, corr, sum);
        if (__any_sync(0xFFFFFFFFu, top != m)) o.scale(__shfl_sync(0xFFFFFFFFu, corr, 8 * t), __shfl_sync(0xFFFFFFFFu, corr, 8 * t + 4));
        m = top;
        C::add(o, values, w, v, lane);
        __syncwarp();
        stage ^= 1;
      }
      m *= unit;
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
      if constexpr (C::kShareBits > 0) {
        constexpr float kBack = 1.0f / (1 << C::kShareBits);
        l *= kBack;
        o.scale(kBack, kBack);
      }
      bool odd[2] = {};  // NaN in a column of head 2t, 2t + 1
#pragma unroll
      for (int i = 0; i < kPairs; ++i) odd[i & 1] |= isnan(o.pair(i).x) || isnan(o.pair(i).y);
      const uint32_t evens = __ballot_sync(0xFFFFFFFFu, odd[0]), odds = __ballot_sync(0xFFFFFFFFu, odd[1]), sums = __ballot_sync(0xFFFFFFFFu, isnan(l));
      if (evens | odds | sums) {
        float* const out = reinterpret_cast<float*>(mine + ld_stage * kStageBytes);  // [8][HDT] in the free stage
#pragma unroll 1
        for (int i = 0; i < min(kDecodeHeads, G - part * kDecodeHeads); ++i) {
          if (!((i & 1 ? odds : evens) & 0x11111111u << i / 2) && !(sums >> 4 * i & 15)) continue;
          const float2 ml = plain_head<C, HDT>(p, ws, at, x, n, in_group, wg, i, out + i * HDT);
          __syncwarp();
          if (g == i) {
            m = ml.x;
            l = ml.y;
          }
          if (i / 2 == t) {
#pragma unroll
            for (int e = 0; e < HDT / 16; ++e) {
              const float* from = out + i * HDT + C::column(e, g);
              if (i & 1) {
                o.x[e][1] = from[0];
                o.x[e][3] = from[C::kApart];
              } else {
                o.x[e][0] = from[0];
                o.x[e][2] = from[C::kApart];
              }
            }
          }
        }
        __syncwarp();
      }
      x += n;
      if (x < end) at.next_segment(p, rows, parts);
    }

    if (to && wg == 1) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) to[32 * i + lane] = o.pair(i);
      if (t == 0) to[32 * kPairs + g] = make_float2(m, l);
      continue;
    }
    // The group's warps join in shared memory, each in the stage that it loads
    // next: nothing uses that until then.
    const int heads = min(kDecodeHeads, G - part * kDecodeHeads), h0 = kvh * G + part * kDecodeHeads;
    float2* mo = reinterpret_cast<float2*>(mine + ld_stage * kStageBytes);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) mo[32 * i + lane] = o.pair(i);
    if (t == 0) {
      join_ml[warp][g][0] = m;
      join_ml[warp][g][1] = l;
    }
    if (lane == 0) join_at[warp] = (warp * kStages + ld_stage) * kStageBytes;
    group_sync();
    // a lane weighs head lane % 8, and asks others for those of its pairs
    const int mine_h = lane % kDecodeHeads;
    const float its_sink = __shfl_sync(0xFFFFFFFFu, sink, 4 * mine_h);
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < wg) top = fmaxf(top, join_ml[w0 + w][mine_h][0]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w >= wg) break;
      sum = fmaf(join_ml[w0 + w][mine_h][1], exp_diff(join_ml[w0 + w][mine_h][0], top), sum);
    }
    float f = 1.0f;
    if (to) {
      if (tid < kDecodeHeads) to[32 * kPairs + tid] = make_float2(top, sum);
    } else if (mine_h < heads) {
      const float2 y = finish(its_sink, p.quiet, top, sum);
      f = y.x * (p.c.v_scale ? p.c.v_scale[kvh] : 1.0f);
      if (tid < kDecodeHeads) store_lse(p, ws, row, h0 + mine_h, y.y);
    }
    __syncwarp();
#pragma unroll 1
    for (int i = tid; i < 32 * kPairs; i += nt) {
      const int head = 2 * t + (i / 32 & 1);
      const float its_top = __shfl_sync(0xFFFFFFFFu, top, head), its_f = __shfl_sync(0xFFFFFFFFu, f, head);
      float a = 0.0f, b = 0.0f;
#pragma unroll 4
      for (int w = w0; w < w0 + wg; ++w) {
        const float e = exp_diff(join_ml[w][head][0], its_top);
        const float2 y = reinterpret_cast<const float2*>(ring + join_at[w])[i];
        a = fmaf(y.x, e, a);
        b = fmaf(y.y, e, b);
      }
      if (to)
        to[i] = make_float2(a, b);
      else if (head < heads)
        store_out<C::kApart>(p, row, h0 + head, C::column(i / 64, g), a * its_f, b * its_f);
    }
    group_sync();  // the stages are free again
  }
  cp_wait<0>();
  // The last warp to leave sets the counter back.
  if (cut.kept > 0 && lane == 0 && atomicAdd(ws.taken + 1, 1) == cut.n_workers - 1) {
    ws.taken[0] = 0;
    ws.taken[1] = 0;
  }
}

// The segments that several ranges hold: a block joins a slice of the columns
// of one, its warps every eighth part, in the ranges' order; the loads of
// kAtOnce parts are in flight at once.
template <class C, int HDT, int kSlice, int kAtOnce>
__global__ void __launch_bounds__(256) join_kernel(const DecodeParams p, const DecodeScratch ws) {
  constexpr int kPairs = HDT / 8, kPartPairs = 32 * kPairs + kDecodeHeads;
  static_assert(kPairs % kSlice == 0 && kSlice <= 8, "slices cover the columns");
  __shared__ float2 outs[8][32 * kSlice], ml[8][kDecodeHeads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, p0 = blockIdx.y * kSlice;
  const int H = p.c.kv_heads, G = p.c.n_heads / H, parts = (G + kDecodeHeads - 1) / kDecodeHeads, segs = H * parts;
  griddep_wait();
  griddep_launch_dependents();
#pragma unroll 1
  for (int s = blockIdx.x; s < p.rows * segs; s += gridDim.x) {
    const int2 held = __ldcg(ws.held + s);
    const int row = s / segs, kvh = (s - row * segs) / parts, part = s - row * segs - kvh * parts;
    const int first = held.x, last = held.y;
    if (first == last) continue;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {};  // of heads 2t and 2t + 1
    float2 o[kSlice];
#pragma unroll
    for (int i = 0; i < kSlice; ++i) o[i] = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (int w = first + warp; w <= last; w += 8 * kAtOnce) {
      float4 y[kAtOnce];
      float2 z[kAtOnce][kSlice];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int v = w + 8 * j;
        y[j] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
#pragma unroll
        for (int i = 0; i < kSlice; ++i) z[j][i] = make_float2(0.0f, 0.0f);
        if (v > last) continue;
        const float2* from = reinterpret_cast<const float2*>(ws.part) + (2 * v + (v == first ? 1 : 0)) * kPartPairs;
        y[j] = __ldcg(reinterpret_cast<const float4*>(from + 32 * kPairs) + t);
#pragma unroll
        for (int i = 0; i < kSlice; ++i) z[j][i] = __ldcg(from + 32 * (p0 + i) + lane);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        float a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ym = e ? y[j].z : y[j].x, top = fmaxf(m[e], ym);
          a[e] = exp_diff(m[e], top);
          b[e] = exp_diff(ym, top);
          m[e] = top;
          l[e] = l[e] * a[e] + (e ? y[j].w : y[j].y) * b[e];
        }
#pragma unroll
        for (int i = 0; i < kSlice; ++i) {
          o[i].x = fmaf(z[j][i].x, b[i & 1], o[i].x * a[i & 1]);
          o[i].y = fmaf(z[j][i].y, b[i & 1], o[i].y * a[i & 1]);
        }
      }
    }
    __syncthreads();  // the segment before is read out
#pragma unroll
    for (int i = 0; i < kSlice; ++i) outs[warp][32 * i + lane] = o[i];
    if (g < 2) ml[warp][2 * t + g] = make_float2(g ? m[1] : m[0], g ? l[1] : l[0]);
    __syncthreads();
    const int used = min(8, last - first + 1), head = 2 * t + (warp & 1), h = kvh * G + part * kDecodeHeads + head;
    if (warp >= kSlice || part * kDecodeHeads + head >= G) continue;
    float top = -INFINITY, sum = 0.0f, a = 0.0f, b = 0.0f;
    for (int w = 0; w < used; ++w) top = fmaxf(top, ml[w][head].x);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w >= used) break;
      const float e = exp_diff(ml[w][head].x, top);
      const float2 y = outs[w][32 * warp + lane];
      sum = fmaf(ml[w][head].y, e, sum);
      a = fmaf(y.x, e, a);
      b = fmaf(y.y, e, b);
    }
    const float2 f = finish(p.sinks ? p.sinks[h] : -INFINITY, p.quiet, top, sum);
    const float by = f.x * (p.c.v_scale ? p.c.v_scale[kvh] : 1.0f);
    if (p0 == 0 && warp < 2 && g == 0) store_lse(p, ws, row, h, f.y);
    store_out<C::kApart>(p, row, h, C::column((p0 + warp) / 2, g), a * by, b * by);
  }
}

template <class C, int HDT>
cudaError_t launch(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  static_assert(kStages * C::kWarps * C::kStageBytes <= kRingBytes, "the rings fit");
  const auto fn = attend_kernel<C, HDT>;
  // the warps' rings, and 128 bytes that a read past the last row may touch
  constexpr size_t smem = C::kWarps * kStages * C::kStageBytes + 128;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fn), smem);
  if (e != cudaSuccess) return e;
  e = launch_kernel(fn, dim3(plan.grid), dim3(32 * C::kWarps), smem, st, p, ws, plan);
  if (e != cudaSuccess || plan.whole) return e;
  const int G = p.c.n_heads / p.c.kv_heads, n_segs = p.rows * p.c.kv_heads * ((G + kDecodeHeads - 1) / kDecodeHeads);
  // Few segments are long ones: narrow slices, so that their parts are read by
  // more blocks, eight at once (2 of 50001 tokens 26.8 us in all against 27.8).
  // Many would not all be resident that way (512 of 8192 tokens 196 us against
  // 186); fewer parts at once than four are slower where a segment has 20 and
  // more (64 of 2K to 16K tokens in 8 bits 47 us against 44).
  constexpr int kWide = HDT / 8 % 4 ? 2 : 4;
  if (n_segs * HDT / 16 <= 2 * plan.grid)
    return launch_kernel(join_kernel<C, HDT, 2, 8>, dim3(n_segs, HDT / 16), dim3(256), 0, st, p, ws);
  return launch_kernel(join_kernel<C, HDT, kWide, 4>, dim3(n_segs < 4 * plan.grid ? n_segs : 4 * plan.grid, HDT / 8 / kWide), dim3(256),
                       0, st, p, ws);
}

}  // namespace decode

cudaError_t launch_attend_bf16(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_bf16_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_e4m3(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_e4m3_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);
cudaError_t launch_attend_f32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st);

}  // namespace mxmoe
