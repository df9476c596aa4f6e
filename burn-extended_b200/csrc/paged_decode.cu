// paged_decode.cu -- attention of one new token per row over a paged cache.
//
// For row r, query head h and its key head g, over the keys n in
// [max(0, len - window), len):
//   s_n = scale q . k_n + bias_n,   m = max(s_n, sink_h, [quiet] 0)
//   L = sum_n e^(s_n - m) + e^(sink_h - m) + [quiet] e^(-m)
//   o = sum_n e^(s_n - m) v_n / L
// A row without keys, or whose scores are all -inf, gives zeros.  With track
// the shares e^(s_n - m) / L of the heads that read key head g are added to the
// weight of slot n: the attention kernel leaves the scores and each head's log
// of the normalizer, and a second kernel turns them into shares once the
// normalizers are known.
#include "paged_decode.cuh"

#include <algorithm>
#include <cstdint>

namespace mxmoe {
namespace {

// The register arrays' head size that the kernels are built for.
int padded_head(const PagedView& c) {
  for (const int d : {64, 80, 96, 128})
    if (c.head_dim <= d && (d != 80 || c.dtype != MXMOE_E4M3)) return d;
  return 256;
}

int warps_of(const PagedView& c) {
  return decode::warps_for(decode::stage_bytes(padded_head(c), c.dtype == MXMOE_F32 ? 4 : c.dtype == MXMOE_BF16 ? 2 : 1));
}

// One warp per tile of cached keys of a (row, key head): the 8 lanes that hold
// one key's scores of 8 heads sum their shares, lane j adds key j's to its
// slot.  Moves 8 bytes of weight and 32 of scores per key and 8 heads; bound by
// the latency of its chain (lengths, page table, weight; normalizer, scores):
// 16 rows of 1000 to 4096 tokens, 8 key heads, 13 MB in 9 us, of which the first
// three loads overlap the join.
template <int NT>
__global__ void __launch_bounds__(256) weigh_kernel(const DecodeParams p, const DecodeScratch ws) {
  __shared__ int before[kDecodeMaxRows + 1];
  __shared__ int len_of[kDecodeMaxRows];
  const decode::Rows rows{before, len_of};
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int H = p.c.kv_heads, G = p.c.n_heads / H, hgroups = (G + kDecodeHeads - 1) / kDecodeHeads;
  // This kernel starts when every block of the one before it has seen the end of
  // the work before that: lengths, tables and weights are ready.  Only the
  // normalizers, and the scores where no join came between, have to be waited
  // for, once the first slots and weights are on their way.
  decode::list_rows(p, rows, 16 * NT);
  const int total = before[p.rows] * H, step = gridDim.x * (blockDim.x / 32);
  bool waited = false;
  for (int x = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); x < total; x += step) {
    decode::Place at;
    at.find(p, rows, 1, x);
    const int first = (before[at.row] * H + at.kvh * at.tiles) * hgroups + at.tile;
    // The slot of the key that lane (g, t) will add to, and its weight.
    const int n = at.lo + at.tile * 16 * NT + 8 * (g >> 1) + 2 * t + (g & 1);
    int64_t slot = -1;
    if (g < 4 * NT && n < at.len) slot = slot_of(p.c, p.t, at.row, n);
    float* const weight = p.c.weight + slot + static_cast<int64_t>(at.kvh) * p.c.page_size;
    const float old = slot >= 0 ? *weight : 0.0f;
    if (!waited) griddep_wait();
    waited = true;
    float w[4 * NT] = {};
    for (int hg = 0; hg < hgroups; ++hg) {
      const int h = hg * kDecodeHeads + g;
      const int64_t tile = first + hg * at.tiles;
      if (h >= G || tile >= ws.score_tiles) continue;
      const float lse = ws.lse[at.row * p.c.n_heads + at.kvh * G + h];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float4 s = *reinterpret_cast<const float4*>(ws.scores + ((tile * NT + u) * 32 + lane) * 4);
        w[4 * u] += decode::exp_diff(s.x, lse);
        w[4 * u + 1] += decode::exp_diff(s.y, lse);
        w[4 * u + 2] += decode::exp_diff(s.z, lse);
        w[4 * u + 3] += decode::exp_diff(s.w, lse);
      }
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) w[i] += __shfl_xor_sync(0xFFFFFFFFu, w[i], o);
    // w[i] is key 8 (i / 2) + 2t + i % 2; lane (g, t) takes i = g
    float add = w[0];
#pragma unroll
    for (int i = 1; i < 4 * NT; ++i) add = g == i ? w[i] : add;
    if (slot >= 0) *weight = old + add;
  }
  if (!waited) griddep_wait();
  griddep_launch_dependents();
}

}  // namespace

int decode_tile(const PagedView& c) {
  const int es = c.dtype == MXMOE_F32 ? 4 : c.dtype == MXMOE_BF16 ? 2 : 1;
  return 16 * decode::tile_halves(padded_head(c) * es);
}

// Two for each range of the tile list: one range for each warp, and twice as
// many, and one more, of those kept back.
size_t decode_part_floats(const PagedView& c, int sms) {
  return static_cast<size_t>(2) * (3 * sms * warps_of(c) + 1) * kDecodeHeads * (padded_head(c) + 2);
}

int decode_rows_at_once(const PagedView& c, int max_pages) {
  const int G = c.n_heads / c.kv_heads, segs = c.kv_heads * ((G + kDecodeHeads - 1) / kDecodeHeads);
  const int64_t most = (static_cast<int64_t>(max_pages) * c.page_size / decode_tile(c) + 1) * segs;
  return static_cast<int>(std::min<int64_t>(kDecodeMaxRows, INT32_MAX / most));
}

cudaError_t launch_paged_decode(const DecodeParams& all, const DecodeScratch& ws, int sms, cudaStream_t st) {
  const int64_t longest = std::min<int64_t>(static_cast<int64_t>(all.t.max_pages) * all.c.page_size, all.window ? all.window : INT32_MAX);
  const DecodePlan plan{sms, longest <= kWholeTiles * decode_tile(all.c)};
  const int chunk = decode_rows_at_once(all.c, all.t.max_pages);
  if (chunk < 1) return cudaErrorInvalidValue;
  for (int r0 = 0; r0 < all.rows; r0 += chunk) {
    DecodeParams p = all;
    const int act = all.q_dtype == MXMOE_F32 ? 4 : 2, oact = all.out_dtype == MXMOE_F32 ? 4 : 2;
    p.rows = std::min(chunk, all.rows - r0);
    p.q = static_cast<const char*>(all.q) + r0 * all.q_row * act;
    p.out = static_cast<char*>(all.out) + r0 * all.out_row * oact;
    p.lens += r0;
    p.t.tables += r0 * all.t.stride;
    p.t.n_rows = p.rows;
    if (p.lse) p.lse += static_cast<int64_t>(r0) * all.c.n_heads;
    if (p.bias) p.bias += r0 * all.bias_row;
    // 32-bit queries or outputs keep 22 bits and more of queries and shares
    const bool x32 = p.q_dtype == MXMOE_F32 || p.out_dtype == MXMOE_F32;
    const auto attend = p.c.dtype == MXMOE_F32    ? launch_attend_f32
                        : p.c.dtype == MXMOE_BF16 ? (x32 ? launch_attend_bf16_x32 : launch_attend_bf16)
                                                  : (x32 ? launch_attend_e4m3_x32 : launch_attend_e4m3);
    const cudaError_t e = attend(p, ws, plan, st);
    if (e != cudaSuccess) return e;
    if (!p.track) continue;
    const cudaError_t f = launch_kernel(decode_tile(p.c) == 32 ? weigh_kernel<2> : weigh_kernel<1>, dim3(8 * sms), dim3(256), 0, st, p, ws);
    if (f != cudaSuccess) return f;
  }
  return cudaSuccess;
}

}  // namespace mxmoe
