// paged.h -- what the paged key-value cache's entry points (paged_api.cu) and
// kernels (paged_append.cu, paged_decode.cu, paged_evict.cu) share.
//
// Keys and values lie in pools [n_pages][kv_heads][page_size][head_dim]; the
// cache index n of a sequence is slot n % page_size of the page that its table
// row names at n / page_size.  Every kernel checks table entries, indexes and
// positions against these bounds before it forms an address: what is out of
// range is skipped (a read gives zero) and leaves its bit in the status word.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace mxmoe {

// Bits of the cache's status word.
constexpr int kPagedBadPage = 1;      // a table entry outside [0, n_pages)
constexpr int kPagedBadIndex = 2;     // a cache index, length or row outside its table
constexpr int kPagedBadPosition = 4;  // a position outside the rotary table

struct PagedView {
  void* k;
  void* v;
  const float* k_scale;  // [kv_heads] (8-bit cache) or null: 1
  const float* v_scale;
  float* weight;      // [n_pages][kv_heads][page_size] or null
  int32_t* position;  // the same shape, or null
  int* status;
  int n_pages, page_size, n_heads, kv_heads, head_dim, dtype;
  uint32_t page_mul, page_shift;  // n / page_size = umulhi(n, page_mul) >> page_shift for 0 <= n < 2^31
};

struct PagedTables {
  const int32_t* tables;  // [n_rows][max_pages], rows `stride` apart
  int64_t stride;
  int n_rows, max_pages;
};

struct AppendParams {
  PagedView c;
  PagedTables t;
  const void *q, *k, *v;  // [tokens][heads][head_dim], strides in elements
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  void *q_out, *k_out;
  int64_t qo_token, qo_head, ko_token, ko_head;
  int dtype, tokens;
  const int32_t *rows, *index, *positions;
  const float *cos, *sin;  // [n_positions][rot / 2]
  int rot, n_positions, interleaved;
  float sign;  // -1: the inverse rotation
};

struct DecodeParams {
  PagedView c;
  PagedTables t;
  const void* q;
  int64_t q_row, q_head;
  int q_dtype;
  int q_wide;  // four columns of q can be loaded at once
  void* out;
  int64_t out_row, out_head;
  int out_dtype;
  int out_wide;  // two bf16 columns of out can be stored at once
  float* lse;  // [rows][n_heads] or null
  int rows;
  const int32_t* lens;
  float scale;
  int window;
  const float* sinks;
  int quiet;
  const float* bias;  // [rows][n_heads][bias_len] by strides, or null
  int64_t bias_row, bias_head;
  int bias_len;
  int track;
};

struct EvictParams {
  PagedView c;
  PagedTables t;
  int rows;
  const int32_t *lens, *seen;
  int32_t* new_lens;
  int budget, sink, recent;
};

constexpr int kDecodeMaxRows = 512;   // rows per launch: their prefix sums lie in shared memory
constexpr int kDecodeHeads = 8;       // query heads of a segment
constexpr int kDecodeWarps = 8;       // of a block, at most

// Device memory that decode needs beside its arguments.
struct DecodeScratch {
  float* part;    // [2 * ranges][8 * (padded head_dim + 2)] partial outputs, maxima and sums
  int2* held;     // [kDecodeMaxRows][segments] the first and last range that a segment falls to
  int* taken;     // [2] ranges taken, warps that have left; zero between calls
  float* scores;  // [score_tiles][tile / 16][32 lanes][4] (track)
  int64_t score_tiles;
  float* lse;  // [kDecodeMaxRows][n_heads] (track)
};

cudaError_t launch_paged_append(const AppendParams& p, int sms, cudaStream_t st);
cudaError_t launch_paged_decode(const DecodeParams& p, const DecodeScratch& ws, int sms, cudaStream_t st);
int decode_tile(const PagedView& c);                     // keys of a tile
// Rows of one launch, whose tiles are numbered in 32 bits; 0: not even one under a table that wide.
int decode_rows_at_once(const PagedView& c, int max_pages);
size_t decode_part_floats(const PagedView& c, int sms);  // of DecodeScratch::part
inline bool apart(const int32_t* a, const int32_t* b, int64_t n) {  // two arrays of n
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), bytes = static_cast<uintptr_t>(n) * 4;
  return x + bytes <= y || y + bytes <= x;
}
cudaError_t launch_paged_evict(const EvictParams& p, int sms, cudaStream_t st);
cudaError_t launch_rotary_table(const double* inv_freq, int half, int64_t first, int n, double factor, float* cos,
                                float* sin, cudaStream_t st);

#ifdef __CUDACC__
__device__ __forceinline__ int page_of(const PagedView& c, int n) {
  return c.page_mul ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), c.page_mul) >> c.page_shift) : n;
}

// The slot of cache index n of a table row: (page * kv_heads + 0) * page_size + n % page_size, head h's is
// page_size * h further.  -1 where the table has none; its bit joins `bad`.
__device__ __forceinline__ int64_t slot_of(const PagedView& c, const PagedTables& t, int row, int n, int& bad) {
  const int pi = page_of(c, n);
  const bool in = n >= 0 && pi < t.max_pages;
  const int page = in ? __ldg(t.tables + row * t.stride + pi) : 0;
  const bool ok = page >= 0 && page < c.n_pages;
  bad |= !in ? kPagedBadIndex : !ok ? kPagedBadPage : 0;
  return in && ok ? static_cast<int64_t>(page) * c.kv_heads * c.page_size + (n - pi * c.page_size) : -1;
}
// The same, its bit set in the status word at once.
__device__ __forceinline__ int64_t slot_of(const PagedView& c, const PagedTables& t, int row, int n) {
  int bad = 0;
  const int64_t s = slot_of(c, t, row, n, bad);
  if (bad) atomicOr(c.status, bad);
  return s;
}
#endif

}  // namespace mxmoe
