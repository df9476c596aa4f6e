// paged_api.cu -- C entry points of the paged key-value cache: argument
// checks, the cache handle and its status word.  Kernels in paged_append.cu,
// paged_decode.cu and paged_evict.cu.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

#include "../../include/mxmoe.h"
#include "launch_util.h"
#include "paged.h"

namespace mxmoe {
int set_last_error(int code, const char* msg);  // api.cu
}

struct mxmqa_paged_cache {
  mxmqa_paged_config cfg{};
  mxmoe::PagedView view{};
  mxmoe::DecodeScratch scratch{};
  void* workspace = nullptr;
  int sms = 148;
};

namespace {

int pfail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return mxmoe::set_last_error(code, buf);
}

#define P_CUDA(expr)                                                                              \
  do {                                                                                            \
    const cudaError_t e_ = (expr);                                                                \
    if (e_ != cudaSuccess) return pfail(MXMOE_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)
#define P_CHECK(cond, ...)                                        \
  do {                                                            \
    if (!(cond)) return pfail(MXMOE_ERR_INVALID_ARG, __VA_ARGS__); \
  } while (0)

struct PDevice {
  int prev = -1;
  explicit PDevice(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
    else prev = -1;
  }
  ~PDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

constexpr uint64_t kMaxTokens = 0x7FFFFFFFu;
constexpr uint64_t kMaxIndexes = (1u << 31) - 1024;  // of a row: kernels walk them in 32 bits, up to 1024 at a step

bool act_dtype(int d) { return d == MXMOE_F32 || d == MXMOE_BF16; }
size_t elem_bytes(int d) { return d == MXMOE_F32 ? 4 : d == MXMOE_BF16 ? 2 : 1; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The tables of a call, and that cache indexes of a row stay a step below 2^31.
int check_tables(const mxmqa_paged_cache* c, const int32_t* tables, int64_t stride, uint32_t rows, uint32_t max_pages,
                 mxmoe::PagedTables& t) {
  P_CHECK(tables != nullptr, "null tables");
  P_CHECK(aligned(tables, 4), "tables must be 4-byte aligned");
  P_CHECK(rows > 0 && rows <= 65535, "rows must be 1 to 65535");
  P_CHECK(max_pages > 0 && static_cast<uint64_t>(max_pages) * c->cfg.page_size <= kMaxIndexes,
          "max_pages x page_size must be 1 to 2^31 - 1024");
  t.tables = tables;
  t.stride = stride;
  t.n_rows = static_cast<int>(rows);
  t.max_pages = static_cast<int>(max_pages);
  return MXMOE_OK;
}

// Zeros device memory and waits for that on a stream of its own: a memset
// returns before it is done, and the caller's streams need not wait for the
// legacy stream, nor this call for what is queued there.
cudaError_t zero_now(void* p, size_t n) {
  cudaStream_t st = nullptr;
  cudaError_t e = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
  if (e != cudaSuccess) return e;
  e = cudaMemsetAsync(p, 0, n, st);
  const cudaError_t f = cudaStreamSynchronize(st);
  cudaStreamDestroy(st);
  return e != cudaSuccess ? e : f;
}

// The inverse frequencies of one rotary table in 64 bits.
int rotary_frequencies(const mxmqa_rotary_config* r, std::vector<double>& f, double& factor) {
  const int half = static_cast<int>(r->rot_dim) / 2;
  const double base0 = r->theta, s = r->scaling_factor;
  const double two_pi = 6.283185307179586476925286766559;
  double base = base0;
  factor = 1.0;
  if (r->scaling == MXMQA_ROTARY_NTK && half > 1) base = base0 * std::pow(s, half / (half - 1.0));
  f.resize(half);
  for (int i = 0; i < half; ++i) f[i] = std::pow(base, -static_cast<double>(i) / half);
  if (r->scaling == MXMQA_ROTARY_LINEAR)
    for (double& x : f) x /= s;
  if (r->scaling == MXMQA_ROTARY_YARN && s > 1.0) {
    // pairs that turn more than ntk_beta times within the first context keep
    // their frequency, those below ntk_alpha turns are interpolated
    const double low = half * std::log(r->initial_context / (r->ntk_beta * two_pi)) / std::log(base0);
    const double high = half * std::log(r->initial_context / (r->ntk_alpha * two_pi)) / std::log(base0);
    for (int i = 0; i < half; ++i) {
      const double ramp = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 1e-3)));
      f[i] = f[i] / s * ramp + f[i] * (1.0 - ramp);
    }
    factor = 0.1 * std::log(s) + 1.0;
  }
  if (r->scaling == MXMQA_ROTARY_STREAMING && s > 1.0) {
    // the interpolation of mxmqa_set_rope (src/rope/mod.rs:11-50): the factor
    // divides the high frequencies
    const double d = 4.0 * half, dh = d / 2.0, lb = std::log(base0);
    const double low = dh * std::log(r->initial_context / (r->ntk_beta * two_pi)) / lb;
    const double high = dh * std::log(r->initial_context / (r->ntk_alpha * two_pi)) / lb;
    if (!(low > 0.0 && high > 0.0 && low < high && high < dh - 1.0))
      return pfail(MXMOE_ERR_INVALID_ARG, "NTK/YaRN thresholds out of range (low %g, high %g)", low, high);
    for (double& x : f) {
      const double idx = std::log(x) * (-d / 2.0 / lb);
      const double ramp = std::min(1.0, std::max(0.0, (idx - low) / (high - low)));
      x = x / s * (1.0 - ramp) + x * ramp;
    }
    factor = 0.1 * std::log(s) + 1.0;
  }
  return MXMOE_OK;
}

int check_rotary(const float* cos, const float* sin, uint32_t rot_dim, uint32_t n_positions, uint32_t head_dim) {
  P_CHECK(rot_dim % 2 == 0 && rot_dim <= head_dim, "rot_dim must be even and at most head_dim");
  if (rot_dim == 0) return MXMOE_OK;
  P_CHECK(cos && sin && aligned(cos, 16) && aligned(sin, 16), "the rotary table must be given, 16-byte aligned");
  P_CHECK(n_positions > 0 && n_positions <= kMaxTokens, "an empty rotary table");
  return MXMOE_OK;
}

}  // namespace

extern "C" {

int mxmqa_paged_create(const mxmqa_paged_config* cfg, const mxmqa_paged_buffers* buf, mxmqa_paged_cache** out) {
  P_CHECK(cfg && buf && out, "null argument");
  *out = nullptr;
  P_CHECK(cfg->n_pages > 0 && cfg->page_size > 0 && cfg->n_heads > 0 && cfg->kv_heads > 0 && cfg->head_dim > 0,
          "zero dimension");
  P_CHECK(cfg->n_heads % cfg->kv_heads == 0, "n_heads must be divisible by kv_heads");
  P_CHECK(cfg->dtype == MXMOE_F32 || cfg->dtype == MXMOE_BF16 || cfg->dtype == MXMOE_E4M3, "bad cache dtype");
  P_CHECK(buf->k && buf->v, "null k or v");
  P_CHECK(aligned(buf->k, 16) && aligned(buf->v, 16), "k and v must be 16-byte aligned");
  P_CHECK(aligned(buf->weight, 4) && aligned(buf->position, 4) && aligned(buf->k_scale, 4) && aligned(buf->v_scale, 4),
          "weight, position and scales must be 4-byte aligned");
  if (cfg->n_pages > kMaxTokens || cfg->page_size > 65536 || cfg->n_heads > 1024 || cfg->head_dim > 256 ||
      cfg->head_dim % (cfg->dtype == MXMOE_E4M3 ? 16 : 8) != 0)
    return pfail(MXMOE_ERR_UNSUPPORTED,
                 "head_dim must be a multiple of 8 (16 in an 8-bit cache) and at most 256, page_size at most 65536, "
                 "n_heads at most 1024");
  P_CHECK(cfg->dtype == MXMOE_E4M3 || (!buf->k_scale && !buf->v_scale), "scales are for the 8-bit cache");
  if (static_cast<uint64_t>(cfg->n_pages) * cfg->page_size > kMaxTokens / cfg->kv_heads)
    return pfail(MXMOE_ERR_UNSUPPORTED, "n_pages x page_size x kv_heads must be below 2^31");
  mxmqa_paged_cache* c = new (std::nothrow) mxmqa_paged_cache();
  if (!c) return pfail(MXMOE_ERR_OOM, "host allocation failed");
  c->cfg = *cfg;
  mxmoe::PagedView& w = c->view;
  w.k = buf->k;
  w.v = buf->v;
  w.k_scale = buf->k_scale;
  w.v_scale = buf->v_scale;
  w.weight = buf->weight;
  w.position = buf->position;
  w.n_pages = static_cast<int>(cfg->n_pages);
  w.page_size = static_cast<int>(cfg->page_size);
  w.n_heads = static_cast<int>(cfg->n_heads);
  w.kv_heads = static_cast<int>(cfg->kv_heads);
  w.head_dim = static_cast<int>(cfg->head_dim);
  w.dtype = static_cast<int>(cfg->dtype);
  // n / d for n < 2^31 by a product: with 2^(l-1) < d <= 2^l and
  // m = floor(2^(31+l) / d) + 1 the error n (m d - 2^(31+l)) < 2^31 d stays
  // below 2^(31+l), so floor(n m / 2^(31+l)) = floor(n / d).
  if (cfg->page_size > 1) {
    uint32_t l = 1;
    while ((1u << l) < cfg->page_size) ++l;
    w.page_mul = static_cast<uint32_t>((1ull << (31 + l)) / cfg->page_size + 1);
    w.page_shift = l - 1;
  }
  PDevice g(cfg->device);
  if (cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, cfg->device) != cudaSuccess || c->sms < 1) {
    cudaGetLastError();
    delete c;
    return pfail(MXMOE_ERR_CUDA, "device %d is not available", cfg->device);
  }
  // Everything that the calls need is allocated here, once and in one piece: a
  // tracked decode keeps the scores of every cached token (32 bytes per token,
  // key head and 8 query heads).
  mxmoe::DecodeScratch& ws = c->scratch;
  const size_t group = cfg->n_heads / cfg->kv_heads, segs = cfg->kv_heads * ((group + mxmoe::kDecodeHeads - 1) / mxmoe::kDecodeHeads);
  const size_t tile = mxmoe::decode_tile(w);
  if (w.weight)
    ws.score_tiles = static_cast<int64_t>((static_cast<uint64_t>(cfg->n_pages) * cfg->page_size / tile + mxmoe::kDecodeMaxRows) * segs);
  size_t bytes = 0;
  auto room = [&bytes](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  const size_t head = room(3 * sizeof(int)), held = room(mxmoe::kDecodeMaxRows * segs * sizeof(int2));
  const size_t part = room(mxmoe::decode_part_floats(w, c->sms) * sizeof(float));
  const size_t lse = room(w.weight ? mxmoe::kDecodeMaxRows * cfg->n_heads * sizeof(float) : 0);
  const size_t scores = room(static_cast<size_t>(ws.score_tiles) * tile * 8 * sizeof(float));
  char* base = nullptr;
  int rc = MXMOE_OK;
  const cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&base), bytes);
  if (e != cudaSuccess) {
    rc = pfail(MXMOE_ERR_OOM, "cudaMalloc(%zu bytes): %s", bytes, cudaGetErrorString(e));
  } else if (const cudaError_t z = zero_now(base + head, 3 * sizeof(int)); z != cudaSuccess) {
    cudaFree(base);
    rc = pfail(MXMOE_ERR_CUDA, "zeroing the workspace: %s", cudaGetErrorString(z));
  }
  if (rc != MXMOE_OK) {
    cudaGetLastError();
    delete c;
    return rc;
  }
  c->workspace = base;
  w.status = reinterpret_cast<int*>(base + head);
  ws.taken = w.status + 1;
  ws.held = reinterpret_cast<int2*>(base + held);
  ws.part = reinterpret_cast<float*>(base + part);
  ws.lse = reinterpret_cast<float*>(base + lse);
  ws.scores = reinterpret_cast<float*>(base + scores);
  *out = c;
  return MXMOE_OK;
}

int mxmqa_paged_destroy(mxmqa_paged_cache* c) {
  if (!c) return MXMOE_OK;
  PDevice g(c->cfg.device);
  cudaFree(c->workspace);
  delete c;
  return MXMOE_OK;
}

int mxmqa_paged_status(mxmqa_paged_cache* c, void* stream) {
  P_CHECK(c, "null cache");
  PDevice g(c->cfg.device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int bits = 0;
  P_CUDA(cudaMemcpyAsync(&bits, c->view.status, sizeof(int), cudaMemcpyDeviceToHost, st));
  P_CUDA(cudaMemsetAsync(c->view.status, 0, sizeof(int), st));
  P_CUDA(cudaStreamSynchronize(st));
  if (bits == 0) return MXMOE_OK;
  return pfail(MXMOE_ERR_INVALID_ARG, "%s%s%sthe entries concerned were skipped",
               bits & mxmoe::kPagedBadPage ? "a table entry is outside the pool; " : "",
               bits & mxmoe::kPagedBadIndex ? "a row, length or cache index is outside its table; " : "",
               bits & mxmoe::kPagedBadPosition ? "a position is outside the rotary table; " : "");
}

int mxmqa_paged_append(mxmqa_paged_cache* c, const mxmqa_paged_append_args* a, void* stream) {
  P_CHECK(c && a, "null argument");
  P_CHECK(act_dtype(a->dtype), "bad dtype");
  P_CHECK(a->tokens <= 1u << 30, "more than 2^30 tokens");
  if (a->tokens == 0) return MXMOE_OK;
  P_CHECK(a->k && a->v && a->index, "null k, v or index");
  P_CHECK((a->q == nullptr) == (a->q_out == nullptr), "q and q_out go together");
  const size_t es = elem_bytes(a->dtype);
  P_CHECK(aligned(a->q, es) && aligned(a->k, es) && aligned(a->v, es) && aligned(a->q_out, es) && aligned(a->k_out, es),
          "q, k, v and the outputs must be aligned to their element");
  P_CHECK(aligned(a->rows, 4) && aligned(a->index, 4) && aligned(a->positions, 4),
          "rows, index and positions must be 4-byte aligned");
  if (const int rc = check_rotary(a->cos, a->sin, a->rot_dim, a->n_positions, c->cfg.head_dim)) return rc;
  mxmoe::AppendParams p{};
  if (const int rc = check_tables(c, a->tables, a->table_stride, a->n_rows, a->max_pages, p.t)) return rc;
  P_CHECK(a->rows || a->tokens == a->n_rows, "%u tokens for %u table rows need `rows`", a->tokens, a->n_rows);
  p.c = c->view;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.qo_token = a->q_out_token;
  p.qo_head = a->q_out_head;
  p.ko_token = a->k_out_token;
  p.ko_head = a->k_out_head;
  p.dtype = static_cast<int>(a->dtype);
  p.tokens = static_cast<int>(a->tokens);
  p.rows = a->rows;
  p.index = a->index;
  p.positions = a->positions;
  p.cos = a->cos;
  p.sin = a->sin;
  p.rot = static_cast<int>(a->rot_dim);
  p.n_positions = static_cast<int>(a->n_positions);
  p.interleaved = a->interleaved ? 1 : 0;
  p.sign = 1.0f;
  PDevice g(c->cfg.device);
  mxmoe::PdlScope pdl(true);  // every kernel waits for the one before it in the stream
  P_CUDA(mxmoe::launch_paged_append(p, c->sms, static_cast<cudaStream_t>(stream)));
  return MXMOE_OK;
}

int mxmqa_paged_decode(mxmqa_paged_cache* c, const mxmqa_paged_decode_args* a, void* stream) {
  P_CHECK(c && a, "null argument");
  P_CHECK(act_dtype(a->q_dtype) && act_dtype(a->out_dtype), "bad dtype");
  if (a->rows == 0) return MXMOE_OK;
  P_CHECK(a->q && a->out && a->lens, "null q, out or lens");
  P_CHECK(aligned(a->q, elem_bytes(a->q_dtype)) && aligned(a->out, elem_bytes(a->out_dtype)),
          "q and out must be aligned to their element");
  P_CHECK(aligned(a->lens, 4) && aligned(a->sinks, 4) && aligned(a->bias, 4) && aligned(a->lse, 4),
          "lens, sinks, bias and lse must be 4-byte aligned");
  P_CHECK(std::isfinite(a->scale), "the scale must be finite");
  P_CHECK(a->window <= kMaxTokens && a->bias_len <= kMaxTokens, "window or bias_len above 2^31 - 1");
  P_CHECK(!a->track || c->view.weight, "track needs a cache with a weight buffer");
  P_CHECK(!a->track || a->window == 0, "a tracked cache attends in full: window must be 0");
  mxmoe::DecodeParams p{};
  if (const int rc = check_tables(c, a->tables, a->table_stride, a->rows, a->max_pages, p.t)) return rc;
  if (static_cast<uint64_t>(a->max_pages) * c->cfg.page_size * c->cfg.n_heads > 16ull * kMaxTokens)
    return pfail(MXMOE_ERR_UNSUPPORTED, "max_pages x page_size x n_heads must be below 2^35");
  if (mxmoe::decode_rows_at_once(c->view, p.t.max_pages) < 1)
    return pfail(MXMOE_ERR_UNSUPPORTED,
                 "max_pages too large: (max_pages x page_size / %d + 1) x kv_heads x (query heads per key head / 8, rounded up) must be below 2^31",
                 mxmoe::decode_tile(c->view));
  p.c = c->view;
  p.q = a->q;
  p.q_row = a->q_row;
  p.q_head = a->q_head;
  p.q_dtype = static_cast<int>(a->q_dtype);
  p.q_wide = aligned(a->q, 4 * elem_bytes(a->q_dtype)) && a->q_row % 4 == 0 && a->q_head % 4 == 0;
  p.out = a->out;
  p.out_row = a->out_row;
  p.out_head = a->out_head;
  p.out_dtype = static_cast<int>(a->out_dtype);
  p.out_wide = aligned(a->out, 4) && a->out_row % 2 == 0 && a->out_head % 2 == 0;
  p.lse = a->lse;
  p.rows = static_cast<int>(a->rows);
  p.lens = a->lens;
  p.scale = a->scale;
  p.window = static_cast<int>(a->window);
  p.sinks = a->sinks;
  p.quiet = a->quiet ? 1 : 0;
  p.bias = a->bias_len ? a->bias : nullptr;
  p.bias_row = a->bias_row;
  p.bias_head = a->bias_head;
  p.bias_len = static_cast<int>(a->bias_len);
  p.track = a->track ? 1 : 0;
  PDevice g(c->cfg.device);
  mxmoe::PdlScope pdl(true);  // every kernel waits for the one before it in the stream
  P_CUDA(mxmoe::launch_paged_decode(p, c->scratch, c->sms, static_cast<cudaStream_t>(stream)));
  return MXMOE_OK;
}

int mxmqa_paged_evict(mxmqa_paged_cache* c, const mxmqa_paged_evict_args* a, void* stream) {
  P_CHECK(c && a, "null argument");
  if (a->rows == 0) return MXMOE_OK;
  P_CHECK(a->lens && a->seen && a->new_lens, "null lens, seen or new_lens");
  P_CHECK(aligned(a->lens, 4) && aligned(a->seen, 4) && aligned(a->new_lens, 4),
          "lens, seen and new_lens must be 4-byte aligned");
  P_CHECK(a->new_lens == a->lens || mxmoe::apart(a->new_lens, a->lens, a->rows), "new_lens may be lens, but not overlap a part of it");
  P_CHECK(c->view.weight && c->view.position, "evict needs a cache with weight and position buffers");
  P_CHECK(a->budget > 0 && a->budget <= kMaxTokens, "budget must be 1 to 2^31 - 1");
  P_CHECK(static_cast<uint64_t>(a->sink) + a->recent <= a->budget, "sink + recent above the budget");
  mxmoe::EvictParams p{};
  if (const int rc = check_tables(c, a->tables, a->table_stride, a->rows, a->max_pages, p.t)) return rc;
  p.c = c->view;
  p.rows = static_cast<int>(a->rows);
  p.lens = a->lens;
  p.seen = a->seen;
  p.new_lens = a->new_lens;
  p.budget = static_cast<int>(a->budget);
  p.sink = static_cast<int>(a->sink);
  p.recent = static_cast<int>(a->recent);
  PDevice g(c->cfg.device);
  mxmoe::PdlScope pdl(true);  // every kernel waits for the one before it in the stream
  P_CUDA(mxmoe::launch_paged_evict(p, c->sms, static_cast<cudaStream_t>(stream)));
  return MXMOE_OK;
}

int mxmqa_rotary_table(const mxmqa_rotary_config* r, uint32_t first, uint32_t n, float* cos, float* sin, int32_t device,
                       void* stream) {
  P_CHECK(r && cos && sin, "null argument");
  P_CHECK(r->rot_dim > 0 && r->rot_dim % 2 == 0 && r->rot_dim <= 256, "rot_dim must be even, 2 to 256");
  P_CHECK(r->scaling <= MXMQA_ROTARY_STREAMING, "bad scaling");
  P_CHECK(r->theta > 0.0f && std::isfinite(r->theta), "theta must be positive");
  P_CHECK(r->scaling == MXMQA_ROTARY_PLAIN || (r->scaling_factor > 0.0f && std::isfinite(r->scaling_factor)),
          "scaling_factor must be positive");
  if (r->scaling == MXMQA_ROTARY_YARN || r->scaling == MXMQA_ROTARY_STREAMING)
    P_CHECK(r->initial_context > 0.0f && r->ntk_alpha > 0.0f && r->ntk_beta > 0.0f && r->theta != 1.0f,
            "initial_context, ntk_alpha and ntk_beta must be positive, theta not 1");
  P_CHECK(static_cast<uint64_t>(first) + n <= kMaxTokens, "positions above 2^31 - 1");
  if (n == 0) return MXMOE_OK;
  try {
    std::vector<double> f;
    double factor = 1.0;
    if (const int rc = rotary_frequencies(r, f, factor)) return rc;
    PDevice g(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* dev = nullptr;
    if (cudaMalloc(reinterpret_cast<void**>(&dev), f.size() * sizeof(double)) != cudaSuccess) {
      cudaGetLastError();
      return pfail(MXMOE_ERR_OOM, "cudaMalloc(%zu bytes) failed", f.size() * sizeof(double));
    }
    cudaError_t e = cudaMemcpyAsync(dev, f.data(), f.size() * sizeof(double), cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess)
      e = mxmoe::launch_rotary_table(dev, static_cast<int>(f.size()), first, static_cast<int>(n), factor, cos, sin, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    cudaFree(dev);
    if (e != cudaSuccess) return pfail(MXMOE_ERR_CUDA, "rotary table: %s", cudaGetErrorString(e));
  } catch (const std::bad_alloc&) {
    return pfail(MXMOE_ERR_OOM, "host allocation failed");
  }
  return MXMOE_OK;
}

int mxmqa_rotary(const mxmqa_rotary_args* a, void* stream) {
  P_CHECK(a, "null argument");
  P_CHECK(act_dtype(a->dtype), "bad dtype");
  P_CHECK(a->tokens <= 1u << 30 && a->heads <= 65535 && a->head_dim <= 65536, "too many tokens, heads or columns");
  if (a->tokens == 0 || a->heads == 0 || a->head_dim == 0) return MXMOE_OK;
  P_CHECK(a->x && a->out && (a->positions || a->rot_dim == 0), "null x, out or positions");
  const size_t es = elem_bytes(a->dtype);
  P_CHECK(aligned(a->x, es) && aligned(a->out, es) && aligned(a->positions, 4), "x, out or positions misaligned");
  if (const int rc = check_rotary(a->cos, a->sin, a->rot_dim, a->n_positions, a->head_dim)) return rc;
  // a token's pairs and passing columns are numbered in 32 bits, 256 at a step
  if (static_cast<uint64_t>(a->heads) * (a->head_dim - a->rot_dim / 2) > kMaxTokens - 256)
    return pfail(MXMOE_ERR_UNSUPPORTED, "heads x (head_dim - rot_dim / 2) must be below 2^31 - 256");
  mxmoe::AppendParams p{};
  p.c.n_heads = static_cast<int>(a->heads);
  p.c.head_dim = static_cast<int>(a->head_dim);
  p.q = a->x;
  p.q_token = a->x_token;
  p.q_head = a->x_head;
  p.q_out = a->out;
  p.qo_token = a->out_token;
  p.qo_head = a->out_head;
  p.dtype = static_cast<int>(a->dtype);
  p.tokens = static_cast<int>(a->tokens);
  p.positions = a->positions;
  p.cos = a->cos;
  p.sin = a->sin;
  p.rot = static_cast<int>(a->rot_dim);
  p.n_positions = static_cast<int>(a->n_positions);
  p.interleaved = a->interleaved ? 1 : 0;
  p.sign = a->inverse ? -1.0f : 1.0f;
  PDevice g(a->device);
  mxmoe::PdlScope pdl(true);  // every kernel waits for the one before it in the stream
  int sms = 0;
  P_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, a->device));
  P_CUDA(mxmoe::launch_paged_append(p, sms, static_cast<cudaStream_t>(stream)));
  return MXMOE_OK;
}

}  // extern "C"
