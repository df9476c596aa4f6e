// paged_decode.cpp -- the paged key-value cache from C++ (include/mxmoe.hpp):
// one conversation of n tokens enters the cache, its last token attends, and
// the output is compared with dense attention on the host.
//
//   paged_decode [n]            prints the largest distance
//   paged_decode --check-errors exercises argument validation only (no GPU)
#include <cuda_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "mxmoe.hpp"

namespace be = burn_extended;

static void* to_device(const void* host, size_t bytes) {
  void* p = nullptr;
  if (cudaMalloc(&p, bytes) != cudaSuccess) throw std::runtime_error("cudaMalloc failed");
  if (host) cudaMemcpy(p, host, bytes, cudaMemcpyHostToDevice);
  else cudaMemset(p, 0, bytes);
  return p;
}

static int check_errors() {
  int caught = 0;
  alignas(16) static char fake[64];
  const mxmqa_paged_buffers buffers{fake, fake, nullptr, nullptr, nullptr, nullptr};
  for (const mxmqa_paged_config& bad : {mxmqa_paged_config{4, 16, 8, 3, 64, MXMOE_F32, 0},    // heads not divisible
                                        mxmqa_paged_config{4, 0, 8, 2, 64, MXMOE_F32, 0},     // no page size
                                        mxmqa_paged_config{4, 16, 8, 2, 60, MXMOE_F32, 0}}) {  // head_dim
    try {
      be::attention::PagedKvCache cache(bad, buffers);
    } catch (const be::Error& e) {
      ++caught;
      std::printf("caught %d: %s\n", e.status(), e.what());
    }
  }
  std::printf("errors caught: %d\n", caught);
  return caught == 3 ? 0 : 1;
}

static float noise(uint32_t& s) {
  s = s * 1664525u + 1013904223u;
  return static_cast<float>(s >> 8) / 8388608.0f - 1.0f;
}

int main(int argc, char** argv) {
  if (argc > 1 && std::strcmp(argv[1], "--check-errors") == 0) return check_errors();
  const int n = argc > 1 ? std::atoi(argv[1]) : 300;
  const int H = 2, G = 4, nH = H * G, hd = 64, page = 16, pages = (n + page - 1) / page;
  uint32_t seed = 1;
  std::vector<float> q(nH * hd), k(n * H * hd), v(k.size()), out(q.size());
  for (auto* x : {&q, &k, &v})
    for (float& y : *x) y = noise(seed);
  std::vector<int32_t> table(pages), index(n), row(n, 0), len{n};
  for (int i = 0; i < pages; ++i) table[i] = pages - 1 - i;
  for (int i = 0; i < n; ++i) index[i] = i;

  const size_t pool = static_cast<size_t>(pages) * H * page * hd * 4;
  const mxmqa_paged_buffers buffers{to_device(nullptr, pool), to_device(nullptr, pool), nullptr, nullptr, nullptr, nullptr};
  const mxmqa_paged_config cfg{static_cast<uint32_t>(pages), page, nH, H, hd, MXMOE_F32, 0};
  be::attention::PagedKvCache cache(cfg, buffers);

  mxmqa_paged_append_args a{};  // keys and values only, without rotation
  a.k = to_device(k.data(), k.size() * 4);
  a.v = to_device(v.data(), v.size() * 4);
  a.k_token = a.v_token = H * hd;
  a.k_head = a.v_head = hd;
  a.dtype = MXMOE_F32;
  a.tokens = n;
  a.tables = static_cast<int32_t*>(to_device(table.data(), table.size() * 4));
  a.table_stride = a.max_pages = pages;
  a.n_rows = 1;
  a.rows = static_cast<int32_t*>(to_device(row.data(), row.size() * 4));
  a.index = static_cast<int32_t*>(to_device(index.data(), index.size() * 4));
  cache.append(a);

  mxmqa_paged_decode_args d{};
  d.q = to_device(q.data(), q.size() * 4);
  d.out = to_device(nullptr, out.size() * 4);
  d.q_row = d.out_row = nH * hd;
  d.q_head = d.out_head = hd;
  d.q_dtype = d.out_dtype = MXMOE_F32;
  d.rows = 1;
  d.max_pages = pages;
  d.tables = a.tables;
  d.table_stride = pages;
  d.lens = static_cast<int32_t*>(to_device(len.data(), 4));
  d.scale = 0.125f;
  cache.decode(d);
  cache.sync_status();
  cudaMemcpy(out.data(), d.out, out.size() * 4, cudaMemcpyDeviceToHost);

  double far = 0.0;
  for (int h = 0; h < nH; ++h) {
    std::vector<double> p(n), o(hd, 0.0);
    double sum = 0.0;
    for (int i = 0; i < n; ++i) {
      double s = 0.0;
      for (int c = 0; c < hd; ++c) s += static_cast<double>(q[h * hd + c]) * k[(i * H + h / G) * hd + c];
      sum += p[i] = std::exp(s * 0.125);
    }
    for (int i = 0; i < n; ++i)
      for (int c = 0; c < hd; ++c) o[c] += p[i] / sum * v[(i * H + h / G) * hd + c];
    for (int c = 0; c < hd; ++c) far = std::fmax(far, std::fabs(o[c] - out[h * hd + c]));
  }
  std::printf("largest distance from dense attention: %.2e\n", far);
  return far < 3e-5 ? 0 : 1;
}
