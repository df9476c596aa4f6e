#define _GNU_SOURCE
/* A CUDA runtime without a device, preloaded before the library to test its host side: what runs on a
 * stream is only counted, memory comes from the host's heap, and nothing is ever launched. */
#include <dlfcn.h>
#include <stddef.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

enum { kStreams = 64 };
static int pending[kStreams]; /* work handed to a stream that nobody has waited for; 0 is the legacy stream */
static int streams, launches, most_launches = 100000;

int fake_pending(void) {
  int n = 0;
  for (int i = 0; i < kStreams; ++i) n += pending[i];
  return n;
}
int fake_launches(void) { return launches; }

static int no_memory;
void fake_no_memory(int on) { no_memory = on; }
void* _Znwm(size_t n) { /* operator new */
  if (no_memory) ((void (*)(void))dlsym(dlopen("libstdc++.so.6", RTLD_LAZY), "_ZSt17__throw_bad_allocv"))();
  return malloc(n);
}

int cudaGetDevice(int* d) { return *d = 0; }
int cudaSetDevice(int d) { return d ? 101 : 0; }
int cudaDeviceGetAttribute(int* v, int attr, int d) { return *v = 148, 0; }
int cudaGetLastError(void) { return 0; }
const char* cudaGetErrorString(int e) { return "an error of the fake runtime"; }
int cudaMalloc(void** p, size_t n) {
  *p = malloc(n);
  if (*p) memset(*p, 0xA5, n < 4096 ? n : 4096);
  return *p ? 0 : 2;
}
int cudaFree(void* p) { return free(p), 0; }
int cudaFuncSetAttribute(const void* f, int a, int v) { return 0; }
int cudaStreamCreateWithFlags(void** s, unsigned flags) {
  if (++streams == kStreams) abort();
  return *s = (void*)(size_t)streams, 0;
}
int cudaStreamDestroy(void* s) { return 0; } /* does not wait */
int cudaStreamSynchronize(void* s) { return pending[(size_t)s] = 0; }
int cudaDeviceSynchronize(void) { return memset(pending, 0, sizeof pending), 0; }
int cudaMemset(void* p, int v, size_t n) { return ++pending[0], 0; } /* of device memory: not waited for */
int cudaMemsetAsync(void* p, int v, size_t n, void* s) { return ++pending[(size_t)s], 0; }
int cudaMemcpyAsync(void* d, const void* s, size_t n, int kind, void* st) { return ++pending[(size_t)st], 0; }
int cudaLaunchKernelExC(const void* cfg, const void* f, void** args) {
  if (++launches > most_launches) _exit(3); /* a loop that does not end */
  return 0;
}
