// The host side of the key/value cache's calls, with no device: this program stands in for the runtime's functions and notes what the
// library asks of them and on which device.  `kv_host_calls <case>` exits with 0 when that is right.
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "tpuhip.h"

namespace {
struct Note {
  std::string what;
  int device;
  size_t size;                 // bytes, or workgroups
};
std::vector<Note> notes;
int current = 0;
bool capturing = false;
dim3 grid, block;
void note(const char *what, size_t size = 0) { notes.push_back({what, current, size}); }
size_t count(const char *what) {
  size_t n = 0;
  for (auto &x : notes) n += x.what == what;
  return n;
}
}  // namespace

extern "C" {
hipError_t hipGetDeviceCount(int *n) { return *n = 2, hipSuccess; }
hipError_t hipSetDevice(int d) { return current = d, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *s) { return *p = const_cast<void *>(s), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { return *s = (hipStream_t)malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return free((void *)s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return note("wait"), hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  return *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes) { return note("malloc", bytes), *p = malloc(16), hipSuccess; }
hipError_t hipFree(void *p) { return note("free"), free(p), hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t bytes, hipStream_t) { return note("memset", bytes), hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return grid = g, block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *shared, hipStream_t *s) {
  return *g = grid, *b = block, *shared = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3 g, dim3 b, void **, size_t, hipStream_t) {
  if ((uint64_t)g.x * b.x > UINT32_MAX || g.y > 65535) return hipErrorInvalidValue;
  return note("launch", (size_t)g.x * g.y), hipSuccess;
}
}

namespace {
void expect(bool held, const char *what) {
  if (!held) throw std::runtime_error(what);
}
void check(int status) {
  if (status != TPUHIP_OK) throw std::runtime_error(tpuhip_last_error());
}

struct Cache {
  tpuhip_ctx *ctx = nullptr;
  tpuhip_kv_cache *cache = nullptr;
  explicit Cache(int device, int kv_heads = 2, int dim = 64, int pages = 64) {
    check(tpuhip_ctx_create(device, &ctx));
    const tpuhip_kv_desc d = {pages, 32, kv_heads, dim, 4};
    check(tpuhip_kv_cache_create(ctx, &d, &cache));
  }
  ~Cache() {
    tpuhip_kv_cache_destroy(ctx, cache);
    tpuhip_ctx_destroy(ctx);
  }
};

tpuhip_kv_attention_desc attention(int n_seq, int heads, int total, int max_q, int max_kv, int dim) {
  return {n_seq, heads, TPUHIP_BF16, total, max_q, max_kv, 0, 0, 1 << 20, 1.0f, (int64_t)heads * dim, dim, (int64_t)heads * dim, dim};
}
int attend(tpuhip_ctx *ctx, const tpuhip_kv_cache *cache, const tpuhip_kv_attention_desc &d, bool table = true) {
  static int32_t there[4];
  static uint16_t q, out;
  return tpuhip_kv_attention(ctx, cache, &d, &q, &out, there, there, table ? there : nullptr);
}

// no tokens at all: a launch that writes zeros, in every form of the kernel
void no_tokens() {
  for (int dim : {64, 128, 192, 256})
    for (int q : {1, 5, 16, 40, 400, 20000}) {
      Cache c(0, 2, dim);
      notes.clear();
      check(attend(c.ctx, c.cache, attention(3, 4, 3 * q, q, 0, dim), q % 2));
      expect(count("launch") == 1, "not one launch");
    }
}

// a context's first attention to another one's cache, on a thread where another device is current: its workspace is its device's
void workspace_device() {
  Cache c(1);
  tpuhip_ctx *other = nullptr;
  check(tpuhip_ctx_create(1, &other));
  (void)hipSetDevice(0);
  notes.clear();
  check(attend(other, c.cache, attention(1, 4, 1, 1, 4096, 64)));
  expect(count("malloc") == 1 && count("memset") == 1 && count("launch") >= 1, "no splits");
  (void)hipSetDevice(0);
  static uint16_t k, v;
  static int32_t slot;
  const tpuhip_kv_rows rows = {1, TPUHIP_BF16, &k, &v, 128, 64, 128, 64};
  check(tpuhip_kv_write(other, c.cache, &rows, &slot));
  (void)hipSetDevice(0);
  check(tpuhip_kv_read(other, c.cache, &rows, &slot));
  for (auto &n : notes) expect(n.device == 1, n.what.c_str());
  check(tpuhip_ctx_destroy(other));
}

// a cache that has been made can be used from any context: its pages are clear
void pages_are_clear() {
  tpuhip_ctx *ctx = nullptr;
  check(tpuhip_ctx_create(0, &ctx));
  notes.clear();
  const tpuhip_kv_desc d = {4, 32, 2, 64, 4};
  tpuhip_kv_cache *cache = nullptr;
  check(tpuhip_kv_cache_create(ctx, &d, &cache));
  size_t cleared = 0, waited = 0;
  for (size_t i = 0; i < notes.size(); ++i) {
    if (notes[i].what == "launch") cleared = i + 1;
    if (notes[i].what == "wait") waited = i + 1;
  }
  expect(cleared && waited > cleared, "the call returned before its pages were clear");
  check(tpuhip_kv_cache_destroy(ctx, cache));
  check(tpuhip_ctx_destroy(ctx));
}

// many rows in one call: only those are refused that the launches cannot hold, and only for a launch that is made
void many_rows() {
  struct {
    int n_seq, heads, max_q, max_kv, kv_heads, dim;
  } const calls[] = {{1, 71, 60000, 60000, 1, 64},   {1, 64, 65536, 65536, 1, 64},   {1, 64, 1 << 20, 1 << 20, 1, 128},
                     {50000, 64, 40, 40, 1, 128},    {40000, 32, 64, 4096, 8, 64},   {60000, 8, 300, 300, 1, 256},
                     {65535, 8, 1, 131072, 8, 64},   {65535, 256, 1, 64, 256, 64}};
  for (auto &x : calls) {
    Cache c(0, x.kv_heads, x.dim);
    notes.clear();
    check(attend(c.ctx, c.cache, attention(x.n_seq, x.heads, x.n_seq * x.max_q, x.max_q, x.max_kv, x.dim)));
    expect(count("launch") == 1, "not one launch");
  }
  Cache c(0, 2048, 64);
  expect(attend(c.ctx, c.cache, attention(65535, 2048, 65535, 1, 64, 64)) == TPUHIP_ERR_INVALID, "2^27 tiles were not refused");
  // few queries and long contexts: split, and joined by the last workgroups or by a launch
  for (int max_kv : {4096, 1 << 20}) {
    notes.clear();
    check(attend(c.ctx, c.cache, attention(1, 2048, 1, 1, max_kv, 64)));
    expect(count("launch") >= 1, "no launch");
  }
  Cache few(0, 2, 64);
  notes.clear();
  check(attend(few.ctx, few.cache, attention(1, 4, 1, 1, 1 << 20, 64)));
  expect(count("launch") == 2, "many splits are joined by a launch");
  notes.clear();
  check(attend(few.ctx, few.cache, attention(65535, 4, 1, 1, 1 << 20, 64)));   // all but one of them without a query
}

// while the context's stream is being recorded, a cache is neither made nor freed, and the recording is not touched; calls are recorded, and
// take no memory
void recording() {
  Cache c(0);
  tpuhip_ctx *fresh = nullptr;
  check(tpuhip_ctx_create(0, &fresh));
  capturing = true;
  notes.clear();
  const tpuhip_kv_desc d = {4, 32, 2, 64, 4};
  tpuhip_kv_cache *other = nullptr;
  expect(tpuhip_kv_cache_create(c.ctx, &d, &other) == TPUHIP_ERR_INVALID && !other, "a cache was made");
  expect(tpuhip_kv_cache_destroy(c.ctx, c.cache) == TPUHIP_ERR_INVALID, "a cache was freed");
  expect(notes.empty(), "the runtime was asked for something");
  check(attend(c.ctx, c.cache, attention(1, 4, 1, 1, 4096, 64)));
  check(attend(fresh, c.cache, attention(1, 4, 1, 1, 4096, 64)));
  expect(count("launch") == notes.size(), "more than launches");
  capturing = false;
  check(tpuhip_ctx_destroy(fresh));
}
}  // namespace

int main(int argc, char **argv) {
  const struct {
    const char *name;
    std::function<void()> run;
  } cases[] = {{"no_tokens", no_tokens}, {"workspace_device", workspace_device}, {"pages_are_clear", pages_are_clear}, {"many_rows", many_rows}, {"recording", recording}};
  try {
    for (auto &c : cases)
      if (argc == 2 && !strcmp(argv[1], c.name)) {
        c.run();
        return 0;
      }
    throw std::runtime_error("no such case");
  } catch (const std::exception &e) {
    fprintf(stderr, "%s\n", e.what());
    return 1;
  }
}
