// The host side of the calls on microscaled numbers and on a batch's pages, with no device: this program stands in for the runtime's functions and
// notes what the library asks of them and on which device.  `mx_host_calls <case>` exits with 0 when that is right.
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>

#include <climits>
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
bool capturing = false, memory = true;
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
hipError_t hipMalloc(void **p, size_t bytes) {
  if (!memory) return hipErrorOutOfMemory;
  return note("malloc", bytes), *p = malloc(16), hipSuccess;
}
hipError_t hipFree(void *p) { return note("free"), free(p), hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t bytes, hipStream_t) { return note("memset", bytes), hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return grid = g, block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *shared, hipStream_t *s) {
  return *g = grid, *b = block, *shared = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3 g, dim3 b, void **, size_t, hipStream_t) {
  if ((uint64_t)g.x * b.x > UINT32_MAX || g.x == 0 || g.y != 1 || g.z != 1 || b.x > 1024) return hipErrorInvalidValue;
  return note("launch", g.x), hipSuccess;
}
}

namespace {
void expect(bool held, const std::string &what) {
  if (!held) throw std::runtime_error(what + ": " + tpuhip_last_error());
}
void check(int status) {
  if (status != TPUHIP_OK) throw std::runtime_error(tpuhip_last_error());
}

struct Context {
  tpuhip_ctx *ctx = nullptr;
  explicit Context(int device = 0) { check(tpuhip_ctx_create(device, &ctx)); }
  ~Context() { tpuhip_ctx_destroy(ctx); }
  operator tpuhip_ctx *() const { return ctx; }
};

alignas(16) uint8_t there[64];   // nothing is read from where the calls point
tpuhip_mx_matrix matrix(int rows, int cols) {
  const int blocks = cols / 32 + (cols % 32 != 0);
  return {rows, cols, there, there + 1, (int64_t)blocks * 16, blocks};
}
tpuhip_mx_product_desc result(int cols, int dtype = TPUHIP_BF16) { return {dtype, cols, cols, nullptr, nullptr}; }
int product(tpuhip_ctx *c, int rows, int cols, int n) {
  const auto x = matrix(rows, cols), w = matrix(n, cols);
  const auto d = result(n);
  return tpuhip_mx_product(c, &d, &x, &w, there);
}
int linear(tpuhip_ctx *c, int rows, int cols, int n) {
  const auto x = matrix(rows, cols), w = matrix(n, cols);
  const auto d = result(n);
  return tpuhip_mx_linear(c, &d, there, TPUHIP_BF16, cols, &x, &w, there);
}
int32_t ints[8];
tpuhip_kv_pages pages(int n_seq = 4, int count = 16, int tokens = 32, int most = 4) { return {n_seq, count, tokens, most, most, ints, ints, ints, ints}; }

// every argument that a call cannot take is refused, with nothing asked of the runtime's device
void refusals() {
  Context c;
  const auto refused = [&](const char *what, int status, const char *says) {
    expect(status == TPUHIP_ERR_INVALID && strstr(tpuhip_last_error(), says), what);
    for (auto &n : notes) expect(n.what != "launch", what);
  };
  notes.clear();
  auto m = matrix(4, 100);
  refused("no context", tpuhip_mx_quantize(nullptr, &m, there, TPUHIP_F32, 100), "NULL");
  refused("no matrix", tpuhip_mx_quantize(c, nullptr, there, TPUHIP_F32, 100), "NULL");
  refused("no x", tpuhip_mx_quantize(c, &m, nullptr, TPUHIP_F32, 100), "NULL");
  refused("a type", tpuhip_mx_quantize(c, &m, there, 3, 100), "type");
  refused("a type", tpuhip_mx_read(c, &m, there, -1, 100), "type");
  refused("in an element", tpuhip_mx_quantize(c, &m, there + 1, TPUHIP_BF16, 100), "begin");
  refused("in an element", tpuhip_mx_read(c, &m, there + 2, TPUHIP_F32, 100), "begin");
  refused("overlapping rows", tpuhip_mx_read(c, &m, there, TPUHIP_F32, 99), "apart");
  refused("backwards", tpuhip_mx_quantize(c, &m, there, TPUHIP_F32, -1), "apart");
  refused("far apart", tpuhip_mx_quantize(c, &m, there, TPUHIP_F32, INT64_MAX / 4), "apart");
  const struct {
    const char *what;
    std::function<void(tpuhip_mx_matrix &)> change;
    const char *says;
  } changes[] = {
      {"no codes", [](auto &v) { v.codes = nullptr; }, "NULL"},
      {"no scales", [](auto &v) { v.scales = nullptr; }, "NULL"},
      {"codes anywhere", [](auto &v) { v.codes = there + 8; }, "begin"},
      {"codes' stride", [](auto &v) { v.codes_stride = 72; }, "apart"},
      {"codes overlap", [](auto &v) { v.codes_stride = 48; }, "apart"},
      {"codes backwards", [](auto &v) { v.codes_stride = -64; }, "apart"},
      {"scales overlap", [](auto &v) { v.scales_stride = 3; }, "apart"},
      {"scales far apart", [](auto &v) { v.scales_stride = INT64_MAX / 2; }, "apart"},
      {"rows", [](auto &v) { v.rows = -1; }, "rows"},
      {"no columns", [](auto &v) { v.cols = 0; }, "columns"},
      {"wide", [](auto &v) { v.cols = (1 << 24) + 1; }, "columns"},
  };
  const auto w = matrix(7, 100);
  for (auto &x : changes) {
    auto v = m;
    x.change(v);
    refused(x.what, tpuhip_mx_quantize(c, &v, there, TPUHIP_F32, 1 << 25), x.says);
    refused(x.what, tpuhip_mx_read(c, &v, there, TPUHIP_F32, 1 << 25), x.says);
    const auto d = result(7);
    refused(x.what, tpuhip_mx_product(c, &d, &v, &w, there), x.says);
    refused(x.what, tpuhip_mx_linear(c, &d, there, TPUHIP_F32, 100, &v, &w, there), x.says);
    const auto e = result(4);
    refused(x.what, tpuhip_mx_product(c, &e, &w, &v, there), x.says);
  }
  auto d = result(7);
  refused("no desc", tpuhip_mx_product(c, nullptr, &m, &w, there), "NULL");
  refused("no x", tpuhip_mx_product(c, &d, nullptr, &w, there), "NULL");
  refused("no w", tpuhip_mx_product(c, &d, &m, nullptr, there), "NULL");
  refused("no y", tpuhip_mx_product(c, &d, &m, &w, nullptr), "NULL");
  refused("no x", tpuhip_mx_linear(c, &d, nullptr, TPUHIP_F32, 100, &m, &w, there), "NULL");
  refused("x's type", tpuhip_mx_linear(c, &d, there, 7, 100, &m, &w, there), "type");
  const auto other = matrix(7, 132), none = matrix(0, 100);
  refused("columns", tpuhip_mx_product(c, &d, &m, &other, there), "columns");
  refused("no columns of y", tpuhip_mx_product(c, &d, &m, &none, there), "rows");
  auto far = m;
  far.codes_stride = 1 << 24;
  refused("codes far apart", tpuhip_mx_product(c, &d, &far, &w, there), "apart");
  d.dtype = 5;
  refused("y's type", tpuhip_mx_product(c, &d, &m, &w, there), "type");
  d = result(6);
  refused("overlapping rows", tpuhip_mx_product(c, &d, &m, &w, there), "apart");
  d = result(7);
  d.residual = there + 1;
  refused("residual", tpuhip_mx_product(c, &d, &m, &w, there), "residual");
  d.residual = there;
  d.residual_stride = -7;
  refused("residual", tpuhip_mx_product(c, &d, &m, &w, there), "residual");
  d = result(7);
  d.bias = (const float *)(there + 2);
  refused("bias", tpuhip_mx_product(c, &d, &m, &w, there), "bias");
  const auto many = matrix(1 << 30, 64);
  refused("many blocks", tpuhip_mx_quantize(c, &many, there, TPUHIP_BF16, 64), "one call");

  int32_t v = 0;
  auto p = pages();
  refused("no context", tpuhip_kv_pages_clear(nullptr, &p), "NULL");
  refused("no pages", tpuhip_kv_pages_clear(c, nullptr), "NULL");
  refused("no wishes", tpuhip_kv_pages_grow(c, &p, nullptr, 4, &v, &v, &v), "NULL");
  refused("no starts", tpuhip_kv_pages_grow(c, &p, &v, 4, nullptr, &v, &v), "NULL");
  refused("no slots", tpuhip_kv_pages_grow(c, &p, &v, 4, &v, nullptr, &v), "NULL");
  refused("capacity", tpuhip_kv_pages_grow(c, &p, &v, -1, &v, &v, &v), "room");
  refused("no keep", tpuhip_kv_pages_trim(c, &p, nullptr), "NULL");
  const tpuhip_kv_pages bad[] = {pages(0), pages(65536), pages(4, 0), pages(4, 16, 0), pages(4, 16, 33), pages(4, 1 << 26, 32), pages(4, 16, 32, 0)};
  for (auto &b : bad) {
    refused("sizes", tpuhip_kv_pages_clear(c, &b), "pages_clear");
    refused("sizes", tpuhip_kv_pages_grow(c, &b, &v, 4, &v, &v, &v), "pages_grow");
    refused("sizes", tpuhip_kv_pages_trim(c, &b, &v), "pages_trim");
  }
  p.table_stride = 3;
  refused("rows of the table", tpuhip_kv_pages_clear(c, &p), "apart");
  for (int i = 0; i < 4; ++i) {
    p = pages();
    (i == 0 ? p.lens : i == 1 ? p.table : i == 2 ? p.free_pages : p.n_free) = nullptr;
    refused("arrays", tpuhip_kv_pages_grow(c, &p, &v, 4, &v, &v, &v), "NULL");
  }
  expect(notes.empty(), "the runtime was asked for something");
}

// calls of all sizes: one launch, two where x is quantised before, and none for no rows
void launches() {
  Context c;
  for (int rows : {0, 1, 3, 16, 17, 64, 200, 777, 5000, 100000})
    for (int cols : {1, 32, 100, 2050, 4096, 16384, 100000})
      for (int n : {1, 16, 1000, 4096, 65536, 300000}) {
        if ((int64_t)rows * cols > (int64_t)1 << 32) continue;
        notes.clear();
        check(product(c, rows, cols, n));
        expect(count("launch") == (rows ? 1 : 0), "product");
        notes.clear();
        check(linear(c, rows, cols, n));
        const int chunks = (cols + 511) / 512;
        expect(count("launch") == (rows == 0 ? 0 : rows <= 16 && rows * chunks <= 32 ? 1 : 2), "linear");
      }
  notes.clear();
  const auto m = matrix((1 << 25) - 2, 1000), over = matrix((1 << 25) - 1, 1000), none = matrix(0, 1000), one = matrix(1, 1 << 24);
  check(tpuhip_mx_quantize(c, &m, there, TPUHIP_F32, 1000));
  check(tpuhip_mx_read(c, &m, there, TPUHIP_F32, 1000));
  check(tpuhip_mx_read(c, &one, there, TPUHIP_F32, 0));
  check(tpuhip_mx_quantize(c, &none, nullptr, TPUHIP_F32, 1000));
  expect(count("launch") == 3, "rows");
  expect(tpuhip_mx_read(c, &over, there, TPUHIP_F32, 1000) == TPUHIP_ERR_INVALID, "2^32 threads");
  expect(product(c, 1 << 30, 32, 1 << 30) == TPUHIP_ERR_INVALID, "more workgroups than a launch has");
  for (int capacity : {0, 1, 1024, 5000, 1 << 20, INT_MAX})
    for (int n : {1, 256, 257, 65535}) {
      notes.clear();
      const auto p = pages(n, 100000, 64, 1000);
      check(tpuhip_kv_pages_grow(c, &p, ints, capacity, ints, ints, nullptr));
      check(tpuhip_kv_pages_trim(c, &p, ints));
      check(tpuhip_kv_pages_clear(c, &p));
      expect(count("launch") == 3, "pages");
    }
}

// on a thread where another device is current: everything on the context's own
void devices() {
  Context c(1);
  const auto m = matrix(40, 16384);
  const auto p = pages(300, 100000, 64, 1000);
  const std::function<int()> calls[] = {[&] { return tpuhip_mx_quantize(c, &m, there, TPUHIP_BF16, 16384); },
                                        [&] { return tpuhip_mx_read(c, &m, there, TPUHIP_BF16, 16384); },
                                        [&] { return product(c, 40, 16384, 1000); },
                                        [&] { return linear(c, 1, 4096, 1000); },
                                        [&] { return linear(c, 300, 4096, 1000); },
                                        [&] { return tpuhip_kv_pages_grow(c, &p, ints, 1 << 20, ints, ints, nullptr); },
                                        [&] { return tpuhip_kv_pages_trim(c, &p, ints); },
                                        [&] { return tpuhip_kv_pages_clear(c, &p); }};
  notes.clear();
  for (auto &call : calls) {
    current = 0;
    check(call());
  }
  for (auto &n : notes) expect(n.device == 1, n.what);
  expect(count("malloc") == 1 && count("memset") == 1, "partial sums once");
}

// calls are recorded, and take no memory: sums that would be shared are not, where the context has none for them
void recording() {
  Context fresh, used;
  check(product(used, 40, 16384, 1000));
  const auto p = pages(300, 100000, 64, 1000);
  capturing = true;
  for (tpuhip_ctx *c : {fresh.ctx, used.ctx}) {
    notes.clear();
    check(product(c, 40, 16384, 1000));
    const size_t works = notes.at(0).size;
    expect(c == fresh ? works == 16 * 2 : works > 16 * 2, "splits");   // 64 x 64 or 32 x 64 tiles
    check(linear(c, 40, 16384, 1000));
    check(linear(c, 1, 4096, 1000));
    check(tpuhip_kv_pages_grow(c, &p, ints, 1 << 20, ints, ints, nullptr));
    expect((notes.back().size > 1) == (c == used.ctx), "workgroups without counters");
    check(tpuhip_kv_pages_trim(c, &p, ints));
    expect(count("launch") == notes.size(), "more than launches");
  }
  capturing = false;
  // no memory for partial sums is no error
  Context poor;
  memory = false;
  check(product(poor, 40, 16384, 1000));
  memory = true;
}
}  // namespace

int main(int argc, char **argv) {
  const struct {
    const char *name;
    void (*run)();
  } cases[] = {{"refusals", refusals}, {"launches", launches}, {"devices", devices}, {"recording", recording}};
  try {
    for (auto &c : cases)
      if (argc == 2 && !strcmp(argv[1], c.name)) {
        c.run();
        return 0;
      }
  } catch (const std::exception &e) {
    fprintf(stderr, "%s\n", e.what());
    return 1;
  }
  fprintf(stderr, "unknown case\n");
  return 2;
}
