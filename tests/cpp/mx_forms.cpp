// Which kernels the products of microscaled numbers launch, with no device: this program stands in for the runtime's functions.  It reads lines
//   <product|linear> <rows> <columns of x> <columns of y> <type of y> <residual: 0 or 1>
// of calls (linear: x of the type of y) and answers each with a line of "kernel workgroups" pairs.  A line "capture 1" or "capture 0" begins or ends a
// recording, "context" makes the context anew; both are answered by an empty line.
#define __HIP_PLATFORM_AMD__
#include <cxxabi.h>
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <iostream>
#include <map>
#include <sstream>
#include <string>

#include "tpuhip.h"

namespace {
std::map<const void *, std::string> &names() {   // the library's kernels come before main() does
  static std::map<const void *, std::string> all;
  return all;
}
std::string answer;
bool capturing = false;
dim3 grid, block;

// "mx_tile_kernel<32, 64, 1, 2, 4>" without its blanks, of a kernel's whole name
std::string plain(const char *mangled) {
  int status = 0;
  char *p = abi::__cxa_demangle(mangled, nullptr, nullptr, &status);
  std::string s = status == 0 ? p : mangled, out;
  free(p);
  if (const size_t at = s.find("tpuhip::"); at != s.npos) s = s.substr(at + 8);
  for (char c : s.substr(0, s.find('(')))
    if (c != ' ') out += c;
  return out;
}
}  // namespace

extern "C" {
void __hipRegisterFunction(void **, const void *f, char *, const char *name, unsigned, void *, void *, dim3 *, dim3 *, int *) { names()[f] = plain(name); }
hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *s) { return *p = const_cast<void *>(s), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { return *s = (hipStream_t)malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return free((void *)s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  return *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipMalloc(void **p, size_t) { return capturing ? hipErrorStreamCaptureUnsupported : (*p = malloc(16), hipSuccess); }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return capturing ? hipErrorStreamCaptureUnsupported : hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return grid = g, block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *shared, hipStream_t *s) {
  return *g = grid, *b = block, *shared = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3, void **, size_t, hipStream_t) {
  answer += (answer.empty() ? "" : " ") + names()[f] + " " + std::to_string(g.x);
  return hipSuccess;
}
}

int main() {
  alignas(16) static uint8_t there[64];   // nothing is read from where the calls point
  const auto matrix = [&](int rows, int cols) {
    const int blocks = cols / 32 + (cols % 32 != 0);
    return tpuhip_mx_matrix{rows, cols, there, there + 16, (int64_t)blocks * 16, blocks};
  };
  tpuhip_ctx *ctx = nullptr;
  if (tpuhip_ctx_create(0, &ctx) != TPUHIP_OK) return 1;
  for (std::string line; std::getline(std::cin, line);) {
    std::istringstream in(line);
    std::string what;
    answer.clear();
    in >> what;
    if (what == "capture") {
      in >> capturing;
    } else if (what == "context") {
      tpuhip_ctx_destroy(ctx);
      if (tpuhip_ctx_create(0, &ctx) != TPUHIP_OK) return 1;
    } else {
      int rows, cols, n, dtype, residual;
      if (!(in >> rows >> cols >> n >> dtype >> residual)) return 2;
      const auto x = matrix(rows, cols), w = matrix(n, cols);
      const tpuhip_mx_product_desc d = {dtype, n, n, nullptr, residual ? there : nullptr};
      const int rc = what == "linear" ? tpuhip_mx_linear(ctx, &d, there, dtype, cols, &x, &w, there) : tpuhip_mx_product(ctx, &d, &x, &w, there);
      if (rc != TPUHIP_OK) {
        fprintf(stderr, "%s: %s\n", line.c_str(), tpuhip_last_error());
        return 1;
      }
    }
    std::cout << answer << "\n";
  }
  tpuhip_ctx_destroy(ctx);
}
