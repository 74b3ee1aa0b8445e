// The pages that a batch's sequences have in a key/value cache: which ones new tokens take, where their rows go, which ones are free again.
#include "common.hpp"

#include <algorithm>
#include <climits>

namespace tpuhip {

struct KvPagesArgs {
  int32_t *lens, *table, *free_pages, *n_free;
  const int32_t *wishes;        // new tokens, or tokens to keep
  int32_t *q_starts, *slots, *refused;
  FastDiv page;                 // tokens of a page
  int64_t most_tokens;          // of a sequence
  int64_t table_stride;
  int n_seq, pages, capacity;
};

constexpr int kPagesThreads = 1024, kPagesWaves = kPagesThreads / 64;

// Sums over a workgroup's threads, of those up to and with each one, of up to three numbers at once
template <int N>
struct ScanRoom {
  int64_t waves[N][kPagesWaves];
};
template <int N>
__device__ __forceinline__ void scan(ScanRoom<N> &room, int64_t (&v)[N], int64_t (&total)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t below = __shfl_up(v[i], d);
      if (lane >= d) v[i] += below;
    }
  __syncthreads();                                             // the room may still be read
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) room.waves[i][wave] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    total[i] = 0;
    int64_t before = 0;
    for (int k = 0; k < kPagesWaves; ++k) {
      if (k < wave) before += room.waves[i][k];
      total[i] += room.waves[i][k];
    }
    v[i] += before;
  }
}

// the last of the threads' ascending starts that is not above `at`
__device__ __forceinline__ int find(const int32_t *starts, int at) {
  int low = 0;
#pragma unroll
  for (int step = kPagesThreads / 2; step; step >>= 1)
    if (starts[low + step] <= at) low += step;
  return low;
}

__device__ __forceinline__ int pages_of(const KvPagesArgs &a, int tokens) {
  uint32_t t = (uint32_t)tokens;
  const uint32_t whole = a.page.split(t);
  return (int)(whole + (t != 0));
}
__device__ __forceinline__ int length(const KvPagesArgs &a, int i) {
  return (int)min((int64_t)max(a.lens[i], 0), a.most_tokens);
}

// One workgroup: sums over the sequences say which pages and slots are whose; each thread has a sequence, 1024 of them at a time, and then pages
// and tokens of any.
__global__ __launch_bounds__(kPagesThreads) void kv_grow_kernel(KvPagesArgs a) {
  __shared__ ScanRoom<2> room;
  __shared__ int32_t page_starts[kPagesThreads], token_starts[kPagesThreads], first_pages[kPagesThreads], first_tokens[kPagesThreads];
  const int t = threadIdx.x;
  const int n_free = min(max(a.n_free[0], 0), a.pages);
  int64_t wanted_pages = 0, wanted_tokens = 0;                 // of the sequences before these
  int tokens = 0, pages = 0, refused = 0;                      // that those got, and did not get
  for (int base = 0; base < a.n_seq; base += kPagesThreads) {
    const int i = base + t;
    const bool there = i < a.n_seq;
    const int len = there ? length(a, i) : 0, have = pages_of(a, len);
    const int wish = there ? max(a.wishes[i], 0) : 0;
    const bool fits = (int64_t)len + wish <= a.most_tokens;
    const int need = fits ? pages_of(a, len + wish) - have : 0;
    int64_t upto[2] = {need, fits ? wish : 0}, all[2];
    scan(room, upto, all);
    const bool served = fits && wanted_tokens + upto[1] <= a.capacity && (need == 0 || wanted_pages + upto[0] <= n_free);
    wanted_pages += all[0];
    wanted_tokens += all[1];
    int64_t got[2] = {served ? wish : 0, (served ? (int64_t)need << 32 : 0) + (there && !served && wish > 0)}, sums[2];
    scan(room, got, sums);
    const int new_tokens = (int)sums[0], new_pages = (int)(sums[1] >> 32);
    const int end = (int)got[0], end_page = (int)(got[1] >> 32);
    if (there) {
      a.q_starts[i + 1] = tokens + end;
      if (served && wish) a.lens[i] = len + wish;
    }
    page_starts[t] = end_page - (served ? need : 0);
    token_starts[t] = end - (served ? wish : 0);
    first_pages[t] = have;
    first_tokens[t] = len;
    __syncthreads();
    for (int p = t; p < new_pages; p += kPagesThreads) {
      const int s = find(page_starts, p);
      a.table[(base + s) * a.table_stride + first_pages[s] + p - page_starts[s]] = a.free_pages[n_free - 1 - pages - p];
    }
    __syncthreads();
    for (int k = t; k < new_tokens; k += kPagesThreads) {
      const int s = find(token_starts, k);
      uint32_t place = (uint32_t)(first_tokens[s] + k - token_starts[s]);
      const int page = (int)a.page.split(place), at = a.table[(base + s) * a.table_stride + page];
      a.slots[tokens + k] = (unsigned)at < (unsigned)a.pages ? (int)(at * a.page.d + place) : -1;
    }
    tokens += new_tokens;
    pages += new_pages;
    refused += (int)(uint32_t)sums[1];
    __syncthreads();
  }
  for (int k = tokens + t; k < a.capacity; k += kPagesThreads) a.slots[k] = -1;
  if (t == 0) {
    a.q_starts[0] = 0;
    a.n_free[0] = n_free - pages;
    if (a.refused) a.refused[0] = refused;
  }
}

__global__ __launch_bounds__(kPagesThreads) void kv_trim_kernel(KvPagesArgs a) {
  __shared__ ScanRoom<1> room;
  __shared__ int32_t page_starts[kPagesThreads], first_pages[kPagesThreads];
  const int t = threadIdx.x;
  const int n_free = min(max(a.n_free[0], 0), a.pages);
  const auto gone = [&](int i, int &left, int &keep) {
    const int len = length(a, i);
    keep = min(max(a.wishes[i], 0), len);
    left = pages_of(a, keep);
    return pages_of(a, len) - left;
  };
  int left, keep;
  int64_t all[1] = {0}, sum[1] = {0};
  for (int i = t; i < a.n_seq; i += kPagesThreads) sum[0] += gone(i, left, keep);
  scan(room, sum, all);
  const int64_t freed = all[0];                                // of all sequences
  int64_t pages = 0;
  for (int base = 0; base < a.n_seq; base += kPagesThreads) {
    const int i = base + t;
    const bool there = i < a.n_seq;
    left = keep = 0;
    const int go = there ? gone(i, left, keep) : 0;
    sum[0] = go;
    scan(room, sum, all);
    page_starts[t] = (int)min(sum[0] - go, (int64_t)INT_MAX);
    first_pages[t] = left;
    if (there) a.lens[i] = keep;
    __syncthreads();
    for (int p = t; p < all[0]; p += kPagesThreads) {
      const int s = find(page_starts, p);
      int32_t *entry = a.table + (base + s) * a.table_stride + first_pages[s] + p - page_starts[s];
      const int64_t to = n_free + freed - 1 - pages - p;
      if (to < a.pages) a.free_pages[to] = *entry;             // more pages than there are come back from a table that is wrong
      *entry = -1;
    }
    pages += all[0];
    __syncthreads();
  }
  if (t == 0) a.n_free[0] = (int)min(n_free + freed, (int64_t)a.pages);
}

__global__ void kv_pages_clear_kernel(KvPagesArgs a) {
  const int64_t step = (int64_t)gridDim.x * blockDim.x, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < a.pages; i += step) a.free_pages[i] = (int)(a.pages - 1 - i);   // the last is the first to go
  for (int64_t i = first; i < a.n_seq; i += step) a.lens[i] = 0;
  for (int64_t i = first; i < (int64_t)a.n_seq * a.capacity; i += step) a.table[i / a.capacity * a.table_stride + i % a.capacity] = -1;
  if (first == 0) a.n_free[0] = a.pages;
}

static int pages_args(tpuhip_ctx *ctx, const tpuhip_kv_pages *p, const char *what, KvPagesArgs *a) {
  TPUHIP_REQUIRE(ctx && p, "%s: NULL argument", what);
  TPUHIP_REQUIRE(p->n_seq >= 1 && p->n_seq <= 65535, "%s: %d sequences", what, p->n_seq);
  TPUHIP_REQUIRE(p->page_tokens >= 32 && p->page_tokens % 32 == 0 && p->pages >= 1 && (int64_t)p->pages * p->page_tokens <= INT_MAX, "%s: %d pages of %d tokens", what,
                 p->pages, p->page_tokens);
  TPUHIP_REQUIRE(p->max_pages >= 1 && p->table_stride >= (p->n_seq > 1 ? p->max_pages : 0), "%s: %d pages a sequence in rows %d apart", what,
                 p->max_pages, p->table_stride);
  TPUHIP_REQUIRE(p->lens && p->table && p->free_pages && p->n_free, "%s: NULL argument", what);
  *a = KvPagesArgs{};
  a->lens = p->lens;
  a->table = p->table;
  a->free_pages = p->free_pages;
  a->n_free = p->n_free;
  a->page = FastDiv(p->page_tokens);
  a->most_tokens = std::min<int64_t>((int64_t)p->max_pages * p->page_tokens, 1 << 30);   // as many as attention takes
  a->table_stride = p->table_stride;
  a->n_seq = p->n_seq;
  a->pages = p->pages;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  return TPUHIP_OK;
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

int tpuhip_kv_pages_clear(tpuhip_ctx *ctx, const tpuhip_kv_pages *pages) {
  KvPagesArgs a;
  if (int rc = pages_args(ctx, pages, "tpuhip_kv_pages_clear", &a)) return rc;
  a.capacity = pages->max_pages;
  const int64_t entries = std::max<int64_t>(a.pages, (int64_t)a.n_seq * a.capacity);
  launch(ctx, kv_pages_clear_kernel, dim3((unsigned)std::min<int64_t>(ceil_div64(entries, 256), 4096)), dim3(256), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

int tpuhip_kv_pages_grow(tpuhip_ctx *ctx, const tpuhip_kv_pages *pages, const int32_t *new_tokens, int capacity, int32_t *q_starts,
                         int32_t *slots, int32_t *refused) {
  const char *what = "tpuhip_kv_pages_grow";
  KvPagesArgs a;
  if (int rc = pages_args(ctx, pages, what, &a)) return rc;
  TPUHIP_REQUIRE(capacity >= 0, "%s: room for %d tokens", what, capacity);
  TPUHIP_REQUIRE(new_tokens && q_starts && (slots || capacity == 0), "%s: NULL argument", what);
  a.wishes = new_tokens;
  a.capacity = capacity;
  a.q_starts = q_starts;
  a.slots = slots;
  a.refused = refused;
  launch(ctx, kv_grow_kernel, dim3(1), dim3(kPagesThreads), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

int tpuhip_kv_pages_trim(tpuhip_ctx *ctx, const tpuhip_kv_pages *pages, const int32_t *keep) {
  const char *what = "tpuhip_kv_pages_trim";
  KvPagesArgs a;
  if (int rc = pages_args(ctx, pages, what, &a)) return rc;
  TPUHIP_REQUIRE(keep, "%s: NULL argument", what);
  a.wishes = keep;
  launch(ctx, kv_trim_kernel, dim3(1), dim3(kPagesThreads), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

}  // extern "C"
