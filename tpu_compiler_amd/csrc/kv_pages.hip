// The pages that a batch's sequences have in a key/value cache: which ones new tokens take, where their rows go, which ones are free again.
#include "kv_cache.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace tpuhip {

struct KvPagesArgs {
  int32_t *lens, *table, *free_pages, *n_free;
  const int32_t *wishes;        // new tokens, or tokens to keep
  int32_t *q_starts, *slots, *refused;
  int *counter;                 // workgroups that have ended, where there are several
  FastDiv page;                 // tokens of a page
  int64_t most_tokens;          // of a sequence
  int64_t table_stride;
  int n_seq, pages, capacity;
};

constexpr int kPagesMost = 128;   // workgroups of a launch

// Sums over a workgroup's threads, of those up to and with each one.  They stop at 2^32 - 1, which no number they are compared with reaches.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t sums16(uint32_t v) {       // over rows of 16 lanes
  v = dpp_add<0x111, 0xf>(v);
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  return dpp_add<0x118, 0xf>(v);
}
template <int THREADS, int N>
struct Scan {
  static constexpr int kWaves = THREADS / 64;
  static_assert(kWaves <= 16);
  uint32_t waves[2][N][16];
  // v: the sums; total: of all threads.  Calls alternate between `room` 0 and 1.
  __device__ __forceinline__ void operator()(int room, uint32_t (&v)[N], uint32_t (&total)[N]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = sums16(v[i]);
      v[i] = dpp_add<0x142, 0xa>(v[i]);                        // from lane 15 to 16..31 and 47 to 48..63,
      v[i] = dpp_add<0x143, 0xc>(v[i]);                        // from lane 31 to 32..63
      if (kWaves > 1 && lane == 63) waves[room][i][wave] = v[i];
    }
    if (kWaves == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) total[i] = (uint32_t)__builtin_amdgcn_readlane((int)v[i], 63);
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t upto = sums16(lane < kWaves ? waves[room][i][lane] : 0u);
      total[i] = (uint32_t)__builtin_amdgcn_readlane((int)upto, kWaves - 1);
      v[i] = __builtin_elementwise_add_sat(v[i], wave ? (uint32_t)__builtin_amdgcn_readlane((int)upto, wave - 1) : 0u);
    }
  }
};

// the last of THREADS ascending starts that is not above `at`
template <int THREADS>
__device__ __forceinline__ int find(const uint32_t *starts, uint32_t at) {
  int low = 0;
#pragma unroll
  for (int step = THREADS / 2; step; step >>= 1)
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

// Whether this workgroup is the last of the launch to come here: all have read the batch's state, which it may write then
__device__ __forceinline__ bool last_of(const KvPagesArgs &a) {
  if (gridDim.x == 1) return true;
  __shared__ int last;
  __syncthreads();                                             // all of this one's reads have been used
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(a.counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = before == (int)gridDim.x - 1;
    if (last) __hip_atomic_store(a.counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
  }
  __syncthreads();
  return last;
}

// Sums over the sequences say which pages and slots are whose: each thread has a sequence, THREADS of them at a time, and then pages and slots of any.
// Every workgroup makes the sums for itself and writes its part of pages and slots; the last one to end writes the state that all have read.
// Bound by latency: lengths, sums, pages, slots are a chain of three loads and two barriers.  64 sequences that get a token each take 3.2 us; 700
// sequences, 315000 new tokens, 6.4 us on 118 workgroups, 1.3 MB of slots.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_grow_kernel(KvPagesArgs a) {
  __shared__ Scan<THREADS, 3> scan;
  __shared__ uint32_t page_starts[THREADS], token_starts[THREADS];
  __shared__ int32_t first_pages[THREADS], first_tokens[THREADS];
  const int t = threadIdx.x, step = (int)gridDim.x * THREADS, first = (int)blockIdx.x * THREADS + t;
  const int n_free = min(max(a.n_free[0], 0), a.pages);
  uint32_t wanted_pages = 0, wanted_tokens = 0;                // of the sequences before these
  uint32_t tokens = 0, pages = 0, refused = 0;                 // that those got, and did not get
  const auto sequences = [&](int base, auto f) {
    const int i = base + t;
    const bool there = i < a.n_seq;
    const int len = there ? length(a, i) : 0, have = pages_of(a, len);
    const int wish = there ? max(a.wishes[i], 0) : 0;
    const bool fits = (int64_t)len + wish <= a.most_tokens;
    const uint32_t need = fits ? (uint32_t)(pages_of(a, len + wish) - have) : 0u;
    uint32_t upto[3] = {need, fits ? (uint32_t)wish : 0u, fits ? 0u : 1u}, all[3];
    scan(0, upto, all);
    const uint32_t pages_upto = __builtin_elementwise_add_sat(wanted_pages, upto[0]), tokens_upto = __builtin_elementwise_add_sat(wanted_tokens, upto[1]);
    wanted_pages = __builtin_elementwise_add_sat(wanted_pages, all[0]);
    wanted_tokens = __builtin_elementwise_add_sat(wanted_tokens, all[1]);
    const bool served = fits && tokens_upto <= (uint32_t)a.capacity && (need == 0 || pages_upto <= (uint32_t)n_free);
    if (all[2] || wanted_pages > (uint32_t)n_free || wanted_tokens > (uint32_t)a.capacity) {   // not all of them are
      upto[0] = served ? need : 0u;
      upto[1] = served ? (uint32_t)wish : 0u;
      upto[2] = there && !served && wish > 0;
      scan(1, upto, all);
    }
    f(i, there, len, have, served ? wish : 0, served ? need : 0u, upto[0], upto[1], all[0], all[1]);
    tokens += all[1];
    pages += all[0];
    refused += all[2];
  };
  int more = 0, new_len = 0;                                   // of this thread's sequence, where there is one
  for (int base = 0; base < a.n_seq; base += THREADS)
    sequences(base, [&](int i, bool there, int len, int have, int got, uint32_t got_pages, uint32_t page_end, uint32_t token_end, uint32_t new_pages, uint32_t new_tokens) {
      more = there ? got : 0;
      new_len = len + got;
      if (blockIdx.x == 0 && there) a.q_starts[i + 1] = (int)(tokens + token_end);
      page_starts[t] = page_end - got_pages;
      token_starts[t] = token_end - (uint32_t)got;
      first_pages[t] = have;
      first_tokens[t] = len;
      __syncthreads();
      const int32_t *next = a.free_pages + (n_free - 1 - (int)pages);   // the next pages to go are next[0], next[-1], ...
#pragma unroll 2
      for (int64_t p = first; p < new_pages; p += step) {
        const int s = find<THREADS>(page_starts, (uint32_t)p);
        a.table[(base + s) * a.table_stride + first_pages[s] + ((int)p - (int)page_starts[s])] = next[-p];
      }
#pragma unroll 2
      for (int64_t k = first; k < new_tokens; k += step) {
        const int s = find<THREADS>(token_starts, (uint32_t)k);
        uint32_t place = (uint32_t)(first_tokens[s] + ((int)k - (int)token_starts[s]));
        const int page = (int)a.page.split(place), fresh = page - first_pages[s];   // of a page that is not in the table yet: which of the new ones
        const int at = fresh < 0 ? a.table[(base + s) * a.table_stride + page] : next[-((int)page_starts[s] + fresh)];
        a.slots[(int)tokens + k] = (unsigned)at < (unsigned)a.pages ? (int)(at * a.page.d + place) : -1;
      }
      if (base + THREADS < a.n_seq) __syncthreads();           // the starts are written again
    });
  for (int64_t k = (int64_t)tokens + first; k < a.capacity; k += step) a.slots[k] = -1;
  if (blockIdx.x == 0 && t == 0) {
    a.q_starts[0] = 0;
    if (a.refused) a.refused[0] = (int)refused;
  }
  const uint32_t taken = pages;
  if (!last_of(a)) return;
  if (t == 0) a.n_free[0] = n_free - (int)taken;
  if (a.n_seq <= THREADS) {
    if (more) a.lens[t] = new_len;
    return;
  }
  wanted_pages = wanted_tokens = tokens = pages = 0;           // once more, what each of them got
  for (int base = 0; base < a.n_seq; base += THREADS) {
    __syncthreads();
    sequences(base, [&](int i, bool there, int len, int, int got, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {
      if (there && got) a.lens[i] = len + got;
    });
  }
}

// As above; a page that a sequence leaves goes to the place on the stack that it was taken from, if nobody has taken one since.  64 sequences 2.6 us, 700
// that lose up to 900 tokens each 4.6 us.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_trim_kernel(KvPagesArgs a) {
  __shared__ Scan<THREADS, 1> scan;
  __shared__ uint32_t page_starts[THREADS];
  __shared__ int32_t first_pages[THREADS];
  const int t = threadIdx.x, step = (int)gridDim.x * THREADS, first = (int)blockIdx.x * THREADS + t;
  const int n_free = min(max(a.n_free[0], 0), a.pages);
  const auto gone = [&](int i, int &left, int &keep) {
    left = keep = 0;
    if (i >= a.n_seq) return 0u;
    const int len = length(a, i);
    keep = min(max(a.wishes[i], 0), len);
    left = pages_of(a, keep);
    return (uint32_t)(pages_of(a, len) - left);
  };
  int left, keep;
  uint32_t all[1] = {0}, sum[1] = {0};
  if (a.n_seq > THREADS) {                                     // pages of all sequences
    for (int i = t; i < a.n_seq; i += THREADS) sum[0] = __builtin_elementwise_add_sat(sum[0], gone(i, left, keep));
    scan(1, sum, all);
  }
  uint32_t freed = all[0], pages = 0;
  for (int base = 0; base < a.n_seq; base += THREADS) {
    const uint32_t go = gone(base + t, left, keep);
    sum[0] = go;
    scan(base / THREADS & 1, sum, all);
    if (a.n_seq <= THREADS) freed = all[0];
    page_starts[t] = sum[0] - go;
    first_pages[t] = left;
    __syncthreads();
    const int64_t few = min((int64_t)all[0], (int64_t)a.pages - min(pages, (uint32_t)a.pages));   // lengths that are wrong may want more than there are
#pragma unroll 4
    for (int64_t p = first; p < few; p += step) {
      const int s = find<THREADS>(page_starts, (uint32_t)p);
      int32_t *entry = a.table + (base + s) * a.table_stride + first_pages[s] + ((int)p - (int)page_starts[s]);
      const int64_t to = (int64_t)n_free + freed - 1 - pages - p;
      if (to < a.pages) a.free_pages[to] = *entry;             // and give more
      *entry = -1;
    }
    pages = __builtin_elementwise_add_sat(pages, all[0]);
    if (base + THREADS < a.n_seq) __syncthreads();             // the starts are written again
  }
  if (!last_of(a)) return;
  for (int i = t; i < a.n_seq; i += THREADS) {
    gone(i, left, keep);
    a.lens[i] = keep;
  }
  if (t == 0) a.n_free[0] = (int)min((int64_t)n_free + freed, (int64_t)a.pages);
}

__global__ void kv_pages_clear_kernel(KvPagesArgs a) {
  const int64_t step = (int64_t)gridDim.x * blockDim.x, first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < a.pages; i += step) a.free_pages[i] = (int)(a.pages - 1 - i);   // the last is the first to go
  for (int64_t i = first; i < a.n_seq; i += step) a.lens[i] = 0;
  for (int64_t i = first; i < (int64_t)a.n_seq * a.capacity; i += step) a.table[i / a.capacity * a.table_stride + i % a.capacity] = -1;
  if (first == 0) a.n_free[0] = a.pages;
}

// Workgroups of a launch: one for each `share` pages or slots that there may be, as each makes all sums, and one alone where the context has no
// counters; 256 threads of it, if they are enough (64 sequences that grow by a token: 3.2 us, with 1024 threads 3.6).  700 sequences grow in 6.4 us
// with 2048 slots a workgroup, 7.4 with 4096, 15.2 with 16384, and no sooner with fewer than 2048; they are trimmed in 4.6 us with 8192 pages a
// workgroup, 6.9 with 16384, 9.0 by one, 4.8 with 2048.
template <typename F>
static int launch_pages(tpuhip_ctx *ctx, KvPagesArgs &a, int64_t items, int share, F kernel_of) {
  int works = (int)std::min<int64_t>(std::max<int64_t>(ceil_div64(items, share), 1), kPagesMost);
  if (works > 1) {
    if (int rc = attention_workspace(ctx)) return rc;
    a.counter = (int *)ctx->join;
    if (!a.counter) works = 1;
  }
  if (works == 1 && a.n_seq <= 256 && items <= 1024)
    launch(ctx, kernel_of(std::integral_constant<int, 256>{}), dim3(1), dim3(256), a);
  else
    launch(ctx, kernel_of(std::integral_constant<int, 1024>{}), dim3((unsigned)works), dim3(1024), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
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
  return launch_pages(ctx, a, capacity, 2048, [](auto threads) { return kv_grow_kernel<decltype(threads)::value>; });
}

int tpuhip_kv_pages_trim(tpuhip_ctx *ctx, const tpuhip_kv_pages *pages, const int32_t *keep) {
  const char *what = "tpuhip_kv_pages_trim";
  KvPagesArgs a;
  if (int rc = pages_args(ctx, pages, what, &a)) return rc;
  TPUHIP_REQUIRE(keep, "%s: NULL argument", what);
  a.wishes = keep;
  const int64_t most = std::min<int64_t>(a.pages, (int64_t)a.n_seq * pages->max_pages);
  return launch_pages(ctx, a, most, 8192, [](auto threads) { return kv_trim_kernel<decltype(threads)::value>; });
}

}  // extern "C"
