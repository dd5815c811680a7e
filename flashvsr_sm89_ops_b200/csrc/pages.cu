// Pages of a paged cache: making room, branching, dropping and compacting.
//
// A cache is pools k, v [layers][pages][page rows] of one block of bytes a page, a table
// [sequences][width] of page numbers (-1 for none), the tokens each sequence holds and how many
// sequences hold each page (0: free).  All of it is device memory and every step is a kernel, so
// a captured graph can allocate: nothing waits for the host.  Free pages are given out lowest
// first in the order of sequences and of their pages, which makes every result a function of the
// state alone.  A page held by several sequences is always full: a fork copies a partly filled
// last page at once, so no append ever writes to a shared page.
//
// The bookkeeping is one block: it scans refs (4 bytes a page) and touches one table row a
// sequence, microseconds against the copies.  Copies are bound by memory: read and written once,
// 64 bytes in flight a thread over all layers' k and v in one launch (100 pages of 128 x 12 x 128 in 4
// layers: 629 MB in 101 us, 6.2 TB/s).  The bookkeeping of a step takes 3.5-6 us, a chain of dependent
// accesses.  A step whose arguments or
// whose room do not suffice changes nothing and records a code in `status`; a reserve also records in
// `refused` whether it was done, for the appends behind it (the host does not know).
//
// Keys stay as they were rotated when a sequence's first pages are given back, so its next tokens'
// positions go on from all that it ever held: `dropped` counts what it held before lens.  A sequence
// without tokens begins at 0 again (there is no key that a distance could be wrong to).
#include "common.cuh"

namespace fvb {
namespace pages {

constexpr int kThreads = 1024;
constexpr int kSmall = 2048;  // lists up to this long are kept in shared memory
constexpr int kNoPages = 1, kNoWidth = 2, kBadArgs = 4;

struct Copy {
  int32_t from, to, rows, pad;
};

// Every kernel of this file is launched while its predecessor still runs, lets its own successor do
// the same, and touches memory only after the predecessor's end: a chain of steps costs their
// latencies, not their launches.
__device__ __forceinline__ void chain() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

// one bit a sequence, in shared memory
__device__ __forceinline__ bool test_and_set(uint32_t* bits, int64_t i) {
  return atomicOr(bits + (i >> 5), 1u << (i & 31)) >> (i & 31) & 1;
}

// exclusive prefix sum over the block of one value a thread; total gets the sum
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums of an earlier scan have been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// The `need` lowest free pages into list; returns how many were found.
__device__ int free_pages(const int32_t* refs, int64_t pages, int need, int32_t* list, int* sums) {
  int found = 0;
  for (int64_t at = 0; at < pages && found < need; at += kThreads * 4) {
    const int64_t p0 = at + threadIdx.x * 4;
    int free = 0, n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + i < pages && refs[p0 + i] == 0) free |= 1 << i, ++n;
    int total;
    int r = found + block_scan(n, sums, total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (free >> i & 1) {
        if (r < need) list[r] = (int32_t)(p0 + i);
        ++r;
      }
    found += total;
  }
  __syncthreads();
  return found < need ? found : need;
}

struct Cache {
  int32_t *table, *lens, *refs, *status, *refused;
  int64_t* dropped;
  int64_t seqs, width, pages;
  int page;
};

__device__ __forceinline__ int64_t held(const Cache& c, int64_t len) {  // pages of len tokens
  const int64_t n = len <= 0 ? 0 : (len + c.page - 1) / c.page;
  return n < c.width ? n : c.width;
}

// ws: prefix [seqs + 1], list [pages]
__global__ void __launch_bounds__(kThreads) reserve_kernel(const Cache c, const int32_t* more,
                                                           int32_t* ws) {
  __shared__ int sums[32];
  __shared__ int32_t s_prefix[kSmall], s_list[kSmall];
  int32_t* const prefix = c.seqs <= kSmall ? s_prefix : ws;
  chain();
  int64_t need = 0;
  int bad = 0;
  for (int64_t at = 0; at < c.seqs; at += kThreads) {
    const int64_t b = at + threadIdx.x;
    int n = 0;
    if (b < c.seqs) {
      const int64_t len = c.lens[b], add = more[b];
      const int64_t want = (len + add + c.page - 1) / c.page;
      if (len < 0 || add < 0 || len + add > INT32_MAX) bad |= kBadArgs;
      else if (want > c.width) bad |= kNoWidth;
      else n = (int)(want - held(c, len));
    }
    int total;
    const int before = block_scan(n, sums, total);
    if (b < c.seqs) prefix[b] = (int32_t)(need + before);
    need += total;
  }
  bad = __syncthreads_or(bad & kBadArgs) ? kBadArgs : __syncthreads_or(bad & kNoWidth) ? kNoWidth : 0;
  if (!bad && need > c.pages) bad = kNoPages;
  int32_t* const list = need <= kSmall ? s_list : ws + c.seqs + 1;
  if (!bad && free_pages(c.refs, c.pages, (int)need, list, sums) < need) bad = kNoPages;
  if (threadIdx.x == 0) {
    if (bad) atomicOr(c.status, bad);
    if (c.refused) *c.refused = bad != 0;
  }
  if (bad) return;
  for (int i = threadIdx.x; i < need; i += kThreads) {
    int64_t lo = 0, hi = c.seqs;  // the last sequence whose pages start at or before i
    while (lo + 1 < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (prefix[mid] <= i) lo = mid; else hi = mid;
    }
    c.table[lo * c.width + held(c, c.lens[lo]) + (i - prefix[lo])] = list[i];
    c.refs[list[i]] = 1;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < c.seqs; b += kThreads) {
    const int32_t len = c.lens[b];
    c.lens[b] = len + more[b];
    if (c.dropped && len == 0) c.dropped[b] = 0;  // begins anew
  }
}

// ws: count, copies [n], list [n]
__global__ void __launch_bounds__(kThreads) fork_kernel(const Cache c, const int32_t* src,
                                                        const int32_t* dst, int n, int32_t* ws) {
  extern __shared__ uint32_t branch[];  // a bit a sequence: it is a branch
  __shared__ int sums[32];
  __shared__ int32_t s_list[kSmall];
  __shared__ int32_t s_rank[kSmall];
  Copy* copies = reinterpret_cast<Copy*>(ws + 4);
  for (int i = threadIdx.x; i < (int)((c.seqs + 31) >> 5); i += kThreads) branch[i] = 0;
  chain();
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t a = src[i], d = dst[i];
    if (a < 0 || a >= c.seqs || d < 0 || d >= c.seqs) bad = kBadArgs;
    else if (test_and_set(branch, d) || c.lens[d] != 0 || c.lens[a] < 0) bad = kBadArgs;
  }
  bad = __syncthreads_or(bad) ? kBadArgs : 0;
  int need = 0;
  if (!bad) {
    for (int at = 0; at < n; at += kThreads) {
      const int i = at + threadIdx.x;
      int part = 0;
      int32_t len = 0;
      int64_t a = 0;
      if (i < n) {
        a = src[i];
        if (branch[a >> 5] >> (a & 31) & 1) bad = kBadArgs;
        len = c.lens[a];
        part = len % c.page;
      }
      int total;
      const int r = need + block_scan(part > 0, sums, total);
      if (i < n) {
        if (n <= kSmall) s_rank[i] = r;
        const int64_t full = len / c.page;
        int32_t from = full < c.width ? c.table[a * c.width + full] : -1;
        if (from < 0 || from >= c.pages) part = 0, from = 0;
        copies[i] = {from, r, part, 0};  // rows 0: nothing to copy
      }
      need += total;
    }
    bad = __syncthreads_or(bad) ? kBadArgs : 0;
  }
  int32_t* const list = n <= kSmall ? s_list : ws + 4 + 4 * (int64_t)n;
  if (!bad && (need > c.pages || free_pages(c.refs, c.pages, need, list, sums) < need)) bad = kNoPages;
  if (bad) {
    if (threadIdx.x == 0) {
      atomicOr(c.status, bad);
      ws[0] = 0;
    }
    return;
  }
  __syncthreads();
  if (threadIdx.x == 0) ws[0] = n;
  // a thread an entry of the branches' rows
  for (int64_t e = threadIdx.x; e < n * c.width; e += kThreads) {
    const int i = (int)(e / c.width);
    const int64_t j = e - i * c.width, a = src[i], d = dst[i];
    const int32_t len = c.lens[a], full = len / c.page;
    int32_t p = -1;
    if (j < full) {
      p = c.table[a * c.width + j];
      if (p >= 0 && p < c.pages) atomicAdd(c.refs + p, 1);
    } else if (j == full && len % c.page) {
      p = list[n <= kSmall ? s_rank[i] : copies[i].to];
      c.refs[p] = 1;
    }
    c.table[d * c.width + j] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int32_t a = src[i], d = dst[i], len = c.lens[a];
    const int64_t before = c.dropped ? c.dropped[a] : 0;
    copies[i].to = len % c.page ? list[n <= kSmall ? s_rank[i] : copies[i].to] : 0;
    c.lens[d] = len;
    if (c.dropped) c.dropped[d] = before;
  }
}

// drop NULL: everything; else leading pages, the others move to the front.
__global__ void __launch_bounds__(kThreads) release_kernel(const Cache c, const int32_t* seqs,
                                                           const int32_t* drop, int n) {
  extern __shared__ uint32_t named[];  // a bit a sequence
  for (int i = threadIdx.x; i < (int)((c.seqs + 31) >> 5); i += kThreads) named[i] = 0;
  chain();
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t b = seqs[i];
    if (b < 0 || b >= c.seqs || (drop && drop[i] < 0) || test_and_set(named, b)) bad = 1;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) atomicOr(c.status, kBadArgs);
    return;
  }
  // a thread an entry of the rows that go as a whole, a warp a row of the others
  for (int64_t e = threadIdx.x; e < n * c.width; e += kThreads) {
    const int i = (int)(e / c.width);
    const int64_t j = e - i * c.width, b = seqs[i], have = held(c, c.lens[b]);
    if (j >= have || (drop && drop[i] < have)) continue;
    const int32_t p = c.table[b * c.width + j];
    c.table[b * c.width + j] = -1;
    if (p >= 0 && p < c.pages) atomicSub(c.refs + p, 1);
  }
  const int lane = threadIdx.x & 31;
  if (drop)
    for (int i = threadIdx.x >> 5; i < n; i += kThreads / 32) {
      const int64_t b = seqs[i], have = held(c, c.lens[b]), gone = drop[i];
      int32_t* row = c.table + b * c.width;
      if (gone >= have) continue;
      for (int64_t j = lane; j < gone; j += 32) {
        const int32_t p = row[j];
        if (p >= 0 && p < c.pages) atomicSub(c.refs + p, 1);
      }
      __syncwarp();
      // 32 entries at a time: read, then written, so that a shift by less than 32 is safe
      for (int64_t j0 = 0; j0 < have; j0 += 32) {
        const int64_t j = j0 + lane;
        const int32_t p = j + gone < have ? row[j + gone] : -1;
        __syncwarp();
        if (j < have) row[j] = p;
        __syncwarp();
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t b = seqs[i], len = c.lens[b], have = held(c, len);
    const int64_t before = drop && c.dropped ? c.dropped[b] : 0;
    const int64_t left = len - (int64_t)(drop ? drop[i] : 0) * c.page;
    const int32_t now = !drop || drop[i] >= have ? 0 : (int32_t)(left > 0 ? left : 0);
    c.lens[b] = now;
    if (c.dropped) c.dropped[b] = now ? before + (len - now) : 0;
  }
}

// ws: count, copies [pages / 2 + 1], map [pages].  Pages at or behind the number in use move to
// the holes before it, both in ascending order.
__global__ void __launch_bounds__(kThreads) compact_kernel(const Cache c, int32_t* ws) {
  __shared__ int sums[32];
  Copy* copies = reinterpret_cast<Copy*>(ws + 4);
  int32_t* map = ws + 4 + 4 * (c.pages / 2 + 1);
  chain();
  int64_t used = 0;
  for (int64_t p = threadIdx.x; p < c.pages; p += kThreads) used += c.refs[p] > 0;
  int total;
  block_scan((int)used, sums, total);
  used = total;
  int holes = 0, movers = 0;
  for (int64_t at = 0; at < c.pages; at += kThreads) {
    const int64_t p = at + threadIdx.x;
    const int in_use = p < c.pages && c.refs[p] > 0;
    const int hole = p < used && !in_use, mover = p >= used && in_use;
    int nh, nm;
    const int rh = holes + block_scan(hole, sums, nh);
    const int rm = movers + block_scan(mover, sums, nm);
    if (hole) copies[rh].to = (int32_t)p;
    if (mover) copies[rm].from = (int32_t)p;
    if (p < c.pages) map[p] = (int32_t)p;
    holes += nh;
    movers += nm;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kThreads) {
    const int32_t from = copies[i].from, to = copies[i].to;
    copies[i].rows = c.page;
    map[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) ws[0] = movers;
}

struct Pools {
  uint8_t *k, *v;
  int64_t layers, layer_stride, page_stride;  // bytes
  int64_t row_bytes, page_bytes;
};

constexpr int kCopyThreads = 256;
constexpr int kChunk = kCopyThreads * 4 * 16;  // bytes a block copies at a time

// count and copies from ws; the table's pages through map (NULL: the table is as it should be)
__global__ void __launch_bounds__(kCopyThreads)
    copy_kernel(const Pools p, const int32_t* ws, const int32_t* map, int32_t* table,
                int64_t entries, int64_t pages) {
  chain();
  const int64_t count = ws[0];
  const Copy* copies = reinterpret_cast<const Copy*>(ws + 4);
  if (map) {
    const int64_t step = (int64_t)gridDim.x * kCopyThreads;
    for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < entries; i += step) {
      const int32_t was = table[i];
      if (was >= 0 && was < pages) table[i] = map[was];
    }
  }
  const int64_t chunks = (p.page_bytes + kChunk - 1) / kChunk;
  const int64_t tasks = count * 2 * p.layers * chunks;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int64_t chunk = task % chunks;
    int64_t r = task / chunks;
    const int64_t layer = r % p.layers;
    r /= p.layers;
    uint8_t* pool = (r & 1 ? p.v : p.k) + layer * p.layer_stride;
    const Copy c = copies[r >> 1];
    const int64_t bytes = c.rows * p.row_bytes;
    const int64_t at = chunk * kChunk + threadIdx.x * 16;
    const uint8_t* from = pool + c.from * p.page_stride + at;
    uint8_t* to = pool + c.to * p.page_stride + at;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * kCopyThreads * 16 < bytes)
        v[i] = ld_stream(reinterpret_cast<const uint4*>(from + i * kCopyThreads * 16));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * kCopyThreads * 16 < bytes)
        *reinterpret_cast<uint4*>(to + i * kCopyThreads * 16) = v[i];
  }
}

template <typename... P, typename... A>
int launch(const char* what, cudaStream_t stream, void (*kernel)(P...), int64_t grid, int threads, size_t smem,
           A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &early;
  c.numAttrs = 1;
  FVB_CUDA_TRY(cudaLaunchKernelEx(&c, kernel, args...), what);
  return FVB_OK;
}

int cache_of(const fvb_pages* p, Cache& c, const char* what) {
  FVB_REQUIRE(p, "%s: NULL pointer", what);
  // a bit a sequence has to fit in shared memory beside the lists
  FVB_REQUIRE(p->seqs >= 0 && p->seqs <= (1 << 17) && p->width >= 0 && p->width < (1ll << 31) &&
                  p->pages >= 0 && p->pages < (1ll << 31) && p->page > 0 && p->page < (1 << 24) &&
                  p->seqs * p->width < (1ll << 31),
              "%s: cache of %lld sequences x %lld pages of %lld, pool of %lld", what, (long long)p->seqs,
              (long long)p->width, (long long)p->page, (long long)p->pages);
  FVB_REQUIRE(p->table && p->lens && p->refs && p->status && p->workspace, "%s: NULL pointer", what);
  FVB_REQUIRE(aligned16(p->workspace), "%s: workspace must be 16-byte aligned", what);
  c = {p->table, p->lens, p->refs, p->status, p->refused, p->dropped, p->seqs, p->width, p->pages, (int)p->page};
  return FVB_OK;
}

int pools_of(const fvb_pages* p, Pools& q, const char* what) {
  FVB_REQUIRE(p->layers >= 0 && p->row_bytes > 0 && p->row_bytes % 16 == 0 &&
                  p->layer_stride % 16 == 0 && p->page_stride % 16 == 0,
              "%s: rows and strides must be multiples of 16 bytes", what);
  FVB_REQUIRE(p->layers == 0 || (p->k && p->v && aligned16(p->k) && aligned16(p->v)),
              "%s: pools must be 16-byte aligned", what);
  q = {(uint8_t*)p->k, (uint8_t*)p->v, p->layers, p->layer_stride, p->page_stride, p->row_bytes,
       p->row_bytes * p->page};
  return FVB_OK;
}

inline size_t bits(int64_t seqs) { return (size_t)((seqs + 31) / 32 * 4); }  // a bit a sequence

int launch_copy(const Pools& p, const int32_t* ws, const int32_t* map, const Cache& c, int64_t most,
                cudaStream_t stream, const char* what) {
  const int64_t chunks = (p.page_bytes + kChunk - 1) / kChunk;
  int64_t grid = most * 2 * p.layers * chunks;
  const int64_t full = (int64_t)sm_count() * 8;
  if (grid > full) grid = full;
  if (grid < 1) grid = 1;
  return launch(what, stream, copy_kernel, grid, kCopyThreads, 0, p, ws, map, c.table, c.seqs * c.width,
                c.pages);
}

}  // namespace pages
}  // namespace fvb

extern "C" {

size_t fvb_pages_workspace_bytes(int64_t seqs, int64_t pages) {
  if (seqs < 0 || pages < 0) return 0;
  const int64_t reserve = seqs + 1 + pages;
  const int64_t fork = 4 + 4 * seqs + seqs;
  const int64_t compact = 4 + 4 * (pages / 2 + 1) + pages;
  int64_t m = reserve > fork ? reserve : fork;
  if (compact > m) m = compact;
  return (size_t)(4 * m + 16);
}

int fvb_pages_reserve(const fvb_pages* p, const int32_t* more, fvb_stream_t stream) {
  using namespace fvb;
  pages::Cache c;
  int rc = pages::cache_of(p, c, "fvb_pages_reserve");
  if (rc || p->seqs == 0) return rc;
  FVB_REQUIRE(more, "fvb_pages_reserve: NULL pointer");
  return pages::launch("fvb_pages_reserve", (cudaStream_t)stream, pages::reserve_kernel, 1, pages::kThreads, 0,
                       c, more, (int32_t*)p->workspace);
}

int fvb_pages_fork(const fvb_pages* p, const int32_t* src, const int32_t* dst, int64_t n,
                   fvb_stream_t stream) {
  using namespace fvb;
  pages::Cache c;
  pages::Pools pools;
  int rc = pages::cache_of(p, c, "fvb_pages_fork");
  if (!rc) rc = pages::pools_of(p, pools, "fvb_pages_fork");
  if (rc) return rc;
  FVB_REQUIRE(n >= 0 && n <= p->seqs, "fvb_pages_fork: %lld branches of %lld sequences", (long long)n,
              (long long)p->seqs);
  if (n == 0) return FVB_OK;
  FVB_REQUIRE(src && dst, "fvb_pages_fork: NULL pointer");
  int32_t* ws = (int32_t*)p->workspace;
  rc = pages::launch("fvb_pages_fork", (cudaStream_t)stream, pages::fork_kernel, 1, pages::kThreads,
                     pages::bits(p->seqs), c, src, dst, (int)n, ws);
  if (rc) return rc;
  return pages::launch_copy(pools, ws, nullptr, c, n, (cudaStream_t)stream, "fvb_pages_fork");
}

int fvb_pages_release(const fvb_pages* p, const int32_t* rows, const int32_t* drop, int64_t n,
                      fvb_stream_t stream) {
  using namespace fvb;
  pages::Cache c;
  int rc = pages::cache_of(p, c, "fvb_pages_release");
  if (rc) return rc;
  FVB_REQUIRE(n >= 0 && n < (1 << 28), "fvb_pages_release: %lld sequences", (long long)n);
  if (n == 0) return FVB_OK;
  FVB_REQUIRE(rows, "fvb_pages_release: NULL pointer");
  return pages::launch("fvb_pages_release", (cudaStream_t)stream, pages::release_kernel, 1, pages::kThreads,
                       pages::bits(p->seqs), c, rows, drop, (int)n);
}

int fvb_pages_compact(const fvb_pages* p, fvb_stream_t stream) {
  using namespace fvb;
  pages::Cache c;
  pages::Pools pools;
  int rc = pages::cache_of(p, c, "fvb_pages_compact");
  if (!rc) rc = pages::pools_of(p, pools, "fvb_pages_compact");
  if (rc || p->pages == 0) return rc;
  int32_t* ws = (int32_t*)p->workspace;
  rc = pages::launch("fvb_pages_compact", (cudaStream_t)stream, pages::compact_kernel, 1, pages::kThreads, 0, c,
                     ws);
  if (rc) return rc;
  return pages::launch_copy(pools, ws, ws + 4 + 4 * (p->pages / 2 + 1), c, p->pages / 2 + 1,
                            (cudaStream_t)stream, "fvb_pages_compact");
}

}  // extern "C"
