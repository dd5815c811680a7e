// Attention of a chunk of new tokens over a paged cache.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  j <= len - n + i (causal) or j < len
// for the n new tokens i of each sequence, len its tokens in the cache (the new ones included),
// query head h on key head h / g.  The g query heads of a key head are rows of one tile ("packed
// row" i * g + h % g), so a key is read once for all of them.
//
// Work is cut the same way in both kernels.  An item is (sequence, key head, tile of packed
// rows); its length is the number of key tiles that its last row sees.  The items of all
// sequences lie end to end on one line of key tiles, and each CTA takes an equal stretch of it:
// uneven sequences and causal triangles balance by themselves, few rows over a long cache spread
// over the machine, and a last partial wave does not exist.  An item cut by a boundary leaves
// unnormalised partial sums (fp32 O, row maximum and sum) that merge_kernel joins in the order of
// the cut, so results do not depend on timing.  Where there are many rows and items enough, whole
// items are dealt out by length instead (see chunk_kernel).  Lengths are read on the device only:
// every CTA counts the work itself, and a captured graph follows them.
//
//   decode_kernel  up to 16 packed rows a tile: single tokens, a few drafted ones.  Bound by the
//                  bytes of the cache.
//   chunk_kernel   256 packed rows a tile on the tcgen05 tensor cores.  Bound by them and by the
//                  exponentials.
//
// Keys past a sequence's end are never seen: their scores are -inf whatever the page holds, and
// their values are zeros in shared memory, so NaNs left in a recycled page do not spread.  A
// page number outside the pool reads as zeros.
#include "common.cuh"

#include <cuda_fp16.h>

namespace fvb {
namespace pattn {

// Keys of a sequence: the end of their last tile, and of tiles loaded ahead of it, is an int.
constexpr int64_t kMostKeys = (1ll << 31) - 1024;

struct Args {
  const void* q;
  void* out;
  int64_t q_token, q_head, o_token, o_head;  // strides, elements
  const void *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  const int32_t *table, *lens, *cu;  // cu NULL: one token a sequence
  int64_t T, width, pages;
  int B, Hk, g, page, causal, ctas;
  int rows, tokens;  // packed rows of an item's tile: whole tokens
  int few_rows;      // rows that the caller's bound on new tokens announces
  float scale_log2;
  float* part;    // [2 ctas][rows][D]: O of an item begun before the CTA, of one begun in it
  float* part_ml; // [2 ctas][rows][2]
  int32_t* rec;   // [ctas][8]: the item begun in the CTA that other CTAs end
};

struct Seq {
  int n, len, off;  // new tokens, keys, keys before the first new token
  int64_t t0;
};

__device__ __forceinline__ Seq get_seq(const Args& a, int b) {
  Seq s;
  int64_t c0 = b, c1 = b + 1;
  if (a.cu) c0 = a.cu[b], c1 = a.cu[b + 1];
  const int len = a.lens[b];
  const int64_t most = a.width * a.page;
  s.len = len < 0 ? 0 : (len < most ? len : (int)most);
  s.off = (int)(len - (c1 - c0));
  if (c1 > a.T) c1 = a.T;
  s.n = c0 < 0 || c1 <= c0 ? 0 : (int)(c1 - c0);
  s.t0 = c0;
  return s;
}

// keys that the sequence's first `i` new tokens see
__device__ __forceinline__ int seen_by(const Args& a, const Seq& s, int i) {
  if (!a.causal) return s.len;
  const int v = s.off + i;
  return v < 0 ? 0 : (v < s.len ? v : s.len);
}

// key tiles of tokens [i0, i1): 0 if there are no such tokens
template <int KT>
__device__ __forceinline__ int tiles_of(const Args& a, const Seq& s, int i0, int i1) {
  if (i0 >= s.n) return 0;
  return (int)(((uint32_t)seen_by(a, s, i1 < s.n ? i1 : s.n) + KT - 1) / KT);
}

struct Segment {  // key tiles [t0, t1) of an item's [0, tiles)
  int b, h, rt, t0, t1, tiles;
  Seq s;
};

// Walks over a CTA's segments.  Items with no key count as one tile, so that their rows (zeros)
// have an owner.
template <int KT>
struct Walk {
  int64_t unit, end;
  int b, h, rt, t0;
  Seq s;

  __device__ int item_tiles(const Args& a) const {
    const int t = tiles_of<KT>(a, s, rt * a.tokens, (rt + 1) * a.tokens);
    return t > 0 ? t : 1;
  }
  __device__ bool next(const Args& a, Segment& g) {
    if (unit >= end) return false;
    const int tiles = item_tiles(a);
    g.b = b, g.h = h, g.rt = rt, g.t0 = t0, g.tiles = tiles, g.s = s;
    g.t1 = (int64_t)(tiles - t0) < end - unit ? tiles : t0 + (int)(end - unit);
    unit += g.t1 - t0;
    t0 = 0;
    if (unit < end) {
      if (++rt * a.tokens >= s.n) {
        rt = 0;
        if (++h == a.Hk) {
          h = 0;
          do s = get_seq(a, ++b); while (s.n == 0);
        }
      }
    }
    return true;
  }
};

struct Found {
  int64_t rem, head;  // the walk's place in its sequence, tiles of a key head there
  int b;
};

// What all items together are.
struct Total {
  int64_t units, items;
  int most;  // the longest item
};

template <int KT>
__device__ __forceinline__ int item_units(const Args& a, const Seq& s, int rt) {
  const int t = tiles_of<KT>(a, s, rt * a.tokens, (rt + 1) * a.tokens);
  return t > 0 ? t : 1;
}

// Work on all sequences, `lanes` threads a sequence (a power of two, a warp at most).
template <int KT, int kThreads>
struct Crew {
  int lanes, seqs, me, at;  // sequences side by side; this thread's among them, and its place there

  __device__ explicit Crew(int B) {
    lanes = 32;
    while (lanes > 1 && B * lanes > kThreads) lanes >>= 1;
    seqs = kThreads / lanes;
    me = threadIdx.x / lanes;
    at = threadIdx.x & (lanes - 1);
  }
  // units of one key head of sequence b, on all of its threads; 0 past the last
  __device__ int64_t head_units(const Args& a, int64_t b, int& tiles) const {
    tiles = 0;
    int64_t u = 0;
    if (b < a.B) {
      const Seq s = get_seq(a, (int)b);
      tiles = (s.n + a.tokens - 1) / a.tokens;
      if (a.causal) {
        for (int r = at; r < tiles; r += lanes) u += item_units<KT>(a, s, r);
      } else if (at == 0 && tiles) {
        u = (int64_t)tiles * item_units<KT>(a, s, 0);
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    return u;
  }
};

// Inclusive prefix sum over the warp.
template <typename I>
__device__ __forceinline__ I warp_scan(I x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// What a thread knows of its sequence of the first round: tiles of a key head, of all, and of the
// sequences before it.
struct First {
  int64_t head, units, before;
};

// Every thread of the block.  kItems: also their number and the longest one.
template <int KT, int kThreads, bool kItems>
__device__ Total count_all(const Args& a, const Crew<KT, kThreads>& crew, First& first, int64_t* sums) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t units = 0, items = 0;
  int most = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += crew.seqs) {
    int tiles;
    const int64_t hu = crew.head_units(a, b0 + crew.me, tiles);
    const int64_t u = crew.at == 0 ? hu * a.Hk : 0;
    if (b0 == 0) first.head = hu, first.units = u;
    units += u;
    if (kItems && crew.at == 0 && tiles) {
      items += (int64_t)tiles * a.Hk;
      most = max(most, item_units<KT>(a, get_seq(a, (int)(b0 + crew.me)), tiles - 1));
    }
  }
  // with one round the sum's own prefix is the place of each sequence
  const int64_t x = warp_scan(units);
  if (lane == 31) sums[warp] = x;
  if (kItems) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      items += __shfl_xor_sync(0xffffffffu, items, o);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    if (lane == 0) sums[kWarps + warp] = items, sums[2 * kWarps + warp] = most;
  }
  __syncthreads();
  Total t = {0, 0, 0};
  first.before = x - units;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) first.before += sums[i];
    t.units += sums[i];
    if (kItems) t.items += sums[kWarps + i], t.most = max(t.most, (int)sums[2 * kWarps + i]);
  }
  return t;
}

// Every thread of the block; finds the walk of this CTA, `per` tiles a CTA.
template <int KT, int kThreads>
__device__ void start_walk(const Args& a, const Crew<KT, kThreads>& crew, const Total& total,
                           const First& first, int64_t per, Walk<KT>& w, Found* sh, int64_t* sums) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = (int64_t)blockIdx.x * per;
  w.unit = unit;
  w.end = unit + per < total.units ? unit + per : total.units;
  if (unit >= total.units) return;  // nothing here (the same for every thread)
  if (a.B <= crew.seqs) {
    if (first.units > 0 && first.before <= unit && unit < first.before + first.units)
      sh->b = crew.me, sh->rem = unit - first.before, sh->head = first.head;
    __syncthreads();
  } else {
    int64_t base = 0;
    for (int64_t b0 = 0; b0 < a.B; b0 += crew.seqs) {
      int tiles;
      const int64_t hu = crew.head_units(a, b0 + crew.me, tiles);
      const int64_t u = crew.at == 0 ? hu * a.Hk : 0;
      const int64_t x = warp_scan(u);
      __syncthreads();
      if (lane == 31) sums[warp] = x;
      __syncthreads();
      int64_t before = base + x - u, all = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sums[i];
        all += sums[i];
      }
      if (u > 0 && before <= unit && unit < before + u)
        sh->b = (int)(b0 + crew.me), sh->rem = unit - before, sh->head = hu;
      base += all;
      __syncthreads();
      if (base > unit) break;
    }
  }
  w.b = sh->b;
  int64_t rem = sh->rem;
  w.s = get_seq(a, w.b);
  w.h = (int)(rem / sh->head);
  rem -= w.h * sh->head;
  w.rt = 0;
  if (!a.causal) {
    const int t = w.item_tiles(a);
    w.rt = (int)(rem / t);
    rem -= (int64_t)w.rt * t;
  } else {
    // a warp at a time: 32 items
    for (;; w.rt += 32) {
      const int x = warp_scan(item_units<KT>(a, w.s, w.rt + lane));
      const uint32_t past = __ballot_sync(0xffffffffu, x > rem);
      const int to = past ? __ffs(past) - 1 : 32;
      rem -= to ? __shfl_sync(0xffffffffu, x, to - 1) : 0;
      if (past) {
        w.rt += to;
        break;
      }
    }
  }
  w.t0 = (int)rem;
}

// One warp: item number `place` of all items in the order of their length, longest first.  Items
// of a sequence grow along it, so how many have at least t tiles follows from one division; a
// binary search over t, a sum over the sequences a step, finds the length at that place.  `mine`:
// sequence number `lane`, read once.
template <int KT>
__device__ Segment item_at(const Args& a, uint32_t place, int most, const Seq& mine) {
  const int lane = threadIdx.x & 31;
  auto seq = [&](int b) { return b < 32 ? mine : get_seq(a, b); };  // b % 32 == lane
  // items of a key head of sequence b with at least t tiles (every item counts as one)
  auto at_least = [&](const Seq& s, int t) -> int {
    const int tiles = (int)((uint32_t)(s.n + a.tokens - 1) / (uint32_t)a.tokens);
    if (t <= 1 || tiles == 0) return tiles;
    const int64_t x = (int64_t)(t - 1) * KT;  // seen keys > x
    if (s.len <= x) return 0;
    if (!a.causal) return tiles;
    const int64_t i = x - s.off;  // tokens of the chunk that do not reach
    if (i >= s.n) return 0;
    const int first = i < 0 ? 0 : (int)((uint32_t)i / (uint32_t)a.tokens);
    return tiles - min(first, tiles - 1);
  };
  auto all_at_least = [&](int t) {  // there are fewer than 2^30 items
    uint32_t n = 0;
    for (int b = lane; b < a.B; b += 32) n += at_least(seq(b), t);
    return __reduce_add_sync(0xffffffffu, n) * (uint32_t)a.Hk;
  };
  int lo = 1, hi = most;  // the largest t with more than `place` items of at least t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (all_at_least(mid) > place) lo = mid; else hi = mid - 1;
  }
  uint32_t k = place - all_at_least(lo + 1);  // among those of lo tiles
  Segment g;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    Seq s = {};
    int n = 0, above = 0;
    if (b < a.B) {
      s = seq(b);
      above = at_least(s, lo + 1);
      n = at_least(s, lo) - above;
    }
    const uint32_t x = warp_scan((uint32_t)n * (uint32_t)a.Hk);
    const uint32_t past = __ballot_sync(0xffffffffu, x > k);
    if (!past) {
      if (b0 + 32 >= a.B) {  // not reached: every place has an item
        g.b = -1;
        return g;
      }
      k -= __shfl_sync(0xffffffffu, x, 31);
      continue;
    }
    const int to = __ffs(past) - 1;
    k -= __shfl_sync(0xffffffffu, x - (uint32_t)n * (uint32_t)a.Hk, to);
    n = __shfl_sync(0xffffffffu, n, to);
    above = __shfl_sync(0xffffffffu, above, to);
    g.b = b0 + to;
    g.s.n = __shfl_sync(0xffffffffu, s.n, to);
    g.s.len = __shfl_sync(0xffffffffu, s.len, to);
    g.s.off = __shfl_sync(0xffffffffu, s.off, to);
    g.s.t0 = __shfl_sync(0xffffffffu, s.t0, to);
    g.h = (int)(k / (uint32_t)n);
    g.rt = (int)((uint32_t)(g.s.n + a.tokens - 1) / (uint32_t)a.tokens) - above - 1 - ((int)k - g.h * n);
    g.t0 = 0;
    g.t1 = g.tiles = item_units<KT>(a, g.s, g.rt);
    return g;
  }
}

// One thread: the record of an item that begins in this CTA and ends in another.
template <int KT>
__device__ void write_rec(const Args& a, Walk<KT> w, int64_t per) {
  int32_t* r = a.rec + (int64_t)blockIdx.x * 8;
  Segment g;
  int valid = 0;
  int64_t at = w.unit;
  while (w.next(a, g)) {
    if (g.t0 == 0 && g.t1 < g.tiles) {
      valid = 1;
      r[1] = g.b, r[2] = g.h, r[3] = g.rt;
      r[4] = (int32_t)((at + g.tiles - 1) / per);
    }
    at += g.t1 - g.t0;
  }
  r[0] = valid;
}

// Lets the merge kernel be set up while this one runs.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// kRange: the largest power of two that weights have room for.  A weight is rounded to the type for
// its product with v, and below the type's normal numbers that is no longer relative to it: in fp16 the
// many small weights of a long cache would be lost beside one that is 2^25 times each of them.  So all
// weights carry a factor 2^shift, sum and O alike, that takes the largest near the top of the range;
// it drops out in the division.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;  // tcgen05 operand format
  static constexpr float kRange = 0.f;  // normal numbers go down to 2^-126: no need
  __device__ static uint32_t pack(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
  }
  __device__ static void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Pair<__half> {
  static constexpr uint32_t kFmt = 0;
  static constexpr float kRange = 15.f;
  __device__ static uint32_t pack(float lo, float hi) {
    __half2 b = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
  }
  __device__ static void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// ===========================================================================
// Few rows: 16 packed rows against 64 keys a step, 16 of them a warp.
//
// Each warp streams its own 16-key strips (cp.async into its own ring, no block barrier in the
// loop), multiplies them with mma.sync (a 128-row tensor-memory tile would be 7/8 empty, and at
// these rates the cache's bytes bound the loop, not the products) and keeps its own maximum, sum
// and O; the four warps join through shared memory at the end of a segment.
// ===========================================================================
namespace dec {

constexpr int kThreads = 128, kRows = 16, kKeys = 64, kLeast = 2;
constexpr int kRing = 96 * 1024;  // two CTAs an SM: 192 KB in flight

template <int D>
struct Shape {
  static constexpr int kRowBytes = D * 2, kChunks = D / 8;
  static constexpr int kStage = 2 * 16 * kRowBytes;           // K and V strip of a warp
  static constexpr int kStages = kRing / (4 * kStage);
  static_assert(kStage == 16 * D * 4, "a stage holds 16 rows of floats");
};

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(take ? 16 : 0)
               : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) decode_kernel(const Args a) {
  using S = Shape<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Found found;
  __shared__ int64_t sums[3 * kThreads / 32];
  __shared__ float s_ml[4][kRows][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  let_next_start();
  Walk<kKeys> w;
  const Crew<kKeys, kThreads> crew(a.B);
  First first;
  const Total total = count_all<kKeys, kThreads, false>(a, crew, first, sums);
  int64_t per = (total.units + a.ctas - 1) / a.ctas;
  if (per < kLeast) per = kLeast;
  start_walk<kKeys>(a, crew, total, first, per, w, &found, sums);
  if (threadIdx.x == 0) write_rec(a, w, per);

  uint8_t* ring = smem + warp * (S::kStages * S::kStage);
  const uint32_t ring_u = smem_u32(ring);
  const T* const kp = reinterpret_cast<const T*>(a.k);
  const T* const vp = reinterpret_cast<const T*>(a.v);
  const int qrow = lane >> 2, qcol = (lane & 3) * 2;

  int base = 0;  // ring stage of a segment's first strip
  int pid = -1;  // page of the strip that is loaded next
  auto strip = [&](const Segment& g, int j) { return (g.t0 + j) * kKeys + warp * 16; };
  // keys that the tile's last token sees: those past them are not loaded
  auto last_seen = [&](const Segment& g) { return seen_by(a, g.s, min(g.s.n, (g.rt + 1) * a.tokens)); };
  auto page_of = [&](const Segment& g, int vis, int j) {  // (pages are multiples of 16 rows)
    const int key = strip(g, j);
    return j < g.t1 - g.t0 && key < vis ? __ldg(a.table + (int64_t)g.b * a.width + key / a.page) : -1;
  };
  auto load = [&](const Segment& g, int vis, int j, int stage) {
    const int key = strip(g, j);
    if (j < g.t1 - g.t0 && key < vis) {
      const bool in = pid >= 0 && pid < a.pages;
      const int slot = key % a.page;
      const int64_t p = in ? pid : 0;
      const T* ks = kp + p * a.k_page + (int64_t)slot * a.k_slot + g.h * a.k_head;
      const T* vs = vp + p * a.v_page + (int64_t)slot * a.v_slot + g.h * a.v_head;
      const uint32_t st = ring_u + (uint32_t)(stage * S::kStage);
      const int c = lane % S::kChunks;
#pragma unroll
      for (int i = 0; i < S::kChunks / 2; ++i) {
        const int r = i * (32 / S::kChunks) + lane / S::kChunks;
        const uint32_t dst = st + (uint32_t)(r * S::kRowBytes + ((c ^ (r & 7)) << 4));
        const bool take = in && key + r < g.s.len;
        const int rr = take ? r : 0;
        cp_async16_or_zero(dst, ks + rr * a.k_slot + c * 8, take);
        cp_async16_or_zero(dst + S::kStage / 2, vs + rr * a.v_slot + c * 8, take);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // a segment's first strips, but for one stage of the ring; page numbers are fetched one strip
  // ahead of the strip that needs them
  auto begin = [&](const Segment& g, int vis) {
    pid = page_of(g, vis, 0);
#pragma unroll 1
    for (int j = 0; j < S::kStages - 1; ++j) {
      const int nx = page_of(g, vis, j + 1);
      load(g, vis, j, (base + j) % S::kStages);
      pid = nx;
    }
  };

  // Q of a segment: fragments of its tile, and the keys that this thread's two rows see
  uint32_t qf[D / 16][4];
  int lim[2], row0, rows;
  auto load_q = [&](const Segment& g) {
    row0 = g.rt * a.rows;
    rows = min(g.s.n * a.g - row0, a.rows);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = qrow + 8 * hh;
      const bool ok = r < rows;
      const int pr = row0 + (ok ? r : 0);
      const int i = pr / a.g;
      const T* qp = reinterpret_cast<const T*>(a.q) + (g.s.t0 + i) * a.q_token +
                    (int64_t)(g.h * a.g + pr - i * a.g) * a.q_head + qcol;
      lim[hh] = ok ? seen_by(a, g.s, i + 1) : 0;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][hh] = ok ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
        qf[kk][hh + 2] = ok ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
      }
    }
  };

  Segment g;
  bool more = w.next(a, g);
  int vis = more ? last_seen(g) : 0;
  if (more) {
    begin(g, vis);
    load_q(g);
  }
  while (more) {
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const int steps = g.t1 - g.t0;
    int stage = base;  // of strip j; the one before it is loaded next
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const int nx = page_of(g, vis, j + S::kStages);
      cp_async_wait<S::kStages - 2>();
      __syncwarp();  // strip j is there for every lane, strip j - 1 has been read by every lane
      load(g, vis, j + S::kStages - 1, stage == 0 ? S::kStages - 1 : stage - 1);
      pid = nx;
      const int key0 = strip(g, j);
      const uint32_t ks = ring_u + (uint32_t)(stage * S::kStage);
      const uint32_t vs = ks + S::kStage / 2;
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      if (key0 >= vis) continue;
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        const int r = ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];
          ldsm4(ks + (uint32_t)(r * S::kRowBytes + (((kk * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4)), b);
          Pair<T>::mma(sc[0], qf[kk], b[0], b[1]);
          Pair<T>::mma(sc[1], qf[kk], b[2], b[3]);
        }
      }
      float alpha[2];
      bool grew = false;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[t][hh * 2 + e];
            x = key0 + t * 8 + qcol + e < lim[hh] ? x * a.scale_log2 : -INFINITY;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[hh], mx);
        alpha[hh] = mn == -INFINITY ? 1.f : ex2_approx(m[hh] - mn);
        grew |= mn > m[hh];
        m[hh] = mn;
        const float sub = mn == -INFINITY ? 0.f : mn;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[t][hh * 2 + e];
            x -= sub;
            if (Pair<T>::kRange > 0.f) x += Pair<T>::kRange;  // (of the difference: exact however large x is)
            x = ex2_approx(x);
            sum += x;
          }
        l[hh] = l[hh] * alpha[hh] + sum;  // this lane's four keys; the quad joins at the end
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= alpha[0], o[i][1] *= alpha[0];
          o[i][2] *= alpha[1], o[i][3] *= alpha[1];
        }
      }
      // P rounded to 16 bits, as the tensor cores take it: off by up to 2^-8 (bf16) or 2^-11 (fp16) of a
      // weight (fp16: or 2^-40 of the largest, if that is more); the sum takes it unrounded
      const uint32_t p[4] = {Pair<T>::pack(sc[0][0], sc[0][1]), Pair<T>::pack(sc[0][2], sc[0][3]),
                             Pair<T>::pack(sc[1][0], sc[1][1]), Pair<T>::pack(sc[1][2], sc[1][3])};
      const int r = (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t b[4];
        ldsm4t(vs + (uint32_t)(r * S::kRowBytes + (((i * 2 + (lane >> 4)) ^ (r & 7)) << 4)), b);
        Pair<T>::mma(o[2 * i], p, b[0], b[1]);
        Pair<T>::mma(o[2 * i + 1], p, b[2], b[3]);
      }
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
      l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
    }
    __syncwarp();  // every lane has read the last strip
    // The next segment's first strips are loaded while this one is joined; the join takes the
    // stage that they leave out, the last strip's: 16 rows of D floats fill it, its 16-byte chunks
    // in an order of their row's against bank conflicts.
    base = stage;
    const int free_stage = (stage == 0 ? S::kStages : stage) - 1;
    const Segment was = g;
    const int was_row0 = row0, was_rows = rows;
    more = w.next(a, g);
    if (more) {
      vis = last_seen(g);
      begin(g, vis);
      load_q(g);
    }
    auto joint = [&](int wp, int r, int chunk) {
      return reinterpret_cast<float*>(smem + (wp * S::kStages + free_stage) * S::kStage) + r * D +
             ((chunk ^ (r & 7)) << 2);
    };
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = qrow + 8 * hh;
      if (r < was_rows) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(joint(warp, r, i * 2 + (qcol >> 2)) + (qcol & 3)) =
              make_float2(o[i][2 * hh], o[i][2 * hh + 1]);
        if ((lane & 3) == 0) s_ml[warp][r][0] = m[hh], s_ml[warp][r][1] = l[hh];
      }
    }
    __syncthreads();
    const bool whole = was.t0 == 0 && was.t1 == was.tiles;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (was.t0 == 0);
    for (int idx = threadIdx.x; idx < was_rows * (D / 4); idx += kThreads) {
      const int r = idx / (D / 4), c = (idx % (D / 4)) * 4;
      float mm = s_ml[0][r][0];
#pragma unroll
      for (int i = 1; i < 4; ++i) mm = fmaxf(mm, s_ml[i][r][0]);
      const float sub = mm == -INFINITY ? 0.f : mm;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float ll = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = ex2_approx(s_ml[i][r][0] - sub);
        const float4 v = *reinterpret_cast<const float4*>(joint(i, r, c >> 2));
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
        ll = fmaf(f, s_ml[i][r][1], ll);
      }
      if (whole) {
        const int pr = was_row0 + r, i = pr / a.g;
        // A row that sees no key is 0, whatever the values that other rows of its tile see.  One that
        // sees some is not: without a finite score its maximum is -inf too, and the result NaN.
        const bool sees = seen_by(a, was.s, i + 1) > 0;
        const float inv = sees ? 1.f / ll : 0.f;
        if (!sees) acc = make_float4(0.f, 0.f, 0.f, 0.f);
        T* dst = reinterpret_cast<T*>(a.out) + (was.s.t0 + i) * a.o_token +
                 (int64_t)(was.h * a.g + pr - i * a.g) * a.o_head + c;
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * kRows + r) * D + c) = acc;
        if (c == 0)
          *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = make_float2(mm, ll);
      }
    }
    __syncthreads();  // the joint's stage is loaded again
  }
  cp_async_wait<0>();
}

}  // namespace dec

// ===========================================================================
// Many rows: 256 packed rows (two tiles of 128, "A" and "B") against 128 keys a step.
//
// Both tiles read the same key and value tiles from one ring, so a key crosses L2 once for 256
// rows.  Per tile a warpgroup of softmax threads (a thread owns a row) and one warp that issues
// its MMAs; one warp loads, one works the segments out.  Tensor memory: one score buffer that the tiles take in turn (a tile's
// softmax copies its scores to registers, and the buffer is the other's), P_A, P_B as packed
// 16-bit pairs, O_A, O_B.  O stays there for a whole segment; the running maximum is raised only
// when a tile's exceeds it by more than 2^8, and O is rescaled in place then.
// ===========================================================================
namespace chunk {

constexpr int kThreads = 384, kRows = 256, kKeys = 128, kLeast = 2;
constexpr int kCut = 12;  // key tiles, see where items are dealt out
constexpr int kAtom = 128 * 128;  // 128 rows x 64 channels of 16 bits, 128-byte swizzle
constexpr float kLazy = 8.0f;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;
// the factor of all weights: with kLazy above it they fill the range.  Maxima from kShifted on do
// without it: their difference from it would be rounded, by whole powers of two in the end.
template <typename T>
constexpr float kShift = Pair<T>::kRange > kLazy ? Pair<T>::kRange - kLazy : 0.f;
constexpr float kShifted = 1048576.f;

template <int D>
struct Shape {
  static constexpr int kTile = D * 256;  // bytes of 128 rows
  static constexpr int kSlots = D == 128 ? 2 : 4;  // of K and of V
  static constexpr size_t kSmem = (size_t)kTile * (2 + 2 * kSlots) + 1024 + 1024;  // alignment, barriers
};

// p = 2^(round(s c) - m) of 64 scores, m one of those products: near it the difference is exact.  In one
// rounding, 2^(s c - m), every weight would carry what the maximum's own product was rounded by, up to
// half a step of m: by it fp16 overflows from scores of 2^27 on, bf16 from 2^31 (finite scores, NaN
// results).  `zero` keeps the compiler from joining the two.  That costs 1-6%: 7 of up to 1537 tokens over
// up to 1001, 16 / 4 x 64, 64.7 -> 66.5 us; 8448 over 33792 keys 1675 -> 1697 under lasting load; 32 of
// up to 600 over up to 600, 32 / 8 x 128, pages of 16, 160 -> 170.  Branches to a rare exact path cost
// 10-15%, predicated differences 20-30%.
//
// Packed as 16 bits (a weight is off by up to 2^-8 of itself in bf16, by 2^-11 or 2^-32 of the largest in
// fp16); fp32 row sum of the unrounded ones into acc2.  All on the special-function unit: an eighth or a
// quarter of them as polynomials on the FMA pipe took 8448 over 33792 keys from 1424 to 1412 us, the
// ragged chunks above from 169 to 186-189 us, those of D 64 from 65 to 66-67 (before `zero`).
template <typename T>
__device__ __forceinline__ void exp_pack64(const uint32_t* s, uint64_t cc, uint64_t zero, uint64_t nm,
                                           uint64_t& acc2, uint32_t* pk) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint64_t xv =
        f2_add(f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), cc, zero), nm);
    float x0, x1;
    f2_unpack(xv, x0, x1);
    const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
    acc2 = f2_add(acc2, f2_pack(p0, p1));
    pk[i] = Pair<T>::pack(p0, p1);
  }
}

// the largest of 64 scores
__device__ __forceinline__ float max64(const uint32_t* s) {
  float mx[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
    mx[t] = fmax3(__uint_as_float(s[t]), __uint_as_float(s[4 + t]), __uint_as_float(s[8 + t]));
#pragma unroll
  for (int i = 12; i < 60; i += 8) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      mx[t] = fmax3(mx[t], __uint_as_float(s[i + t]), __uint_as_float(s[i + 4 + t]));
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) mx[t] = fmaxf(mx[t], __uint_as_float(s[60 + t]));
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

__device__ __forceinline__ void add_release(uint32_t* p, uint32_t v) {
  asm volatile("red.release.cta.shared::cta.add.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
// Bounded wait, as mbar_wait, for a count in shared memory to reach `v`.
__device__ __forceinline__ bool wait_count(uint32_t* p, uint32_t v, unsigned code) {
  uint64_t t0 = 0;
  for (uint32_t i = 0;; ++i) {
    uint32_t x;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(x) : "r"(smem_u32(p)) : "memory");
    if ((int32_t)(x - v) >= 0) return true;
    if ((i & 255u) == 255u) {
      const uint64_t t = globaltimer_ns();
      if (!t0) t0 = t;
      if (t - t0 > kWaitLimitNs) break;
    }
  }
  atomicCAS(&g_device_error, 0u, code);
  return false;
}

// A segment as one warp works it out for the others.
struct Desc {
  int more;       // 0: there are no further segments
  int cnt[2], all;  // key tiles of either half, and of the longer one
  int key_t0, b, h, len;
  int n, off, row0, whole;
  int64_t t0;
};
constexpr int kDescs = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const int box, const Args a) {
  using S = Shape<D>;
  constexpr int kSlots = S::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* const sQ = base;
  uint8_t* const sK = base + 2 * S::kTile;
  uint8_t* const sV = sK + kSlots * S::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kSlots * S::kTile);
  enum { Q_FULL = 0, Q_EMPTY, S_FULL, S_FREE, P_FULL, PV_DONE, DRAIN, kNB };
  auto BAR = [&](int x, int i) { return bars + x * kNB + i; };
  uint64_t* const k_full = bars + 2 * kNB;
  uint64_t* const k_empty = k_full + kSlots;
  uint64_t* const v_full = k_empty + kSlots;
  uint64_t* const v_empty = v_full + kSlots;
  uint64_t* const d_full = v_empty + kSlots;  // segments: one writer, 11 readers
  uint64_t* const d_empty = d_full + kDescs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + kDescs);
  __shared__ Desc descs[kDescs];
  // Score tiles that each tile's softmax has copied out, counted at the end of a segment (four
  // warps each).  A parity names a phase only to a waiter that is at most one behind, and a tile
  // that sits out keys which the other one sees falls further behind than that.
  __shared__ uint32_t s_copied[2];
  __shared__ Found found;
  __shared__ int64_t sums[3 * kThreads / 32];

  const int warp = warp_id_uniform();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_copied[0] = s_copied[1] = 0;
    for (int x = 0; x < 2; ++x)
      for (int b = 0; b < kNB; ++b)
        mbar_init(BAR(x, b), (b == S_FREE || b == P_FULL) ? 4u : 1u);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(k_empty + i, 2);
      mbar_init(v_empty + i, 2);
    }
    for (int i = 0; i < kDescs; ++i) {
      mbar_init(d_full + i, 1);
      mbar_init(d_empty + i, 11);
    }
    fence_mbar_init();
  }
  if (warp == 10) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  let_next_start();
  // Cut items at CTA boundaries, or whole ones to each CTA, longest first and there and back (so the
  // longest is paired with the shortest of the next round)?  A cut costs both CTAs a write of 256 rows
  // of floats and the join their reads: 18 us for all, about kCut tiles' time.  Whole items cost
  // what the last, incomplete round leaves idle, or an item longer than a CTA's share.
  Walk<kKeys> w = {};
  const Crew<kKeys, kThreads> crew(a.B);
  First first;
  const Total total = count_all<kKeys, kThreads, true>(a, crew, first, sums);
  int64_t per = (total.units + a.ctas - 1) / a.ctas;
  if (per < kLeast) per = kLeast;
  const int64_t rounds = (total.items + a.ctas - 1) / a.ctas;
  const bool cut = total.items < a.ctas || total.most > per + kCut ||
                   (rounds * a.ctas - total.items) * total.units > kCut * a.ctas * total.items;
  if (cut) start_walk<kKeys>(a, crew, total, first, per, w, &found, sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  uint32_t seg = 0;  // segments seen
  auto DESC = [&]() -> const Desc& { return descs[seg % kDescs]; };
  // the next segment; false at the end, or after a time-out
  auto next_segment = [&]() {
    return mbar_wait(d_full + seg % kDescs, (seg / kDescs) & 1u, 0x90eu) && DESC().more;
  };

  if (warp == 8) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    const int boxes = kKeys / box;
    const int half_rows = a.rows >> 1;
    bool ok = true;
    int64_t nk = 0, nv = 0;       // tiles issued
    uint32_t nq[2] = {0, 0};
    // a tile is `boxes` boxes of `box` rows, each inside one page; lane i loads box i.  Page
    // numbers are fetched a tile ahead, and V takes K's.
    struct Place {
      int row, page;  // in the page; past the sequence's end, and numbers outside the pool: zeros
    };
    auto look = [&](int j) {
      const Desc& g = DESC();
      const int key = (g.key_t0 + j) * kKeys + lane * box;
      const int at = (int)((uint32_t)key / (uint32_t)a.page);
      Place p = {key - at * a.page, -1};
      if (lane < boxes && key < g.len) p.page = __ldg(a.table + g.b * a.width + at);
      return p;
    };
    auto tile = [&](uint8_t* ring, const CUtensorMap& tm, uint64_t* full, uint64_t* empty,
                    int64_t& count, const Place& p) {
      const int s = (int)(count % kSlots);
      const uint32_t ph = (uint32_t)(count / kSlots) & 1u;
      if (!__all_sync(0xffffffffu, mbar_wait(empty + s, ph ^ 1u, 0x901u))) return false;
      if (lane == 0) mbar_arrive_expect_tx(full + s, S::kTile);
      __syncwarp();
      if (lane < boxes) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(ring + s * S::kTile + c * kAtom + lane * box * 128, &tm, full + s, c * 64, DESC().h,
                      p.row, p.page);
      }
      ++count;
      return true;
    };
    while (ok && __all_sync(0xffffffffu, next_segment())) {
      const int all = DESC().all;
      Place now = look(0), before = now;
      // Q of both halves: boxes of a token's g heads for 128 / g tokens (rows past the
      // sequence's end are other tokens', or zeros: nobody stores them)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!ok || DESC().cnt[x] == 0) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(BAR(x, Q_EMPTY), (nq[x] & 1u) ^ 1u, 0x912u))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const Desc& g = DESC();
          mbar_arrive_expect_tx(BAR(x, Q_FULL), (uint32_t)(half_rows * D * 2));
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(sQ + x * S::kTile + c * kAtom, &tmQ, BAR(x, Q_FULL), c * 64, g.h * a.g,
                        (int)g.t0 + (g.row0 + x * half_rows) / a.g, 0);
        }
        __syncwarp();
        ++nq[x];
      }
      // the MMA threads take K(0) K(1) V(0) K(2) V(1) ...
      for (int j = 0; j <= all && all > 0 && ok; ++j) {
        const Place next = j + 1 < all ? look(j + 1) : now;
        if (j < all) ok = tile(sK, tmK, k_full, k_empty, nk, now);
        if (ok && j >= 1) ok = tile(sV, tmV, v_full, v_empty, nv, before);
        before = now;
        now = next;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(d_empty + seg % kDescs);
      ++seg;
    }
    // no load may still be writing shared memory when the CTA exits
    if (lane == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (nq[x]) mbar_wait(BAR(x, Q_FULL), (nq[x] - 1) & 1u, 0x902u);
      for (int64_t i = nk > kSlots ? nk - kSlots : 0; i < nk; ++i)
        mbar_wait(k_full + i % kSlots, (uint32_t)(i / kSlots) & 1u, 0x902u);
      for (int64_t i = nv > kSlots ? nv - kSlots : 0; i < nv; ++i)
        mbar_wait(v_full + i % kSlots, (uint32_t)(i / kSlots) & 1u, 0x902u);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ segments
    const Walk<kKeys> start = w;
    Seq mine = {};
    if (lane < a.B) mine = get_seq(a, lane);
    Segment g;
    int64_t round = 0;
    for (bool more = true; more; ++seg) {
      if (cut) {
        more = w.next(a, g);
      } else {
        const int64_t place = round * a.ctas + (round & 1 ? a.ctas - 1 - blockIdx.x : blockIdx.x);
        more = place < total.items;
        if (more) g = item_at<kKeys>(a, (uint32_t)place, total.most, mine);
        more = more && g.b >= 0;
        ++round;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(d_empty + seg % kDescs, ((seg / kDescs) & 1u) ^ 1u, 0x90fu)))
        break;
      if (lane == 0) {
        Desc& d = descs[seg % kDescs];
        d.more = more;
        if (more) {
          const int half = a.tokens >> 1, i0 = g.rt * a.tokens;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int tl = tiles_of<kKeys>(a, g.s, i0 + x * half, i0 + (x + 1) * half);
            const int e = tl < g.t1 ? tl : g.t1;
            d.cnt[x] = e > g.t0 ? e - g.t0 : 0;
          }
          d.all = d.cnt[0] > d.cnt[1] ? d.cnt[0] : d.cnt[1];
          d.key_t0 = g.t0, d.b = g.b, d.h = g.h, d.len = g.s.len, d.n = g.s.n, d.off = g.s.off;
          d.row0 = g.rt * a.rows, d.whole = g.t0 == 0 && g.t1 == g.tiles, d.t0 = g.s.t0;
        }
        mbar_arrive(d_full + seg % kDescs);
      }
      __syncwarp();
    }
    if (lane == 0) {
      if (cut) write_rec(a, start, per);
      else a.rec[(int64_t)blockIdx.x * 8] = 0;
    }
  } else if (warp >= 10) {
    // ------------------------------------------------------------ MMA issuer of tile x
    // The whole warp walks the loop, so that descriptors and addresses stay warp-uniform (the form
    // the tensor instructions take them in), and one elected lane issues: from a branch of one
    // lane the eight instructions of a product took 800 clocks to issue, 512 to run.
    const int x = warp - 10;
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = make_idesc(Pair<T>::kFmt, Pair<T>::kFmt, 0, 0, 128, 128);
    constexpr uint32_t idesc_o = make_idesc(Pair<T>::kFmt, Pair<T>::kFmt, 0, 1, 128, D);
    const uint64_t dq = smem_desc_sw128(smem_u32(sQ + x * S::kTile), 16, 1024);
    const uint64_t dk = smem_desc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t dv = smem_desc_sw128(smem_u32(sV), (uint32_t)kAtom, 1024);
    const uint32_t tP = tmem + kColP + (uint32_t)(x * 64);
    const uint32_t tO = tmem + kColO + (uint32_t)(x * 128);
    uint64_t* const free_mine = BAR(x, S_FREE);
    uint64_t* const free_other = BAR(x ^ 1, S_FREE);
    bool ok = true;
    uint32_t mine = 0, other = 0, segs = 0;  // tiles of x, of the other, segments
    uint32_t ks = 0, kph = 0, vs = 0, vph = 0;  // ring slots and their parities
    auto wait = [&](uint64_t* bar, uint32_t index, unsigned code) {
      if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, index & 1u, code))) ok = false;
    };
    auto step = [&](uint32_t& slot, uint32_t& parity) {
      if (++slot == kSlots) slot = 0, parity ^= 1u;
    };
    while (ok && __all_sync(0xffffffffu, next_segment())) {
      const int cm = __shfl_sync(0xffffffffu, DESC().cnt[x], 0);
      const int co = __shfl_sync(0xffffffffu, DESC().cnt[x ^ 1], 0);
      const int all = __shfl_sync(0xffffffffu, DESC().all, 0);
      if (leader) mbar_arrive(d_empty + seg % kDescs);
      ++seg;
      if (cm > 0) wait(BAR(x, Q_FULL), segs, 0x903u);
      // The score buffer holds S_A(0) S_B(0) S_A(1) S_B(1) ... (a tile past its count drops
      // out); S_x(j) waits until the softmax of the occupant before it has copied it out.
      auto issue_s = [&](int j) {
        if (!ok || j >= cm) return;
        if (j == 0) {  // the buffer is free of the last segment's scores
          if (!__all_sync(0xffffffffu, wait_count(s_copied + (x ^ 1), 4 * other, 0x904u) &&
                                           wait_count(s_copied + x, 4 * mine, 0x904u)))
            ok = false;
        }
        if (x == 0) {
          if (j >= 1) {
            if (j - 1 < co) wait(free_other, other + j - 1, 0x904u);
            else wait(free_mine, mine + j - 1, 0x904u);
          }
        } else {
          if (j < co) wait(free_other, other + j, 0x904u);
          else if (j >= 1) wait(free_mine, mine + j - 1, 0x904u);
        }
        wait(k_full + ks, kph, 0x905u);
        if (!ok) return;
        tc_fence_after();
        const uint64_t k0 = dk + ks * (uint32_t)(S::kTile >> 4);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (uint32_t)((kk >> 2) * kAtom + (kk & 3) * 32) >> 4;
            mma_f16(tmem + kColS, dq + off, k0 + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          tc_commit(BAR(x, S_FULL));
          tc_commit(k_empty + ks);
          if (j == cm - 1) tc_commit(BAR(x, Q_EMPTY));
        }
        __syncwarp();
        step(ks, kph);
      };
      auto issue_pv = [&](int j) {
        if (!ok) return;
        wait(BAR(x, P_FULL), mine + j, 0x906u);
        wait(v_full + vs, vph, 0x907u);
        if (!ok) return;
        tc_fence_after();
        const uint64_t v0 = dv + vs * (uint32_t)(S::kTile >> 4);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // keys [16 kk, 16 kk + 16) are P columns [8 kk, 8 kk + 8)
            mma_f16_ts(tO, tP + (uint32_t)(kk * 8), v0 + (uint32_t)(kk * 16 * 128 >> 4), idesc_o,
                       (j > 0 || kk > 0) ? 1u : 0u);
          tc_commit(v_empty + vs);
          tc_commit(BAR(x, PV_DONE));
        }
        __syncwarp();
        step(vs, vph);
      };
      issue_s(0);
      issue_s(1);
      for (int j = 0; j < cm && ok; ++j) {
        issue_pv(j);
        issue_s(j + 2);
      }
      for (int j = cm; j < all && ok; ++j) {  // tiles that only the other one reads
        wait(k_full + ks, kph, 0x908u);
        if (ok && leader) mbar_arrive(k_empty + ks);
        wait(v_full + vs, vph, 0x908u);
        if (ok && leader) mbar_arrive(v_empty + vs);
        __syncwarp();
        step(ks, kph);
        step(vs, vph);
      }
      mine += cm;
      other += co;
      segs += cm > 0;
    }
    // every MMA issued above completes before tensor memory is freed
    if (leader) {
      tc_commit(BAR(x, DRAIN));
      mbar_wait(BAR(x, DRAIN), 0, 0x909u);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax of tile x
    const int x = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + kColS + lane_addr;
    const uint32_t tP = tmem + kColP + (uint32_t)(x * 64) + lane_addr;
    const uint32_t tO = tmem + kColO + (uint32_t)(x * 128) + lane_addr;
    const float c = a.scale_log2;
    const float zero = fminf(c, 0.f);  // c is positive, which the compiler does not know
    // what a maximum's weights are taken relative to
    auto ref = [](float m) { return kShift<T> > 0.f && fabsf(m) < kShifted ? m - kShift<T> : m; };
    const int half_rows = a.rows >> 1;
    bool ok = true;
    uint32_t kv = 0, mine = 0;
    while (ok && __all_sync(0xffffffffu, next_segment())) {
      const int cnt = DESC().cnt[x], key_t0 = DESC().key_t0, len = DESC().len;
      int lim = 0;  // keys that this row sees
      if (cnt > 0) {
        const Desc& g = DESC();
        const int pr = g.row0 + x * half_rows + row;
        if (row < half_rows && pr < g.n * a.g) {
          const int v = a.causal ? min(g.off + pr / a.g + 1, len) : len;
          lim = v > 0 ? v : 0;
        }
      }
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < cnt; ++j) {
        if (!__all_sync(0xffffffffu, mbar_wait(BAR(x, S_FULL), (mine + j) & 1u, 0x90au))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[128];
        tmem_ld_32x32b_x32(tS, s);
        tmem_ld_32x32b_x32(tS + 32, s + 32);
        tmem_ld_32x32b_x32(tS + 64, s + 64);
        tmem_ld_32x32b_x32(tS + 96, s + 96);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(x, S_FREE));
        const int key0 = (key_t0 + j) * kKeys;
        const bool masked = __any_sync(0xffffffffu, key0 + kKeys > lim);
        if (masked) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key0 + i >= lim) s[i] = __float_as_uint(-INFINITY);
        }
        const float mb = fmaxf(max64(s), max64(s + 64)) * c;  // log2 domain
        float alpha = 1.f;
        const bool raise = mb > m_used + kLazy;
        if (raise) {
          alpha = (m_used == -INFINITY) ? 0.f : ex2_approx(ref(m_used) - ref(mb));
          m_used = mb;
        }
        // tcgen05.ld / st are warp-wide: the warp rescales when any of its rows does
        const bool rescale = __any_sync(0xffffffffu, raise);
        const float msub = (m_used == -INFINITY) ? 0.f : ref(m_used);
        const uint64_t cc = f2_pack(c, c), zz = f2_pack(zero, zero);
        const uint64_t nm = f2_pack(-msub, -msub);
        uint64_t acc2 = f2_pack(0.f, 0.f);
        uint32_t pk[32];
        // twice the same: with the two kinds of tiles apart the compiler keeps all scores in registers
        // (ragged chunks of D 64 65.3 us; in one path it spills ten of them, 67.1)
        if (masked) exp_pack64<T>(s, cc, zz, nm, acc2, pk);
        else exp_pack64<T>(s, cc, zz, nm, acc2, pk);
        if (j > 0) {
          // P_x and O_x are free once the product of tile j - 1 is done
          if (!__all_sync(0xffffffffu,
                          mbar_wait(BAR(x, PV_DONE), (mine + j - 1) & 1u, 0x90bu))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (rescale) {
#pragma unroll 1
            for (int hh = 0; hh < D / 32; ++hh) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tO + (uint32_t)(hh * 32), o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32b_x32(tO + (uint32_t)(hh * 32), o);
            }
          }
        }
        tmem_st_32x32b_x32(tP, pk);
        if (masked) exp_pack64<T>(s + 64, cc, zz, nm, acc2, pk);
        else exp_pack64<T>(s + 64, cc, zz, nm, acc2, pk);
        tmem_st_32x32b_x32(tP + 32, pk);
        float la, lb;
        f2_unpack(acc2, la, lb);
        l = l * alpha + (la + lb);
        if (key0 + kKeys > len) {
          // values past the sequence's end: what a recycled page holds there is replaced by
          // zeros (0 * NaN is NaN).  Both tiles write the same zeros before their own product.
          const uint32_t vs = (kv + j) % kSlots;
          if (!__all_sync(0xffffffffu,
                          mbar_wait(v_full + vs, ((kv + j) / kSlots) & 1u, 0x90cu))) {
            ok = false;
            break;
          }
          if (key0 + row >= len) {
            uint8_t* dst = sV + vs * S::kTile + row * 128;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
              *reinterpret_cast<uint4*>(dst + (i >> 3) * kAtom + ((i & 7) << 4)) =
                  make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(x, P_FULL));
      }
      if (ok && cnt > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) add_release(s_copied + x, (uint32_t)cnt);
      }
      const bool have_o = __all_sync(
          0xffffffffu,
          ok && cnt > 0 && mbar_wait(BAR(x, PV_DONE), (mine + cnt - 1) & 1u, 0x90du));
      if (have_o) tc_fence_after();
      else if (cnt > 0) ok = false;
      const Desc& g = DESC();
      const int pr = g.row0 + x * half_rows + row;
      const bool row_ok = row < half_rows && pr < g.n * a.g;
      const bool whole = g.whole;
      const float inv = (have_o && lim > 0) ? 1.0f / l : 0.f;
      const int64_t prow = ((int64_t)blockIdx.x * 2 + (key_t0 == 0)) * kRows + x * half_rows + row;
      const int tok = pr / a.g;
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + (g.t0 + tok) * a.o_token +
                                            (int64_t)(g.h * a.g + pr - tok * a.g) * a.o_head);
      float4* pdst = reinterpret_cast<float4*>(a.part + prow * D);
#pragma unroll 1
      for (int hh = 0; hh < D / 32; ++hh) {
        uint32_t o[32];
        if (have_o) {
          tmem_ld_32x32b_x32(tO + (uint32_t)(hh * 32), o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (row_ok && whole) {
          // a row that sees no key is 0, whatever the values that other rows of its tile see; one that
          // has no finite score (its maximum is -inf too) is NaN by its sum, 0 or NaN
          if (lim == 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
#pragma unroll
          for (int cch = 0; cch < 4; ++cch) {
            uint4 v;
            uint32_t* vw = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              vw[i] = Pair<T>::pack(__uint_as_float(o[8 * cch + 2 * i]) * inv,
                                    __uint_as_float(o[8 * cch + 2 * i + 1]) * inv);
            dst[hh * 4 + cch] = v;
          }
        } else if (row_ok && have_o) {  // without keys there is only the maximum (-inf) to say so
#pragma unroll
          for (int i = 0; i < 8; ++i)
            pdst[hh * 8 + i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                           __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
        }
      }
      if (row_ok && !whole)
        *reinterpret_cast<float2*>(a.part_ml + prow * 2) =
            make_float2(have_o ? ref(m_used) : -INFINITY, have_o ? l : 0.f);
      tc_fence_before();
      kv += g.all;
      mine += cnt;
      __syncwarp();
      if (lane == 0) mbar_arrive(d_empty + seg % kDescs);
      ++seg;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace chunk

// ===========================================================================
// Joins the parts of an item that CTA boundaries cut, in their order.  A part whose maximum is -inf and
// whose sum is 0 has no weight (its O may not have been written); with a sum of NaN it has NaN scores,
// which the result shows.  D / 8 lanes (a group) take a
// row.  With few rows an item can have hundreds of parts: beyond kWide a block takes a row, its groups
// every G-th part, four in flight, and the groups are joined through shared memory.  Launched while
// the kernel before it still runs, it waits for that one's end before it reads anything.
// ===========================================================================
template <typename T, int D, int R, bool FEW>
__global__ void __launch_bounds__(256) merge_kernel(const Args a) {
  constexpr int kLanes = D / 8, G = 256 / kLanes, kFlight = 4, kWide = 8;
  __shared__ float s_o[FEW ? G : 1][D];
  __shared__ float s_l[FEW ? G : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int gl = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int c0 = blockIdx.x;
  const int4 rec = *reinterpret_cast<const int4*>(a.rec + (int64_t)c0 * 8);  // valid, b, h, rt
  if (!rec.x) return;
  const int parts = a.rec[(int64_t)c0 * 8 + 4] - c0 + 1;
  const bool wide = FEW && parts > kWide;
  const Seq s = get_seq(a, rec.y);
  const int rows = min(a.rows, s.n * a.g - rec.w * a.rows);
  // wide: a row a block; else a row a group (a few rows are one block's)
  if (FEW && !wide && blockIdx.y) return;
  for (int row0 = wide ? blockIdx.y : blockIdx.y * G; row0 < rows; row0 += wide ? gridDim.y : gridDim.y * G) {
    const int row = wide ? row0 : row0 + group;
    const bool live = row < rows;
    auto slot = [&](int p) { return ((int64_t)(c0 + p) * 2 + (p == 0)) * R + row; };
    float mm = -INFINITY;
    if (live)
      for (int p = wide ? threadIdx.x & 31 : gl; p < parts; p += wide ? 32 : kLanes)
        mm = fmaxf(mm, a.part_ml[slot(p) * 2]);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    if (wide) {
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    }
    float acc[8], l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    if (live) {
      const int step = wide ? G : 1;
      for (int p0 = wide ? group : 0; p0 < parts; p0 += step * kFlight) {
        float2 ml[kFlight];
        float4 x[kFlight], y[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const int p = p0 + i * step;
          ml[i] = make_float2(-INFINITY, 0.f);
          if (p >= parts) continue;
          ml[i] = *reinterpret_cast<const float2*>(a.part_ml + slot(p) * 2);
          const float4* o = reinterpret_cast<const float4*>(a.part + slot(p) * D + gl * 8);
          x[i] = o[0], y[i] = o[1];  // whatever it is where the part saw no key: not used then
        }
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;
          const float f = ex2_approx(ml[i].x - mm);
          acc[0] = fmaf(f, x[i].x, acc[0]), acc[1] = fmaf(f, x[i].y, acc[1]);
          acc[2] = fmaf(f, x[i].z, acc[2]), acc[3] = fmaf(f, x[i].w, acc[3]);
          acc[4] = fmaf(f, y[i].x, acc[4]), acc[5] = fmaf(f, y[i].y, acc[5]);
          acc[6] = fmaf(f, y[i].z, acc[6]), acc[7] = fmaf(f, y[i].w, acc[7]);
          l = fmaf(f, ml[i].y, l);
        }
      }
    }
    if (wide) {
      __syncthreads();  // the last row's sums have been read
#pragma unroll
      for (int i = 0; i < 8; ++i) s_o[FEW ? group : 0][gl * 8 + i] = acc[i];
      if (gl == 0) s_l[FEW ? group : 0] = l;
      __syncthreads();
      if (group) continue;
      for (int q = 1; q < G && q < parts; ++q) {
        l += s_l[FEW ? q : 0];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += s_o[FEW ? q : 0][gl * 8 + i];
      }
    }
    if (live) {
      const int64_t pr = (int64_t)rec.w * a.rows + row, i = pr / a.g;
      const float inv = seen_by(a, s, (int)i + 1) > 0 ? 1.f / l : 0.f;
      T* dst = reinterpret_cast<T*>(a.out) + (s.t0 + i) * a.o_token +
               ((int64_t)rec.z * a.g + pr - i * a.g) * a.o_head + gl * 8;
      *reinterpret_cast<uint4*>(dst) = make_uint4(
          Pair<T>::pack(acc[0] * inv, acc[1] * inv), Pair<T>::pack(acc[2] * inv, acc[3] * inv),
          Pair<T>::pack(acc[4] * inv, acc[5] * inv), Pair<T>::pack(acc[6] * inv, acc[7] * inv));
    }
  }
}

// Whether the rows of the longest sequence fit a tile of the few-rows kernel.  16 streams of up to 4000
// keys, D 128, few rows against many: 1 row a key head 29.5 and 46.2 us, 4 rows 35.1 and 48.9, 16 rows
// 34.0 and 44.6; 32 rows, two tiles of it that read the cache twice, 50.2 and 49.9.
inline bool few_rows(int64_t max_new, int64_t g) { return max_new <= dec::kRows / g; }  // (max_new may be huge)
inline int ctas_of(bool few) { return sm_count() * (few ? 2 : 1); }

int launch_merge(void (*kernel)(Args), dim3 grid, const Args& a, cudaStream_t stream) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(256);
  c.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &early;
  c.numAttrs = 1;
  FVB_CUDA_TRY(cudaLaunchKernelEx(&c, kernel, a), "fvb_paged_attn merge launch");
  return FVB_OK;
}

template <typename T, int D>
int launch(Args& a, bool few, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    FVB_CUDA_TRY(cudaFuncSetAttribute(dec::decode_kernel<T, D>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, dec::kRing),
                 "fvb_paged_attn smem attribute");
    FVB_CUDA_TRY(cudaFuncSetAttribute(chunk::chunk_kernel<T, D>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)chunk::Shape<D>::kSmem),
                 "fvb_paged_attn smem attribute");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  if (few) {
    dec::decode_kernel<T, D><<<a.ctas, dec::kThreads, dec::kRing, stream>>>(a);
    int rc = check_launch("fvb_paged_attn");
    if (rc) return rc;
    return launch_merge(merge_kernel<T, D, dec::kRows, true>, dim3(a.ctas, a.few_rows < 4 ? a.few_rows : 4), a,
                        stream);
  }
  // rows of a TMA box: a power of two that divides the page, at most a tile
  int box = 16;
  while (box < chunk::kKeys && a.page % (2 * box) == 0) box *= 2;
  CUtensorMap tq, tk, tv;
  const CUtensorMapDataType dt = Pair<T>::kFmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)a.Hk, (uint64_t)a.page, (uint64_t)a.pages};
  const uint64_t sk[3] = {(uint64_t)a.k_head * 2, (uint64_t)a.k_slot * 2, (uint64_t)a.k_page * 2};
  const uint64_t sv[3] = {(uint64_t)a.v_head * 2, (uint64_t)a.v_slot * 2, (uint64_t)a.v_page * 2};
  const uint32_t bx[4] = {64, 1, (uint32_t)box, 1};
  int rc = make_tmap_4d(&tk, a.k, dt, dims, sk, bx);
  if (rc) return rc;
  rc = make_tmap_4d(&tv, a.v, dt, dims, sv, bx);
  if (rc) return rc;
  const uint64_t dq[4] = {(uint64_t)D, (uint64_t)a.Hk * a.g, (uint64_t)a.T, 1};
  const uint64_t sq[3] = {(uint64_t)a.q_head * 2, (uint64_t)a.q_token * 2, (uint64_t)a.q_token * 2};
  const uint32_t bq[4] = {64, (uint32_t)a.g, (uint32_t)(128 / a.g), 1};
  rc = make_tmap_4d(&tq, a.q, dt, dq, sq, bq);
  if (rc) return rc;
  chunk::chunk_kernel<T, D><<<a.ctas, chunk::kThreads, chunk::Shape<D>::kSmem, stream>>>(tq, tk, tv, box, a);
  rc = check_launch("fvb_paged_attn");
  if (rc) return rc;
  return launch_merge(merge_kernel<T, D, chunk::kRows, false>, dim3(a.ctas, chunk::kRows * (D / 8) / 256), a,
                      stream);
}

struct Workspace {
  int64_t part, ml, rec, total;  // byte offsets
};
inline Workspace workspace(bool few, int64_t D) {
  const int64_t n = ctas_of(few), rows = few ? dec::kRows : chunk::kRows;
  Workspace w;
  w.part = 0;
  w.ml = w.part + 2 * n * rows * D * 4;
  w.rec = w.ml + 2 * n * rows * 2 * 4;
  w.total = w.rec + n * 8 * 4;
  return w;
}

}  // namespace pattn
}  // namespace fvb

extern "C" size_t fvb_paged_attn_workspace_bytes(int64_t max_new, int64_t Hq, int64_t Hk, int64_t D) {
  if (max_new < 1 || Hk < 1 || Hq < Hk || D < 1) return 0;
  return (size_t)fvb::pattn::workspace(fvb::pattn::few_rows(max_new, Hq / Hk), D).total;
}

extern "C" int fvb_paged_attn(const fvb_paged_attn_args* p, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(p, "fvb_paged_attn: NULL pointer");
  FVB_REQUIRE(p->dtype == FVB_BF16 || p->dtype == FVB_F16, "fvb_paged_attn: dtype %d", (int)p->dtype);
  if (p->D != 64 && p->D != 128)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attn: head_dim must be 64 or 128 (got %lld)", (long long)p->D);
  FVB_REQUIRE(p->Hk > 0 && p->Hq > 0 && p->Hq % p->Hk == 0 && p->Hq < (1 << 20),
              "fvb_paged_attn: %lld query heads on %lld key heads", (long long)p->Hq, (long long)p->Hk);
  FVB_REQUIRE(p->page > 0 && p->page % 16 == 0 && p->page < (1 << 24),
              "fvb_paged_attn: pages must hold a multiple of 16 tokens (got %lld)", (long long)p->page);
  FVB_REQUIRE(p->T >= 0 && p->B >= 0 && p->B < (1 << 30) && p->width >= 0 && p->width < (1ll << 31) &&
                  p->pages > 0 && p->pages < (1ll << 31) && p->width * p->page <= pattn::kMostKeys &&
                  p->T < (1ll << 30) && p->T * p->Hq < (1ll << 30),
              "fvb_paged_attn: shape");
  // (one that is 0 in fp32 would make -inf * 0 of masked scores)
  const float scale_log2 = (float)(p->scale * 1.4426950408889634);
  FVB_REQUIRE(p->scale > 0 && p->scale < 1e30 && scale_log2 > 0.f, "fvb_paged_attn: scale %g", p->scale);
  FVB_REQUIRE(p->max_new >= 1, "fvb_paged_attn: max_new %lld", (long long)p->max_new);
  if (p->T == 0 || p->B == 0) return FVB_OK;
  FVB_REQUIRE(p->cu || p->T == p->B, "fvb_paged_attn: %lld tokens of %lld sequences need cu_seqlens",
              (long long)p->T, (long long)p->B);
  FVB_REQUIRE(p->q && p->lens && p->out && p->workspace && (p->width == 0 || p->table) && p->k && p->v,
              "fvb_paged_attn: NULL pointer");
  FVB_REQUIRE(aligned16(p->q) && aligned16(p->k) && aligned16(p->v) && aligned16(p->out) &&
                  aligned16(p->workspace),
              "fvb_paged_attn: pointers must be 16-byte aligned");
  FVB_REQUIRE((p->q_token | p->q_head | p->k_page | p->k_slot | p->k_head | p->v_page | p->v_slot |
               p->v_head | p->o_token | p->o_head) % 8 == 0,
              "fvb_paged_attn: strides must be multiples of 8 elements");
  const bool few = pattn::few_rows(p->max_new, p->Hq / p->Hk);
  if (!few && p->Hq / p->Hk > 128)
    return fail(FVB_ERR_UNSUPPORTED, "fvb_paged_attn: more than 128 query heads on a key head");
  const pattn::Workspace w = pattn::workspace(few, p->D);
  char* const ws = (char*)p->workspace;
  pattn::Args a = {};
  a.q = p->q;
  a.out = p->out;
  a.q_token = p->q_token, a.q_head = p->q_head, a.o_token = p->o_token, a.o_head = p->o_head;
  a.k = p->k, a.v = p->v;
  a.k_page = p->k_page, a.k_slot = p->k_slot, a.k_head = p->k_head;
  a.v_page = p->v_page, a.v_slot = p->v_slot, a.v_head = p->v_head;
  a.table = p->table, a.lens = p->lens, a.cu = p->cu;
  a.T = p->T, a.width = p->width, a.pages = p->pages;
  a.B = (int)p->B, a.Hk = (int)p->Hk, a.g = (int)(p->Hq / p->Hk), a.page = (int)p->page;
  a.causal = p->causal != 0;
  a.ctas = pattn::ctas_of(few);
  // whole tokens in a tile, and with many rows in each half of it
  a.tokens = few ? pattn::dec::kRows / a.g : 2 * (128 / a.g);
  a.rows = a.tokens * a.g;
  a.few_rows = (int)(few ? p->max_new * a.g : a.rows);
  a.scale_log2 = scale_log2;
  a.part = (float*)(ws + w.part);
  a.part_ml = (float*)(ws + w.ml);
  a.rec = (int32_t*)(ws + w.rec);
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == FVB_BF16)
    return p->D == 128 ? pattn::launch<__nv_bfloat16, 128>(a, few, st)
                       : pattn::launch<__nv_bfloat16, 64>(a, few, st);
  return p->D == 128 ? pattn::launch<__half, 128>(a, few, st) : pattn::launch<__half, 64>(a, few, st);
}
