// Rotary positions, and the append of a chunk's keys and values to a paged cache.
//
// The first `rot` channels of a head are pairs; pair i of a token at position p is turned by
// p * w_i.  interleaved: pair i is channels (2i, 2i+1); half: channels (i, i + rot/2).
//   y_a = m (a cos - b sin),  y_b = m (b cos + a sin)
// and with the sine negated the inverse rotation, which is the gradient.  m is the factor of a
// scaling for long contexts.
//
// Angles: w_i / 2 pi is held as a 64-bit fraction of a turn, so p * w_i modulo one turn is an
// integer product that drops whole turns exactly: the angle is good to fp32 up to positions of about
// 2^30, where p * w in fp32 has lost it by p = 2^16.  (w itself comes from a 64-bit float: beyond, the
// angle is off by up to p w 2^-52.)  One angle a token and pair, in shared memory, serves every head
// of q and k.
//
// Bound by memory: q and k are read and written once (append: q, k and v, with k and v written
// to their pages).  Measured (B200, cold inputs): 8448 tokens of 12 + 12 heads of 128 in bf16 19.5 us
// (104 MB at 5.3 TB/s), 16896 tokens appended 51.6 us (261 MB at 5.1 TB/s), 4099 tokens of 24 + 4 heads
// of 80 in fp32 11.4 us (73 MB at 6.4 TB/s).  Where vectors do not fit, an element at a time: 8448
// tokens of 12 + 12 heads of 96 in bf16, 24 of them turned in halves, 57 us (1.4 TB/s; 32 of them,
// with vectors, 14.4).  An earlier form that dealt rows of heads to threads
// spent 63% of its issue slots on indexes (27, 54 and 21 us); one that kept blocks resident and
// prefetched the next tokens' angles held too many registers to cover latency (34, 74 and 20 us).
#include "common.cuh"

#include <cuda_fp16.h>

namespace fvb {
namespace rope {

constexpr int kThreads = 512;      // most threads of a block
constexpr int kManyThreads = 192;  // where there are tokens enough for every SM
constexpr int kMaxTokens = 32;     // tokens a block
constexpr int kMaxDim = 256;

struct Part {  // q, k or v: heads of a token, and where they go
  const void* src;
  int64_t src_token, src_head;  // strides, elements
  void* dst;
  int64_t dst_token, dst_head;
  int heads;
  int paged;  // dst is a pool of pages, the token's row given by its page (dst_token unused)
  int turned;
};

struct Args {
  Part part[3];
  int parts, heads;  // heads: of all parts together
  int64_t T;
  int D, rot, tokens;  // tokens: a block's share
  int units, turned_units;  // places of a head, those that are turned
  int lanes, side;          // threads of a token, tokens side by side
  const void* pos;  // NULL: the token's place in its sequence, dropped tokens counted
  int pos64, axes;
  const uint64_t* freq;  // [rot / 2] turns a position, 2^64 to a turn
  const int32_t* axis;   // [rot / 2]
  float scale;
  int inverse;
  // append
  const int32_t *cu, *lens, *table;
  int64_t B, width, pages;
  int page;
  int64_t page_stride, slot_stride;  // of the pools
  const int32_t* refused;  // not 0: the chunk has no room (NULL: it has)
  const int32_t* refs;     // sequences that hold a page (NULL: one)
  const int64_t* dropped;  // tokens that a sequence had before those of lens (NULL: none)
  int32_t* status;
};

constexpr int kNotAppended = 8;  // in status

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kV = 4;
  __device__ static void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  __device__ static float get(float v) { return v; }
  __device__ static float put(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kV = 8;
  __device__ static void unpack(const uint4& u, float* f) { bf16x8_to_f32(u, f); }
  __device__ static uint4 pack(const float* f) { return f32_to_bf16x8(f); }
  __device__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static constexpr int kV = 8;
  __device__ static void unpack(const uint4& u, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  __device__ static uint4 pack(const float* f) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return u;
  }
  __device__ static float get(__half v) { return __half2float(v); }
  __device__ static __half put(float v) { return __float2half_rn(v); }
};

// 16 bytes that are read once (not as read-only data: the output may be the input)
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// two pairs at once: (a, b) -> (a c - b s, b c + a s)
__device__ __forceinline__ void turn2(float& a0, float& a1, float& b0, float& b1, float c0, float c1,
                                      float s0, float s1) {
  const uint64_t a = f2_pack(a0, a1), b = f2_pack(b0, b1), c = f2_pack(c0, c1), s = f2_pack(s0, s1);
  const uint64_t x = f2_fma(a, c, f2_mul(b, f2_pack(-s0, -s1)));
  const uint64_t y = f2_fma(b, c, f2_mul(a, s));
  f2_unpack(x, a0, a1);
  f2_unpack(y, b0, b1);
}

// A token's work is `heads * units` places: a 16-byte vector (interleaved, or not turned) or two half
// a rotation apart (VEC: strides, pointers, D and the rotated part are multiples of them), else one
// pair or one untouched channel.  A thread keeps its place over the block's tokens, kBatch of them
// in flight, so that a token costs it two additions of strides; the first ones are on their way
// while the angles are formed.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_kernel(const Args a) {
  constexpr int V = VEC ? Elem<T>::kV : 1;
  constexpr int kBatch = HALF ? 2 : 4;  // tokens in flight a thread: 64 bytes either way
  extern __shared__ __align__(16) float cs_all[];  // [tokens][cos, sin][rot / 2]
  __shared__ int64_t s_pos[kMaxTokens];
  __shared__ int64_t s_slot[kMaxTokens];  // offset of the token's row in the pools, -1: leave it
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)min((int64_t)a.tokens, a.T - t0);
  const int half_rot = a.rot >> 1;
  const int work = a.heads * a.units;
  // tokens side by side when a token's work is smaller than the block
  const int lane_token = threadIdx.x / a.lanes, first = threadIdx.x - lane_token * a.lanes;
  const bool works = lane_token < a.side && first < work;

  uint4 va[kBatch], vb[kBatch];
  float fa[kBatch], fb[kBatch];
  const T* src;
  T* dst;
  int64_t src_step, dst_step;
  int u, ch2, paged;
  bool two, tr;
  // the place w of a token: which part, head and channels
  auto place = [&](int w) {
    int h = w / a.units;
    u = w - h * a.units;
    int i = 0;
    if (h >= a.part[0].heads) {
      h -= a.part[0].heads, i = 1;
      if (a.parts > 2 && h >= a.part[1].heads) h -= a.part[1].heads, i = 2;
    }
    const Part& pt = a.part[i];
    const bool rotates = u < a.turned_units;
    int ch;
    if (VEC)
      ch = HALF ? (rotates ? u * V : a.rot + (u - a.turned_units) * V) : u * V;
    else
      ch = rotates ? (HALF ? u : 2 * u) : a.rot + (u - a.turned_units);
    two = rotates && (HALF || !VEC);
    ch2 = HALF ? half_rot : 1;  // how far on the second one is
    tr = rotates && pt.turned;
    paged = pt.paged;
    src_step = a.side * pt.src_token;
    dst_step = pt.paged ? 0 : a.side * pt.dst_token;
    const int64_t t = t0 + lane_token;
    src = reinterpret_cast<const T*>(pt.src) + t * pt.src_token + h * pt.src_head + ch;
    dst = reinterpret_cast<T*>(pt.dst) + (pt.paged ? 0 : t * pt.dst_token) + h * pt.dst_head + ch;
  };
  auto load = [&](int tk) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (tk + i * a.side >= n) break;
      if (VEC) {
        va[i] = ld_once(src);
        if (two) vb[i] = ld_once(src + ch2);
      } else {
        fa[i] = Elem<T>::get(src[0]);
        if (two) fb[i] = Elem<T>::get(src[ch2]);
      }
      src += src_step;
    }
  };
  if (works) {
    place(first);
    load(lane_token);
  }

  int32_t refs = 0;  // sequences that hold this thread's token's page: they arrive while the angles are formed
  if (a.cu) {
    if (threadIdx.x < n) {
      const int32_t refused = a.refused ? *a.refused : 0;
      const int64_t t = t0 + threadIdx.x;
      // last sequence that starts at or before t; tokens behind the last sequence are left alone
      int64_t lo = 0, hi = a.B;
      while (lo + 1 < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int64_t c0 = a.cu[lo], c1 = a.cu[lo + 1];
      bool live = c0 <= t && t < c1;
      // without the room that a reserve makes, the places counted back from lens are cached tokens'
      if (live && refused) {
        live = false;
        atomicOr(a.status, kNotAppended);
      }
      const int64_t before = a.dropped ? a.dropped[lo] : 0;
      const int64_t at = (int64_t)a.lens[lo] - (c1 - c0) + (t - c0);
      int64_t slot = -1;
      if (live && at >= 0) {
        const int64_t j = at / a.page;
        const int32_t p = j < a.width ? a.table[lo * a.width + j] : -1;
        if (p >= 0 && p < a.pages) {
          if (a.refs) refs = a.refs[p];
          slot = p * a.page_stride + (at - j * a.page) * a.slot_stride;
        }
      }
      s_pos[threadIdx.x] = at + before;
      s_slot[threadIdx.x] = live ? slot : -2;  // -1: no place in the pool, -2: no token at all
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n * half_rot; i += blockDim.x) {
    const int tk = i / half_rot, pr = i - tk * half_rot;
    int64_t p;
    if (a.pos) {
      const int64_t at = (t0 + tk) * a.axes + (a.axes > 1 ? a.axis[pr] : 0);
      p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at]
                  : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[at];
    } else {
      p = s_pos[tk];
    }
    // turns in [-1/2, 1/2), to 2^-32 of one
    const int32_t f = (int32_t)(((uint64_t)p * a.freq[pr]) >> 32);
    float s, c;
    sincospif((float)f * 4.656612873077393e-10f /* 2^-31 */, &s, &c);
    float* cs = cs_all + tk * a.rot + pr;
    cs[0] = c * a.scale;
    cs[half_rot] = (a.inverse ? -s : s) * a.scale;
  }
  if (refs > 1) {  // other sequences' tokens too
    s_slot[threadIdx.x] = -1;
    atomicOr(a.status, kNotAppended);
  }
  __syncthreads();
  if (!works) return;

  for (int w = first; w < work; w += a.lanes) {
    if (w != first) place(w);
    for (int tk = lane_token; tk < n; tk += a.side * kBatch) {
      if (w != first || tk != lane_token) load(tk);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int k = tk + i * a.side;
        if (k >= n) break;
        T* d = dst;
        dst += dst_step;
        if (a.cu) {
          const int64_t slot = s_slot[k];
          if (slot < (paged ? 0 : -1)) continue;
          if (paged) d += slot;
        }
        if (VEC) {
          if (tr) {
            const float* cs = cs_all + k * a.rot;
            float x[V];
            Elem<T>::unpack(va[i], x);
            if (HALF) {
              float y[V];
              Elem<T>::unpack(vb[i], y);
              cs += u * V;
#pragma unroll
              for (int j = 0; j < V; j += 4) {
                const float4 c = *reinterpret_cast<const float4*>(cs + j);
                const float4 s = *reinterpret_cast<const float4*>(cs + half_rot + j);
                turn2(x[j], x[j + 1], y[j], y[j + 1], c.x, c.y, s.x, s.y);
                turn2(x[j + 2], x[j + 3], y[j + 2], y[j + 3], c.z, c.w, s.z, s.w);
              }
              vb[i] = Elem<T>::pack(y);
            } else {
              cs += u * (V / 2);
#pragma unroll
              for (int j = 0; j < V; j += 4) {
                const float2 c = *reinterpret_cast<const float2*>(cs + j / 2);
                const float2 s = *reinterpret_cast<const float2*>(cs + half_rot + j / 2);
                turn2(x[j], x[j + 2], x[j + 1], x[j + 3], c.x, c.y, s.x, s.y);
              }
            }
            va[i] = Elem<T>::pack(x);
          }
          *reinterpret_cast<uint4*>(d) = va[i];
          if (two) *reinterpret_cast<uint4*>(d + ch2) = vb[i];
        } else {
          if (tr) {
            const float c = cs_all[k * a.rot + u], s = cs_all[k * a.rot + half_rot + u];
            const float x = fa[i], y = fb[i];
            fa[i] = fmaf(x, c, -(y * s));
            fb[i] = fmaf(y, c, x * s);
          }
          d[0] = Elem<T>::put(fa[i]);
          if (two) d[ch2] = Elem<T>::put(fb[i]);
        }
      }
    }
  }
}

inline bool mult(int64_t v, int m) { return v % m == 0; }

// Sizes, the path and the launch, for both entry points.
template <typename T>
int launch(Args& a, bool half, cudaStream_t stream, const char* what) {
  constexpr int V = Elem<T>::kV;
  bool vec = mult(a.D, V) && mult(a.rot, half ? 2 * V : V);
  for (int i = 0; i < a.parts; ++i) {
    const Part& p = a.part[i];
    vec = vec && aligned16(p.src) && aligned16(p.dst) && mult(p.src_token, V) && mult(p.src_head, V) &&
          mult(p.dst_head, V) && mult(p.paged ? 0 : p.dst_token, V);
    if (p.paged) vec = vec && mult(a.page_stride, V) && mult(a.slot_stride, V);
  }
  const int v = vec ? V : 1;
  // places of a head: pairs of vectors (half) or vectors (interleaved); scalar: pairs; and what
  // is not turned, a vector or a channel each
  a.turned_units = (half || !vec) ? a.rot / (2 * v) : a.rot / v;
  a.units = a.turned_units + (a.D - a.rot) / v;
  // Threads: as many as a token has places, in equal rounds, or several tokens side by side.  Up to
  // 512 of them where a block's latency is what counts (one token of 12 + 12 heads 2.4 us, with
  // 256 3.1; 64 tokens appended 4.45, with 256 5.1), 192 where the blocks of an SM cover each other's
  // (4099 tokens of 24 + 4 heads of 80 in fp32 11.6 us, with 128 12.5, with 256 13.3; 16896 tokens
  // appended 51.5, 52.9 and 51.5; 8448 tokens of 12 + 12 heads in bf16 19.2, 17.3 and 19.2).
  const int most = a.T < 2 * (int64_t)sm_count() ? kThreads : kManyThreads;
  const int work = a.heads * a.units;
  const int rounds = (work + most - 1) / most;
  a.lanes = (work + rounds - 1) / rounds;
  a.side = most / a.lanes > 1 ? most / a.lanes : 1;
  if (a.side > kMaxTokens / 4) a.side = kMaxTokens / 4;
  const int threads = (a.lanes * a.side + 31) / 32 * 32;
  // one token a block (a side) until that fills the machine several times over, then more
  const int64_t want = (int64_t)sm_count() * 8;
  int64_t tokens = (a.T + want - 1) / want;
  tokens = (tokens + a.side - 1) / a.side * a.side;
  a.tokens = (int)(tokens < kMaxTokens ? tokens : kMaxTokens / a.side * a.side);
  const int64_t grid = (a.T + a.tokens - 1) / a.tokens;
  const size_t smem = (size_t)a.tokens * a.rot * sizeof(float);
  const dim3 g((unsigned)grid), b((unsigned)threads);
  if (half) {
    if (vec) rope_kernel<T, true, true><<<g, b, smem, stream>>>(a);
    else rope_kernel<T, true, false><<<g, b, smem, stream>>>(a);
  } else {
    if (vec) rope_kernel<T, false, true><<<g, b, smem, stream>>>(a);
    else rope_kernel<T, false, false><<<g, b, smem, stream>>>(a);
  }
  return check_launch(what);
}

int launch_dtype(Args& a, int dtype, bool half, cudaStream_t stream, const char* what) {
  if (dtype == FVB_BF16) return launch<__nv_bfloat16>(a, half, stream, what);
  if (dtype == FVB_F16) return launch<__half>(a, half, stream, what);
  return launch<float>(a, half, stream, what);
}

}  // namespace rope
}  // namespace fvb

extern "C" int fvb_rope(const fvb_rope_args* p, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(p, "fvb_rope: NULL pointer");
  FVB_REQUIRE(p->dtype >= FVB_BF16 && p->dtype <= FVB_F32, "fvb_rope: dtype %d", (int)p->dtype);
  FVB_REQUIRE(p->T >= 0 && p->D > 0 && p->D <= rope::kMaxDim, "fvb_rope: T %lld, D %lld (1..%d)",
              (long long)p->T, (long long)p->D, rope::kMaxDim);
  FVB_REQUIRE(p->rot >= 0 && p->rot <= p->D && p->rot % 2 == 0, "fvb_rope: rot %lld of %lld channels",
              (long long)p->rot, (long long)p->D);
  FVB_REQUIRE(p->Hq >= 0 && p->Hk >= 0 && p->Hq <= 4096 && p->Hk <= 4096 - p->Hq,
              "fvb_rope: %lld + %lld heads", (long long)p->Hq, (long long)p->Hk);
  FVB_REQUIRE(p->axes >= 1 && p->axes <= 16, "fvb_rope: %lld axes", (long long)p->axes);
  if (p->T == 0 || p->Hq + p->Hk == 0) return FVB_OK;
  FVB_REQUIRE((p->Hq == 0 || (p->q && p->q_out)) && (p->Hk == 0 || (p->k && p->k_out)),
              "fvb_rope: NULL pointer");
  FVB_REQUIRE(p->rot == 0 || (p->pos && p->freq && (p->axes == 1 || p->axis)), "fvb_rope: NULL pointer");
  rope::Args a = {};
  if (p->Hq)
    a.part[a.parts++] = {p->q, p->q_token, p->q_head, p->q_out, p->qo_token, p->qo_head, (int)p->Hq, 0, 1};
  if (p->Hk)
    a.part[a.parts++] = {p->k, p->k_token, p->k_head, p->k_out, p->ko_token, p->ko_head, (int)p->Hk, 0, 1};
  a.heads = (int)(p->Hq + p->Hk);
  a.T = p->T;
  a.D = (int)p->D;
  a.rot = (int)p->rot;
  a.pos = p->pos;
  a.pos64 = p->pos64 != 0;
  a.axes = (int)p->axes;
  a.freq = p->freq;
  a.axis = p->axis;
  a.scale = (float)p->scale;
  a.inverse = p->inverse != 0;
  return rope::launch_dtype(a, (int)p->dtype, p->half != 0, (cudaStream_t)stream, "fvb_rope");
}

extern "C" int fvb_kv_append(const fvb_kv_append_args* p, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(p, "fvb_kv_append: NULL pointer");
  FVB_REQUIRE(p->dtype == FVB_BF16 || p->dtype == FVB_F16, "fvb_kv_append: dtype %d", (int)p->dtype);
  FVB_REQUIRE(p->T >= 0 && p->D > 0 && p->D <= rope::kMaxDim, "fvb_kv_append: T %lld, D %lld (1..%d)",
              (long long)p->T, (long long)p->D, rope::kMaxDim);
  FVB_REQUIRE(p->rot >= 0 && p->rot <= p->D && p->rot % 2 == 0,
              "fvb_kv_append: rot %lld of %lld channels", (long long)p->rot, (long long)p->D);
  FVB_REQUIRE(p->Hq >= 0 && p->Hk > 0 && p->Hq <= 4096 && p->Hk <= 2048 && p->Hq + 2 * p->Hk <= 4096,
              "fvb_kv_append: %lld + 2 x %lld heads", (long long)p->Hq, (long long)p->Hk);
  FVB_REQUIRE(p->B >= 0 && p->width >= 0 && p->pages >= 0 && p->page > 0 && p->page < (1 << 24),
              "fvb_kv_append: cache shape");
  FVB_REQUIRE(p->axes >= 1 && p->axes <= 16 && (p->axes == 1 || p->pos),
              "fvb_kv_append: %lld axes need positions", (long long)p->axes);
  if (p->T == 0 || p->B == 0) return FVB_OK;
  FVB_REQUIRE((p->Hq == 0 || (p->q && p->q_out)) && p->k && p->v && p->cu && p->lens && p->table &&
                  p->k_pool && p->v_pool,
              "fvb_kv_append: NULL pointer");
  FVB_REQUIRE(p->rot == 0 || (p->freq && (p->axes == 1 || p->axis)), "fvb_kv_append: NULL pointer");
  FVB_REQUIRE((!p->refused && !p->refs) || p->status, "fvb_kv_append: refused and refs need status");
  const int turned = p->rot > 0;
  rope::Args a = {};
  if (p->Hq)
    a.part[a.parts++] = {p->q, p->q_token, p->q_head, p->q_out, p->qo_token, p->qo_head, (int)p->Hq, 0, turned};
  a.part[a.parts++] = {p->k, p->k_token, p->k_head, p->k_pool, 0, p->D, (int)p->Hk, 1, turned};
  a.part[a.parts++] = {p->v, p->v_token, p->v_head, p->v_pool, 0, p->D, (int)p->Hk, 1, 0};
  a.heads = (int)(p->Hq + 2 * p->Hk);
  a.T = p->T;
  a.D = (int)p->D;
  a.rot = (int)p->rot;
  a.pos = p->pos;
  a.pos64 = p->pos64 != 0;
  a.axes = (int)p->axes;
  a.freq = p->freq;
  a.axis = p->axis;
  a.scale = (float)p->scale;
  a.cu = p->cu;
  a.lens = p->lens;
  a.table = p->table;
  a.B = p->B;
  a.width = p->width;
  a.pages = p->pages;
  a.page = (int)p->page;
  a.page_stride = p->page_stride;
  a.slot_stride = p->Hk * p->D;
  a.refused = p->refused;
  a.refs = p->refs;
  a.dropped = p->dropped;
  a.status = p->status;
  return rope::launch_dtype(a, (int)p->dtype, p->half != 0, (cudaStream_t)stream, "fvb_kv_append");
}
