// Rotary positions, and the append of a chunk's keys and values to a paged cache.
//
// The first `rot` channels of a head are pairs; pair i of a token at position p is turned by
// p * w_i.  interleaved: pair i is channels (2i, 2i+1); half: channels (i, i + rot/2).
//   y_a = m (a cos - b sin),  y_b = m (b cos + a sin)
// and with the sine negated the inverse rotation, which is the gradient.  m is the factor of a
// scaling for long contexts.
//
// Angles: w_i / 2 pi is held as a 64-bit fraction of a turn, so p * w_i modulo one turn is an
// integer product that drops whole turns exactly: the angle of a position of any size is good to
// fp32, where p * w in fp32 has lost it by p = 2^16.  One angle a token and pair, in shared
// memory, serves every head of q and k.
//
// Bound by memory: q and k are read and written once (append: q, k and v, with k and v written
// to their pages).  A thread keeps one place of a head (one 16-byte vector, or two half a
// rotation apart) and walks over (token, head) rows with kRopeBatch rows in flight.
#include "common.cuh"

#include <cuda_fp16.h>

namespace fvb {
namespace rope {

constexpr int kThreads = 256;
constexpr int kBatch = 4;       // rows in flight a thread
constexpr int kMaxTokens = 8;   // tokens a block
constexpr int kMaxDim = kThreads;  // a place of a head is one thread's at the narrowest

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
  uint32_t heads_inv;  // ceil(2^32 / heads)
  int units, turned_units, rows_at_once;
  const void* pos;  // NULL: the token's place in its sequence
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
};

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

__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float x = a, y = b;
  a = fmaf(x, cs.x, -(y * cs.y));
  b = fmaf(y, cs.x, x * cs.y);
}

// VEC: 16-byte vectors (strides, pointers, D and the rotated part are multiples of them), else
// one pair or one untouched channel at a time.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_kernel(const Args a) {
  constexpr int V = VEC ? Elem<T>::kV : 1;
  extern __shared__ float2 cs_all[];  // [tokens][rot / 2] cos, sin
  __shared__ int64_t s_pos[kMaxTokens];
  __shared__ int64_t s_slot[kMaxTokens];  // offset of the token's row in the pools, -1: none
  __shared__ int s_live[kMaxTokens];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)min((int64_t)a.tokens, a.T - t0);
  const int half_rot = a.rot >> 1;

  if (threadIdx.x < n) {
    const int64_t t = t0 + threadIdx.x;
    int64_t slot = -1, place = 0;
    int live = 1;
    if (a.cu) {
      // last sequence that starts at or before t; tokens behind the last sequence are left alone
      int64_t lo = 0, hi = a.B;
      while (lo + 1 < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int64_t c0 = a.cu[lo], c1 = a.cu[lo + 1];
      live = c0 <= t && t < c1;
      place = (int64_t)a.lens[lo] - (c1 - c0) + (t - c0);
      if (live && place >= 0) {
        const int64_t j = place / a.page;
        const int32_t p = j < a.width ? a.table[lo * a.width + j] : -1;
        if (p >= 0 && p < a.pages) slot = p * a.page_stride + (place - j * a.page) * a.slot_stride;
      }
    }
    s_pos[threadIdx.x] = place;
    s_slot[threadIdx.x] = slot;
    s_live[threadIdx.x] = live;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * half_rot; i += kThreads) {
    const int tk = i / half_rot, pr = i - tk * half_rot;
    int64_t p;
    if (a.pos) {
      const int64_t at = (t0 + tk) * a.axes + (a.axes > 1 ? a.axis[pr] : 0);
      p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at]
                  : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[at];
    } else {
      p = s_pos[tk];
    }
    const int64_t f = (int64_t)((uint64_t)p * a.freq[pr]);  // in [-1/2, 1/2) turns
    float s, c;
    sincospif(__ll2float_rn(f) * 1.0842021724855044e-19f /* 2^-63 */, &s, &c);
    cs_all[i] = make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
  }
  __syncthreads();

  const int u = threadIdx.x % a.units;  // this thread's place in a head
  const int r0 = threadIdx.x / a.units;
  if (r0 >= a.rows_at_once) return;
  const bool rotates = u < a.turned_units;
  // first channel of the place; the second of a half-layout pair lies half_rot on
  int ch;
  if (VEC)
    ch = HALF ? (rotates ? u * V : a.rot + (u - a.turned_units) * V) : u * V;
  else
    ch = rotates ? (HALF ? u : 2 * u) : a.rot + (u - a.turned_units);
  const bool two = rotates && (HALF || !VEC);
  const int ch2 = HALF ? ch + half_rot : ch + 1;

  const int rows = n * a.heads;
  for (int base = r0; base < rows; base += a.rows_at_once * kBatch) {
    const T* src[kBatch];
    T* dst[kBatch];
    int tok[kBatch];
    bool turned[kBatch];
    uint4 va[kBatch], vb[kBatch];
    float fa[kBatch], fb[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = base + i * a.rows_at_once;
      dst[i] = nullptr;
      if (r >= rows) continue;
      const int tk = a.heads > 1 ? (int)__umulhi((uint32_t)r, a.heads_inv) : r;
      int h = r - tk * a.heads;
      tok[i] = tk;
      if (!s_live[tk]) continue;
      const Part* pt = &a.part[0];
      if (h >= pt->heads) {
        h -= pt->heads;
        ++pt;
        if (a.parts > 2 && h >= pt->heads) h -= pt->heads, ++pt;
      }
      const int64_t t = t0 + tk;
      if (pt->paged) {
        if (s_slot[tk] < 0) continue;
        dst[i] = reinterpret_cast<T*>(pt->dst) + s_slot[tk] + h * pt->dst_head;
      } else {
        dst[i] = reinterpret_cast<T*>(pt->dst) + t * pt->dst_token + h * pt->dst_head;
      }
      src[i] = reinterpret_cast<const T*>(pt->src) + t * pt->src_token + h * pt->src_head;
      turned[i] = pt->turned != 0;
      if (VEC) {
        va[i] = *reinterpret_cast<const uint4*>(src[i] + ch);
        if (two) vb[i] = *reinterpret_cast<const uint4*>(src[i] + ch2);
      } else {
        fa[i] = Elem<T>::get(src[i][ch]);
        if (two) fb[i] = Elem<T>::get(src[i][ch2]);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (!dst[i]) continue;
      const float2* cs = cs_all + tok[i] * half_rot;
      const bool tr = rotates && turned[i];
      if (VEC) {
        if (tr) {
          if (HALF) {
            float x[V], y[V];
            Elem<T>::unpack(va[i], x);
            Elem<T>::unpack(vb[i], y);
#pragma unroll
            for (int j = 0; j < V; ++j) turn(x[j], y[j], cs[u * V + j]);
            va[i] = Elem<T>::pack(x);
            vb[i] = Elem<T>::pack(y);
          } else {
            float x[V];
            Elem<T>::unpack(va[i], x);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) turn(x[2 * j], x[2 * j + 1], cs[u * (V / 2) + j]);
            va[i] = Elem<T>::pack(x);
          }
        }
        *reinterpret_cast<uint4*>(dst[i] + ch) = va[i];
        if (two) *reinterpret_cast<uint4*>(dst[i] + ch2) = vb[i];
      } else {
        if (tr) turn(fa[i], fb[i], cs[u]);
        dst[i][ch] = Elem<T>::put(fa[i]);
        if (two) dst[i][ch2] = Elem<T>::put(fb[i]);
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
  a.rows_at_once = kThreads / a.units;
  // row / heads as a multiplication: rows < 8 * 4096, so the reciprocal's excess (< heads) cannot
  // carry (one head needs no division, and its reciprocal would not fit)
  a.heads_inv = a.heads > 1 ? (uint32_t)(((1ull << 32) + a.heads - 1) / a.heads) : 0;
  // one token a block until that fills the machine several times over, then as many as keep it full
  const int64_t want = (int64_t)sm_count() * 8;
  a.tokens = (int)(a.T / want);
  if (a.tokens < 1) a.tokens = 1;
  if (a.tokens > kMaxTokens) a.tokens = kMaxTokens;
  const int64_t grid = (a.T + a.tokens - 1) / a.tokens;
  FVB_REQUIRE(grid < (1ll << 31), "%s: too many tokens", what);
  const size_t smem = (size_t)a.tokens * (a.rot / 2) * sizeof(float2);
  const dim3 g((unsigned)grid), b(kThreads);
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
  return rope::launch_dtype(a, (int)p->dtype, p->half != 0, (cudaStream_t)stream, "fvb_kv_append");
}
