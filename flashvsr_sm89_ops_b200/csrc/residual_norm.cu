// The seam between two branches of a sandwich-normed block, in one pass over the stream:
//
//   z  = post(y) * pw + pb                    post: RMSNorm, LayerNorm or nothing
//   x' = rs * x + gate * z                    the residual stream, stored in bf16
//   h  = (norm(x') * w + b) * (1 + scale) + shift     norm: RMSNorm or LayerNorm
//
// h is stored in bf16 and / or as microscaled 4-bit codes (fp4.cuh).  Everything between the
// loads and the stores is fp32: h is normed from x' before its rounding to bf16, and the codes
// are those of h before its rounding, so nothing is rounded twice.
//
// HBM bounds it: x and y are read once, x' and h (or its codes) written once, so what is spent
// on an element has to stay near 15 instructions.  A block works on rows of one batch item and
// folds the per-column operands into fp32 vectors in shared memory first:
//   x' = rs * x + n1 * A1      A1 = gate * pw,  n1 = post norm of y
//   h  = n2 * A2 + B2          A2 = w * (1 + scale), B2 = b * (1 + scale) + shift
// (with a gate per row or a post-norm bias, A1 = pw and the other two are read as they are).
// WPR warps own a row and hold it in registers as fp32 pairs, thread t the 16-byte vectors
// t, t + 32 WPR, ...; statistics are two-pass in registers (mean, then centred squares); the
// next row's loads go out as soon as the current row's registers are free.  Measured on
// 2 x 8448 x 1536 (208 MB moved): 37.4 us, 5.6 TB/s (60 us with every operand unpacked for every
// row, 45 instructions an element); 8448 x 1536 with nv codes for h: 21.7 us (20.9 with a
// bare product in place of the quotient, which put some midpoints on their wrong side).
#include <atomic>

#include "fp4.cuh"

namespace fvb {
namespace resnorm {

enum { kNone = 0, kRms = 1, kLayer = 2 };
constexpr size_t kStaticSmem = 8 * 4;  // red_all, which counts toward the 48 KB that need no asking

struct Args {
  const __nv_bfloat16* x;
  const __nv_bfloat16* y;
  const __nv_bfloat16* gate;   // [B, D], or [rows, D] with gate_rows; NULL: 1
  const __nv_bfloat16* pw;     // [D] or NULL
  const __nv_bfloat16* pb;
  const __nv_bfloat16* w;
  const __nv_bfloat16* b;
  const __nv_bfloat16* scale;  // [B, D] or NULL
  const __nv_bfloat16* shift;
  int64_t L;
  int D, post, norm, gate_rows;
  float rs, eps, post_eps;
  __nv_bfloat16* x_out;
  __nv_bfloat16* out;          // NULL: no bf16 h
  int fmt;                     // 0: no codes
  uint8_t* codes;
  uint8_t* scales;
  float* row_scale;
  int64_t pitch, tiles;
  int64_t chunk;               // rows of a block
  int blocks;                  // blocks of a batch item
};

// The row's threads: a warp, or WPR warps of the block meeting at named barrier 1 + team.
template <int WPR>
__device__ __forceinline__ void team_sync(int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * WPR) : "memory");
}
template <int WPR, typename Op>
__device__ __forceinline__ float team_reduce(float v, float* red, int team, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (WPR > 1) {
    const int w = (threadIdx.x >> 5) % WPR;
    team_sync<WPR>(team);  // the last reduction's readers are done
    if ((threadIdx.x & 31) == 0) red[w] = v;
    team_sync<WPR>(team);
    v = red[0];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v = op(v, red[i]);
  }
  return v;
}

__device__ __forceinline__ void unpack8(const uint4& u, uint64_t* f) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 pack8(const uint64_t* f) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(f[i], a, b);
    h[i] = __floats2bfloat162_rn(a, b);
  }
  return u;
}

// normed = f * scale + off (a pair each, the same in both halves): (f - mean) * rstd.  kRms has
// mean 0, kNone is the identity.  Vectors past the row hold zeros and count for nothing.
template <int NV, int WPR, bool FULL>
__device__ __forceinline__ void row_norm(const uint64_t (*f)[4], int t, int nvec, float dim, int kind,
                                         float eps, float* red, int team, uint64_t& scale,
                                         uint64_t& off) {
  const auto add = [](float a, float b) { return a + b; };
  float a, b, mean = 0.f;
  if (kind == kNone) {
    scale = f2_pack(1.f, 1.f);
    off = f2_pack(0.f, 0.f);
    return;
  }
  if (kind == kLayer) {
    uint64_t s2 = f2_pack(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s2 = f2_add(s2, f[j][i]);
    f2_unpack(s2, a, b);
    // a true quotient: the mean of a constant row is that constant, so its variance is 0
    mean = __fdiv_rn(team_reduce<WPR>(a + b, red, team, add), dim);
  }
  const uint64_t nm = f2_pack(-mean, -mean);
  uint64_t q2 = f2_pack(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (FULL || t + j * 32 * WPR < nvec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t d = f2_add(f[j][i], nm);
        q2 = f2_fma(d, d, q2);
      }
    }
  f2_unpack(q2, a, b);
  const float r = rsqrtf(__fdiv_rn(team_reduce<WPR>(a + b, red, team, add), dim) + eps);
  scale = f2_pack(r, r);
  off = nm;
}

// EXTRA: a gate per row or a post-norm bias.  FMT: format of the emitted codes, 0 for none.
// FULL: the row fills every thread's NV vectors.
template <int NV, int WPR, bool FULL, bool EXTRA, int FMT>
__global__ void __launch_bounds__(256, NV == 8 ? 1 : 2) residual_norm_kernel(const Args a) {
  constexpr int T = 32 * WPR, TEAMS = 8 / WPR;
  // A1, A2, B2: for each first the lower, then the upper four floats of every vector, so that a
  // warp's 16-byte reads fall on all banks
  extern __shared__ float4 cols[];
  __shared__ float red_all[kStaticSmem / 4];
  const int team = WPR == 1 ? threadIdx.x >> 5 : threadIdx.x / T;
  const int t = threadIdx.x % T;
  float* red = red_all + team * WPR;
  const int nvec = a.D >> 3;
  // the block's rows: [first, last) of batch item bi, dealt to the teams in turn
  const int64_t bi = blockIdx.x / a.blocks;
  const int64_t first = bi * a.L + (int64_t)(blockIdx.x % a.blocks) * a.chunk;
  const int64_t end = (bi + 1) * a.L;
  const int64_t last = first + a.chunk < end ? first + a.chunk : end;
  int64_t row = first + team;

  uint4 xv[NV], yv[NV];
  auto load = [&](uint4* v, const __nv_bfloat16* p, int64_t r) {
    const uint4* src = reinterpret_cast<const uint4*>(p + r * a.D);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      v[j] = r < last && (FULL || t + j * T < nvec) ? ld_stream(src + t + j * T)
                                                    : make_uint4(0u, 0u, 0u, 0u);
  };
  load(yv, a.y, row);
  load(xv, a.x, row);

  for (int v = threadIdx.x; v < nvec; v += 256) {
    float p[8], q[8], s[8], sh[8];
    auto get = [&](const __nv_bfloat16* src, float* d, float fill) {
      if (src) {
        bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(src) + v), d);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fill;
      }
    };
    auto put = [&](int k, const float* d) {
      cols[2 * k * nvec + v] = make_float4(d[0], d[1], d[2], d[3]);
      cols[(2 * k + 1) * nvec + v] = make_float4(d[4], d[5], d[6], d[7]);
    };
    get(!EXTRA && a.gate ? a.gate + bi * a.D : nullptr, s, 1.f);
    get(a.pw, p, 1.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] *= s[i];
    put(0, p);
    get(a.scale ? a.scale + bi * a.D : nullptr, s, 0.f);
    get(a.w, p, 1.f);
    get(a.b, q, 0.f);
    get(a.shift ? a.shift + bi * a.D : nullptr, sh, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = 1.0f + s[i];
      p[i] *= m;
      q[i] = __fmaf_rn(q[i], m, sh[i]);
    }
    put(1, p);
    put(2, q);
  }
  __syncthreads();
  auto column = [&](int k, int v, uint64_t* d) {  // vector v of column operand k, as pairs
    const float4 u = cols[2 * k * nvec + v], w = cols[(2 * k + 1) * nvec + v];
    d[0] = f2_pack(u.x, u.y);
    d[1] = f2_pack(u.z, u.w);
    d[2] = f2_pack(w.x, w.y);
    d[3] = f2_pack(w.z, w.w);
  };

  const uint64_t rs2 = f2_pack(a.rs, a.rs);
  const float dim = (float)a.D;
  for (; row < last; row += TEAMS) {
    uint64_t f[NV][4], sc, of;
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack8(yv[j], f[j]);
    load(yv, a.y, row + TEAMS);
    row_norm<NV, WPR, FULL>(f, t, nvec, dim, a.post, a.post_eps, red, team, sc, of);
    uint4* xo = reinterpret_cast<uint4*>(a.x_out + row * a.D);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = t + j * T;
      if (FULL || v < nvec) {
        uint64_t x[4], c[4], pb[4], g[4];
        unpack8(xv[j], x);
        column(0, v, c);
        if (EXTRA) {
          const int64_t gr = a.gate_rows ? row : bi;
          if (a.pb) unpack8(__ldg(reinterpret_cast<const uint4*>(a.pb) + v), pb);
          if (a.gate) unpack8(__ldg(reinterpret_cast<const uint4*>(a.gate + gr * a.D) + v), g);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t n = f2_mul(f2_add(f[j][i], of), sc);
          if (EXTRA) {
            const uint64_t z = a.pb ? f2_fma(n, c[i], pb[i]) : f2_mul(n, c[i]);
            const uint64_t y = f2_mul(rs2, x[i]);
            f[j][i] = a.gate ? f2_fma(z, g[i], y) : f2_add(z, y);
          } else {
            f[j][i] = f2_fma(n, c[i], f2_mul(rs2, x[i]));
          }
        }
        xo[v] = pack8(f[j]);
      }
    }
    load(xv, a.x, row + TEAMS);
    row_norm<NV, WPR, FULL>(f, t, nvec, dim, a.norm, a.eps, red, team, sc, of);
    uint4* ho = reinterpret_cast<uint4*>(a.out + row * a.D);
    float am[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = t + j * T;
      am[j] = 0.f;
      if (FULL || v < nvec) {
        uint64_t c1[4], c2[4];
        column(1, v, c1);
        column(2, v, c2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[j][i] = f2_fma(f2_mul(f2_add(f[j][i], of), sc), c1[i], c2[i]);
          if (FMT) am[j] = fp4::max_abs_nan(am[j], f[j][i]);
        }
        if (a.out) ho[v] = pack8(f[j]);
      }
    }
    if (FMT == 0) continue;
    // 4-bit codes: a block is 2 (nv) or 4 (mx) neighbouring lanes' vectors.  The whole warp
    // takes every turn (shuffles).  The padding of the last scale tile ends within the turns: they
    // cover whole tiles, 8 or 16 vectors
    const auto mx = [](float x, float y) { return fmaxf(x, y); };
    uint32_t bad = 0u;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t any = __ballot_sync(0xffffffffu, !(am[j] < INFINITY));
      if (any) {  // a block with a non-finite value: NaN scale, its finite values still count
        const uint32_t mine = FMT == FVB_FP4_NV ? 3u << (t & 30) : 15u << (t & 28);
        if (any & mine) bad |= 1u << j;
        if (!(am[j] < INFINITY)) {
          am[j] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float u, w;
            f2_unpack(f[j][i], u, w);
            if (fabsf(u) < INFINITY) am[j] = fmaxf(am[j], fabsf(u));
            if (fabsf(w) < INFINITY) am[j] = fmaxf(am[j], fabsf(w));
          }
        }
      }
      am[j] = fmaxf(am[j], __shfl_xor_sync(0xffffffffu, am[j], 1));
      if (FMT == FVB_FP4_MX) am[j] = fmaxf(am[j], __shfl_xor_sync(0xffffffffu, am[j], 2));
    }
    float rs = 1.f, ik = 1.f;
    if (FMT == FVB_FP4_NV) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) top = fmaxf(top, am[j]);
      const int k = fp4::row_exponent(team_reduce<WPR>(top, red, team, mx));
      rs = fp4::pow2i(k);
      ik = fp4::pow2i(-k);
      if (t == 0) a.row_scale[row] = rs;
    }
    const int npad = (int)(a.tiles * (FMT == FVB_FP4_NV ? 8 : 16));  // vectors under the scale tiles
    uint32_t* cp = reinterpret_cast<uint32_t*>(a.codes + row * a.pitch);
    // scale_at(row, j): a thread's blocks of successive turns are whole tiles apart
    constexpr int PER = FMT == FVB_FP4_NV ? 2 : 4;  // vectors per block
    uint8_t* sp = a.scales + fp4::scale_at(row, t / PER, a.tiles);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = t + j * T;
      if (v >= npad) break;
      uint32_t byte, code;
      float q[8];
      if (FMT == FVB_FP4_NV) {
        byte = fp4::nv_scale(am[j], ik);
        const float d = fp4::e4m3_value(byte) * rs, r = byte == 0u ? 0.f : __frcp_rn(d);
        const uint64_t r2 = f2_pack(r, r), nd2 = f2_pack(-d, -d);
        // fp4::quotient on pairs: a bare product with r puts some midpoints on their wrong side
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t p = f2_mul(f[j][i], r2);
          f2_unpack(f2_fma(f2_fma(p, nd2, f[j][i]), r2, p), q[2 * i], q[2 * i + 1]);
        }
      } else {
        const int e = fp4::mx_exponent(am[j]);
        const float r = fp4::pow2i(-e);
        byte = (uint32_t)(e + 127);
#pragma unroll
        for (int i = 0; i < 4; ++i) f2_unpack(f2_mul(f[j][i], f2_pack(r, r)), q[2 * i], q[2 * i + 1]);
      }
      code = fp4::e2m1x8(q);
      if ((bad >> j) & 1u) {
        code = 0u;
        byte = FMT == FVB_FP4_NV ? 0x7Fu : 0xFFu;
      }
      if (!FULL && v >= nvec) code = byte = 0u;
      if (v * 4 < a.pitch) cp[v] = code;
      if (t % PER == 0) sp[(int64_t)j * (T / PER / 4) * 512] = (uint8_t)byte;
    }
  }
}

template <int NV, int WPR, bool FULL, bool EXTRA, int FMT>
static int launch_as(Args a, int64_t B, cudaStream_t st) {
  auto kern = residual_norm_kernel<NV, WPR, FULL, EXTRA, FMT>;
  const size_t smem = (size_t)3 * a.D * 4;
  constexpr size_t most_smem = (size_t)3 * NV * WPR * 256 * 4;  // of the widest row it takes
  if (most_smem + kStaticSmem > 48 * 1024) {
    // the same limit whoever sets it: calls of several threads and widths may meet here
    static std::atomic<bool> configured[64];
    int dev = 0;
    FVB_CUDA_TRY(cudaGetDevice(&dev), "fvb_residual_norm device");
    FVB_REQUIRE(dev >= 0 && dev < 64, "fvb_residual_norm: device ordinal %d", dev);
    if (!configured[dev].load(std::memory_order_acquire)) {
      FVB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem),
                   "fvb_residual_norm smem attribute");
      configured[dev].store(true, std::memory_order_release);
    }
  }
  // two blocks per SM, rows split evenly; no block without a row for each of its teams if
  // there are enough
  constexpr int TEAMS = 8 / WPR;
  int64_t blocks = (2 * (int64_t)sm_count() + B - 1) / B;
  const int64_t most = (a.L + TEAMS - 1) / TEAMS;
  if (blocks > most) blocks = most;
  a.chunk = (a.L + blocks - 1) / blocks;
  blocks = (a.L + a.chunk - 1) / a.chunk;
  a.blocks = (int)blocks;
  FVB_REQUIRE(blocks * B < (1ll << 31), "fvb_residual_norm: batch");
  kern<<<(unsigned)(blocks * B), 256, smem, st>>>(a);
  return check_launch("fvb_residual_norm");
}

template <int NV, int WPR, int FMT>
static int launch_fmt(const Args& a, int64_t B, cudaStream_t st) {
  // without FULL's instances the widths that fill the registers take 5-13% longer: 8448 x 1536 18.3
  // us against 17.4 (bf16), 23.3 against 21.4 (nv), 21.1 against 19.0 (mx); 25344 x 512 17.7 : 16.3
  const bool full = a.D == NV * WPR * 256, extra = a.gate_rows || a.pb;
  if (full && extra) return launch_as<NV, WPR, true, true, FMT>(a, B, st);
  if (full) return launch_as<NV, WPR, true, false, FMT>(a, B, st);
  if (extra) return launch_as<NV, WPR, false, true, FMT>(a, B, st);
  return launch_as<NV, WPR, false, false, FMT>(a, B, st);
}
template <int NV, int WPR>
static int launch_codes(const Args& a, int64_t B, cudaStream_t st) {
  return a.fmt == FVB_FP4_NV ? launch_fmt<NV, WPR, FVB_FP4_NV>(a, B, st)
                             : launch_fmt<NV, WPR, FVB_FP4_MX>(a, B, st);
}
template <int NV, int WPR>
static int launch(const Args& a, int64_t B, cudaStream_t st) {
  return a.fmt ? launch_codes<NV, WPR>(a, B, st) : launch_fmt<NV, WPR, 0>(a, B, st);
}

}  // namespace resnorm
}  // namespace fvb

extern "C" int fvb_residual_norm(const void* x, const void* y, const void* gate, int gate_rows,
                                 float residual_scale, int post, const void* post_w,
                                 const void* post_b, float post_eps, int norm, const void* w,
                                 const void* b, const void* scale, const void* shift, float eps,
                                 int64_t B, int64_t L, int64_t D, void* x_out, void* out, int fmt,
                                 void* codes, void* scales, float* row_scale,
                                 fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(B >= 0 && L >= 0 && D > 0, "fvb_residual_norm: shape");
  FVB_REQUIRE(D % 8 == 0 && D <= 16384, "fvb_residual_norm: D=%lld must be a multiple of 8, at most 16384",
              (long long)D);
  FVB_REQUIRE(post >= FVB_NORM_NONE && post <= FVB_NORM_LAYER, "fvb_residual_norm: post norm %d", post);
  FVB_REQUIRE(norm == FVB_NORM_RMS || norm == FVB_NORM_LAYER, "fvb_residual_norm: norm %d", norm);
  FVB_REQUIRE(fmt == 0 || fmt == FVB_FP4_NV || fmt == FVB_FP4_MX, "fvb_residual_norm: format %d", fmt);
  if (B == 0 || L == 0) return FVB_OK;
  FVB_REQUIRE(B < (1ll << 31) && L < (1ll << 31) && B * L < (1ll << 31), "fvb_residual_norm: rows");
  FVB_REQUIRE(x && y && x_out, "fvb_residual_norm: NULL pointer");
  FVB_REQUIRE(out || fmt, "fvb_residual_norm: neither a bf16 nor a 4-bit output");
  FVB_REQUIRE(!fmt || (codes && scales && (fmt == FVB_FP4_MX || row_scale)),
              "fvb_residual_norm: NULL 4-bit output");
  for (const void* p : {x, y, gate, post_w, post_b, w, b, scale, shift, (const void*)x_out,
                        (const void*)out, (const void*)codes, (const void*)scales})
    FVB_REQUIRE(!p || aligned16(p), "fvb_residual_norm: pointers must be 16-byte aligned");
  resnorm::Args a;
  a.x = (const __nv_bfloat16*)x;
  a.y = (const __nv_bfloat16*)y;
  a.gate = (const __nv_bfloat16*)gate;
  a.gate_rows = gate && gate_rows;
  a.pw = (const __nv_bfloat16*)post_w;
  a.pb = (const __nv_bfloat16*)post_b;
  a.w = (const __nv_bfloat16*)w;
  a.b = (const __nv_bfloat16*)b;
  a.scale = (const __nv_bfloat16*)scale;
  a.shift = (const __nv_bfloat16*)shift;
  a.L = L;
  a.D = (int)D;
  a.post = post;
  a.norm = norm;
  a.rs = residual_scale;
  a.eps = eps;
  a.post_eps = post_eps;
  a.x_out = (__nv_bfloat16*)x_out;
  a.out = (__nv_bfloat16*)out;
  a.fmt = fmt;
  a.codes = (uint8_t*)codes;
  a.scales = (uint8_t*)scales;
  a.row_scale = row_scale;
  a.pitch = fp4::code_pitch(D);
  a.tiles = fmt ? fp4::scale_tiles(D, fmt) : 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (D <= 256) return resnorm::launch<1, 1>(a, B, st);
  if (D <= 512) return resnorm::launch<2, 1>(a, B, st);
  if (D <= 1024) return resnorm::launch<4, 1>(a, B, st);
  // One warp a row or two.  With codes one, which leaves their blocks and row maxima within a warp,
  // once the rows give every SM a block of such warps; below that two.  us, one : two
  //   nv   512 x 1032 5.1 : 4.1   512 x 1536 5.2 : 4.0   2112 x 1536 7.2 : 7.6   16896 x 1536 36.5 : 37.7
  //   mx   512 x 1032 4.8 : 3.7   512 x 1536 4.7 : 3.6   2112 x 1536 6.4 : 6.6   16896 x 1536 32.0 : 31.9
  // Without codes two: 512 x 1536 4.1 : 3.3, 16896 x 1536 37.5 : 36.8 (38.4 : 37.3 with a post-norm),
  // though one is faster for narrow rows in numbers, 16896 x 1032 25.1 : 26.2
  if (D <= 1536)
    return fmt && B * L > 8 * (int64_t)sm_count() ? resnorm::launch_codes<6, 1>(a, B, st)
                                                  : resnorm::launch<3, 2>(a, B, st);
  if (D <= 2048) return resnorm::launch<4, 2>(a, B, st);
  if (D <= 4096) return resnorm::launch<4, 4>(a, B, st);
  if (D <= 8192) return resnorm::launch<4, 8>(a, B, st);
  return resnorm::launch<8, 8>(a, B, st);
}
