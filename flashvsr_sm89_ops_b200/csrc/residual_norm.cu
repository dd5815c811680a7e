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
// HBM bounds it: x and y are read once, x' and h (or its codes) written once.  WPR warps own a
// row and hold it in registers, thread t the 16-byte vectors t, t + 32 WPR, ...; statistics are
// two-pass in registers (mean, then centred squares).
#include "fp4.cuh"

namespace fvb {
namespace resnorm {

enum { kNone = 0, kRms = 1, kLayer = 2 };

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
  int64_t rows, L;
  int D, post, norm, gate_rows;
  float rs, eps, post_eps;
  __nv_bfloat16* x_out;
  __nv_bfloat16* out;          // NULL: no bf16 h
  int fmt;                     // 0: no codes
  uint8_t* codes;
  uint8_t* scales;
  float* row_scale;
  int64_t pitch, tiles;
};

template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if (WPR > 1) {
    __syncthreads();  // the last reduction's readers are done with red
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v += red[i];
  }
  return v;
}
template <int WPR>
__device__ __forceinline__ float row_max(float v, float* red) {
  v = warp_max(v);
  if (WPR > 1) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v = fmaxf(v, red[i]);
  }
  return v;
}

__device__ __forceinline__ void ld8(const __nv_bfloat16* p, int v, float* f) {
  bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(p) + v), f);
}

// f <- the row normed: (f - mean) * rsqrt(mean of squares + eps); kRms: no mean.
// Vectors past the row hold zeros and stay zeros.
template <int NV, int WPR>
__device__ __forceinline__ void norm_row(float (*f)[8], int t, int nvec, int D, int kind, float eps,
                                         float* red) {
  if (kind == kLayer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += f[j][i];
    // a true quotient: the mean of a constant row is that constant, so its variance is 0
    const float mean = __fdiv_rn(row_sum<WPR>(s, red), (float)D);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (t + j * 32 * WPR < nvec) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] -= mean;
      }
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) q = __fmaf_rn(f[j][i], f[j][i], q);
  const float r = rsqrtf(__fdiv_rn(row_sum<WPR>(q, red), (float)D) + eps);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) f[j][i] *= r;
}

template <int NV, int WPR>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 32 * WPR) residual_norm_kernel(const Args a) {
  constexpr int T = 32 * WPR;
  __shared__ float red[WPR];
  const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (row >= a.rows) return;  // whole warps; with WPR > 1 the grid has exactly the rows
  const int t = WPR == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int nvec = a.D >> 3;
  const int64_t bi = row / a.L;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.D);
  const uint4* yr = reinterpret_cast<const uint4*>(a.y + row * a.D);
  uint4 xv[NV], yv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = t + j * T;
    yv[j] = v < nvec ? ld_stream(yr + v) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = t + j * T;
    xv[j] = v < nvec ? ld_stream(xr + v) : make_uint4(0u, 0u, 0u, 0u);
  }
  float f[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) bf16x8_to_f32(yv[j], f[j]);
  if (a.post != kNone) norm_row<NV, WPR>(f, t, nvec, a.D, a.post, a.post_eps, red);
  const __nv_bfloat16* gate = a.gate ? a.gate + (a.gate_rows ? row : bi) * a.D : nullptr;
  uint4* xo = reinterpret_cast<uint4*>(a.x_out + row * a.D);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = t + j * T;
    if (v < nvec) {
      float p[8], x[8];
      if (a.pw) {
        ld8(a.pw, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] *= p[i];
      }
      if (a.pb) {
        ld8(a.pb, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] += p[i];
      }
      if (gate) {
        ld8(gate, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] *= p[i];
      }
      bf16x8_to_f32(xv[j], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = __fmaf_rn(a.rs, x[i], f[j][i]);
      xo[v] = f32_to_bf16x8(f[j]);
    }
  }
  norm_row<NV, WPR>(f, t, nvec, a.D, a.norm, a.eps, red);
  const __nv_bfloat16* scale = a.scale ? a.scale + bi * a.D : nullptr;
  const __nv_bfloat16* shift = a.shift ? a.shift + bi * a.D : nullptr;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = t + j * T;
    if (v < nvec) {
      float p[8];
      if (a.w) {
        ld8(a.w, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] *= p[i];
      }
      if (a.b) {
        ld8(a.b, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] += p[i];
      }
      if (scale) {
        ld8(scale, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] *= 1.0f + p[i];
      }
      if (shift) {
        ld8(shift, v, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[j][i] += p[i];
      }
      if (a.out) reinterpret_cast<uint4*>(a.out + row * a.D)[v] = f32_to_bf16x8(f[j]);
    }
  }
  if (a.fmt == 0) return;
  // 4-bit codes: a block is 2 (nv) or 4 (mx) neighbouring lanes' vectors
  float am[NV];
  uint32_t bad = 0u;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float m = 0.f;
    bool nf = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = fabsf(f[j][i]);
      nf |= !(v < INFINITY);
      if (v < INFINITY) m = fmaxf(m, v);
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    nf = __shfl_xor_sync(0xffffffffu, (int)nf, 1) || nf;
    if (a.fmt == FVB_FP4_MX) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      nf = __shfl_xor_sync(0xffffffffu, (int)nf, 2) || nf;
    }
    am[j] = m;
    bad |= (uint32_t)nf << j;
  }
  float rs = 1.f, ik = 1.f;
  if (a.fmt == FVB_FP4_NV) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) top = fmaxf(top, am[j]);
    const int k = fp4::row_exponent(row_max<WPR>(top, red));
    rs = fp4::pow2i(k);
    ik = fp4::pow2i(-k);
    if (t == 0) a.row_scale[row] = rs;
  }
  const int npad = (int)(a.tiles * (a.fmt == FVB_FP4_NV ? 8 : 16));  // vectors under the scale tiles
#pragma unroll
  for (int j = 0; j < NV + 1; ++j) {
    // one more turn than the registers hold: the padding of the last scale tile may start
    // past the row's last vector
    const int v = t + j * T;
    if (v >= npad) break;
    const bool nf = j < NV && ((bad >> j) & 1u);
    float q[8];
    uint32_t byte;
    if (a.fmt == FVB_FP4_NV) {
      byte = j < NV ? fp4::nv_scale(am[j < NV ? j : 0], ik) : 0u;
      const float d = fp4::e4m3_value(byte) * rs;
      const float r = __frcp_rn(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = j < NV ? f[j < NV ? j : 0][i] : 0.f;
        q[i] = byte == 0u ? 0.f * h : fp4::quotient(h, d, r);
      }
    } else {
      const int e = j < NV ? fp4::mx_exponent(am[j < NV ? j : 0]) : -127;
      byte = (uint32_t)(e + 127);
      const float r = fp4::pow2i(-e);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = (j < NV ? f[j < NV ? j : 0][i] : 0.f) * r;
    }
    if (v * 4 < a.pitch)
      *reinterpret_cast<uint32_t*>(a.codes + row * a.pitch + v * 4) = nf ? 0u : fp4::e2m1x8(q);
    if (a.fmt == FVB_FP4_NV) {
      if ((t & 1) == 0) a.scales[fp4::scale_at(row, v >> 1, a.tiles)] = (uint8_t)(nf ? 0x7Fu : byte);
    } else {
      if ((t & 3) == 0) a.scales[fp4::scale_at(row, v >> 2, a.tiles)] = (uint8_t)(nf ? 0xFFu : byte);
    }
  }
}

template <int NV, int WPR>
static int launch(const Args& a, cudaStream_t st) {
  const unsigned grid = (unsigned)(WPR == 1 ? (a.rows + 7) / 8 : a.rows);
  residual_norm_kernel<NV, WPR><<<grid, WPR == 1 ? 256 : 32 * WPR, 0, st>>>(a);
  return check_launch("fvb_residual_norm");
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
  a.gate_rows = gate_rows;
  a.pw = (const __nv_bfloat16*)post_w;
  a.pb = (const __nv_bfloat16*)post_b;
  a.w = (const __nv_bfloat16*)w;
  a.b = (const __nv_bfloat16*)b;
  a.scale = (const __nv_bfloat16*)scale;
  a.shift = (const __nv_bfloat16*)shift;
  a.rows = B * L;
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
  if (D <= 256) return resnorm::launch<1, 1>(a, st);
  if (D <= 512) return resnorm::launch<2, 1>(a, st);
  if (D <= 1024) return resnorm::launch<4, 1>(a, st);
  if (D <= 1536) return resnorm::launch<6, 1>(a, st);
  if (D <= 2048) return resnorm::launch<2, 4>(a, st);
  if (D <= 4096) return resnorm::launch<4, 4>(a, st);
  if (D <= 8192) return resnorm::launch<4, 8>(a, st);
  return resnorm::launch<8, 8>(a, st);
}
