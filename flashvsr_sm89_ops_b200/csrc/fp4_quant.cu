// Quantisation to microscaled 4-bit and back (fp4.cuh has the formats and the layout).
//
// Both directions move each element once and compute a few operations on it, so HBM bounds
// them.  A thread's unit is 16 elements of one row: one nv block, or half an mx block whose
// other half is the neighbouring lane's.  nv needs the row's amax before its first code, so
// the row waits in registers (one warp up to 2048 elements, four warps up to 16384); longer
// rows are read twice.  mx blocks and the way back need nothing of the rest of their row.
// Measured at 8448 x 8960 (193 MB read and written): mx 32.1 us from fp16 (6.0 TB/s, 93% of
// a plain copy), nv 39 us from bf16, the way back 35 us; 8448 x 1536: nv 7.9 us, back 6.9 us;
// rows of an odd length, 4000 x 7001: mx 19.8 us, nv 25.7, back 17.5 (159 when each thread wrote
// its 16 elements one by one).
#include "fp4.cuh"

namespace fvb {
namespace fp4 {

// Units of a row that a warp takes (mx), and the order of a grid of 8-row blocks: reading, the
// row blocks of one segment follow each other (32 us against 33 the other way round); writing,
// the segments of one row block do, or DRAM's pages are written in pieces (35 us against 44)
constexpr int kSegUnits = 128;

template <typename T>
struct Raw {
  static constexpr int kVec = (int)sizeof(T);  // 16-byte vectors of 16 elements
  uint4 v[kVec];
};

__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }

// 32 bytes at once (one whole sector per lane), p 32-byte aligned
__device__ __forceinline__ void ld32(const uint4* p, uint4& a, uint4& b) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}
__device__ __forceinline__ void st32(uint4* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y),
               "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// How a matrix's rows are aligned: 2 = 32 bytes, 1 = 16, 0 = less
__host__ __forceinline__ int row_alignment(const void* p, int64_t pitch_bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes;
  return (a & 31u) == 0 ? 2 : (a & 15u) == 0 ? 1 : 0;
}

// elements [k0, k0 + 16) of a row of K; zeros past its end
template <typename T, bool WIDE = false>
__device__ __forceinline__ void load16(Raw<T>& r, const T* __restrict__ row, int64_t k0, int64_t K,
                                       int align) {
  if (align && k0 + 16 <= K) {
    const uint4* p = reinterpret_cast<const uint4*>(row + k0);
#pragma unroll
    for (int i = 0; i < Raw<T>::kVec; i += 2) {
      if (WIDE && align == 2) {
        ld32(p + i, r.v[i], r.v[i + 1]);
      } else {
        r.v[i] = ld_stream(p + i);
        r.v[i + 1] = ld_stream(p + i + 1);
      }
    }
  } else {
    T* e = reinterpret_cast<T*>(r.v);
#pragma unroll
    for (int i = 0; i < Raw<T>::kVec; ++i) r.v[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k0 + i < K) e[i] = row[k0 + i];
  }
}

// The same for a whole warp, lane l the unit u0 + l.  Rows that are not 16-byte aligned go
// through the warp's 512 elements of shared memory: element by element in row order (a lane
// that read its own 16 one by one would touch 32 sectors with each load).  STAGED: they do; a
// kernel of its own, since the branch and its buffer cost the aligned one 8 of 32 us (mx).
template <typename T, bool WIDE, bool STAGED>
__device__ __forceinline__ void load_units(Raw<T>& r, const T* __restrict__ row, int64_t u0, int64_t K,
                                           int align, T* stage) {
  const int lane = threadIdx.x & 31;
  if (!STAGED) {
    load16<T, WIDE>(r, row, (u0 + lane) * 16, K, align);
    return;
  }
  using U = typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type;
  const U* src = reinterpret_cast<const U*>(row) + u0 * 16;
  U* st = reinterpret_cast<U*>(stage);
  const int64_t left = K - u0 * 16;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = j * 32 + lane;
    st[i] = i < left ? __ldg(src + i) : (U)0;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < Raw<T>::kVec; ++i)
    r.v[i] = reinterpret_cast<const uint4*>(stage)[lane * Raw<T>::kVec + i];
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void unpack16(const Raw<T>& r, float* f) {
  const T* e = reinterpret_cast<const T*>(r.v);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = to_f32(e[i]);
}

// largest finite magnitude of the 16; bad: whether one is not finite
template <typename T>
__device__ __forceinline__ float amax16(const Raw<T>& r, bool& bad) {
  float m;
  if constexpr (sizeof(T) == 2) {
    // packed 16-bit maxima that keep a NaN
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(r.v);
    T2 a = __habs2(p[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) a = __hmax2_nan(a, __habs2(p[i]));
    const T* e = reinterpret_cast<const T*>(&a);
    m = to_f32(__hmax_nan(e[0], e[1]));
  } else {
    uint32_t b = 0u;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(r.v);
#pragma unroll
    for (int i = 0; i < 16; ++i) b = max(b, p[i] & 0x7FFFFFFFu);
    m = __uint_as_float(b);
  }
  bad = !(m < INFINITY);
  if (bad) {
    float f[16];
    unpack16(r, f);
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float a = fabsf(f[i]);
      if (a < INFINITY) m = fmaxf(m, a);
    }
  }
  return m;
}

template <typename T>
struct QuantArgs {
  const T* x;
  int64_t ld, M, K;
  uint8_t* codes;
  uint8_t* scales;
  float* row_scale;
  int64_t pitch;  // bytes of one row of codes
  int64_t tiles;  // scale tiles along a row
  int align;  // row_alignment of x
  unsigned row_blocks;  // of 8 rows (mx)
};

// codes and scale of one nv unit
template <typename T>
__device__ __forceinline__ void nv_store(const QuantArgs<T>& a, int64_t m, int64_t u,
                                         const Raw<T>& r, float amax, bool bad, float rs, float ik) {
  const uint32_t c = nv_scale(amax, ik);
  if (u * 8 < a.pitch) {
    float f[16];
    unpack16(r, f);
    *reinterpret_cast<uint2*>(a.codes + m * a.pitch + u * 8) =
        bad ? make_uint2(0u, 0u) : nv_codes16(f, c, rs);
  }
  a.scales[scale_at(m, u, a.tiles)] = (uint8_t)(bad ? 0x7Fu : c);
}

// nv, the row held in registers: WPR warps a row, NB units a thread
template <typename T, int NB, int WPR, bool STAGED>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 32 * WPR) quant_nv_kernel(const QuantArgs<T> a) {
  constexpr int T_ROW = 32 * WPR;
  const int64_t m = WPR == 1 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (m >= a.M) return;  // whole warps, and with WPR > 1 no block has such a row
  const int t = WPR == 1 ? threadIdx.x & 31 : threadIdx.x;
  const T* row = a.x + m * a.ld;
  const int units = (int)(a.tiles * 4);
  Raw<T> r[NB];
  __shared__ __align__(16) T stage[WPR == 1 ? 8 : WPR][STAGED ? 512 : 1];
  const int64_t w0 = t & ~31;  // the warp's first unit
#pragma unroll
  for (int i = 0; i < NB; ++i)
    // 32 bytes a load: 7.9 us against 9.0 at 8448 x 1536, but 40.7 against 39.2 at 8448 x 8960
    load_units<T, WPR == 1, STAGED>(r[i], row, w0 + i * T_ROW, a.K, a.align, stage[threadIdx.x >> 5]);
  float am[NB], top = 0.f;
  uint32_t bad = 0u;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    bool b;
    am[i] = amax16(r[i], b);
    bad |= (uint32_t)b << i;
    top = fmaxf(top, am[i]);
  }
  top = warp_max(top);
  if (WPR > 1) {
    __shared__ float red[WPR];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = fmaxf(top, red[i]);
  }
  const int k = row_exponent(top);
  const float rs = pow2i(k), ik = pow2i(-k);
  if (t == 0) a.row_scale[m] = rs;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int u = t + i * T_ROW;
    if (u < units) nv_store(a, m, u, r[i], am[i], (bad >> i) & 1u, rs, ik);
  }
}

// nv, rows too long for the registers of four warps: the row is read twice (the second time
// from L2, which holds the rows in flight)
template <typename T>
__global__ void __launch_bounds__(256) quant_nv_long_kernel(const QuantArgs<T> a) {
  const int64_t m = blockIdx.x;
  const T* row = a.x + m * a.ld;
  const int64_t units = a.tiles * 4;
  float top = 0.f;
  for (int64_t u = threadIdx.x; u < units; u += 256) {
    Raw<T> r;
    bool b;
    load16(r, row, u * 16, a.K, a.align);
    top = fmaxf(top, amax16(r, b));
  }
  __shared__ float red[8];
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, red[i]);
  const int k = row_exponent(top);
  const float rs = pow2i(k), ik = pow2i(-k);
  if (threadIdx.x == 0) a.row_scale[m] = rs;
  for (int64_t u = threadIdx.x; u < units; u += 256) {
    Raw<T> r;
    bool b;
    load16(r, row, u * 16, a.K, a.align);
    const float am = amax16(r, b);
    nv_store(a, m, u, r, am, b, rs, ik);
  }
}

// mx: lanes 2i and 2i + 1 share a block; a block of threads is 8 rows x 32 units
template <typename T, bool STAGED>
__global__ void __launch_bounds__(256) quant_mx_kernel(const QuantArgs<T> a) {
  const int64_t m = (int64_t)(blockIdx.x % a.row_blocks) * 8 + (threadIdx.x >> 5);
  if (m >= a.M) return;  // whole warps
  const int lane = threadIdx.x & 31;
  const int64_t units = a.tiles * 8;  // a multiple of 8, so both lanes of a block are in or out
  const T* row = a.x + m * a.ld;
  uint8_t* codes = a.codes + m * a.pitch;
  __shared__ __align__(16) T stage[8][STAGED ? 512 : 1];
  const int64_t u1 = (int64_t)(blockIdx.x / a.row_blocks) * kSegUnits;
#pragma unroll 2
  for (int64_t u0 = u1; u0 < units && u0 < u1 + kSegUnits; u0 += 32) {
    const int64_t u = u0 + lane;
    Raw<T> r;
    load_units<T, false, STAGED>(r, row, u0, a.K, a.align, stage[threadIdx.x >> 5]);
    bool bad;
    float am = amax16(r, bad);
    am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
    const bool other = __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;  // by every lane
    bad = bad || other;
    if (u >= units) continue;
    const int e = mx_exponent(am);
    if (u * 8 < a.pitch) {
      float f[16];
      unpack16(r, f);
      *reinterpret_cast<uint2*>(codes + u * 8) = bad ? make_uint2(0u, 0u) : mx_codes16(f, e);
    }
    // scales past the last block are 0, the exponent byte of an empty block
    if ((u & 1) == 0) a.scales[scale_at(m, u >> 1, a.tiles)] = (uint8_t)(bad ? 0xFF : e + 127);
  }
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}

// p * r for a p of few bits and any r, such that from_f32<T> of it is the product rounded once:
// for a 16-bit T the fp32 product is cut off and its last bit holds whether anything was lost
template <typename T>
__device__ __forceinline__ float scaled(float p, float r) {
  if (sizeof(T) == 4) return __fmul_rn(p, r);
  const float a = fabsf(p), b = fabsf(r), t = __fmul_rz(a, b);
  const uint32_t lost = __fmaf_ru(a, b, -t) > 0.f ? 1u : 0u;
  const uint32_t sign = (__float_as_uint(p) ^ __float_as_uint(r)) & 0x80000000u;
  return __uint_as_float(sign | __float_as_uint(t) | lost);
}

// the values that codes stand for; one thread per 16 elements, 8 rows x 32 units a block
template <typename T, int FMT, bool STAGED>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales,
                                                      const float* __restrict__ row_scale,
                                                      int rs_row, int64_t M, int64_t K,
                                                      int64_t pitch, int64_t tiles, int align,
                                                      unsigned segs, T* __restrict__ out) {
  const int64_t m = (int64_t)(blockIdx.x / segs) * 8 + (threadIdx.x >> 5);
  if (m >= M) return;
  const int lane = threadIdx.x & 31;
  const int64_t u0 = (int64_t)(blockIdx.x % segs) * 32, u = u0 + lane;
  __shared__ __align__(16) T stage[8][STAGED ? 512 : 1];
  T* st = stage[threadIdx.x >> 5];
  if (u < (K + 15) / 16) {
    const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + m * pitch + u * 8));
    const uint32_t b = __ldg(scales + scale_at(m, FMT == FVB_FP4_NV ? u : u >> 1, tiles));
    // code times s is exact; so it stays with a row scale that is a power of two (quantisation
    // makes no other), away from the ends of the range.  Any other multiplies last (warp-uniform).
    float s, rs = 1.0f;
    bool apart = false;
    if (FMT == FVB_FP4_NV) {
      s = e4m3_value(b);
      if (row_scale) rs = __ldg(row_scale + (rs_row ? m : 0));
      const uint32_t bits = __float_as_uint(rs);
      apart = (bits & 0x7FFFFFu) != 0u || (bits >> 23) - 17u > 228u;  // 2^-110 .. 2^118
      if (!apart) s *= rs;
    } else {
      s = b == 0xFFu ? __uint_as_float(0x7FC00000u) : pow2i((int)b - 127);
    }
    uint32_t h[8];
    e2m1x8_to_f16(c.x, h);
    e2m1x8_to_f16(c.y, h + 4);
    float v[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      v[2 * j] = f.x * s;
      v[2 * j + 1] = f.y * s;
    }
    if (apart) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = scaled<T>(v[j], rs);
    }
    Raw<T> o;
    T* e = reinterpret_cast<T*>(o.v);
#pragma unroll
    for (int j = 0; j < 16; ++j) e[j] = from_f32<T>(v[j]);
    T* p = out + m * K + u * 16;
    if (!STAGED && align == 2 && u * 16 + 16 <= K) {
#pragma unroll
      for (int j = 0; j < Raw<T>::kVec; j += 2) st32(reinterpret_cast<uint4*>(p) + j, o.v[j], o.v[j + 1]);
    } else if (!STAGED && u * 16 + 16 <= K) {
#pragma unroll
      for (int j = 0; j < Raw<T>::kVec; ++j) reinterpret_cast<uint4*>(p)[j] = o.v[j];
    } else if (!STAGED) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (u * 16 + j < K) p[j] = e[j];
    } else {
#pragma unroll
      for (int j = 0; j < Raw<T>::kVec; ++j) reinterpret_cast<uint4*>(st)[lane * Raw<T>::kVec + j] = o.v[j];
    }
  }
  if (!STAGED) return;
  // rows that are not 16-byte aligned: element by element in row order
  __syncwarp();
  T* p = out + m * K + u0 * 16;
  const int64_t left = K - u0 * 16;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j * 32 + lane < left) p[j * 32 + lane] = st[j * 32 + lane];
}

template <typename T, bool STAGED>
static void quant_nv(const QuantArgs<T>& a, int64_t units, cudaStream_t st) {
  const unsigned g8 = (unsigned)((a.M + 7) / 8), g1 = (unsigned)a.M;
  if (units <= 32)
    quant_nv_kernel<T, 1, 1, STAGED><<<g8, 256, 0, st>>>(a);
  else if (units <= 64)
    quant_nv_kernel<T, 2, 1, STAGED><<<g8, 256, 0, st>>>(a);
  else if (units <= 96)
    quant_nv_kernel<T, 3, 1, STAGED><<<g8, 256, 0, st>>>(a);
  else if (units <= 128)
    quant_nv_kernel<T, 4, 1, STAGED><<<g8, 256, 0, st>>>(a);
  else if (units <= 256)
    quant_nv_kernel<T, 2, 4, STAGED><<<g1, 128, 0, st>>>(a);
  else if (units <= 640)
    quant_nv_kernel<T, 5, 4, STAGED><<<g1, 128, 0, st>>>(a);
  else
    quant_nv_kernel<T, 8, 4, STAGED><<<g1, 128, 0, st>>>(a);
}

template <typename T>
static int quant(const void* x, int64_t ld, int64_t M, int64_t K, int fmt, void* codes,
                 void* scales, float* row_scale, cudaStream_t st) {
  QuantArgs<T> a;
  a.x = (const T*)x;
  a.ld = ld;
  a.M = M;
  a.K = K;
  a.codes = (uint8_t*)codes;
  a.scales = (uint8_t*)scales;
  a.row_scale = row_scale;
  a.pitch = code_pitch(K);
  a.tiles = scale_tiles(K, fmt);
  a.align = row_alignment(x, ld * (int64_t)sizeof(T));
  if (fmt == FVB_FP4_MX) {
    const int64_t segs = (a.tiles * 8 + kSegUnits - 1) / kSegUnits, blocks = (M + 7) / 8 * segs;
    FVB_REQUIRE(blocks < (1ll << 31), "fvb_quant_fp4: size");
    a.row_blocks = (unsigned)((M + 7) / 8);
    if (a.align) quant_mx_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>(a);
    else quant_mx_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>(a);
    return check_launch("fvb_quant_fp4");
  }
  const int64_t units = a.tiles * 4;
  const unsigned g1 = (unsigned)M;
  if (units > 1024)
    quant_nv_long_kernel<T><<<g1, 256, 0, st>>>(a);
  else if (a.align)
    quant_nv<T, false>(a, units, st);
  else
    quant_nv<T, true>(a, units, st);
  return check_launch("fvb_quant_fp4");
}

template <typename T>
static int dequant(const void* codes, const void* scales, const float* row_scale, int rs_row,
                   int64_t M, int64_t K, int fmt, void* out, cudaStream_t st) {
  const int64_t segs64 = ((K + 15) / 16 + 31) / 32, blocks = (M + 7) / 8 * segs64;
  FVB_REQUIRE(blocks < (1ll << 31), "fvb_dequant_fp4: size");
  const unsigned grid = (unsigned)blocks, segs = (unsigned)segs64;
  const int64_t pitch = code_pitch(K), tiles = scale_tiles(K, fmt);
  const int align = row_alignment(out, K * (int64_t)sizeof(T));
  const auto c = (const uint8_t*)codes;
  const auto f = (const uint8_t*)scales;
#define FVB_DQ(FMT, STAGED)                                                                      \
  dequant_kernel<T, FMT, STAGED><<<grid, 256, 0, st>>>(c, f, row_scale, rs_row, M, K, pitch, tiles, \
                                                       align, segs, (T*)out)
  if (fmt == FVB_FP4_NV) {
    if (align) FVB_DQ(FVB_FP4_NV, false);
    else FVB_DQ(FVB_FP4_NV, true);
  } else {
    if (align) FVB_DQ(FVB_FP4_MX, false);
    else FVB_DQ(FVB_FP4_MX, true);
  }
#undef FVB_DQ
  return check_launch("fvb_dequant_fp4");
}

}  // namespace fp4
}  // namespace fvb

extern "C" {

size_t fvb_fp4_codes_bytes(int64_t M, int64_t K) {
  return M > 0 && K > 0 ? (size_t)(M * fvb::fp4::code_pitch(K)) : 0;
}

size_t fvb_fp4_scales_bytes(int64_t M, int64_t K, int fmt) {
  if (M <= 0 || K <= 0 || (fmt != FVB_FP4_NV && fmt != FVB_FP4_MX)) return 0;
  return (size_t)((M + 127) / 128 * fvb::fp4::scale_tiles(K, fmt)) * 512;
}

int fvb_quant_fp4(const void* x, int dtype, int64_t ld, int64_t M, int64_t K, int fmt, void* codes,
                  void* scales, float* row_scale, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(M >= 0 && K >= 0, "fvb_quant_fp4: negative size");
  FVB_REQUIRE(M < (1ll << 31) && K < (1ll << 31), "fvb_quant_fp4: size");
  FVB_REQUIRE(fmt == FVB_FP4_NV || fmt == FVB_FP4_MX, "fvb_quant_fp4: format %d", fmt);
  FVB_REQUIRE(dtype == FVB_BF16 || dtype == FVB_F16 || dtype == FVB_F32, "fvb_quant_fp4: dtype %d",
              dtype);
  if (M == 0 || K == 0) return FVB_OK;
  if (ld == 0) ld = K;
  FVB_REQUIRE(ld >= K || M == 1, "fvb_quant_fp4: row pitch %lld < K %lld", (long long)ld,
              (long long)K);
  FVB_REQUIRE(x && codes && scales, "fvb_quant_fp4: NULL pointer");
  FVB_REQUIRE(fmt == FVB_FP4_MX || row_scale, "fvb_quant_fp4: nv needs row_scale");
  FVB_REQUIRE(aligned16(codes) && aligned16(scales),
              "fvb_quant_fp4: codes and scales must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FVB_BF16)
    return fp4::quant<__nv_bfloat16>(x, ld, M, K, fmt, codes, scales, row_scale, st);
  if (dtype == FVB_F16) return fp4::quant<__half>(x, ld, M, K, fmt, codes, scales, row_scale, st);
  return fp4::quant<float>(x, ld, M, K, fmt, codes, scales, row_scale, st);
}

int fvb_dequant_fp4(const void* codes, const void* scales, const float* row_scale, int rs_mode,
                    int64_t M, int64_t K, int fmt, int dtype, void* out, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(M >= 0 && K >= 0, "fvb_dequant_fp4: negative size");
  FVB_REQUIRE(M < (1ll << 31) && K < (1ll << 31), "fvb_dequant_fp4: size");
  FVB_REQUIRE(fmt == FVB_FP4_NV || fmt == FVB_FP4_MX, "fvb_dequant_fp4: format %d", fmt);
  FVB_REQUIRE(dtype == FVB_BF16 || dtype == FVB_F16 || dtype == FVB_F32,
              "fvb_dequant_fp4: dtype %d", dtype);
  FVB_REQUIRE(rs_mode == FVB_SCALE_TENSOR || rs_mode == FVB_SCALE_ROW, "fvb_dequant_fp4: rs_mode");
  if (M == 0 || K == 0) return FVB_OK;
  FVB_REQUIRE(codes && scales && out, "fvb_dequant_fp4: NULL pointer");
  FVB_REQUIRE(aligned16(codes) && aligned16(scales) && aligned16(out),
              "fvb_dequant_fp4: pointers must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  const int rr = rs_mode == FVB_SCALE_ROW;
  if (dtype == FVB_BF16)
    return fp4::dequant<__nv_bfloat16>(codes, scales, row_scale, rr, M, K, fmt, out, st);
  if (dtype == FVB_F16)
    return fp4::dequant<__half>(codes, scales, row_scale, rr, M, K, fmt, out, st);
  return fp4::dequant<float>(codes, scales, row_scale, rr, M, K, fmt, out, st);
}

}  // extern "C"
