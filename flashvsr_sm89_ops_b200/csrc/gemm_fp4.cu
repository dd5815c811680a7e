// Product of two microscaled 4-bit matrices on the 5th-generation tensor cores, with the
// epilogues of a DiT block's linears (fp4.cuh has the formats and the layout).
//
//   acc[m, n] = sum_k A[m, k] W[n, k]      codes times block scales, fp32, in the tensor core
//   y = acc * sa[m] * sw[n] + bias[n]      sa, sw: the nv formats' row scales (mx: 1)
//   out = bf16(y)  or  bf16(res + gate[n] * y)  or  mx codes of GELU(tanh)(y)
//
// Two kernels.  Products with many output tiles run on persistent CTA pairs (cta_group::2, one
// CTA per SM, 256 x 256 tiles of which each CTA holds 128 rows), warp-specialised; those with few
// on a tile per cluster of CTAs that share its K loop (further down).  Measured: 8448 x 4608 x 1536
// nv 33 us (3.6 PFLOP/s), mx 28.5; 8448 x 1536 x 8960 nv 46 us (5.0 PFLOP/s), with the gated
// residual 50; the MMAs of the latter alone 36.5.
//   warp 0      TMA producer: 256-element (128-byte) K blocks of A and W and their scale tiles
//               into a ring of shared-memory stages
//   warp 1      MMA issuer: copies a K block's scale tiles into TMEM (tcgen05.cp), then issues
//               its four block-scaled MMAs (K = 64 each) into the fp32 accumulator
//   warps 2..   epilogue: the warps of a TMEM lane quarter take the tile's 64-column chunks in
//               turn; bf16 through a swizzled staging buffer and a TMA store, a residual into
//               the same buffer by TMA while the tile is still being multiplied
//
// TMEM (512 columns): two accumulators of 256 columns, so that a tile's epilogue runs under the
// next tile's MMAs, and two or more buffers of a K block's scales.  That is more than 512, so
// the second accumulator starts at column 128: the two share half their columns, the epilogue's
// warps read those first, and the next tile's MMAs start when they have been read.  Tiles 192
// wide with separate accumulators move more operands for each flop and measured 39.8 us against
// 36.4 on 8448 x 4608 x 1536 and 62 against 50 on 8448 x 1536 x 8960.
//
// A scale buffer is overwritten after a wait for the MMAs that read it: the issue order puts a
// copy before the MMAs after it, but nothing puts an MMA before a copy after it.  The wait is on
// the ring stage's own barrier; a commit and a wait for every scale tile measured 84.6 us on
// 8448 x 1536 x 8960, where one for every K block took 49.
//
// Shared-memory bandwidth (128 bytes a clock per SM) is what the operands, their TMA writes and
// the epilogue share, and it is nearly used up: a 256-element K block of a 256 x 256 pair tile
// reads 32 KB and writes 38 KB per CTA in the 512 clocks of its MMAs.  So the epilogue reads
// TMEM in the 16x256b shape, where a thread holds 2 columns of every 8 for 4 rows: a 64-column
// chunk's scales and biases then cost a warp 24 wavefronts of shared memory, where a thread
// that holds a whole row reads all 64 columns' and costs it 128.  They travel by shuffles, each
// warp with the two columns a lane that it read one chunk ahead: no barrier between the warps.
#include <atomic>

#include "fp4.cuh"

namespace fvb {
namespace gemm4 {

constexpr int BM = 128;
constexpr int kRowBytes = 128;  // one K block of a row: 256 elements
constexpr int kStageOut = 32 * 128;  // an epilogue warp's staging: 32 rows x 64 bf16

constexpr int kStageCodes = 32 * 32;  // with GELU: 32 rows x 64 codes

enum { kPlain = 0, kResidual = 1, kGeluMx = 2 };

// Epilogue warps per TMEM lane quarter.  The GELU epilogue is the longer part of its product
// (1.5 special functions and the codes for every element), so it has three: they take the
// 64-column chunks of successive tiles in turn and drift out of step, so that one's special
// functions run beside another's sums and conversions.  8448 x 8960 x 1536 (nv) measured 75 us
// with three (78 with gelu2's tail), 87 with two; four leave 96 registers a thread and spill.  The
// others need a 4 KB staging buffer a warp, and a third would cost them a ring stage.
__host__ __device__ constexpr int epi_per_quarter(int epi) { return epi == kGeluMx ? 3 : 2; }

struct Args {
  int M, N, K;
  const float* sa;  // NULL: 1
  const float* sw;
  int sa_row, sw_row;
  const __nv_bfloat16* bias;  // [N] or NULL
  const __nv_bfloat16* res;   // kResidual: [M, N], row pitch ldr
  const __nv_bfloat16* gate;  // kResidual: [N] or NULL (1)
  __nv_bfloat16* out;         // row pitch ldo
  int64_t ldr, ldo;
  int tma_out;      // whether `out` suits a TMA store
  int tma_res;      // whether `res` suits a TMA load
  uint8_t* hcodes;  // kGeluMx
  uint8_t* hscales;
  int64_t hpitch, htiles;
};

template <int FMT, int EPI>
struct Shape {
  static constexpr int BN = 256;
  static constexpr int kEpiWarps = 4 * epi_per_quarter(EPI);
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kOut = EPI == kGeluMx ? kStageCodes : kStageOut;
  static constexpr int kOutBytes = kEpiWarps * kOut;
  static constexpr int kTilesK = FMT == FVB_FP4_NV ? 4 : 2;  // scale tiles per K block
  static constexpr int kMmas = 4 / kTilesK;                  // MMAs (K = 64) per scale tile
  static constexpr int kRowsB = BN / 2;                      // W rows a CTA of the pair stages
  static constexpr int kSfTilesB = BN / 128;                 // 128-row scale tiles of W
  static constexpr int kBytesA = BM * kRowBytes;
  static constexpr int kBytesB = kRowsB * kRowBytes;
  static constexpr int kBytesSfA = kTilesK * 512;
  static constexpr int kBytesSfB = kTilesK * kSfTilesB * 512;
  static constexpr int kBytes = kBytesA + kBytesB + kBytesSfA + kBytesSfB;
  static constexpr int kFixed = kOutBytes + 1024 /*align*/ + 384 /*barriers*/;
  static constexpr int kFit = (227 * 1024 - kFixed) / kBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr size_t kSmem = (size_t)kStages * kBytes + kFixed;
  // TMEM columns
  static constexpr int kAcc1 = BN / 2;                // start of the second accumulator
  static constexpr int kSf = kAcc1 + BN;              // start of the scale buffers
  static constexpr int kSfA = 4 * kTilesK, kSfB = 4 * kTilesK * kSfTilesB;  // columns of one
  static constexpr int kFitSf = (512 - kSf) / (kSfA + kSfB);
  static constexpr int kSfBufs = kFitSf > kStages ? kStages : kFitSf;
  static_assert(kSfBufs >= 2, "TMEM columns");
  static_assert(kStages >= 3, "ring");
};

// D[tmem] (+)= A[smem] * W[smem], E2M1 with block scales in TMEM
template <int FMT, bool PAIR>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define FVB_MMA4(group, kind, vec)                                                           \
  asm volatile(                                                                              \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                      \
      "tcgen05.mma.cta_group::" group ".kind::" kind ".block_scale.scale_vec::" vec          \
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                     \
      "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                      \
      : "memory")
  if (FMT == FVB_FP4_NV) {
    if (PAIR) FVB_MMA4("2", "mxf4nvf4", "4X");
    else FVB_MMA4("1", "mxf4nvf4", "4X");
  } else {
    if (PAIR) FVB_MMA4("2", "mxf4", "2X");
    else FVB_MMA4("1", "mxf4", "2X");
  }
#undef FVB_MMA4
}

// descriptor of one 512-byte scale tile: unswizzled 8-row x 16-byte core matrices, 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// the tile -> 4 TMEM columns of 32 lanes, repeated in the four lane quarters
template <bool PAIR>
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t desc) {
  if (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

// 16 lanes x 64 columns of 32-bit TMEM: register 4 g + 2 h + e of lane l is row l / 4 + 8 h,
// column 8 g + 2 (l % 4) + e
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// four 8 x 8 matrices of 16-bit values: lane l names row l % 8 of matrix l / 8, and register m
// holds row l / 4, columns 2 (l % 4) + {0, 1} of matrix m
__device__ __forceinline__ void stmatrix_x4(uint32_t saddr, const uint32_t* r) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(saddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// into this CTA's shared memory, counted on the barrier at shared::cluster address bar_caddr
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map,
                                                 uint32_t bar_caddr, int32_t x, int32_t y,
                                                 int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_caddr), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// arrive on a barrier of the pair without releasing this thread's earlier stores: what it
// signals is TMEM that has been read (tcgen05.wait::ld), and a release at cluster scope waits
// for the thread's global stores in flight (1300 clocks a tile in the GELU epilogue)
__device__ __forceinline__ void mbar_arrive_remote_relaxed(uint32_t caddr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(caddr) : "memory");
}

// instruction descriptor: E2M1 operands, scale type, M x N; the scale ids (byte of the 4-byte
// scale column an mx MMA starts at) are added per MMA
template <int FMT>
__host__ __device__ constexpr uint32_t idesc4(int M, int N) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
         ((FMT == FVB_FP4_MX ? 1u : 0u) << 23) | ((uint32_t)(M >> 4) << 24);
}

// GELU(tanh) of two values in fp32: x * sigmoid(2 u) = x / (1 + 2^v), u = sqrt(2/pi) (x + c x^3),
// v = -2 u log2(e).  One reciprocal of the product serves both, 1 / a = b / (a b): the
// special-function unit (16 a clock per SM) would bound the epilogue with two for each value.
// So that the product stays finite, x below -7.5 (v = 60.7, GELU = -4e-18) counts as 0; -inf
// becomes NaN there, as 0.5 x (1 + tanh u) has it.  Holding v at 60 instead (3 us of the FFN's 126
// at 8448 x 1536 x 8960 less) leaves x / 2^60: -8.7e11 of -1e30, and a block of nothing but such
// values would be scaled to them.  One minimum over a thread's 64 values and these selects behind a
// branch measured 128 us.
__device__ __forceinline__ uint64_t gelu2(uint64_t x) {
  const float k1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, k3 = k1 * 0.044715f;
  float x0, x1, z0, z1, v0, v1, a, b;
  f2_unpack(x, x0, x1);
  f2_unpack(f2_mul(x, f2_pack(-0.0f, -0.0f)), z0, z1);
  x = f2_pack(x0 < -7.5f ? z0 : x0, x1 < -7.5f ? z1 : x1);
  f2_unpack(f2_mul(x, f2_fma(f2_mul(x, x), f2_pack(k3, k3), f2_pack(k1, k1))), v0, v1);
  f2_unpack(f2_add(f2_pack(ex2_approx(v0), ex2_approx(v1)), f2_pack(1.0f, 1.0f)), a, b);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  return f2_mul(x, f2_pack(b * r, a * r));
}
// GELU and mx quantisation of an epilogue chunk (32 rows x 64 columns, v as in the kernel): the
// codes into the staging buffer at shared address `stg` (32 rows x 32 bytes, 32-byte swizzle),
// the two scale bytes of row lr + 8 k returned in sb[k] by every lane of the row.
// A row's block lies in four neighbouring lanes: its exponent is the maximum of theirs, and the
// code bytes (one per pair of columns) are transposed within the four, so that lane j ends up
// with columns 8 j .. 8 j + 7 of the block as one word.
__device__ __forceinline__ void gelu_mx(uint64_t (&v)[4][8], int col0, int N, int lane, uint32_t stg,
                                        uint32_t* sb) {
  const int lr = lane >> 2, lq = lane & 3;
  if (col0 + 64 > N) {  // columns past N carry whatever scales lie past W's rows
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const int left = N - (col0 + g * 8 + 2 * lq);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (left < 1) v[k][g] &= 0xFFFFFFFF00000000ull;
        if (left < 2) v[k][g] &= 0x00000000FFFFFFFFull;
      }
    }
  }
  // the exponent fields of the 4 rows x 2 blocks, two to a word (255: not finite)
  uint32_t ex[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      v[k][g] = gelu2(v[k][g]);
      m[g >> 2] = fp4::max_abs_nan(m[g >> 2], v[k][g]);
    }
    ex[k] = __byte_perm(__float_as_uint(m[0]) >> 23, __float_as_uint(m[1]) >> 23, 0x5410);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) ex[k] = __vmaxu2(ex[k], __shfl_xor_sync(0xffffffffu, ex[k], 1));
#pragma unroll
  for (int k = 0; k < 4; ++k) ex[k] = __vmaxu2(ex[k], __shfl_xor_sync(0xffffffffu, ex[k], 2));
  uint32_t w[2][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sb[k] = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t e = h ? ex[k] >> 16 : ex[k] & 0xFFFFu;
      // scale byte: amax's exponent field - 2, at least 0; 1 / scale = 2^(127 - byte)
      const uint32_t byte = e > 2u ? e - 2u : 0u;
      const bool bad = e == 255u;
      sb[k] |= (bad ? 255u : byte) << (8 * h);
      const float rs = __uint_as_float((254u - byte) << 23);
      const uint64_t rs2 = f2_pack(rs, rs);
      float x[8];
#pragma unroll
      for (int g = 0; g < 4; ++g) f2_unpack(f2_mul(v[k][4 * h + g], rs2), x[2 * g], x[2 * g + 1]);
      w[h][k] = bad ? 0u : fp4::e2m1x8(x);
    }
  }
  // 4 x 4 byte transposes in each group of four lanes, two words (rows k, k + 1) per exchange:
  // lane bit 0 trades odd for even bytes, lane bit 1 the upper for the lower pair
  const bool o = lane & 1, u = lane & 2;
  const uint32_t give1 = o ? 0x6420u : 0x7531u, keep1p = o ? 0x3514u : 0x5240u,
                 keep1q = o ? 0x3716u : 0x7260u, give2 = u ? 0x5410u : 0x7632u,
                 keep2p = u ? 0x3254u : 0x5410u, keep2q = u ? 0x3276u : 0x7610u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      uint32_t p = w[h][k], q = w[h][k + 1];
      uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(p, q, give1), 1);
      p = __byte_perm(p, got, keep1p);
      q = __byte_perm(q, got, keep1q);
      got = __shfl_xor_sync(0xffffffffu, __byte_perm(p, q, give2), 2);
      w[h][k] = __byte_perm(p, got, keep2p);
      w[h][k + 1] = __byte_perm(q, got, keep2q);
    }
  }
  // 16-byte chunk h of row l lies at chunk h ^ (l / 4 % 2)
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = stg + (lr + 8 * k) * 32 + ((h ^ ((lr >> 2) & 1)) << 4) + lq * 4;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w[h][k]) : "memory");
    }
}

template <int FMT, int EPI>
__global__ void __launch_bounds__(64 + 128 * epi_per_quarter(EPI), 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSfA,
                    const __grid_constant__ CUtensorMap tmSfB,
                    const __grid_constant__ CUtensorMap tmOut,
                    const __grid_constant__ CUtensorMap tmRes, const Args args) {
  using S = Shape<FMT, EPI>;
  constexpr int BN = S::BN;
  constexpr int STAGES = S::kStages;
  constexpr int TM = 2 * BM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = sA + STAGES * S::kBytesA;
  uint8_t* sSfA = sB + STAGES * S::kBytesB;
  uint8_t* sSfB = sSfA + STAGES * S::kBytesSfA;
  uint8_t* sOut = sSfB + STAGES * S::kBytesSfB;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + S::kOutBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;   // [2] accumulator finished
  uint64_t* tempty = tfull + 2;       // [2] the columns shared with the other accumulator read
  uint64_t* tdone = tempty + 2;       // [2] the other columns read
  uint64_t* drain = tdone + 2;        // every MMA this CTA issued finished
  uint64_t* rfull = drain + 1;        // [epilogue warps] residual arrived
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + S::kEpiWarps);
  uint32_t* pair_ok = tmem_slot + 1;

  const int warp = warp_id_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int unit = (int)(blockIdx.x >> 1);
  const int units = (int)(gridDim.x >> 1);
  const int m_tiles = (args.M + TM - 1) / TM;
  const int n_tiles = (args.N + BN - 1) / BN;
  const int num_tiles = m_tiles * n_tiles;
  const int kblocks = (args.K + 255) / 256;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);  // 2 CTAs x 4 lane quarters x 2 chunks
      mbar_init(&tdone[b], 16);
    }
    mbar_init(drain, 1);
    for (int w = 0; w < S::kEpiWarps; ++w) mbar_init(&rfull[w], 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSfA);
    prefetch_tmap(&tmSfB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  if (threadIdx.x == 0)
    *pair_ok = ld_shared_cluster_u32(mapa_shared(smem_u32(tmem_slot), rank ^ 1u)) == *tmem_slot;
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // a pair whose TMEM addresses differ (never expected) does no work and reports it
  const bool run = *pair_ok != 0u;
  if (!run && threadIdx.x == 0 && rank == 0) atomicCAS(&g_device_error, 0u, 0x40Cu);
  const uint32_t full0_c = mapa_shared(smem_u32(full), 0u);
  const uint32_t tempty0_c = mapa_shared(smem_u32(tempty), 0u);

  if (!run) {
    // straight to the teardown
  } else if (warp == 0) {
    // ------------------------------------------------------------ producer
    // like the MMA issuer below, the whole warp walks the loop and one elected lane issues
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int64_t issued = 0;
    for (int tile = unit; tile < num_tiles && ok; tile += units) {
      const int m0 = (tile / n_tiles) * TM + (int)rank * BM;
      const int nt = (tile % n_tiles) * BN;
      const int n0 = nt + (int)rank * S::kRowsB;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, 0x401u))) {
          ok = false;
          break;
        }
        if (leader) {
          uint8_t* a = sA + stage * S::kBytesA;
          uint8_t* b = sB + stage * S::kBytesB;
          uint8_t* fa = sSfA + stage * S::kBytesSfA;
          uint8_t* fb = sSfB + stage * S::kBytesSfB;
          // scale tiles past the last of a row are filled with zeros
          // the even CTA arms its barrier for both CTAs' bytes
          const uint32_t bar = full0_c + 8u * stage;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], (uint32_t)(2 * S::kBytes));
          tma_load_2d_pair(a, &tmA, bar, kb * kRowBytes, m0);
          tma_load_2d_pair(b, &tmB, bar, kb * kRowBytes, n0);
          tma_load_3d_pair(fa, &tmSfA, bar, 0, kb * S::kTilesK, m0 >> 7);
          tma_load_3d_pair(fb, &tmSfB, bar, 0, kb * S::kTilesK, nt >> 7);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // no load may still be writing shared memory when its CTA exits: the last STAGES loads
    // are the newest phase of their stages' full barriers (a pair's are the even CTA's)
    if (rank == 0)
      for (int64_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
        mbar_wait(&full[i % STAGES], (uint32_t)((i / STAGES) & 1), 0x40Au);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop, so addresses and descriptors stay warp-uniform (the form
    // the tensor instructions take them in); one elected lane issues.
    if (rank == 0) {
      constexpr uint32_t idesc = idesc4<FMT>(TM, BN);
      const bool leader = elect_one();
      const int ksteps = (args.K + 63) / 64;
      const uint64_t descA = smem_desc_sw128(smem_u32(sA), 16, 1024);
      const uint64_t descB = smem_desc_sw128(smem_u32(sB), 16, 1024);
      const uint64_t descFA = scale_desc(smem_u32(sSfA));
      const uint64_t descFB = scale_desc(smem_u32(sSfB));
      int stage = 0;
      uint32_t phase = 0;
      int t = 0;
      int sbuf = 0;  // scale buffer, and the stage and parity of the K block that had it last
      int old_stage = 0;
      uint32_t old_phase = 0;
      bool reuse = false;
      bool ok = true, any = false;
      for (int tile = unit; tile < num_tiles && ok; tile += units, ++t) {
        const int buf = t & 1;
        // until the columns shared with the previous tile were read, and the others of the tile
        // before it, whose accumulator this is
        const bool clear =
            (t < 1 || mbar_wait(&tempty[buf ^ 1], (uint32_t)((t - 1) >> 1) & 1u, 0x402u)) &&
            (t < 2 || mbar_wait(&tdone[buf], (uint32_t)((t - 2) >> 1) & 1u, 0x407u));
        if (!__all_sync(0xffffffffu, clear)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * S::kAcc1);
        for (int kb = 0; kb < kblocks && ok; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, 0x403u))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = descA + (uint32_t)(stage * (S::kBytesA >> 4));
          const uint64_t db = descB + (uint32_t)(stage * (S::kBytesB >> 4));
          const uint64_t fa = descFA + (uint32_t)(stage * (S::kBytesSfA >> 4));
          const uint64_t fb = descFB + (uint32_t)(stage * (S::kBytesSfB >> 4));
          const int left = ksteps - kb * 4;  // K steps from this block on
          if (reuse && S::kSfBufs < STAGES) {
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[old_stage], old_phase, 0x405u))) {
              ok = false;
              break;
            }
            if (++old_stage == STAGES) {
              old_stage = 0;
              old_phase ^= 1u;
            }
          }
          const uint32_t sfa = tmem + (uint32_t)(S::kSf + sbuf * (S::kSfA + S::kSfB));
          const uint32_t sfb = sfa + (uint32_t)S::kSfA;
          if (leader) {
#pragma unroll
            for (int i = 0; i < S::kTilesK; ++i) {
              cp_scales<true>(sfa + 4u * i, fa + i * 512 / 16);
#pragma unroll
              for (int r = 0; r < S::kSfTilesB; ++r)
                cp_scales<true>(sfb + (uint32_t)(4 * (S::kSfTilesB * i + r)),
                                fb + (r * S::kTilesK + i) * 512 / 16);
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              // an mx MMA takes two bytes of the four in a scale column
              const uint32_t i = ks / S::kMmas, id = 2u * (ks % S::kMmas);
              if (ks < left)
                mma_fp4<FMT, true>(d, da + 2 * ks, db + 2 * ks, idesc | (id << 4) | (id << 29),
                                   sfa + 4u * i, sfb + 4u * S::kSfTilesB * i,
                                   (kb | ks) != 0 ? 1u : 0u);
            }
            tc_commit_pair_both(&empty[stage], 0x3);
            if (kb + 1 == kblocks) tc_commit_pair_both(&tfull[buf], 0x3);
          }
          __syncwarp();
          any = true;
          if (++sbuf == S::kSfBufs) {
            sbuf = 0;
            reuse = true;
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every MMA issued above completes before TMEM is freed
      if (any) {
        if (leader) tc_commit_pair(drain);
        __syncwarp();
        mbar_wait(drain, 0, 0x40Bu);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // A tile is four 64-column chunks; chunk n = 4 * (tile's number) + position goes to the warp
    // n % G of its lane quarter.  Positions 0 and 1 are the columns shared with the other
    // accumulator (the first accumulator's last two chunks, the second's first two).
    constexpr int G = epi_per_quarter(EPI);
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const int lr = lane >> 2, lc = 2 * (lane & 3);  // this thread's rows lr + 8 k, columns 8 g + lc + {0, 1}
    uint8_t* stg = sOut + (size_t)(warp - 2) * S::kOut;
    uint64_t* rbar = &rfull[warp - 2];
    const uint32_t tdone0_c = mapa_shared(smem_u32(tdone), 0u);
    const bool tma_res = EPI == kResidual && args.tma_res;
    // A chunk's vectors, two columns and four rows a lane, loaded one chunk ahead and left as they
    // arrive (any arithmetic on them here would wait for the loads); the lanes that need a column
    // get it by shuffles
    struct Vectors {
      float s0, s1, sa[4];
      uint16_t b0, b1, g0, g1;
    };
    auto place = [&](int n, int& m0, int& col0) {  // false past the last tile
      const int tile = unit + (n >> 2) * units;
      if (tile >= num_tiles) return false;
      m0 = (tile / n_tiles) * TM + (int)rank * BM + q * 32;
      col0 = (tile % n_tiles) * BN + (((n & 3) + (n & 4 ? 0 : 2)) & 3) * 64;
      return true;
    };
    auto vectors = [&](int n) {
      Vectors c = {1.f, 1.f, {1.f, 1.f, 1.f, 1.f}, 0, 0, 0x3F80, 0x3F80};
      int m0, col0;
      if (place(n, m0, col0)) {
        const int col = col0 + 2 * lane;
        const bool in0 = col < args.N, in1 = col + 1 < args.N;
        const uint16_t* bias = reinterpret_cast<const uint16_t*>(args.bias) + col;
        const uint16_t* gate = reinterpret_cast<const uint16_t*>(args.gate) + col;
        if (args.sw && in0) c.s0 = __ldg(args.sw + (args.sw_row ? col : 0));
        if (args.sw && in1) c.s1 = __ldg(args.sw + (args.sw_row ? col + 1 : 0));
        if (args.bias && in0) c.b0 = __ldg(bias);
        if (args.bias && in1) c.b1 = __ldg(bias + 1);
        if (EPI == kResidual && args.gate && in0) c.g0 = __ldg(gate);
        if (EPI == kResidual && args.gate && in1) c.g1 = __ldg(gate + 1);
        if (args.sa) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = m0 + lr + 8 * k;
            if (row < args.M) c.sa[k] = __ldg(args.sa + (args.sa_row ? row : 0));
          }
        }
      }
      return c;
    };
    auto unpack = [](uint32_t w) {
      return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    };
    int n = (warp - 2) >> 2, m0, col0;
    Vectors ahead = vectors(n);
    uint32_t rphase = 0;
#pragma unroll 1
    for (; place(n, m0, col0); n += G) {
      const int t = n >> 2, buf = t & 1;
      const bool cols_ok = col0 < args.N;  // warp-uniform
      {
        if (tma_res && cols_ok && lane == 0) {  // the chunk's residual into the staging buffer
          tma_store_wait_read<0>();               // which the last store has left
          mbar_arrive_expect_tx(rbar, kStageOut);
          tma_load_2d(stg, &tmRes, rbar, col0, m0);
        }
        const Vectors vec = ahead;
        ahead = vectors(n + G);
        const uint32_t bias = __byte_perm(vec.b0, vec.b1, 0x5410);
        uint64_t sa2[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) sa2[k] = f2_pack(vec.sa[k], vec.sa[k]);
        if (!__all_sync(0xffffffffu, mbar_wait(&tfull[buf], (uint32_t)(t >> 1) & 1u, 0x404u))) {
          if (tma_res && cols_ok) mbar_wait(rbar, rphase, 0x406u);
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) +
                             (uint32_t)(buf * S::kAcc1 + (((n & 3) + (n & 4 ? 0 : 2)) & 3) * 64);
        uint32_t r[64];
        // v[k][g]: row lr + 8 k, columns 8 g + lc and the next, as an fp32 pair
        tmem_ld_16x256b_x8(acc, r);
        tmem_ld_16x256b_x8(acc + (16u << 16), r + 32);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_relaxed(((n & 3) < 2 ? tempty0_c : tdone0_c) + 8u * buf);
        uint64_t v[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int i0 = (k >> 1) * 32 + g * 4 + (k & 1) * 2;
            v[k][g] = f2_pack(__uint_as_float(r[i0]), __uint_as_float(r[i0 + 1]));
          }
        if (cols_ok) {
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int from = 4 * g + (lane & 3);
            const uint64_t b2 = unpack(__shfl_sync(0xffffffffu, bias, from));
            if (args.sw) {
              const uint64_t s2 = f2_pack(__shfl_sync(0xffffffffu, vec.s0, from),
                                          __shfl_sync(0xffffffffu, vec.s1, from));
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k][g] = f2_fma(v[k][g], f2_mul(sa2[k], s2), b2);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k][g] = f2_fma(v[k][g], sa2[k], b2);
            }
          }
        }
        if constexpr (EPI == kGeluMx) {
          uint32_t sb[4] = {0u, 0u, 0u, 0u};  // past the last block: the next product reads whole tiles
          if (cols_ok) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            gelu_mx(v, col0, args.N, lane, smem_u32(stg), sb);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {  // ends at the rows' pitch
              tma_store_2d(&tmOut, stg, col0 >> 1, m0);
              tma_store_commit();
            }
          }
          // scale_at(row, col0 / 32): the warp's rows are one 4-byte column of their tile; lane
          // lq of a row's four stores row lr + 8 lq
          const int k = lane & 3;
          const uint32_t b = k == 0 ? sb[0] : k == 1 ? sb[1] : k == 2 ? sb[2] : sb[3];
          if (m0 + lr + 8 * k < args.M && (col0 >> 7) < args.htiles)
            *reinterpret_cast<uint16_t*>(args.hscales + ((m0 >> 7) * args.htiles + (col0 >> 7)) * 512 +
                                         (lr + 8 * k) * 16 + q * 4 + ((col0 >> 5) & 3)) = (uint16_t)b;
          continue;
        }
        if (!cols_ok) continue;
        // 128-byte swizzle of the staging rows: 16-byte chunk g of row l lies at chunk g ^ (l % 8);
        // lane l names row l of a group's 32 rows x 8 columns
        const uint32_t srow = smem_u32(stg) + lane * 128;
        if (EPI == kResidual) {
          if (tma_res) {
            if (!__all_sync(0xffffffffu, mbar_wait(rbar, rphase, 0x406u))) break;
            rphase ^= 1u;
          }
          const uint32_t gate = __byte_perm(vec.g0, vec.g1, 0x5410);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            uint32_t x[4];
            if (tma_res) {
              ldmatrix_x4(x, srow + ((g ^ (lane & 7)) << 4));
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int row = m0 + lr + 8 * k, col = col0 + g * 8 + lc;
                const __nv_bfloat16* rp = args.res + (int64_t)row * args.ldr + col;
                __nv_bfloat162 p = __float2bfloat162_rn(0.f);
                if (row < args.M && col < args.N) p.x = rp[0];
                if (row < args.M && col + 1 < args.N) p.y = rp[1];
                x[k] = *reinterpret_cast<uint32_t*>(&p);
              }
            }
            const uint64_t g2 = unpack(__shfl_sync(0xffffffffu, gate, 4 * g + (lane & 3)));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[k][g] = f2_fma(g2, v[k][g], unpack(x[k]));
            }
          }
        }
        if (args.tma_out) {
          if (!tma_res && lane == 0) tma_store_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float v0, v1;
              f2_unpack(v[k][g], v0, v1);
              const __nv_bfloat162 p = __floats2bfloat162_rn(v0, v1);
              o[k] = *reinterpret_cast<const uint32_t*>(&p);
            }
            stmatrix_x4(srow + ((g ^ (lane & 7)) << 4), o);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, stg, col0, m0);
            tma_store_commit();
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = m0 + lr + 8 * k;
            __nv_bfloat16* op = args.out + (int64_t)row * args.ldo + col0;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              float v0, v1;
              f2_unpack(v[k][g], v0, v1);
              const int col = col0 + g * 8 + lc;
              if (row < args.M && col < args.N) op[g * 8 + lc] = __float2bfloat16_rn(v0);
              if (row < args.M && col + 1 < args.N) op[g * 8 + lc + 1] = __float2bfloat16_rn(v1);
            }
          }
          if (tma_res) {  // the next residual load writes what this warp has read
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) tma_store_wait0();
  }
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// Few output tiles: a 128 x 128 tile for each cluster of Z CTAs, each CTA a part of K.
//
// What bounds such a product is not a rate but how many SMs read the weight and how long one of
// them is in its K loop: 129 x 1536 x 8960 has 6 pair tiles, 12 of 148 SMs for 16.6 us.  The
// CTAs of a cluster leave their fp32 partial tiles in their own shared memory (the ring's, which
// is free by then) and each adds up and finishes a share of the rows, reading the others' over
// the cluster in the order of their ranks, so the sums do not depend on timing.  No workspace.
// ---------------------------------------------------------------------------------------------
template <int FMT>
struct Split {
  static constexpr int BN = 128;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kTilesK = FMT == FVB_FP4_NV ? 4 : 2;
  static constexpr int kMmas = 4 / kTilesK;
  static constexpr int kBytesA = BM * kRowBytes, kBytesB = BN * kRowBytes, kBytesSf = kTilesK * 512;
  static constexpr int kBytes = kBytesA + kBytesB + 2 * kBytesSf;
  static constexpr int kStages = 6;
  static constexpr size_t kSmem = (size_t)kStages * kBytes + BM * 4 /*row scales*/ + 1024 + 256;
  static constexpr int kSf = BN;             // TMEM: accumulator, then a scale buffer per stage
  static constexpr int kSfCols = 8 * kTilesK;
  static_assert(kSf + kStages * kSfCols <= 512, "TMEM columns");
  static_assert(kStages * (kBytesA + kBytesB) >= BM * BN * 4, "partial tile");
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t caddr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(caddr));
  return v;
}

// SPLIT: Z > 1
template <int FMT, int EPI, bool SPLIT>
__global__ void __launch_bounds__(Split<FMT>::kThreads, 1)
    fp4_gemm_split_kernel(const __grid_constant__ CUtensorMap tmA,
                          const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmSfA,
                          const __grid_constant__ CUtensorMap tmSfB, const Args args, const int Z) {
  using S = Split<FMT>;
  constexpr int STAGES = S::kStages, BN = S::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = sA + STAGES * S::kBytesA;
  uint8_t* sSfA = sB + STAGES * S::kBytesB;
  uint8_t* sSfB = sSfA + STAGES * S::kBytesSf;
  float* sRow = reinterpret_cast<float*>(sSfB + STAGES * S::kBytesSf);  // the tile's row scales
  uint64_t* full = reinterpret_cast<uint64_t*>(sRow + BM);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);

  const int warp = warp_id_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t z = SPLIT ? cluster_ctarank() : 0u;
  const int tile = (int)(blockIdx.x >> (31 - __clz(Z)));
  const int n_tiles = (args.N + BN - 1) / BN;
  const int m0 = tile / n_tiles * BM, n0 = tile % n_tiles * BN;
  const int kblocks = (args.K + 255) / 256;
  // Z is 1, 2, 4 or 8
  const int zs = 31 - __clz(Z), k0 = (kblocks * (int)z) >> zs, k1 = (kblocks * ((int)z + 1)) >> zs;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(tfull, 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSfA);
    prefetch_tmap(&tmSfB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const bool leader = elect_one();
    int issued = 0, stage = 0;
    uint32_t phase = 0;
    for (int kb = k0; kb < k1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, 0x421u))) break;
      if (leader) {
        mbar_arrive_expect_tx(&full[stage], (uint32_t)S::kBytes);
        tma_load_2d(sA + stage * S::kBytesA, &tmA, &full[stage], kb * kRowBytes, m0);
        tma_load_2d(sB + stage * S::kBytesB, &tmB, &full[stage], kb * kRowBytes, n0);
        tma_load_3d(sSfA + stage * S::kBytesSf, &tmSfA, &full[stage], 0, kb * S::kTilesK, m0 >> 7);
        tma_load_3d(sSfB + stage * S::kBytesSf, &tmSfB, &full[stage], 0, kb * S::kTilesK, n0 >> 7);
      }
      __syncwarp();
      ++issued;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // no load may still be writing shared memory when the partial tile goes there or the CTA exits
    for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
      mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u, 0x42Au);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = idesc4<FMT>(BM, BN);
    const bool leader = elect_one();
    const uint64_t descA = smem_desc_sw128(smem_u32(sA), 16, 1024);
    const uint64_t descB = smem_desc_sw128(smem_u32(sB), 16, 1024);
    const uint64_t descFA = scale_desc(smem_u32(sSfA));
    const uint64_t descFB = scale_desc(smem_u32(sSfB));
    const int ksteps = (args.K + 63) / 64;
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = k0; kb < k1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, 0x423u))) break;
      tc_fence_after();
      const uint64_t da = descA + (uint32_t)(stage * (S::kBytesA >> 4));
      const uint64_t db = descB + (uint32_t)(stage * (S::kBytesB >> 4));
      const uint64_t fa = descFA + (uint32_t)(stage * (S::kBytesSf >> 4));
      const uint64_t fb = descFB + (uint32_t)(stage * (S::kBytesSf >> 4));
      const int left = ksteps - kb * 4;
      // the stage's own scale columns: its last MMAs are done, or the stage were not full again
      const uint32_t sfa = tmem + (uint32_t)(S::kSf + stage * S::kSfCols);
      const uint32_t sfb = sfa + (uint32_t)(4 * S::kTilesK);
      if (leader) {
#pragma unroll
        for (int i = 0; i < S::kTilesK; ++i) {
          cp_scales<false>(sfa + 4u * i, fa + i * 512 / 16);
          cp_scales<false>(sfb + 4u * i, fb + i * 512 / 16);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t i = ks / S::kMmas, id = 2u * (ks % S::kMmas);
          if (ks < left)
            mma_fp4<FMT, false>(tmem, da + 2 * ks, db + 2 * ks, idesc | (id << 4) | (id << 29),
                                sfa + 4u * i, sfb + 4u * i, kb != k0 || ks != 0 ? 1u : 0u);
        }
        tc_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // every MMA issued above has finished when this arrives
    if (leader) tc_commit(tfull);
    __syncwarp();
    mbar_wait(tfull, 0, 0x42Bu);
  }

  // ------------------------------------------------------------ partial tiles, sum, epilogue
  const int et = (int)threadIdx.x - 64;
  const int u = et & 15;  // this thread's 8 columns of every row it finishes
  const int col = n0 + u * 8;
  float sw[8], bias[8], gate[8];
  bool ok = true;
  if (warp >= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = col + i < args.N;
      sw[i] = args.sw ? (args.sw_row ? (in ? __ldg(args.sw + col + i) : 0.f) : __ldg(args.sw)) : 1.f;
      bias[i] = args.bias && in ? __bfloat162float(args.bias[col + i]) : 0.f;
      gate[i] = EPI == kResidual && args.gate && in ? __bfloat162float(args.gate[col + i]) : 1.f;
    }
    if (et < BM)
      sRow[et] = args.sa && m0 + et < args.M ? __ldg(args.sa + (args.sa_row ? m0 + et : 0)) : 1.f;
    ok = __all_sync(0xffffffffu, mbar_wait(tfull, 0, 0x424u));
    tc_fence_after();
    const int q = warp & 3, c = (warp - 2) >> 2;
    uint32_t r[64];
    const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(c * 64);
    tmem_ld_16x256b_x8(acc, r);
    tmem_ld_16x256b_x8(acc + (16u << 16), r + 32);
    tmem_ld_wait();
    // row pitch 512 bytes, 32-byte units of 8 columns: unit w of row l at w ^ (l % 8)
    const int lr = lane >> 2, lq = lane & 3;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const int row = q * 32 + lr + 8 * k, w = (c * 8 + g) ^ (row & 7);
        const int i0 = (k >> 1) * 32 + g * 4 + (k & 1) * 2;
        *reinterpret_cast<uint2*>(base + row * 512 + w * 32 + lq * 8) = make_uint2(r[i0], r[i0 + 1]);
      }
  }
  tc_fence_before();
  if (SPLIT) cluster_sync_all();
  else __syncthreads();
  if (warp >= 2) {
    const int rows = args.M - m0 < BM ? args.M - m0 : BM;
    const uint32_t base_u = smem_u32(base);
    // whole warps go round (the GELU form shuffles); two rows a warp
#pragma unroll 4
    for (int it = (int)z * 16 + (et >> 4); (it & ~1) < rows; it += Z * 16) {
      const int rl = it, row = m0 + rl;
      const bool in = rl < rows && ok;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      if (in) {
        const uint32_t at = base_u + rl * 512 + ((u ^ (rl & 7)) << 5);
        if (!SPLIT) {
          const float4* own = reinterpret_cast<const float4*>(base + (at - base_u));
          const float4 a = own[0], b = own[1];
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
          v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
        // four ranks' values on their way at once (one at a time, eight cost 3 us)
        for (int p0 = 0; SPLIT && p0 < Z; p0 += 4) {
          float4 a[4], b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p0 + j < Z) {
              const uint32_t ca = mapa_shared(at, (uint32_t)(p0 + j));
              a[j] = ld_cluster_f4(ca);
              b[j] = ld_cluster_f4(ca + 16);
            }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p0 + j < Z) {
              v[0] += a[j].x; v[1] += a[j].y; v[2] += a[j].z; v[3] += a[j].w;
              v[4] += b[j].x; v[5] += b[j].y; v[6] += b[j].z; v[7] += b[j].w;
            }
        }
      }
      const float sa = sRow[rl & (BM - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmaf_rn(v[i], sa * sw[i], bias[i]);
      if constexpr (EPI == kGeluMx) {
        uint64_t p[4];
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (col + 2 * i >= args.N) v[2 * i] = 0.f;
          if (col + 2 * i + 1 >= args.N) v[2 * i + 1] = 0.f;
          p[i] = gelu2(f2_pack(v[2 * i], v[2 * i + 1]));
          m = fp4::max_abs_nan(m, p[i]);
        }
        uint32_t e = __float_as_uint(m) >> 23;  // amax's exponent field over the block's four lanes
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
        const uint32_t byte = e > 2u ? e - 2u : 0u;
        const float rs = __uint_as_float((254u - byte) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) f2_unpack(f2_mul(p[i], f2_pack(rs, rs)), v[2 * i], v[2 * i + 1]);
        if (in) {
          if ((col >> 1) < args.hpitch)
            *reinterpret_cast<uint32_t*>(args.hcodes + (int64_t)row * args.hpitch + (col >> 1)) =
                e == 255u ? 0u : fp4::e2m1x8(v);
          if ((u & 3) == 0)
            args.hscales[fp4::scale_at(row, col >> 5, args.htiles)] = (uint8_t)(e == 255u ? 255u : byte);
        }
      } else if (in && col < args.N) {
        if (EPI == kResidual) {
          const __nv_bfloat16* rp = args.res + (int64_t)row * args.ldr + col;
          float x[8];
          if (args.tma_res && col + 8 <= args.N) {  // 16-byte aligned rows
            bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(rp)), x);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = col + i < args.N ? __bfloat162float(rp[i]) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __fmaf_rn(gate[i], v[i], x[i]);
        }
        __nv_bfloat16* op = args.out + (int64_t)row * args.ldo + col;
        if (args.tma_out && col + 8 <= args.N) {
          *reinterpret_cast<uint4*>(op) = f32_to_bf16x8(v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col + i < args.N) op[i] = __float2bfloat16_rn(v[i]);
        }
      }
    }
  }
  // neither shared memory that a peer reads nor TMEM goes before everybody is done
  if (SPLIT) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct Operand {
  const void* codes;
  const void* scales;
};

// codes of A in boxes of 128 rows and of W in boxes of `rows_b`, a K block wide; the scale tiles
// of a K block for one 128-row band of A and for `bands_b` of W
template <int FMT>
static int operand_maps(const Args& a, const Operand& A, const Operand& W, int rows_b, int bands_b,
                        CUtensorMap& tmA, CUtensorMap& tmB, CUtensorMap& tmSfA, CUtensorMap& tmSfB) {
  const int64_t pitch = fp4::code_pitch(a.K);
  const int64_t tiles = fp4::scale_tiles(a.K, FMT);
  constexpr int kTilesK = FMT == FVB_FP4_NV ? 4 : 2;
  int rc = make_tmap_2d(&tmA, A.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)pitch,
                        (uint64_t)a.M, (uint64_t)pitch, kRowBytes, BM, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_tmap_2d(&tmB, W.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)pitch, (uint64_t)a.N,
                    (uint64_t)pitch, kRowBytes, (uint32_t)rows_b, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  // scales as 32-bit words of [band of 128 rows][tile][128 words]
  rc = make_tmap_3d(&tmSfA, A.scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 128, (uint64_t)tiles,
                    (uint64_t)((a.M + 127) / 128), 512, (uint64_t)tiles * 512, 128, kTilesK, 1);
  if (rc) return rc;
  return make_tmap_3d(&tmSfB, W.scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 128, (uint64_t)tiles,
                      (uint64_t)((a.N + 127) / 128), 512, (uint64_t)tiles * 512, 128, kTilesK,
                      (uint32_t)bands_b);
}

template <int FMT, int EPI>
static int launch(const Args& a, const Operand& A, const Operand& W, cudaStream_t st) {
  using S = Shape<FMT, EPI>;
  CUtensorMap tmA, tmB, tmSfA, tmSfB, tmO, tmR;
  int rc = operand_maps<FMT>(a, A, W, S::kRowsB, S::kSfTilesB, tmA, tmB, tmSfA, tmSfB);
  if (rc) return rc;
  tmO = tmA;  // unused unless tma_out
  if (EPI == kGeluMx) {
    rc = make_tmap_2d(&tmO, a.hcodes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)a.hpitch,
                      (uint64_t)a.M, (uint64_t)a.hpitch, 32, 32, CU_TENSOR_MAP_SWIZZLE_32B);
    if (rc) return rc;
  } else if (a.tma_out) {
    rc = make_tmap_2d(&tmO, a.out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.N,
                      (uint64_t)a.M, (uint64_t)a.ldo * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  tmR = tmA;  // unused unless tma_res
  if (a.tma_res) {
    rc = make_tmap_2d(&tmR, a.res, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.N,
                      (uint64_t)a.M, (uint64_t)a.ldr * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  auto kern = fp4_gemm_kernel<FMT, EPI>;
  constexpr size_t smem = S::kSmem;
  static_assert(smem <= 227 * 1024, "fp4 gemm: shared memory");
  static std::atomic<bool> configured[64];  // calls of several threads may meet here
  static std::atomic<int> pair_slots[64];
  int dev = 0;
  FVB_CUDA_TRY(cudaGetDevice(&dev), "fp4 gemm device");
  FVB_REQUIRE(dev >= 0 && dev < 64, "fp4 gemm: device ordinal %d", dev);
  constexpr int TM = 2 * BM;
  const int64_t n_tiles64 = (int64_t)((a.M + TM - 1) / TM) * ((a.N + S::BN - 1) / S::BN);
  FVB_REQUIRE(n_tiles64 < (1ll << 31) - 4096, "fp4 gemm: too many output tiles");
  const int num = (int)n_tiles64;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!configured[dev].load(std::memory_order_acquire)) {
    FVB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                 "fp4 gemm smem attribute");
    int clusters = 0;
    cfg.gridDim = dim3(2 * (sm_count() / 2));
    FVB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg), "fp4 gemm cluster occupancy");
    FVB_REQUIRE(clusters > 0, "fp4 gemm: no 2-CTA cluster fits on this device");
    pair_slots[dev].store(clusters, std::memory_order_relaxed);
    configured[dev].store(true, std::memory_order_release);
  }
  const int slots = pair_slots[dev].load(std::memory_order_relaxed);
  cfg.gridDim = dim3(2 * (num < slots ? num : slots));
  FVB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmSfA, tmSfB, tmO, tmR, a),
               "fp4 gemm launch");
  return check_launch("fp4 gemm");
}

template <int FMT, int EPI, bool SPLIT>
static int launch_split(const Args& a, const Operand& A, const Operand& W, int Z, cudaStream_t st) {
  using S = Split<FMT>;
  CUtensorMap tmA, tmB, tmSfA, tmSfB;
  int rc = operand_maps<FMT>(a, A, W, S::BN, 1, tmA, tmB, tmSfA, tmSfB);
  if (rc) return rc;
  auto kern = fp4_gemm_split_kernel<FMT, EPI, SPLIT>;
  static std::atomic<bool> configured[64];  // calls of several threads may meet here
  int dev = 0;
  FVB_CUDA_TRY(cudaGetDevice(&dev), "fp4 gemm device");
  FVB_REQUIRE(dev >= 0 && dev < 64, "fp4 gemm: device ordinal %d", dev);
  if (!configured[dev].load(std::memory_order_acquire)) {
    FVB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem),
                 "fp4 gemm smem attribute");
    configured[dev].store(true, std::memory_order_release);
  }
  const int64_t tiles = (int64_t)((a.M + BM - 1) / BM) * ((a.N + S::BN - 1) / S::BN);
  FVB_REQUIRE(tiles * Z < (1ll << 31), "fp4 gemm: too many output tiles");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(S::kThreads);
  cfg.gridDim = dim3((unsigned)(tiles * Z));
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  if (SPLIT) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = Z;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  FVB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmSfA, tmSfB, a, Z), "fp4 gemm launch");
  return check_launch("fp4 gemm");
}

// Pair tiles for products that fill the machine with them, split tiles for the rest: whichever
// the fitted times (in 10 ns) call shorter.  A K block takes a pair tile 0.37 us and a split tile
// 0.25, a wave 1.3 and 3.0 us besides (fill and epilogue, which split tiles do not overlap), and
// Z parts of K cost their exchange.  Measured (us), pair / Z = 1 / 2 / 4:
//   129 x 1536 x 8960  16.6 / 11.9 / 10.6 / 10.0     16 x 1536 x 8960    16.0 / 10.6 / 8.5 / 7.4
//   1024 x 1536 x 1536  8.1 /  6.3 / 14.1 / 24.7     517 x 1544 x 1000    7.6 /  5.5 / 7.6 / 15.9
//   2048 x 1536 x 1536  8.5 / 10.8                   1024 x 1536 x 8960  18.1 / 12.9
// Clusters that do not all fit at once (more than about 128 CTAs) lose more than they give.
template <int FMT, int EPI>
static int dispatch(const Args& a, const Operand& A, const Operand& W, cudaStream_t st) {
  const int64_t kb = (a.K + 255) / 256, sms = sm_count();
  const int64_t pairs = (int64_t)((a.M + 255) / 256) * ((a.N + 255) / 256);
  const int64_t tiles = (int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128);
  const int64_t pair_cost = (pairs + sms / 2 - 1) / (sms / 2) * (37 * kb + 130) + 500;
  int best = 1;
  int64_t split_cost = (tiles + sms - 1) / sms * (25 * kb + 300) + 50;
  for (int z = 2; z <= 8 && z <= kb && tiles * z <= 128; z *= 2) {
    const int64_t cost = 25 * ((kb + z - 1) / z) + 470 + 60 * z;
    if (cost < split_cost) {
      split_cost = cost;
      best = z;
    }
  }
  if (pair_cost <= split_cost) return launch<FMT, EPI>(a, A, W, st);
  return best > 1 ? launch_split<FMT, EPI, true>(a, A, W, best, st)
                  : launch_split<FMT, EPI, false>(a, A, W, 1, st);
}

template <int EPI>
static int dispatch_fmt(int fmt, const Args& a, const Operand& A, const Operand& W, cudaStream_t st) {
  return fmt == FVB_FP4_NV ? dispatch<FVB_FP4_NV, EPI>(a, A, W, st)
                           : dispatch<FVB_FP4_MX, EPI>(a, A, W, st);
}

// checks shared by the entry points; fills the operand half of `g`
static int operands(const char* who, const void* A, const void* sfA, const float* rsA, int a_mode,
                    const void* W, const void* sfW, const float* rsW, int w_mode, int fmt,
                    int64_t M, int64_t N, int64_t K, Args& g, Operand& oa, Operand& ow) {
  FVB_REQUIRE(K > 0, "%s: K=%lld must be positive", who, (long long)K);
  FVB_REQUIRE(A && sfA && W && sfW, "%s: NULL pointer", who);
  FVB_REQUIRE(aligned16(A) && aligned16(sfA) && aligned16(W) && aligned16(sfW),
              "%s: codes and scales must be 16-byte aligned", who);
  g = Args{};
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  if (fmt == FVB_FP4_NV) {
    g.sa = rsA;
    g.sw = rsW;
    g.sa_row = a_mode == FVB_SCALE_ROW;
    g.sw_row = w_mode == FVB_SCALE_ROW;
  }
  oa = Operand{A, sfA};
  ow = Operand{W, sfW};
  return FVB_OK;
}

}  // namespace gemm4
}  // namespace fvb

extern "C" {

int fvb_fp4_gemm(const void* A, const void* sfA, const float* rsA, int a_mode, const void* W,
                 const void* sfW, const float* rsW, int w_mode, int fmt, const void* bias,
                 const void* residual, int64_t ldr, const void* gate, int64_t M, int64_t N,
                 int64_t K, void* out, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(M >= 0 && N >= 0 && K >= 0, "fvb_fp4_gemm: negative size");
  FVB_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && K < (1ll << 31) - 256,
              "fvb_fp4_gemm: size");
  FVB_REQUIRE(fmt == FVB_FP4_NV || fmt == FVB_FP4_MX, "fvb_fp4_gemm: format %d", fmt);
  FVB_REQUIRE(a_mode == FVB_SCALE_TENSOR || a_mode == FVB_SCALE_ROW, "fvb_fp4_gemm: a_mode");
  FVB_REQUIRE(w_mode == FVB_SCALE_TENSOR || w_mode == FVB_SCALE_ROW, "fvb_fp4_gemm: w_mode");
  FVB_REQUIRE(residual || !gate, "fvb_fp4_gemm: gate without a residual");
  if (M == 0 || N == 0) return FVB_OK;
  gemm4::Args a;
  gemm4::Operand oa, ow;
  int rc = gemm4::operands("fvb_fp4_gemm", A, sfA, rsA, a_mode, W, sfW, rsW, w_mode, fmt, M, N, K,
                           a, oa, ow);
  if (rc) return rc;
  FVB_REQUIRE(out != nullptr, "fvb_fp4_gemm: NULL pointer");
  if (ldr == 0) ldr = N;
  FVB_REQUIRE(!residual || ldr >= N || M == 1, "fvb_fp4_gemm: residual row pitch");
  a.bias = (const __nv_bfloat16*)bias;
  a.res = (const __nv_bfloat16*)residual;
  a.gate = (const __nv_bfloat16*)gate;
  a.ldr = ldr;
  a.out = (__nv_bfloat16*)out;
  a.ldo = N;
  a.tma_out = aligned16(out) && N % 8 == 0;
  a.tma_res = residual && aligned16(residual) && ldr % 8 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (residual) return gemm4::dispatch_fmt<gemm4::kResidual>(fmt, a, oa, ow, st);
  return gemm4::dispatch_fmt<gemm4::kPlain>(fmt, a, oa, ow, st);
}

size_t fvb_fp4_ffn_workspace_bytes(int64_t M, int64_t F) {
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  return up(fvb_fp4_codes_bytes(M, F)) + up(fvb_fp4_scales_bytes(M, F, FVB_FP4_MX));
}

int fvb_fp4_ffn(const void* A, const void* sfA, const float* rsA, int a_mode, const void* W0,
                const void* sfW0, const float* rsW0, int w_mode, int fmt, const void* b0,
                const void* W2, const void* sfW2, const void* b2, const void* residual, int64_t ldr,
                const void* gate, int64_t M, int64_t D, int64_t F, int64_t N, void* out,
                void* workspace, fvb_stream_t stream) {
  using namespace fvb;
  FVB_REQUIRE(M >= 0 && D > 0 && F > 0 && N >= 0, "fvb_fp4_ffn: shape");
  FVB_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && D < (1ll << 31) - 256 &&
                  F < (1ll << 31) - 256,
              "fvb_fp4_ffn: size");
  FVB_REQUIRE(fmt == FVB_FP4_NV || fmt == FVB_FP4_MX, "fvb_fp4_ffn: format %d", fmt);
  FVB_REQUIRE(a_mode == FVB_SCALE_TENSOR || a_mode == FVB_SCALE_ROW, "fvb_fp4_ffn: a_mode");
  FVB_REQUIRE(w_mode == FVB_SCALE_TENSOR || w_mode == FVB_SCALE_ROW, "fvb_fp4_ffn: w_mode");
  if (M == 0 || N == 0) return FVB_OK;
  FVB_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
              "fvb_fp4_ffn: workspace must be 256-byte aligned");
  // what the second product would refuse, before the first is launched
  FVB_REQUIRE(W2 && sfW2 && out, "fvb_fp4_ffn: NULL pointer");
  FVB_REQUIRE(aligned16(W2) && aligned16(sfW2), "fvb_fp4_ffn: codes and scales must be 16-byte aligned");
  FVB_REQUIRE(residual || !gate, "fvb_fp4_ffn: gate without a residual");
  FVB_REQUIRE(!residual || ldr == 0 || ldr >= N || M == 1, "fvb_fp4_ffn: residual row pitch");
  gemm4::Args a;
  gemm4::Operand oa, ow;
  int rc = gemm4::operands("fvb_fp4_ffn", A, sfA, rsA, a_mode, W0, sfW0, rsW0, w_mode, fmt, M, F,
                           D, a, oa, ow);
  if (rc) return rc;
  uint8_t* hc = static_cast<uint8_t*>(workspace);
  uint8_t* hs = hc + ((fvb_fp4_codes_bytes(M, F) + 255) & ~(size_t)255);
  a.bias = (const __nv_bfloat16*)b0;
  a.hcodes = hc;
  a.hscales = hs;
  a.hpitch = fp4::code_pitch(F);
  a.htiles = fp4::scale_tiles(F, FVB_FP4_MX);
  rc = gemm4::dispatch_fmt<gemm4::kGeluMx>(fmt, a, oa, ow, (cudaStream_t)stream);
  if (rc) return rc;
  return fvb_fp4_gemm(hc, hs, nullptr, FVB_SCALE_TENSOR, W2, sfW2, nullptr, FVB_SCALE_TENSOR,
                      FVB_FP4_MX, b2, residual, ldr, gate, M, N, F, out, stream);
}

}  // extern "C"
