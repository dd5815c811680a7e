// Product of two microscaled 4-bit matrices on the 5th-generation tensor cores, with the
// epilogues of a DiT block's linears (fp4.cuh has the formats and the layout).
//
//   acc[m, n] = sum_k A[m, k] W[n, k]      codes times block scales, fp32, in the tensor core
//   y = acc * sa[m] * sw[n] + bias[n]      sa, sw: the nv formats' row scales (mx: 1)
//   out = bf16(y)  or  bf16(res + gate[n] * y)  or  mx codes of GELU(tanh)(y)
//
// One persistent CTA per SM, or one CTA pair per two SMs, warp-specialised:
//   warp 0      TMA producer: 256-element (128-byte) K blocks of A and W and their scale tiles
//               into a ring of shared-memory stages
//   warp 1      MMA issuer: copies a group of scale tiles into TMEM (tcgen05.cp), then issues
//               the group's block-scaled MMAs (K = 64 each) into the fp32 accumulator
//   warps 2..   epilogue (8 warps, 16 with GELU): the warps of a TMEM lane quarter take the
//               tile's 64-column chunks in turn, each thread one row; bf16 through a swizzled
//               staging buffer and a TMA store.  A chunk is two mx blocks of a row, so the
//               4-bit output needs no exchange between threads and the hidden state of an FFN
//               never exists in 16 bits.
//
// TMEM (512 columns): two accumulators of BN columns and two buffers of scale columns.  With
// BN = 256 that is more than 512, so the second accumulator starts at column 192: the tiles'
// accumulators share 64 columns, the epilogue reads those first, and the next tile's MMAs start
// when they have been read instead of when the whole tile has.
//
// The scale columns of a group are overwritten two groups later, after a wait for the MMAs that
// read them: the issue order orders a copy before the MMAs after it, but nothing orders an MMA
// before a copy after it.
#include "fp4.cuh"

namespace fvb {
namespace gemm4 {

constexpr int BM = 128;
constexpr int kRowBytes = 128;  // one K block of a row: 256 elements
constexpr int kStageOut = 32 * 128;  // an epilogue warp's staging: 32 rows x 64 bf16

enum { kPlain = 0, kResidual = 1, kGeluMx = 2 };

// epilogue warps, a multiple of 4
__host__ __device__ constexpr int epi_warps(int epi) { return epi == kGeluMx ? 16 : 8; }

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
  int vec_res;      // whether res may be read 16 bytes at a time
  uint8_t* hcodes;  // kGeluMx
  uint8_t* hscales;
  int64_t hpitch, htiles;
};

template <int FMT, int BN, int EPI, bool PAIR>
struct Shape {
  static constexpr int kEpiWarps = epi_warps(EPI);
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kOutBytes = EPI == kGeluMx ? 0 : kEpiWarps * kStageOut;
  static constexpr int kColBytes = 3 * BN * 4;  // the tile's column scales, biases and gates
  static constexpr int kTilesK = FMT == FVB_FP4_NV ? 4 : 2;  // scale tiles per K block
  static constexpr int kGroups = kTilesK / 2;                // TMEM groups of two scale tiles
  static constexpr int kMmas = 4 / kGroups;                  // MMAs (K = 64) per group
  static constexpr int kRowsB = PAIR ? BN / 2 : BN;          // W rows this CTA stages
  static constexpr int kSfTilesB = BN > 128 ? BN / 128 : 1;  // 128-row tiles of W's scales
  static constexpr int kBytesA = BM * kRowBytes;
  static constexpr int kBytesB = kRowsB * kRowBytes;
  static constexpr int kBytesSfA = kGroups * 1024;
  static constexpr int kBytesSfB = kGroups * kSfTilesB * 1024;
  static constexpr int kBytes = kBytesA + kBytesB + kBytesSfA + kBytesSfB;
  static constexpr int kFixed = kOutBytes + kColBytes + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int kFit = (227 * 1024 - kFixed) / kBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr size_t kSmem = (size_t)kStages * kBytes + kFixed;
  // TMEM columns
  static constexpr int kAcc1 = BN == 256 ? 192 : BN;  // start of the second accumulator
  static constexpr bool kOverlap = BN == 256;
  static constexpr int kSf = kAcc1 + BN;                    // start of the scale columns
  static constexpr int kSfCols = 8 + 8 * kSfTilesB;         // one group's
  static_assert(kSf + 2 * kSfCols <= 512, "TMEM columns");
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

// instruction descriptor: E2M1 operands, scale type, M x N; the scale ids (byte of the 4-byte
// scale column an mx MMA starts at) are added per MMA
template <int FMT>
__host__ __device__ constexpr uint32_t idesc4(int M, int N) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
         ((FMT == FVB_FP4_MX ? 1u : 0u) << 23) | ((uint32_t)(M >> 4) << 24);
}

// GELU(tanh) of two values in fp32: x * sigmoid(2 u) = x / (1 + 2^v), u = sqrt(2/pi) (x + c x^3),
// v = -2 u log2(e).  One reciprocal of the product serves both: 1 / a = b / (a b).  v is held
// at 60 so the product stays finite; x / 2^60 is then already far below any step of the codes
// next to it, and 0.5 x (1 + tanh u) in fp32 has long been 0.
__device__ __forceinline__ void gelu2(float& x0, float& x1) {
  const float k1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, k3 = k1 * 0.044715f;
  const uint64_t x = f2_pack(x0, x1);
  const uint64_t v = f2_mul(x, f2_fma(f2_mul(x, x), f2_pack(k3, k3), f2_pack(k1, k1)));
  float v0, v1;
  f2_unpack(v, v0, v1);
  const float a = 1.0f + ex2_approx(fminf(v0, 60.0f)), b = 1.0f + ex2_approx(fminf(v1, 60.0f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  f2_unpack(f2_mul(f2_mul(x, f2_pack(r, r)), f2_pack(b, a)), x0, x1);
}
__device__ __forceinline__ float max_nan(float a, float b) {  // keeps a NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void load_cols8(const __nv_bfloat16* p, int c, int N, bool vec, float* v) {
  if (vec && c + 8 <= N) {
    bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(p + c)), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < N ? __bfloat162float(p[c + i]) : 0.f;
  }
}
template <int FMT, int BN, int EPI, bool PAIR>
__global__ void __launch_bounds__(64 + 32 * epi_warps(EPI), 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSfA,
                    const __grid_constant__ CUtensorMap tmSfB,
                    const __grid_constant__ CUtensorMap tmOut, const Args args) {
  using S = Shape<FMT, BN, EPI, PAIR>;
  constexpr int STAGES = S::kStages;
  constexpr int TM = PAIR ? 2 * BM : BM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = sA + STAGES * S::kBytesA;
  uint8_t* sSfA = sB + STAGES * S::kBytesB;
  uint8_t* sSfB = sSfA + STAGES * S::kBytesSfA;
  uint8_t* sOut = sSfB + STAGES * S::kBytesSfB;
  float* sCol = reinterpret_cast<float*>(sOut + S::kOutBytes);  // [3][BN]
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + S::kOutBytes + S::kColBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;   // [2] accumulator finished
  uint64_t* tempty = tfull + 2;       // [2] accumulator (its shared columns) read
  uint64_t* sfree = tempty + 2;       // [2] the MMAs of a scale buffer finished
  uint64_t* drain = sfree + 2;        // every MMA this CTA issued finished
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  uint32_t* pair_ok = tmem_slot + 1;

  const int warp = warp_id_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
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
      mbar_init(&tempty[b], PAIR ? 2 * S::kEpiWarps : S::kEpiWarps);
      mbar_init(&sfree[b], 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSfA);
    prefetch_tmap(&tmSfB);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (PAIR) {
    cluster_sync_all();
    if (threadIdx.x == 0)
      *pair_ok = ld_shared_cluster_u32(mapa_shared(smem_u32(tmem_slot), rank ^ 1u)) == *tmem_slot;
    __syncthreads();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // a pair whose TMEM addresses differ (never expected) does no work and reports it
  const bool run = !PAIR || *pair_ok != 0u;
  if (!run && threadIdx.x == 0 && rank == 0) atomicCAS(&g_device_error, 0u, 0x40Cu);
  const uint32_t full0_c = PAIR ? mapa_shared(smem_u32(full), 0u) : 0u;
  const uint32_t tempty0_c = PAIR ? mapa_shared(smem_u32(tempty), 0u) : 0u;

  if (!run) {
    // straight to the teardown
  } else if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int64_t issued = 0;
      for (int tile = unit; tile < num_tiles && ok; tile += units) {
        const int m0 = (tile / n_tiles) * TM + (int)rank * BM;
        const int nt = (tile % n_tiles) * BN;
        const int n0 = nt + (int)rank * (PAIR ? S::kRowsB : 0);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, 0x401u)) {
            ok = false;
            break;
          }
          uint8_t* a = sA + stage * S::kBytesA;
          uint8_t* b = sB + stage * S::kBytesB;
          uint8_t* fa = sSfA + stage * S::kBytesSfA;
          uint8_t* fb = sSfB + stage * S::kBytesSfB;
          if (PAIR) {
            const uint32_t bar = full0_c + 8u * stage;
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], (uint32_t)(2 * S::kBytes));
            tma_load_2d_pair(a, &tmA, bar, kb * kRowBytes, m0);
            tma_load_2d_pair(b, &tmB, bar, kb * kRowBytes, n0);
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
              // two scale tiles = 256 words; past the last tile of a row TMA fills zeros
              const int x = (kb * S::kTilesK + 2 * g) * 128;
              tma_load_2d_pair(fa + g * 1024, &tmSfA, bar, x, m0 >> 7);
              tma_load_2d_pair(fb + g * S::kSfTilesB * 1024, &tmSfB, bar, x, nt >> 7);
            }
          } else {
            mbar_arrive_expect_tx(&full[stage], (uint32_t)S::kBytes);
            tma_load_2d(a, &tmA, &full[stage], kb * kRowBytes, m0);
            tma_load_2d(b, &tmB, &full[stage], kb * kRowBytes, n0);
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
              const int x = (kb * S::kTilesK + 2 * g) * 128;
              tma_load_2d(fa + g * 1024, &tmSfA, &full[stage], x, m0 >> 7);
              tma_load_2d(fb + g * S::kSfTilesB * 1024, &tmSfB, &full[stage], x, nt >> 7);
            }
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // no load may still be writing shared memory when its CTA exits: the last STAGES loads
      // are the newest phase of their stages' full barriers (a pair's are the even CTA's)
      if (!PAIR || rank == 0)
        for (int64_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
          mbar_wait(&full[i % STAGES], (uint32_t)((i / STAGES) & 1), 0x40Au);
    }
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
      uint32_t grp = 0;  // scale groups issued
      bool ok = true, any = false;
      for (int tile = unit; tile < num_tiles && ok; tile += units, ++t) {
        const int buf = t & 1;
        // shared columns: wait until the previous tile's were read; else until this
        // accumulator's last tile was
        const bool clear =
            S::kOverlap
                ? (t == 0 || mbar_wait(&tempty[buf ^ 1], (uint32_t)((t - 1) >> 1) & 1u, 0x402u))
                : mbar_wait(&tempty[buf], ((uint32_t)(t >> 1) & 1u) ^ 1u, 0x402u);
        if (!__all_sync(0xffffffffu, clear)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf ? S::kAcc1 : 0);
        const int nt = (tile % n_tiles) * BN;
        const uint32_t shift = BN < 128 ? (uint32_t)((nt & 127) >> 5) : 0u;
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
#pragma unroll
          for (int g = 0; g < S::kGroups; ++g) {
            if (g * S::kMmas < left) {
              const uint32_t sb = grp & 1u;
              if (!__all_sync(0xffffffffu, mbar_wait(&sfree[sb], ((grp >> 1) & 1u) ^ 1u, 0x405u))) {
                ok = false;
                break;
              }
              const uint32_t sfa = tmem + (uint32_t)S::kSf + sb * (uint32_t)S::kSfCols;
              const uint32_t sfb = sfa + 8u;
              if (leader) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  cp_scales<PAIR>(sfa + 4u * i, fa + (g * 1024 + i * 512) / 16);
#pragma unroll
                  for (int r = 0; r < S::kSfTilesB; ++r)
                    cp_scales<PAIR>(sfb + (uint32_t)(4 * S::kSfTilesB * i + 4 * r),
                                    fb + ((g * S::kSfTilesB + r) * 1024 + i * 512) / 16);
                }
#pragma unroll
                for (int i = 0; i < S::kMmas; ++i) {
                  const int ks = g * S::kMmas + i;  // K step inside the block
                  if (ks < left) {
                    const int ti = FMT == FVB_FP4_NV ? i : i >> 1;            // scale tile
                    const uint32_t id = FMT == FVB_FP4_NV ? 0u : (i & 1) * 2u;  // byte in its column
                    mma_fp4<FMT, PAIR>(d, da + 2 * ks, db + 2 * ks, idesc | (id << 4) | (id << 29),
                                       sfa + 4u * ti, sfb + (uint32_t)(4 * S::kSfTilesB * ti) + shift,
                                       (kb | ks) != 0 ? 1u : 0u);
                  }
                }
                if (PAIR) tc_commit_pair(&sfree[sb]);
                else tc_commit(&sfree[sb]);
              }
              ++grp;
              any = true;
            }
          }
          if (!ok) break;
          if (leader) {
            if (PAIR) tc_commit_pair_both(&empty[stage], 0x3);
            else tc_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && leader) {
          if (PAIR) tc_commit_pair_both(&tfull[buf], 0x3);
          else tc_commit(&tfull[buf]);
        }
        __syncwarp();
      }
      // every MMA issued above completes before TMEM is freed
      if (any) {
        if (leader) {
          if (PAIR) tc_commit_pair(drain);
          else tc_commit(drain);
        }
        __syncwarp();
        mbar_wait(drain, 0, 0x40Bu);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // G warps per TMEM lane quarter (warp % 4) take the tile's 64-column chunks in turn, each
    // thread one row of a chunk
    constexpr int G = S::kEpiWarps / 4;
    constexpr int kChunks = BN / 64;
    const int q = warp & 3;
    const int sub = (warp - 2) >> 2;
    const int et = (int)threadIdx.x - 64;
    uint8_t* stg = sOut + (size_t)(warp - 2) * kStageOut;
    auto release = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_remote(tempty0_c + 8u * b);
        else mbar_arrive(&tempty[b]);
      }
    };
    // the tile's column vectors go through shared memory: read from global one tile ahead,
    // so that no thread waits for them between the accumulator and the store
    float cs = 1.f, cb = 0.f, cg = 1.f;
    auto columns = [&](int tile) {
      const int c = (tile % n_tiles) * BN + et;
      if (tile < num_tiles && et < BN && c < args.N) {
        if (args.sw) cs = __ldg(args.sw + (args.sw_row ? c : 0));
        if (args.bias) cb = __bfloat162float(args.bias[c]);
        if (EPI == kResidual && args.gate) cg = __bfloat162float(args.gate[c]);
      }
    };
    columns(unit);
    bool ok = true;
    int t = 0;
    for (int tile = unit; tile < num_tiles; tile += units, ++t) {
      const int buf = t & 1;
      const int m0 = (tile / n_tiles) * TM + (int)rank * BM;
      const int n0 = (tile % n_tiles) * BN;
      const int row = m0 + q * 32 + lane;
      const bool row_ok = row < args.M;
      float sa = 1.0f;
      if (args.sa) sa = args.sa_row ? (row_ok ? __ldg(args.sa + row) : 0.f) : __ldg(args.sa);
      asm volatile("bar.sync 1, %0;" ::"r"(S::kEpiWarps * 32) : "memory");  // last tile's readers
      if (et < BN) {
        sCol[et] = cs;
        sCol[BN + et] = cb;
        if (EPI == kResidual) sCol[2 * BN + et] = cg;
      }
      asm volatile("bar.sync 1, %0;" ::"r"(S::kEpiWarps * 32) : "memory");
      columns(tile + units);
      // a warp whose wait ran out goes on to the barriers above, which its neighbours may be at,
      // and does nothing else
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&tfull[buf], (uint32_t)(t >> 1) & 1u, 0x404u));
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf ? S::kAcc1 : 0);
      const uint64_t sa2 = f2_pack(sa, sa);
      // chunk order: the columns shared with the other accumulator first (the first
      // accumulator's last chunk, the second's first)
      const int first = S::kOverlap && buf == 0 ? kChunks - 1 : 0;
      if (sub >= kChunks || (S::kOverlap && sub != 0)) release(buf);  // reads no shared column
#pragma unroll 1
      for (int i = sub; i < kChunks; i += G) {
        const int c = (i + first) & (kChunks - 1);
        const int col0 = n0 + c * 64;
        uint32_t r[64];
        tmem_ld_32x32b_x32(acc + (uint32_t)(c * 64), r);
        tmem_ld_32x32b_x32(acc + (uint32_t)(c * 64 + 32), r + 32);
        tmem_ld_wait();
        if (S::kOverlap ? i == 0 : i + G >= kChunks) release(buf);
        float* v = reinterpret_cast<float*>(r);
        if (col0 < args.N) {  // warp-uniform
          const float4* s4 = reinterpret_cast<const float4*>(sCol + c * 64);
          const float4* b4 = reinterpret_cast<const float4*>(sCol + BN + c * 64);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float4 s = s4[j], b = b4[j];
            f2_unpack(f2_fma(f2_pack(v[4 * j], v[4 * j + 1]), f2_mul(sa2, f2_pack(s.x, s.y)),
                             f2_pack(b.x, b.y)),
                      v[4 * j], v[4 * j + 1]);
            f2_unpack(f2_fma(f2_pack(v[4 * j + 2], v[4 * j + 3]), f2_mul(sa2, f2_pack(s.z, s.w)),
                             f2_pack(b.z, b.w)),
                      v[4 * j + 2], v[4 * j + 3]);
          }
        }
        if (EPI == kGeluMx) {
          // two mx blocks of this row
          uint32_t byte[2] = {0u, 0u};
          uint4 code[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            code[h] = make_uint4(0u, 0u, 0u, 0u);
            const int cb0 = col0 + h * 32;
            if (cb0 >= args.N) continue;  // past the last block: a zero scale
            float* x = v + h * 32;
            float am = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              gelu2(x[j], x[j + 1]);
              if (cb0 + 32 > args.N) {  // columns past N carry whatever scales lie past W's rows
                if (cb0 + j >= args.N) x[j] = 0.f;
                if (cb0 + j + 1 >= args.N) x[j + 1] = 0.f;
              }
              am = max_nan(max_nan(am, fabsf(x[j])), fabsf(x[j + 1]));
            }
            if (am < INFINITY) {
              const int e = fp4::mx_exponent(am);
              byte[h] = (uint32_t)(e + 127);
              const uint2 lo = fp4::mx_codes16(x, e), hi = fp4::mx_codes16(x + 16, e);
              code[h] = make_uint4(lo.x, lo.y, hi.x, hi.y);
            } else {
              byte[h] = 0xFFu;
            }
          }
          if (row_ok && (col0 >> 5) < args.htiles * 4) {
            uint8_t* hp = args.hcodes + (int64_t)row * args.hpitch + (col0 >> 1);
            if (col0 < args.N) *reinterpret_cast<uint4*>(hp) = code[0];
            if (col0 + 32 < args.N) *reinterpret_cast<uint4*>(hp + 16) = code[1];
            *reinterpret_cast<uint16_t*>(args.hscales + fp4::scale_at(row, col0 >> 5, args.htiles)) =
                (uint16_t)(byte[0] | (byte[1] << 8));
          }
          continue;
        }
        if (col0 >= args.N) continue;
        if (EPI == kResidual) {
          const __nv_bfloat16* rp = args.res + (int64_t)row * args.ldr;
          const float4* g4 = reinterpret_cast<const float4*>(sCol + 2 * BN + c * 64);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float x[8];
            load_cols8(rp, row_ok ? col0 + g * 8 : args.N, args.N, args.vec_res, x);
            const float4 ga = g4[2 * g], gb = g4[2 * g + 1];
            float* y = v + g * 8;
            y[0] = __fmaf_rn(ga.x, y[0], x[0]);
            y[1] = __fmaf_rn(ga.y, y[1], x[1]);
            y[2] = __fmaf_rn(ga.z, y[2], x[2]);
            y[3] = __fmaf_rn(ga.w, y[3], x[3]);
            y[4] = __fmaf_rn(gb.x, y[4], x[4]);
            y[5] = __fmaf_rn(gb.y, y[5], x[5]);
            y[6] = __fmaf_rn(gb.z, y[6], x[6]);
            y[7] = __fmaf_rn(gb.w, y[7], x[7]);
          }
        }
        if (args.tma_out) {
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
          // 128-byte swizzle: 16-byte chunk g of row l lands at chunk g ^ (l % 8)
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((g ^ (lane & 7)) << 4)) =
                f32_to_bf16x8(v + g * 8);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, stg, col0, m0 + q * 32);
            tma_store_commit();
          }
        } else if (row_ok) {
          __nv_bfloat16* op = args.out + (int64_t)row * args.ldo;
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (col0 + j < args.N) op[col0 + j] = __float2bfloat16_rn(v[j]);
        }
      }
    }
    if (lane == 0) tma_store_wait0();
  }
  tc_fence_before();
  if (PAIR)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR)
      tmem_dealloc_pair(tmem, 512);
    else
      tmem_dealloc(tmem, 512);
  }
}

struct Operand {
  const void* codes;
  const void* scales;
  const float* rs;
  int rs_row;
};

template <int FMT, int BN, int EPI, bool PAIR>
static int launch(const Args& a, const Operand& A, const Operand& W, cudaStream_t st) {
  using S = Shape<FMT, BN, EPI, PAIR>;
  const int64_t pitch = fp4::code_pitch(a.K);
  const int64_t tiles = fp4::scale_tiles(a.K, FMT);
  CUtensorMap tmA, tmB, tmSfA, tmSfB, tmO;
  int rc = make_tmap_2d(&tmA, A.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)pitch,
                        (uint64_t)a.M, (uint64_t)pitch, kRowBytes, BM, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_tmap_2d(&tmB, W.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)pitch, (uint64_t)a.N,
                    (uint64_t)pitch, kRowBytes, S::kRowsB, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  // scales as 32-bit words: a row of the map is one 128-row band, two tiles are 256 words
  rc = make_tmap_2d(&tmSfA, A.scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, (uint64_t)tiles * 128,
                    (uint64_t)((a.M + 127) / 128), (uint64_t)tiles * 512, 256, 1,
                    CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  rc = make_tmap_2d(&tmSfB, W.scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, (uint64_t)tiles * 128,
                    (uint64_t)((a.N + 127) / 128), (uint64_t)tiles * 512, 256, S::kSfTilesB,
                    CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  tmO = tmA;  // unused unless tma_out
  if (a.tma_out) {
    rc = make_tmap_2d(&tmO, a.out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)a.N,
                      (uint64_t)a.M, (uint64_t)a.ldo * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  auto kern = fp4_gemm_kernel<FMT, BN, EPI, PAIR>;
  constexpr size_t smem = S::kSmem;
  static_assert(smem <= 227 * 1024, "fp4 gemm: shared memory");
  static bool configured[64] = {false};
  static int pair_slots[64] = {0};
  int dev = 0;
  FVB_CUDA_TRY(cudaGetDevice(&dev), "fp4 gemm device");
  FVB_REQUIRE(dev >= 0 && dev < 64, "fp4 gemm: device ordinal %d", dev);
  constexpr int TM = PAIR ? 2 * BM : BM;
  const int64_t n_tiles64 = (int64_t)((a.M + TM - 1) / TM) * ((a.N + BN - 1) / BN);
  FVB_REQUIRE(n_tiles64 < (1ll << 31) - 4096, "fp4 gemm: too many output tiles");
  const int num = (int)n_tiles64;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  if (PAIR) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  if (!configured[dev]) {
    FVB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                 "fp4 gemm smem attribute");
    if (PAIR) {
      int clusters = 0;
      cfg.gridDim = dim3(2 * (sm_count() / 2));
      FVB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg),
                   "fp4 gemm cluster occupancy");
      FVB_REQUIRE(clusters > 0, "fp4 gemm: no 2-CTA cluster fits on this device");
      pair_slots[dev] = clusters;
    }
    configured[dev] = true;
  }
  int grid;
  if (PAIR)
    grid = 2 * (num < pair_slots[dev] ? num : pair_slots[dev]);
  else
    grid = num < sm_count() ? num : sm_count();
  cfg.gridDim = dim3(grid);
  FVB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmSfA, tmSfB, tmO, a), "fp4 gemm launch");
  return check_launch("fp4 gemm");
}

template <int FMT, int EPI>
static int dispatch(const Args& a, const Operand& A, const Operand& W, cudaStream_t st) {
  if (a.M > BM && a.N > 128) return launch<FMT, 256, EPI, true>(a, A, W, st);
  return launch<FMT, 128, EPI, false>(a, A, W, st);
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
  oa = Operand{A, sfA, rsA, g.sa_row};
  ow = Operand{W, sfW, rsW, g.sw_row};
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
  a.vec_res = residual && aligned16(residual) && ldr % 8 == 0;
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
