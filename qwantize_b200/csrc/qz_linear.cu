// qz_linear.cu -- y = x W^T with W in packed NVFP4 (block 16) or MXFP4 (block
// 32) and x quantized to the same format on the way in, on the block-scaled
// tcgen05 tensor cores.
//
//   y[t, n] = p_t * w * sum_b sx[t, b] * sw[n, b] * sum_{k in b} qx[t, k] * qw[n, k]  (+ bias[n])
//
// qx, sx: the naive E2M1 codes and block scales of row t (the same rounding as
// qz_quantize); for NVFP4 on the row divided by p_t, the smallest power of two
// with max|x_t| <= 448 * 6 * p_t, so that the E4M3 scales fit whatever the row's
// magnitude (MXFP4 scales reach any fp32 magnitude: p_t = 1).  The division
// is exact, so 16-bit inputs keep their 11 significant bits and the rounding
// shortcut of qz_common.cuh holds.  w is the weight's tensor scale.
//
// Two launches: quantize_rows_kernel (one CTA per row), then linear_kernel.
//
// linear_kernel, one persistent CTA per SM, 192 threads: warp 0 feeds a ring of
// stages (256 values of K: 128-byte swizzled rows of A and B by TMA, their
// scales by bulk copies), warp 1 copies the stage's scales to TMEM
// (tcgen05.cp) and issues four block-scaled MMAs of K = 64, warps 2-5 drain the
// accumulator.  The wide form (BN = 256) has 128 token rows as A and 256 rows
// of W as B.  The narrow forms (BN = 16 .. 128) swap the operands: 128 rows of
// W are A and BN tokens are B, so that a decode step multiplies few padded
// rows, and W streams through the ring once.  With few tiles K is cut into
// splits; the last CTA of a tile adds the splits' fp32 partials in split order
// (the order of arrival changes nothing).
//
// Scales in memory, for both operands: row tiles of 128 rows (x, narrow form:
// BN rows), groups of 4 blocks of K; a group is 512 bytes, row r at
// (r % 32) * 16 + (r / 32) * 4, one byte per block: what tcgen05.cp
// 32x128b.warpx4 spreads over the 128 TMEM lanes as 4 columns.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/qwantize_b200.h"
#include "qz_common.cuh"
#include "qz_kernels.h"
#include "qz_tc.cuh"

namespace qz {

int fail(int code, const char* fmt, ...);
int cuda_status(cudaError_t e, const char* what);
int current_sms(int* sms);

constexpr int kStepK = 256;      // values of K per pipeline stage: one 128-byte swizzled row of codes
constexpr int kGroupBytes = 512; // scales of 128 rows x 4 blocks

template <int BS>
struct Fmt {
  static constexpr int kBlocks = kStepK / BS;                       // scale blocks per row and stage
  static constexpr int kGroups = kBlocks / 4;                       // scale groups per stage: 4 (NVFP4), 2 (MXFP4)
  static constexpr int kSfBytes = kGroups * kGroupBytes;            // per 128 rows and stage
};

// ---------------------------------------------------------------------------
// activations to FP4
// ---------------------------------------------------------------------------
// One CTA per row, one thread per block of BS values.  Bound by HBM for many
// rows and by one DRAM round trip for few; the second read of the row (after
// its maximum is known) comes from L1 / L2.
template <int BS, int DT>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t K,
                                                            uint8_t* __restrict__ packed, int64_t ldp,
                                                            uint8_t* __restrict__ sf, int gran, int64_t n_steps,
                                                            float* __restrict__ row_scale, int* __restrict__ counters,
                                                            int n_counters) {
  __shared__ uint32_t s_max[16];
  const int64_t row = blockIdx.x;
  const char* base = static_cast<const char*>(x) + row * ldx * Elem<DT>::kSize;
  const int64_t nb = K / BS, nb_pad = n_steps * Fmt<BS>::kBlocks, nb_packed = ldp * 2 / BS;
  const int tid = threadIdx.x, nt = blockDim.x;
  if (row == 0)
    for (int i = tid; i < n_counters; i += nt) counters[i] = 0;
  float inv = 1.0f, p = 1.0f;
  if (BS == 16) {
    uint32_t m = 0;
    for (int64_t b = tid; b < nb; b += nt) {
      float v[BS];
      load_block<BS, DT>(base, b, v);
#pragma unroll
      for (int i = 0; i < BS; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < (nt >> 5); ++w) m = max(m, s_max[w]);
    // smallest e with max <= 1.3125 * 2^(11 + e); 0 for an all-zero row and for inf / NaN
    int e = 0;
    if (m != 0 && m < 0x7f800000u) {
      e = (int)(m >> 23) - 127 - 11 + ((m & 0x7fffffu) > 0x280000u ? 1 : 0);
      e = max(e, -120);
    }
    inv = pow2f(-e);
    p = pow2f(e);
  }
  if (tid == 0) row_scale[row] = p;
  uint8_t* sf_row = sf + (row / gran) * n_steps * Fmt<BS>::kSfBytes + (row % gran % 32) * 16 + (row % gran / 32) * 4;
  for (int64_t b0 = 0; b0 < nb_pad; b0 += nt) {
    const int64_t b = b0 + tid;
    uint32_t code = 0;
    uint32_t words[BS / 8] = {};
    if (b < nb) {
      float v[BS];
      load_block<BS, DT>(base, b, v);
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < BS; ++i) {
        v[i] = __fmul_rn(v[i], inv);
        am = max(am, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      float s;
      if (BS == 16) {
        s = e4m3_snap_nonneg(__fdiv_rn(__uint_as_float(am), 6.0f));
        code = e4m3_code(s);
      } else {
        code = is_nan_bits(am) ? 255u : (uint32_t)ue8m0_naive_exp(am);
        s = code == 255u ? __uint_as_float(kMxNanBits) : pow2f((int)code - 127);
      }
      if (s > 0.0f) {  // a zero (or NaN) scale keeps codes 0
        if (DT != kDtF32) {
          const float c = __fmul_rn(__frcp_rn(s), kBiasDown);
#pragma unroll
          for (int i = 0; i < BS; i += 2) {
            const uint32_t lo = __float_as_uint(v[i]) >> 31, hi = __float_as_uint(v[i + 1]) >> 31;
            words[i / 8] |= (e2m1x2_rn(__fmul_rn(fabsf(v[i]), c), __fmul_rn(fabsf(v[i + 1]), c)) | lo << 3 | hi << 7)
                            << (4 * (i % 8));
          }
        } else {
#pragma unroll
          for (int i = 0; i < BS; ++i) {
            const float q = __fdiv_rn(fabsf(v[i]), s);
            uint32_t n = __float_as_uint(v[i]) >> 31 << 3;
#pragma unroll
            for (int k = 0; k < 7; ++k) n += q > bnd(k) ? 1u : 0u;
            words[i / 8] |= n << (4 * (i % 8));
          }
        }
      }
    }
    if (b < nb_packed) {
      if (BS == 16) *reinterpret_cast<uint2*>(packed + row * ldp + b * 8) = make_uint2(words[0], words[1]);
      else *reinterpret_cast<uint4*>(packed + row * ldp + b * 16) = make_uint4(words[0], words[1], words[BS / 16], words[BS / 8 - 1]);
    }
    // four neighbouring blocks share one scale word
    uint32_t w = code | __shfl_down_sync(0xffffffffu, code, 1) << 8;
    w |= __shfl_down_sync(0xffffffffu, w, 2) << 16;
    if ((tid & 3) == 0 && b < nb_pad) *reinterpret_cast<uint32_t*>(sf_row + (b >> 2) * kGroupBytes) = w;
  }
}

// Scale bytes (N, nb) of a weight -> the group layout (row tiles padded to
// n_tiles, K to whole stages; padding gets scale 0).  One thread per word.
__global__ void scale_layout_kernel(const uint8_t* __restrict__ codes, int64_t N, int64_t nb, int64_t n_groups,
                                    int64_t n_tiles, uint32_t* __restrict__ out) {
  const int64_t total = n_tiles * n_groups * 128;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t word = i % 128, group = i / 128 % n_groups, tile = i / (128 * n_groups);
    const int64_t row = tile * 128 + (word & 3) * 32 + (word >> 2);
    uint32_t w = 0;
    for (int k = 0; k < 4; ++k) {
      const int64_t b = group * 4 + k;
      if (row < N && b < nb) w |= (uint32_t)codes[row * nb + b] << (8 * k);
    }
    out[i] = w;
  }
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
struct LinearParams {
  int64_t T, N;                       // tokens, output features
  int64_t tiles_a, tiles_b;           // 128-row A tiles, BN-row B tiles
  int splits, n_steps;                // K splits, stages over the whole of K
  int64_t n_units;
  const uint8_t *sf_a, *sf_b;         // scales: tile-major, n_steps * kSfBytes each
  float* partial;                     // splits > 1: (tile, split, column, 128) fp32
  int* counters;                      // splits > 1: arrivals per tile, zeroed by the quantization launch
  const float* row_scale;             // p_t
  float w_scale;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t ldo;
  int vec;                            // 16-byte stores are aligned (wide form, 16-bit outputs)
};

template <int BN, int BS>
struct LinGeo {
  static constexpr bool kSwap = BN < 256;  // A = weight rows, B = tokens
  static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
  static constexpr int kBTiles = BN > 128 ? BN / 128 : 1;  // 128-row scale tiles of B
  static constexpr int kSf = Fmt<BS>::kSfBytes;
  static constexpr int kStageBytes = kABytes + kBBytes + kSf * (1 + kBTiles);
  static constexpr int kMaxStages = (232448 - 1024 - 512) / kStageBytes;
  static constexpr int kStages = kMaxStages > 10 ? 10 : kMaxStages;
  static constexpr int kSmem = kStages * kStageBytes + 1024 + 512;
  static constexpr int kAccs = BN > 128 ? 1 : 2;
  // TMEM: accumulators, then kSfBufs buffers of scales (kGroups * 4 columns per 128 rows)
  static constexpr int kSfCols = Fmt<BS>::kGroups * 4 * (1 + kBTiles);
  static constexpr int kSfBufs = BN > 128 ? 2 : 4;
  static constexpr int kAccCols = BN > 128 ? 256 : 2 * BN;
  static_assert(kAccCols + kSfBufs * kSfCols <= 512, "TMEM columns");
};

// Block-scaled MMA, E2M1 x E2M1 -> fp32, K = 64, scales of A and B in TMEM:
// one E4M3 scale per 16 values (NVFP4) or one power of two per 32 (MXFP4).
template <int BS>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accumulate) {
  if constexpr (BS == 16)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}

// Instruction descriptor of the block-scaled kinds: E2M1 operands, K-major;
// scale type E4M3 (0) or power of two (1); sf_id: the byte of the 32-bit TMEM
// scale word that the MMA starts from (MXFP4 takes two of the four).
template <int BS>
__host__ __device__ constexpr uint32_t idesc_fp4(int N, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((BS == 32 ? 1u : 0u) << 23) |
         ((uint32_t)(128 >> 4) << 24) | (sf_id << 29);
}

// 32 rows of 16 bytes (512 contiguous bytes) -> 4 TMEM columns, spread to all
// four 32-lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
  // no swizzle; 8-row groups 128 bytes apart
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 |
                        (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == kDtF32) return static_cast<const float*>(p)[i];
  const uint32_t h = static_cast<const uint16_t*>(p)[i];
  return dtype == kDtBF16 ? bf16_bits_to_float(h) : f16_bits_to_float(h);
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
  uint32_t r;
  if (dtype == kDtBF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == kDtF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)(pack16(v, 0.0f, dtype) & 0xffffu);
}

struct LinUnit {
  int64_t a, b, tile;
  int split, s0, s1;
};

// Units: the splits of one tile side by side; wide tiles in bands of 16 token
// tiles, so that the ~148 tiles in flight are about as many token rows as
// weight rows and share both through L2.
template <bool SWAP>
__device__ __forceinline__ LinUnit lin_unit(const LinearParams& p, int64_t t) {
  LinUnit u;
  u.split = (int)(t % p.splits);
  u.tile = t / p.splits;
  if (SWAP) {
    u.a = u.tile % p.tiles_a;
    u.b = u.tile / p.tiles_a;
  } else {
    const int64_t per = 16 * p.tiles_b, band = u.tile / per, r = u.tile % per;
    const int64_t left = p.tiles_a - band * 16, rows = left < 16 ? left : 16;
    u.b = r / rows;
    u.a = band * 16 + r % rows;
  }
  u.s0 = (int)((int64_t)u.split * p.n_steps / p.splits);
  u.s1 = (int)((int64_t)(u.split + 1) * p.n_steps / p.splits);
  return u;
}

template <int BN, int BS>
__global__ void __launch_bounds__(192, 1)
    linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, LinearParams p) {
  using G = LinGeo<BN, BS>;
  constexpr bool SWAP = G::kSwap;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // operands first (1024-byte swizzle atoms), then the scales of all stages, then barriers
  unsigned char* smem_sf = smem + G::kStages * (G::kABytes + G::kBBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::kStages * G::kStageBytes);
  uint64_t* empty = full + G::kStages;
  uint64_t* tfull = empty + G::kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  volatile int* last_s = abort_s + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, 128); }
    mbar_init(mma_done, 1);
    *abort_s = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_base_s, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_s;

  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned err) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
      if (*abort_s) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        atomicOr(&qz_device_error, err);
        *abort_s = 1;
        return false;
      }
    }
    return true;
  };

  if (warp == 0) {
    // ---------------- producer ----------------
    if (lane == 0) {
      uint32_t it = 0;
      for (int64_t t = blockIdx.x; t < p.n_units; t += gridDim.x) {
        const LinUnit u = lin_unit<SWAP>(p, t);
        for (int ks = u.s0; ks < u.s1; ++ks, ++it) {
          const int s = it % G::kStages;
          if (!wait(empty + s, ((it / G::kStages) & 1) ^ 1, kDevErrLoadTimeout)) goto producer_done;
          unsigned char* sa = smem + s * (G::kABytes + G::kBBytes);
          unsigned char* sf = smem_sf + s * G::kSf * (1 + G::kBTiles);
          mbar_arrive_expect_tx(full + s, G::kStageBytes);
          tma_load_2d(sa, &map_a, ks * 128, (int)(u.a * 128), full + s);
          tma_load_2d(sa + G::kABytes, &map_b, ks * 128, (int)(u.b * BN), full + s);
          bulk_load(sf, p.sf_a + (u.a * p.n_steps + ks) * G::kSf, G::kSf, full + s);
#pragma unroll
          for (int h = 0; h < G::kBTiles; ++h)
            bulk_load(sf + (1 + h) * G::kSf, p.sf_b + ((u.b * G::kBTiles + h) * p.n_steps + ks) * G::kSf, G::kSf, full + s);
        }
      }
    producer_done:
      // every load issued must have landed before the CTA can exit (bounded)
      for (uint32_t k = it > (uint32_t)G::kStages ? it - G::kStages : 0u; k < it; ++k)
        mbar_wait_bounded(full + (k % G::kStages), (k / G::kStages) & 1, kDevErrLoadTimeout);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      uint32_t it = 0, lt = 0;
      for (int64_t t = blockIdx.x; t < p.n_units; t += gridDim.x, ++lt) {
        const LinUnit u = lin_unit<SWAP>(p, t);
        const uint32_t acc = G::kAccs == 2 ? (lt & 1) : 0u;
        const uint32_t phase = G::kAccs == 2 ? ((lt >> 1) & 1) : (lt & 1);
        if (!wait(tempty + acc, phase ^ 1, kDevErrMmaTimeout)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        bool ok = true;
        for (int ks = u.s0; ks < u.s1; ++ks, ++it) {
          const int s = it % G::kStages;
          if (!wait(full + s, (it / G::kStages) & 1, kDevErrMmaTimeout)) { ok = false; break; }
          // this scale buffer was last read by the MMAs kSfBufs stages ago
          if (it >= (uint32_t)G::kSfBufs) {
            const uint32_t j = it - G::kSfBufs;
            if (!wait(empty + j % G::kStages, (j / G::kStages) & 1, kDevErrMmaTimeout)) { ok = false; break; }
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * (G::kABytes + G::kBBytes)), sb = sa + G::kABytes;
          const uint32_t sf = smem_u32(smem_sf + s * G::kSf * (1 + G::kBTiles));
          const uint32_t t_sfa = tmem_base + G::kAccCols + (it % G::kSfBufs) * G::kSfCols;
          const uint32_t t_sfb = t_sfa + Fmt<BS>::kGroups * 4;
#pragma unroll
          for (int q = 0; q < Fmt<BS>::kGroups; ++q) {
            tmem_cp_scales(t_sfa + 4 * q, sf + q * kGroupBytes);
#pragma unroll
            for (int h = 0; h < G::kBTiles; ++h)
              tmem_cp_scales(t_sfb + (q * G::kBTiles + h) * 4, sf + (1 + h) * G::kSf + q * kGroupBytes);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int q = BS == 16 ? kk : kk / 2;
            umma_fp4<BS>(d_tmem, smem_desc(sa + kk * 32, 16, 1024), smem_desc(sb + kk * 32, 16, 1024),
                         idesc_fp4<BS>(BN, BS == 16 ? 0u : (kk & 1) * 2u), t_sfa + 4 * q, t_sfb + 4 * q * G::kBTiles,
                         (ks > u.s0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(empty + s);
        }
        if (!ok) break;
        umma_commit(tfull + acc);
      }
      // the MMAs issued must retire before TMEM is freed (also after an abort)
      umma_commit(mma_done);
      mbar_wait_bounded(mma_done, 0u, kDevErrMmaTimeout);
    }
  } else {
    // ---------------- epilogue (warps 2-5) ----------------
    const int row = (warp & 3) * 32 + lane;  // accumulator row of this thread
    uint32_t lt = 0;
    for (int64_t t = blockIdx.x; t < p.n_units; t += gridDim.x, ++lt) {
      const LinUnit u = lin_unit<SWAP>(p, t);
      const uint32_t acc = G::kAccs == 2 ? (lt & 1) : 0u;
      const uint32_t phase = G::kAccs == 2 ? ((lt >> 1) & 1) : (lt & 1);
      uint32_t go = wait(tfull + acc, phase, kDevErrEpilogueTimeout) ? 1u : 0u;
      if (p.splits > 1)  // all epilogue threads go on or all stop: the barriers below count on it
        asm volatile(
            "{\n .reg .pred a, b;\n setp.ne.u32 a, %0, 0;\n barrier.cta.red.and.aligned.pred b, 1, 128, a;\n selp.u32 %0, 1, 0, b;\n}\n"
            : "+r"(go)::"memory");
      if (!go) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * BN;
      const int64_t ra = u.a * 128 + row;       // swapped: output feature; wide: token
      const int64_t cb = u.b * BN;              // swapped: first token; wide: first output feature
      const int64_t cols_left = (SWAP ? p.T : p.N) - cb;
      const int cols = cols_left < BN ? (int)cols_left : BN;
      // finish 16 columns: scale, bias, round once, store
      auto finish = [&](int c, const float(&v)[16]) {
        if (ra >= (SWAP ? p.N : p.T)) return;
        if constexpr (SWAP) {
          const float bias = p.bias ? load_any(p.bias, p.bias_dtype, ra) : 0.0f;
#pragma unroll
          for (int q = 0; q < 16; ++q)
            if (c + q < cols) {
              const int64_t tok = cb + c + q;
              store_any(p.out, p.out_dtype, tok * p.ldo + ra, __fmaf_rn(v[q], p.row_scale[tok] * p.w_scale, bias));
            }
        } else {
          const float sc = p.row_scale[ra] * p.w_scale;
          float o[16];
#pragma unroll
          for (int q = 0; q < 16; ++q)
            o[q] = __fmaf_rn(v[q], sc, p.bias && c + q < cols ? load_any(p.bias, p.bias_dtype, cb + c + q) : 0.0f);
          const int64_t at = ra * p.ldo + cb + c;
          if (p.vec && c + 16 <= cols) {
            uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
            d[0] = make_uint4(pack16(o[0], o[1], p.out_dtype), pack16(o[2], o[3], p.out_dtype),
                              pack16(o[4], o[5], p.out_dtype), pack16(o[6], o[7], p.out_dtype));
            d[1] = make_uint4(pack16(o[8], o[9], p.out_dtype), pack16(o[10], o[11], p.out_dtype),
                              pack16(o[12], o[13], p.out_dtype), pack16(o[14], o[15], p.out_dtype));
          } else {
#pragma unroll
            for (int q = 0; q < 16; ++q)
              if (c + q < cols) store_any(p.out, p.out_dtype, at + q, o[q]);
          }
        }
      };
      if (p.splits == 1) {
#pragma unroll 1
        for (int c = 0; c < cols; c += 16) {
          float v[16];
          tmem_ld16(taddr + c, v);
          finish(c, v);
        }
        tc_fence_before();
        mbar_arrive(tempty + acc);
        continue;
      }
      float* part = p.partial + (u.tile * p.splits + u.split) * (int64_t)(BN * 128) + row;
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        float v[16];
        tmem_ld16(taddr + c, v);
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (c + q < cols) part[(c + q) * 128] = v[q];
      }
      tc_fence_before();
      mbar_arrive(tempty + acc);
      __threadfence();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (threadIdx.x == 64) *last_s = atomicAdd(p.counters + u.tile, 1) == p.splits - 1;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool last = *last_s != 0;
      asm volatile("bar.sync 1, 128;" ::: "memory");  // last_s is read before the next unit writes it
      if (!last) continue;
      __threadfence();
      const float* all = p.partial + u.tile * p.splits * (int64_t)(BN * 128) + row;
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        float v[16] = {};
        for (int sp = 0; sp < p.splits; ++sp) {
#pragma unroll
          for (int q = 0; q < 16; ++q)
            if (c + q < cols) v[q] += __ldcg(all + sp * (int64_t)(BN * 128) + (c + q) * 128);
        }
        finish(c, v);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
cudaError_t read_device_error_linear(unsigned* out, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(out, qz_device_error, sizeof(unsigned));
  if (e != cudaSuccess || !clear) return e;
  unsigned zero = 0;
  return cudaMemcpyToSymbol(qz_device_error, &zero, sizeof(unsigned));
}

// Rows of packed codes: `inner` bytes each, `rows` rows `stride` bytes apart.
static int code_map(CUtensorMap* m, const void* base, uint64_t inner, uint64_t rows, uint64_t stride, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(QZ_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {inner, rows};
  cuuint64_t strides[1] = {stride};
  cuuint32_t box[2] = {128, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QZ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return QZ_OK;
}

// Tile form and K splits of one call, and its workspace.
struct LinPlan {
  int bn, splits, n_steps;
  int64_t tiles_a, tiles_b, ldp;
  int64_t off_sf, off_scale, off_counter, off_partial, bytes;
};

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

static LinPlan plan_linear(int64_t T, int64_t K, int64_t N, int bs, int sms) {
  LinPlan best{};
  double best_cost = -1.0;
  const int n_steps = (int)((K + kStepK - 1) / kStepK);
  for (int bn : {16, 32, 64, 128, 256}) {
    if (bn < 128 && T > 4 * bn) continue;
    const bool swap = bn < 256;
    const int64_t ta = swap ? (N + 127) / 128 : (T + 127) / 128;
    const int64_t tb = swap ? (T + bn - 1) / bn : (N + 255) / 256;
    const double stage = 128.0 * 128 + 128.0 * bn + 128.0 * 256 / bs * (1 + (bn > 128 ? 2 : 1));
    for (int sp = 1; sp <= n_steps && sp <= 32; ++sp) {
      const int64_t units = ta * tb * sp;
      if (sp > 1 && units > 4 * sms) break;
      const double waves = (double)((units + sms - 1) / sms);
      // clocks: a stage's bytes at about 40 per clock and SM, or its MMAs; a unit's fill and epilogue
      const double step = stage / 40.0 > 2.0 * bn ? stage / 40.0 : 2.0 * bn;
      const double cost = waves * ((n_steps + sp - 1) / sp * step + 1200.0 + 6.0 * bn) + (sp > 1 ? 1500.0 + 4.0 * sp * (T < bn ? T : bn) : 0.0);
      if (best_cost < 0 || cost < best_cost) {
        best_cost = cost;
        best.bn = bn; best.splits = sp; best.tiles_a = ta; best.tiles_b = tb;
      }
    }
  }
  best.n_steps = n_steps;
  best.ldp = up(K, 32) / 2;
  const int gran = best.bn < 128 ? best.bn : 128;
  const int64_t sf_tiles = (T + gran - 1) / gran;
  best.off_sf = up(T * best.ldp, 256);
  best.off_scale = best.off_sf + up(sf_tiles * n_steps * (int64_t)(kStepK / bs / 4 * kGroupBytes), 256);
  best.off_counter = best.off_scale + up(T * 4, 256);
  const int64_t tiles = best.tiles_a * best.tiles_b;
  best.off_partial = best.off_counter + (best.splits > 1 ? up(tiles * 4, 256) : 0);
  best.bytes = best.off_partial + (best.splits > 1 ? tiles * best.splits * best.bn * 128 * 4 : 0);
  return best;
}

template <int BS>
static cudaError_t launch_quantize_rows(const void* x, int dt, int64_t ldx, int64_t T, int64_t K, uint8_t* packed,
                                        int64_t ldp, uint8_t* sf, int gran, int64_t n_steps, float* row_scale,
                                        int* counters, int n_counters, cudaStream_t st) {
  const int64_t nb = n_steps * Fmt<BS>::kBlocks;
  const int nt = nb >= 512 ? 512 : (nb < 64 ? 64 : (int)up(nb, 32));
  const unsigned grid = (unsigned)T;
  if (dt == kDtBF16)
    quantize_rows_kernel<BS, kDtBF16><<<grid, nt, 0, st>>>(x, ldx, K, packed, ldp, sf, gran, n_steps, row_scale, counters, n_counters);
  else if (dt == kDtF16)
    quantize_rows_kernel<BS, kDtF16><<<grid, nt, 0, st>>>(x, ldx, K, packed, ldp, sf, gran, n_steps, row_scale, counters, n_counters);
  else
    quantize_rows_kernel<BS, kDtF32><<<grid, nt, 0, st>>>(x, ldx, K, packed, ldp, sf, gran, n_steps, row_scale, counters, n_counters);
  return cudaGetLastError();
}

template <int BN, int BS>
static int launch_linear(const CUtensorMap& a, const CUtensorMap& b, const LinearParams& p, int sms, cudaStream_t st) {
  using G = LinGeo<BN, BS>;
  static bool attr_set[64] = {false};  // per device (a benign race: every thread sets the same value)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_kernel<BN, BS>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t grid = p.n_units < sms ? p.n_units : sms;
  linear_kernel<BN, BS><<<(unsigned)grid, 192, G::kSmem, st>>>(a, b, p);
  return cuda_status(cudaGetLastError(), "linear launch");
}

template <int BS>
static int run_linear(int bn, const CUtensorMap& a, const CUtensorMap& b, const LinearParams& p, int sms, cudaStream_t st) {
  switch (bn) {
    case 16: return launch_linear<16, BS>(a, b, p, sms, st);
    case 32: return launch_linear<32, BS>(a, b, p, sms, st);
    case 64: return launch_linear<64, BS>(a, b, p, sms, st);
    case 128: return launch_linear<128, BS>(a, b, p, sms, st);
    default: return launch_linear<256, BS>(a, b, p, sms, st);
  }
}

static int check_sizes(int64_t T, int64_t K, int64_t N, int format, int* bs) {
  if (format != QZ_FMT_NVFP4 && format != QZ_FMT_MXFP4)
    return fail(QZ_ERR_INVALID, "the FP4 product takes NVFP4 (blocks of 16) and MXFP4 (blocks of 32), got format %d", format);
  *bs = format == QZ_FMT_NVFP4 ? 16 : 32;
  if (T < 0 || K <= 0 || N <= 0) return fail(QZ_ERR_INVALID, "need T >= 0, K > 0 and N > 0");
  if (K % *bs) return fail(QZ_ERR_INVALID, "K=%lld must be a multiple of the block size %d", (long long)K, *bs);
  if (T > 2147483647LL || K > 1073741824LL || N > 2147483647LL) return fail(QZ_ERR_INVALID, "T, K and N must fit in int32");
  return QZ_OK;
}

}  // namespace qz

using namespace qz;

extern "C" int qz_fp4_scale_layout_bytes(int64_t N, int64_t K, int format, int64_t* bytes) {
  int bs = 0;
  const int s = check_sizes(0, K, N, format, &bs);
  if (s != QZ_OK) return s;
  if (!bytes) return fail(QZ_ERR_INVALID, "NULL pointer");
  *bytes = up(N, 256) / 128 * ((K + kStepK - 1) / kStepK) * (kStepK / bs / 4 * kGroupBytes);
  return QZ_OK;
}

extern "C" int qz_fp4_scale_layout(const uint8_t* scale_codes, int64_t N, int64_t K, int format, uint8_t* out, void* stream) {
  int bs = 0, sms = 0;
  int s = check_sizes(0, K, N, format, &bs);
  if (s != QZ_OK) return s;
  if (!scale_codes || !out) return fail(QZ_ERR_INVALID, "NULL pointer");
  if (reinterpret_cast<uintptr_t>(out) % 16) return fail(QZ_ERR_INVALID, "out must be 16-byte aligned");
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  const int64_t groups = (K + kStepK - 1) / kStepK * (kStepK / bs / 4), tiles = up(N, 256) / 128;
  const int64_t ctas = (tiles * groups * 128 + 255) / 256;
  scale_layout_kernel<<<(unsigned)(ctas < sms * 16 ? ctas : sms * 16), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      scale_codes, N, K / bs, groups, tiles, reinterpret_cast<uint32_t*>(out));
  return cuda_status(cudaGetLastError(), "scale layout launch");
}

extern "C" int qz_fp4_linear_workspace(int64_t T, int64_t K, int64_t N, int format, int64_t* bytes) {
  int bs = 0, sms = 0;
  int s = check_sizes(T, K, N, format, &bs);
  if (s != QZ_OK) return s;
  if (!bytes) return fail(QZ_ERR_INVALID, "NULL pointer");
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  *bytes = T == 0 ? 0 : plan_linear(T, K, N, bs, sms).bytes;
  return QZ_OK;
}

extern "C" int qz_fp4_linear(const void* x, int x_dtype, int64_t ldx, int64_t T, int64_t K, int64_t N, int format,
                             const uint8_t* packed, int64_t ldp, const uint8_t* scales, float tensor_scale,
                             const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  int bs = 0, sms = 0;
  int s = check_sizes(T, K, N, format, &bs);
  if (s != QZ_OK) return s;
  for (int d : {x_dtype, out_dtype, bias ? bias_dtype : QZ_DTYPE_F32})
    if (d != QZ_DTYPE_F32 && d != QZ_DTYPE_BF16 && d != QZ_DTYPE_F16) return fail(QZ_ERR_INVALID, "unknown dtype %d", d);
  if (T == 0) return QZ_OK;
  if (!x || !packed || !scales || !out || !workspace) return fail(QZ_ERR_INVALID, "NULL pointer");
  const int xs = x_dtype == QZ_DTYPE_F32 ? 4 : 2;
  if (ldx < K || ldx * xs % 16) return fail(QZ_ERR_INVALID, "rows of x must be at least K apart and 16-byte aligned");
  if (ldp < up(K, 32) / 2 || ldp % 16)
    return fail(QZ_ERR_INVALID, "packed rows must be at least %lld bytes apart and 16-byte aligned", (long long)(up(K, 32) / 2));
  if (ldo < N) return fail(QZ_ERR_INVALID, "rows of out must be at least N apart");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(scales)) % 16 ||
      reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(QZ_ERR_INVALID, "x, packed and scales must be 16-byte aligned, workspace 256-byte");
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  const LinPlan pl = plan_linear(T, K, N, bs, sms);
  if (workspace_bytes < pl.bytes)
    return fail(QZ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)pl.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool swap = pl.bn < 256;
  CUtensorMap mx, mw;
  s = code_map(&mx, ws, (uint64_t)pl.ldp, (uint64_t)T, (uint64_t)pl.ldp, swap ? pl.bn : 128);
  if (s == QZ_OK) s = code_map(&mw, packed, (uint64_t)pl.ldp, (uint64_t)N, (uint64_t)ldp, swap ? 128 : 256);
  if (s != QZ_OK) return s;
  LinearParams p{};
  p.T = T; p.N = N;
  p.tiles_a = pl.tiles_a; p.tiles_b = pl.tiles_b;
  p.splits = pl.splits; p.n_steps = pl.n_steps;
  p.n_units = pl.tiles_a * pl.tiles_b * pl.splits;
  p.sf_a = swap ? scales : ws + pl.off_sf;
  p.sf_b = swap ? ws + pl.off_sf : scales;
  p.row_scale = reinterpret_cast<float*>(ws + pl.off_scale);
  p.counters = reinterpret_cast<int*>(ws + pl.off_counter);
  p.partial = reinterpret_cast<float*>(ws + pl.off_partial);
  p.w_scale = tensor_scale;
  p.bias = bias; p.bias_dtype = bias_dtype;
  p.out = out; p.out_dtype = out_dtype; p.ldo = ldo;
  p.vec = out_dtype != QZ_DTYPE_F32 && ldo % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const int n_counters = pl.splits > 1 ? (int)(pl.tiles_a * pl.tiles_b) : 0;
  const int gran = pl.bn < 128 ? pl.bn : 128;
  float* rs = reinterpret_cast<float*>(ws + pl.off_scale);
  s = cuda_status(bs == 16 ? launch_quantize_rows<16>(x, x_dtype, ldx, T, K, ws, pl.ldp, ws + pl.off_sf, gran, pl.n_steps,
                                                      rs, p.counters, n_counters, st)
                           : launch_quantize_rows<32>(x, x_dtype, ldx, T, K, ws, pl.ldp, ws + pl.off_sf, gran, pl.n_steps,
                                                      rs, p.counters, n_counters, st),
                  "quantize rows launch");
  if (s != QZ_OK) return s;
  const CUtensorMap &ma = swap ? mw : mx, &mb = swap ? mx : mw;
  return bs == 16 ? run_linear<16>(pl.bn, ma, mb, p, sms, st) : run_linear<32>(pl.bn, ma, mb, p, sms, st);
}
