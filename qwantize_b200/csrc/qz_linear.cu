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
// Two launches: quantize_rows_kernel (one CTA per row), then the product, in one
// of two forms; both walk K in stages of 256 values (128-byte swizzled rows of A
// and B by TMA, their scales by bulk copies) with a ring of stages per CTA:
//
//   linear_kernel (few tokens; BN = 16, 32 or 64): 128 rows of W are A and BN tokens
//   are B, so that a decode step multiplies few padded rows, and W streams through
//   the ring once: the bytes of W bound it.  Where the tiles leave SMs idle, a
//   cluster of 2 or 4 CTAs cuts K among them and adds the fp32 parts, in order,
//   through distributed shared memory, each CTA finishing its share of the columns.
//   1 x 2560 x 9728: 8.1 us, 1 x 8192 x 28672: 27 us (132 MB), with the quantization.
//
//   linear_pair_kernel (prompts): a pair of CTAs on 256 tokens x 256 features; the
//   tensor cores bound it.
//
// A single token goes without the first launch: each CTA quantizes it for itself.
//
// The second launch starts before the first has ended and fetches its first
// stages of W meanwhile.  Issuing a copy or an MMA takes about 30 clocks from an
// elected lane of a converged warp and about 60 from a branch on the lane, so
// each role has a warp of its own and stays converged.
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
// The largest magnitude of 16 bytes of elements: fp32 bits for fp32, else two
// 16-bit patterns side by side that order like the magnitudes (NaN above inf).
template <int DT>
__device__ __forceinline__ uint32_t abs_max(uint32_t m, const uint4& w) {
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (DT == kDtF32) m = max(m, ww[k] & 0x7fffffffu);
    else m = __vmaxu2(m, ww[k] & 0x7fff7fffu);
  }
  return m;
}
// ... as fp32 bits
template <int DT>
__device__ __forceinline__ uint32_t abs_bits(uint32_t m) {
  if (DT == kDtF32) return m;
  m = max(m >> 16, m & 0xffffu);
  return DT == kDtBF16 ? m << 16 : __float_as_uint(f16_bits_to_float(m));
}

template <int DT, int VEC, int BS>
__device__ __forceinline__ void unpack(const uint4 (&w)[VEC], float (&v)[BS]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == kDtF32) {
        v[4 * i + k] = __uint_as_float(ww[k]);
      } else {
        v[8 * i + 2 * k] = DT == kDtBF16 ? bf16_bits_to_float(ww[k] & 0xffffu) : f16_bits_to_float(ww[k] & 0xffffu);
        v[8 * i + 2 * k + 1] = DT == kDtBF16 ? bf16_bits_to_float(ww[k] >> 16) : f16_bits_to_float(ww[k] >> 16);
      }
    }
  }
}

// The power of two p of a row with the largest magnitude m (fp32 bits): the
// exponent e, smallest with max <= 1.3125 * 2^(11 + e); 0 for an all-zero row and
// for inf / NaN.
__device__ __forceinline__ int row_power(uint32_t m) {
  if (m == 0 || m >= 0x7f800000u) return 0;
  return max((int)(m >> 23) - 127 - 11 + ((m & 0x7fffffu) > 0x280000u ? 1 : 0), -120);
}

// One block of x / p (inv = 1 / p; a power of two moves no bit of a 16-bit value):
// its scale code, its values' codes in words.
template <int BS, int DT, int VEC>
__device__ __forceinline__ uint32_t quantize_block(const uint4 (&w)[VEC], uint32_t largest, float inv, uint32_t (&words)[BS / 8]) {
  const uint32_t y = __float_as_uint(__fmul_rn(__uint_as_float(largest), inv));
  uint32_t code;
  float s;
  if (BS == 16) {
    s = e4m3_snap_nonneg(__fdiv_rn(__uint_as_float(y), 6.0f));
    code = e4m3_code(s);
  } else {
    code = is_nan_bits(y) ? 255u : (uint32_t)ue8m0_naive_exp(y);
    s = code == 255u ? __uint_as_float(kMxNanBits) : pow2f((int)code - 127);
  }
  if (!(s > 0.0f)) return code;  // a zero (or NaN) scale keeps codes 0
  float v[BS];
  unpack<DT, VEC>(w, v);
  if (DT != kDtF32) {
    // the conversion rounds the magnitude and keeps the sign
    const float c = __fmul_rn(__frcp_rn(s), kBiasDown);
    const bool in_range = inv >= 0x1p-60f && inv <= 0x1p60f;  // inv * c is exact: one product per value
    const float ci = in_range ? __fmul_rn(c, inv) : c;
#pragma unroll
    for (int i = 0; i < BS; i += 2) {
      float lo = v[i], hi = v[i + 1];
      if (!in_range) { lo = __fmul_rn(lo, inv); hi = __fmul_rn(hi, inv); }
      words[i / 8] |= e2m1x2_rn(__fmul_rn(lo, ci), __fmul_rn(hi, ci)) << (4 * (i % 8));
    }
  } else {
#pragma unroll
    for (int i = 0; i < BS; ++i) {
      const float q = __fdiv_rn(fabsf(__fmul_rn(v[i], inv)), s);
      uint32_t n = __float_as_uint(v[i]) >> 31 << 3;
#pragma unroll
      for (int k = 0; k < 7; ++k) n += q > bnd(k) ? 1u : 0u;
      words[i / 8] |= n << (4 * (i % 8));
    }
  }
  return code;
}

// One CTA per row.  A thread keeps its first R blocks of BS values in registers
// between the row's maximum and the rounding (later ones of very long rows
// are read again, from L2): R = 1 for few rows, where the latency of one row
// counts, R = 4 (NVFP4) or 2 (MXFP4) for many, where loads in flight do.  With the
// product, 64 rows of 8192: 16.9 us with R = 1, 18.0 with 4; 256 rows: 18.8 with
// both; 1024: 27.1 and 25.9; 8192: 90.8 and 72.1.
template <int BS, int DT, int R>
__global__ void __launch_bounds__(R == 1 ? 512 : 256)
    quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t K, uint8_t* __restrict__ packed, int64_t ldp,
                         uint8_t* __restrict__ sf, int gran, int64_t n_steps, float* __restrict__ row_scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ uint32_t s_max[16];
  constexpr int kVec = BS * Elem<DT>::kSize / 16;  // 16-byte loads per block
  const int64_t row = blockIdx.x;
  const uint4* base = reinterpret_cast<const uint4*>(static_cast<const char*>(x) + row * ldx * Elem<DT>::kSize);
  const int64_t nb = K / BS, nb_pad = n_steps * Fmt<BS>::kBlocks, nb_packed = ldp * 2 / BS;
  const int tid = threadIdx.x, nt = blockDim.x;
  uint4 raw[R][kVec];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int64_t b = tid + (int64_t)r * nt;
      raw[r][v] = b < nb ? __ldg(base + b * kVec + v) : make_uint4(0, 0, 0, 0);
    }
  float inv = 1.0f, p = 1.0f;
  uint32_t am[R];  // the blocks' largest magnitudes
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) m = abs_max<DT>(m, raw[r][v]);
    am[r] = abs_bits<DT>(m);
  }
  if (BS == 16) {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) m = max(m, am[r]);
    for (int64_t b = tid + (int64_t)R * nt; b < nb; b += nt) {
      uint32_t o = 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) o = abs_max<DT>(o, __ldg(base + b * kVec + v));
      m = max(m, abs_bits<DT>(o));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < (nt >> 5); ++w) m = max(m, s_max[w]);
    const int e = row_power(m);
    inv = pow2f(-e);
    p = pow2f(e);
  }
  if (tid == 0) row_scale[row] = p;
  uint8_t* sf_row = sf + (row / gran) * n_steps * Fmt<BS>::kSfBytes + (row % gran % 32) * 16 + (row % gran / 32) * 4;
  auto block = [&](int64_t b, const uint4 (&w)[kVec], uint32_t largest) {
    uint32_t code = 0;
    uint32_t words[BS / 8] = {};
    if (b < nb) code = quantize_block<BS, DT>(w, largest, inv, words);
    if (b < nb_packed) {
      if (BS == 16) *reinterpret_cast<uint2*>(packed + row * ldp + b * 8) = make_uint2(words[0], words[1]);
      else *reinterpret_cast<uint4*>(packed + row * ldp + b * 16) = make_uint4(words[0], words[1], words[BS / 16], words[BS / 8 - 1]);
    }
    // four neighbouring blocks share one scale word
    uint32_t sw = code | __shfl_down_sync(0xffffffffu, code, 1) << 8;
    sw |= __shfl_down_sync(0xffffffffu, sw, 2) << 16;
    if ((tid & 3) == 0 && b < nb_pad) *reinterpret_cast<uint32_t*>(sf_row + (b >> 2) * kGroupBytes) = sw;
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
    if ((int64_t)r * nt < nb_pad) block(tid + (int64_t)r * nt, raw[r], am[r]);
  for (int64_t b0 = (int64_t)R * nt; b0 < nb_pad; b0 += nt) {
    uint4 w[kVec];
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      w[v] = b0 + tid < nb ? __ldg(base + (b0 + tid) * kVec + v) : make_uint4(0, 0, 0, 0);
      m = abs_max<DT>(m, w[v]);
    }
    block(b0 + tid, w, abs_bits<DT>(m));
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
  int split;                          // CTAs of a cluster that share a tile (1: no cluster)
  int n_steps;                        // stages over the whole of K
  const uint8_t *sf_a, *sf_b;         // scales: tile-major, n_steps * kSfBytes each
  const float* row_scale;             // p_t
  float w_scale;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t ldo;
  const void* x;                      // the token that the product's own kernel quantizes, K elements
  int64_t K;
  int tma_out;                        // map_out is valid (pair form, 16-bit output, 16-byte rows)
};

// The form of few tokens: A = weight rows, B = tokens.  HERE: the CTA quantizes a
// single token itself and keeps the codes and scales of all its stages.  CTAS per SM:
// two where there are more tiles than SMs (16 and 32 tokens; for 64 the ring would
// be too short): all stream at once instead of in one full wave and one that is not.
// 4 x 8192 x 28672: 29.8 us with one, 27.0 with two; 4 x 2560 x 19456: 14.7, 11.3;
// 48 x 9728 x 2560: 14.5, 12.3; 17 x 4096 x 4096, the one loss seen: 9.5, 10.0.
constexpr int kHereStages = 16;
template <int BN, int BS, bool HERE, int CTAS>
struct LinGeo {
  static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
  static constexpr int kSf = Fmt<BS>::kSfBytes;
  static constexpr int kRing = HERE ? kABytes : kABytes + kBBytes, kRingSf = HERE ? kSf : 2 * kSf;  // of a stage
  static constexpr int kKeep = HERE ? kHereStages * (kBBytes + kSf) : 0;
  static constexpr int kMaxStages = ((CTAS == 1 ? 232448 : 115712) - 1024 - 768 - kKeep) / (kRing + kRingSf);
  static constexpr int kStages = kMaxStages > 10 ? 10 : kMaxStages;
  static constexpr int kSmem = kStages * (kRing + kRingSf) + kKeep + 1024 + 768;
  // TMEM columns: two accumulators, then kSfBufs buffers of scales (kGroups * 4 of A, as many of B)
  static constexpr int kSfCols = Fmt<BS>::kGroups * 4 * 2;
  static constexpr int kSfBufs = 4;
  static constexpr int kAccCols = 2 * BN, kTmemCols = 512 / CTAS;
  static_assert(kAccCols + kSfBufs * kSfCols <= kTmemCols && kStages >= kSfBufs, "TMEM columns");
};

// Block-scaled MMA, E2M1 x E2M1 -> fp32, K = 64, scales of A and B in TMEM:
// one E4M3 scale per 16 values (NVFP4) or one power of two per 32 (MXFP4).
// a, b: low words of the operands' descriptors (address / 16, K-major rows of
// 128 swizzled bytes, 8-row groups 1024 bytes apart).
constexpr uint32_t kDescRows = 1u << 16, kDescRowsHi = (1024u >> 4) | 1u << 14 | 2u << 29;
template <int BS>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accumulate) {
  if constexpr (BS == 16)
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %7};\n mov.b64 y, {%2, %7};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], x, y, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "r"(a | kDescRows), "r"(b | kDescRows), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(kDescRowsHi)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %7};\n mov.b64 y, {%2, %7};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "r"(a | kDescRows), "r"(b | kDescRows), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(kDescRowsHi)
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

// 32 rows of 16 bytes (512 contiguous bytes at 16 * lo, no swizzle, 8-row groups
// 128 bytes apart) -> 4 TMEM columns, spread to all four 32-lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t lo) {
  asm volatile(
      "{\n .reg .b64 x;\n mov.b64 x, {%1, %2};\n tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], x;\n}\n" ::"r"(taddr),
      "r"(lo | (128u >> 4) << 16), "n"((128u >> 4) | 1u << 14)
      : "memory");
}

// 32 lanes x 32 bits, C consecutive columns per thread.
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[C]) {
  if constexpr (C == 16) {
    tmem_ld16(taddr, v);
  } else {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  }
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

// One CTA's work: every gridDim-th tile, or its cluster's tile and its share of
// the stages.
template <bool SWAP>
struct LinWork {
  const LinearParams& p;
  int64_t a, b;  // tile coordinates
  int s0, s1;    // stages [s0, s1) of it
  int64_t tile;

  __device__ __forceinline__ explicit LinWork(const LinearParams& q) : p(q), tile(blockIdx.x / (SWAP ? q.split : 2)) {
    const int rank = SWAP ? blockIdx.x % p.split : 0, parts = SWAP ? p.split : 1;
    s0 = rank * p.n_steps / parts;
    s1 = (rank + 1) * p.n_steps / parts;
  }
  __device__ __forceinline__ bool next() {
    if (tile >= p.tiles_a * p.tiles_b) return false;
    if (SWAP) {
      a = tile % p.tiles_a;
      b = tile / p.tiles_a;
    } else {
      // bands of 8 tiles of tokens: the ~74 tiles in flight are about as many
      // token rows as weight rows and share both through L2
      const int64_t per = 8 * p.tiles_b, band = tile / per, r = tile % per;
      const int64_t left = p.tiles_a - band * 8, rows = left < 8 ? left : 8;
      b = r / rows;
      a = band * 8 + r % rows;
    }
    tile += gridDim.x / (SWAP ? p.split : 2);
    return true;
  }
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float load_peer(uint32_t saddr, int rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// Where a tile's sums go (few tokens): this thread's accumulator row is an output feature, columns are tokens.
template <int BN>
struct LinOutTokens {
  static constexpr int C = BN < 32 ? BN : 32;  // columns drained at a time
  const LinearParams& p;
  int row, lane, cols;  // accumulator row; tokens of the tile that exist
  int64_t ra, cb;       // output feature, first token
  bool in;
  float bias;
  const float* scales;  // of the tile's tokens

  __device__ __forceinline__ LinOutTokens(const LinearParams& q, const LinWork<true>& u, const float* here) : p(q) {
    lane = threadIdx.x & 31;
    row = (threadIdx.x >> 5 & 3) * 32 + lane;
    ra = u.a * 128 + row;
    cb = u.b * BN;
    cols = p.T - cb < BN ? (int)(p.T - cb) : BN;
    in = ra < p.N;
    bias = in && p.bias ? load_any(p.bias, p.bias_dtype, ra) : 0.0f;
    scales = here ? here : p.row_scale + cb;
  }
  // lane q: the scale of token c + q
  __device__ __forceinline__ float column(int c) const {
    return c + lane < cols && lane < C ? scales[c + lane] * p.w_scale : 0.0f;
  }
  __device__ __forceinline__ void store(int c, float v, float scale) const {
    if (in) store_any(p.out, p.out_dtype, (cb + c) * p.ldo + ra, __fmaf_rn(v, scale, bias));
  }
  // C columns from c: scale, bias, round once, store.  The output type is asked for once: with a branch on it in every
  // column their conversions and stores do not overlap.
  template <int DT>
  __device__ __forceinline__ void finish_as(int c, float (&v)[C], float col) const {
    const int64_t at = (cb + c) * p.ldo + ra;
#pragma unroll
    for (int q = 0; q < C; ++q) {
      const float y = __fmaf_rn(v[q], __shfl_sync(0xffffffffu, col, q), bias);
      if (in && c + q < cols) store_any(p.out, DT, at + q * p.ldo, y);
    }
  }
  __device__ __forceinline__ void finish(int c, float (&v)[C], float col) const {
    if (p.out_dtype == kDtBF16) finish_as<kDtBF16>(c, v, col);
    else if (p.out_dtype == kDtF16) finish_as<kDtF16>(c, v, col);
    else finish_as<kDtF32>(c, v, col);
  }
};

// The same for a tile of a prompt: rows are tokens, columns are output features.
struct LinOutRows {
  static constexpr int BN = 256, C = 32;
  const LinearParams& p;
  int row, lane, cols;   // accumulator row; features of the tile that exist
  int64_t ra, ra0, cb;   // token, first token, first feature
  bool in;
  float scale;           // of this token

  __device__ __forceinline__ LinOutRows(const LinearParams& q, const LinWork<false>& u) : p(q) {
    lane = threadIdx.x & 31;
    row = (threadIdx.x >> 5 & 3) * 32 + lane;
    ra0 = u.a * 128;
    ra = ra0 + row;
    cb = u.b * BN;
    cols = p.N - cb < BN ? (int)(p.N - cb) : BN;
    in = ra < p.T;
    // an ordinary load: the launch before this one may still write them when this one begins
    scale = in ? p.row_scale[ra] * p.w_scale : 0.0f;
  }
  // C columns from c: scale, bias, round once, store
  __device__ __forceinline__ void finish(int c, float (&v)[C], const CUtensorMap& map_out, unsigned char* smem_out) const {
    if (p.bias) {
      const float b = c + lane < cols ? load_any(p.bias, p.bias_dtype, cb + c + lane) : 0.0f;
#pragma unroll
      for (int q = 0; q < C; ++q) v[q] = __fmaf_rn(v[q], scale, __shfl_sync(0xffffffffu, b, q));
    } else {
#pragma unroll
      for (int q = 0; q < C; ++q) v[q] = __fmul_rn(v[q], scale);
    }
    // 32 rows of 64 bytes per warp, 16-byte pieces swizzled: a row at a time leaves for memory from here, since
    // lanes that each write their own row touch 32 sectors with every store (3841 x 1424 x 2630: 140 us with the call,
    // 39 this way, 29 with 16-byte rows and TMA)
    const int64_t r0 = ra0 + (row & ~31);
    if (r0 >= p.T) return;
    unsigned char* stage = smem_out + (row >> 5) * 2048;
    auto piece = [&](int r, int q) { return stage + r * 64 + ((q ^ (r >> 1 & 3)) << 4); };
    if (p.out_dtype == kDtF32) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(piece(lane, q)) =
              make_float4(v[16 * half + 4 * q], v[16 * half + 4 * q + 1], v[16 * half + 4 * q + 2], v[16 * half + 4 * q + 3]);
        __syncwarp();
        const int k = lane & 15, col = c + 16 * half + k;
        float* to = static_cast<float*>(p.out) + (r0 + (lane >> 4)) * p.ldo + cb + col;
#pragma unroll 1
        for (int r = lane >> 4; r < 32; r += 16) {
          float x[8];  // all loads before the first store
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const float*>(piece(r + 2 * i, k >> 2) + (k & 3) * 4);
#pragma unroll
          for (int i = 0; i < 8; ++i, to += 2 * p.ldo)
            if (r0 + r + 2 * i < p.T && col < cols) *to = x[i];
        }
      }
      return;
    }
    if (p.tma_out && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4*>(piece(lane, q)) =
          make_uint4(pack16(v[8 * q], v[8 * q + 1], p.out_dtype), pack16(v[8 * q + 2], v[8 * q + 3], p.out_dtype),
                     pack16(v[8 * q + 4], v[8 * q + 5], p.out_dtype), pack16(v[8 * q + 6], v[8 * q + 7], p.out_dtype));
    if (p.tma_out) {  // the tensor map clips rows and columns beyond the result
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&map_out),
                     "r"((int)cb + c), "r"((int)r0), "r"(smem_u32(stage))
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else {  // rows that are not 16-byte aligned
      __syncwarp();
      uint16_t* to = static_cast<uint16_t*>(p.out) + r0 * p.ldo + cb + c + lane;
#pragma unroll 1
      for (int r = 0; r < 32; r += 8) {
        uint16_t x[8];  // all loads before the first store
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint16_t*>(piece(r + i, lane >> 3) + (lane & 7) * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i, to += p.ldo)
          if (r0 + r + i < p.T && c + lane < cols) *to = x[i];
      }
    }
  }
};

constexpr int kLinThreads = 224;

// One token's codes and scales of stages [s0, s1), in the layout that TMA and the
// bulk copies would give the stages of a ring, by the 128 threads of warps 2-5.
// The row's maximum takes all of it, also where a cluster cuts K.
template <int BS, int DT>
__device__ __forceinline__ void quantize_here(const LinearParams& p, int s0, int s1, int stage_bytes, unsigned char* codes,
                                              unsigned char* sf, float* scale, uint32_t* s_max) {
  constexpr int kVec = BS * Elem<DT>::kSize / 16, kBlocks = Fmt<BS>::kBlocks, kMost = kHereStages * kBlocks / 128;
  const int tid = threadIdx.x - 64, nb = (int)(p.K / BS), blocks = (s1 - s0) * kBlocks;
  const uint4* row = static_cast<const uint4*>(p.x);
  uint4 w[kMost][kVec];
#pragma unroll
  for (int i = 0; i < kMost; ++i)
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int j = tid + i * 128, b = s0 * kBlocks + j;
      w[i][v] = j < blocks && b < nb ? __ldg(row + b * kVec + v) : make_uint4(0, 0, 0, 0);
    }
  int e = 0;
  if (BS == 16) {
    uint32_t m = 0;
#pragma unroll 4
    for (int v = tid; v < nb * kVec; v += 128) m = abs_max<DT>(m, __ldg(row + v));
    m = __reduce_max_sync(0xffffffffu, abs_bits<DT>(m));
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    asm volatile("barrier.sync 1, 128;" ::: "memory");
    e = row_power(max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3])));
  }
  const float inv = pow2f(-e);
  if (tid == 0) *scale = pow2f(e);
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int j = tid + i * 128, kb = j % kBlocks;
    if (j >= blocks) break;
    uint32_t m = 0, words[BS / 8] = {}, code = 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) m = abs_max<DT>(m, w[i][v]);
    if (s0 * kBlocks + j < nb) code = quantize_block<BS, DT>(w[i], abs_bits<DT>(m), inv, words);
    unsigned char* to = codes + j / kBlocks * stage_bytes;  // row 0 of the swizzle: in order
    if constexpr (BS == 16) *reinterpret_cast<uint2*>(to + kb * 8) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint4*>(to + kb * 16) = make_uint4(words[0], words[1], words[BS / 16], words[BS / 8 - 1]);
    sf[j / kBlocks * Fmt<BS>::kSfBytes + kb / 4 * kGroupBytes + kb % 4] = (uint8_t)code;
  }
  fence_proxy_async_smem();
  asm volatile("barrier.sync 1, 128;" ::: "memory");  // the scale
}

// HERE: the type of the one token that this kernel quantizes itself (-1: an earlier launch does)
template <int BN, int BS, int HERE, int CTAS>
__global__ void __launch_bounds__(kLinThreads, CTAS)
    linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ LinearParams p) {
  // 224 threads: warp 0 feeds the ring, warp 6 copies a stage's scales to TMEM (tcgen05.cp), warp 1 issues its four
  // block-scaled MMAs of K = 64, warps 2-5 drain the accumulator
  constexpr bool kHere = HERE >= 0;
  using G = LinGeo<BN, BS, kHere, CTAS>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // operands (1024-byte swizzle atoms), the scales of all stages, barriers
  unsigned char* smem_x = smem + G::kStages * G::kRing;  // kHere: the token's codes, then its scales (the other 15 rows of B are whatever is there)
  unsigned char* smem_xsf = smem_x + kHereStages * G::kBBytes;
  unsigned char* smem_sf = smem_x + G::kKeep;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_sf + G::kStages * G::kRingSf);
  uint64_t* empty = full + G::kStages;
  uint64_t* tfull = empty + G::kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* sf_full = tempty + 2;
  uint64_t* mma_done = sf_full + G::kSfBufs;
  uint64_t* sf_done = mma_done + 1;
  uint64_t* x_here = sf_done + 1;  // kHere: the token is in shared memory
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(x_here + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  float* scale_here = reinterpret_cast<float*>(tmem_base_s + 2);
  uint32_t* s_max = reinterpret_cast<uint32_t*>(scale_here + 1);
  constexpr int C = LinOutTokens<BN>::C;
  float* part = reinterpret_cast<float*>(smem);  // (BN, 128) fp32, over the ring's first stages
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull + a, 1); mbar_init(tempty + a, 128); }
    for (int b = 0; b < G::kSfBufs; ++b) mbar_init(sf_full + b, 1);
    mbar_init(mma_done, 1);
    mbar_init(sf_done, 1);
    mbar_init(x_here, 128);
    *abort_s = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_base_s, G::kTmemCols);
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
    // ---------------- producer (the warp stays converged: one elected lane issues) ----------------
    auto load_w = [&](const LinWork<true>& u, int ks, int s) {
      mbar_arrive_expect_tx(full + s, G::kRing + G::kRingSf);
      tma_load_2d(smem + s * G::kRing, &map_a, ks * 128, (int)(u.a * 128), full + s);
      bulk_load(smem_sf + s * G::kRingSf, p.sf_a + (u.a * p.n_steps + ks) * G::kSf, G::kSf, full + s);
    };
    auto load_x = [&](const LinWork<true>& u, int ks, int s) {
      if (kHere) return;
      tma_load_2d(smem + s * G::kRing + G::kABytes, &map_b, ks * 128, (int)(u.b * BN), full + s);
      bulk_load(smem_sf + s * G::kRingSf + G::kSf, p.sf_b + (u.b * p.n_steps + ks) * G::kSf, G::kSf, full + s);
    };
    // the first ring of weights does not wait for the quantization launch
    uint32_t ahead = 0;
    for (LinWork<true> u(p); ahead < (uint32_t)G::kStages && u.next();)
      for (int ks = u.s0; ks < u.s1 && ahead < (uint32_t)G::kStages; ++ks, ++ahead) {
        if (elect_one()) load_w(u, ks, ahead);
        __syncwarp();
      }
    if (!kHere) asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t it = 0, s = 0, ph = 1;
    bool ok = true;
    for (LinWork<true> u(p); ok && u.next();) {
      for (int ks = u.s0; ks < u.s1; ++ks, ++it) {
        if (it >= ahead) {
          ok = __all_sync(0xffffffffu, wait(empty + s, ph, kDevErrLoadTimeout));
          if (!ok) break;
        }
        if (elect_one()) {
          if (it >= ahead) load_w(u, ks, s);
          load_x(u, ks, s);
        }
        __syncwarp();
        if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
      }
    }
    // every load issued must have landed before the CTA can exit (bounded)
    for (uint32_t k = it > (uint32_t)G::kStages ? it - G::kStages : 0u; k < it; ++k)
      mbar_wait_bounded(full + (k % G::kStages), (k / G::kStages) & 1, kDevErrLoadTimeout);
  } else if (warp == 1) {
    // ---------------- MMA issuer (the warp waits together, one lane issues) ----------------
    // low words of the descriptors of stage 0; a stage further is an addition
    const uint32_t lo_a = smem_u32(smem) >> 4, lo_b = kHere ? smem_u32(smem_x) >> 4 : lo_a + (G::kABytes >> 4);
    const bool ready = !kHere || wait(x_here, 0, kDevErrMmaTimeout);
    uint32_t lt = 0, s = 0, ph = 0, sb = 0, sph = 0;  // stage, scale buffer, their phases
    for (LinWork<true> u(p); u.next(); ++lt) {
      const uint32_t acc = lt & 1;
      bool ok = ready && wait(tempty + acc, (lt >> 1 & 1) ^ 1, kDevErrMmaTimeout);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int ks = u.s0; ks < u.s1; ++ks) {
        ok = wait(full + s, ph, kDevErrMmaTimeout) && wait(sf_full + sb, sph, kDevErrMmaTimeout);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t da = lo_a + s * (G::kRing >> 4), db = lo_b + (kHere ? (ks - u.s0) * (G::kBBytes >> 4) : s * (G::kRing >> 4));
        const uint32_t t_sfa = tmem_base + G::kAccCols + sb * G::kSfCols, t_sfb = t_sfa + Fmt<BS>::kGroups * 4;
        const uint32_t first = ks > u.s0 ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int q = BS == 16 ? kk : kk / 2;
            umma_fp4<BS>(d_tmem, da + 2 * kk, db + 2 * kk, idesc_fp4<BS>(BN, BS == 16 ? 0u : (kk & 1) * 2u), t_sfa + 4 * q,
                         t_sfb + 4 * q, kk > 0 ? 1u : first);
          }
          umma_commit(empty + s);
          if (ks + 1 == u.s1) umma_commit(tfull + acc);
        }
        __syncwarp();
        if (++sb == (uint32_t)G::kSfBufs) { sb = 0; sph ^= 1; }
        if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
      }
      if (!ok) break;
    }
    // the MMAs issued must retire before TMEM is freed (also after an abort)
    __syncwarp();
    if (elect_one()) umma_commit(mma_done);
    __syncwarp();
    mbar_wait_bounded(mma_done, 0u, kDevErrMmaTimeout);
  } else if (warp == 6) {
    // ---------------- scales to TMEM ----------------
    const uint32_t lo_sf = smem_u32(smem_sf) >> 4;
    uint32_t s = 0, ph = 0, sb = 0, warm = 0;  // warm: scale buffers used so far, up to kSfBufs
    const uint32_t lo_xsf = smem_u32(smem_xsf) >> 4;
    bool ok = !kHere || __all_sync(0xffffffffu, wait(x_here, 0, kDevErrMmaTimeout));
    for (LinWork<true> u(p); ok && u.next();) {
      for (int ks = u.s0; ks < u.s1; ++ks) {
        ok = wait(full + s, ph, kDevErrMmaTimeout);
        // this scale buffer was last read by the MMAs kSfBufs stages ago
        if (warm == (uint32_t)G::kSfBufs) {
          const bool wrap = s < (uint32_t)G::kSfBufs;
          ok = ok && wait(empty + (wrap ? s + G::kStages - G::kSfBufs : s - G::kSfBufs), wrap ? ph ^ 1 : ph, kDevErrMmaTimeout);
        } else {
          ++warm;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ds = lo_sf + s * (G::kRingSf >> 4);
        const uint32_t ds_b = kHere ? lo_xsf + (ks - u.s0) * (G::kSf >> 4) : ds + (G::kSf >> 4);
        const uint32_t t_sfa = tmem_base + G::kAccCols + sb * G::kSfCols, t_sfb = t_sfa + Fmt<BS>::kGroups * 4;
        if (elect_one()) {
#pragma unroll
          for (int q = 0; q < Fmt<BS>::kGroups; ++q) {
            tmem_cp_scales(t_sfa + 4 * q, ds + q * (kGroupBytes >> 4));
            tmem_cp_scales(t_sfb + 4 * q, ds_b + q * (kGroupBytes >> 4));
          }
          umma_commit(sf_full + sb);
        }
        __syncwarp();
        if (++sb == (uint32_t)G::kSfBufs) sb = 0;
        if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
      }
    }
    // the copies issued must have ended before TMEM is freed (also after an abort)
    __syncwarp();
    if (elect_one()) umma_commit(sf_done);
    __syncwarp();
    mbar_wait_bounded(sf_done, 0u, kDevErrMmaTimeout);
  } else {
    // ---------------- epilogue (warps 2-5) ----------------
    if constexpr (kHere) {
      LinWork<true> u(p);
      quantize_here<BS, HERE>(p, u.s0, u.s1, G::kBBytes, smem_x, smem_xsf, scale_here, s_max);
      mbar_arrive(x_here);
    } else {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // row scales are the quantization launch's
    }
    uint32_t lt = 0;
    for (LinWork<true> u(p); u.next(); ++lt) {
      const uint32_t acc = lt & 1, phase = lt >> 1 & 1;
      LinOutTokens<BN> out(p, u, kHere ? scale_here : nullptr);
      if (!__all_sync(0xffffffffu, wait(tfull + acc, phase, kDevErrEpilogueTimeout))) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * BN;
      float col = out.column(0);
#pragma unroll 1
      for (int c = 0; c < BN; c += C) {
        const float now = col;
        col = out.column((c + C) % BN);
        float v[C];
        if (c < out.cols) tmem_ld<C>(taddr + c, v);
        if (c + C == BN) {
          tc_fence_before();
          mbar_arrive(tempty + acc);
        }
        if (c >= out.cols) continue;
        if (p.split > 1) {  // this CTA's part, to be added below (the ring is idle: all its MMAs are done)
#pragma unroll
          for (int q = 0; q < C; ++q) part[(c + q) * 128 + out.row] = v[q];
        } else {
          out.finish(c, v, now);
        }
      }
    }
  }
  if (p.split > 1) {
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && warp < 6) {
      LinWork<true> u(p);
      if (u.next()) {
        // rank r finishes columns [r, r + 1) * BN / split, which lie in one group of C
        static_assert(BN / 2 <= C, "columns of a rank");
        LinOutTokens<BN> out(p, u, kHere ? scale_here : nullptr);
        const int rank = blockIdx.x % p.split, per = BN / p.split;
        const float col = out.column(rank * per / C * C);
        const uint32_t at = smem_u32(part) + out.row * 4;
        const int c_end = (rank + 1) * per < out.cols ? (rank + 1) * per : out.cols;
        for (int c0 = rank * per; c0 < c_end; c0 += 4) {
          float x[4][4];  // all loads of four columns before the first sum
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q][w] = w < p.split && c0 + q < c_end ? load_peer(at + (c0 + q) * 512, w) : 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v = x[q][0];
#pragma unroll
            for (int w = 1; w < 4; ++w) v += x[q][w];
            const float scale = __shfl_sync(0xffffffffu, col, (c0 + q) % C);
            if (c0 + q < c_end) out.store(c0 + q, v, scale);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();  // the parts have been read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, G::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// the product of a prompt: two CTAs on one tile
// ---------------------------------------------------------------------------
// 256 tokens x 256 output features by a cluster of two CTAs (cta_group::2): each
// has 128 token rows of A, 128 of the tile's 256 rows of W, and the sums of its
// own tokens; the tensor cores of both read both halves of B.  A stage is then
// 38 KB per SM for 512 clocks of MMAs, where one CTA on 128 x 256 needs 55 KB: the
// SMs take about 64 bytes per clock from L2, and that bounded a form of one CTA
// per tile (945 clocks a stage, 829 us for 8192 x 8192 x 28672).  This one: 610 clocks
// a stage, 673 us alone (5.7 PFLOP/s, tensor pipe 82% active); in a row the board
// reaches its power limit and the clock falls: 770 to 885 us a call, as long as it
// lasts.
//
// 320 threads: warp 0 feeds this CTA's ring; its tiles signal the leader (rank 0),
// its scales this CTA.  Warps 6-9 put a stage's scales in this CTA's TMEM (its
// tokens', and those of all 256 features) and tell the leader, whose warp 1 issues
// the MMAs of the pair; commits free a stage and publish the sums in both CTAs;
// warps 2-5 drain.  TMEM holds two accumulators that share 96 columns, so that two
// buffers of scales fit beside them; the epilogue takes the shared columns into
// registers first, and the next tile begins once it has (with 160 shared columns
// and three buffers: 695 clocks a stage).  Everything another CTA reads or signals
// lies between the cluster barriers at both ends.
template <int BS>
struct PairGeo {
  static constexpr int BN = LinOutRows::BN;
  static constexpr int kABytes = 128 * 128, kBBytes = 128 * 128;
  static constexpr int kSf = Fmt<BS>::kSfBytes;
  static constexpr int kStageBytes = kABytes + kBBytes + 3 * kSf;
  static constexpr int kOutBytes = 4 * 2048;
  static constexpr int kMaxStages = (232448 - 1024 - 512 - kOutBytes) / kStageBytes;
  static constexpr int kStages = kMaxStages > 6 ? 6 : kMaxStages;
  static constexpr int kSmem = kStages * kStageBytes + kOutBytes + 1024 + 512;
  // TMEM columns: two accumulators that share kOverlap columns, then kSfBufs buffers of scales
  static constexpr int kSfCols = Fmt<BS>::kGroups * 4 * 3;
  static constexpr int kOverlap = 96;
  static constexpr int kAccCols = 2 * BN - kOverlap;
  static constexpr int kSfBufs = (512 - kAccCols) / kSfCols;
  static_assert(kSfBufs >= 2 && kStages > kSfBufs && kOverlap % LinOutRows::C == 0, "TMEM columns");
};
constexpr int kPairThreads = 320;

template <int BS>
__device__ __forceinline__ void umma_fp4_pair(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                              uint32_t accumulate) {
  if constexpr (BS == 16)
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %7};\n mov.b64 y, {%2, %7};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], x, y, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "r"(a | kDescRows), "r"(b | kDescRows), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(kDescRowsHi)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %7};\n mov.b64 y, {%2, %7};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "r"(a | kDescRows), "r"(b | kDescRows), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(kDescRowsHi)
        : "memory");
}

// Arrive on the barrier at this offset in both CTAs once the pair's MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "{\n .reg .b16 m;\n mov.b16 m, 3;\n"
      " tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// Arrivals at the leader's barrier and waits for the pair's. They are relaxed: what they order is in TMEM (the
// tcgen05 fences beside them do that) or was loaded into registers that have been used; the operands themselves signal
// the leader's barrier directly. With release.cluster an arrival took about 1300 clocks, and every stage waits for one.
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %0, 0;\n"
      " mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [at];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A tile into this CTA's memory that signals the leader's barrier at this offset.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "{\n .reg .b32 at;\n mapa.shared::cluster.u32 at, %4, 0;\n"
      " cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[at];\n}\n" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// C columns of 32 bits from registers to TMEM, one row per lane.
template <int C>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t* r) {
  if constexpr (C == 32)
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
        "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
  else if constexpr (C == 16)
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

template <int BS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_out, const __grid_constant__ LinearParams p) {
  using G = PairGeo<BS>;
  constexpr int BN = G::BN;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* smem_out = smem + G::kStages * (G::kABytes + G::kBBytes);
  unsigned char* smem_sf = smem_out + G::kOutBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::kStages * G::kStageBytes + G::kOutBytes);  // the leader's: operands
  uint64_t* sf_in = full + G::kStages;       // this CTA's scales of a stage are in shared memory
  uint64_t* empty = sf_in + G::kStages;
  uint64_t* tfull = empty + G::kStages;
  uint64_t* tempty = tfull + 2;              // the leader's: both CTAs' shared columns are drained
  uint64_t* sf_full = tempty + 1;            // the leader's: both CTAs' scales are in TMEM
  uint64_t* mma_done = sf_full + G::kSfBufs;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) { mbar_init(full + s, 1); mbar_init(sf_in + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) mbar_init(tfull + a, 1);
    mbar_init(tempty, 2 * 128);
    for (int b = 0; b < G::kSfBufs; ++b) mbar_init(sf_full + b, 2 * 4);
    mbar_init(mma_done, 1);
    *abort_s = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_base_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers and TMEM exist
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_s;

  // data: the wait is for loads that this CTA's threads or the tensor core read from shared memory
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned err, bool data = false) -> bool {
    if (data ? mbar_try_wait(bar, parity) : mbar_try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!(data ? mbar_try_wait(bar, parity) : mbar_try_wait_cluster(bar, parity))) {
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
    // ---------------- producer (the warp stays converged: one elected lane issues) ----------------
    auto load_w = [&](const LinWork<false>& u, int ks, int s) {
      unsigned char* sb = smem + s * (G::kABytes + G::kBBytes) + G::kABytes;
      unsigned char* sf = smem_sf + s * 3 * G::kSf;
      if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * (G::kABytes + G::kBBytes));
      mbar_arrive_expect_tx(sf_in + s, 3 * G::kSf);
      tma_load_2d_pair(sb, &map_b, ks * 128, (int)(u.b * BN) + rank * 128, full + s);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        bulk_load(sf + (1 + h) * G::kSf, p.sf_b + ((u.b * 2 + h) * p.n_steps + ks) * G::kSf, G::kSf, sf_in + s);
    };
    auto load_x = [&](const LinWork<false>& u, int ks, int s) {
      const int64_t a = u.a * 2 + rank;
      tma_load_2d_pair(smem + s * (G::kABytes + G::kBBytes), &map_a, ks * 128, (int)(a * 128), full + s);
      bulk_load(smem_sf + s * 3 * G::kSf, p.sf_a + (a * p.n_steps + ks) * G::kSf, G::kSf, sf_in + s);
    };
    // the first ring of weights does not wait for the quantization launch
    uint32_t ahead = 0;
    for (LinWork<false> u(p); ahead < (uint32_t)G::kStages && u.next();)
      for (int ks = u.s0; ks < u.s1 && ahead < (uint32_t)G::kStages; ++ks, ++ahead) {
        if (elect_one()) load_w(u, ks, ahead);
        __syncwarp();
      }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t it = 0, s = 0, ph = 1;
    bool ok = true;
    for (LinWork<false> u(p); ok && u.next();) {
      for (int ks = u.s0; ks < u.s1; ++ks, ++it) {
        if (it >= ahead) {
          ok = __all_sync(0xffffffffu, wait(empty + s, ph, kDevErrLoadTimeout));
          if (!ok) break;
        }
        if (elect_one()) {
          if (it >= ahead) load_w(u, ks, s);
          load_x(u, ks, s);
        }
        __syncwarp();
        if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
      }
    }
    // every load issued must have landed before the CTA can exit (bounded)
    for (uint32_t k = it > (uint32_t)G::kStages ? it - G::kStages : 0u; k < it; ++k) {
      mbar_wait_bounded(sf_in + (k % G::kStages), (k / G::kStages) & 1, kDevErrLoadTimeout);
      if (rank == 0) mbar_wait_bounded(full + (k % G::kStages), (k / G::kStages) & 1, kDevErrLoadTimeout);
    }
    // after an abort the leader may not have waited for this CTA's last operands
    if (rank == 1 && *abort_s)
      for (int k = 0; k < 100; ++k) __nanosleep(1000);
  } else if (warp == 1) {
    // ---------------- MMA issuer (the leader's) ----------------
    if (rank == 0) {
      const uint32_t lo_a = smem_u32(smem) >> 4, lo_b = lo_a + (G::kABytes >> 4);
      uint32_t lt = 0, s = 0, ph = 0, sb = 0, sph = 0;
      for (LinWork<false> u(p); u.next(); ++lt) {
        const uint32_t acc = lt & 1;
        bool ok = lt == 0 || wait(tempty, (lt - 1) & 1, kDevErrMmaTimeout);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * (BN - G::kOverlap);
        for (int ks = u.s0; ks < u.s1; ++ks) {
          ok = wait(full + s, ph, kDevErrMmaTimeout, true);
          ok = __all_sync(0xffffffffu, ok && wait(sf_full + sb, sph, kDevErrMmaTimeout));
          if (!ok) break;
          tc_fence_after();
          const uint32_t da = lo_a + s * ((G::kABytes + G::kBBytes) >> 4), db = lo_b + s * ((G::kABytes + G::kBBytes) >> 4);
          const uint32_t t_sfa = tmem_base + G::kAccCols + sb * G::kSfCols, t_sfb = t_sfa + Fmt<BS>::kGroups * 4;
          const uint32_t first = ks > u.s0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const int q = BS == 16 ? kk : kk / 2;
              // M = 256: the descriptor's field counts 16 rows, as for 128
              constexpr uint32_t m256 = (uint32_t)(256 >> 4) << 24, m128 = (uint32_t)(128 >> 4) << 24;
              umma_fp4_pair<BS>(d_tmem, da + 2 * kk, db + 2 * kk, idesc_fp4<BS>(BN, BS == 16 ? 0u : (kk & 1) * 2u) - m128 + m256,
                                t_sfa + 4 * q, t_sfb + 8 * q, kk > 0 ? 1u : first);
            }
            umma_commit_pair(empty + s);
            if (ks + 1 == u.s1) umma_commit_pair(tfull + acc);
          }
          __syncwarp();
          if (++sb == (uint32_t)G::kSfBufs) { sb = 0; sph ^= 1; }
          if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
      }
      // the MMAs issued must retire before either CTA's TMEM is freed (also after an abort)
      __syncwarp();
      if (elect_one()) umma_commit_pair(mma_done);
      __syncwarp();
      mbar_wait_bounded(mma_done, 0u, kDevErrMmaTimeout);
    }
  } else if (warp >= 6) {
    // ---------------- scales to TMEM (warps 6-9, one quarter of the lanes each) ----------------
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s = 0, ph = 0, sb = 0, warm = 0;  // warm: scale buffers used so far, up to kSfBufs
    bool ok = true;
    for (LinWork<false> u(p); ok && u.next();) {
      for (int ks = u.s0; ks < u.s1; ++ks) {
        ok = wait(sf_in + s, ph, kDevErrMmaTimeout, true);
        uint32_t r[G::kSfCols];
        const unsigned char* sf = smem_sf + s * 3 * G::kSf + lane * 16;
#pragma unroll
        for (int q = 0; q < Fmt<BS>::kGroups; ++q) {
          *reinterpret_cast<uint4*>(r + 4 * q) = *reinterpret_cast<const uint4*>(sf + q * kGroupBytes);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<uint4*>(r + (Fmt<BS>::kGroups + 2 * q + h) * 4) =
                *reinterpret_cast<const uint4*>(sf + (1 + h) * G::kSf + q * kGroupBytes);
        }
        // this scale buffer was last read by the MMAs kSfBufs stages ago
        if (warm == (uint32_t)G::kSfBufs) {
          const bool wrap = s < (uint32_t)G::kSfBufs;
          ok = ok && wait(empty + (wrap ? s + G::kStages - G::kSfBufs : s - G::kSfBufs), wrap ? ph ^ 1 : ph, kDevErrMmaTimeout);
        } else {
          ++warm;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_sf = tmem_base + quarter + G::kAccCols + sb * G::kSfCols;
        constexpr int kLow = G::kSfCols == 48 ? 32 : 16;
        tmem_st<kLow>(t_sf, r);
        tmem_st<G::kSfCols - kLow>(t_sf + kLow, r + kLow);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(sf_full + sb);
        if (++sb == (uint32_t)G::kSfBufs) sb = 0;
        if (++s == (uint32_t)G::kStages) { s = 0; ph ^= 1; }
      }
    }
  } else {
    // ---------------- epilogue (warps 2-5) ----------------
    asm volatile("griddepcontrol.wait;" ::: "memory");  // row scales are the quantization launch's
    constexpr int C = LinOutRows::C, kShared = G::kOverlap / C;
    uint32_t lt = 0;
    for (LinWork<false> u(p); u.next(); ++lt) {
      const uint32_t acc = lt & 1, phase = lt >> 1 & 1;
      u.a = u.a * 2 + rank;  // this CTA's 128 rows
      LinOutRows out(p, u);
      if (!__all_sync(0xffffffffu, wait(tfull + acc, phase, kDevErrEpilogueTimeout))) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * (BN - G::kOverlap);
      // the columns shared with the next tile's accumulator come first
      const int c_first = acc == 0 ? BN - G::kOverlap : 0;
      float v[kShared][C];
#pragma unroll
      for (int i = 0; i < kShared; ++i)
        if (c_first + i * C < out.cols) tmem_ld<C>(taddr + c_first + i * C, v[i]);
      tc_fence_before();
      mbar_arrive_leader(tempty);
#pragma unroll
      for (int i = 0; i < kShared; ++i) {
        const int c = c_first + i * C;
        if (c < out.cols) out.finish(c, v[i], map_out, smem_out);
      }
#pragma unroll 1
      for (int i = kShared; i < BN / C; ++i) {
        const int c = (c_first + i * C) % BN;
        if (c >= out.cols) continue;
        tmem_ld<C>(taddr + c, v[0]);
        out.finish(c, v[0], map_out, smem_out);
      }
    }
    // staged output has been written (the staging area goes away with the CTA)
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // the last of the leader's signals: all before it have come
  if (warp == 1 && rank == 1) mbar_wait_bounded(mma_done, 0u, kDevErrMmaTimeout);
  __syncthreads();
  cluster_sync();  // neither CTA's memory is read or signalled any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
  __syncwarp();
  cluster_sync();  // both CTAs take part in freeing the pair's TMEM
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

// 16-bit output (T, N), written in boxes of 32 x 32.
static int out_map(CUtensorMap* m, void* base, uint64_t N, uint64_t T, uint64_t ldo) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(QZ_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {N, T};
  cuuint64_t strides[1] = {ldo * 2};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QZ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return QZ_OK;
}

// Tile form and cluster size of one call, and its workspace.
struct LinPlan {
  int bn, split, n_steps;
  int gran;   // rows of a tile of x's scales
  bool here;  // the product's kernel quantizes the token itself
  bool two;   // two CTAs per SM
  int64_t tiles_a, tiles_b, ldp;
  int64_t off_sf, off_scale, bytes;
};

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Chooses the form by an estimate in microseconds: waves of tiles x stages x time
// of a stage (1.4 of it where two CTAs share an SM), what follows the last stage,
// and a cluster's exchange of sums.  Checked against every form that can run, at 16
// numbers of tokens from 1 to 2048 and (K, N) = (1024, 1024), (2560, 9728), (9728, 2560),
// (4096, 4096), (2560, 1000), (8192, 1024), (2560, 19456), (8192, 2048) and (8192, 28672),
// MXFP4 at the first three (per call in a graph of 100, over weights that exceed L2
// together; repeats agree within 0.1 us): the choice is the fastest or within 10% of
// it in 179 of 189.  The others: 64 tokens of 1024 x 1024 (10.3%), and 333 to 1024 tokens
// of weights with about 1000 features and K up to 2560, which the limit of eight
// passes over W keeps from the narrow forms (1024 x 1024, 333 tokens: 9.8 us, 16
// columns 7.8; 2560 x 1000: 13.2, 10.8).
// Some, in microseconds with the quantization: 2560 x 9728, 64 tokens: 32 columns (two
// CTAs per SM) 11.1, 64 13.0, 16 14.0, pair 13.0; 192 tokens: 15.7, 17.5, 21.8, pair 13.3.
// 9728 x 2560, 1 token: clusters of 4, 2, 1: 9.9, 13.0, 17.8; 64 tokens, clusters of 4: 32
// columns (two CTAs per SM) 12.6, 64 columns 13.6; 16 alone 18.2.  8192 x 28672, 64
// tokens: 64 columns 33.4, 32 42.1, pair 35.3.  Not built: clusters of 8, which gained 10%
// or lost 30% as they found room on the GPU (8192 x 2048, 17 and 32 tokens), and 128
// columns, never the fastest by more than 8% (both from a timer with steps of 2 us).
struct LinForm {
  int bn;               // tokens of a tile (256: the pair form)
  double stage, last, join;
};
constexpr LinForm kForms[] = {{16, 0.27, 0.0, 1.0}, {32, 0.32, 0.0, 1.8}, {64, 0.40, 1.2, 2.4}, {256, 0.36, 4.0, 0.0}};

static LinPlan plan_linear(int64_t T, int64_t K, int64_t N, int bs, int sms) {
  LinPlan best{};
  double best_cost = -1.0;
  const int n_steps = (int)((K + kStepK - 1) / kStepK);
  for (const LinForm& f : kForms) {
    const bool pair = f.bn == 256;
    if (!pair && T > 8 * f.bn) continue;  // W would pass through L2 more than eight times
    const int64_t ta = pair ? (T + 255) / 256 : (N + 127) / 128;
    const int64_t tb = pair ? (N + 255) / 256 : (T + f.bn - 1) / f.bn;
    for (int split : {1, 2, 4}) {
      const bool two = f.bn <= 32 && ta * tb * split > sms;
      if (split > 1 && (pair || split > n_steps || ta * tb * split > (f.bn <= 32 ? 2 * sms : sms))) break;
      const int64_t slots = pair ? sms / 2 : two ? sms * 2 : sms;
      const double waves = (double)((ta * tb * split + slots - 1) / slots) * (two ? 1.4 : 1.0);
      const double cost = waves * ((n_steps + split - 1) / split) * f.stage + f.last + (split > 1 ? f.join : 0.0);
      if (best_cost < 0 || cost < best_cost) {
        best_cost = cost;
        best.bn = f.bn; best.split = split; best.two = two; best.tiles_a = ta; best.tiles_b = tb;
      }
    }
  }
  best.n_steps = n_steps;
  // a single token, quantized by every CTA for itself: no first launch.  On the device 8.1 us instead of 10.3
  // (NVFP4) and 7.8 instead of 9.7 (MXFP4) at 2560 x 9728, 9.9 instead of 10.7 at 9728 x 2560, 5.9 instead of 6.9 at
  // 2560 x 1000, and a launch less for the host.  A form of it for several tokens gained nothing from 2 on, and took 13
  // (MXFP4) and 21 us (NVFP4) for 8, where two launches take 10.3.
  best.here = best.bn == 16 && T == 1 && !best.two && (n_steps + best.split - 1) / best.split <= kHereStages;
  best.ldp = up(K, 32) / 2;
  best.gran = best.bn < 128 ? best.bn : 128;
  const int64_t sf_tiles = best.bn == 256 ? best.tiles_a * 2 : best.tiles_b;
  best.off_sf = up(T * best.ldp, 256);
  best.off_scale = best.off_sf + up(sf_tiles * n_steps * (int64_t)(kStepK / bs / 4 * kGroupBytes), 256);
  best.bytes = best.off_scale + up(T * 4, 256);
  return best;
}

struct QuantizeRows {
  const void* x;
  int dtype;
  int64_t ldx, T, K;
  uint8_t* packed;
  int64_t ldp;
  uint8_t* sf;
  int gran;
  int64_t n_steps;
  float* row_scale;
};

template <int BS, int R>
static cudaError_t launch_quantize_rows(const QuantizeRows& q, cudaStream_t st) {
  const int64_t threads = (q.n_steps * Fmt<BS>::kBlocks + R - 1) / R;
  const int64_t most = R == 1 ? 512 : 256;
  const int nt = threads >= most ? (int)most : (threads < 64 ? 64 : (int)up(threads, 32));
  const unsigned grid = (unsigned)q.T;
#define QZ_ROWS(DT)                                                                                                     \
  quantize_rows_kernel<BS, DT, R><<<grid, nt, 0, st>>>(q.x, q.ldx, q.K, q.packed, q.ldp, q.sf, q.gran, q.n_steps,       \
                                                       q.row_scale)
  if (q.dtype == kDtBF16) QZ_ROWS(kDtBF16);
  else if (q.dtype == kDtF16) QZ_ROWS(kDtF16);
  else QZ_ROWS(kDtF32);
#undef QZ_ROWS
  return cudaGetLastError();
}

template <int BN, int BS, int HERE, int CTAS>
static int launch_linear(const CUtensorMap& a, const CUtensorMap& b, const LinearParams& p, int sms, cudaStream_t st) {
  using G = LinGeo<BN, BS, (HERE >= 0), CTAS>;
  static bool attr_set[64] = {false};  // per device (a benign race: every thread sets the same value)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_kernel<BN, BS, HERE, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchAttribute at[2] = {};
  int n = 0;
  if (HERE < 0) {  // the quantization launch is before it
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.split > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n++].val.clusterDim = {(unsigned)p.split, 1, 1};
  }
  const int64_t ctas = p.tiles_a * p.tiles_b * p.split;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ctas < sms * CTAS ? ctas : sms * CTAS));
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cuda_status(cudaLaunchKernelEx(&cfg, linear_kernel<BN, BS, HERE, CTAS>, a, b, p), "linear launch");
}

template <int BS>
static int launch_pair(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, const LinearParams& p, int sms,
                       cudaStream_t st) {
  using G = PairGeo<BS>;
  static bool attr_set[64] = {false};  // per device (a benign race: every thread sets the same value)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(linear_pair_kernel<BS>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  const int64_t pairs = p.tiles_a * p.tiles_b;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(2 * (pairs < sms / 2 ? pairs : sms / 2)));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, linear_pair_kernel<BS>, a, b, o, p), "linear launch");
}

template <int BS>
static int run_linear(int bn, bool two, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, const LinearParams& p, int sms,
                      cudaStream_t st) {
  switch (bn) {
    case 16: return two ? launch_linear<16, BS, -1, 2>(a, b, p, sms, st) : launch_linear<16, BS, -1, 1>(a, b, p, sms, st);
    case 32: return two ? launch_linear<32, BS, -1, 2>(a, b, p, sms, st) : launch_linear<32, BS, -1, 1>(a, b, p, sms, st);
    case 64: return launch_linear<64, BS, -1, 1>(a, b, p, sms, st);
    default: return launch_pair<BS>(a, b, o, p, sms, st);
  }
}
template <int BS>
static int run_linear_here(int x_dtype, const CUtensorMap& a, const LinearParams& p, int sms, cudaStream_t st) {
  if (x_dtype == kDtBF16) return launch_linear<16, BS, kDtBF16, 1>(a, a, p, sms, st);
  if (x_dtype == kDtF16) return launch_linear<16, BS, kDtF16, 1>(a, a, p, sms, st);
  return launch_linear<16, BS, kDtF32, 1>(a, a, p, sms, st);
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
  if (s == QZ_OK) s = code_map(&mw, packed, (uint64_t)pl.ldp, (uint64_t)N, (uint64_t)ldp, 128);
  if (s != QZ_OK) return s;
  LinearParams p{};
  p.T = T; p.N = N;
  p.tiles_a = pl.tiles_a; p.tiles_b = pl.tiles_b;
  p.split = pl.split;
  p.n_steps = pl.n_steps;
  p.sf_a = swap ? scales : ws + pl.off_sf;
  p.sf_b = swap ? ws + pl.off_sf : scales;
  p.row_scale = reinterpret_cast<float*>(ws + pl.off_scale);
  p.w_scale = tensor_scale;
  p.bias = bias; p.bias_dtype = bias_dtype;
  p.out = out; p.out_dtype = out_dtype; p.ldo = ldo;
  p.tma_out = !swap && out_dtype != QZ_DTYPE_F32 && ldo % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  p.x = x; p.K = K;
  if (pl.here) return bs == 16 ? run_linear_here<16>(x_dtype, mw, p, sms, st) : run_linear_here<32>(x_dtype, mw, p, sms, st);
  CUtensorMap mo = mx;
  if (p.tma_out && (s = out_map(&mo, out, (uint64_t)N, (uint64_t)T, (uint64_t)ldo)) != QZ_OK) return s;
  const QuantizeRows q{x, x_dtype, ldx, T, K, ws, pl.ldp, ws + pl.off_sf, pl.gran, pl.n_steps,
                       reinterpret_cast<float*>(ws + pl.off_scale)};
  const bool few = T < 2 * sms;
  s = cuda_status(bs == 16 ? (few ? launch_quantize_rows<16, 1>(q, st) : launch_quantize_rows<16, 4>(q, st))
                           : (few ? launch_quantize_rows<32, 1>(q, st) : launch_quantize_rows<32, 2>(q, st)),
                  "quantize rows launch");
  if (s != QZ_OK) return s;
  const CUtensorMap &ma = swap ? mw : mx, &mb = swap ? mx : mw;
  return bs == 16 ? run_linear<16>(pl.bn, pl.two, ma, mb, mo, p, sms, st) : run_linear<32>(pl.bn, pl.two, ma, mb, mo, p, sms, st);
}
