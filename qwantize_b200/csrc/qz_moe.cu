// qz_moe.cu -- a whole mixture-of-experts layer for a few tokens, with the
// experts' weights in packed NVFP4 (block 16) or MXFP4 (block 32):
//
//   logits = x R^T,   S_t = the top_k largest logits of token t (ties: lowest index)
//   y_t = sum_{e in S_t} c_te D_e (silu(G_e x_t) * (U_e x_t)),   c_t = softmax over S_t
//         (or the softmax over all experts, taken at S_t)
//
// Few tokens make this a stream of weights: every chosen expert's 3 H I codes
// are read once, and the floor is their bytes over the HBM rate.  Activations
// stay in 16 bits (quantizing them would save nothing).
//
// Two launches.  moe_router_kernel, a cluster of 8 CTAs per 4 tokens: the CTAs
// share the experts' logits, send them to the CTA of their token through
// distributed shared memory, and that one chooses; it also writes the token
// as fp16 in the order of the matrix instructions' B fragments.
// moe_experts_kernel, cooperative, one CTA of 16 warps per SM: each CTA groups the
// choices by expert, then the CTAs share the units of the gate / up product; a grid
// barrier; the units of the down product; a grid barrier; the weighted sum over
// each token's experts in a fixed order.
//
// A unit is 32 weight rows of one expert times up to 16 of its tokens (more would
// be bound by the matrix instructions and gain nothing).  A CTA has a run of
// neighbouring units, so its warps share an expert's tokens in L1; a warp takes
// a unit alone and streams its weights through its own ring of bulk copies,
// never waiting for another warp.  The units that are left when every warp has had
// its share are cut along K by up to 8 warps each, which add up through shared
// memory.
//
// Weights are laid out once in the order of the A fragments of mma.m16n8k16
// (fp16, fp32 accumulation): a lane's 16 bytes hold its 4 steps of one 16-row
// tile and 64-column chunk.  The codes convert exactly to fp16 by hardware; an
// NVFP4 scale (one per step) is multiplied in there, exactly (6 significant
// bits, 2^-10 .. 2688), an MXFP4 scale (one per two steps, any power of two)
// multiplies the fp32 partial product.  A gate / up tile interleaves 8 gate rows
// with the 8 up rows of the same outputs, so a lane holds both and the
// activation function needs no exchange.  tcgen05 would need 128 weight rows per
// instruction and 16-bit operands in shared memory; with 1 to 32 tokens per expert
// the matrix work is a tenth of what mma.sync can do while HBM delivers the codes.
//
// Measured, router and experts: 1 token, 8 of 128 experts of 2048 x 768, NVFP4: 8.9
// and 22.9 us (21 MB; latency of launches, routing and barriers); 64 tokens, 8 of 64
// of 2560 x 1280: 10.3 and 111 us (354 MB, 3.2 TB/s).  There a warp spends about 120
// instructions on a chunk of 64 columns, half of them on unpacking and scaling,
// and four warps per scheduler cover the latencies between them to 43% of the
// issue slots; more warps leave too few registers (12, 16, 20 and 24 were tried).
//
// fp16 operands: a bf16 token is scaled by the power of two that puts its
// largest magnitude in [2^14, 2^15), exact for values within 2^-28 of it.  An
// activation row is scaled by a power of two from the bound |silu(g) u| <= |g| |u|
// <= |x|^2 max(|G row| |U row|) over its outputs (kept with the weights), so it cannot
// overflow whatever the data, and rounded to 11 bits, or to 2^-40 of the bound where
// that is more; for fp16 outputs, whose own rounding is no coarser, the remainder is
// kept as a second fp16 operand.  The largest activation of normal data lies near
// 2^-14 of the bound; where a token's norm comes from a channel that the weights
// suppress, it lies lower, and the first bit goes at about 2^-26 (a channel 10,000
// times the others, its weights as much smaller; at 100,000 seven bits are left).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/qwantize_b200.h"
#include "qz_common.cuh"
#include "qz_kernels.h"
#include "qz_moe_walk.cuh"
#include "qz_ptx.cuh"
#include "qz_tc.cuh"

namespace qz {

int fail(int code, const char* fmt, ...);
int cuda_status(cudaError_t e, const char* what);
int current_sms(int* sms);

constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTop = 16;
constexpr int kMoeThreads = kMoeWarps * 32;
constexpr int kMoeMaxSlots = kMoeMaxTokens * kMoeMaxTop;
constexpr int kMoeGroup = 16;                                                  // tokens of a unit
constexpr int kMoeMaxGroups = kMoeMaxExperts + kMoeMaxSlots / kMoeGroup;
constexpr int kMoeStages = 2;                                                  // copies in flight per warp

struct MoeParams {
  int T, H, I, E, top;
  int hc, ic;                       // 64-column chunks of H and I
  int dtype;                        // of x and out
  const int* choice;                // (T, top) experts
  const float* choice_weight;       // (T, top)
  const uint8_t *up_codes, *up_scales;      // (E, I / 16 units, hc chunks, 2 tiles) 512 and 8 * 2 * 64 / bs bytes
  const uint8_t *down_codes, *down_scales;  // (E, H / 32 units, ic chunks, 2 tiles)
  const float* norms;               // (E, 2): factors of the bound of |G row| |U row|, without the tensor scale
  float up_scale, down_scale;       // tensor scales
  const __half* xh;                 // (T, hc, 64) in fragment order
  const int2* xp;                   // (T): power of two of the token, exponent bound of its scaled squared norm
  __half* act;                      // (parts, T * top, ic, 64) in fragment order: the rounded row, then the remainder
  int64_t act_part;                 // elements of one part
  float* y;                         // (T * top, H)
  int* barrier;
  void* out;                        // (T, H)
};

// ---------------------------------------------------------------------------
// weights to fragment order
// ---------------------------------------------------------------------------
// Lane (g, t) of a 16-row tile and 64-column chunk: word j (one mma step, 16
// columns) holds columns 16j + 4t .. + 3 of row g (low half) and row g + 8 (high
// half).  gate_up: rows 0-7 of tile i are gate rows 8i .., rows 8-15 the up rows
// rows / 2 + 8i ...  Scales: those of row g and row g + 8 side by side.  A chunk's
// two tiles of a unit are neighbours.
template <int BS>
__global__ void moe_layout_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales, int64_t E,
                                  int64_t rows, int64_t K, int gate_up, uint32_t* __restrict__ codes_out,
                                  uint8_t* __restrict__ scales_out) {
  const int64_t chunks = (K + 63) / 64, tiles = rows / 16;
  const int64_t total = E * tiles * chunks * 128;  // words
  constexpr int kSc = 64 / BS;                     // scales per row and chunk
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int j = i & 3, lane = (int)(i >> 2) & 31, g = lane >> 2, t = lane & 3;
    const int64_t chunk = i / 256 % chunks, unit = i / 256 / chunks % (tiles / 2), e = i / 256 / chunks / (tiles / 2);
    const int64_t tile = unit * 2 + (i / 128 & 1);
    const int64_t col = chunk * 64 + 16 * j + 4 * t;
    uint32_t w = 0;
    for (int h = 0; h < 2; ++h) {
      const int64_t row = gate_up ? (h ? rows / 2 : 0) + tile * 8 + g : tile * 16 + h * 8 + g;
      const uint8_t* p = packed + (e * rows + row) * (K / 2) + col / 2;
      if (col < K) w |= ((uint32_t)p[0] | (uint32_t)p[1] << 8) << (16 * h);
      if (j == 0 && t < kSc) {  // lane t < kSc of the quad writes scale t of both rows
        const int64_t b = chunk * kSc + t;
        scales_out[((i / 128 * 8 + g) * 2 + h) * kSc + t] =
            b < K / BS ? scales[(e * rows + row) * (K / BS) + b] : 0;
      }
    }
    codes_out[i] = w;
  }
}

// A bound of every output's |G row| |U row|, a warp per pair of rows: the largest sum of
// the two norms' exponent bounds (the row of one output and the row of another do not
// meet, so neither do their norms), as whole numbers in the first word of `norms`.
// Rows of zeros and rows that are not finite count for nothing: their activations are
// zero, or spoil the token whatever its scale.
template <int BS>
__global__ void moe_bound_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales, int64_t E, int64_t rows,
                                 int64_t K, int* __restrict__ norms) {
  const int lane = threadIdx.x & 31;
  const int64_t n_warps = (int64_t)gridDim.x * (blockDim.x >> 5), outputs = rows / 2;
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < E * outputs; i += n_warps) {
    int both = 0;
    bool counts = true;
    for (int h = 0; h < 2; ++h) {
      const int64_t r = i / outputs * rows + h * outputs + i % outputs;
      double sum = 0.0;
      for (int64_t b = lane; b < K / BS; b += 32) {
        const uint32_t c = scales[r * (K / BS) + b];
        const float s = BS == 32 ? (c == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(c == 0 ? 0x00400000u : c << 23))
                      : c == 127 ? __uint_as_float(0x7fffffffu) : e4m3_value((int)c);
        float q2 = 0.0f;
        for (int k = 0; k < BS / 2; ++k) {
          const float2 v = e2m1x2_to_float2(packed[r * (K / 2) + b * (BS / 2) + k]);
          q2 += v.x * v.x + v.y * v.y;
        }
        sum += (double)q2 * s * s;  // an MXFP4 scale's square does not fit in fp32
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (sum > 0.0 && isfinite(sum)) both += ilogb(sqrt(sum)) + 1;
      else counts = false;
    }
    if (lane == 0 && counts) atomicMax(norms + i / outputs * 2, both);
  }
}
// ... as two powers of two whose exponent bounds add up to it.
__global__ void moe_factors_kernel(float2* norms, int64_t E) {
  const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (e >= E) return;
  // below (2^-126)^2 nothing is left of an activation in fp32
  const int both = min(max(__float_as_int(norms[e].x), -250), 256), half = both >> 1;
  norms[e] = make_float2(ldexpf(1.0f, half - 1), ldexpf(1.0f, both - half - 1));
}

// ---------------------------------------------------------------------------
// router logits, fp16 tokens
// ---------------------------------------------------------------------------
// 8 consecutive elements as fp32.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  if (DT == kDtF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = DT == kDtBF16 ? bf16_bits_to_float(ww[k] & 0xffffu) : f16_bits_to_float(ww[k] & 0xffffu);
    v[2 * k + 1] = DT == kDtBF16 ? bf16_bits_to_float(ww[k] >> 16) : f16_bits_to_float(ww[k] >> 16);
  }
}

// e with x * 2^-e in [2^14, 2^15) for the largest magnitude (its bits m); 0
// for 0, inf and NaN
__device__ __forceinline__ int f16_power(uint32_t m) {
  if (m == 0 || m >= 0x7f800000u) return 0;
  const int e = (int)(m >> 23) - 127 - 14;
  return e < -112 ? -112 : e;
}

// Smallest e with |v| < 2^e for a finite v > 0 (a bound of its exponent); 0 else
__device__ __forceinline__ int exponent_bound(float v) {
  const uint32_t u = __float_as_uint(v);
  return v > 0.0f && u < 0x7f800000u ? (int)(u >> 23) - 126 : 0;
}

// Ascending order of the bits is ascending order of the floats, NaN on top;
// never 0.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The top_k largest of a token's logits, by one warp: lane l holds experts W l .. W
// l + W - 1, so the lowest index among equal logits is in the lowest lane.
template <int W>
__device__ __forceinline__ void choose(const float* logits, int E, int top, int renorm, int* ids, float* weights) {
  const int lane = threadIdx.x & 31;
  uint32_t key[W];  // 0: not there, or taken
  auto logit = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); };
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    key[i] = lane * W + i < E ? order_bits(logits[lane * W + i]) : 0u;
    m = max(m, key[i]);
  }
  const float best = logit(__reduce_max_sync(0xffffffffu, m));
  float sum = 0.0f;
  if (!renorm)
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (key[i]) sum += expf(logit(key[i]) - best);
  uint32_t chosen = 0;  // lane k keeps choice k
  int mine = 0;
#pragma unroll 1
  for (int k = 0; k < top; ++k) {
    m = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) m = max(m, key[i]);
    const uint32_t most = __reduce_max_sync(0xffffffffu, m);
    const int src = __ffs(__ballot_sync(0xffffffffu, m == most)) - 1;
    int at = 0;
#pragma unroll
    for (int i = W - 1; i >= 0; --i)
      if (key[i] == most) at = i;
    if (lane == src) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i == at) key[i] = 0;
    }
    at = __shfl_sync(0xffffffffu, at, src);
    if (lane == k) { chosen = most; mine = src * W + at; }
  }
  const float e = lane < top ? expf(logit(chosen) - best) : 0.0f;
  if (renorm) sum = e;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane < top) {
    ids[lane] = mine;
    weights[lane] = __fdiv_rn(e, sum);
  }
}

// A cluster of kRouterCtas CTAs has up to kRouterTokens tokens: CTA r computes the
// logits of every kRouterCtas-th expert for all of them and owns token r.
constexpr int kRouterCtas = 8, kRouterTokens = 4, kRouterThreads = 512;
template <int DT, int RDT, int NTK>  // NTK: tokens of a cluster
__global__ void __cluster_dims__(kRouterCtas, 1, 1) __launch_bounds__(kRouterThreads)
    moe_router_kernel(const void* __restrict__ x, int64_t ldx, const void* __restrict__ router, int T, int H, int E, int top,
                      int renorm, int* __restrict__ ids, float* __restrict__ weights, uint4* __restrict__ xh,
                      int2* __restrict__ xp, int* __restrict__ barrier) {
  constexpr int kWarps = kRouterThreads / 32;
  __shared__ float s_logits[kMoeMaxExperts];
  __shared__ float s_part[kWarps][NTK];
  __shared__ float s_norm[kRouterThreads / 32];
  __shared__ uint32_t s_max[kRouterThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % kRouterCtas, t0 = blockIdx.x / kRouterCtas * NTK;
  const int nt = T - t0 < NTK ? T - t0 : NTK, t = rank < nt ? t0 + rank : T;  // T: no token
  if (blockIdx.x == 0 && tid < 2) barrier[tid] = 0;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // every CTA has begun before another writes to it
  // warps per expert of this CTA, so that all are busy: they split H
  const int mine = (E - rank + kRouterCtas - 1) / kRouterCtas;
  int cut = 1;
  while (cut < kWarps && mine * cut * 2 <= kWarps) cut *= 2;
  for (int i0 = 0; i0 < mine; i0 += kWarps / cut) {
    const int i = i0 + warp / cut, e = rank + i * kRouterCtas;
    float acc[NTK] = {};
    if (i < mine) {
#pragma unroll(NTK == 1 ? 8 : 2)
      for (int h = (warp % cut * 32 + lane) * 8; h < H; h += cut * 256) {
        float r[8];
        uint4 raw[NTK];  // all loads before the first product
        load8<RDT>(router, (int64_t)e * H + h, r);
#pragma unroll
        for (int n = 0; n < NTK; ++n)
          raw[n] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + (t0 + (n < nt ? n : 0)) * ldx + h));
#pragma unroll
        for (int n = 0; n < NTK; ++n) {
          const uint32_t ww[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            acc[n] = fmaf(DT == kDtBF16 ? bf16_bits_to_float(ww[k] & 0xffffu) : f16_bits_to_float(ww[k] & 0xffffu), r[2 * k], acc[n]);
            acc[n] = fmaf(DT == kDtBF16 ? bf16_bits_to_float(ww[k] >> 16) : f16_bits_to_float(ww[k] >> 16), r[2 * k + 1], acc[n]);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NTK; ++n) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[n] += __shfl_xor_sync(0xffffffffu, acc[n], o);
      if (lane == 0) s_part[warp][n] = acc[n];
    }
    __syncthreads();
    if (i0 == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    // thread (expert, token): the parts in order, to the token's CTA
    if (tid < kWarps / cut * NTK) {
      const int j = tid / NTK, n = tid % NTK;
      if (i0 + j < mine && n < nt) {
        float v = 0.0f;
        for (int q = 0; q < cut; ++q) v += s_part[j * cut + q][n];
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(s_logits + rank + (i0 + j) * kRouterCtas)), "r"(n));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
      }
    }
    __syncthreads();
  }
  if (mine <= 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  // this CTA's token as fp16
  int e = 0;
  if (DT == kDtBF16 && t < T) {
    uint32_t m = 0;
    for (int h = tid * 8; h < H; h += kRouterThreads * 8) {
      float v[8];
      load8<DT>(x, t * ldx + h, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
    m = s_max[lane % (kRouterThreads / 32)];
    e = f16_power(__reduce_max_sync(0xffffffffu, m));
  }
  const float inv = pow2f(-e);
  const int hc = (H + 63) / 64;
  float norm2 = 0.0f;
  if (t < T) {
    // thread: 8 halves; lane t' of the fragment takes columns 4t' .. + 3 of two blocks of 16
    for (int i = tid; i < hc * 8; i += kRouterThreads) {
      const int col = (i >> 2) * 32 + (i & 3) * 4;  // and 16 further
      uint32_t w[4] = {0, 0, 0, 0};
      if (col < H) {  // H is a multiple of 32
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint2 raw = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(x) + t * ldx + col + 16 * k));
          const uint32_t rr[2] = {raw.x, raw.y};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float a = (DT == kDtBF16 ? bf16_bits_to_float(rr[q] & 0xffffu) : f16_bits_to_float(rr[q] & 0xffffu)) * inv;
            const float b = (DT == kDtBF16 ? bf16_bits_to_float(rr[q] >> 16) : f16_bits_to_float(rr[q] >> 16)) * inv;
            norm2 = fmaf(a, a, fmaf(b, b, norm2));
            const __half2 h = __floats2half2_rn(a, b);
            w[2 * k + q] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
      }
      xh[(int64_t)t * hc * 8 + i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) norm2 += __shfl_xor_sync(0xffffffffu, norm2, o);
  if (lane == 0) s_norm[warp] = norm2;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (t >= T) return;
  if (warp == 0) {
    int* id = ids + (int64_t)t * top;
    float* w = weights + (int64_t)t * top;
    if (E <= 32) choose<1>(s_logits, E, top, renorm, id, w);
    else if (E <= 64) choose<2>(s_logits, E, top, renorm, id, w);
    else if (E <= 128) choose<4>(s_logits, E, top, renorm, id, w);
    else choose<kMoeMaxExperts / 32>(s_logits, E, top, renorm, id, w);
  } else if (tid == 32) {
    float sum = 0.0f;
    for (int i = 0; i < kRouterThreads / 32; ++i) sum += s_norm[i];
    xp[t] = make_int2(e, exponent_bound(sum));
  }
}

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------
struct MoeShared {
  float weight[kMoeMaxSlots];
  uint16_t id[kMoeMaxSlots], rank[kMoeMaxSlots];  // a slot's expert, its place among the expert's slots
  uint16_t list[kMoeMaxSlots];            // slots (token * top + k) grouped by expert, tokens ascending
  uint16_t count[kMoeMaxExperts];
  uint16_t start[kMoeMaxExperts];
  // groups: up to kMoeGroup tokens of one expert, experts ascending
  uint16_t g_expert[kMoeMaxGroups], g_begin[kMoeMaxGroups], g_count[kMoeMaxGroups];
  uint16_t g_cost[kMoeMaxGroups + 1];     // cost of one unit of each group before this one
  int n_groups, ok;
  int bound[4];                           // this CTA's first unit and the one behind its last: gate / up, down
  uint64_t full[kMoeWarps * kMoeStages];  // the warps' rings
  float x_scale[kMoeMaxTokens];           // power of two of a token times the tensor scale
  int16_t act_exp[kMoeMaxSlots];          // e: |activation| of the slot < 2^(e + 15)
  float part[kMoeWarps][16 * 32];         // sums of warps that share a unit: (value, lane)
};

// All CTAs arrive, then wait for each other (they are all resident: cooperative
// launch).  Bounded: on timeout the error flag is set and the kernel ends.
__device__ __forceinline__ bool grid_barrier(int* counter, MoeShared& s) {
  __syncthreads();  // one thread's release and acquire stand for the CTA's
  if (threadIdx.x == 0) {
    int ok = 1;
    asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(counter) : "memory");
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
      int v;
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
      if (v >= (int)gridDim.x) break;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        atomicOr(&qz_device_error, kDevErrEpilogueTimeout);
        ok = 0;
        break;
      }
    }
    s.ok = ok;
  }
  __syncthreads();
  return s.ok != 0;
}

// Relative time of a unit with one or two tiles of 8 tokens: a chunk's unpacking is
// shared, its products are not.  Microseconds with 1:1, 4:5, 5:7, 2:3, 64 tokens: 8 of 64
// experts of 2560 x 1280, NVFP4: 120, 109, 111, 115 (fp16: 144, 130, 129, 131), MXFP4: 144,
// 134, 138, 147; 8 of 128 of 2048 x 768, NVFP4: 116, 105, 100, 102 (fp16: 142, 125, 115, 113).
// Up to 32 tokens all are alike.
__device__ __forceinline__ int unit_cost(int tokens) { return tokens <= 8 ? 5 : 7; }

__device__ __forceinline__ void route(const MoeParams& p, MoeShared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = p.T * p.top;
  for (int i = threadIdx.x; i < n; i += kMoeThreads) {
    s.id[i] = (uint16_t)__ldg(p.choice + i);
    s.weight[i] = __ldg(p.choice_weight + i);
  }
  __syncthreads();
  // asked for here, used at the end
  constexpr int kPer = kMoeMaxSlots / kMoeThreads;
  int2 xp[kPer];
  float2 norm[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = k * kMoeThreads + threadIdx.x;
    if (i < n) {
      xp[k] = __ldg(p.xp + i / p.top);
      norm[k] = __ldg(reinterpret_cast<const float2*>(p.norms) + s.id[i]);
    }
  }
  // a warp numbers the slots of every kMoeWarps-th expert in ascending order
  {
    uint16_t ids[kMoeMaxSlots / 32];
#pragma unroll
    for (int i = 0; i < kMoeMaxSlots / 32; ++i) ids[i] = i * 32 + lane < n ? s.id[i * 32 + lane] : (uint16_t)0xffffu;
#pragma unroll 1
    for (int e = warp; e < p.E; e += kMoeWarps) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kMoeMaxSlots / 32; ++i) {
        if (i * 32 >= n) break;
        const unsigned same = __ballot_sync(0xffffffffu, ids[i] == e);
        if (ids[i] == e) s.rank[i * 32 + lane] = (uint16_t)(c + __popc(same & ((1u << lane) - 1u)));
        c += __popc(same);
      }
      if (lane == 0) s.count[e] = (uint16_t)c;
    }
  }
  __syncthreads();
  // one warp lays out the groups
  if (warp == 0) {
    int at = 0, groups = 0, cost = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int c = e0 + lane < p.E ? s.count[e0 + lane] : 0, m = (c + kMoeGroup - 1) / kMoeGroup;
      const int z = m == 0 ? 0 : (m - 1) * unit_cost(kMoeGroup) + unit_cost(c - (m - 1) * kMoeGroup);
      // inclusive prefix sums of the three in one word: slots <= 1024, groups <= 128, cost <= 896
      static_assert(kMoeMaxSlots <= 1024 && kMoeMaxTokens <= 4 * kMoeGroup, "fields of the word");
      unsigned sums = (unsigned)c | (unsigned)m << 11 | (unsigned)z << 20;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += x;
      }
      const int a = sums & 2047, b = sums >> 11 & 511, d = sums >> 20;
      if (e0 + lane < p.E) s.start[e0 + lane] = (uint16_t)(at + a - c);
      for (int k = 0; k < m; ++k) {
        const int g = groups + b - m + k;
        s.g_expert[g] = (uint16_t)(e0 + lane);
        s.g_begin[g] = (uint16_t)(at + a - c + k * kMoeGroup);
        s.g_count[g] = (uint16_t)(c - k * kMoeGroup < kMoeGroup ? c - k * kMoeGroup : kMoeGroup);
        s.g_cost[g] = (uint16_t)(cost + d - z + k * unit_cost(kMoeGroup));
      }
      sums = __shfl_sync(0xffffffffu, sums, 31);
      at += sums & 2047;
      groups += sums >> 11 & 511;
      cost += sums >> 20;
    }
    if (lane == 0) {
      s.n_groups = groups;
      s.g_cost[groups] = (uint16_t)cost;
    }
    __syncwarp();
    if (lane < 4) {
      // the first unit at or behind this CTA's (the next one's) share of the phase's cost
      const int units = lane < 2 ? p.I / 16 : p.H / 32;
      const int64_t at = (int64_t)cost * units * (blockIdx.x + (lane & 1)) / gridDim.x;
      int lo = 0, hi = groups;  // last group that begins at or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)s.g_cost[mid] * units <= at) lo = mid; else hi = mid;
      }
      const int one = s.g_cost[lo + 1] - s.g_cost[lo];
      s.bound[lane] = lo * units + ((int)(at - (int64_t)s.g_cost[lo] * units) + one - 1) / one;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = k * kMoeThreads + threadIdx.x;
    if (i >= n) break;
    s.list[s.start[s.id[i]] + s.rank[i]] = (uint16_t)i;
    const int bound = xp[k].y + 2 * xp[k].x + exponent_bound(norm[k].x) + exponent_bound(norm[k].y) + 2 * exponent_bound(fabsf(p.up_scale)) - 15;
    s.act_exp[i] = (int16_t)min(max(bound, -140), 113);  // an fp32 activation is below 2^128; below 2^-125 nothing is left
    if (i % p.top == 0) s.x_scale[i / p.top] = pow2f(xp[k].x) * p.up_scale;
  }
  __syncthreads();
}

__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, __half2 b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four E4M3 scales of a word as fp16 pairs (s, s) (the multiplication reads one half twice).
__device__ __forceinline__ void scales_nv(uint32_t w, __half2 (&s)[4]) {
  uint32_t h0, h1;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(h0), "=r"(h1)
      : "r"(w));
  const __half2 x = *reinterpret_cast<const __half2*>(&h0), y = *reinterpret_cast<const __half2*>(&h1);
  s[0] = __low2half2(x);
  s[1] = __high2half2(x);
  s[2] = __low2half2(y);
  s[3] = __high2half2(y);
}
__device__ __forceinline__ float scale_mx(uint32_t c) {
  return __uint_as_float(c == 0 ? 0x00400000u : c == 255 ? 0x7fffffffu : c << 23);
}

// One chunk (64 columns) of a unit: two 16-row tiles of weights in shared memory
// (a lane's 16 bytes of each, its rows' scales) times NT tiles of 8 tokens, whose
// B words come in `PARTS` addends.
template <int NT, int BS, int PARTS>
__device__ __forceinline__ void chunk_product(const uint8_t* codes, const uint8_t* scales, const uint32_t (&b)[PARTS][NT][8],
                                              float (&acc)[2][NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
  uint32_t w[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint4 w4 = *reinterpret_cast<const uint4*>(codes + r * 512 + lane * 16);
    w[r][0] = w4.x; w[r][1] = w4.y; w[r][2] = w4.z; w[r][3] = w4.w;
  }
  // the two tiles side by side: their chains of conversions and products are independent
  if constexpr (BS == 16) {
    __half2 s0[2][4], s1[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint2 sc = *reinterpret_cast<const uint2*>(scales + r * 64 + g * 8);
      scales_nv(sc.x, s0[r]);
      scales_nv(sc.y, s1[r]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[2][4];  // row g, columns 0-1 and 2-3; row g + 8
#pragma unroll
      for (int r = 0; r < 2; ++r) e2m1x8_to_f16(w[r][j], a[r]);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        a[r][0] = mul_f16x2(a[r][0], s0[r][j]);
        a[r][1] = mul_f16x2(a[r][1], s0[r][j]);
        a[r][2] = mul_f16x2(a[r][2], s1[r][j]);
        a[r][3] = mul_f16x2(a[r][3], s1[r][j]);
      }
#pragma unroll
      for (int q = 0; q < PARTS; ++q)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) mma_f16(acc[r][n], a[r][0], a[r][2], a[r][1], a[r][3], b[q][n][2 * j], b[q][n][2 * j + 1]);
    }
  } else {
    uint32_t sc[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) sc[r] = *reinterpret_cast<const uint32_t*>(scales + r * 32 + g * 4);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      float d[2][NT][4];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) d[r][n][0] = d[r][n][1] = d[r][n][2] = d[r][n][3] = 0.0f;
#pragma unroll
      for (int k = j; k < j + 2; ++k) {
        uint32_t a[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) e2m1x8_to_f16(w[r][k], a[r]);
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) mma_f16(d[r][n], a[r][0], a[r][2], a[r][1], a[r][3], b[q][n][2 * k], b[q][n][2 * k + 1]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float s0 = scale_mx(sc[r] >> (4 * j) & 255u), s1 = scale_mx(sc[r] >> (16 + 4 * j) & 255u);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[r][n][0] = fmaf(d[r][n][0], s0, acc[r][n][0]);
          acc[r][n][1] = fmaf(d[r][n][1], s0, acc[r][n][1]);
          acc[r][n][2] = fmaf(d[r][n][2], s1, acc[r][n][2]);
          acc[r][n][3] = fmaf(d[r][n][3], s1, acc[r][n][3]);
        }
      }
    }
  }
}

// The weighted results of token t's experts, columns 4 h .. + 3, added in order and rounded once.
__device__ __forceinline__ void add_experts(const MoeParams& p, int t, int h) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int k = 0; k < p.top; ++k) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p.y + (int64_t)(t * p.top + k) * p.H) + h);
    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
  }
  uint32_t lo, hi;
  if (p.dtype == kDtBF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(v.y), "f"(v.x));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(v.w), "f"(v.z));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(v.y), "f"(v.x));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(v.w), "f"(v.z));
  }
  reinterpret_cast<uint2*>(p.out)[(int64_t)t * (p.H / 4) + h] = make_uint2(lo, hi);
}

// The ring of one warp: pieces of up to kMoePiece chunks.
template <int BS>
struct MoeRing {
  static constexpr int kCodes = 1024, kScales = 1024 * 2 / BS;  // bytes per chunk
  static constexpr int kStage = kMoePiece * (kCodes + kScales);
  static constexpr int kBytes = kMoeWarps * kMoeStages * kStage;
};

// `warps` neighbouring warps wait for each other at barrier `id`: whether all are well.
__device__ __forceinline__ bool meet(bool ok, int id, int warps) {
  uint32_t go = ok ? 1u : 0u;
  asm volatile(
      "{\n .reg .pred a, b;\n setp.ne.u32 a, %0, 0;\n barrier.cta.red.and.aligned.pred b, %1, %2, a;\n selp.u32 %0, 1, 0, b;\n}\n"
      : "+r"(go)
      : "r"(id), "r"(warps * 32)
      : "memory");
  return go != 0;
}

// One phase: every group times its units.  UP: gate / up and the activation from
// x; else: down from the activations (in PARTS addends), weighted.
// ready: called once when the first copies are on their way, waits for the
// phase's other operand.
template <int BS, bool UP, int PARTS, class Ready>
__device__ __forceinline__ bool run_phase(const MoeParams& p, MoeShared& s, uint8_t* ring, uint32_t& it, Ready ready) {
  using R = MoeRing<BS>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint8_t* codes = UP ? p.up_codes : p.down_codes;
  const uint8_t* scales = UP ? p.up_scales : p.down_scales;
  const int units = UP ? p.I / 16 : p.H / 32, chunks = UP ? p.hc : p.ic;
  MoeWalk w(s.bound + (UP ? 0 : 2), units, chunks, warp), ahead = w;
  uint8_t* mine = ring + warp * kMoeStages * R::kStage;
  uint64_t* full = s.full + warp * kMoeStages;
  int64_t at_unit = 0;  // first chunk of the unit that is loaded
  auto locate = [&]() {
    if (!ahead.done()) at_unit = ((int64_t)s.g_expert[ahead.group] * units + ahead.unit) * chunks;
  };
  auto issue = [&](uint32_t i) {  // one lane: the piece at `ahead` into stage i % kMoeStages
    const int st = i % kMoeStages, n = ahead.piece();
    const int64_t chunk = at_unit + ahead.c;
    mbar_arrive_expect_tx(full + st, n * (R::kCodes + R::kScales));
    bulk_load(mine + st * R::kStage, codes + chunk * R::kCodes, n * R::kCodes, full + st);
    bulk_load(mine + st * R::kStage + kMoePiece * R::kCodes, scales + chunk * R::kScales, n * R::kScales, full + st);
  };
  locate();
  uint32_t issued = it;
  for (int k = 0; k < kMoeStages && !ahead.done(); ++k, ++issued) {
    if (elect_one()) issue(issued);
    __syncwarp();
    if (ahead.advance()) locate();
  }
  bool ok = ready();
  auto unit_of = [&](auto nt_tag) {
    constexpr int NT = decltype(nt_tag)::value;
    const int u = w.unit, count = s.g_count[w.group], share = w.whole ? 1 : w.share, part = w.part;
    const uint16_t* slots = s.list + s.g_begin[w.group];
    // this lane's B rows: token g of each tile of 8 (rows beyond the count repeat the last)
    const uint4* row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int i = n * 8 + g, slot = slots[i < count ? i : count - 1];
      row[n] = reinterpret_cast<const uint4*>(UP ? p.xh + (int64_t)(slot / p.top) * p.hc * 64 : p.act + (int64_t)slot * p.ic * 64) + t;
    }
    float acc[2][NT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][n][c] = 0.0f;
    // the B words of chunk c
    auto load_b = [&](uint32_t(&b)[PARTS][NT][8], int c) {
#pragma unroll
      for (int q = 0; q < PARTS; ++q)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4* from = row[n] + (UP ? 0 : q * (p.act_part / 8)) + c * 8;
          const uint4 lo = UP ? __ldg(from) : *from, hi = UP ? __ldg(from + 4) : from[4];
          b[q][n][0] = lo.x; b[q][n][1] = lo.y; b[q][n][2] = lo.z; b[q][n][3] = lo.w;
          b[q][n][4] = hi.x; b[q][n][5] = hi.y; b[q][n][6] = hi.z; b[q][n][7] = hi.w;
        }
    };
    // the B words are asked for kAhead chunks before their product, as far as registers allow (0: at once)
    constexpr int kAhead = NT * PARTS == 1 ? 2 : NT * PARTS == 2 ? 1 : 0, kBuffers = kAhead ? kAhead : 1;
    static_assert(kMoePiece % kBuffers == 0, "a piece begins with the first buffer");
    uint32_t b[kBuffers][PARTS][NT][8];
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
      if (w.c + d < w.c1) load_b(b[d], w.c + d);
    bool more = true;
    while (more) {
      const int st = it % kMoeStages, pieces = w.piece();
      if (!mbar_wait_warp(full + st, it / kMoeStages & 1, kDevErrLoadTimeout)) { ok = false; break; }
      const uint8_t* at = mine + st * R::kStage;
#pragma unroll 1
      for (int k = 0; k < pieces; k += kBuffers) {
#pragma unroll
        for (int d = 0; d < kBuffers; ++d) {
          if (k + d >= pieces) break;
          if (kAhead == 0) load_b(b[d], w.c + k + d);
          chunk_product<NT, BS, PARTS>(at + (k + d) * R::kCodes, at + kMoePiece * R::kCodes + (k + d) * R::kScales, b[d], acc);
          if (kAhead != 0 && w.c + k + d + kAhead < w.c1) load_b(b[d], w.c + k + d + kAhead);
        }
      }
      __syncwarp();  // every lane has read the stage
      if (!ahead.done()) {
        if (elect_one()) issue(issued);
        __syncwarp();
        if (ahead.advance()) locate();
        ++issued;
      }
      ++it;
      more = !w.advance();
    }
    if (share > 1) {
      // the unit's warps meet twice: sums written, sums read (a warp whose copy did
      // not come takes the others with it)
      float* mem = s.part[warp];
      if (part > 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) mem[((r * NT + n) * 4 + c) * 32 + lane] = acc[r][n][c];
      }
      w.met = true;
      ok = meet(ok, 1 + warp / share, share);
      if (!ok) return;
      if (part == 0) {
        for (int q = 1; q < share; ++q)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[r][n][c] += s.part[warp + q][((r * NT + n) * 4 + c) * 32 + lane];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / share), "r"(share * 32) : "memory");
      if (part > 0) return;
    }
    if (!ok) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = n * 8 + 2 * t + c;
        if (i >= count) continue;
        const int slot = slots[i], e = s.act_exp[slot], e1 = e / 2;
        if constexpr (UP) {
          const float f = s.x_scale[slot / p.top], q1 = pow2f(-e1), q2 = pow2f(e1 - e);  // 2^-e in two factors
          // column 16 u + 8 r + g: block j = u % 4 of its chunk, lane (8 r + g) / 4 of the fragment
          const int j = u & 3;
          __half* to = p.act + ((int64_t)slot * p.ic + (u >> 2)) * 64 + (j >> 1) * 32 + (g >> 2) * 8 + (j & 1) * 4 + (g & 3);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float gate = acc[r][n][c] * f, up = acc[r][n][c + 2] * f;
            // Gate far below 0: the exponential overflows and the quotient is -0.  The fast exponential is off by
            // |gate| 2^-24 of itself, which moves the activation by 1.3 2^-24 |up| at most, the fast quotient by 2^-22
            // of itself: nothing beside the 11 bits that bf16 tokens keep, as much as the 22 of fp16 tokens.
            const float v = __fdividef(gate, 1.0f + __expf(-gate)) * up * q1 * q2;
            const __half hi = __float2half_rn(v);
            to[r * 16] = hi;
            if (p.dtype == kDtF16) to[r * 16 + p.act_part] = __float2half_rn(v - __half2float(hi));
            if (u + 1 == units && (units & 3))  // the other half of the last chunk is padding
              for (int q = 0; q < 2; ++q) {
                __half* pad = to + r * 16 + 32 - (j & 1) * 4 + q * 4;
                *pad = __float2half_rn(0.0f);
                if (p.dtype == kDtF16) pad[p.act_part] = __float2half_rn(0.0f);
              }
          }
        } else {
          const float f = p.down_scale * s.weight[slot], q1 = pow2f(e1), q2 = pow2f(e - e1);
          float* to = p.y + (int64_t)slot * p.H + u * 32 + g;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            to[r * 16] = acc[r][n][c] * q1 * q2 * f;
            to[r * 16 + 8] = acc[r][n][c + 2] * q1 * q2 * f;
          }
        }
      }
  };
  while (ok && !w.done()) {
    if (s.g_count[w.group] <= 8) unit_of(std::integral_constant<int, 1>());
    else unit_of(std::integral_constant<int, 2>());
  }
  if (!ok && w.owes_meeting()) meet(false, 1 + warp / w.share, w.share);
  if (!ok)  // copies in flight must land before the CTA exits (bounded)
    for (; it < issued; ++it) mbar_wait_bounded(full + it % kMoeStages, it / kMoeStages & 1, kDevErrLoadTimeout);
  return ok;
}

template <int BS, int PARTS>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_experts_kernel(const __grid_constant__ MoeParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  MoeShared& s = *reinterpret_cast<MoeShared*>(ring + MoeRing<BS>::kBytes);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMoeWarps * kMoeStages; ++i) mbar_init(s.full + i, 1);
    fence_barrier_init();
  }
  route(p, s);
  uint32_t it = 0;  // pieces this warp has consumed
  run_phase<BS, true, 1>(p, s, ring, it, [] { return true; });
  run_phase<BS, false, PARTS>(p, s, ring, it, [&] { return grid_barrier(p.barrier, s); });
  if (!grid_barrier(p.barrier + 1, s)) return;
  const int h4 = p.H / 4;
  for (int i = blockIdx.x * kMoeThreads + threadIdx.x; i < p.T * h4; i += gridDim.x * kMoeThreads) add_experts(p, i / h4, i % h4);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
cudaError_t read_device_error_moe(unsigned* out, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(out, qz_device_error, sizeof(unsigned));
  if (e != cudaSuccess || !clear) return e;
  unsigned zero = 0;
  return cudaMemcpyToSymbol(qz_device_error, &zero, sizeof(unsigned));
}

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

struct MoeWorkspace {
  int64_t choice, weight, xh, xp, act, y, barrier, bytes;
};

static MoeWorkspace moe_workspace(int64_t T, int64_t H, int64_t I, int64_t top) {
  MoeWorkspace w;
  w.choice = 0;
  w.weight = up256(T * top * 4);
  w.xh = 2 * w.weight;
  w.xp = w.xh + up256(T * ((H + 63) / 64) * 128);
  w.act = w.xp + up256(T * 8);
  w.y = w.act + 2 * up256(T * top * ((I + 63) / 64) * 128);
  w.barrier = w.y + up256(T * top * H * 4);
  w.bytes = w.barrier + 256;
  return w;
}

static int check_moe(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top, int format) {
  if (format != QZ_FMT_NVFP4 && format != QZ_FMT_MXFP4)
    return fail(QZ_ERR_INVALID, "the experts are NVFP4 (blocks of 16) or MXFP4 (blocks of 32), got format %d", format);
  if (H <= 0 || I <= 0 || H % 32 || I % 32 || H > (1 << 20) || I > (1 << 20))
    return fail(QZ_ERR_INVALID, "H=%lld and I=%lld must be positive multiples of 32", (long long)H, (long long)I);
  if (E < 1 || E > kMoeMaxExperts) return fail(QZ_ERR_INVALID, "%lld experts, expected 1 to %d", (long long)E, kMoeMaxExperts);
  if (T < 0 || T > kMoeMaxTokens) return fail(QZ_ERR_INVALID, "%lld tokens, expected at most %d", (long long)T, kMoeMaxTokens);
  if (top < 1 || top > E || top > kMoeMaxTop)
    return fail(QZ_ERR_INVALID, "top_k=%lld, expected 1 to %d and at most the number of experts", (long long)top, kMoeMaxTop);
  return QZ_OK;
}

}  // namespace qz

using namespace qz;

extern "C" int qz_moe_layout(const uint8_t* scale_codes, const uint8_t* packed, int64_t E, int64_t rows, int64_t K,
                             int format, int gate_up, uint8_t* codes_out, uint8_t* scales_out, float* norms_out,
                             void* stream) {
  if (format != QZ_FMT_NVFP4 && format != QZ_FMT_MXFP4)
    return fail(QZ_ERR_INVALID, "the experts are NVFP4 (blocks of 16) or MXFP4 (blocks of 32), got format %d", format);
  if (E < 1 || E > kMoeMaxExperts || rows <= 0 || rows % 32 || K <= 0 || K % 32)
    return fail(QZ_ERR_INVALID, "need 1 to %d experts, rows and K positive multiples of 32", kMoeMaxExperts);
  if (!scale_codes || !packed || !codes_out || !scales_out || (gate_up && !norms_out)) return fail(QZ_ERR_INVALID, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(codes_out) | reinterpret_cast<uintptr_t>(scales_out)) % 16 ||
      (gate_up && reinterpret_cast<uintptr_t>(norms_out) % 8))
    return fail(QZ_ERR_INVALID, "codes_out and scales_out must be 16-byte aligned, norms_out 8-byte");
  int sms = 0;
  const int s = current_sms(&sms);
  if (s != QZ_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t* co = reinterpret_cast<uint32_t*>(codes_out);
  if (format == QZ_FMT_NVFP4) moe_layout_kernel<16><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, gate_up, co, scales_out);
  else moe_layout_kernel<32><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, gate_up, co, scales_out);
  int r = cuda_status(cudaGetLastError(), "moe layout launch");
  if (r != QZ_OK || !gate_up) return r;
  // 0x80 in every byte: below any bound
  if ((r = cuda_status(cudaMemsetAsync(norms_out, 0x80, (size_t)E * 8, st), "cudaMemsetAsync")) != QZ_OK) return r;
  int* norms = reinterpret_cast<int*>(norms_out);
  if (format == QZ_FMT_NVFP4) moe_bound_kernel<16><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, norms);
  else moe_bound_kernel<32><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, norms);
  if ((r = cuda_status(cudaGetLastError(), "moe bound launch")) != QZ_OK) return r;
  moe_factors_kernel<<<(unsigned)((E + 127) / 128), 128, 0, st>>>(reinterpret_cast<float2*>(norms_out), E);
  return cuda_status(cudaGetLastError(), "moe bound launch");
}

extern "C" int qz_moe_workspace(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k, int64_t* bytes) {
  const int s = check_moe(T, H, I, E, top_k, QZ_FMT_NVFP4);
  if (s != QZ_OK) return s;
  if (!bytes) return fail(QZ_ERR_INVALID, "NULL pointer");
  *bytes = moe_workspace(T, H, I, top_k).bytes;
  return QZ_OK;
}

extern "C" int qz_moe(const void* x, int dtype, int64_t ldx, int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k,
                      int renormalize, const void* router, int router_dtype, int format, const uint8_t* up_codes,
                      const uint8_t* up_scales, const float* up_norms, float up_tensor_scale, const uint8_t* down_codes,
                      const uint8_t* down_scales, float down_tensor_scale, void* out, int* ids, float* weights,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  int s = check_moe(T, H, I, E, top_k, format);
  if (s != QZ_OK) return s;
  if (dtype != QZ_DTYPE_BF16 && dtype != QZ_DTYPE_F16) return fail(QZ_ERR_INVALID, "x must be bf16 or fp16, got dtype %d", dtype);
  if (router_dtype != QZ_DTYPE_F32 && router_dtype != QZ_DTYPE_BF16 && router_dtype != QZ_DTYPE_F16)
    return fail(QZ_ERR_INVALID, "unknown dtype %d", router_dtype);
  if (T == 0) return QZ_OK;
  if (!x || !router || !up_codes || !up_scales || !up_norms || !down_codes || !down_scales || !out || !workspace)
    return fail(QZ_ERR_INVALID, "NULL pointer");
  if (ldx < H || ldx % 8) return fail(QZ_ERR_INVALID, "rows of x must be at least H apart and 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(up_codes) |
       reinterpret_cast<uintptr_t>(up_scales) | reinterpret_cast<uintptr_t>(down_codes) |
       reinterpret_cast<uintptr_t>(down_scales)) % 16 || reinterpret_cast<uintptr_t>(workspace) % 256 ||
      (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(up_norms)) % 8)  // pairs of norms, four results at once
    return fail(QZ_ERR_INVALID, "inputs must be 16-byte aligned, up_norms and out 8-byte, workspace 256-byte");
  const MoeWorkspace w = moe_workspace(T, H, I, top_k);
  if (workspace_bytes < w.bytes)
    return fail(QZ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.bytes);
  int sms = 0;
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeParams p{};
  p.T = (int)T; p.H = (int)H; p.I = (int)I; p.E = (int)E; p.top = (int)top_k;
  p.hc = (int)((H + 63) / 64); p.ic = (int)((I + 63) / 64);
  p.dtype = dtype;
  if (!ids) ids = reinterpret_cast<int*>(ws + w.choice);
  if (!weights) weights = reinterpret_cast<float*>(ws + w.weight);
  p.choice = ids; p.choice_weight = weights;
  p.up_codes = up_codes; p.up_scales = up_scales; p.norms = up_norms;
  p.down_codes = down_codes; p.down_scales = down_scales;
  p.up_scale = up_tensor_scale; p.down_scale = down_tensor_scale;
  p.xh = reinterpret_cast<const __half*>(ws + w.xh);
  p.xp = reinterpret_cast<const int2*>(ws + w.xp);
  p.act = reinterpret_cast<__half*>(ws + w.act);
  p.act_part = up256(T * top_k * p.ic * 128) / 2;
  p.y = reinterpret_cast<float*>(ws + w.y);
  p.barrier = reinterpret_cast<int*>(ws + w.barrier);
  p.out = out;
  const unsigned grid = (unsigned)((T + kRouterTokens - 1) / kRouterTokens * kRouterCtas);
#define QZ_ROUTER_N(DT, RDT, NTK)                                                                                       \
  moe_router_kernel<DT, RDT, NTK><<<grid, kRouterThreads, 0, st>>>(x, ldx, router, p.T, p.H, p.E, p.top, renormalize,     \
                                                                   ids, weights, reinterpret_cast<uint4*>(ws + w.xh),   \
                                                                   reinterpret_cast<int2*>(ws + w.xp), p.barrier)
#define QZ_ROUTER(DT, RDT)                                                                                              \
  if (T == 1) QZ_ROUTER_N(DT, RDT, 1);                                                                                  \
  else QZ_ROUTER_N(DT, RDT, kRouterTokens)
#define QZ_ROUTER_OF(DT)                                                                                                \
  if (router_dtype == QZ_DTYPE_F32) { QZ_ROUTER(DT, kDtF32); }                                                          \
  else if (router_dtype == QZ_DTYPE_BF16) { QZ_ROUTER(DT, kDtBF16); }                                                   \
  else { QZ_ROUTER(DT, kDtF16); }
  if (dtype == QZ_DTYPE_BF16) { QZ_ROUTER_OF(kDtBF16) }
  else { QZ_ROUTER_OF(kDtF16) }
#undef QZ_ROUTER_OF
#undef QZ_ROUTER
#undef QZ_ROUTER_N
  if ((s = cuda_status(cudaGetLastError(), "moe router launch")) != QZ_OK) return s;
  const bool nv = format == QZ_FMT_NVFP4, two = dtype == QZ_DTYPE_F16;
  const void* fn = nv ? (two ? reinterpret_cast<const void*>(&moe_experts_kernel<16, 2>) : reinterpret_cast<const void*>(&moe_experts_kernel<16, 1>))
                      : (two ? reinterpret_cast<const void*>(&moe_experts_kernel<32, 2>) : reinterpret_cast<const void*>(&moe_experts_kernel<32, 1>));
  const int smem = (nv ? MoeRing<16>::kBytes : MoeRing<32>::kBytes) + (int)sizeof(MoeShared);
  static bool attr_set[4][64] = {};  // per kernel and device (a benign race: every thread sets the same value)
  int dev = 0;
  if ((s = cuda_status(cudaGetDevice(&dev), "cudaGetDevice")) != QZ_OK) return s;
  bool* done = dev >= 0 && dev < 64 ? &attr_set[(nv ? 0 : 2) + (two ? 1 : 0)][dev] : nullptr;
  if (!done || !*done) {
    s = cuda_status(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute");
    if (s != QZ_OK) return s;
    if (done) *done = true;
  }
  void* args[] = {&p};
  return cuda_status(cudaLaunchCooperativeKernel(fn, dim3((unsigned)sms), dim3(kMoeThreads), args, (size_t)smem, st),
                     "moe experts launch");
}
