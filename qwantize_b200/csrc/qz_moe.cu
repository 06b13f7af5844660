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
// Two launches.  moe_router_kernel: the logits, and x as fp16 in the order of
// the matrix instructions' B fragments.  moe_experts_kernel, cooperative, every
// CTA resident: each CTA derives the routing from the logits for itself (they
// are a few KB), then the CTAs share the (expert, row tile) units of the
// gate / up product; a grid barrier; the units of the down product; a grid
// barrier; the weighted sum over each token's experts in a fixed order.
//
// A unit is 16 weight rows; a CTA's 8 warps split K and add up through shared
// memory.  Weights are laid out once in the order of the A fragments of
// mma.m16n8k16 (fp16, fp32 accumulation): a lane's 16 bytes hold its 4 mma
// steps of one 64-column chunk.  One mma step covers one NVFP4 scale block (two
// an MXFP4 block), so the block scale multiplies the fp32 partial product and
// the codes convert exactly to fp16 by hardware.  A gate / up tile interleaves 8
// gate rows with the 8 up rows of the same outputs, so the activation function
// needs no second pass.  tcgen05 would need 128 weight rows per instruction and
// 16-bit operands in shared memory; with 1 to 32 tokens per expert the
// fragments go straight from HBM to registers instead.
//
// fp16 operands: a bf16 token is scaled by the power of two that puts its
// largest magnitude in [2^14, 2^15), exact for values within 2^-28 of it
// (smaller ones lose bits below 2^-39 of it); an activation row likewise, one
// rounding to 11 bits, a quarter of the step of the 16-bit result's.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/qwantize_b200.h"
#include "qz_common.cuh"
#include "qz_kernels.h"
#include "qz_ptx.cuh"

namespace qz {

int fail(int code, const char* fmt, ...);
int cuda_status(cudaError_t e, const char* what);
int current_sms(int* sms);

constexpr int kMoeMaxTokens = 64, kMoeMaxExperts = 512, kMoeMaxTop = 16;
constexpr int kMoeWarps = 8, kMoeThreads = kMoeWarps * 32;
constexpr int kMoeMaxSlots = kMoeMaxTokens * kMoeMaxTop;

struct MoeParams {
  int T, H, I, E, top;
  int hc, ic;                       // 64-column chunks of H and I
  int renorm;
  int dtype;                        // of x and out
  const float* logits;              // (T, E)
  const uint4* up_codes;            // (E, I / 8 tiles, hc chunks, 32 lanes) 16 bytes
  const uint32_t* up_scales;        // (E, I / 8 tiles, hc chunks, 8 row pairs): words of scales
  const uint4* down_codes;          // (E, H / 16 tiles, ic chunks, 32 lanes)
  const uint32_t* down_scales;
  float up_scale, down_scale;       // tensor scales
  const uint4* xh;                  // (T, hc, 64) fp16 in fragment order
  const float* xs;                  // (T) power of two of each token
  float* act;                       // (T * top, I)
  unsigned* act_max;                // (T * top) bits of the largest |act|
  float* y;                         // (T * top, H)
  int* barrier;
  void* out;                        // (T, H)
  int* ids;                         // (T, top) or NULL
  float* weights;                   // (T, top) or NULL
};

// ---------------------------------------------------------------------------
// weights to fragment order
// ---------------------------------------------------------------------------
// Lane (g, t) of a 16-row tile and 64-column chunk: word j (one mma step, 16
// columns) holds columns 16j + 4t .. + 3 of row g (low half) and row g + 8 (high
// half).  gate_up: rows 0-7 of tile i are gate rows 8i .., rows 8-15 the up rows
// rows / 2 + 8i ...  Scales: the words of row g and row g + 8 side by side.
template <int BS>
__global__ void moe_layout_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales, int64_t E,
                                  int64_t rows, int64_t K, int gate_up, uint32_t* __restrict__ codes_out,
                                  uint8_t* __restrict__ scales_out) {
  const int64_t chunks = (K + 63) / 64, tiles = rows / 16;
  const int64_t total = E * tiles * chunks * 128;  // words
  constexpr int kSc = 64 / BS;                     // scales per row and chunk
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int j = i & 3, lane = (int)(i >> 2) & 31, g = lane >> 2, t = lane & 3;
    const int64_t chunk = i / 128 % chunks, tile = i / 128 / chunks % tiles, e = i / 128 / chunks / tiles;
    const int64_t col = chunk * 64 + 16 * j + 4 * t;
    uint32_t w = 0;
    for (int h = 0; h < 2; ++h) {
      const int64_t row = gate_up ? (h ? rows / 2 : 0) + tile * 8 + g : tile * 16 + h * 8 + g;
      const uint8_t* p = packed + (e * rows + row) * (K / 2) + col / 2;
      if (col < K) w |= ((uint32_t)p[0] | (uint32_t)p[1] << 8) << (16 * h);
      if (j == 0 && t < kSc) {  // lane t < kSc of the quad writes scale t of both rows
        const int64_t b = chunk * kSc + t;
        scales_out[((((e * tiles + tile) * chunks + chunk) * 8 + g) * 2 + h) * kSc + t] =
            b < K / BS ? scales[(e * rows + row) * (K / BS) + b] : 0;
      }
    }
    codes_out[i] = w;
  }
}

// ---------------------------------------------------------------------------
// router logits, fp16 tokens
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t i, float (&v)[8]) {
  if (dtype == kDtF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = dtype == kDtBF16 ? bf16_bits_to_float(ww[k] & 0xffffu) : f16_bits_to_float(ww[k] & 0xffffu);
    v[2 * k + 1] = dtype == kDtBF16 ? bf16_bits_to_float(ww[k] >> 16) : f16_bits_to_float(ww[k] >> 16);
  }
}

// 2^e with x * 2^-e in [2^14, 2^15) for the largest magnitude (its bits m); 1
// for 0, inf and NaN
__device__ __forceinline__ int f16_power(uint32_t m) {
  if (m == 0 || m >= 0x7f800000u) return 0;
  const int e = (int)(m >> 23) - 127 - 14;
  return e < -112 ? -112 : e;
}

// Blocks [0, E * ceil(T / 8)): one expert and 8 tokens, the 4 warps splitting H.
// The T blocks after them: one token to fp16, and the counters' zeroing.
constexpr int kRouterThreads = 128;
__global__ void __launch_bounds__(kRouterThreads)
    moe_router_kernel(const void* __restrict__ x, int64_t ldx, int dtype, const void* __restrict__ router, int rdtype,
                      int T, int H, int E, float* __restrict__ logits, __half* __restrict__ xh, float* __restrict__ xs,
                      unsigned* __restrict__ act_max, int n_slots, int* __restrict__ barrier) {
  __shared__ float s_part[4][8];
  __shared__ uint32_t s_max[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int groups = (T + 7) / 8;
  if ((int)blockIdx.x < E * groups) {
    const int e = blockIdx.x % E, t0 = blockIdx.x / E * 8;
    const int nt = T - t0 < 8 ? T - t0 : 8;
    float acc[8] = {};
    for (int h = tid * 8; h < H; h += kRouterThreads * 8) {
      float r[8];
      load8(router, rdtype, (int64_t)e * H + h, r);
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (n >= nt) break;
        float v[8];
        load8(x, dtype, (t0 + n) * ldx + h, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[n] = fmaf(v[k], r[k], acc[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[n] += __shfl_xor_sync(0xffffffffu, acc[n], o);
      if (lane == 0) s_part[warp][n] = acc[n];
    }
    __syncthreads();
    if (tid < nt) logits[(int64_t)(t0 + tid) * E + e] = (s_part[0][tid] + s_part[1][tid]) + (s_part[2][tid] + s_part[3][tid]);
    return;
  }
  const int t = blockIdx.x - E * groups;
  if (t == 0) {
    for (int i = tid; i < n_slots; i += kRouterThreads) act_max[i] = 0u;
    if (tid < 2) barrier[tid] = 0;
  }
  float p = 1.0f, inv = 1.0f;
  if (dtype == kDtBF16) {
    uint32_t m = 0;
    for (int h = tid * 8; h < H; h += kRouterThreads * 8) {
      float v[8];
      load8(x, dtype, t * ldx + h, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
    m = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    const int e = f16_power(m);
    p = pow2f(e);
    inv = pow2f(-e);
  }
  if (tid == 0) xs[t] = p;
  const int hc = (H + 63) / 64;
  // thread: 8 halves = (half, t) of a chunk: columns 16 (2 half + i / 4) + 4 t + i % 4
  for (int i = tid; i < hc * 8; i += kRouterThreads) {
    const int chunk = i >> 3, half = (i >> 2) & 1, q = i & 3;
    __half v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int col = chunk * 64 + 16 * (2 * half + k / 4) + 4 * q + k % 4;
      float f = 0.0f;
      if (col < H) {
        const uint32_t b = static_cast<const uint16_t*>(x)[t * ldx + col];
        f = (dtype == kDtBF16 ? bf16_bits_to_float(b) : f16_bits_to_float(b)) * inv;
      }
      v[k] = __float2half_rn(f);
    }
    *reinterpret_cast<uint4*>(xh + ((int64_t)t * hc + chunk) * 64 + half * 32 + q * 8) = *reinterpret_cast<uint4*>(v);
  }
}

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------
struct MoeShared {
  float weight[kMoeMaxSlots];
  uint16_t id[kMoeMaxSlots];
  uint16_t list[kMoeMaxSlots];       // slots (token * top + k) grouped by expert, tokens ascending
  uint16_t start[kMoeMaxExperts + 1];
  uint16_t active[kMoeMaxExperts];   // experts with tokens, ascending
  int n_active, ok;
  float part[kMoeWarps * 16 * 32];   // per warp: 16 rows x up to 32 tokens
};

// All CTAs arrive, then wait for each other (they are all resident: cooperative
// launch).  Bounded: on timeout the error flag is set and the kernel ends.
__device__ __forceinline__ bool grid_barrier(int* counter, MoeShared& s) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int ok = 1;
    atomicAdd(counter, 1);
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
  __threadfence();
  return s.ok != 0;
}

// Ascending order of the bits is ascending order of the floats, NaN on top.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ void route(const MoeParams& p, MoeShared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = warp; t < p.T; t += kMoeWarps) {
    uint32_t key[kMoeMaxExperts / 32];
    float top0 = 0.0f, sum = 0.0f;
    uint32_t taken_key = 0, mine = 0;
    float val[kMoeMaxExperts / 32];
#pragma unroll
    for (int i = 0; i < kMoeMaxExperts / 32; ++i) {
      const int e = i * 32 + lane;
      val[i] = e < p.E ? __ldcg(p.logits + (int64_t)t * p.E + e) : 0.0f;
      key[i] = e < p.E ? max(order_bits(val[i]), 1u) : 0u;  // 0: not there, or taken
    }
    float chosen = 0.0f;  // lane k keeps the logit of choice k
    for (int k = 0; k < p.top; ++k) {
      taken_key = 0;
#pragma unroll
      for (int i = 0; i < kMoeMaxExperts / 32; ++i) taken_key = max(taken_key, key[i]);
      taken_key = __reduce_max_sync(0xffffffffu, taken_key);
      uint32_t e = 0xffffffffu;
      float v = 0.0f;
#pragma unroll
      for (int i = kMoeMaxExperts / 32 - 1; i >= 0; --i)
        if (key[i] == taken_key) e = i * 32 + lane;
      e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
      for (int i = 0; i < kMoeMaxExperts / 32; ++i)
        if (e == (uint32_t)(i * 32 + lane)) { v = val[i]; key[i] = 0; }
      v = __shfl_sync(0xffffffffu, v, e & 31);
      if (k == 0) top0 = v;
      if (lane == k) { chosen = v; mine = e; }
    }
    if (p.renorm) {
      sum = lane < p.top ? expf(chosen - top0) : 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < kMoeMaxExperts / 32; ++i)
        if (i * 32 + lane < p.E) sum += expf(val[i] - top0);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < p.top) {
      const float w = __fdiv_rn(expf(chosen - top0), sum);
      s.id[t * p.top + lane] = (uint16_t)mine;
      s.weight[t * p.top + lane] = w;
      if (blockIdx.x == 0) {
        if (p.ids) p.ids[t * p.top + lane] = (int)mine;
        if (p.weights) p.weights[t * p.top + lane] = w;
      }
    }
  }
  __syncthreads();
  // counts, starts and lists per expert
  const int n = p.T * p.top;
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
    int c = 0;
    for (int i = 0; i < n; ++i) c += s.id[i] == e;
    s.start[e + 1] = (uint16_t)c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int a = 0, at = 0;
    for (int e = 0; e < p.E; ++e) {
      const int c = s.start[e + 1];
      s.start[e] = (uint16_t)at;
      if (c) s.active[a++] = (uint16_t)e;
      at += c;
    }
    s.start[p.E] = (uint16_t)at;
    s.n_active = a;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
    int at = s.start[e];
    if (at == s.start[e + 1]) continue;
    for (int i = 0; i < n; ++i)
      if (s.id[i] == e) s.list[at++] = (uint16_t)i;
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

// Four E4M3 scales of a word, or two power-of-two ones of a half word.
__device__ __forceinline__ void scales_nv(uint32_t w, float (&s)[4]) {
  uint32_t h0, h1;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(h0), "=r"(h1)
      : "r"(w));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h0)), b = __half22float2(*reinterpret_cast<__half2*>(&h1));
  s[0] = a.x; s[1] = a.y; s[2] = b.x; s[3] = b.y;
}
__device__ __forceinline__ float scale_mx(uint32_t c) {
  return __uint_as_float(c == 0 ? 0x00400000u : c == 255 ? 0x7fffffffu : c << 23);
}

// One 16-row tile times up to 8 NT tokens: this warp's chunks (warp, warp + 8,
// ...) of K.  load_b(chunk, n, b): the 8 B words of n-tile n and this lane.
template <int NT, int BS, typename LoadB>
__device__ __forceinline__ void tile_product(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales,
                                             int chunks, float (&acc)[NT][4], LoadB&& load_b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
  constexpr int kBatch = 4;
  for (int c0 = warp; c0 < chunks; c0 += kMoeWarps * kBatch) {
    uint4 w[kBatch];
    uint2 sc[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int c = c0 + i * kMoeWarps;
      if (c < chunks) {
        w[i] = __ldcs(codes + c * 32 + lane);
        if constexpr (BS == 16) sc[i] = __ldcs(reinterpret_cast<const uint2*>(scales) + c * 8 + g);
        else sc[i].x = __ldcs(scales + c * 8 + g);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int c = c0 + i * kMoeWarps;
      if (c >= chunks) break;
      float s0[4], s1[4];
      if constexpr (BS == 16) {
        scales_nv(sc[i].x, s0);
        scales_nv(sc[i].y, s1);
      } else {
        s0[0] = s0[1] = scale_mx(sc[i].x & 255u);
        s0[2] = s0[3] = scale_mx(sc[i].x >> 8 & 255u);
        s1[0] = s1[1] = scale_mx(sc[i].x >> 16 & 255u);
        s1[2] = s1[3] = scale_mx(sc[i].x >> 24);
      }
      const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      uint32_t b[NT][8];
#pragma unroll
      for (int n = 0; n < NT; ++n) load_b(c, n, b[n]);
#pragma unroll
      for (int j = 0; j < 4; j += BS / 16) {
        float d[NT][4] = {};
#pragma unroll
        for (int q = 0; q < BS / 16; ++q) {
          uint32_t a[4];
          e2m1x8_to_f16(ww[j + q], a);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(d[n], a[0], a[2], a[1], a[3], b[n][2 * (j + q)], b[n][2 * (j + q) + 1]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(d[n][0], s0[j], acc[n][0]);
          acc[n][1] = fmaf(d[n][1], s0[j], acc[n][1]);
          acc[n][2] = fmaf(d[n][2], s1[j], acc[n][2]);
          acc[n][3] = fmaf(d[n][3], s1[j], acc[n][3]);
        }
      }
    }
  }
}

// Partial sums of the 8 warps, added in warp order: row r, token n of the tile.
template <int NT>
__device__ __forceinline__ void put_partials(MoeShared& s, const float (&acc)[NT][4]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* part = s.part + warp * (16 * NT * 8);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    part[(n * 8 + 2 * t) * 16 + g] = acc[n][0];
    part[(n * 8 + 2 * t + 1) * 16 + g] = acc[n][1];
    part[(n * 8 + 2 * t) * 16 + g + 8] = acc[n][2];
    part[(n * 8 + 2 * t + 1) * 16 + g + 8] = acc[n][3];
  }
}
template <int NT>
__device__ __forceinline__ float sum_partials(const MoeShared& s, int n, int r) {
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < kMoeWarps; ++w) v += s.part[w * (16 * NT * 8) + n * 16 + r];
  return v;
}

// slots: the tokens of this unit (count <= 8 NT), in the expert's list
template <int NT, int BS>
__device__ __forceinline__ void up_unit(const MoeParams& p, MoeShared& s, int e, int tile, const uint16_t* slots, int count) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t at = ((int64_t)e * (p.I / 8) + tile) * p.hc;
  const uint4* xrow[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = n * 8 + g;
    xrow[n] = p.xh + (int64_t)(slots[i < count ? i : count - 1] / p.top) * p.hc * 8 + t;
  }
  float acc[NT][4] = {};
  tile_product<NT, BS>(p.up_codes + at * 32, p.up_scales + at * 8 * (BS == 16 ? 2 : 1), p.hc, acc,
                       [&](int c, int n, uint32_t(&b)[8]) {
                         const uint4 lo = __ldg(xrow[n] + c * 8), hi = __ldg(xrow[n] + c * 8 + 4);
                         b[0] = lo.x; b[1] = lo.y; b[2] = lo.z; b[3] = lo.w;
                         b[4] = hi.x; b[5] = hi.y; b[6] = hi.z; b[7] = hi.w;
                       });
  put_partials<NT>(s, acc);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 64; i += kMoeThreads) {
    const int n = i >> 3, r = i & 7;
    const bool there = n < count;
    float a = 0.0f;
    const int slot = slots[there ? n : 0];
    if (there) {
      const float f = p.xs[slot / p.top] * p.up_scale;
      const float gate = sum_partials<NT>(s, n, r) * f, up = sum_partials<NT>(s, n, r + 8) * f;
      a = __fdiv_rn(gate, 1.0f + expf(-gate)) * up;  // gate far below 0: expf overflows and the quotient is -0
      p.act[(int64_t)slot * p.I + tile * 8 + r] = a;
    }
    uint32_t m = __float_as_uint(a) & 0x7fffffffu;
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
    if (there && r == 0) atomicMax(p.act_max + slot, m);  // a maximum: order changes nothing
  }
  __syncthreads();
}

template <int NT, int BS>
__device__ __forceinline__ void down_unit(const MoeParams& p, MoeShared& s, int e, int tile, const uint16_t* slots, int count) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t at = ((int64_t)e * (p.H / 16) + tile) * p.ic;
  const float* arow[NT];
  float inv[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = n * 8 + g;
    const int slot = slots[i < count ? i : count - 1];
    arow[n] = p.act + (int64_t)slot * p.I + 4 * t;
    inv[n] = pow2f(-f16_power(__ldcg(p.act_max + slot)));
  }
  float acc[NT][4] = {};
  tile_product<NT, BS>(p.down_codes + at * 32, p.down_scales + at * 8 * (BS == 16 ? 2 : 1), p.ic, acc,
                       [&](int c, int n, uint32_t(&b)[8]) {
#pragma unroll
                         for (int j = 0; j < 4; ++j) {
                           float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                           if (c * 64 + j * 16 < p.I) v = __ldcg(reinterpret_cast<const float4*>(arow[n] + c * 64 + j * 16));
                           const __half2 lo = __floats2half2_rn(v.x * inv[n], v.y * inv[n]);
                           const __half2 hi = __floats2half2_rn(v.z * inv[n], v.w * inv[n]);
                           b[2 * j] = *reinterpret_cast<const uint32_t*>(&lo);
                           b[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&hi);
                         }
                       });
  put_partials<NT>(s, acc);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 128; i += kMoeThreads) {
    const int n = i >> 4, r = i & 15;
    if (n >= count) continue;
    const int slot = slots[n];
    const float f = pow2f(f16_power(__ldcg(p.act_max + slot))) * p.down_scale * s.weight[slot];
    p.y[(int64_t)slot * p.H + tile * 16 + r] = sum_partials<NT>(s, n, r) * f;
  }
  __syncthreads();
}

// Runs f(expert, tile, slots, count) for this CTA's units: every active expert,
// its tokens in groups of at most 32, its tiles.
template <typename F>
__device__ __forceinline__ void for_units(const MoeShared& s, int tiles, F&& f) {
  int first = 0;  // index of the group's first unit
  for (int a = 0; a < s.n_active; ++a) {
    const int e = s.active[a], begin = s.start[e], end = s.start[e + 1];
    for (int b = begin; b < end; b += 32) {
      // units first .. first + tiles - 1 belong to CTA (unit % grid)
      int u = (int)((blockIdx.x + gridDim.x - first % gridDim.x) % gridDim.x);
      for (; u < tiles; u += gridDim.x) f(e, u, s.list + b, end - b < 32 ? end - b : 32);
      first += tiles;
    }
  }
}

template <int BS>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_experts_kernel(const __grid_constant__ MoeParams p) {
  __shared__ MoeShared s;
  route(p, s);
  for_units(s, p.I / 8, [&](int e, int tile, const uint16_t* slots, int count) {
    if (count <= 8) up_unit<1, BS>(p, s, e, tile, slots, count);
    else if (count <= 16) up_unit<2, BS>(p, s, e, tile, slots, count);
    else up_unit<4, BS>(p, s, e, tile, slots, count);
  });
  if (!grid_barrier(p.barrier, s)) return;
  for_units(s, p.H / 16, [&](int e, int tile, const uint16_t* slots, int count) {
    if (count <= 8) down_unit<1, BS>(p, s, e, tile, slots, count);
    else if (count <= 16) down_unit<2, BS>(p, s, e, tile, slots, count);
    else down_unit<4, BS>(p, s, e, tile, slots, count);
  });
  if (!grid_barrier(p.barrier + 1, s)) return;
  for (int i = blockIdx.x * kMoeThreads + threadIdx.x; i < p.T * p.H; i += gridDim.x * kMoeThreads) {
    const int t = i / p.H, h = i % p.H;
    float v = 0.0f;
    for (int k = 0; k < p.top; ++k) v += __ldcg(p.y + (int64_t)(t * p.top + k) * p.H + h);
    if (p.dtype == kDtBF16) {
      uint16_t r;
      asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
      static_cast<uint16_t*>(p.out)[i] = r;
    } else {
      static_cast<__half*>(p.out)[i] = __float2half_rn(v);
    }
  }
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
  int64_t logits, xh, xs, act, act_max, y, barrier, bytes;
};

static MoeWorkspace moe_workspace(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top) {
  MoeWorkspace w;
  w.logits = 0;
  w.xh = up256(T * E * 4);
  w.xs = w.xh + up256(T * ((H + 63) / 64) * 128);
  w.act = w.xs + up256(T * 4);
  w.act_max = w.act + up256(T * top * I * 4);
  w.y = w.act_max + up256(T * top * 4);
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
                             int format, int gate_up, uint8_t* codes_out, uint8_t* scales_out, void* stream) {
  if (format != QZ_FMT_NVFP4 && format != QZ_FMT_MXFP4)
    return fail(QZ_ERR_INVALID, "the experts are NVFP4 (blocks of 16) or MXFP4 (blocks of 32), got format %d", format);
  if (E < 1 || E > kMoeMaxExperts || rows <= 0 || rows % 32 || K <= 0 || K % 32)
    return fail(QZ_ERR_INVALID, "need 1 to %d experts, rows and K positive multiples of 32", kMoeMaxExperts);
  if (!scale_codes || !packed || !codes_out || !scales_out) return fail(QZ_ERR_INVALID, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(codes_out) | reinterpret_cast<uintptr_t>(scales_out)) % 16)
    return fail(QZ_ERR_INVALID, "codes_out and scales_out must be 16-byte aligned");
  int sms = 0;
  const int s = current_sms(&sms);
  if (s != QZ_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (format == QZ_FMT_NVFP4)
    moe_layout_kernel<16><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, gate_up,
                                                   reinterpret_cast<uint32_t*>(codes_out), scales_out);
  else
    moe_layout_kernel<32><<<sms * 8, 256, 0, st>>>(packed, scale_codes, E, rows, K, gate_up,
                                                   reinterpret_cast<uint32_t*>(codes_out), scales_out);
  return cuda_status(cudaGetLastError(), "moe layout launch");
}

extern "C" int qz_moe_workspace(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k, int64_t* bytes) {
  const int s = check_moe(T, H, I, E, top_k, QZ_FMT_NVFP4);
  if (s != QZ_OK) return s;
  if (!bytes) return fail(QZ_ERR_INVALID, "NULL pointer");
  *bytes = moe_workspace(T, H, I, E, top_k).bytes;
  return QZ_OK;
}

extern "C" int qz_moe(const void* x, int dtype, int64_t ldx, int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k,
                      int renormalize, const void* router, int router_dtype, int format, const uint8_t* up_codes,
                      const uint8_t* up_scales, float up_tensor_scale, const uint8_t* down_codes,
                      const uint8_t* down_scales, float down_tensor_scale, void* out, int* ids, float* weights,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  int s = check_moe(T, H, I, E, top_k, format);
  if (s != QZ_OK) return s;
  if (dtype != QZ_DTYPE_BF16 && dtype != QZ_DTYPE_F16) return fail(QZ_ERR_INVALID, "x must be bf16 or fp16, got dtype %d", dtype);
  if (router_dtype != QZ_DTYPE_F32 && router_dtype != QZ_DTYPE_BF16 && router_dtype != QZ_DTYPE_F16)
    return fail(QZ_ERR_INVALID, "unknown dtype %d", router_dtype);
  if (T == 0) return QZ_OK;
  if (!x || !router || !up_codes || !up_scales || !down_codes || !down_scales || !out || !workspace)
    return fail(QZ_ERR_INVALID, "NULL pointer");
  if (ldx < H || ldx % 8) return fail(QZ_ERR_INVALID, "rows of x must be at least H apart and 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(up_codes) |
       reinterpret_cast<uintptr_t>(up_scales) | reinterpret_cast<uintptr_t>(down_codes) |
       reinterpret_cast<uintptr_t>(down_scales)) % 16 || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(QZ_ERR_INVALID, "inputs must be 16-byte aligned, workspace 256-byte");
  const MoeWorkspace w = moe_workspace(T, H, I, E, top_k);
  if (workspace_bytes < w.bytes)
    return fail(QZ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.bytes);
  int sms = 0;
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeParams p{};
  p.T = (int)T; p.H = (int)H; p.I = (int)I; p.E = (int)E; p.top = (int)top_k;
  p.hc = (int)((H + 63) / 64); p.ic = (int)((I + 63) / 64);
  p.renorm = renormalize; p.dtype = dtype;
  p.logits = reinterpret_cast<float*>(ws + w.logits);
  p.up_codes = reinterpret_cast<const uint4*>(up_codes); p.up_scales = reinterpret_cast<const uint32_t*>(up_scales);
  p.down_codes = reinterpret_cast<const uint4*>(down_codes); p.down_scales = reinterpret_cast<const uint32_t*>(down_scales);
  p.up_scale = up_tensor_scale; p.down_scale = down_tensor_scale;
  p.xh = reinterpret_cast<const uint4*>(ws + w.xh);
  p.xs = reinterpret_cast<float*>(ws + w.xs);
  p.act = reinterpret_cast<float*>(ws + w.act);
  p.act_max = reinterpret_cast<unsigned*>(ws + w.act_max);
  p.y = reinterpret_cast<float*>(ws + w.y);
  p.barrier = reinterpret_cast<int*>(ws + w.barrier);
  p.out = out; p.ids = ids; p.weights = weights;
  const int groups = (int)((T + 7) / 8);
  moe_router_kernel<<<(unsigned)(E * groups + T), kRouterThreads, 0, st>>>(
      x, ldx, dtype, router, router_dtype, p.T, p.H, p.E, reinterpret_cast<float*>(ws + w.logits),
      reinterpret_cast<__half*>(ws + w.xh), reinterpret_cast<float*>(ws + w.xs), p.act_max, (int)(T * top_k), p.barrier);
  if ((s = cuda_status(cudaGetLastError(), "moe router launch")) != QZ_OK) return s;
  void* args[] = {&p};
  const void* fn = format == QZ_FMT_NVFP4 ? reinterpret_cast<const void*>(&moe_experts_kernel<16>)
                                          : reinterpret_cast<const void*>(&moe_experts_kernel<32>);
  static int per_sm[2] = {0, 0};  // resident CTAs per SM (a benign race: every thread computes the same value)
  int& occ = per_sm[format == QZ_FMT_NVFP4 ? 0 : 1];
  if (!occ) {
    int n = 0;
    s = cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, kMoeThreads, 0), "moe occupancy");
    if (s != QZ_OK) return s;
    if (n < 1) return fail(QZ_ERR_CUDA, "moe kernel does not fit an SM");
    occ = n > 2 ? 2 : n;
  }
  return cuda_status(cudaLaunchCooperativeKernel(fn, dim3((unsigned)(sms * occ)), dim3(kMoeThreads), args, 0, st),
                     "moe experts launch");
}
