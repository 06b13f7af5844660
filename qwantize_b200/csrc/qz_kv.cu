// qz_kv.cu -- a paged key / value cache held in 8 bits (int8 or E4M3) with one
// fp32 scale per page of 64 tokens and head: append, read back, and attention
// of one query token per sequence over it.
//
//   append     s' = max(s, max|new| * fp32(1 / top)), s = 0 for a page without
//              tokens; codes of the page's older tokens are taken over by s / s', new
//              ones are x / s'; slots behind the last token are zero   (top = 127 / 448)
//   attention  o_h = sum_n p_n v_n, p = softmax_n(scale q_h . k_n), the query heads
//              of a group sharing one head of the cache
//
// The attention reads each code once and is bound by HBM: 2 D bytes per token and
// head (32 sequences up to 32768 tokens, 8 heads of 128, E4M3: 1.09 GB in 180 us,
// 6.0 TB/s).  Layout inside a (page, head) block of 64 D bytes, so that a warp's
// 16-byte loads are contiguous and are the A fragments of mma.m16n8k16 after an
// exact conversion to fp16 (int8 and E4M3 both fit):
//   keys    token n = 16 t + 2 j + e, value d at ((j D/64 + d/64) 8 + 2 t + e) 64 + d % 64
//   values  transposed: token n, value d at 64 d + n
// Key tiles 2i and 2i + 1 (8 tokens each) are the 16 rows of score tile i, and a
// lane's 4 bytes of a value row are its part of the value product's step i.
//
// Work: the pages of all (sequence, head) pairs, in order, are cut into equal
// runs, one per warp of the grid (lengths live on the device, so the cut is made
// there); a warp streams its run through its own ring of bulk copies with a
// running maximum and sum, and never waits for another warp.  A pair that one warp
// covers is written at once; of the others each warp leaves a partial result and
// a second kernel joins them in order.  Few short sequences go without the second
// launch: a CTA per pair, joined through shared memory.
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

constexpr int kPage = 64;           // tokens per page
constexpr int kKvInt8 = 0, kKvE4M3 = 1;
constexpr int kKvMaxSeqs = 4096;    // sequences per attention call (their prefix sums sit in shared memory)

// Byte offsets inside a (page, head) block.
__host__ __device__ __forceinline__ int key_at(int n, int d, int D) {
  return (((n >> 1 & 7) * (D / 64) + d / 64) * 8 + (n >> 4) * 2 + (n & 1)) * 64 + d % 64;
}
__host__ __device__ __forceinline__ int value_at(int n, int d) { return d * 64 + n; }
// The token of byte `at` of a key block.
__device__ __forceinline__ int key_token(int at, int D) {
  const int j = at / (D * 8), g = at / 64 % 8;
  return (g >> 1) * 16 + 2 * j + (g & 1);
}

template <int KV>
__device__ __forceinline__ float decode8(uint32_t b) {
  if (KV == kKvInt8) return (float)(int8_t)b;
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)b));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

template <int KV>
__device__ __forceinline__ uint32_t encode8(float y) {
  if (KV == kKvInt8) return (uint32_t)(int)fminf(fmaxf(rintf(y), -127.0f), 127.0f) & 255u;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(y));
  return r & 255u;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendParams {
  uint8_t *k, *v;
  float *ks, *vs;
  int64_t num_pages;
  int Hkv;
  const uint16_t *nk, *nv;      // new tokens: (token, head, D), strides in elements
  int64_t k_tok, k_head, v_tok, v_head, N;
  const int* table;             // (B, max_pages)
  int64_t ld_table;
  int max_pages;
  const int* lengths;           // tokens before the append
  const int* cu;                // (B + 1) prefix sums of the new tokens, or NULL: one per sequence
  int64_t max_new;
};

// Codes of y = x / s, the quotient correctly rounded, four to a word.  lo and hi
// are the reciprocal of s, 2^-21 down and up: their products enclose the quotient
// (each of reciprocal, its scaling and product is off by 2^-24 at most), and
// rounding is monotonic, so where both give the same code it is the quotient's.
// `near` is set where they do not, and the caller divides.
struct Reciprocal {
  float2 lo, hi;
};
__device__ __forceinline__ Reciprocal reciprocal(float s) {
  const float r = __frcp_rn(s), a = __fmul_rn(r, 1.0f - 0x1p-21f), b = __fmul_rn(r, 1.0f + 0x1p-21f);
  return {make_float2(a, a), make_float2(b, b)};
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 x, x, y, z;\n"
      " mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x4(float2 a, float2 b) {
  uint32_t w;
  asm("{\n .reg .b16 x, y;\n cvt.rn.satfinite.e4m3x2.f32 x, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 y, %4, %3;\n mov.b32 %0, {x, y};\n}\n"
      : "=r"(w)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return w;
}
template <int KV>
__device__ __forceinline__ uint32_t encode4(float2 a, float2 b, const Reciprocal& r, bool& near) {
  if constexpr (KV == kKvInt8) {
    const float2 magic = make_float2(12582912.0f, 12582912.0f);  // 1.5 * 2^23: the sum's low byte is the rounded product
    const float2 l0 = fma2(a, r.lo, magic), l1 = fma2(b, r.lo, magic), h0 = fma2(a, r.hi, magic), h1 = fma2(b, r.hi, magic);
    near |= ((__float_as_uint(l0.x) ^ __float_as_uint(h0.x)) | (__float_as_uint(l0.y) ^ __float_as_uint(h0.y)) |
             (__float_as_uint(l1.x) ^ __float_as_uint(h1.x)) | (__float_as_uint(l1.y) ^ __float_as_uint(h1.y))) != 0;
    return __byte_perm(__byte_perm(__float_as_uint(h0.x), __float_as_uint(h0.y), 0x0040),
                       __byte_perm(__float_as_uint(h1.x), __float_as_uint(h1.y), 0x0040), 0x5410);
  } else {
    const uint32_t w = e4m3x4(mul2(a, r.hi), mul2(b, r.hi));
    near |= w != e4m3x4(mul2(a, r.lo), mul2(b, r.lo));
    return w;
  }
}
template <int KV>
__device__ __noinline__ uint32_t encode4_div(float a, float b, float c, float d, float s) {
  return encode8<KV>(__fdiv_rn(a, s)) | encode8<KV>(__fdiv_rn(b, s)) << 8 | encode8<KV>(__fdiv_rn(c, s)) << 16 |
         encode8<KV>(__fdiv_rn(d, s)) << 24;
}

template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int i) {
  const uint32_t h = i ? w >> 16 : w & 0xffffu;
  return DT == kDtBF16 ? bf16_bits_to_float(h) : f16_bits_to_float(h);
}
// The larger magnitudes of two pairs of 16-bit values, as 16 bits that order like them (NaN above all).
__device__ __forceinline__ uint32_t abs_max16(uint32_t m, uint32_t w) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(w & 0x7fff7fffu));
  return r;
}

// One CTA per (page a sequence touches, head, keys or values, sequence).  All
// it reads -- the new values, the page's block and scale -- is asked for at once and
// kept in registers; the block is rebuilt in shared memory and written whole.  A
// decode step is one such round trip.  Threads own 8 values of a token (keys) or
// two values of 4 neighbouring slots (values), so that a word of the block has one
// owner.  Prompts are bound by instructions, 16 per value: 8 of 1900 tokens, 8 heads
// of 128, E4M3, in 26 us (69% of the issue slots).  64 single tokens: 12.5 to 13.7 us
// for 1024 CTAs in 1.4 waves; a warp's 630 instructions, nearly all of them on the
// page's older codes, take half of the issue slots, and of the stalls half are waits
// for the reads (length, table, block) and at the CTA's barriers.
template <int KV, int D, int DT>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kStride = 68;  // bytes between value rows in shared memory: words of neighbouring rows in different banks
  constexpr int kVecs = kPage * D / 16 / 256, kNew = kPage * D / 8 / 256;  // 16-byte vectors of codes, of new values per thread
  __shared__ __align__(16) uint8_t s_block[D * kStride];
  __shared__ uint32_t s_max[8];
  const int tid = threadIdx.x, which = blockIdx.y & 1, head = blockIdx.y >> 1, b = blockIdx.z;
  int64_t first = b, end = b + 1;
  if (p.cu) { first = p.cu[b]; end = p.cu[b + 1]; }
  const int64_t old = p.lengths[b];
  if (old < 0 || first < 0 || end > p.N || end <= first) return;
  if (end - first > p.max_new) end = first + p.max_new;
  const int64_t blk = old / kPage + blockIdx.x;
  if (blk >= p.max_pages) return;
  const int64_t t0 = blk * kPage > old ? blk * kPage : old;   // position of the first new token in this page
  int64_t t1 = old + (end - first);
  if (t1 > (blk + 1) * kPage) t1 = (blk + 1) * kPage;
  if (t0 >= t1) return;
  const int64_t page = p.table[b * p.ld_table + blk];
  if (page < 0 || page >= p.num_pages) return;
  const int off = (int)(t0 - blk * kPage), fill = (int)(t1 - blk * kPage);  // new tokens take slots [off, fill)
  const int64_t at = page * p.Hkv + head;
  const int64_t tok = which ? p.v_tok : p.k_tok;
  const uint16_t* x = (which ? p.nv + head * p.v_head : p.nk + head * p.k_head) + (first + (t0 - old) - off) * tok;  // slot 0's row
  float* scale_p = (which ? p.vs : p.ks) + at;
  uint8_t* block = (which ? p.v : p.k) + at * (int64_t)(kPage * D);
  const float per_top = KV == kKvInt8 ? 1.0f / 127.0f : 1.0f / 448.0f;  // rounded once, a constant

  // new values: keys 8 of a slot; values two (d, d + 1) of 4 slots in x, y, z, w
  uint4 raw[kNew];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kNew; ++i) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (which == 0) {
      const int n = (tid + i * 256) / (D / 8), d = (tid + i * 256) % (D / 8) * 8;
      if (n >= off && n < fill) raw[i] = __ldg(reinterpret_cast<const uint4*>(x + n * tok + d));
    } else {
      const int n = (tid + i * 256) / (D / 2) * 4, d = (tid + i * 256) % (D / 2) * 2;
      const uint16_t* from = x + n * tok + d;
      if (n >= off && n < fill) raw[i].x = __ldg(reinterpret_cast<const uint32_t*>(from));
      if (n + 1 >= off && n + 1 < fill) raw[i].y = __ldg(reinterpret_cast<const uint32_t*>(from + tok));
      if (n + 2 >= off && n + 2 < fill) raw[i].z = __ldg(reinterpret_cast<const uint32_t*>(from + 2 * tok));
      if (n + 3 >= off && n + 3 < fill) raw[i].w = __ldg(reinterpret_cast<const uint32_t*>(from + 3 * tok));
    }
  }
  uint4 have[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
    have[i] = off > 0 ? *reinterpret_cast<const uint4*>(block + (tid + i * 256) * 16) : make_uint4(0, 0, 0, 0);
  const float before = off > 0 ? *scale_p : 0.0f;
#pragma unroll
  for (int i = 0; i < kNew; ++i) m = abs_max16(abs_max16(abs_max16(abs_max16(m, raw[i].x), raw[i].y), raw[i].z), raw[i].w);
  m = __reduce_max_sync(0xffffffffu, max(m >> 16, m & 0xffffu));
  if ((tid & 31) == 0) s_max[tid >> 5] = m;
  __syncthreads();
  m = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) m = max(m, s_max[w]);
  m = __float_as_uint(half_of<DT>(m, 0));
  const float need = __fmul_rn(__uint_as_float(m), per_top);
  float s = before > need ? before : need;
  // a value that is not finite, now or earlier, leaves the page's scale NaN and its codes 0
  const bool fine = m < 0x7f800000u && before <= 3.0e38f;
  if (!fine) s = __uint_as_float(0x7fc00000u);
  const float ratio = s > 0.0f ? __fdiv_rn(before, s) : 0.0f;
  // older tokens (slots below off), zeros elsewhere; a page that new tokens fill has neither
  const bool whole = off == 0 && fill == kPage && fine && s > 0.0f;
  if (!whole) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = (tid + i * 256) * 16, kt = key_token(v, D);
      uint32_t ww[4] = {have[i].x, have[i].y, have[i].z, have[i].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // bytes of slots below off
        const int left = which ? off - (v % 64 + 4 * q) : (kt < off ? 4 : 0);
        ww[q] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        if (!fine) ww[q] = 0;
        if (ratio != 1.0f && ww[q]) {
          uint32_t r = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) r |= encode8<KV>(__fmul_rn(decode8<KV>(ww[q] >> (8 * c) & 255u), ratio)) << (8 * c);
          ww[q] = r;
        }
        *reinterpret_cast<uint32_t*>(s_block + (which ? v / 64 * kStride + v % 64 : v) + 4 * q) = ww[q];
      }
    }
    __syncthreads();
  }
  if (fine && s > 0.0f) {
    const Reciprocal r = reciprocal(s);
    const bool slow = s < 0x1p-100f;  // the reciprocal or its products may leave fp32's normal range
#pragma unroll
    for (int i = 0; i < kNew; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      const int n = which ? (tid + i * 256) / (D / 2) * 4 : (tid + i * 256) / (D / 8);
      if (which ? n + 3 < off || n >= fill : n < off || n >= fill) continue;
      float2 f[2][2];  // keys: values 0-3, 4-7; values: row d, row d + 1
      bool near = slow;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          f[h][c] = which ? make_float2(half_of<DT>(w[2 * c], h), half_of<DT>(w[2 * c + 1], h))
                          : make_float2(half_of<DT>(w[2 * h + c], 0), half_of<DT>(w[2 * h + c], 1));
      uint32_t code[2] = {encode4<KV>(f[0][0], f[0][1], r, near), encode4<KV>(f[1][0], f[1][1], r, near)};
      if (near) {
#pragma unroll
        for (int h = 0; h < 2; ++h) code[h] = encode4_div<KV>(f[h][0].x, f[h][0].y, f[h][1].x, f[h][1].y, s);
      }
      if (which == 0) {
        *reinterpret_cast<uint2*>(s_block + key_at(n, (tid + i * 256) % (D / 8) * 8, D)) = make_uint2(code[0], code[1]);
      } else {
        // slots without a new token have code 0 here, and their old code in the block
        const int d = (tid + i * 256) % (D / 2) * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t* to = reinterpret_cast<uint32_t*>(s_block + (d + h) * kStride + n);
          *to = whole ? code[h] : *to | code[h];
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = (tid + i * 256) * 16;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(s_block + (which ? v / 64 * kStride + v % 64 : v));
    *reinterpret_cast<uint4*>(block + v) = make_uint4(from[0], from[1], from[2], from[3]);
  }
  if (tid == 0) *scale_p = s;
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
template <int KV>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (KV == kKvInt8) {
    // 0x6400 | (code + 128) is 1024 + code + 128 in fp16
    w ^= 0x80808080u;
    lo = __byte_perm(w, 0x64646464u, 0x4140);
    hi = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 c = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), c), b = __hsub2(*reinterpret_cast<__half2*>(&hi), c);
    lo = *reinterpret_cast<uint32_t*>(&a);
    hi = *reinterpret_cast<uint32_t*>(&b);
  } else {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

template <int DT>
__device__ __forceinline__ void store16or32(void* out, int64_t i, float v) {
  if (DT == kDtF32) static_cast<float*>(out)[i] = v;
  else if (DT == kDtF16) static_cast<__half*>(out)[i] = __float2half_rn(v);
  else {
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    static_cast<uint16_t*>(out)[i] = r;
  }
}

// One CTA per (page of the list, head, keys or values): codes times scale, (n,
// Hkv, 64, D).  Bound by the writes: four times the codes' bytes for fp32 (91 MB in
// 17.2 us).
template <int KV, int D, int DT>
__global__ void __launch_bounds__(256) kv_read_kernel(const uint8_t* __restrict__ k, const uint8_t* __restrict__ v,
                                                      const float* __restrict__ ks, const float* __restrict__ vs,
                                                      int64_t num_pages, int Hkv, const int* __restrict__ pages,
                                                      void* __restrict__ ok, void* __restrict__ ov) {
  constexpr int kStride = 68, kVecs = kPage * D / 16 / 256;
  __shared__ __align__(16) uint8_t s_block[D * kStride];
  const int tid = threadIdx.x, which = blockIdx.x & 1, head = blockIdx.x >> 1;
  void* out = which ? ov : ok;
  if (!out) return;
  const int64_t n = blockIdx.y, page = pages[n], at = page * Hkv + head;
  const bool there = page >= 0 && page < num_pages;
  const uint8_t* block = (which ? v : k) + at * (int64_t)(kPage * D);
  const float s = there ? __ldg((which ? vs : ks) + at) : __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int b = (tid + i * 256) * 16;
    const uint4 w = there ? __ldg(reinterpret_cast<const uint4*>(block + b)) : make_uint4(0, 0, 0, 0);
    uint32_t* d = reinterpret_cast<uint32_t*>(s_block + (which ? b / 64 * kStride + b % 64 : b));
    d[0] = w.x; d[1] = w.y; d[2] = w.z; d[3] = w.w;
  }
  __syncthreads();
  const int64_t o0 = (n * Hkv + head) * kPage * D;
#pragma unroll 4
  for (int i = tid; i < kPage * D / 4; i += 256) {
    // keys: four values of a token; values: four tokens of a value, neighbouring lanes' stores side by side
    const int tkn = which ? i / D * 4 : i / (D / 4), d = which ? i % D : i % (D / 4) * 4;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(s_block + (which ? d * kStride + tkn : key_at(tkn, d, D)));
    uint32_t lo, hi;
    codes_to_f16<KV>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    const float f[4] = {__fmul_rn(a.x, s), __fmul_rn(a.y, s), __fmul_rn(b.x, s), __fmul_rn(b.y, s)};
    const int64_t o = o0 + tkn * D + d;
    if (which) {
#pragma unroll
      for (int q = 0; q < 4; ++q) store16or32<DT>(out, o + q * D, f[q]);
    } else if constexpr (DT == kDtF32) {
      *reinterpret_cast<float4*>(static_cast<float*>(out) + o) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      uint32_t x, y;
      if (DT == kDtBF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(f[1]), "f"(f[0]));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(f[3]), "f"(f[2]));
      } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(f[1]), "f"(f[0]));
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(f[3]), "f"(f[2]));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) = make_uint2(x, y);
    }
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
struct AttnParams {
  const uint8_t *k, *v;
  const float *ks, *vs;
  int64_t num_pages;
  int B, Hkv, G;                 // G query heads per cache head ...
  int row_tiles, rows_per_tile;  // ... in row_tiles tiles of 8 or 16
  int join_rows;                 // rows of a CTA of the joining launch
  const uint16_t* q;             // (B, Hkv * G, D), strides in elements
  int64_t q_seq, q_head;
  int dtype;
  const int* table;
  int64_t ld_table;
  int max_pages;
  const int* lengths;
  float scale_log2;              // softmax scale * log2(e)
  float* part_o;                 // (warps, 2, 16, D) partial sums
  float* part_ml;                // (warps, 2, 16, 2) maximum (base 2) and sum
  void* out;                     // (B, Hkv * G, D), contiguous
};

__device__ __forceinline__ int pages_of(const AttnParams& p, int b) {
  const int len = p.lengths[b];
  if (len <= 0) return 0;
  const int nb = (len - 1) / kPage + 1;  // any length of 32 bits, also one that stands for "all"
  return nb < p.max_pages ? nb : p.max_pages;
}

// prefix[b] = pages of the sequences before b, b = 0 .. B (all threads of the CTA)
__device__ __forceinline__ void page_prefix(const AttnParams& p, int* prefix) {
  if (threadIdx.x < 32) {
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + threadIdx.x;
      int n = b < p.B ? pages_of(p, b) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int m = __shfl_up_sync(0xffffffffu, n, o);
        if ((int)threadIdx.x >= o) n += m;
      }
      if (b < p.B) prefix[b + 1] = base + n;
      base += __shfl_sync(0xffffffffu, n, 31);
    }
    if (threadIdx.x == 0) prefix[0] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}

// Transpose of an 8 x 8 tile of 16-bit values (row g, columns 2t, 2t + 1 per lane).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 units of the last place; 0 for -inf
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Four values of a result, joined from partial sums in order.
struct Joined {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -INFINITY, l = 0.0f;

  __device__ __forceinline__ void take(const float2 ml, const float4 o) {
    const float n = fmaxf(m, ml.x), z = n == -INFINITY ? 0.0f : n;
    const float c = exp2_fast(m - z), cw = exp2_fast(ml.x - z);
    v = make_float4(v.x * c + o.x * cw, v.y * c + o.y * cw, v.z * c + o.z * cw, v.w * c + o.w * cw);
    l = l * c + ml.y * cw;
    m = n;
  }
  // divided by the sum (0 where nothing was attended to) and rounded once
  __device__ __forceinline__ void store(const AttnParams& p, int64_t at) const {
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    uint32_t x, y;
    if (p.dtype == kDtBF16) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(v.y * inv), "f"(v.x * inv));
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(v.w * inv), "f"(v.z * inv));
    } else {
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(v.y * inv), "f"(v.x * inv));
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(v.w * inv), "f"(v.z * inv));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(x, y);
  }
};

// Probabilities go to the value product as fp16 at 2^15 times their value over the
// largest so far: one above 2^-29 of the largest keeps 11 bits, and none is off by
// more than 2^-40 of it (at their own value: 2^-14 and 2^-25, and where the largest
// has a small value, thousands of small ones make up the result).  For fp16 results,
// whose own rounding is no coarser, the remainder is a second fp16 operand (PARTS = 2:
// 2^-22 of a probability; 32 sequences of 16384 tokens, 8 heads of 128, int8, groups
// of 8: 169-171 us, as without, groups of 16: 260 instead of 213).  Their sum is of
// the unrounded ones, in fp32.
constexpr float kProbUp = 0x1p15f, kProbDown = 0x1p-15f;

// NH tiles of 8 query heads share the warp's pass over a page.  Warps per SM:
// what the registers allow (D = 128: 12 of at most 168 with one tile; two tiles
// keep twice the sums: 8) and the ring, one page of keys and values per warp.
template <int D, int NH>
struct AttnGeo {
  static constexpr int kBlock = kPage * D;               // bytes of keys (or values) of one page and head
  static constexpr int kWarps = D == 128 ? (NH == 1 ? 12 : 8) : (NH == 1 ? 16 : 12);
  static constexpr int kRing = kWarps * 2 * kBlock;
  static int smem(int B) { return kRing + kWarps * 2 * 8 + (B + 1) * 4; }
};
constexpr int kAttnMaxWarps = 16;

// Scores as S^T = K Q^T and sums as O^T = V^T P^T: the cache is the 16-row A
// operand, 8 query heads the N side, so a group of up to 8 heads wastes nothing
// and a page costs 4 D/16 + 4 D/16 matrix instructions.  The codes' conversion to
// fp16 (2 instructions per 4 E4M3 codes, 5 per 4 int8) is the largest part of
// the rest.
//
// ONE: a CTA has one pair of the list to itself, its warps cut the pair's pages and
// join through shared memory, so short sequences need no second launch.
template <int D, int KV, int NH, bool ONE, int PARTS>
__global__ void __launch_bounds__(AttnGeo<D, NH>::kWarps * 32, 1) kv_attention_kernel(const __grid_constant__ AttnParams p) {
  using G = AttnGeo<D, NH>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bar_k = reinterpret_cast<uint64_t*>(smem + G::kRing) + warp * 2;
  uint64_t* bar_v = bar_k + 1;
  int* prefix = reinterpret_cast<int*>(smem + G::kRing + G::kWarps * 16);
  uint8_t* ring = smem + warp * 2 * G::kBlock;
  if (lane == 0) {
    mbar_init(bar_k, 1);
    mbar_init(bar_v, 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int HR = p.Hkv * p.row_tiles;
  // position in the work list: sequence b, head and row tile hr, page pg of nb
  struct Pos { int b, hr, pg, nb; };
  Pos cur;
  int64_t me, u0, u1;  // this warp's place; its units (a page of a pair each)
  if constexpr (ONE) {
    cur.b = blockIdx.x / HR;
    cur.hr = blockIdx.x % HR;
    cur.nb = pages_of(p, cur.b);
    me = warp;
    u0 = (int64_t)warp * cur.nb / G::kWarps;
    u1 = (int64_t)(warp + 1) * cur.nb / G::kWarps;
    cur.pg = (int)u0;
  } else {
    page_prefix(p, prefix);
    const int64_t total = (int64_t)prefix[p.B] * HR, warps = (int64_t)gridDim.x * G::kWarps;
    me = (int64_t)warp * gridDim.x + blockIdx.x;  // neighbours in work on different SMs
    u0 = me * total / warps;
    u1 = (me + 1) * total / warps;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (u0 >= u1) return;
    int lo = 0, hi = p.B;  // last b with prefix[b] * HR <= u0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)prefix[mid] * HR <= u0) lo = mid; else hi = mid;
    }
    cur.b = lo;
    cur.nb = prefix[lo + 1] - prefix[lo];
    const int64_t r = u0 - (int64_t)prefix[lo] * HR;
    cur.hr = (int)(r / cur.nb);
    cur.pg = (int)(r % cur.nb);
  }
  auto advance = [&](Pos& x) {
    if (++x.pg < x.nb || ONE) return;
    x.pg = 0;
    if (++x.hr < HR) return;
    x.hr = 0;
    do ++x.b; while (x.b < p.B && prefix[x.b + 1] == prefix[x.b]);
    x.nb = x.b < p.B ? prefix[x.b + 1] - prefix[x.b] : 1;
  };
  // the cache block of a position, -1 if the table names no page of the cache
  auto block_of = [&](const Pos& x) -> int64_t {
    const int64_t page = __ldg(p.table + (int64_t)x.b * p.ld_table + x.pg);
    return page < 0 || page >= p.num_pages ? -1 : page * p.Hkv + x.hr / p.row_tiles;
  };
  int issued_k = 0, issued_v = 0;
  auto issue = [&](const uint8_t* base, int64_t block, uint8_t* dst, uint64_t* bar) {  // lane 0
    if (block < 0) {  // nothing is read, the tokens are masked
      mbar_arrive(bar);
      return;
    }
    mbar_arrive_expect_tx(bar, G::kBlock);
    bulk_load(dst, base + block * G::kBlock, G::kBlock, bar);
  };

  Pos next = cur;
  int64_t blk = -1, blk_next = -1;
  if (!ONE || u0 < u1) {
    blk = block_of(cur);
    if (lane == 0) {
      issue(p.k, blk, ring, bar_k);
      issue(p.v, blk, ring + G::kBlock, bar_v);
    }
    issued_k = issued_v = 1;
  }
  float ks = blk >= 0 ? __ldg(p.ks + blk) : 0.0f, vs = blk >= 0 ? __ldg(p.vs + blk) : 0.0f;
  advance(next);
  if (u0 + 1 < u1) blk_next = block_of(next);

  uint32_t qb[NH][D / 16][2];
  float o[D / 16][NH][4], m[NH][2], l[NH][2], qs[NH][2];
  bool fresh = true, ok = true;
  int64_t seg_begin = u0;
  uint32_t parity = 0;
  for (int64_t u = u0; u < u1; ++u, parity ^= 1) {
    const int head = cur.hr / p.row_tiles, r0 = cur.hr % p.row_tiles * (8 * NH);
    const bool more = u + 1 < u1;
    // one page ahead: its scales; two ahead: its place in the table
    float ks_next = 0.0f, vs_next = 0.0f;
    if (more && blk_next >= 0) {
      ks_next = __ldg(p.ks + blk_next);
      vs_next = __ldg(p.vs + blk_next);
    }
    Pos after = next;
    int64_t blk_after = -1;
    if (u + 2 < u1) {
      advance(after);
      blk_after = block_of(after);
    }
    int valid = blk >= 0 ? __ldg(p.lengths + cur.b) - cur.pg * kPage : 0;
    if (valid > kPage) valid = kPage;
    if (fresh) {
      // this pair's query heads as fp16, each on the power of two that puts its
      // largest magnitude in [2^14, 2^15) (fp16 heads as they are)
      fresh = false;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const int row = r0 + 8 * n + g;
        const uint16_t* qp = p.q + cur.b * p.q_seq + (int64_t)(head * p.G + (row < p.G ? row : 0)) * p.q_head;
        uint32_t x = 0;
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int v = 0; v < 2; ++v) {  // lane t takes values 64 h + 16 t .. + 15 of head g
            const uint4 w = row < p.G ? __ldg(reinterpret_cast<const uint4*>(qp + 64 * h + 16 * t + 8 * v)) : make_uint4(0, 0, 0, 0);
            qb[n][4 * h + 2 * v][0] = w.x; qb[n][4 * h + 2 * v][1] = w.y;
            qb[n][4 * h + 2 * v + 1][0] = w.z; qb[n][4 * h + 2 * v + 1][1] = w.w;
          }
        float sc = 1.0f;
        if (p.dtype == kDtBF16) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) x = max(x, max(qb[n][i][c] & 0x7fff0000u, qb[n][i][c] << 16 & 0x7fff0000u));
          x = max(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = max(x, __shfl_xor_sync(0xffffffffu, x, 2));
          const int e = x == 0 || x >= 0x7f800000u ? 0 : max((int)(x >> 23) - 141, -112);
          const float inv = pow2f(-e);
          sc = pow2f(e);
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const __half2 h = __floats2half2_rn(bf16_bits_to_float(qb[n][i][c] & 0xffffu) * inv, bf16_bits_to_float(qb[n][i][c] >> 16) * inv);
              qb[n][i][c] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        // the sums' columns are heads 2t and 2t + 1
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          qs[n][c] = __shfl_sync(0xffffffffu, sc, (2 * t + c) * 4) * p.scale_log2;
          m[n][c] = -INFINITY;
          l[n][c] = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][n][c] = 0.0f;
    }
    if (!mbar_wait_warp(bar_k, parity, kDevErrLoadTimeout)) { ok = false; break; }
    // scores: 4 tiles of 16 tokens; row g (g + 8) of tile i is token 16 (g / 2) + 4 i + g % 2 (+ 2)
    float s[4][NH][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][n][c] = 0.0f;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(ring + (2 * i * (D / 64) + h) * 512 + lane * 16);
        const uint4 w1 = *reinterpret_cast<const uint4*>(ring + ((2 * i + 1) * (D / 64) + h) * 512 + lane * 16);
        const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t a0, a1, a2, a3;
          codes_to_f16<KV>(x0[q], a0, a2);
          codes_to_f16<KV>(x1[q], a1, a3);
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_16816(s[i][n], a0, a1, a2, a3, qb[n][4 * h + q]);
        }
      }
    }
    __syncwarp();  // every lane has read its keys
    if (more) {
      if (lane == 0) issue(p.k, blk_next, ring, bar_k);
      ++issued_k;
    }
    float corr[NH][2];
    uint32_t pb[PARTS][4][NH][2];  // probabilities, fp16: the B fragments of the value product
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float z[2], sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float f = ks * qs[n][c];
        float x = m[n][c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i][n][c] *= f;
          s[i][n][c + 2] *= f;
          if (valid < kPage) {
            const int tok = 16 * (g >> 1) + 4 * i + (g & 1);
            if (tok >= valid) s[i][n][c] = -INFINITY;
            if (tok + 2 >= valid) s[i][n][c + 2] = -INFINITY;
          }
          x = fmaxf(x, fmaxf(s[i][n][c], s[i][n][c + 2]));
        }
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        z[c] = x == -INFINITY ? 0.0f : x;  // nothing unmasked yet
        corr[n][c] = exp2_fast(m[n][c] - z[c]);
        m[n][c] = x;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][n][c] = exp2_fast(s[i][n][c] - z[c & 1]);
        sum[0] += s[i][n][0] + s[i][n][2];
        sum[1] += s[i][n][1] + s[i][n][3];
        const float2 up = make_float2(kProbUp, kProbUp);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 f = mul2(make_float2(s[i][n][2 * h], s[i][n][2 * h + 1]), up);
          const __half2 x = __float22half2_rn(f);
          pb[0][i][n][h] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&x));
          if constexpr (PARTS == 2) {
            const float2 b = __half22float2(x);
            const __half2 y = __floats2half2_rn(f.x - b.x, f.y - b.y);
            pb[1][i][n][h] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&y));
          }
        }
      }
      l[n][0] = fmaf(l[n][0], corr[n][0], sum[0]);
      l[n][1] = fmaf(l[n][1], corr[n][1], sum[1]);
    }
    if (!mbar_wait_warp(bar_v, parity, kDevErrLoadTimeout)) { ok = false; break; }
    const float v_scale = vs * kProbDown;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint4 w0 = *reinterpret_cast<const uint4*>(ring + G::kBlock + i * 1024 + lane * 16);
      const uint4 w1 = *reinterpret_cast<const uint4*>(ring + G::kBlock + i * 1024 + 512 + lane * 16);
      uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
      float d[NH][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) d[n][c] = 0.0f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (valid < kPage) {  // what lies behind the last token may decode to NaN
          const int left = valid - (16 * t + 4 * q);
          const uint32_t mask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
          x0[q] &= mask;
          x1[q] &= mask;
        }
        uint32_t a0, a1, a2, a3;
        codes_to_f16<KV>(x0[q], a0, a2);
        codes_to_f16<KV>(x1[q], a1, a3);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_16816(d[n], a0, a1, a2, a3, pb[part][q][n]);
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][n][c] = fmaf(d[n][c], v_scale, o[i][n][c] * corr[n][c & 1]);
    }
    __syncwarp();  // every lane has read its values
    if (more) {
      if (lane == 0) issue(p.v, blk_next, ring + G::kBlock, bar_v);
      ++issued_v;
    }
    const bool pair_ends = cur.pg + 1 == cur.nb;
    if (pair_ends || !more) {
      const bool whole = pair_ends && u + 1 - seg_begin == cur.nb;
      const int64_t slot = me * 2 + (seg_begin == u0 ? 0 : 1);
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // a head's sum lies in the eight lanes of its column
          float sum = l[n][c];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = 8 * n + 2 * t + c;  // of the row tile
          if (r0 + row >= p.G) continue;
          if (whole) {
            const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
            uint16_t* out = static_cast<uint16_t*>(p.out) + (((int64_t)cur.b * p.Hkv + head) * p.G + r0 + row) * D;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float v = o[i][n][2 * h + c] * inv;
                uint16_t r;
                if (p.dtype == kDtBF16) asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
                else r = __half_as_ushort(__float2half_rn(v));
                out[16 * i + 8 * h + g] = r;
              }
          } else {
            // ONE: in this warp's ring, which is idle now
            float* po = ONE ? reinterpret_cast<float*>(ring) + row * D : p.part_o + (slot * 16 + row) * D;
            float* ml = ONE ? reinterpret_cast<float*>(ring) + 16 * D + row * 2 : p.part_ml + (slot * 16 + row) * 2;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              po[16 * i + g] = o[i][n][c];
              po[16 * i + 8 + g] = o[i][n][2 + c];
            }
            if (g == 0) *reinterpret_cast<float2*>(ml) = make_float2(m[n][c], sum);
          }
        }
      fresh = true;
      seg_begin = u + 1;
    }
    cur = next;
    next = after;
    blk = blk_next;
    blk_next = blk_after;
    ks = ks_next;
    vs = vs_next;
  }
  if (!ok) {  // copies in flight must land before the CTA exits (bounded)
    mbar_wait_bounded(bar_k, (issued_k - 1) & 1, kDevErrLoadTimeout);
    mbar_wait_bounded(bar_v, (issued_v - 1) & 1, kDevErrLoadTimeout);
  }
  if constexpr (ONE) {
    __syncthreads();
    const int64_t nb = cur.nb;
    if (nb == 1) return;  // the page's warp wrote the result
    const int head = cur.hr / p.row_tiles, r0 = cur.hr % p.row_tiles * (8 * NH);
    const int rows = p.G - r0 < 8 * NH ? p.G - r0 : 8 * NH;
    for (int i = threadIdx.x; i < rows * (D / 4); i += G::kWarps * 32) {
      const int row = i / (D / 4), d4 = i % (D / 4);
      Joined a;
      for (int w = 0; w < G::kWarps; ++w) {
        if (w * nb / G::kWarps == (w + 1) * nb / G::kWarps) continue;  // it had no page
        const float* from = reinterpret_cast<const float*>(smem + w * 2 * G::kBlock);
        a.take(*reinterpret_cast<const float2*>(from + 16 * D + row * 2), *reinterpret_cast<const float4*>(from + row * D + d4 * 4));
      }
      a.store(p, (((int64_t)cur.b * p.Hkv + head) * p.G + r0 + row) * D + d4 * 4);
    }
  }
}

// Joins the partial results of the (sequence, head, row tile) pairs that several
// warps share, in the order of their pages; writes zeros for empty sequences.
// One CTA per pair and join_rows rows: a thread owns four values of one row and one
// of `split` interleaved shares of the partial results (a long sequence has
// hundreds), which then meet in shared memory.
constexpr int kJoinThreads = 512;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const __grid_constant__ AttnParams p, int64_t warps) {
  extern __shared__ int prefix[];
  __shared__ float4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  const int HR = p.Hkv * p.row_tiles;
  const int b = blockIdx.x / HR, hr = blockIdx.x % HR, head = hr / p.row_tiles, rt = hr % p.row_tiles * p.rows_per_tile;
  const int first_row = blockIdx.y * p.join_rows, r0 = rt + first_row;  // of the row tile; of the head's group
  const int last = rt + p.rows_per_tile < p.G ? rt + p.rows_per_tile : p.G;
  const int rows = last - r0 < p.join_rows ? last - r0 : p.join_rows;
  if (rows <= 0) return;
  const int per = rows * (D / 4), split = kJoinThreads / per;
  const int part = threadIdx.x / per, row = threadIdx.x % per / (D / 4), d4 = threadIdx.x % (D / 4);
  page_prefix(p, prefix);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // in every CTA with rows: this grid ends after the one before it
  const int64_t total = (int64_t)prefix[p.B] * HR;
  const int nb = prefix[b + 1] - prefix[b];
  Joined a;
  if (nb > 0) {
    const int64_t u0 = (int64_t)prefix[b] * HR + (int64_t)hr * nb, u1 = u0 + nb;
    // the warp of unit u is the last w with w * total / warps <= u; with fewer
    // units than warps every unit has a warp of its own
    const int64_t w0 = ((u0 + 1) * warps - 1) / total, w1 = (u1 * warps - 1) / total;
    if (w0 == w1) return;  // one warp had all of it
    const int count = total >= warps ? (int)(w1 - w0 + 1) : nb;
    const int first = w0 * total / warps >= u0 ? 0 : 1;  // w0 began with an earlier pair
    if (part < split) {
#pragma unroll 4
      for (int i = part; i < count; i += split) {
        const int64_t w = total >= warps ? w0 + i : ((u0 + i + 1) * warps - 1) / total;
        const int64_t at = (w * 2 + (i == 0 ? first : 0)) * 16 + first_row + row;
        a.take(__ldcg(reinterpret_cast<const float2*>(p.part_ml) + at), __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D) + d4));
      }
    }
    s_o[threadIdx.x] = a.v;
    s_ml[threadIdx.x] = make_float2(a.m, a.l);
    __syncthreads();
    if (part > 0) return;
    for (int i = 1; i < split; ++i) a.take(s_ml[i * per + threadIdx.x], s_o[i * per + threadIdx.x]);
  } else if (part > 0) {
    return;
  }
  a.store(p, (((int64_t)b * p.Hkv + head) * p.G + r0 + row) * D + d4 * 4);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
cudaError_t read_device_error_kv(unsigned* out, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(out, qz_device_error, sizeof(unsigned));
  if (e != cudaSuccess || !clear) return e;
  unsigned zero = 0;
  return cudaMemcpyToSymbol(qz_device_error, &zero, sizeof(unsigned));
}

static int check_cache(int kv_dtype, int64_t num_pages, int64_t Hkv, int64_t D) {
  if (kv_dtype != QZ_KV_INT8 && kv_dtype != QZ_KV_E4M3) return fail(QZ_ERR_INVALID, "unknown cache type %d", kv_dtype);
  if (D != 64 && D != 128) return fail(QZ_ERR_INVALID, "head dimension %lld, expected 64 or 128", (long long)D);
  if (Hkv < 1 || Hkv > 1024) return fail(QZ_ERR_INVALID, "%lld cache heads, expected 1 to 1024", (long long)Hkv);
  if (num_pages < 0 || num_pages > 2147483647LL) return fail(QZ_ERR_INVALID, "num_pages must fit in int32");
  return QZ_OK;
}

static bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

// Whether each (sequence, head, row tile) pair is given to one CTA, in one launch,
// instead of cutting all pages evenly and joining in a second one: with at most a
// CTA per SM, and at most two pages in a row for a warp by the table's width.
// Microseconds alone / evenly (a call in a graph of 60), 8 cache heads of 128, groups
// of 4, int8: 1 sequence of 300 tokens 7.4 / 9.5, of 1000 10.6 / 10.6, of 2000 14.4 / 12.4, of
// 8000 41 / 26; 8 of 1000 11.7 / 13.7, 32 of 1000 (256 pairs) 24.6 / 21.7.  With heads of 64 and
// 128, groups of 1, 4 and 16, both cache types and 16 batches from 1 x 60 to 32 x 1000 the
// rule is within 12% of the faster (worst: 1 of 1000, groups of 1: 10.5 / 9.3).  The width
// stands for the lengths, which the host does not know: in a wide table short
// sequences pay for the second launch.
static bool attention_alone(int64_t pairs, int64_t max_pages, int sms, int warps) {
  return pairs <= sms && max_pages <= 2 * warps;
}

template <int D, int KV, int NH, bool ONE, int PARTS>
static int prepare_attention() {
  static bool attr_set[64] = {false};  // per device (a benign race: every thread sets the same value)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "cudaGetDevice");
  if (dev >= 0 && dev < 64 && attr_set[dev]) return QZ_OK;
  e = cudaFuncSetAttribute(kv_attention_kernel<D, KV, NH, ONE, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           AttnGeo<D, NH>::smem(kKvMaxSeqs));
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute");
  if (dev >= 0 && dev < 64) attr_set[dev] = true;
  return QZ_OK;
}

template <int D, int KV, int NH, int PARTS>
static int launch_attention(AttnParams p, int sms, cudaStream_t st) {
  using G = AttnGeo<D, NH>;
  p.rows_per_tile = 8 * NH;
  p.row_tiles = (p.G + 8 * NH - 1) / (8 * NH);
  const int64_t pairs = (int64_t)p.B * p.Hkv * p.row_tiles;
  if (attention_alone(pairs, p.max_pages, sms, G::kWarps)) {
    const int s = prepare_attention<D, KV, NH, true, PARTS>();
    if (s != QZ_OK) return s;
    kv_attention_kernel<D, KV, NH, true, PARTS><<<(unsigned)pairs, G::kWarps * 32, G::smem(0), st>>>(p);
    return cuda_status(cudaGetLastError(), "kv attention launch");
  }
  // few pairs have many partial results each: more CTAs share a pair's (1 sequence of 4528 tokens, 128 heads on 8: 43.4
  // us with 16 rows per CTA, 19.5 with 4; 16 of 2000: 28.8 and 29.6; 32 of 300: 19.6 and 26.7)
  p.join_rows = pairs <= sms ? 4 : p.rows_per_tile;
  int s = prepare_attention<D, KV, NH, false, PARTS>();
  if (s != QZ_OK) return s;
  kv_attention_kernel<D, KV, NH, false, PARTS><<<sms, G::kWarps * 32, G::smem(p.B), st>>>(p);
  if ((s = cuda_status(cudaGetLastError(), "kv attention launch")) != QZ_OK) return s;
  // the join may begin while the last pages are read; it waits for the kernel's end before it reads results
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)pairs, (unsigned)(p.rows_per_tile / p.join_rows));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = (size_t)(p.B + 1) * 4;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kv_join_kernel<D>, p, (int64_t)sms * G::kWarps), "kv join launch");
}

template <int D, int KV>
static int run_attention(const AttnParams& p, int sms, cudaStream_t st) {
  if (p.dtype == kDtF16) return p.G <= 8 ? launch_attention<D, KV, 1, 2>(p, sms, st) : launch_attention<D, KV, 2, 2>(p, sms, st);
  return p.G <= 8 ? launch_attention<D, KV, 1, 1>(p, sms, st) : launch_attention<D, KV, 2, 1>(p, sms, st);
}

}  // namespace qz

using namespace qz;

extern "C" int qz_kv_append(uint8_t* k, float* k_scale, uint8_t* v, float* v_scale, int kv_dtype, int64_t num_pages,
                            int64_t Hkv, int64_t D, const void* new_k, int64_t k_tok, int64_t k_head, const void* new_v,
                            int64_t v_tok, int64_t v_head, int dtype, int64_t N, const int* table, int64_t ld_table,
                            int64_t max_pages, const int* lengths, const int* cu_new, int64_t max_new, int64_t B,
                            void* stream) {
  int s = check_cache(kv_dtype, num_pages, Hkv, D);
  if (s != QZ_OK) return s;
  if (dtype != QZ_DTYPE_BF16 && dtype != QZ_DTYPE_F16) return fail(QZ_ERR_INVALID, "new tokens must be bf16 or fp16, got dtype %d", dtype);
  if (B < 0 || B > 65535 || N < 0 || N > 2147483647LL || max_new < 0 || max_pages < 0 || max_pages > 2147483647LL || ld_table < max_pages)
    return fail(QZ_ERR_INVALID, "need 0 <= B <= 65535, 0 <= N < 2^31, max_new >= 0 and table rows of max_pages");
  if (!cu_new && N != B) return fail(QZ_ERR_INVALID, "without cu_new there is one new token per sequence: N=%lld, B=%lld", (long long)N, (long long)B);
  if (B == 0 || N == 0 || max_new == 0 || max_pages == 0) return QZ_OK;
  if (!k || !v || !k_scale || !v_scale || !new_k || !new_v || !table || !lengths) return fail(QZ_ERR_INVALID, "NULL pointer");
  if (off16(k) || off16(v) || off16(new_k) || off16(new_v) || k_tok % 8 || k_head % 8 || v_tok % 8 || v_head % 8)
    return fail(QZ_ERR_INVALID, "caches and rows of new tokens must be 16-byte aligned");
  int sms = 0;
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  if (max_new > N) max_new = N;
  // a run of max_new tokens touches at most this many pages, wherever it starts
  int64_t touched = (max_new + kPage - 2) / kPage + 1;
  if (touched > max_pages) touched = max_pages;
  AppendParams p{k, v, k_scale, v_scale, num_pages, (int)Hkv, static_cast<const uint16_t*>(new_k),
                 static_cast<const uint16_t*>(new_v), k_tok, k_head, v_tok, v_head, N, table, ld_table, (int)max_pages,
                 lengths, cu_new, max_new};
  const dim3 grid((unsigned)touched, (unsigned)(Hkv * 2), (unsigned)B);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define QZ_APPEND(KV, DIM)                                                                     \
  if (dtype == QZ_DTYPE_BF16) kv_append_kernel<KV, DIM, kDtBF16><<<grid, 256, 0, st>>>(p);     \
  else kv_append_kernel<KV, DIM, kDtF16><<<grid, 256, 0, st>>>(p)
  if (kv_dtype == QZ_KV_INT8 && D == 128) { QZ_APPEND(kKvInt8, 128); }
  else if (kv_dtype == QZ_KV_INT8) { QZ_APPEND(kKvInt8, 64); }
  else if (D == 128) { QZ_APPEND(kKvE4M3, 128); }
  else { QZ_APPEND(kKvE4M3, 64); }
#undef QZ_APPEND
  return cuda_status(cudaGetLastError(), "kv append launch");
}

extern "C" int qz_kv_read(const uint8_t* k, const float* k_scale, const uint8_t* v, const float* v_scale, int kv_dtype,
                          int64_t num_pages, int64_t Hkv, int64_t D, const int* pages, int64_t n, void* out_k,
                          void* out_v, int out_dtype, void* stream) {
  int s = check_cache(kv_dtype, num_pages, Hkv, D);
  if (s != QZ_OK) return s;
  if (out_dtype != QZ_DTYPE_F32 && out_dtype != QZ_DTYPE_BF16 && out_dtype != QZ_DTYPE_F16)
    return fail(QZ_ERR_INVALID, "unknown dtype %d", out_dtype);
  if (n < 0) return fail(QZ_ERR_INVALID, "n must be >= 0");
  if (n == 0) return QZ_OK;
  if (!k || !v || !k_scale || !v_scale || !pages) return fail(QZ_ERR_INVALID, "NULL pointer");
  if (off16(k) || off16(v) || off16(out_k) || off16(out_v)) return fail(QZ_ERR_INVALID, "caches and outputs must be 16-byte aligned");
  int sms = 0;
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t out_page = (size_t)Hkv * kPage * D * (out_dtype == QZ_DTYPE_F32 ? 4 : 2);
  for (int64_t n0 = 0; n0 < n; n0 += 65535) {  // the grid's y dimension
    const unsigned ny = (unsigned)(n - n0 < 65535 ? n - n0 : 65535);
    uint8_t *ok = out_k ? static_cast<uint8_t*>(out_k) + n0 * out_page : nullptr, *ov = out_v ? static_cast<uint8_t*>(out_v) + n0 * out_page : nullptr;
    const dim3 grid((unsigned)(Hkv * 2), ny);
#define QZ_READ(KV, DIM, DT) \
  kv_read_kernel<KV, DIM, DT><<<grid, 256, 0, st>>>(k, v, k_scale, v_scale, num_pages, (int)Hkv, pages + n0, ok, ov)
#define QZ_READ_OF(KV, DIM)                                     \
  if (out_dtype == QZ_DTYPE_F32) QZ_READ(KV, DIM, kDtF32);      \
  else if (out_dtype == QZ_DTYPE_BF16) QZ_READ(KV, DIM, kDtBF16); \
  else QZ_READ(KV, DIM, kDtF16)
    if (kv_dtype == QZ_KV_INT8 && D == 128) { QZ_READ_OF(kKvInt8, 128); }
    else if (kv_dtype == QZ_KV_INT8) { QZ_READ_OF(kKvInt8, 64); }
    else if (D == 128) { QZ_READ_OF(kKvE4M3, 128); }
    else { QZ_READ_OF(kKvE4M3, 64); }
#undef QZ_READ_OF
#undef QZ_READ
    s = cuda_status(cudaGetLastError(), "kv read launch");
    if (s != QZ_OK) return s;
  }
  return QZ_OK;
}

extern "C" int qz_kv_attention_workspace(int64_t D, int64_t* bytes) {
  int sms = 0;
  const int s = check_cache(QZ_KV_INT8, 0, 1, D);
  if (s != QZ_OK) return s;
  if (!bytes) return fail(QZ_ERR_INVALID, "NULL pointer");
  const int r = current_sms(&sms);
  if (r != QZ_OK) return r;
  const int64_t warps = (int64_t)sms * kAttnMaxWarps;
  *bytes = warps * 2 * (16 * D + 32) * 4;
  return QZ_OK;
}

extern "C" int qz_kv_attention(const uint8_t* k, const float* k_scale, const uint8_t* v, const float* v_scale, int kv_dtype,
                               int64_t num_pages, int64_t Hkv, int64_t D, const void* q, int64_t q_seq, int64_t q_head,
                               int dtype, int64_t B, int64_t Hq, const int* table, int64_t ld_table, int64_t max_pages,
                               const int* lengths, float scale, void* out, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  int s = check_cache(kv_dtype, num_pages, Hkv, D);
  if (s != QZ_OK) return s;
  if (dtype != QZ_DTYPE_BF16 && dtype != QZ_DTYPE_F16) return fail(QZ_ERR_INVALID, "q must be bf16 or fp16, got dtype %d", dtype);
  if (Hq < 1 || Hq % Hkv || Hq > 65536) return fail(QZ_ERR_INVALID, "%lld query heads are not a multiple of %lld cache heads", (long long)Hq, (long long)Hkv);
  if (B < 0 || B > kKvMaxSeqs) return fail(QZ_ERR_INVALID, "%lld sequences, expected at most %d", (long long)B, kKvMaxSeqs);
  if (max_pages < 0 || ld_table < max_pages || max_pages * (B ? B : 1) > 2147483647LL)
    return fail(QZ_ERR_INVALID, "need table rows of max_pages entries, B * max_pages < 2^31");
  if (B == 0) return QZ_OK;
  if (!k || !v || !k_scale || !v_scale || !q || !lengths || !out || !workspace || (!table && max_pages)) return fail(QZ_ERR_INVALID, "NULL pointer");
  if (off16(k) || off16(v) || off16(q) || off16(out) || off16(workspace) || q_seq % 8 || q_head % 8)
    return fail(QZ_ERR_INVALID, "caches, q, out and workspace must be 16-byte aligned");
  int sms = 0;
  if ((s = current_sms(&sms)) != QZ_OK) return s;
  const int64_t warps = (int64_t)sms * kAttnMaxWarps;
  const int64_t need = warps * 2 * (16 * D + 32) * 4;
  if (workspace_bytes < need) return fail(QZ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  AttnParams p{};
  p.k = k; p.v = v; p.ks = k_scale; p.vs = v_scale; p.num_pages = num_pages;
  p.B = (int)B; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv);
  p.q = static_cast<const uint16_t*>(q); p.q_seq = q_seq; p.q_head = q_head; p.dtype = dtype;
  p.table = table; p.ld_table = ld_table; p.max_pages = (int)max_pages; p.lengths = lengths;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + warps * 2 * 16 * D;
  p.out = out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D == 128) return kv_dtype == QZ_KV_INT8 ? run_attention<128, kKvInt8>(p, sms, st) : run_attention<128, kKvE4M3>(p, sms, st);
  return kv_dtype == QZ_KV_INT8 ? run_attention<64, kKvInt8>(p, sms, st) : run_attention<64, kKvE4M3>(p, sms, st);
}
