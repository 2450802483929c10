// The packed 8-bit format of include/spb_hip.h ("8-bit packing"): what its writers and readers share.
#pragma once
#include "vec8.h"

#define P8_BLOCK 128                  // columns (and, for weights, rows) that share a scale
#define P8_E_LOW (-110)               // smallest / largest exponent of a scale: every value code * 2^e is then a normal bfloat16
#define P8_E_HIGH 120

#define P8_DEPTH_MAX (1 << 23)        // longest row of codes in a product: the rows of a tile are reached by 32-bit offsets
#define P8_SIDE_MAX (1 << 30)         // most rows of B, columns of G: rounded up to a tile they fit an int

static inline int p8_cols(int K) { return (K + 127) / 128 * 128; }          // Kp: bytes of a row of codes
static inline int p8_scales(int K) { return ((K + 127) / 128 + 3) / 4 * 4; } // Sp: bytes of a row of scales

#define P8_THREADS 0xffffffffll        // most threads that a launch holds
static inline bool p8_fits(long long wgs, int threads) { return wgs <= 0x7fffffffll && wgs * threads <= P8_THREADS; }

// exponent of a block from its largest finite magnitude: top = m 2^k with 1 <= m < 2 and 448 = 1.75 * 2^8, so e = k - 8, one more if m > 1.75
__device__ __forceinline__ int p8_exponent(float top) {
  const unsigned u = __float_as_uint(top);
  if (u == 0) return 0;
  const int e = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);     // a subnormal top has k < -126: clamped below
  return e < P8_E_LOW ? P8_E_LOW : (e > P8_E_HIGH ? P8_E_HIGH : e);
}
__device__ __forceinline__ float p8_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float p8_finite_abs(float v) { const float a = fabsf(v); return a < __builtin_inff() ? a : 0.f; }   // inf, NaN: 0

// four codes of x * 2^-e (r = 2^-e), round to nearest even; inf and NaN become NaN codes.  Only in blocks of the highest exponent can a finite
// value round up to 2^128: it takes the code below.
__device__ __forceinline__ unsigned p8_encode4(float a, float b, float c, float d) {
  int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
}
__device__ __forceinline__ uint2 p8_encode8(const float v[8], int e) {
  const float r = p8_pow2(-e);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i] * r;
  if (e == P8_E_HIGH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(x[i]);
      if (a > 240.f && a < __builtin_inff()) x[i] = copysignf(240.f, x[i]);
    }
  }
  return make_uint2(p8_encode4(x[0], x[1], x[2], x[3]), p8_encode4(x[4], x[5], x[6], x[7]));
}
typedef float p8_f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void p8_decode8(uint2 q, float s, float v[8]) {
  const p8_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
  const p8_f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
  v[0] = a.x * s; v[1] = a.y * s; v[2] = b.x * s; v[3] = b.y * s;
  v[4] = c.x * s; v[5] = c.y * s; v[6] = d.x * s; v[7] = d.y * s;
}

// LDS-DMA of 4 bytes a lane (dma16s of common.h with dwords): lane i's dword lands at lds_base + 4 i
__device__ __forceinline__ void dma4s(const void* sbase, unsigned voff, unsigned lds_base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds_base) : "memory");
}

// Four floats of a partial product past the caches: the next launch reads them on other XCDs, and lines left dirty in this one's L2 would be written back before
// it could start (weight gradient 2352 x 1024 x 1280: 26.8 -> 23.8 us).
__device__ __forceinline__ void p8_put_part(float* p, const f32x4_t& v) { __builtin_nontemporal_store(v, reinterpret_cast<f32x4_t*>(p)); }
// Sum of S partial planes in a fixed order, four neighbouring floats a thread (`i` is their number).  GR 1: a thread adds all of them, four requested at a time.
// Many planes (S > P8_JOIN): GR threads take a part of the planes each, whose sums meet in LDS; one of them returns true with the result.
constexpr int P8_JOIN = 16;
template <int GR> __device__ __forceinline__ bool p8_sum_parts(const float* part, int S, long long plane, long long& i, float4& v) {
  constexpr int Q = 256 / GR;
  const int ql = threadIdx.x % Q, gr = threadIdx.x / Q, per = (S + GR - 1) / GR, s0 = gr * per, s1 = s0 + per < S ? s0 + per : S;
  i = (long long)blockIdx.x * Q + ql;
  const bool in = i * 4 < plane;
  const float* p = part + (in ? i * 4 : 0);
  v = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int B = GR == 1 ? 4 : 8;
  for (int s = s0; s < s1; s += B) {
    float4 x[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const f32x4_t q = s + k < s1 ? __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(p + (s + k) * plane)) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
      x[k] = make_float4(q[0], q[1], q[2], q[3]);
    }
#pragma unroll
    for (int k = 0; k < B; ++k)
      if (s + k < s1) { v.x += x[k].x; v.y += x[k].y; v.z += x[k].z; v.w += x[k].w; }
  }
  if constexpr (GR > 1) {
    __shared__ float4 red[GR][Q];
    red[gr][ql] = v;
    __syncthreads();
    if (gr > 0) return false;
#pragma unroll
    for (int k = 1; k < GR; ++k) { const float4 x = red[k][ql]; v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w; }
  }
  return in;
}
inline long long p8_join_blocks(long long plane, int S) { const int q = S > P8_JOIN ? 16 : 256; return (plane / 4 + q - 1) / q; }
