// Weight gradient from an 8-bit checkpoint:  dW[n,k] (+)= sum_m G[m,n] X[m,k],  X packed by rows (include/spb_hip.h "8-bit packing").
//
// A value code * 2^e is exact in bfloat16, so X becomes bfloat16 on its way into LDS (one instruction for two values, scale included) and the
// products run on the bfloat16 matrix cores at half the bytes a 16-bit activation would cost.  The reduction index m is the row of both operands;
// the scale belongs to (m, 128 columns): along the reduction it changes with every step, which is why the 8-bit instructions, whose scale covers 32
// steps of the reduction, do not fit.  G keeps all its bits: it is split by truncation into 1 (bfloat16), 2 (half: 8 + 3 bits) or 3 (float32: 8 + 8 + 8 bits)
// bfloat16 pieces with an exact sum.
//   * 128 x 128 tiles of dW, four waves of 64 x 64; stages of 64 rows in LDS, read with the transpose load ds_read_b64_tr_b16.
//   * Few tiles and many rows: the rows are split over workgroups, each stores its partial tile, and a second launch adds them in order.
#include "pack8.h"

namespace {

typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;
constexpr int WT = 128, WR = 64, WLD = WT + 8;       // tile, rows of a stage, row stride in LDS (elements)

struct Wgrad8Args {
  const void* G; const unsigned char* X; const unsigned char* Xs; float* out;
  long long M, ldg, ldo, plane;                        // plane: distance of two splits' outputs (0: a single one)
  long long rows;                                      // rows of a split, a multiple of WR
  int N, K, Kp, Sp, NT, KT, accumulate;
};

// bfloat16 pieces of 8 gradients: piece p of element i in out[p]
template <int P> __device__ __forceinline__ void split8(const float v[8], uint4 out[P]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    unsigned h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned u = __float_as_uint(r[i]) & 0xffff0000u;
      const bool fin = fabsf(r[i]) < __builtin_inff();
      if (r[i] != r[i]) u = 0x7fc00000u;
      h[i] = u;
      r[i] = fin ? r[i] - __uint_as_float(u) : 0.f;     // exact: what the truncation cut off
    }
    out[p] = make_uint4((h[0] >> 16) | h[1], (h[2] >> 16) | h[3], (h[4] >> 16) | h[5], (h[6] >> 16) | h[7]);
  }
}

template <typename T, int P, bool VEC>
__global__ __launch_bounds__(256) void wgrad8_kernel(const Wgrad8Args g) {
  __shared__ __attribute__((aligned(16))) bf16_t Gs[P][WR * WLD];
  __shared__ __attribute__((aligned(16))) bf16_t Xl[WR * WLD];
  const int t = threadIdx.x, l = t & 63, w = t >> 6, li = l & 15, lq = l >> 4;
  const int wn = w >> 1, wk = w & 1;
  const int lid = xcd_remap(blockIdx.x, gridDim.x);     // the tiles of a split read the same rows: one XCD, back to back
  const int tiles = g.NT * g.KT, tile = lid % tiles, split = lid / tiles;
  const int n0 = (tile / g.KT) * WT, k0 = (tile % g.KT) * WT;
  const long long mb = (long long)split * g.rows, me = mb + g.rows < g.M ? mb + g.rows : g.M;
  const int cv = t & 15, r0 = t >> 4;                    // this thread's 8 columns and its first row of a stage
  const int kb = k0 >> 7;

  f32x4_t acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  typedef s16x4_t __attribute__((address_space(3))) * lds_v4;
  auto trload = [&](const bf16_t* p) {
    union { struct { s16x4_t lo, hi; } s; b16x8_t v; } u;
    u.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p));
    u.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p + 4 * WLD));
    return u.v;
  };
  for (long long m = mb; m < me; m += WR) {
    float gv[4][8];
    uint2 xq[4];
    unsigned char xs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long r = m + r0 + 16 * i, rc = r < me ? r : me - 1;
      const T* row = reinterpret_cast<const T*>(g.G) + rc * g.ldg;
      const int n = n0 + cv * 8;
      if (VEC) {
        ld8<T>(row + (n < g.N ? n : 0), gv[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) gv[i][j] = to_f<T>(row[n + j < g.N ? n + j : 0]);
      }
      xq[i] = *reinterpret_cast<const uint2*>(g.X + rc * g.Kp + k0 + cv * 8);
      xs[i] = g.Xs[rc * g.Sp + kb];
#pragma unroll
      for (int j = 0; j < 8; ++j) gv[i][j] = r < me && n + j < g.N ? gv[i][j] : 0.f;
      if (r >= me) xq[i] = make_uint2(0, 0);
    }
    __syncthreads();                                    // the previous stage has been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = (r0 + 16 * i) * WLD + cv * 8;
      uint4 piece[P];
      split8<P>(gv[i], piece);
#pragma unroll
      for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(Gs[p] + o) = piece[p];
      const float s = p8_pow2((int)xs[i] - 127);
      union { bf2_t h[4]; uint4 u; } x;
      x.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xq[i].x, s, false);
      x.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xq[i].x, s, true);
      x.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xq[i].y, s, false);
      x.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xq[i].y, s, true);
      *reinterpret_cast<uint4*>(Xl + o) = x.u;
    }
    __syncthreads();
#pragma unroll
    for (int mc = 0; mc < WR / 32; ++mc) {
      const int row = (mc * 32 + lq * 8 + (li >> 2)) * WLD + (li & 3) * 4;
      b16x8_t xf[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) xf[b] = trload(Xl + row + (wk * 4 + b) * 16);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const b16x8_t gf = trload(Gs[p] + row + (wn * 4 + a) * 16);
#pragma unroll
          for (int b = 0; b < 4; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(gf, xf[b], acc[a][b], 0, 0, 0);
        }
    }
  }
  float* out = g.out + (long long)split * g.plane;
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + (wn * 4 + a) * 16 + lq * 4 + r;
      if (n >= g.N) continue;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int k = k0 + (wk * 4 + b) * 16 + li;
        float* p = out + (long long)n * g.ldo + k;
        if (k < g.K) *p = acc[a][b][r] + (g.accumulate ? *p : 0.f);
      }
    }
}

// dW (+)= the S partial products, in order
__global__ __launch_bounds__(256) void wgrad8_join_kernel(const float* part, int S, long long plane, float* dW, long long ldw, int N, int K, int accumulate) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= plane) return;
  const long long n = i / K;
  float v = 0.f;
  for (int s = 0; s < S; ++s) v += part[s * plane + i];
  float* p = dW + n * ldw + (i - n * K);
  *p = v + (accumulate ? *p : 0.f);
}

struct Split { int S; long long rows; };
// at least 512 workgroups where the rows allow it (two on each of the 256 compute units), and at least four stages in each
inline Split split_of(long long M, int N, int K) {
  const long long tiles = (long long)((N + WT - 1) / WT) * ((K + WT - 1) / WT), stages = (M + WR - 1) / WR;
  long long S = 512 / tiles;
  if (S > stages / 4) S = stages / 4;
  if (S < 1) S = 1;
  const long long per = (stages + S - 1) / S;
  return {(int)((stages + per - 1) / per), per * WR};
}
template <typename T, int P> void run(const Wgrad8Args& g, unsigned blocks, bool vec, hipStream_t s) {
  if (vec) hipLaunchKernelGGL((wgrad8_kernel<T, P, true>), dim3(blocks), dim3(256), 0, s, g);
  else hipLaunchKernelGGL((wgrad8_kernel<T, P, false>), dim3(blocks), dim3(256), 0, s, g);
}
__global__ __launch_bounds__(256) void wgrad8_zero_kernel(float* dW, long long ldw, int N, int K) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long n = i / K;
  if (n < N) dW[n * ldw + (i - n * K)] = 0.f;
}

}  // namespace

extern "C" long long spb_gemm8_wgrad_bytes(int dtype, long long M, int N, int K) {
  if ((dtype != SPB_F32 && dtype != SPB_BF16) || M < 0 || N < 0 || K < 0) return SPB_E_SHAPE;
  if (M == 0 || N == 0 || K == 0) return 0;
  const Split sp = split_of(M, N, K);
  return sp.S > 1 ? (long long)sp.S * N * K * 4 : 0;
}

extern "C" int spb_gemm8_wgrad(int dtype, const spb_wgrad8_args_t* a, spb_stream_t stream) {
  if (!a || (dtype != SPB_F32 && dtype != SPB_BF16)) return SPB_E_ARG;
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->ldg < 0 || (a->N > 1 && a->ldw < a->K)) return SPB_E_SHAPE;
  if (a->N == 0 || a->K == 0) return 0;
  if (!a->dW) return SPB_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  const long long blocks1 = ((long long)a->N * a->K + 255) / 256;
  if (blocks1 > 0x7fffffffll) return SPB_E_SHAPE;
  if (a->M == 0) {
    if (!a->accumulate) hipLaunchKernelGGL(wgrad8_zero_kernel, dim3((unsigned)blocks1), dim3(256), 0, s, a->dW, a->ldw, a->N, a->K);
    SPB_CHECK_LAUNCH();
    return 0;
  }
  if (!a->G || !a->X || !a->Xs || ((uintptr_t)a->X & 15) || ((uintptr_t)a->Xs & 3)) return SPB_E_ARG;
  const Split sp = split_of(a->M, a->N, a->K);
  if (sp.S > 1 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < spb_gemm8_wgrad_bytes(dtype, a->M, a->N, a->K))) return SPB_E_ARG;
  const int es = dtype == SPB_F32 ? 4 : 2;
  const bool vec = a->N % 8 == 0 && ((uintptr_t)a->G & 15) == 0 && (a->ldg * es) % 16 == 0;
  const long long plane = (long long)a->N * a->K;
  Wgrad8Args g = {a->G, a->X, a->Xs, sp.S > 1 ? (float*)a->ws : a->dW, a->M, a->ldg, sp.S > 1 ? a->K : a->ldw, sp.S > 1 ? plane : 0, sp.rows, a->N, a->K,
                  p8_cols(a->K), p8_scales(a->K), (a->N + WT - 1) / WT, (a->K + WT - 1) / WT, sp.S > 1 ? 0 : a->accumulate};
  const long long blocks = (long long)g.NT * g.KT * sp.S;
  if (blocks > 0x7fffffffll) return SPB_E_SHAPE;
  if (dtype == SPB_F32) run<float, 3>(g, (unsigned)blocks, vec, s);
#ifdef SPB_F16
  else run<bf16_t, 2>(g, (unsigned)blocks, vec, s);
#else
  else run<bf16_t, 1>(g, (unsigned)blocks, vec, s);
#endif
  SPB_CHECK_LAUNCH();
  if (sp.S > 1) {
    hipLaunchKernelGGL(wgrad8_join_kernel, dim3((unsigned)blocks1), dim3(256), 0, s, (const float*)a->ws, sp.S, plane, a->dW, a->ldw, a->N, a->K, a->accumulate);
    SPB_CHECK_LAUNCH();
  }
  return 0;
}
