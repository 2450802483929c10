// Product of two packed 8-bit matrices (format: include/spb_hip.h "8-bit packing"):  Y[m,n] = sum_k A[m,k] B[n,k] + bias[n].
//
// The scales of a block of 128 are powers of two, the reduction step of v_mfma_scale_f32_16x16x128_f8f6f4 is 128 deep, and the instruction
// multiplies by 2^(ea - 127) 2^(eb - 127) itself: a step of a tile is one instruction, and the sums of all blocks stay in one f32 accumulator.
//   * Both operands go global -> LDS by LDS-DMA, 128 bytes of a row for each step, two stages.  The 16-byte slots of a row are XOR-swizzled with
//     (row & 7) on the source address, so the lane-linear DMA image is read back without bank conflicts.
//   * The scales of four steps are one dword a row: they ride the same DMA every fourth step.
//   * The instruction's first operand is B: a lane then holds four neighbouring columns of one row of Y.
// EXACT (f32 output): the 8-bit instruction aligns each 8 neighbouring products to the largest of them and drops what lies below 2^-13 of it (measured;
// products further apart and the accumulator keep 24 bits).  On normal data that is 1.4e-5 of the result's rms, 4e-5 with channels 16 times the
// others, whatever K: far below the rounding of a 16-bit output, but not below f32's.  The parity mode converts the codes to bfloat16 (exact, scale
// included) and uses the bfloat16 instructions.
#include "pack8.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;

struct Gemm8Args {
  const unsigned char* A; const unsigned char* As; const unsigned char* B; const unsigned char* Bs;
  const float* bias; void* Y;
  long long M, ldy;
  int N, Kp, Sp, bshift, vec;
};

template <typename TO> __device__ __forceinline__ void store4(TO* p, const float v[4]);
template <> __device__ __forceinline__ void store4<float>(float* p, const float v[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t* p, const float v[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// BM x BN tile, WM x WN waves
template <int BM, int BN, int WM, int WN, typename TO>
__global__ __launch_bounds__(WM * WN * 64) void gemm8_kernel(const Gemm8Args g) {
  constexpr bool EXACT = sizeof(TO) == 4;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * 128, DI = (BM + BN) / 8 / NW;       // DMA instructions of a stage for each wave: 8 rows each
  constexpr int SI = (BM + BN) / 64;                                    // DMA instructions of four steps' scales: 64 rows each
  extern __shared__ __attribute__((aligned(16))) char smem[];           // [2] stages, [2] scale tables
  const int t = threadIdx.x, l = t & 63, li = l & 15, lq = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / WN, wn = w % WN;
  const int NT = (g.N + BN - 1) / BN;
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  const long long m0 = (long long)(lid / NT) * BM;
  const int n0 = (lid % NT) * BN;
  const int KT = g.Kp >> 7;

  // DMA roles: row r of the stage (A rows, then B rows); rows behind the matrix repeat its last one (their results are not stored)
  const unsigned lds0 = lds_addr(smem);
  const char* abase = reinterpret_cast<const char*>(g.A) + m0 * g.Kp;
  const char* bbase = reinterpret_cast<const char*>(g.B) + (long long)n0 * g.Kp;
  const int mlast = (int)(g.M - 1 - m0 < BM - 1 ? g.M - 1 - m0 : BM - 1), nlast = g.N - 1 - n0 < BN - 1 ? g.N - 1 - n0 : BN - 1;
  const int slot = ((l & 7) ^ (l >> 3)) << 4;
  unsigned off[DI];
#pragma unroll
  for (int i = 0; i < DI; ++i) {
    const int r = (i * NW + w) * 8 + (l >> 3);
    const int rc = r < BM ? (r < mlast ? r : mlast) : (r - BM < nlast ? r - BM : nlast);
    off[i] = (unsigned)rc * (unsigned)g.Kp + (unsigned)slot;
  }
  const char* asb = reinterpret_cast<const char*>(g.As) + m0 * g.Sp;
  const char* bsb = reinterpret_cast<const char*>(g.Bs) + (long long)(n0 >> g.bshift) * g.Sp;
  auto issue = [&](int kt, int buf) {
    const unsigned sb = lds0 + (unsigned)(buf * STAGE);
#pragma unroll
    for (int i = 0; i < DI; ++i) {
      const int r0 = (i * NW + w) * 8;
      dma16s((r0 < BM ? abase : bbase) + (size_t)kt * 128, off[i], sb + (unsigned)(r0 * 128));
    }
    if ((kt & 3) == 0) {
      for (int i = w; i < SI; i += NW) {
        const int r = i * 64 + l;
        const bool isa = i * 64 < BM;
        const int rc = isa ? (r < mlast ? r : mlast) : (r - BM < nlast ? r - BM : nlast);
        // n0 is a multiple of 128 where blocks share scales (BN is): the block of a row is its distance from n0
        const unsigned so = (unsigned)(isa ? rc : rc >> g.bshift) * (unsigned)g.Sp;
        dma4s((isa ? asb : bsb) + kt, so, lds0 + (unsigned)(2 * STAGE + ((kt >> 2) & 1) * (BM + BN) * 4 + i * 256));
      }
    }
  };

  f32x4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int sw = li & 7;
  const unsigned pos0 = (unsigned)((lq ^ sw) << 4), pos1 = (unsigned)(((lq + 4) ^ sw) << 4);
  auto frag = [&](const char* row) {
    union { uint4 u[2]; i32x8_t v; } f;
    f.u[0] = *reinterpret_cast<const uint4*>(row + pos0);
    f.u[1] = *reinterpret_cast<const uint4*>(row + pos1);
    return f.v;
  };

  issue(0, 0);
  wait_vmcnt<0>();
  lds_barrier();
  unsigned sa[TM], sb[TN];
  for (int kt = 0; kt < KT; ++kt) {
    const int buf = kt & 1;
    if (kt + 1 < KT) issue(kt + 1, buf ^ 1);
    const char* stage = smem + buf * STAGE;
    if ((kt & 3) == 0) {
      const unsigned* tab = reinterpret_cast<const unsigned*>(smem + 2 * STAGE) + ((kt >> 2) & 1) * (BM + BN);
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = tab[(wm * TM + i) * 16 + li];
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] = tab[BM + (wn * TN + j) * 16 + li];
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] >>= 8;
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] >>= 8;
    }
    const char* as = stage + (wm * TM * 16 + li) * 128;
    const char* bs = stage + BM * 128 + (wn * TN * 16 + li) * 128;
    if constexpr (!EXACT) {
      i32x8_t b[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = frag(bs + j * 2048);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const i32x8_t a = frag(as + i * 2048);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a, acc[i][j], 0, 0, 0, (int)sb[j], 0, (int)sa[i]);
      }
    } else {
      // 8 of the lane's 32 codes at a time: the same ones of A and B, so any order of the reduction will do
      auto wide = [&](const i32x8_t& f, int h, float s) {
        union { bf2_t p[4]; b16x8_t v; } o;
        o.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h], s, false);
        o.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h], s, true);
        o.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h + 1], s, false);
        o.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h + 1], s, true);
        return o.v;
      };
      i32x8_t b[TN], a[TM];
      float fa[TM], fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) { b[j] = frag(bs + j * 2048); fb[j] = p8_pow2((int)(sb[j] & 255u) - 127); }
#pragma unroll
      for (int i = 0; i < TM; ++i) { a[i] = frag(as + i * 2048); fa[i] = p8_pow2((int)(sa[i] & 255u) - 127); }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        b16x8_t wb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) wb[j] = wide(b[j], h, fb[j]);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const b16x8_t wa = wide(a[i], h, fa[i]);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j], wa, acc[i][j], 0, 0, 0);
        }
      }
    }
    wait_vmcnt<0>();          // this wave's share of the next stage has landed
    lds_barrier();            // everybody's has, and everybody is done with this one
  }

  TO* Y = reinterpret_cast<TO*>(g.Y);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + (wn * TN + j) * 16 + lq * 4;
    float bias[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[r] = g.bias != nullptr && n + r < g.N ? g.bias[n + r] : 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const long long m = m0 + (wm * TM + i) * 16 + li;
      if (m >= g.M) continue;
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] + bias[r];
      TO* p = Y + m * g.ldy + n;
      if (g.vec && n + 4 <= g.N) store4<TO>(p, v);
      else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < g.N) p[r] = from_f<TO>(v[r]);
      }
    }
  }
}

// no reduction (K == 0): the bias alone
template <typename TO> __global__ __launch_bounds__(256) void gemm8_bias_kernel(const Gemm8Args g) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long m = i / g.N;
  const int n = (int)(i - m * g.N);
  if (m < g.M) reinterpret_cast<TO*>(g.Y)[m * g.ldy + n] = from_f<TO>(g.bias ? g.bias[n] : 0.f);
}

template <int BM, int BN, int WM, int WN, typename TO> int run(const Gemm8Args& g, hipStream_t s) {
  constexpr int LDS = 2 * (BM + BN) * 128 + 2 * (BM + BN) * 4;
  const long long tiles = (g.M + BM - 1) / BM * ((g.N + BN - 1) / BN);
  if (tiles > 0x7fffffffll) return SPB_E_SHAPE;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm8_kernel<BM, BN, WM, WN, TO>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL((gemm8_kernel<BM, BN, WM, WN, TO>), dim3((unsigned)tiles), dim3(WM * WN * 64), LDS, s, g);
  SPB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" long long spb_gemm8_bytes(int dtype, long long M, int N, int K) {
  if ((dtype != SPB_F32 && dtype != SPB_BF16) || M < 0 || N < 0 || K < 0) return SPB_E_SHAPE;
  return 0;
}

extern "C" int spb_gemm8(int dtype, const spb_gemm8_args_t* a, spb_stream_t stream) {
  if (!a || (dtype != SPB_F32 && dtype != SPB_BF16) || (a->b_block_rows != 1 && a->b_block_rows != 128)) return SPB_E_ARG;
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->K > (1 << 23) || (a->M > 1 && a->ldy < a->N)) return SPB_E_SHAPE;
  if (a->M == 0 || a->N == 0) return 0;
  if (!a->Y) return SPB_E_ARG;
  const int es = dtype == SPB_F32 ? 4 : 2;
  hipStream_t s = (hipStream_t)stream;
  Gemm8Args g = {a->A, a->As, a->B, a->Bs, a->bias, a->Y, a->M, a->ldy, a->N, p8_cols(a->K), p8_scales(a->K), a->b_block_rows == 128 ? 7 : 0,
                 ((uintptr_t)a->Y % (4 * es)) == 0 && a->ldy % 4 == 0};
  if (a->K == 0) {
    const long long blocks = (a->M * a->N + 255) / 256;
    if (blocks > 0x7fffffffll) return SPB_E_SHAPE;
    if (dtype == SPB_F32) hipLaunchKernelGGL((gemm8_bias_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, s, g);
    else hipLaunchKernelGGL((gemm8_bias_kernel<bf16_t>), dim3((unsigned)blocks), dim3(256), 0, s, g);
    SPB_CHECK_LAUNCH();
    return 0;
  }
  if (!a->A || !a->As || !a->B || !a->Bs || (((uintptr_t)a->A | (uintptr_t)a->B) & 15) || (((uintptr_t)a->As | (uintptr_t)a->Bs) & 3)) return SPB_E_ARG;
  return dtype == SPB_F32 ? run<128, 128, 2, 2, float>(g, s) : run<128, 128, 2, 2, bf16_t>(g, s);
}
