// Product of two packed 8-bit matrices (format: include/spb_hip.h "8-bit packing"):  Y[m,n] = sum_k A[m,k] B[n,k] + bias[n].
//
// The scales of a block of 128 are powers of two, the reduction step of v_mfma_scale_f32_16x16x128_f8f6f4 is 128 deep, and the instruction
// multiplies by 2^(ea - 127) 2^(eb - 127) itself: a step of a tile is one instruction, and the sums of all blocks stay in one f32 accumulator.
//   * Both operands go global -> LDS by LDS-DMA, 128 bytes of a row for each step, two or four stages.  The 16-byte slots of a row are XOR-swizzled with
//     (row & 7) on the source address, so the lane-linear DMA image is read back without bank conflicts.
//   * The scales of four steps are one dword a row: they ride the same DMA every fourth step.
//   * The instruction's first operand is B: a lane then holds four neighbouring columns of one row of Y.
// EXACT (f32 output): the 8-bit instruction aligns each 8 neighbouring products to the largest of them and drops what lies below 2^-13 of it (measured;
// products further apart and the accumulator keep 24 bits).  On normal data that is 1.4e-5 of the result's rms, 4e-5 with channels 16 times the
// others, whatever K: far below the rounding of a 16-bit output, but not below f32's.  The parity mode converts the codes to bfloat16 (exact, scale
// included) and uses the bfloat16 instructions.  So do all products of up to 16 rows: they wait for B's bytes, and it costs 2 to 5 % there (1 x 4096 x 4096 6.0 -> 6.2 us from HBM,
// 16 x 9216 x 9216 29.6 -> 30.9); 48 x 4096 x 9216 would go from 14.2 to 16.9, 16384 x 4096 x 4096 from 207 to 424.
#include "pack8.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;

struct Gemm8Args {
  const unsigned char* A; const unsigned char* As; const unsigned char* B; const unsigned char* Bs;
  const float* bias; void* Y;
  long long M, ldy;
  long long plane;       // distance of two splits' outputs; 0: one split
  int N, Kp, Sp, bshift;
  int steps;             // steps of the reduction for each split
};

// 8 of a lane's 32 codes as bfloat16 values.  A and B give the same 8, so any order of the reduction will do.
__device__ __forceinline__ b16x8_t wide8(const i32x8_t& f, int h, float s) {
  union { bf2_t p[4]; b16x8_t v; } o;
  o.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h], s, false);
  o.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h], s, true);
  o.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h + 1], s, false);
  o.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * h + 1], s, true);
  return o.v;
}
__device__ __forceinline__ float scale_of(unsigned byte) { return p8_pow2((int)(byte & 255u) - 127); }

// LDS-DMA (16 / 4 bytes a lane, lane i behind lds_base in order); m0 is not saved: nothing in these kernels uses it
__device__ __forceinline__ void dma16m(const void* sbase, unsigned voff, unsigned lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ void dma4m(const void* sbase, unsigned voff, unsigned lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase), "s"(lds_base) : "memory", "m0");
}

// bias, rounding and the store of V neighbouring columns of a row, at any alignment
template <int V, typename TO> __device__ __forceinline__ void put(const Gemm8Args& g, TO* Y, long long m, int n, const f32x4_t* acc, const float bias[V]) {
  float v[V];
#pragma unroll
  for (int r = 0; r < V; ++r) v[r] = acc[r / 4][r % 4] + bias[r];
  TO* p = Y + m * g.ldy + n;
  if (n + V <= g.N) {
    if constexpr (sizeof(TO) == 4) __builtin_memcpy(p, v, V * 4);
    else {
      unsigned u[V / 2];
#pragma unroll
      for (int r = 0; r < V / 2; ++r) u[r] = pack_bf16x2(v[2 * r], v[2 * r + 1]);
      __builtin_memcpy(p, u, V * 2);
    }
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r)
      if (n + r < g.N) p[r] = from_f<TO>(v[r]);
  }
}
template <int V> __device__ __forceinline__ void bias_of(const Gemm8Args& g, int n, float bias[V]) {
#pragma unroll
  for (int r = 0; r < V; ++r) bias[r] = g.bias != nullptr && n + r < g.N ? g.bias[n + r] : 0.f;
}

constexpr int BAND = 8;      // tile rows that are walked together
// BM x BN tile, WM x WN waves, a ring of NST stages
template <int BM, int BN, int WM, int WN, int NST, bool EXACT, typename TO>
__global__ __launch_bounds__(WM * WN * 64) void gemm8_kernel(const Gemm8Args g) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int TILE = (BM + BN) * 128, STAGE = TILE + (BM + BN) * 4;   // codes, then the dword of scales that holds this step's
  // Eight waves: the upper four, one on each SIMD, fetch at the head of a step, while the other four, whose instructions go first, multiply.  (All eight
  // fetching between their products: 8192 x 8192 x 8192 419 us, like this 381; f32 16384 x 4096 x 4096 482 and 432; a wave that waits for a DMA instruction to be taken issues no product.)
  constexpr bool LEAD = NW == 8;
  constexpr int DW = LEAD ? NW / 2 : NW, DI = (BM + BN) / 8 / DW;       // waves that fetch; DMA instructions of a stage for each: 8 rows of codes
  constexpr int ST = (BM + BN) / 64, SI = (ST + DW - 1) / DW;           // and 64 rows of scales each (a wave too many repeats an instruction)
  static_assert(DI * 8 * DW == BM + BN && ST * 64 == BM + BN, "whole DMA instructions");
  // 16-bit output: the 16 rows of B in a pair of column tiles alternate in fours, so that a lane holds eight neighbouring columns and four lanes 64 bytes
  constexpr bool PAIR = sizeof(TO) == 2;
  static_assert(!PAIR || (TN % 2 == 0 && NW % 2 == 0), "pairs of column tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int t = threadIdx.x, l = t & 63, li = l & 15, lq = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / WN, wn = w % WN, wd = w % DW;
  // The 32 workgroups that an XCD runs at a time share one L2: eight tile rows times four tile columns of them fetch 12 tiles a step where a line of
  // 32 fetches 33 (8192 x 8192 x 8192: 4 TB/s out of the L2s' misses, half the matrix cores' time spent waiting).
  const int NT = (g.N + BN - 1) / BN, MT = (int)((g.M + BM - 1) / BM);
  const int tiles = MT * NT, wg = xcd_remap(blockIdx.x, gridDim.x), split = wg / tiles;
  const int lid = wg - split * tiles, band = lid / (BAND * NT), in = lid - band * (BAND * NT);
  const int rows = MT - band * BAND < BAND ? MT - band * BAND : BAND;
  const long long m0 = (long long)(band * BAND + in % rows) * BM;
  const int n0 = in / rows * BN;
  const int kbeg = split * g.steps, KT = ((g.Kp >> 7) - kbeg < g.steps ? (g.Kp >> 7) - kbeg : g.steps);     // g.steps is a multiple of 4

  // DMA roles: row r of the stage (A rows, then B rows); rows behind the matrix repeat its last one (their results are not stored)
  const unsigned lds0 = lds_addr(smem);
  const char* abase = reinterpret_cast<const char*>(g.A) + m0 * g.Kp + (long long)kbeg * 128;
  const char* bbase = reinterpret_cast<const char*>(g.B) + (long long)n0 * g.Kp + (long long)kbeg * 128;
  const int mlast = (int)(g.M - 1 - m0 < BM - 1 ? g.M - 1 - m0 : BM - 1), nlast = g.N - 1 - n0 < BN - 1 ? g.N - 1 - n0 : BN - 1;
  const int slot = ((l & 7) ^ (l >> 3)) << 4, slotb = PAIR ? ((l & 7) ^ ((l >> 3 & 3) | (wd & 1) << 2)) << 4 : slot;
  unsigned off[DI], soff[SI];
#pragma unroll
  for (int i = 0; i < DI; ++i) {
    const int r = (i * DW + wd) * 8 + (l >> 3);
    const int rc = r < BM ? (r < mlast ? r : mlast) : (r - BM < nlast ? r - BM : nlast);
    off[i] = (unsigned)rc * (unsigned)g.Kp + (unsigned)((i * DW + wd) * 8 < BM ? slot : slotb);
  }
  const char* asb = reinterpret_cast<const char*>(g.As) + m0 * g.Sp + kbeg;
  const char* bsb = reinterpret_cast<const char*>(g.Bs) + (long long)(n0 >> g.bshift) * g.Sp + kbeg;
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const int r = (i * DW + wd) % ST * 64 + l;
    const int rc = r < BM ? (r < mlast ? r : mlast) : (r - BM < nlast ? r - BM : nlast);
    soff[i] = (unsigned)(r < BM ? rc : ((n0 + rc) >> g.bshift) - (n0 >> g.bshift)) * (unsigned)g.Sp;
  }
  // DMA instruction i of stage kt into buffer `buf`: DI of codes, then SI of scales
  auto issue1 = [&](int i, int kt, int buf) {
    const unsigned sb = lds0 + (unsigned)(buf * STAGE);
    if (i < DI) {
      const int r0 = (i * DW + wd) * 8;
      dma16m((r0 < BM ? abase : bbase) + (size_t)kt * 128, off[i < DI ? i : 0], sb + (unsigned)(r0 * 128));
    } else if (EXACT || NST > 2 || (kt & 3) == 0) {        // (two stages, products: the dwords are read in the step they belong to only)
      const int r0 = ((i - DI) * DW + wd) % ST * 64;
      dma4m((r0 < BM ? asb : bsb) + (kt & ~3), soff[i < DI ? 0 : i - DI], sb + (unsigned)(TILE + r0 * 4));
    }
  };
  auto issue = [&](int kt, int buf) {
    if (LEAD && w >= DW) return;
#pragma unroll
    for (int i = 0; i < DI + SI; ++i) issue1(i, kt, buf);
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

  // this wave's share of stage kt has landed once only the stages behind it are in flight; behind the barrier everybody's has, and everybody is done
  // with stage kt - 1, whose buffer takes stage kt + NST - 1
  auto land = [&](int kt) {
    if (NST > 2 && kt + NST - 2 < KT) wait_vmcnt<(NST - 2) * (DI + SI)>();
    else if (NST > 3 && kt + 1 < KT) wait_vmcnt<DI + SI>();
    else wait_vmcnt<0>();
    lds_barrier();
  };
  const int ao = (wm * TM * 16 + li) * 128, bl = wn * TN * 16 + (PAIR ? (li >> 2) * 8 + (li & 3) : li), bo = BM * 128 + bl * 128;
  const int ato = TILE + (wm * TM * 16 + li) * 4, bto = TILE + (BM + bl) * 4;
  auto brow = [](int j) { return PAIR ? (j >> 1) * 32 + (j & 1) * 4 : j * 16; };      // row of column tile j behind this lane's first
  for (int s = 0; s < NST - 1 && s < KT; ++s) issue(s, s);
  int buf = 0;
  land(0);
  if constexpr (!EXACT) {
    // The operands of row tile i + 1 are read while row tile i is multiplied.  Where every wave fetches, the next stage's DMA goes out between them: at the head of
    // the step its instructions would keep the first operand reads waiting.
    int sa[TM], sb[TN];
    if (LEAD && w >= DW) __builtin_amdgcn_s_setprio(1);
    constexpr int PER = (DI + SI + TM - 1) / TM;
    for (int kt = 0; kt < KT; ++kt) {
      if (kt > 0) land(kt);
      const char* stage = smem + buf * STAGE;
      const int nbuf = buf == 0 ? NST - 1 : buf - 1;
      const bool more = kt + NST - 1 < KT;
      buf = buf == NST - 1 ? 0 : buf + 1;
      i32x8_t b[TN], a[2];
      if (LEAD && more) issue(kt + NST - 1, nbuf);
      a[0] = frag(stage + ao);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = frag(stage + bo + brow(j) * 128);
      if ((kt & 3) == 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j) sb[j] = *reinterpret_cast<const int*>(stage + bto + brow(j) * 4);
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = *reinterpret_cast<const int*>(stage + ato + i * 64);
      } else {
#pragma unroll
        for (int j = 0; j < TN; ++j) sb[j] = (int)((unsigned)sb[j] >> 8);
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = (int)((unsigned)sa[i] >> 8);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i + 1 < TM) a[(i + 1) & 1] = frag(stage + ao + (i + 1) * 2048);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a[i & 1], acc[i][j], 0, 0, 0, sb[j], 0, sa[i]);
        if (!LEAD && more) {
#pragma unroll
          for (int q = i * PER; q < (i + 1) * PER && q < DI + SI; ++q) issue1(q, kt + NST - 1, nbuf);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
    // B's values of a step are converted once, A's a row tile at a time, while the one before is multiplied
    if (LEAD && w >= DW) __builtin_amdgcn_s_setprio(1);
    for (int kt = 0; kt < KT; ++kt) {
      if (kt > 0) land(kt);
      if (kt + NST - 1 < KT) issue(kt + NST - 1, buf == 0 ? NST - 1 : buf - 1);
      const char* stage = smem + buf * STAGE;
      buf = buf == NST - 1 ? 0 : buf + 1;
      const int sh = (kt & 3) * 8;
      i32x8_t a[2];
      float fa[2];
      b16x8_t wb[TN][4];
      a[0] = frag(stage + ao);
      fa[0] = scale_of(*reinterpret_cast<const unsigned*>(stage + ato) >> sh);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const i32x8_t b = frag(stage + bo + brow(j) * 128);
        const float fb = scale_of(*reinterpret_cast<const unsigned*>(stage + bto + brow(j) * 4) >> sh);
#pragma unroll
        for (int h = 0; h < 4; ++h) wb[j][h] = wide8(b, h, fb);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i + 1 < TM) {
          a[(i + 1) & 1] = frag(stage + ao + (i + 1) * 2048);
          fa[(i + 1) & 1] = scale_of(*reinterpret_cast<const unsigned*>(stage + ato + (i + 1) * 64) >> sh);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const b16x8_t wa = wide8(a[i & 1], h, fa[i & 1]);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j][h], wa, acc[i][j], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  constexpr int V = PAIR ? 8 : 4;
  TO* Y = reinterpret_cast<TO*>(g.Y) + split * g.plane;
#pragma unroll
  for (int j = 0; j < TN; j += V / 4) {
    const int n = n0 + wn * TN * 16 + j * 16 + lq * V;
    float bias[V];
    bias_of<V>(g, n, bias);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const long long m = m0 + (wm * TM + i) * 16 + li;
      if (m >= g.M) continue;
      if constexpr (V == 4) {
        if (g.plane) {
          if (n < g.ldy) p8_put_part(reinterpret_cast<float*>(Y) + m * g.ldy + n, acc[i][j]);
          continue;
        }
      }
      put<V, TO>(g, Y, m, n, &acc[i][j], bias);
    }
  }
}

// Few rows (M <= 16): the product is a stream of B.  A workgroup takes 16 columns of Y and its sixteen waves every sixteenth pair of steps of the reduction:
// 256 bytes of each row, straight from memory in operand layout, all requested before the first is used.  No wave prefetches; four on each SIMD
// cover each other.  A comes through L2.  The waves' sums meet in LDS, in order.  (With more rows the half lines that this layout loads of A cost more
// than the tiles' way through LDS: 48 x 4096 x 9216 took 20 us with three row tiles.)
constexpr int SKW = 16;
template <typename TO>
__global__ __launch_bounds__(SKW * 64) void gemm8_rows_kernel(const Gemm8Args g) {
  __shared__ __attribute__((aligned(16))) f32x4_t part[SKW][64];
  const int t = threadIdx.x, l = t & 63, li = l & 15, lq = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n0 = blockIdx.x * 16, KT = g.Kp >> 7;
  const int n = n0 + li < g.N ? n0 + li : g.N - 1;
  const unsigned char* brow = g.B + (long long)n * g.Kp + lq * 16;
  const unsigned char* bsc = g.Bs + (long long)(n >> g.bshift) * g.Sp;
  const long long m = li < g.M ? li : g.M - 1;
  const unsigned char* arow = g.A + m * g.Kp + lq * 16;
  const unsigned char* asc = g.As + m * g.Sp;
  union F { uint4 u[2]; i32x8_t v; };
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int kt = 2 * w; kt < KT; kt += 2 * SKW) {
    const int k1 = kt + 1 < KT ? kt + 1 : kt;            // an odd number of steps: the last pair is one
    F b[2], a[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long o = (long long)(u ? k1 : kt) * 128;
      b[u].u[0] = *reinterpret_cast<const uint4*>(brow + o);
      b[u].u[1] = *reinterpret_cast<const uint4*>(brow + o + 64);
      a[u].u[0] = *reinterpret_cast<const uint4*>(arow + o);
      a[u].u[1] = *reinterpret_cast<const uint4*>(arow + o + 64);
    }
    const unsigned sb = *reinterpret_cast<const unsigned short*>(bsc + kt);            // rows of scales hold a multiple of four
    const unsigned sa = *reinterpret_cast<const unsigned short*>(asc + kt);
    __builtin_amdgcn_sched_barrier(0);                                  // left alone, the compiler trades the loads in flight for fewer registers
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && kt + 1 >= KT) break;
      const float fb = scale_of(sb >> (8 * u)), fa = scale_of(sa >> (8 * u));
#pragma unroll
      for (int h = 0; h < 4; ++h) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide8(b[u].v, h, fb), wide8(a[u].v, h, fa), acc, 0, 0, 0);
    }
  }
  part[w][l] = acc;
  __syncthreads();
  if (w == 0) {
    f32x4_t v = part[0][l];
#pragma unroll
    for (int k = 1; k < SKW; ++k) v += part[k][l];
    const int nn = n0 + lq * 4;
    float bias[4];
    bias_of<4>(g, nn, bias);
    if (li < g.M) put<4, TO>(g, reinterpret_cast<TO*>(g.Y), li, nn, &v, bias);
  }
}

// Y = the S partial products + bias: four columns a thread, partial rows hold a multiple of four
template <typename TO, int GR> __global__ __launch_bounds__(256) void gemm8_join_kernel(const Gemm8Args g, const float* part, int S) {
  long long i;
  float4 x;
  if (!p8_sum_parts<GR>(part, S, g.plane, i, x)) return;
  const int q = (g.N + 3) >> 2;
  const long long m = i / q;
  const int n = (int)(i - m * q) * 4;
  const f32x4_t v = {x.x, x.y, x.z, x.w};
  float bias[4];
  bias_of<4>(g, n, bias);
  put<4, TO>(g, reinterpret_cast<TO*>(g.Y), m, n, &v, bias);
}

// no reduction (K == 0): the bias alone
template <typename TO> __global__ __launch_bounds__(256) void gemm8_bias_kernel(const Gemm8Args g) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < g.M * g.N; i += (long long)gridDim.x * 256) {
    const long long m = i / g.N;
    const int n = (int)(i - m * g.N);
    reinterpret_cast<TO*>(g.Y)[m * g.ldy + n] = from_f<TO>(g.bias ? g.bias[n] : 0.f);
  }
}

template <int BM, int BN, int WM, int WN, int NST, bool EXACT, typename TO> int run(const Gemm8Args& g, int S, hipStream_t s) {
  constexpr int LDS = NST * (BM + BN) * 132;
  const long long wgs = (g.M + BM - 1) / BM * ((g.N + BN - 1) / BN) * S;
  if (!p8_fits(wgs, WM * WN * 64)) return SPB_E_SHAPE;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm8_kernel<BM, BN, WM, WN, NST, EXACT, TO>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL((gemm8_kernel<BM, BN, WM, WN, NST, EXACT, TO>), dim3((unsigned)wgs), dim3(WM * WN * 64), LDS, s, g);
  SPB_CHECK_LAUNCH();
  return 0;
}

// the rows kernel: few rows, and columns for which a launch has threads
inline bool by_rows(long long M, int N) { return M <= 16 && p8_fits((N + 15) / 16, SKW * 64); }
// How a product is cut.  From 144 tiles of 128 x 128 on those or 256 x 256 ones are taken, whichever is estimated to end first: rounds of workgroups over the
// 256 compute units, two of the small tile on each, times a round of KT steps.  Fitted to 130 sizes, in us: large tile 8.4 + 1.2 KT (f32 17.5 + 2.65 KT), small one
// 3.2 + 0.75 KT (f32 8 + 1.55 KT, and 0.65 of that in a last round of one workgroup a compute unit).  Filled tiles and long reductions favour the large one, sides that
// leave part of it empty, or start another round, the small one.  Measured, 256 against 128: 16384 x 4096 x 4096 210 / 255, 2816 x 4096 x 4096 49 / 54,
// 37632 x 700 x 4096 101 / 111, f32 16384 x 896 x 4096 111 / 121; 150528 x 24 x 144 24 / 14, 37632 x 64 x 1024 17 / 11, 37632 x 384 x 4096 87 / 59,
// 2048 x 4096 x 2048 27 / 19, f32 16384 x 2304 x 4096 306 / 274, f32 300 x 40000 x 1024 78 / 41.
// f32 with a side of at most 64 takes 64 x 64 tiles, which convert nothing that is not used (150528 x 24 x 144: 20.5 us, 128: 22.9; 37632 x 64 x 1024 16.3 / 21.4; 16-bit
// results gain nothing: 13.9 / 13.8, 11.2 / 10.7).
// Smaller products take 64 x 64 tiles (2048 x 1024 x 1024, 128 tiles of 128: 7.0 us against 8.3; 2352 x 1024 x 1024, 152 tiles: 10.1 against 8.4), and where even these are fewer than 256 the reduction is split into parts of at least four
// steps, whose sums a second launch adds up, if the steps saved (0.29 us each) are
// worth that launch (3.5 us) and the partial sums' way out and back at 3.5 TB/s: 48 x 4096 x 9216 in four parts 12.4 us, in one 21.7, 300 x 512 x 4096 9.3 and
// 11.1, but 4096 x 128 x 1024 in two parts 9.2, in one 5.1.
struct Cut { int tile, S, steps; };
inline Cut cut_of(bool exact, long long M, int N, int KT) {
  const long long t256 = (M + 255) / 256 * ((N + 255) / 256), t128 = (M + 127) / 128 * ((N + 127) / 128), t64 = (M + 63) / 64 * ((N + 63) / 64);
  if (t256 >= 1 << 20) return {256, 1, (KT + 3) / 4 * 4};         // smaller tiles would be more threads than a launch holds
  if (t128 >= 144 && !(exact && (M <= 64 || N <= 64))) {
    const long long rest = t128 % 512;
    const double large = (double)((t256 + 255) / 256) * (exact ? 17.5 + 2.65 * KT : 8.4 + 1.2 * KT);
    const double small = ((double)(t128 / 512) + (rest == 0 ? 0. : exact && rest <= 256 ? 0.65 : 1.)) * (exact ? 8. + 1.55 * KT : 3.2 + 0.75 * KT);
    return {large < small ? 256 : 128, 1, (KT + 3) / 4 * 4};
  }
  long long S = t64 >= 256 ? 1 : 256 / t64;
  const int quads = (KT + 3) / 4;
  if (S > quads) S = quads;
  int per = (int)((quads + S - 1) / S);
  S = (quads + per - 1) / per;
  if (S > 1 && (quads - per) * 4 * 0.29 < 3.5 + (double)S * (double)M * N * 8 / 3.5e6) { per = quads; S = 1; }
  return {64, (int)S, per * 4};
}
template <bool EXACT, typename TO> int product(const Gemm8Args& g, void* ws, hipStream_t s) {
  if (by_rows(g.M, g.N)) {
    hipLaunchKernelGGL((gemm8_rows_kernel<TO>), dim3((unsigned)((g.N + 15) / 16)), dim3(SKW * 64), 0, s, g);
    SPB_CHECK_LAUNCH();
    return 0;
  }
  const Cut c = cut_of(EXACT, g.M, g.N, g.Kp >> 7);
  Gemm8Args h = g;
  h.steps = c.steps;
  if (c.tile == 256) return run<256, 256, 2, 4, 2, EXACT, TO>(h, 1, s);
  if (c.tile >= 128) {
    // more tiles than compute units: two workgroups on each cover each other's waits (3840 x 2048 x 2048: 25.6 -> 22.1 us); fewer: eight waves and four
    // stages do (4096 x 1024 x 4096: 26.7 -> 24.4 us; f32 2352 x 1024 x 1024 17.1 -> 16.2).  f32 in two workgroups: four waves convert less (45.6 -> 43.4 us).
    if ((g.M + 127) / 128 * ((g.N + 127) / 128) > 256) return run<128, 128, 2, EXACT ? 2 : 4, 2, EXACT, TO>(h, 1, s);
    return run<128, 128, 2, 4, 4, EXACT, TO>(h, 1, s);
  }
  if (c.S == 1) return run<64, 64, 2, 2, 4, EXACT, TO>(h, 1, s);
  const long long q = (g.N + 3) / 4;
  h.Y = ws; h.bias = nullptr; h.ldy = 4 * q; h.plane = g.M * h.ldy;
  const int e = run<64, 64, 2, 2, 4, EXACT, float>(h, c.S, s);
  if (e) return e;
  Gemm8Args j = g;
  j.plane = h.plane;
  const dim3 blocks((unsigned)p8_join_blocks(h.plane, c.S));
  if (c.S > P8_JOIN) hipLaunchKernelGGL((gemm8_join_kernel<TO, 16>), blocks, dim3(256), 0, s, j, (const float*)ws, c.S);
  else hipLaunchKernelGGL((gemm8_join_kernel<TO, 1>), blocks, dim3(256), 0, s, j, (const float*)ws, c.S);
  SPB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" long long spb_gemm8_bytes(int dtype, long long M, int N, int K) {
  if ((dtype != SPB_F32 && dtype != SPB_BF16) || M < 0 || N < 0 || N > P8_SIDE_MAX || K < 0 || K > P8_DEPTH_MAX) return SPB_E_SHAPE;
  if (M == 0 || N == 0 || K == 0 || by_rows(M, N)) return 0;
  const Cut c = cut_of(dtype == SPB_F32, M, N, (K + 127) / 128);
  return c.S > 1 ? (long long)c.S * M * ((N + 3) / 4 * 4) * 4 : 0;
}

extern "C" int spb_gemm8(int dtype, const spb_gemm8_args_t* a, spb_stream_t stream) {
  if (!a || (dtype != SPB_F32 && dtype != SPB_BF16) || (a->b_block_rows != 1 && a->b_block_rows != 128)) return SPB_E_ARG;
  if (a->M < 0 || a->N < 0 || a->N > P8_SIDE_MAX || a->K < 0 || a->K > P8_DEPTH_MAX || (a->M > 1 && a->ldy < a->N)) return SPB_E_SHAPE;
  if (a->M == 0 || a->N == 0) return 0;
  if (!a->Y) return SPB_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  Gemm8Args g = {a->A, a->As, a->B, a->Bs, a->bias, a->Y, a->M, a->ldy, 0, a->N, p8_cols(a->K), p8_scales(a->K), a->b_block_rows == 128 ? 7 : 0, 0};
  if (a->K == 0) {
    const long long all = (a->M * a->N + 255) / 256, blocks = all < 1 << 20 ? all : 1 << 20;
    if (dtype == SPB_F32) hipLaunchKernelGGL((gemm8_bias_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, s, g);
    else hipLaunchKernelGGL((gemm8_bias_kernel<bf16_t>), dim3((unsigned)blocks), dim3(256), 0, s, g);
    SPB_CHECK_LAUNCH();
    return 0;
  }
  if (!a->A || !a->As || !a->B || !a->Bs || (((uintptr_t)a->A | (uintptr_t)a->B) & 15) || (((uintptr_t)a->As | (uintptr_t)a->Bs) & 3)) return SPB_E_ARG;
  const long long need = spb_gemm8_bytes(dtype, a->M, a->N, a->K);
  if (need > 0 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < need)) return SPB_E_ARG;
  return dtype == SPB_F32 ? product<true, float>(g, a->ws, s) : product<false, bf16_t>(g, a->ws, s);
}
