// Weight gradient from an 8-bit checkpoint:  dW[n,k] (+)= sum_m G[m,n] X[m,k],  X packed by rows (include/spb_hip.h "8-bit packing").
//
// A value code * 2^e is exact in bfloat16, so X becomes bfloat16 on its way into LDS (one instruction for two values, scale included) and the
// products run on the bfloat16 matrix cores at half the bytes a 16-bit activation would cost.  The reduction index m is the row of both operands;
// the scale belongs to (m, 128 columns): along the reduction it changes with every step, which is why the 8-bit instructions, whose scale covers 32
// steps of the reduction, do not fit.  G keeps all its bits: it is split by truncation into 1 (bfloat16), 2 (half: 8 + 3 bits) or 3 (float32: 8 + 8 + 8 bits)
// bfloat16 pieces with an exact sum.
//   * Tiles of dW: 256 x 256 with eight waves of 128 x 64, a stage requested ahead; 128 x 128, three stages ahead, with eight waves of 64 x 32; or
//     64 x 64 with four waves of 32 x 32: a stage of the small tiles is multiplied in a fifth of the time that memory takes to answer.
//     Stages of R rows (64; 32 with more than one piece in the larger tiles) in LDS, read with the transpose load ds_read_b64_tr_b16.
//     64 rows of the large tile are 2048 clocks of matrix instructions, and 1536 of reads and 512 of writes in LDS; the two hardly overlap (16384 x 4096 x 4096,
//     counted: matrix cores busy 55 % of the time, LDS 35 %, bank conflicts 7 %).
//   * bfloat16 gradients with 16-byte aligned rows go to LDS by DMA, the others through registers.
//   * Of the two waves on a SIMD one multiplies a stage before it brings the next one into place, the other after it: the matrix cores work while operands are
//     converted (16384 x 4096 x 4096: 459 -> 427 us; 37632 x 1024 x 1280: 183 -> 174).
//   * Few tiles and many rows: the rows are split over workgroups, each stores its partial tile, and a second launch adds them in order.
// LDS rows hold TW columns without padding (the DMA image is linear).  The transpose load reads 32 bytes of 16 rows, r = 8 q + 0 .. 3 (+ 4): the 32-byte
// pairs of a row are XOR-swizzled with (r & 3) + 4 ((r >> 3) & 1), which spreads them over all banks; 64 columns are four pairs, and two rows cover the banks, so
// bits 1 and 3 of r do.
#include "pack8.h"

namespace {

typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;

struct Wgrad8Args {
  const void* G; const unsigned char* X; const unsigned char* Xs; float* out;
  long long M, ldg, ldo, plane;                        // plane: distance of two splits' outputs (0: a single one)
  long long rows;                                      // rows of a split, a multiple of 64
  int N, K, Kp, Sp, NT, KT, accumulate;
};

// bfloat16 pieces of 8 gradients, piece p of all of them in out[p]: the upper half of the bits, then the same of what is left.  The differences are exact.  What is
// subtracted is kept finite: every piece of an infinity is one (inf - inf would make its row of dW NaN where bfloat16 gradients give infinities), and a NaN
// stays one in the second piece whatever its bits.  It costs an instruction an element: f16 16384 x 4096 x 4096 815 -> 823 us, f32 1183 -> 1198.
template <int P> __device__ __forceinline__ void split8(const float v[8], uint4 out[P]) {
  constexpr float TOP = 3.4028234e38f;
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    unsigned u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(r[i]);
    out[p] = make_uint4(__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u),
                        __builtin_amdgcn_perm(u[5], u[4], 0x07060302u), __builtin_amdgcn_perm(u[7], u[6], 0x07060302u));
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] -= __builtin_amdgcn_fmed3f(__uint_as_float(u[i] & 0xffff0000u), -TOP, TOP);
  }
}
// Four neighbouring values of a row (`left` of them inside it), added to what is there or not, at any alignment (element by element: 71 x 3494 x 958
// 14.6 us, like this 9.2).
__device__ __forceinline__ void put4(float* p, f32x4_t v, int left, int accumulate) {
  if (left >= 4) {
    if (accumulate) { f32x4_t o; __builtin_memcpy(&o, p, 16); v += o; }
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) p[r] = v[r] + (accumulate ? p[r] : 0.f);
  }
}
template <int TW> __device__ __forceinline__ int wg_swz(int row) { return TW == 64 ? ((row >> 1) & 1) | ((row >> 2) & 2) : (row & 3) | ((row >> 1) & 4); }

// WN x WK waves of (16 TN) x (16 TK); both sides of the tile are TW wide.  GDMA: G straight to LDS (P == 1, 16-byte aligned rows, MODE 0); otherwise through
// registers (MODE: vec8.h).  Two forms:
//   NST == 2 (large tile): X through registers requested a stage ahead; G by DMA (GDMA) or through registers too.
//   NST > 2 (small tile): codes and scales of X come by DMA into a ring of NST stages and each lane turns what it fetched itself into bfloat16; G by DMA into
//   a ring of its own or through registers.  (Several stages ahead in registers would not do for X: the compiler counts their loads without the DMA
//   between them, and waits for all but the last stage.)
template <typename T, int P, bool GDMA, int MODE, int NST, int WN, int WK, int TN, int TK>
__global__ __launch_bounds__(WN * WK * 64) void wgrad8_kernel(const Wgrad8Args g) {
  constexpr int TW = WN * TN * 16, NW = WN * WK, NTH = NW * 64;
  static_assert(WK * TK * 16 == TW, "square tiles");
  constexpr bool RING = NST > 2;
  static_assert(!GDMA || P == 1, "pieces come from registers");
  constexpr int R = P == 1 || TW == 64 ? 64 : 32, ROWB = TW * 2, PLANE = R * ROWB;
  constexpr int XL = TW / 16, XT = R * XL < NTH ? R * XL : NTH, XR = XT / XL, XP = R / XR;     // lanes of a row of codes (16 each), threads that fetch codes,
                                                                                           // rows of a pass, passes
  constexpr int GL = TW / 8, GRW = NTH / GL, GP = R / GRW;              // the same for 8 gradients a lane
  constexpr int DW = RING ? NW : NW / 2, DI = GDMA ? PLANE / 1024 / DW : 0, RPI = 1024 / ROWB; // direct DMA: waves that issue it (large tile: those that multiply
                                                                        // last), instructions of a stage for each, rows each covers
  constexpr int IPS = DI + (RING ? 2 * XP : 0);
  constexpr int GST = GDMA ? NST : 2 * P;                             // planes of G in LDS
  constexpr int XOFF = GST * PLANE, XRAW = XOFF + 2 * PLANE, XST = XT * XP * 20, XW = XT / 64;
  static_assert(XP * XR == R && GP * GRW == R && (!GDMA || DI * 1024 * DW == PLANE), "whole passes");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // NST > 2: planes of G, two of X, the ring of X;  NST == 2: the planes of G and X of a stage side by side (their reads share address registers)
  auto gplane = [&](int st, int slot) { return smem + (RING ? (GDMA ? slot * PLANE : (st & 1) * (P * PLANE)) : (st & 1) * ((P + 1) * PLANE)); };
  auto xplane = [&](int st) { return smem + (RING ? XOFF + (st & 1) * PLANE : (st & 1) * ((P + 1) * PLANE) + P * PLANE); };
  const int t = threadIdx.x, l = t & 63, li = l & 15, lq = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wn = w / WK, wk = w % WK;
  const bool first = w >= NW / 2;                        // this wave multiplies first
  const int lid = xcd_remap(blockIdx.x, gridDim.x);     // the tiles of a split read the same rows: one XCD, back to back
  const int tiles = g.NT * g.KT, tile = lid % tiles, split = lid / tiles;
  const int n0 = (tile / g.KT) * TW, k0 = (tile % g.KT) * TW;
  const long long mb = (long long)split * g.rows, me = mb + g.rows < g.M ? mb + g.rows : g.M;
  const int nst = (int)((me - mb + R - 1) / R);

  // ---- staging
  const unsigned lds0 = lds_addr(smem);
  const int drow = w * RPI + l / (64 / RPI), dslot = l % (64 / RPI);                         // direct DMA: this lane's row of the first instruction, its 16-byte slot
  int dcol[2];                                             // every other pass has the other half of the swizzle where a pass covers 8 rows
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = n0 + (((dslot >> 1) ^ wg_swz<TW>(drow + i * DW * RPI)) * 2 + (dslot & 1)) * 8;
    dcol[i] = c < g.N ? c : g.N - 8;                       // columns behind the matrix: any (not stored)
  }
  const int xr = t / XL, xc = (t % XL) * 16;
  const int xk = k0 + xc < g.Kp ? k0 + xc : g.Kp - 16;
  const int gr = t / GL, gc = (t % GL) * 8;
  struct Regs { uint4 xq[XP]; unsigned char xs[XP]; Raw8<T> graw[GDMA ? 1 : GP]; } regs;
  auto rows_of = [&](int st) { const long long left = me - (mb + (long long)st * R); return (int)(left < R ? left : R); };
  auto dma = [&](int st, int slot) {                     // what comes by DMA of stage st
    const long long m = mb + (long long)st * R;
    const int last = rows_of(st) - 1;
    if constexpr (GDMA) {
      const char* gb = reinterpret_cast<const char*>(g.G) + m * g.ldg * 2;
#pragma unroll
      for (int i = 0; i < DI; ++i) {
        const int r = drow + i * (DW * RPI), rc = r < last ? r : last;
        dma16s(gb, ((unsigned)rc * (unsigned)g.ldg + (unsigned)dcol[i & 1]) * 2u, lds0 + (unsigned)((RING ? slot * PLANE : (st & 1) * (2 * PLANE)) + (i * DW + w) * 1024));
      }
    }
    if (RING && w < XW) {
      const char* xb = reinterpret_cast<const char*>(g.X) + m * g.Kp;
      const char* sb = reinterpret_cast<const char*>(g.Xs) + m * g.Sp;
#pragma unroll
      for (int i = 0; i < XP; ++i) {
        const int r = xr + i * XR, rc = r < last ? r : last;
        const unsigned to = lds0 + (unsigned)(XRAW + slot * XST);
        dma16s(xb, (unsigned)rc * (unsigned)g.Kp + (unsigned)xk, to + (unsigned)((i * XW + w) * 1024));
        dma4s(sb, (unsigned)rc * (unsigned)g.Sp + (unsigned)((xk >> 7) & ~3), to + (unsigned)(XT * XP * 16 + (i * XW + w) * 256));
      }
    }
  };
  auto fetch = [&](int st) {                             // requests what goes through registers
    const long long m = mb + (long long)st * R;
    const int last = rows_of(st) - 1;
    if constexpr (!GDMA) {
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        const int r = gr + i * GRW, rc = r < last ? r : last, n = n0 + gc;
        const T* row = reinterpret_cast<const T*>(g.G) + (m + rc) * g.ldg;
        if constexpr (MODE == 2) {
          T e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = row[n + j < g.N ? n + j : 0];
          __builtin_memcpy(&regs.graw[i], e, sizeof(regs.graw[i]));
        } else {
          regs.graw[i] = vec_get<T, MODE>(row, n, g.N);
        }
      }
    }
    if constexpr (!RING) {
#pragma unroll
      for (int i = 0; i < XP; ++i) {
        const int r = xr + i * XR, rc = r < last ? r : last;
        regs.xq[i] = *reinterpret_cast<const uint4*>(g.X + (m + rc) * g.Kp + xk);
        regs.xs[i] = g.Xs[(m + rc) * g.Sp + (xk >> 7)];
      }
    }
  };
  auto commit = [&](int st, int slot) {                  // stage st as bfloat16 into its planes; rows behind the last one as zeros
    const int left = rows_of(st);
    if constexpr (!GDMA) {
      char* sb = gplane(st, slot);
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        const int r = gr + i * GRW;
        Raw8<T> raw = regs.graw[i];
        if constexpr (MODE == 1) vec_place<T, MODE>(raw, n0 + gc, g.N);
        float v[8];
        cvt8(raw, v);
        uint4 piece[P];
        split8<P>(v, piece);
#pragma unroll
        for (int p = 0; p < P; ++p)
          *reinterpret_cast<uint4*>(sb + p * PLANE + r * ROWB + (((gc >> 4) ^ wg_swz<TW>(r)) << 5) + ((gc & 8) << 1)) = r < left ? piece[p] : make_uint4(0, 0, 0, 0);
      }
    }
    if (XT < NTH && w >= XW) return;
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int r = xr + i * XR;
      uint4 xq;
      unsigned xs;
      if constexpr (RING) {
        const char* q = smem + XRAW + slot * XST;
        xq = *reinterpret_cast<const uint4*>(q + (i * XT + t) * 16);
        xs = *reinterpret_cast<const unsigned char*>(q + XT * XP * 16 + (i * XT + t) * 4 + ((xk >> 7) & 3));
      } else {
        xq = regs.xq[i];
        xs = regs.xs[i];
      }
      const float s = p8_pow2((int)xs - 127);
      const unsigned c[4] = {xq.x, xq.y, xq.z, xq.w};
      union { bf2_t h[8]; uint4 u[2]; } x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x.h[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r < left ? c[j] : 0u, s, false);
        x.h[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r < left ? c[j] : 0u, s, true);
      }
      // neighbouring lanes are 32 bytes apart: odd ones write their second half first, so that each instruction covers all banks
      char* p = xplane(st) + r * ROWB + (((xc >> 4) ^ wg_swz<TW>(r)) << 5);
      const bool odd = t & 1;
      const uint4 u = x.u[0], v = x.u[1];                // (component by component: a choice between the two would put the array into scratch memory)
      *reinterpret_cast<uint4*>(p + (odd ? 16 : 0)) = make_uint4(odd ? v.x : u.x, odd ? v.y : u.y, odd ? v.z : u.z, odd ? v.w : u.w);
      *reinterpret_cast<uint4*>(p + (odd ? 0 : 16)) = make_uint4(odd ? u.x : v.x, odd ? u.y : v.y, odd ? u.z : v.z, odd ? u.w : v.w);
    }
  };

  // ---- product
  f32x4_t acc[TN][TK];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TK; ++b) acc[a][b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  typedef s16x4_t __attribute__((address_space(3))) * lds_v4;
  const int swz = wg_swz<TW>((lq << 3) + (li >> 2));         // of every row this lane reads
  const int rowo = (lq * 8 + (li >> 2)) * ROWB + (li & 3) * 8;
  auto trload = [&](const char* plane, int mc, int f) {  // 16-column tile f of the 32 rows mc: 8 rows of one column for each lane
    union { struct { s16x4_t lo, hi; } s; b16x8_t v; } u;
    const char* p = plane + mc * (32 * ROWB) + rowo + ((f ^ swz) << 5);
    u.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p));
    u.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p + 4 * ROWB));
    return u.v;
  };
  auto clear = [&](int st, int slot) {                   // direct DMA repeats the last row of a ragged stage: those rows become zeros
    if (GDMA && rows_of(st) < R) {
      for (int i = t + rows_of(st) * (ROWB / 16); i < R * (ROWB / 16); i += NTH) *reinterpret_cast<uint4*>(gplane(st, slot) + i * 16) = make_uint4(0, 0, 0, 0);
      lds_barrier();
    }
  };
  auto multiply = [&](int st, int slot) {
    const char* sb = gplane(st, slot);
    const char* sx = xplane(st);
    if constexpr (RING) {                                 // every operand of the stage is read before the first product: one LDS round trip a stage
      b16x8_t xf[R / 32][TK], gf[R / 32][P * TN];
#pragma unroll
      for (int mc = 0; mc < R / 32; ++mc) {
#pragma unroll
        for (int b = 0; b < TK; ++b) xf[mc][b] = trload(sx, mc, wk * TK + b);
#pragma unroll
        for (int pa = 0; pa < P * TN; ++pa) gf[mc][pa] = trload(sb + pa / TN * PLANE, mc, wn * TN + pa % TN);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int mc = 0; mc < R / 32; ++mc)
#pragma unroll
        for (int pa = 0; pa < P * TN; ++pa)
#pragma unroll
          for (int b = 0; b < TK; ++b) acc[pa % TN][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[mc][b], gf[mc][pa], acc[pa % TN][b], 0, 0, 0);
    } else {
#pragma unroll
      for (int mc = 0; mc < R / 32; ++mc) {
        b16x8_t xf[TK], gf[2];
        gf[0] = trload(sb, mc, wn * TN);
#pragma unroll
        for (int b = 0; b < TK; ++b) xf[b] = trload(sx, mc, wk * TK + b);
#pragma unroll
        for (int pa = 0; pa < P * TN; ++pa) {               // piece pa / TN, row tile pa % TN; the next one's operand is read under these products
          if (pa + 1 < P * TN) gf[(pa + 1) & 1] = trload(sb + (pa + 1) / TN * PLANE, mc, wn * TN + (pa + 1) % TN);
#pragma unroll
          for (int b = 0; b < TK; ++b) acc[pa % TN][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[b], gf[pa & 1], acc[pa % TN][b], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  if constexpr (RING) {
    // NST - 1 stages are in flight.  Before or after stage st is multiplied the buffer of stage st - 1 takes stage st + NST - 1, and this lane's part of stage st + 1, which
    // has landed once only the stages behind it are in flight, goes into its planes.
    // G through registers: the compiler waits for its loads with a count that knows nothing of the DMA, so whatever was requested behind them is waited for
    // too.  The DMA then goes out behind the commit, not in front of it (f32 5472 x 4432 x 640: 198 -> 163 us).
    auto landed = [&](int st) {                          // stages behind st: at most NST - 2 have been requested
      const int behind = nst - 1 - st;
      if (!GDMA) wait_vmcnt<0>();
      else if (behind >= NST - 2) wait_vmcnt<(NST - 2) * IPS>();
      else if (behind == 1) wait_vmcnt<IPS>();
      else wait_vmcnt<0>();
    };
    static_assert(NST == 4, "landed() knows 2, 1 or 0 stages behind");
#pragma unroll
    for (int q = 0; q < NST - 1; ++q)
      if (q < nst) dma(q, q);
    fetch(0);
    landed(0);
    commit(0, 0);
    if (nst > 1) fetch(1);
    lds_barrier();
    int slot = 0;
    for (int st = 0; st < nst; ++st) {
      clear(st, slot);
      const int next = slot == NST - 1 ? 0 : slot + 1;
      if (first) multiply(st, slot);
      if (GDMA && st + NST - 1 < nst) dma(st + NST - 1, slot == 0 ? NST - 1 : slot - 1);
      if (st + 1 < nst) {
        landed(st + 1);
        commit(st + 1, next);
        if (!GDMA && st + NST - 1 < nst) dma(st + NST - 1, slot == 0 ? NST - 1 : slot - 1);
        if (st + 2 < nst) fetch(st + 2);
      }
      if (!first) multiply(st, slot);
      slot = next;
      lds_barrier();
    }
  } else {
    // Before or after stage st is multiplied, stage st + 1 goes into the other buffers, its G by DMA, the rest from registers, which are then requested for
    // stage st + 2.  In this order: the compiler waits for the registers' loads with a count that knows nothing of the DMA, so a DMA in front of the commit
    // would be waited for there.
    if (!first) dma(0, 0);
    fetch(0);
    commit(0, 0);
    if (nst > 1) fetch(1);
    wait_vmcnt<0>();
    lds_barrier();
    for (int st = 0; st < nst; ++st) {
      clear(st, st & 1);
      if (first) multiply(st, st & 1);
      if (st + 1 < nst) {
        commit(st + 1, 0);
        if (!first) dma(st + 1, (st + 1) & 1);
        if (st + 2 < nst) fetch(st + 2);
      }
      if (!first) {
        multiply(st, st & 1);
        // the DMA has landed once only the requests of stage st + 2 (two for each pass over X) are in flight
        if (GDMA) { if (st + 2 < nst) wait_vmcnt<2 * XP>(); else wait_vmcnt<0>(); }
      }
      lds_barrier();
    }
  }
  // a lane holds four neighbouring k of one n
  float* out = g.out + (long long)split * g.plane;
#pragma unroll
  for (int a = 0; a < TN; ++a) {
    const int n = n0 + (wn * TN + a) * 16 + li;
    if (n >= g.N) continue;
#pragma unroll
    for (int b = 0; b < TK; ++b) {
      const int k = k0 + (wk * TK + b) * 16 + lq * 4;
      float* p = out + (long long)n * g.ldo + k;
      f32x4_t v = acc[a][b];
      if (g.plane) {
        if (k < g.ldo) p8_put_part(p, v);
      } else {
        put4(p, v, g.K - k, g.accumulate);
      }
    }
  }
}

// dW (+)= the S partial products: four columns a thread, partial rows hold a multiple of four
template <int GR> __global__ __launch_bounds__(256) void wgrad8_join_kernel(const float* part, int S, long long plane, float* dW, long long ldw, int N, int K, int accumulate) {
  long long i;
  float4 v;
  if (!p8_sum_parts<GR>(part, S, plane, i, v)) return;
  const int q = (K + 3) >> 2;
  const long long n = i / q;
  const int k = (int)(i - n * q) * 4;
  float* p = dW + n * ldw + k;
  put4(p, (f32x4_t){v.x, v.y, v.z, v.w}, K - k, accumulate);
}

// 256 x 256 tiles where at least 192 of them keep the compute units busy and neither side is narrower than half a tile (2352 rows, 256 against 128: f16
// 24 x 50000 116 / 93 us, f32 100 x 50000 158 / 143, bfloat16 alike; f16 200 x 50000 122 / 185; from 2^20 of them on smaller tiles
// would be more threads than a launch holds).  Otherwise 128 x 128 or 64 x 64, the rows split for about 256 workgroups with at
// least four stages of 64 rows each, whichever is estimated to end first: a stage of one piece takes 0.85 or 0.62 us (0.85 for 64 x 64 too where two workgroups
// share a compute unit), two and three pieces take one and a half times and twice as long, and partial products cost a launch of 3.5 us and their way out and
// back at 3.5 TB/s.
// Measured in us, 128 against 64 (rows x N x K): 2352 x 1024 x 1280 24 / 31, 1024 x 1024 x 1024 18 / 12, 4096 x 1024 x 1024 28 / 42, 4096 x 512 x 512 18 / 16,
// 300 x 1024 x 1024 8.9 / 6.2; f16 34 / 42, 21 / 17, 40 / 67, 21 / 20, 12.5 / 7.6; f32 37 / 76, 22 / 19, 42 / 65, 23 / 23, 14 / 8.5.
struct Split { int tile, S; long long rows; };
inline Split split_of(int pieces, long long M, int N, int K) {
  const long long stages = (M + 63) / 64;
  const long long t256 = (long long)((N + 255) / 256) * ((K + 255) / 256);
  if (t256 >= 192 && ((N > 128 && K > 128) || t256 >= 1 << 20)) return {256, 1, stages * 64};
  Split best = {0, 1, 0};
  double least = 0;
  for (int tile = 64; tile <= 128; tile += 64) {
    const long long t = (long long)((N + tile - 1) / tile) * ((K + tile - 1) / tile);
    long long S = 256 / t;
    if (S > stages / 4) S = stages / 4;
    if (S < 1) S = 1;
    const long long per = (stages + S - 1) / S;
    S = (stages + per - 1) / per;
    const long long wgs = t * S;
    const double stage = (tile == 64 ? (wgs <= 256 ? 0.62 : 0.85 * (double)((wgs + 511) / 512)) : 0.85 * (double)((wgs + 255) / 256)) * (1 + pieces) / 2;
    const double us = (double)per * stage + (S > 1 ? 3.5 + (double)S * N * K * 8 / 3.5e6 : 0.);
    if (best.tile == 0 || us < least) { best = {tile, (int)S, per * 64}; least = us; }
  }
  return best;
}
inline int pieces_of(int dtype) {
#ifdef SPB_F16
  return dtype == SPB_F32 ? 3 : 2;
#else
  return dtype == SPB_F32 ? 3 : 1;
#endif
}
inline long long part_plane(int N, int K) { return (long long)N * ((K + 3) / 4 * 4); }

template <typename T, int P, bool GDMA, int MODE, int NST, int WN, int WK, int TN, int TK> int launch(const Wgrad8Args& g, int S, hipStream_t s) {
  constexpr int TW = WN * TN * 16, R = P == 1 || TW == 64 ? 64 : 32, PLANE = R * TW * 2, NTH = WN * WK * 64;
  constexpr int RING = NST > 2 ? NST * (R * TW + R * TW / 4) : 0;      // codes, a dword of scales a lane
  constexpr int LDS = ((GDMA ? NST : 2 * P) + 2) * PLANE + RING;
  static_assert(LDS <= 160 * 1024, "fits a compute unit");
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&wgrad8_kernel<T, P, GDMA, MODE, NST, WN, WK, TN, TK>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL((wgrad8_kernel<T, P, GDMA, MODE, NST, WN, WK, TN, TK>), dim3((unsigned)((long long)g.NT * g.KT * S)), dim3(NTH), LDS, s, g);
  SPB_CHECK_LAUNCH();
  return 0;
}
template <typename T, int P, bool GDMA, int MODE> int run(Wgrad8Args g, const Split& sp, hipStream_t s) {
  g.NT = (g.N + sp.tile - 1) / sp.tile; g.KT = (g.K + sp.tile - 1) / sp.tile;
  if (!p8_fits((long long)g.NT * g.KT * sp.S, 512)) return SPB_E_SHAPE;
  if (sp.tile == 256) return launch<T, P, GDMA, MODE, 2, 2, 4, 8, 4>(g, sp.S, s);
  if (sp.tile == 64) return launch<T, P, GDMA, MODE, 4, 2, 2, 2, 2>(g, sp.S, s);
  return launch<T, P, GDMA, MODE, 4, 2, 4, 4, 2>(g, sp.S, s);
}
template <typename T, int P> int run_regs(const Wgrad8Args& g, const Split& sp, hipStream_t s) {
  const int mode = vec_mode(g.N);
  return mode == 0 ? run<T, P, false, 0>(g, sp, s) : (mode == 1 ? run<T, P, false, 1>(g, sp, s) : run<T, P, false, 2>(g, sp, s));
}
__global__ __launch_bounds__(256) void wgrad8_zero_kernel(float* dW, long long ldw, int N, int K) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)N * K; i += (long long)gridDim.x * 256) {
    const long long n = i / K;
    dW[n * ldw + (i - n * K)] = 0.f;
  }
}

}  // namespace

extern "C" long long spb_gemm8_wgrad_bytes(int dtype, long long M, int N, int K) {
  if ((dtype != SPB_F32 && dtype != SPB_BF16) || M < 0 || N < 0 || N > P8_SIDE_MAX || K < 0 || K > P8_DEPTH_MAX) return SPB_E_SHAPE;
  if (M == 0 || N == 0 || K == 0) return 0;
  const Split sp = split_of(pieces_of(dtype), M, N, K);
  return sp.S > 1 ? (long long)sp.S * part_plane(N, K) * 4 : 0;
}

extern "C" int spb_gemm8_wgrad(int dtype, const spb_wgrad8_args_t* a, spb_stream_t stream) {
  if (!a || (dtype != SPB_F32 && dtype != SPB_BF16)) return SPB_E_ARG;
  if (a->M < 0 || a->N < 0 || a->N > P8_SIDE_MAX || a->K < 0 || a->K > P8_DEPTH_MAX || a->ldg < 0 || (a->N > 1 && a->ldw < a->K)) return SPB_E_SHAPE;
  if (a->N == 0 || a->K == 0) return 0;
  if (!a->dW) return SPB_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (a->M == 0) {
    const long long all = ((long long)a->N * a->K + 255) / 256;
    if (!a->accumulate) hipLaunchKernelGGL(wgrad8_zero_kernel, dim3((unsigned)(all < 1 << 20 ? all : 1 << 20)), dim3(256), 0, s, a->dW, a->ldw, a->N, a->K);
    SPB_CHECK_LAUNCH();
    return 0;
  }
  if (!a->G || !a->X || !a->Xs || ((uintptr_t)a->X & 15) || ((uintptr_t)a->Xs & 3)) return SPB_E_ARG;
  const Split sp = split_of(pieces_of(dtype), a->M, a->N, a->K);
  if (sp.S > 1 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < spb_gemm8_wgrad_bytes(dtype, a->M, a->N, a->K))) return SPB_E_ARG;
  const long long plane = part_plane(a->N, a->K);
  const Wgrad8Args g = {a->G, a->X, a->Xs, sp.S > 1 ? (float*)a->ws : a->dW, a->M, a->ldg, sp.S > 1 ? plane / a->N : a->ldw, sp.S > 1 ? plane : 0, sp.rows, a->N, a->K,
                        p8_cols(a->K), p8_scales(a->K), 0, 0, sp.S > 1 ? 0 : a->accumulate};
  int e;
  if (dtype == SPB_F32) e = run_regs<float, 3>(g, sp, s);
#ifdef SPB_F16
  else e = run_regs<bf16_t, 2>(g, sp, s);
#else
  // by DMA: whole vectors at 16-byte addresses; the offsets of 64 rows fit 32 bits
  else if (a->N % 8 == 0 && ((uintptr_t)a->G & 15) == 0 && a->ldg % 8 == 0 && a->ldg < (1 << 23)) e = run<bf16_t, 1, true, 0>(g, sp, s);
  else e = run_regs<bf16_t, 1>(g, sp, s);
#endif
  if (e) return e;
  if (sp.S > 1) {
    const long long blocks = p8_join_blocks(plane, sp.S);
    if (sp.S > P8_JOIN) hipLaunchKernelGGL((wgrad8_join_kernel<16>), dim3((unsigned)blocks), dim3(256), 0, s, (const float*)a->ws, sp.S, plane, a->dW, a->ldw, a->N, a->K, a->accumulate);
    else hipLaunchKernelGGL((wgrad8_join_kernel<1>), dim3((unsigned)blocks), dim3(256), 0, s, (const float*)a->ws, sp.S, plane, a->dW, a->ldw, a->N, a->K, a->accumulate);
    SPB_CHECK_LAUNCH();
  }
  return 0;
}
