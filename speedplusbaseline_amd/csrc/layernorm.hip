// Layer norm over the last axis of [M, C] rows, forward and backward (spb_layernorm_* in include/spb_hip.h).
//
//   forward    mean = sum x / C,  var = sum (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd gamma + beta
//   backward   h = g gamma,  xh = (x - mean) rstd:   dx = rstd (h - sum(h) / C - xh sum(h xh) / C)
//              dgamma = sum over rows of g xh,  dbeta = sum over rows of g
//
// Both are bound by HBM: the forward reads x and writes y, the backward reads g and x and writes dx, each element once, because a row
// stays in registers between its sums and its output.  The variance is taken from the differences to the mean, not from the sum of
// squares: a row whose mean is far larger than its spread would lose the variance in the subtraction.  Sums over a row are f32.
//   * TPR threads share a row (16, 64 or 256), so that short rows fill a wave (four rows of up to 256 columns) and long rows need no second
//     pass (8192 columns: 32 elements a thread).  Rows longer than that go through memory once per sum (ln_*_long).
//   * Workgroups walk the rows with a stride, gamma and beta stay in registers, and the next row is requested before this one is summed.
//   * dgamma / dbeta: a thread keeps its columns' sums in registers over its rows (f32), the groups of a workgroup join through LDS, a workgroup
//     stores one partial row, and a second launch adds the partial rows in order, both in 64 bits: no atomics, the same bits in every run.
#include "vec8.h"

namespace {

constexpr int LN_REG_MAX = 8192;      // longest row held in registers
constexpr int LN_COLS_MAX = 1 << 30;  // column counters of long rows step past the end
constexpr int LN_SUMS_MAX = (1 << 27) - 64;   // longest row with parameter gradients: the launch that joins their partial rows has 16 threads for each of 2 C sums
constexpr int LN_FWD_WGS = 2048;      // workgroups that walk the rows: eight of 256 threads on each of the 256 compute units
constexpr int LN_BWD_WGS = 512;       // backward: each stores one partial row of 2 C floats, so fewer of them

// The 8 * NV elements of a row that a thread holds.
//   VEC (C a multiple of 8): vectors of 8, a group apart, at any alignment.  Vectors in front of number `last` lie inside the row for every thread, those
//   behind it outside, both the same for the whole launch: only vector `last` is compared with the row's end.
//   Otherwise single elements a group apart: a wave still reads whole lines.  (Vectors at odd addresses, the last one from
//   8 elements in front of the end on, were built and are slower where it matters: backward 16384 x 4095 bfloat16 110 against 96 us.)
template <int TPR, bool VEC> struct RowEnd {
  int C, lane, last;
  __device__ __forceinline__ RowEnd(int C_, int lane_) : C(C_), lane(lane_), last((C_ >> 3) / TPR) {}
  __device__ __forceinline__ int col(int j, int i) const { return VEC ? (j * TPR + lane) * 8 + i : (j * 8 + i) * TPR + lane; }
  // f(j, i, true) for the elements of whole vectors, f(j, i, inside) for the others that may be inside
  template <int NV, typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!VEC || j == last) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f(j, i, VEC ? (j * TPR + lane) * 8 < C : col(j, i) < C);
      } else if (j < last) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f(j, i, true);
      }
    }
  }
};
template <typename T, int TPR, int NV, bool VEC> struct RowRegs {
  Raw8<T> r[NV];
  __device__ __forceinline__ void load(const T* row, const RowEnd<TPR, VEC>& end) {
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j] = vec_get<T, 0>(row, end.col(j, 0), end.C);
  }
  __device__ __forceinline__ void get(float v[NV][8]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) cvt8(r[j], v[j]);
  }
};
template <typename T, int TPR, int NV> struct RowRegs<T, TPR, NV, false> {
  T e[NV][8];
  __device__ __forceinline__ void load(const T* row, const RowEnd<TPR, false>& end) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) e[j][i] = row[end.col(j, i) < end.C ? end.col(j, i) : 0];
  }
  __device__ __forceinline__ void get(float v[NV][8]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = to_f<T>(e[j][i]);
  }
};
template <int TPR, int NV, bool VEC> __device__ __forceinline__ void ln_param(const float* p, float other, const RowEnd<TPR, VEC>& end, float v[NV][8]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = other;
  if (p == nullptr) return;
  RowRegs<float, TPR, NV, VEC> r;
  r.load(p, end);
  r.get(v);
}
template <typename T, int TPR, int NV, bool VEC> __device__ __forceinline__ void ln_store(T* row, const RowEnd<TPR, VEC>& end, const float v[NV][8]) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j <= end.last) vec_put<T, 0>(row, end.col(j, 0), end.C, v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (end.col(j, i) < end.C) row[end.col(j, i)] = from_f<T>(v[j][i]);
  }
}

// sums over the TPR threads of a row's group, in every thread of it.  TPR 256: `red` holds 4 floats for each value; the caller alternates
// between buffers so that one barrier a reduction is enough.
__device__ __forceinline__ float ln_wave_sum(float v) { return xor32_sum(xor16_sum(row16_sum(v))); }
template <int TPR, int NVAL> __device__ __forceinline__ void group_sum(float v[NVAL], float* red) {
#pragma unroll
  for (int k = 0; k < NVAL; ++k) v[k] = TPR == 16 ? row16_sum(v[k]) : ln_wave_sum(v[k]);
  if (TPR == 256) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < NVAL; ++k) red[k * 4 + w] = v[k];
    }
    lds_barrier();
#pragma unroll
    for (int k = 0; k < NVAL; ++k) v[k] = (red[k * 4] + red[k * 4 + 1]) + (red[k * 4 + 2] + red[k * 4 + 3]);
  }
}

template <typename T, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const spb_layernorm_args_t a) {
  constexpr int GR = 256 / TPR;                  // rows a workgroup works on at a time
  __shared__ float red[4][4];
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const int C = a.C;
  const RowEnd<TPR, VEC> end(C, lane);
  const float inv = 1.f / (float)C;
  const T* X = reinterpret_cast<const T*>(a.X);
  T* Y = reinterpret_cast<T*>(a.Y);
  const long long step = (long long)gridDim.x * GR;
  long long m = (long long)blockIdx.x * GR + grp;
  RowRegs<T, TPR, NV, VEC> cur, nxt;
  cur.load(X + (m < a.M ? m : a.M - 1) * a.ldx, end);
  float gm[NV][8], bt[NV][8];
  ln_param<TPR, NV, VEC>(a.gamma, 1.f, end, gm);
  ln_param<TPR, NV, VEC>(a.beta, 0.f, end, bt);
  // a group's row is past the end for whole groups: the sums of a group read its own lanes only, and with TPR 256 (barriers) the group is the workgroup
  int flip = 0;
  for (; m < a.M; m += step, flip ^= 2) {
    const long long mn = m + step;
    nxt.load(X + (mn < a.M ? mn : m) * a.ldx, end);
    float v[NV][8];
    cur.get(v);
    float s[1] = {0.f};
    end.template each<NV>([&](int j, int i, bool in) { s[0] += in ? v[j][i] : 0.f; });
    group_sum<TPR, 1>(s, red[flip]);
    const float mean = s[0] * inv;
    float q[1] = {0.f};
    end.template each<NV>([&](int j, int i, bool in) {
      v[j][i] = in ? v[j][i] - mean : 0.f;
      q[0] += v[j][i] * v[j][i];
    });
    group_sum<TPR, 1>(q, red[flip + 1]);
    const float rstd = 1.f / sqrtf(q[0] * inv + a.eps);
    end.template each<NV>([&](int j, int i, bool) { v[j][i] = v[j][i] * rstd * gm[j][i] + bt[j][i]; });
    ln_store<T, TPR, NV, VEC>(Y + m * a.ldy, end, v);
    if (lane == 0) { a.mean[m] = mean; a.rstd[m] = rstd; }
    cur = nxt;
  }
}

// rows longer than LN_REG_MAX: a workgroup a row, the row read once for each sum and once for the output (from L2 after the first time)
__device__ __forceinline__ float wg_sum(float v, float* red) {
  v = ln_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_long(const spb_layernorm_args_t a) {
  __shared__ float red[4];
  const float inv = 1.f / (float)a.C;
  for (long long m = blockIdx.x; m < a.M; m += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.X) + m * a.ldx;
    T* y = reinterpret_cast<T*>(a.Y) + m * a.ldy;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256) s += to_f<T>(x[c]);
    const float mean = wg_sum(s, red) * inv;
    float q = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256) { const float d = to_f<T>(x[c]) - mean; q += d * d; }
    const float rstd = 1.f / sqrtf(wg_sum(q, red) * inv + a.eps);
    for (int c = threadIdx.x; c < a.C; c += 256)
      y[c] = from_f<T>((to_f<T>(x[c]) - mean) * rstd * (a.gamma ? a.gamma[c] : 1.f) + (a.beta ? a.beta[c] : 0.f));
    if (threadIdx.x == 0) { a.mean[m] = mean; a.rstd[m] = rstd; }
  }
}

template <typename T, int TPR, int NV, bool VEC, bool SUMS>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const spb_layernorm_args_t a) {
  constexpr int GR = 256 / TPR;
  __shared__ float red[2][8];
  __shared__ float join[SUMS && GR > 1 ? GR * TPR * NV * 8 : 1];
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const int C = a.C;
  const RowEnd<TPR, VEC> end(C, lane);
  const float inv = 1.f / (float)C;
  const T* X = reinterpret_cast<const T*>(a.X);
  const T* G = reinterpret_cast<const T*>(a.G);
  T* D = reinterpret_cast<T*>(a.Y);
  const long long step = (long long)gridDim.x * GR;
  long long m = (long long)blockIdx.x * GR + grp;
  RowRegs<T, TPR, NV, VEC> cx, cg, nx, ng;
  float cm, cr, nm, nr;
  {
    const long long mc = m < a.M ? m : a.M - 1;
    cx.load(X + mc * a.ldx, end); cg.load(G + mc * a.ldg, end);
    cm = a.mean[mc]; cr = a.rstd[mc];
  }
  float gm[NV][8], dg[NV][8], db[NV][8];
  ln_param<TPR, NV, VEC>(a.gamma, 1.f, end, gm);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) { dg[j][i] = 0.f; db[j][i] = 0.f; }
  int flip = 0;
  for (; m < a.M; m += step, flip ^= 1) {      // whole groups leave: see the forward kernel
    const long long mn = m + step, mc = mn < a.M ? mn : m;
    nx.load(X + mc * a.ldx, end); ng.load(G + mc * a.ldg, end);
    nm = a.mean[mc]; nr = a.rstd[mc];
    float x[NV][8], g[NV][8];
    cx.get(x); cg.get(g);
    float s[2] = {0.f, 0.f};
    end.template each<NV>([&](int j, int i, bool in) {
      x[j][i] = in ? (x[j][i] - cm) * cr : 0.f;             // xh
      g[j][i] = in ? g[j][i] : 0.f;
      if (SUMS) { dg[j][i] += g[j][i] * x[j][i]; db[j][i] += g[j][i]; }
      g[j][i] *= gm[j][i];                                   // h
      s[0] += g[j][i]; s[1] += g[j][i] * x[j][i];
    });
    group_sum<TPR, 2>(s, red[flip]);
    const float s1 = s[0] * inv, s2 = s[1] * inv;
    end.template each<NV>([&](int j, int i, bool) { g[j][i] = cr * (g[j][i] - s1 - x[j][i] * s2); });
    ln_store<T, TPR, NV, VEC>(D + m * a.ldy, end, g);
    cx = nx; cg = ng; cm = nm; cr = nr;
  }
  if (SUMS) {
    float* out = a.part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (GR > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) join[grp * (TPR * NV * 8) + end.col(j, i)] = half ? db[j][i] : dg[j][i];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256) {
          double v = 0.;
#pragma unroll
          for (int k = 0; k < GR; ++k) v += join[k * (TPR * NV * 8) + c];
          out[half * C + c] = (float)v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = end.col(j, i);
            if (c < C) out[half * C + c] = half ? db[j][i] : dg[j][i];
          }
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_long(const spb_layernorm_args_t a) {
  __shared__ float red[4];
  const float inv = 1.f / (float)a.C;
  for (long long m = blockIdx.x; m < a.M; m += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.X) + m * a.ldx;
    const T* g = reinterpret_cast<const T*>(a.G) + m * a.ldg;
    T* d = reinterpret_cast<T*>(a.Y) + m * a.ldy;
    const float mean = a.mean[m], rstd = a.rstd[m];
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float h = to_f<T>(g[c]) * (a.gamma ? a.gamma[c] : 1.f);
      s += h; q += h * (to_f<T>(x[c]) - mean) * rstd;
    }
    s = wg_sum(s, red) * inv;
    q = wg_sum(q, red) * inv;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float h = to_f<T>(g[c]) * (a.gamma ? a.gamma[c] : 1.f);
      d[c] = from_f<T>(rstd * (h - s - (to_f<T>(x[c]) - mean) * rstd * q));
    }
  }
}
// partial rows of dgamma / dbeta for long rows: a thread a column, blockIdx.y a range of rows.  It runs BEFORE ln_bwd_long, whose output may
// overwrite g.  Rows are added in blocks of 64, whose sums are added up in 64 bits: a single chain would collect a rounding for each of the range's rows.
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols(const spb_layernorm_args_t a, long long rows) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  const long long m0 = (long long)blockIdx.y * rows, m1 = m0 + rows < a.M ? m0 + rows : a.M;
  if (c >= a.C) return;
  double dg = 0., db = 0.;
  for (long long b = m0; b < m1; b += 64) {
    float pg = 0.f, pb = 0.f;
    for (long long m = b, e = b + 64 < m1 ? b + 64 : m1; m < e; ++m) {
      const float g = to_f<T>(reinterpret_cast<const T*>(a.G)[m * a.ldg + c]);
      pg += g * (to_f<T>(reinterpret_cast<const T*>(a.X)[m * a.ldx + c]) - a.mean[m]) * a.rstd[m];
      pb += g;
    }
    dg += pg; db += pb;
  }
  float* out = a.part + (size_t)blockIdx.y * 2 * a.C;
  out[c] = (float)dg; out[a.C + c] = (float)db;
}

// dgamma / dbeta (+)= the P partial rows, in order and in 64 bits (0.6 us of 12 on 2351 x 1001, whose dgamma errs by 6.1e-8 of its norm instead of 1.3e-7): 64 columns a workgroup, its sixteen waves a
// sixteenth of the rows each, eight requested at a time (a loop of dependent additions waits for memory at every row: 128 rows took 35 us, this form takes 4)
constexpr int LN_JOIN = 16;
__global__ __launch_bounds__(LN_JOIN * 64) void ln_join_kernel(const float* part, int P, int C, float* dgamma, float* dbeta, int accumulate) {
  __shared__ double red[LN_JOIN][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long long n = 2ll * C, c = (long long)blockIdx.x * 64 + l, cc = c < n ? c : n - 1;
  const int per = (P + LN_JOIN - 1) / LN_JOIN, p0 = w * per, p1 = p0 + per < P ? p0 + per : P;
  double v = 0.;
  for (int p = p0; p < p1; p += 8) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = part[(p + i < p1 ? p + i : p1 - 1) * n + cc];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p + i < p1 ? x[i] : 0.f;
    v += (((double)x[0] + x[1]) + ((double)x[2] + x[3])) + (((double)x[4] + x[5]) + ((double)x[6] + x[7]));
  }
  red[w][l] = v;
  __syncthreads();
  if (w == 0 && c < n) {
    v = 0.;
#pragma unroll
    for (int k = 0; k < LN_JOIN; k += 4) v += (red[k][l] + red[k + 1][l]) + (red[k + 2][l] + red[k + 3][l]);
    float* dst = c < C ? dgamma : dbeta;
    const int o = (int)(c < C ? c : c - C);
    if (dst) dst[o] = (accumulate ? dst[o] : 0.f) + (float)v;
  }
}

struct LnShape { int tpr, nv; };
// the narrowest group that holds a row in 16 (16 threads), 24 (64) or 32 (256) elements a thread
inline LnShape ln_shape(int C) {
  if (C <= 128) return {16, 1};
  if (C <= 256) return {16, 2};
  if (C <= 512) return {64, 1};
  if (C <= 1024) return {64, 2};
  if (C <= 1536) return {64, 3};
  if (C <= 2048) return {256, 1};
  if (C <= 4096) return {256, 2};
  return {256, 4};
}
inline int ln_bwd_parts(long long M, int C) {
  if (C > LN_REG_MAX) return (int)(M < 64 ? (M > 0 ? M : 1) : 64);
  const long long wgs = (M + 256 / ln_shape(C).tpr - 1) / (256 / ln_shape(C).tpr), rounds = wgs > 0 ? (wgs + LN_BWD_WGS - 1) / LN_BWD_WGS : 1;
  return (int)(wgs > 0 ? (wgs + rounds - 1) / rounds : 1);         // every workgroup as many rounds: fewer partial rows in the same time
}
template <typename T, bool VEC> void launch_fwd(const spb_layernorm_args_t& a, hipStream_t s) {
  const LnShape sh = ln_shape(a.C);
  const long long gr = 256 / sh.tpr, need = (a.M + gr - 1) / gr;
  const dim3 grid((unsigned)(need < LN_FWD_WGS ? need : LN_FWD_WGS)), block(256);
#define LN_F(TPR, NV) hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV, VEC>), grid, block, 0, s, a)
  if (sh.tpr == 16) { if (sh.nv == 1) LN_F(16, 1); else LN_F(16, 2); }
  else if (sh.tpr == 64) { if (sh.nv == 1) LN_F(64, 1); else if (sh.nv == 2) LN_F(64, 2); else LN_F(64, 3); }
  else { if (sh.nv == 1) LN_F(256, 1); else if (sh.nv == 2) LN_F(256, 2); else LN_F(256, 4); }
#undef LN_F
}
template <typename T, bool VEC, bool SUMS> void launch_bwd(const spb_layernorm_args_t& a, hipStream_t s) {
  const LnShape sh = ln_shape(a.C);
  const dim3 grid((unsigned)ln_bwd_parts(a.M, a.C)), block(256);
#define LN_B(TPR, NV) hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV, VEC, SUMS>), grid, block, 0, s, a)
  if (sh.tpr == 16) { if (sh.nv == 1) LN_B(16, 1); else LN_B(16, 2); }
  else if (sh.tpr == 64) { if (sh.nv == 1) LN_B(64, 1); else if (sh.nv == 2) LN_B(64, 2); else LN_B(64, 3); }
  else { if (sh.nv == 1) LN_B(256, 1); else if (sh.nv == 2) LN_B(256, 2); else LN_B(256, 4); }
#undef LN_B
}
template <typename T> void run_fwd(const spb_layernorm_args_t& a, hipStream_t s) {
  if (a.C > LN_REG_MAX) {
    hipLaunchKernelGGL((ln_fwd_long<T>), dim3((unsigned)(a.M < LN_FWD_WGS ? a.M : LN_FWD_WGS)), dim3(256), 0, s, a);
    return;
  }
  if (a.C % 8 == 0) launch_fwd<T, true>(a, s); else launch_fwd<T, false>(a, s);
}
// returns the number of partial rows
template <typename T> int run_bwd(const spb_layernorm_args_t& a, bool sums, hipStream_t s) {
  int P = ln_bwd_parts(a.M, a.C);
  if (a.C > LN_REG_MAX) {
    const long long rows = (a.M + P - 1) / P;
    P = (int)((a.M + rows - 1) / rows);             // ranges that hold a row
    if (sums) hipLaunchKernelGGL((ln_bwd_cols<T>), dim3((unsigned)((a.C + 255) / 256), (unsigned)P), dim3(256), 0, s, a, rows);
    hipLaunchKernelGGL((ln_bwd_long<T>), dim3((unsigned)(a.M < LN_FWD_WGS ? a.M : LN_FWD_WGS)), dim3(256), 0, s, a);
    return P;
  }
  if (sums) { if (a.C % 8 == 0) launch_bwd<T, true, true>(a, s); else launch_bwd<T, false, true>(a, s); }
  else { if (a.C % 8 == 0) launch_bwd<T, true, false>(a, s); else launch_bwd<T, false, false>(a, s); }
  return P;
}

int check_args(int dtype, const spb_layernorm_args_t* a, bool bwd) {
  if (dtype != SPB_F32 && dtype != SPB_BF16) return SPB_E_ARG;
  if (!a || a->C < 1 || a->C > LN_COLS_MAX || a->M < 0) return a ? SPB_E_SHAPE : SPB_E_ARG;
  if (bwd && (a->dgamma || a->dbeta) && a->C > LN_SUMS_MAX) return SPB_E_SHAPE;
  if (a->M == 0) return 0;
  if (!a->X || !a->Y || !a->mean || !a->rstd || (bwd && !a->G)) return SPB_E_ARG;
  if (a->ldx < 0 || a->ldy < (a->M > 1 ? a->C : 0) || (bwd && a->ldg < 0)) return SPB_E_SHAPE;
  if (bwd && a->dgamma && a->dgamma == a->dbeta) return SPB_E_ARG;      // two sums into one buffer
  return 0;
}

}  // namespace

extern "C" int spb_layernorm_fwd(int dtype, const spb_layernorm_args_t* a, spb_stream_t stream) {
  const int bad = check_args(dtype, a, false);
  if (bad) return bad;
  if (a->M == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SPB_F32) run_fwd<float>(*a, s); else run_fwd<bf16_t>(*a, s);
  SPB_CHECK_LAUNCH();
  return 0;
}

extern "C" long long spb_layernorm_bwd_floats(long long M, int C) {
  if (M < 0 || C < 1 || C > LN_SUMS_MAX) return SPB_E_SHAPE;
  return 2ll * C * ln_bwd_parts(M, C);
}

extern "C" int spb_layernorm_bwd(int dtype, const spb_layernorm_args_t* a, spb_stream_t stream) {
  const int bad = check_args(dtype, a, true);
  if (bad) return bad;
  const bool sums = a->dgamma || a->dbeta;
  if (a->M == 0 && (!sums || a->accumulate)) return 0;
  if (sums && a->M > 0 && (!a->part || a->part_cap < spb_layernorm_bwd_floats(a->M, a->C))) return SPB_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  int P = 0;                                        // no rows: the join writes zeros
  if (a->M > 0) P = dtype == SPB_F32 ? run_bwd<float>(*a, sums, s) : run_bwd<bf16_t>(*a, sums, s);
  SPB_CHECK_LAUNCH();
  if (sums) {
    hipLaunchKernelGGL(ln_join_kernel, dim3((unsigned)((2ll * a->C + 63) / 64)), dim3(LN_JOIN * 64), 0, s, a->part, P, a->C, a->dgamma, a->dbeta, a->accumulate);
    SPB_CHECK_LAUNCH();
  }
  return 0;
}
