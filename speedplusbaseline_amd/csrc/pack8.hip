// Packing to 8 bits with one power-of-two scale for each block of 128 (format: include/spb_hip.h "8-bit packing"), and the activations that keep
// their input in that form for the backward pass.
//
//   block top a = max |x| over its finite elements,  e = smallest integer with a <= 448 * 2^e,  code = e4m3(x * 2^-e)
//   act8 forward  y = act(x), checkpoint = pack(x);    backward  dx = g * act'(value(checkpoint))
//
// The scale is a power of two so that packing has ONE rounding (the code's own), its result does not depend on how a quotient is rounded, values
// stay exact in bfloat16, and the matrix instructions apply it themselves.  It costs at most one bit of exponent range, which e4m3 has to spare.
// All of it is bound by HBM: every element is read once and written once.  16 lanes share a block of 128 (8 consecutive elements each: 16-byte
// loads of 16-bit types, 8-byte stores of codes), its top is four vector-ALU exchanges, and neighbouring groups hold neighbouring blocks.
#include "pack8.h"

namespace {

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, spb_dpp_f<0xB1>(v)); v = fmaxf(v, spb_dpp_f<0x4E>(v)); v = fmaxf(v, spb_dpp_f<0x141>(v)); v = fmaxf(v, spb_dpp_f<0x140>(v));
  return v;
}
// 8 elements from column c on (MODE: vec8.h): requested, then put into place with zeros behind K
template <typename T, int MODE> __device__ __forceinline__ Raw8<T> get8(const T* row, int c, int K) {
  if constexpr (MODE == 2) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = row[c + i < K ? c + i : 0];
    return vec_ld<T>(t);
  } else {
    return vec_get<T, MODE>(row, c, K);
  }
}
template <typename T, int MODE> __device__ __forceinline__ void place8(Raw8<T> r, int c, int K, float v[8]) {
  vec_place<T, MODE>(r, c, K);
  cvt8(r, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + (MODE == 0 ? 0 : i) < K ? v[i] : 0.f;
}
template <typename T, int MODE> __device__ __forceinline__ void load8(const T* row, int c, int K, float v[8]) {
  place8<T, MODE>(get8<T, MODE>(row, c, K), c, K, v);
}
// The f32 value is what is rounded, in both forms: without the empty asm the compiler may fold a product into its conversion to half (one rounding
// instead of two) in one of them, and a result would depend on its row's length.
template <typename T, int MODE> __device__ __forceinline__ void store8(T* row, int c, int K, float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("" : "+v"(v[i]));
  vec_put<T, MODE>(row, c, K, v);
}

// act(x) and act'(x) in f32 (ACT 0: none, plain packing), from one exponential and one reciprocal each: with the library's erff, tanhf, expf and the exact
// division both passes were bound by vector instructions (16384 x 4096 bfloat16: 88 / 102 us).
//   sigmoid    s = 1 / (1 + e^-x);   silu = x s,  silu' = s (1 + x (1 - s))
//   gelu tanh  (1 + tanh u) / 2 = sigmoid(2 u),  u = sqrt(2 / pi) (x + 0.044715 x^3)
//   gelu       Phi(x) = 1 - Q or Q, Q = erfc(|x| / sqrt 2) / 2 = t (a1 + t (a2 + ...)) e^(-x^2 / 2) / 2, t = 1 / (1 + p |x| / sqrt 2): Abramowitz and Stegun
//              7.1.26, |error of erf| <= 1.5e-7; the density's exponential is the same one
__device__ __forceinline__ float p8_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float p8_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + p8_exp(-x)); }
__device__ __forceinline__ float p8_phi(float x, float& e) {      // Phi(x); e = e^(-x^2 / 2)
  const float a = fabsf(x);
  e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);
  const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.23164189f, 1.f));
  const float q = fmaf(fmaf(fmaf(fmaf(0.5307027145f, t, -0.7265760135f), t, 0.7107068705f), t, -0.142248368f), t, 0.127414796f) * t * e;
  return x < 0.f ? q : 1.f - q;
}
template <int ACT> __device__ __forceinline__ float act8(float x) {
  float e;
  if (ACT == SPB_ACT_SILU) return x * p8_sigmoid(x);
  if (ACT == SPB_ACT_GELU) return x * p8_phi(x, e);
  return x * p8_sigmoid(1.59576912f * fmaf(0.044715f * x, x * x, x));
}
template <int ACT> __device__ __forceinline__ float act8_slope(float x) {
  if (ACT == SPB_ACT_SILU) { const float s = p8_sigmoid(x); return s * fmaf(x, 1.f - s, 1.f); }
  if (ACT == SPB_ACT_GELU) { float e; const float p = p8_phi(x, e); return fmaf(x * 0.39894228f, e, p); }
  x = x > 16.f ? 16.f : (x < -16.f ? -16.f : x);       // s (1 - s) is 0 from there on; x * x would overflow in 0 * inf.  NaN stays NaN.
  const float s = p8_sigmoid(1.59576912f * fmaf(0.044715f * x, x * x, x));
  return s * fmaf(x * (1.f - s), 1.59576912f * fmaf(0.134145f * x, x, 1.f), 1.f);
}

struct RowArgs {
  const void* X; void* Y; unsigned char* Q; unsigned char* S;
  long long ldx, ldy;
  unsigned blocks;      // M * KB
  int K, KB, Kp, Sp;
};
template <typename T, int MODE, int ACT>
__global__ __launch_bounds__(256) void pack8_rows_kernel(const RowArgs a) {
  const unsigned u = blockIdx.x * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  if (u >= a.blocks) return;                           // whole groups of 16 lanes: the exchanges below stay inside a group
  const unsigned m = u / (unsigned)a.KB;
  const int kb = (int)(u - m * (unsigned)a.KB), c = kb * P8_BLOCK + l * 8;
  float v[8];
  load8<T, MODE>(reinterpret_cast<const T*>(a.X) + (long long)m * a.ldx, c, a.K, v);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, p8_finite_abs(v[i]));
  const int e = p8_exponent(row16_max(top));
  *reinterpret_cast<uint2*>(a.Q + (size_t)m * a.Kp + c) = p8_encode8(v, e);
  unsigned char* s = a.S + (size_t)m * a.Sp;
  if (l == 0) s[kb] = (unsigned char)(e + 127);
  else if (kb == a.KB - 1 && a.KB - 1 + l < a.Sp) s[a.KB - 1 + l] = 127;
  if (ACT != 0) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = act8<ACT>(v[i]);
    store8<T, MODE>(reinterpret_cast<T*>(a.Y) + (long long)m * a.ldy, c, a.K, y);
  }
}

// values of a packed matrix (ACT 0) or g * act'(value): a thread 8 elements
struct UnpackArgs {
  const void* G; void* Y; const unsigned char* Q; const unsigned char* S;
  long long ldg, ldy;
  unsigned vecs;        // M * V
  int K, V, Kp, Sp, shift;
};
template <typename T, int MODE, int ACT>
__global__ __launch_bounds__(256) void unpack8_kernel(const UnpackArgs a) {
  const unsigned u = blockIdx.x * 256 + threadIdx.x;
  if (u >= a.vecs) return;
  const unsigned m = u / (unsigned)a.V;
  const int c = (int)(u - m * (unsigned)a.V) * 8;
  const uint2 q = *reinterpret_cast<const uint2*>(a.Q + (size_t)m * a.Kp + c);
  const float s = p8_pow2((int)a.S[(size_t)(m >> a.shift) * a.Sp + (c >> 7)] - 127);
  float v[8];
  p8_decode8(q, s, v);
  if (ACT != 0) {
    float g[8];
    load8<T, MODE>(reinterpret_cast<const T*>(a.G) + (long long)m * a.ldg, c, a.K, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = g[i] * act8_slope<ACT>(v[i]);
  }
  store8<T, MODE>(reinterpret_cast<T*>(a.Y) + (long long)m * a.ldy, c, a.K, v);
}

// a 128 x 128 block a workgroup: 16 lanes hold 128 columns, a thread 8 columns of 8 neighbouring rows, whose codes it transposes in registers: the 8 codes of a
// column go to LDS as 8 bytes (rows of 136 bytes: neighbouring columns are two banks apart) and come back as 16.
// byte j of a[i] becomes byte i of t[j]
__device__ __forceinline__ void p8_transpose4(const unsigned a[4], unsigned t[4]) {
  const unsigned x0 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), x1 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);
  const unsigned y0 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), y1 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
  t[0] = __builtin_amdgcn_perm(y0, x0, 0x05040100u); t[1] = __builtin_amdgcn_perm(y0, x0, 0x07060302u);
  t[2] = __builtin_amdgcn_perm(y1, x1, 0x05040100u); t[3] = __builtin_amdgcn_perm(y1, x1, 0x07060302u);
}
struct WeightArgs {
  const void* W; unsigned char* Q; unsigned char* S; unsigned char* QT; unsigned char* ST;
  long long ldw;
  int N, K, NB, KB, Kp, Sp, Np, SpT;
};
template <typename T, int MODE>
__global__ __launch_bounds__(256) void pack8_weight_kernel(const WeightArgs a) {
  constexpr int LD = 136;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) unsigned char tile[128 * LD];     // [column][row]
  const int nb = blockIdx.x / a.KB, kb = blockIdx.x - nb * a.KB;
  const int l = threadIdx.x & 15, r0 = (threadIdx.x >> 4) * 8, c = kb * P8_BLOCK + l * 8;
  float v[8][8];
  Raw8<T> raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = nb * P8_BLOCK + r0 + i;
    raw[i] = get8<T, MODE>(reinterpret_cast<const T*>(a.W) + (long long)(n < a.N ? n : 0) * a.ldw, c, a.K);
  }
  __builtin_amdgcn_sched_barrier(0);                   // all requests before the first is used (4096 x 4096 f32: 17.4 -> 16.9 us)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = nb * P8_BLOCK + r0 + i;
    place8<T, MODE>(raw[i], c, a.K, v[i]);
    if (n >= a.N) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, p8_finite_abs(v[i][j]));
  top = row16_max(top);
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  const int e = p8_exponent(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  uint2 q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = nb * P8_BLOCK + r0 + i;
    q[i] = p8_encode8(v[i], e);
    if (n < a.N) *reinterpret_cast<uint2*>(a.Q + (size_t)n * a.Kp + c) = q[i];
  }
  if (a.QT) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {                        // columns 4 h .. 4 h + 3: two 4 x 4 byte transposes
      unsigned lo[4], hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { lo[i] = h ? q[i].y : q[i].x; hi[i] = h ? q[i + 4].y : q[i + 4].x; }
      unsigned tl[4], th[4];
      p8_transpose4(lo, tl);
      p8_transpose4(hi, th);
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint2*>(tile + (l * 8 + h * 4 + j) * LD + r0) = make_uint2(tl[j], th[j]);
    }
  }
  if (threadIdx.x == 0) a.S[(size_t)nb * a.Sp + kb] = (unsigned char)(e + 127);
  else if (kb == a.KB - 1 && kb + (int)threadIdx.x < a.Sp) a.S[(size_t)nb * a.Sp + kb + threadIdx.x] = 127;
  if (a.QT) {
    if (threadIdx.x == 0) a.ST[(size_t)kb * a.SpT + nb] = (unsigned char)(e + 127);
    else if (nb == a.NB - 1 && nb + (int)threadIdx.x < a.SpT) a.ST[(size_t)kb * a.SpT + nb + threadIdx.x] = 127;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int idx = threadIdx.x + 256 * i, col = idx >> 3, part = idx & 7, k = kb * P8_BLOCK + col;
      if (k < a.K)
      {
        const uint2 u0 = *reinterpret_cast<const uint2*>(tile + col * LD + part * 16), u1 = *reinterpret_cast<const uint2*>(tile + col * LD + part * 16 + 8);
        *reinterpret_cast<uint4*>(a.QT + (size_t)k * a.Np + nb * P8_BLOCK + part * 16) = make_uint4(u0.x, u0.y, u1.x, u1.y);
      }
    }
  }
}

inline bool bad_codes(const void* q, const void* s) { return !q || !s || ((uintptr_t)q & 15) || ((uintptr_t)s & 3); }
inline bool bad_dtype(int d) { return d != SPB_F32 && d != SPB_BF16; }

// one instance for each type and row length (MODE)
#define P8_LAUNCH(kernel, grid, ...)                                                                                                        \
  do {                                                                                                                                      \
    const int mode_ = vec_mode(a.K);                                                                                                        \
    if (dtype == SPB_F32) {                                                                                                                 \
      if (mode_ == 0) hipLaunchKernelGGL((kernel<float, 0, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                      \
      else if (mode_ == 1) hipLaunchKernelGGL((kernel<float, 1, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                 \
      else hipLaunchKernelGGL((kernel<float, 2, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                                 \
    } else {                                                                                                                                \
      if (mode_ == 0) hipLaunchKernelGGL((kernel<bf16_t, 0, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                     \
      else if (mode_ == 1) hipLaunchKernelGGL((kernel<bf16_t, 1, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                \
      else hipLaunchKernelGGL((kernel<bf16_t, 2, ##__VA_ARGS__>), grid, dim3(256), 0, s, a);                                                \
    }                                                                                                                                       \
    SPB_CHECK_LAUNCH();                                                                                                                     \
  } while (0)

// as many rows a launch as it has threads for (16 a block; 8 elements each)
template <int ACT> int pack_rows(int dtype, const RowArgs& all, long long M, hipStream_t s) {
  if (M * all.KB > 0xfffffff0ll) return SPB_E_SHAPE;
  const long long most = (P8_THREADS / 256 * 16) / all.KB, es = dtype == SPB_F32 ? 4 : 2;
  for (long long m = 0; m < M; m += most) {
    RowArgs a = all;
    a.blocks = (unsigned)((M - m < most ? M - m : most) * a.KB);
    a.X = (const char*)a.X + m * a.ldx * es; a.Q += m * a.Kp; a.S += m * a.Sp;
    if (ACT != 0) a.Y = (char*)a.Y + m * a.ldy * es;
    P8_LAUNCH(pack8_rows_kernel, dim3(a.blocks / 16 + (a.blocks % 16 ? 1 : 0)), ACT);
  }
  return 0;
}
template <int ACT> int unpack(int dtype, const UnpackArgs& all, long long M, hipStream_t s) {
  if (M * all.V > 0xfffffff0ll) return SPB_E_SHAPE;
  long long most = (P8_THREADS / 256 * 256) / all.V;
  const long long es = dtype == SPB_F32 ? 4 : 2;
  if (most < M && all.shift) most = most >> 7 << 7;       // whole blocks of rows
  if (most == 0) return SPB_E_SHAPE;
  for (long long m = 0; m < M; m += most) {
    UnpackArgs a = all;
    a.vecs = (unsigned)((M - m < most ? M - m : most) * a.V);
    a.Q += m * a.Kp; a.S += (m >> a.shift) * a.Sp; a.Y = (char*)a.Y + m * a.ldy * es;
    if (ACT != 0) a.G = (const char*)a.G + m * a.ldg * es;
    P8_LAUNCH(unpack8_kernel, dim3(a.vecs / 256 + (a.vecs % 256 ? 1 : 0)), ACT);
  }
  return 0;
}

}  // namespace

extern "C" int spb_pack8_rows(int dtype, const void* X, long long ldx, long long M, int K, unsigned char* codes, unsigned char* scales, spb_stream_t stream) {
  if (bad_dtype(dtype)) return SPB_E_ARG;
  if (M < 0 || K < 0 || ldx < 0) return SPB_E_SHAPE;
  if (M == 0 || K == 0) return 0;
  if (!X || bad_codes(codes, scales)) return SPB_E_ARG;
  return pack_rows<0>(dtype, {X, nullptr, codes, scales, ldx, 0, 0, K, (K + 127) / 128, p8_cols(K), p8_scales(K)}, M, (hipStream_t)stream);
}

extern "C" int spb_pack8_weight(int dtype, const void* W, long long ldw, int N, int K, unsigned char* codes, unsigned char* scales, unsigned char* codesT,
                                unsigned char* scalesT, spb_stream_t stream) {
  if (bad_dtype(dtype)) return SPB_E_ARG;
  if (N < 0 || K < 0 || ldw < 0) return SPB_E_SHAPE;
  if (N == 0 || K == 0) return 0;
  if (!W || bad_codes(codes, scales) || (codesT != nullptr) != (scalesT != nullptr) || (codesT && bad_codes(codesT, scalesT))) return SPB_E_ARG;
  const WeightArgs a = {W, codes, scales, codesT, scalesT, ldw, N, K, (N + 127) / 128, (K + 127) / 128, p8_cols(K), p8_scales(K), p8_cols(N), p8_scales(N)};
  if (!p8_fits((long long)a.NB * a.KB, 256)) return SPB_E_SHAPE;
  hipStream_t s = (hipStream_t)stream;
  P8_LAUNCH(pack8_weight_kernel, dim3((unsigned)(a.NB * a.KB)));
  return 0;
}

extern "C" int spb_unpack8(int dtype, const unsigned char* codes, const unsigned char* scales, int block_rows, long long M, int K, void* Y, long long ldy,
                           spb_stream_t stream) {
  if (bad_dtype(dtype) || (block_rows != 1 && block_rows != 128)) return SPB_E_ARG;
  if (M < 0 || K < 0 || (M > 1 && ldy < K)) return SPB_E_SHAPE;
  if (M == 0 || K == 0) return 0;
  if (!Y || bad_codes(codes, scales)) return SPB_E_ARG;
  return unpack<0>(dtype, {nullptr, Y, codes, scales, 0, ldy, 0, K, (K + 7) / 8, p8_cols(K), p8_scales(K), block_rows == 128 ? 7 : 0}, M, (hipStream_t)stream);
}

extern "C" int spb_act8_fwd(int dtype, int act, const void* X, long long ldx, void* Y, long long ldy, long long M, int K, unsigned char* codes,
                            unsigned char* scales, spb_stream_t stream) {
  if (bad_dtype(dtype) || act < SPB_ACT_GELU || act > SPB_ACT_SILU) return SPB_E_ARG;
  if (M < 0 || K < 0 || ldx < 0 || (M > 1 && ldy < K)) return SPB_E_SHAPE;
  if (M == 0 || K == 0) return 0;
  if (!X || !Y || bad_codes(codes, scales)) return SPB_E_ARG;
  const RowArgs a = {X, Y, codes, scales, ldx, ldy, 0, K, (K + 127) / 128, p8_cols(K), p8_scales(K)};
  hipStream_t s = (hipStream_t)stream;
  if (act == SPB_ACT_GELU) return pack_rows<SPB_ACT_GELU>(dtype, a, M, s);
  if (act == SPB_ACT_GELU_TANH) return pack_rows<SPB_ACT_GELU_TANH>(dtype, a, M, s);
  return pack_rows<SPB_ACT_SILU>(dtype, a, M, s);
}

extern "C" int spb_act8_bwd(int dtype, int act, const void* G, long long ldg, const unsigned char* codes, const unsigned char* scales, void* dX,
                            long long ldd, long long M, int K, spb_stream_t stream) {
  if (bad_dtype(dtype) || act < SPB_ACT_GELU || act > SPB_ACT_SILU) return SPB_E_ARG;
  if (M < 0 || K < 0 || ldg < 0 || (M > 1 && ldd < K)) return SPB_E_SHAPE;
  if (M == 0 || K == 0) return 0;
  if (!G || !dX || bad_codes(codes, scales)) return SPB_E_ARG;
  const UnpackArgs a = {G, dX, codes, scales, ldg, ldd, 0, K, (K + 7) / 8, p8_cols(K), p8_scales(K), 0};
  hipStream_t s = (hipStream_t)stream;
  if (act == SPB_ACT_GELU) return unpack<SPB_ACT_GELU>(dtype, a, M, s);
  if (act == SPB_ACT_GELU_TANH) return unpack<SPB_ACT_GELU_TANH>(dtype, a, M, s);
  return unpack<SPB_ACT_SILU>(dtype, a, M, s);
}
