// Vectors of 8 row elements at any alignment: what the kernels on rows of any length and stride share.
//   The hardware loads and stores 16 bytes a lane at any element alignment, so an odd row stride costs no element-wise loop.  A row's length enters
//   through MODE:  0: a multiple of 8;  1: any length >= 8, the last vector is loaded from 8 elements before the row's end and shifted into place
//   (nothing behind the row is touched);  2: shorter than 8, element by element.
#pragma once
#include "common.h"

static inline int vec_mode(int C) { return C < 8 ? 2 : (C % 8 ? 1 : 0); }

template <typename T> __device__ __forceinline__ Raw8<T> vec_ld(const T* p) {
  Raw8<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
// elements s .. 7 move to 0 .. 7 - s (what follows is arbitrary)
__device__ __forceinline__ void vec_shift(Raw8<bf16_t>& r, int s) {
  unsigned long long lo = (unsigned long long)r.u.y << 32 | r.u.x, hi = (unsigned long long)r.u.w << 32 | r.u.z;
  if (s & 4) lo = hi;
  const int b = (s & 3) * 16;
  lo = b ? (lo >> b) | (hi << (64 - b)) : lo;
  hi >>= b;
  r.u = make_uint4((unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32));
}
__device__ __forceinline__ void vec_shift(Raw8<float>& r, int s) {
  // bit masks: of `s & k ? v[i + k] : v[i]` the compiler makes eight comparisons for each element
  unsigned v[8] = {__float_as_uint(r.a.x), __float_as_uint(r.a.y), __float_as_uint(r.a.z), __float_as_uint(r.a.w),
                   __float_as_uint(r.b.x), __float_as_uint(r.b.y), __float_as_uint(r.b.z), __float_as_uint(r.b.w)};
#pragma unroll
  for (int k = 1; k < 8; k <<= 1) {
    const unsigned m = s & k ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i + k < 8; ++i) v[i] = (v[i + k] & m) | (v[i] & ~m);
  }
  r.a = make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
  r.b = make_float4(__uint_as_float(v[4]), __uint_as_float(v[5]), __uint_as_float(v[6]), __uint_as_float(v[7]));
}
// where the vector of column c is loaded from (c >= C: anywhere in the row; its elements are not used)
template <int MODE> __device__ __forceinline__ int vec_from(int c, int C) { return MODE == 0 ? (c < C ? c : 0) : (c + 8 <= C ? c : C - 8); }
// the vector of column c, requested (MODE 0, 1)
template <typename T, int MODE> __device__ __forceinline__ Raw8<T> vec_get(const T* row, int c, int C) { return vec_ld<T>(row + vec_from<MODE>(c, C)); }
// ... and put into place
template <typename T, int MODE> __device__ __forceinline__ void vec_place(Raw8<T>& r, int c, int C) {
  if (MODE == 1) vec_shift(r, c + 8 <= C ? 0 : (c - (C - 8)) & 7);
}
template <typename T, int MODE> __device__ __forceinline__ void vec_put(T* row, int c, int C, const float v[8]) {
  if (MODE == 2 || (MODE == 1 && c + 8 > C)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) row[c + i] = from_f<T>(v[i]);
  } else if (c < C) {
    T t[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = v[i];
      __builtin_memcpy(row + c, t, 32);
    } else {
      const uint4 u = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      __builtin_memcpy(row + c, &u, 16);
    }
  }
}
