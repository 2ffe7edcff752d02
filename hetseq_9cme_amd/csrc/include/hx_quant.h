// 8-bit blocks: 128 consecutive entries share one power-of-two scale 2^e.
//
//   e4m3 : e = the smallest integer with max |x| <= 448 2^e,  code = e4m3(x 2^-e), nearest even
//   int8 : e = the smallest integer with max |x| <= 127 2^e,  code = rint(x 2^-e)
//
// over the block's finite entries (all zero: e = 0), e >= -126 so that 2^e and 2^-e are normal fp32
// numbers.  Scaling by a power of two is exact, so the only rounding is the code's own and any
// order of the same arithmetic gives the same bits; and 2^e is one byte (e + 127), the form the
// scaled matrix instructions take.  A general scale max / 448 would keep at most one bit more of
// range and cost that rounding.  Entries that are not finite: e4m3 NaN, int8 -128.
#pragma once
#include "hx_common.h"

namespace hx {
namespace q8 {

constexpr int kBlock = 128;

// (exponent of the largest code, mantissa bits of the largest code): 448 = 1.75 2^8, 127 = 1.984375 2^6
struct E4M3 {
  static constexpr int top_exp = 8;
  static constexpr uint32_t top_man = 0x600000u;
};
struct Int8 {
  static constexpr int top_exp = 6;
  static constexpr uint32_t top_man = 0x7E0000u;
};

// the block exponent from its largest finite magnitude
template <typename F>
__device__ __forceinline__ int block_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - F::top_exp + ((u & 0x7fffffu) > F::top_man ? 1 : 0);
  return u == 0 ? 0 : (e < -126 ? -126 : e);   // (a subnormal maximum clamps too)
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 .. 127
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;   // inf / NaN do not take part in the maximum
}

// 4 values -> their 4 e4m3 codes at scale s = 2^e in one word: v_cvt_scalef32_pk_fp8_* rounds x / s to
// nearest even, and what is not finite to NaN
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16v2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float s) {
  i16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, s, true));
}
__device__ __forceinline__ uint32_t e4m3x4(uint32_t ab, uint32_t cd, float s) {   // of packed bf16 pairs
  i16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16v2, ab), s, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16v2, cd), s, true));
}
// one scaled value -> its int8 code in the low byte
__device__ __forceinline__ uint32_t int8_of(float v) {
  const float r = rintf(v);
  return fabsf(r) <= 127.f ? (uint32_t)(int)r & 0xffu : 0x80u;
}
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
  return int8_of(a) | (int8_of(b) << 8) | (int8_of(c) << 16) | (int8_of(d) << 24);
}
// byte j of a word of int8 codes -> its value times s
__device__ __forceinline__ float int8_val(uint32_t w, int j, float s) {
  const int c = (int)(w << (24 - 8 * j)) >> 24;
  return c == -128 ? __uint_as_float(0x7fc00000u) : (float)c * s;
}

// 8 int8 codes -> their values times s: a code plus 128 is a byte (one conversion) and b s - 128 s is exact, so
// one fma each; codes of -128 and scales so large that 128 s is not finite take the careful way
__device__ __forceinline__ void int8_vals(uint2 w, float s, float (&v)[8]) {
  const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
  const uint32_t zero = (((a - 0x01010101u) & ~a) | ((b - 0x01010101u) & ~b)) & 0x80808080u;   // some byte is 0
  if (__builtin_expect(zero != 0 || s > 1.329227995784916e36f, 0)) {   // 2^120
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = int8_val(k < 4 ? w.x : w.y, k & 3, s);
    return;
  }
  const float o = -128.f * s;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = fmaf((float)((a >> (8 * k)) & 0xffu), s, o);
    v[4 + k] = fmaf((float)((b >> (8 * k)) & 0xffu), s, o);
  }
}

// two fp32 values -> packed bf16 (one v_cvt_pk_bf16_f32: nearest even, NaN kept)
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16v2));
}

// ---- 16-B accesses at any element: global_load / store_dwordx4 take addresses of any alignment, so rows
// of odd length or stride need no path of their own, only their last elements do
typedef uint32_t u32v4 __attribute__((ext_vector_type(4)));
typedef u32v4 u32v4_any __attribute__((aligned(2)));
__device__ __forceinline__ u32v4 load16(const void* p) { return *reinterpret_cast<const u32v4_any*>(p); }
__device__ __forceinline__ void store16(void* p, u32v4 v) { *reinterpret_cast<u32v4_any*>(p) = v; }

// 8 consecutive elements of a row, of which n (<= 0: none) are inside, as fp32
template <typename T>
__device__ __forceinline__ void load_upto(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const u32v4 a = load16(p), b = load16(p + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = __uint_as_float(a[k]);
        v[4 + k] = __uint_as_float(b[k]);
      }
    } else {
      const u32v4 w = load16(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? io<T>::ld(p + k) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_upto(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      store16(p, u32v4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
      store16(p + 4, u32v4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
    } else {
      store16(p, u32v4{bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7])});
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) io<T>::st(p + k, v[k]);
}

// max over the 16 lanes that hold one block's row (a DPP row): each step joins groups that already agree
__device__ __forceinline__ uint32_t max16u(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));    // lane ^ 1
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));    // lane ^ 2
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));   // mirrored in 8
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, false));   // mirrored in 16
}

}  // namespace q8
}  // namespace hx
