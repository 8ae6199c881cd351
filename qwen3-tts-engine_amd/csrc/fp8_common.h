// The 8-bit K/V pool's row format, shared by the kernels that write it and those that read it (gfx950).
//
// A row is one token of one KV head: 128 e4m3 codes and one exponent byte s, value = code * 2^(s - 127).  The writer takes
// the smallest power of two that brings the row's largest finite magnitude a to at most 448 (the largest e4m3 number):
//   a = f * 2^x with 1 <= f < 2;  448 = 1.75 * 2^8;  e = x - 8 (+ 1 if f > 1.75), at least -117;  s = e + 127.
// A power of two, because x * 2^-e and code * 2^e are then exact: the rounding to e4m3 (nearest even, 4 significant bits,
// half a step 2^-4 of the value at worst) is the only one, the value read back is a bf16 number as it is, and attention over
// the pool equals attention over the bf16 rows read back from it.  A scale with a mantissa would gain at most the one bit
// of range below 2^(e - 6), where e4m3 spaces its codes evenly.  At e = -117 the smallest code, 2^-9, is 2^-126, still a
// normal number; at the largest e, 120, codes stop at 240 (256 * 2^120 would be past the largest bf16, and fp32).
// Elements that are not finite are held as NaN, and do not enter a.
#pragma once

#include "q3a_common.h"

namespace q3a {

constexpr int kRowDims = 128;
constexpr int kMinScaleByte = 10;   // 2^-117
constexpr int kMaxScaleByte = 247;  // 2^120, of rows over 448 * 2^119

// bf16 magnitude bits of the row's largest finite element (0..0x7f7f) -> exponent byte.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bf16) {
  const int s = (int)(amax_bf16 >> 7) - 8 + ((amax_bf16 & 0x7f) > 0x60 ? 1 : 0);
  return (uint32_t)max(s, kMinScaleByte);
}
// 2^(s - 127) and 2^(127 - s) for the bytes that the writer makes (10..247).
__device__ __forceinline__ float fp8_scale(uint32_t s) { return __uint_as_float(s << 23); }
__device__ __forceinline__ float fp8_inv_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Largest magnitude bits over the pairs of n dwords of bf16, elements that are not finite left out; as packed halves.
template <int N>
__device__ __forceinline__ uint32_t bf16_amax_pair(const uint32_t (&w)[N]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) a = pk_max_u16(a, w[i] & 0x7fff7fffu);
  if ((a & 0xffffu) >= 0x7f80u || (a >> 16) >= 0x7f80u) {  // some element is inf or NaN: again without those
    a = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t m = w[i] & 0x7fff7fffu;
      if ((m & 0xffffu) >= 0x7f80u) m &= 0xffff0000u;
      if ((m >> 16) >= 0x7f80u) m &= 0xffffu;
      a = pk_max_u16(a, m);
    }
  }
  return a;
}
__device__ __forceinline__ uint32_t halves_max(uint32_t a) { return max(a & 0xffffu, a >> 16); }

// The same whatever the elements are.
template <int N>
__device__ __forceinline__ uint32_t bf16_any_amax_pair(const uint32_t (&w)[N]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) a = pk_max_u16(a, w[i] & 0x7fff7fffu);
  return a;
}
// The pair with NaN in the halves that are not finite.
__device__ __forceinline__ uint32_t nan_if_not_finite(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w |= 0x7fu;
  if ((w & 0x7f800000u) == 0x7f800000u) w |= 0x7f0000u;
  return w;
}
// Rows with infinities and NaN, or close to the largest bf16, are rare: their codes need care (bf16_amax_pair, fp8_codes4).
// True on all lanes if one's largest magnitude bits tell so.
__device__ __forceinline__ bool any_rare(uint32_t top) { return __builtin_amdgcn_ballot_w64(top >= 0x7f00u) != 0; }

// Two dwords of bf16 (4 elements) -> one dword of e4m3 codes, of finite elements up to 448 scale.
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2_t;
__device__ __forceinline__ uint32_t fp8_finite_codes4(uint32_t w0, uint32_t w1, float scale) {
  s16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w0), scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w1), scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Two dwords of bf16 (4 elements) -> one dword of e4m3 codes at the exponent byte s.
__device__ __forceinline__ uint32_t fp8_codes4(uint32_t w0, uint32_t w1, uint32_t s) {
  const float inv = fp8_inv_scale(s), most = s >= kMaxScaleByte ? 240.f : 448.f;
  auto one = [&](float x) {
    // v_cvt_pk_fp8_f32 of an infinity depends on the mode; here everything that is not finite becomes NaN
    const float y = x * inv;
    return fabsf(y) <= 448.f ? __builtin_amdgcn_fmed3f(y, -most, most) : __builtin_nanf("");
  };
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(one(bf16_lo(w0)), one(bf16_hi(w0)), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(one(bf16_lo(w1)), one(bf16_hi(w1)), r, true);
  return (uint32_t)r;
}

// One half (two codes) of a dword of codes -> a pair of bf16, times the power of two `scale` (exact).
template <bool kHi>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHi));
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u32(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}

// x / d for x < 2^31: with 2^s >= d the multiplier is at most 1 too large, which x carries on by less than 1 / d.
struct Divisor {
  uint32_t d, m;
  int shift;
};
__device__ __forceinline__ uint32_t divide(uint32_t x, const Divisor& d) { return (uint32_t)(((uint64_t)x * d.m) >> d.shift); }
inline Divisor divisor(uint32_t d) {
  int s = 0;
  while (((uint64_t)1 << s) < d) ++s;
  return {d, (uint32_t)(((uint64_t)1 << (31 + s)) / d + 1), 31 + s};
}

// A pool's pointers, strides and sizes as every entry point over it needs them (kv_fp8.hip): Q3A_OK, or the error for the caller.
int check_fp8_pool(const char* who, const void* kc, const void* vc, int64_t sp, int64_t st, int64_t sh, const void* ks,
                   const void* vs, int64_t ss_p, int64_t ss_h, int num_pages, int page_size, int hkv);

// Rows k, v [tokens, hkv, 128] of bf16 and their slots, as the pools' writes and reads take them (kv_fp8.hip).
int check_pool_rows(const char* who, const void* k, const void* v, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                    const void* slots, int64_t tokens, int hkv, int head_dim);

}  // namespace q3a
