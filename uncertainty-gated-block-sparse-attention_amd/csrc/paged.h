// The paged key-value cache of the decode path: pages of 64 tokens (kBlock),
// named by a block table [B, max_pages] int32 (entry j of row b holds tokens
// 64 j .. 64 j + 63 of sequence b).
//
//   K, V    [P, Hk, 64, D] in the call's 16-bit format, or e4m3 bytes with a
//           scale byte per token and head ([P, Hk, 64]): value = code * 2^(byte - 127);
//           or e2m1 codes, two a byte (the even dim below), [P, Hk, 64, D / 2], with a
//           scale byte per 32 dims of a token's head ([P, Hk, D / 32, 64], so that the
//           keys which a lane reads lie side by side; byte 255: the 32 are NaN)
//   planes  [P, Hk, 2, D] in the 16-bit format: K-max and K-min of a page's keys as
//           they were given, the Quest summary of kernel 1, one block a page.  What a
//           page of codes holds of them is rounded, and may lie past the planes by half a
//           step: of e4m3 1/16 of its magnitude, or 2^-10 of the token's scale if that is
//           more; of e2m1 a quarter of its magnitude or of its scale
//
// Power-of-two scales keep every step exact but one: x 2^-e is exact, the
// rounding to e4m3's four significant bits is the only one, and what the write
// stored reads back exactly in its format, bf16 or fp16 (four bits at an exponent the
// unquantised value had; two of e2m1).  A float format loses next to nothing by it: the scale only has to
// place the token's largest magnitude in the top binade.
//
// Lengths and table entries are device data that the host cannot check.  A
// length is taken within [0, 64 max_pages], and a table entry outside [0, P) is
// an absent page: nothing is written to it and its keys take no part.
#pragma once

#include "common.h"
#include "launch.h"

namespace ugbsa {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(1))) u32x4 gu32x4;
typedef const __attribute__((address_space(1))) u32x2 gu32x2;
typedef const __attribute__((address_space(1))) uint32_t gu32;
typedef const __attribute__((address_space(1))) void gvoid;
typedef const __attribute__((address_space(4))) int32_t cint;   // read by scalar loads where the address is uniform

// A load, NT: of data read once, which need not displace other data from the caches.
template <bool NT, typename T>
__device__ __forceinline__ auto stream_load(T* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

// Eight e4m3 codes (lo: dims 0-3, hi: 4-7) times 2^(byte - 127) in E's format (exact).
template <typename E>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t codes, float scale, bool hi) {
  if constexpr (E::code == ElemF16::code)
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
  else
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}
template <typename E>
__device__ __forceinline__ bf16x8 e4m3_x8(uint32_t lo, uint32_t hi, float scale) {
  const u32x4 w = {e4m3_pair<E>(lo, scale, false), e4m3_pair<E>(lo, scale, true),
                   e4m3_pair<E>(hi, scale, false), e4m3_pair<E>(hi, scale, true)};
  return __builtin_bit_cast(bf16x8, w);
}
// Codes 2 SEL and 2 SEL + 1 of eight e2m1 codes, times 2^(byte - 127), in E's format
// (exact; NaN for byte 255).
template <typename E, int SEL>
__device__ __forceinline__ uint32_t e2m1_pair(uint32_t codes, float scale) {
  if constexpr (E::code == ElemF16::code)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
}
// A pair of E's values over scale, rounded to the nearest even code, as codes 2 SEL and
// 2 SEL + 1 of a word; magnitudes past 6 (and NaN) give 6.
template <typename E, int SEL>
__device__ __forceinline__ uint32_t e2m1_codes(uint32_t word, uint32_t pair, float scale) {
  if constexpr (E::code == ElemF16::code)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(f16x2, pair), scale, SEL);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(bf16x2, pair), scale, SEL);
}
template <typename E>
__device__ __forceinline__ u32x4 e2m1_x8(uint32_t codes, float scale) {
  return u32x4{e2m1_pair<E, 0>(codes, scale), e2m1_pair<E, 1>(codes, scale), e2m1_pair<E, 2>(codes, scale),
               e2m1_pair<E, 3>(codes, scale)};
}
__device__ __forceinline__ float e8m0(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ int cached_len(const int32_t* lens, int b, int max_pages) {
  const int64_t most = static_cast<int64_t>(max_pages) * kBlock;
  const int n = lens[b];
  return n < 0 ? 0 : (n > most ? static_cast<int>(most) : n);
}

}  // namespace ugbsa
