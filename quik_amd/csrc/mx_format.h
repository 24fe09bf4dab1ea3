// Blocks of 32 numbers that share a power of two: 4-bit (e2m1) or 8-bit (e4m3) floating-point codes and one byte per block, the biased
// exponent of 2^(byte - 127) (e8m0); the form that the scaled matrix instructions take.
//   byte = max(exponent of the block's largest magnitude - E, 0), E the exponent of the format's largest number (2: 6 = 1.5 * 2^2; 8: 448)
//   code = value / 2^(byte - 127), rounded to the nearest, of two to the even code, at most the largest number
// A block that holds a NaN or an infinity has codes 0 and the byte 255 (NaN): whatever it is multiplied by is a NaN.
// Two 4-bit codes per byte, the even column in the low half.
#pragma once
#include "rows_math.h"

namespace quik {
namespace {

constexpr int kMxBlock = 32;
constexpr uint32_t kMxNan = 255;

template <int BITS>
__device__ __forceinline__ uint32_t block_byte(uint32_t top_bits) {  // of the largest magnitude's fp32 pattern
  const int e = static_cast<int>(top_bits >> 23) - (BITS == 4 ? 2 : 8);
  return top_bits >= 0x7F800000u ? kMxNan : static_cast<uint32_t>(e > 0 ? e : 0);
}
// 2^(byte - 127); the byte 0 is fp32's subnormal 2^-127
__device__ __forceinline__ float block_unit(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }

// Eight values -> eight codes; all products with powers of two are exact.  (byte <= 253 where it is not NaN)
__device__ __forceinline__ uint32_t encode4(const float (&v)[8], uint32_t byte) {
  if (byte == kMxNan) return 0;
  const float unit = block_unit(byte);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], unit, 0);  // (nearest even, at most 6)
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], unit, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], unit, 3);
}
// (the conversion divides by the power of two; it does not stop at 448, but makes a NaN of numbers from 464 on)
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t byte) {
  if (byte == kMxNan) return make_uint2(0, 0);
  typedef short s2 __attribute__((ext_vector_type(2)));
  const float unit = block_unit(byte), most = 448.0f * unit;
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
  s2 lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, t[0], t[1], unit, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, t[2], t[3], unit, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, t[4], t[5], unit, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, t[6], t[7], unit, true);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Eight codes -> eight values (exact in fp32; NaNs where the byte is 255)
template <int BITS>
__device__ __forceinline__ void decode8(uint2 w, uint32_t byte, float (&v)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const float unit = block_unit(byte);
  f2 a, b, c, d;
  if constexpr (BITS == 4) {
    a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 0);
    b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 3);
  } else {
    a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), false);
    b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), true);
    c = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), false);
    d = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), true);
  }
  const float t[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = byte == kMxNan ? __builtin_nanf("") : t[i] * unit;
}

// n / d and n % d for n < 2^31: factor = min(2^32 / d, 2^32 - 1)
struct Divide {
  uint32_t d, factor;
  __device__ __forceinline__ uint32_t operator()(uint32_t n, uint32_t &rest) const {
    uint32_t q = __umulhi(n, factor);
    rest = n - q * d;
    if (rest >= d) {
      ++q;
      rest -= d;
    }
    return q;
  }
};
inline Divide divide_by(int64_t d) {
  const uint64_t f = (uint64_t{1} << 32) / static_cast<uint64_t>(d);
  return Divide{static_cast<uint32_t>(d), static_cast<uint32_t>(f > 0xFFFFFFFFull ? 0xFFFFFFFFull : f)};
}

// at the alignment of one element (global memory takes any)
typedef uint32_t mx_loose1 __attribute__((aligned(1)));

// the largest of four neighbouring lanes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  uint32_t o = static_cast<uint32_t>(dpp_move_i<kDppSwap1>(static_cast<int>(v)));
  v = v > o ? v : o;
  o = static_cast<uint32_t>(dpp_move_i<kDppSwap2>(static_cast<int>(v)));
  return v > o ? v : o;
}

// Eight columns of a 16-bit row, `left` (1 .. 8) of them there, zeros behind.
template <bool WIDE>
__device__ __forceinline__ void load_eight(const uint16_t *from, int left, uint16_t (&v)[8]) {
  if (WIDE || left == 8) {
    if constexpr (WIDE) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(from);
    else *reinterpret_cast<loose4 *>(v) = *reinterpret_cast<const loose4 *>(from);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? from[e] : 0;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store_eight(uint16_t *to, int left, const uint16_t (&v)[8]) {
  if (WIDE || left == 8) {
    if constexpr (WIDE) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(v);
    else *reinterpret_cast<loose4 *>(to) = *reinterpret_cast<const loose4 *>(v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) to[e] = v[e];
  }
}

// The codes of eight columns (`left` of them there; 4 bits: an even number) and, from the first lane of the block, its byte.  All four lanes of a
// block call this together; a lane without columns (left <= 0) has values 0.
template <int BITS, bool WIDE>
__device__ __forceinline__ void store_block(const float (&v)[8], int left, uint8_t *codes, uint8_t *byte_to, bool first) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t m = __float_as_uint(v[e]) & 0x7FFFFFFFu;
    top = top > m ? top : m;
  }
  const uint32_t byte = block_byte<BITS>(quad_max(top));
  if (left <= 0) return;
  if (first) *byte_to = static_cast<uint8_t>(byte);
  if constexpr (BITS == 4) {
    const uint32_t w = encode4(v, byte);
    if constexpr (WIDE) *reinterpret_cast<uint32_t *>(codes) = w;
    else if (left >= 8) *reinterpret_cast<mx_loose1 *>(codes) = w;
    else
      for (int e = 0; 2 * e < left; ++e) codes[e] = static_cast<uint8_t>(w >> (8 * e));
  } else {
    const uint2 w = encode8(v, byte);
    if constexpr (WIDE) *reinterpret_cast<uint2 *>(codes) = w;
    else if (left >= 8) *reinterpret_cast<loose2 *>(codes) = loose2{w.x, w.y};
    else
      for (int e = 0; e < left; ++e) codes[e] = static_cast<uint8_t>((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

}  // namespace
}  // namespace quik
