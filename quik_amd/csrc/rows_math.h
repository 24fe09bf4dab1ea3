// What the row kernels share (rows8.hip: codes with one scale per row; mxrows.hip: codes in blocks of 32): the values of a row, the norm's
// factor, reductions over a workgroup.
#pragma once
#include "common.h"

namespace quik {
namespace {

enum RowOp { kNorm, kNormAdd, kSiluMul };

// gate / (1 + exp(-gate)) * up.  exp2 and reciprocal are the hardware's, good to 1 ulp; with the rounding of exp2's argument a value is off by
// (1.5 |gate| + 10) 2^-24 of it (6e-7 at gates around 0, 3e-6 at -30).  From kFar down exp(-gate) nears the end of fp32's range, where a
// large up still makes a number of the value (and a row of nothing else has a scale): such a gate's exponential comes in halves, on either
// factor, until they are 0 from -175 on (a value below 2^-116 whatever up is); within the same bound.
constexpr uint32_t kFarBits = 0xC2AC0000u;  // -86: bits above are gates below (and negative NaNs)
__device__ __forceinline__ float gated(float gate, float up) {
  return gate * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gate * -1.44269504088896340736f)) * up;
}
__device__ __forceinline__ float gated_far(float gate, float up) {
  const float half = __builtin_amdgcn_exp2f(gate * 0.72134752044448170368f);
  return gate * half * (up * half);
}

template <bool BF16, RowOp OP, bool FAR>
__device__ __forceinline__ float row_value(float a, float b, float gain, uint16_t &h, float &square) {
  if constexpr (OP == kSiluMul) {
    return FAR && __float_as_uint(a) > kFarBits ? gated_far(a, b) : gated(a, b);
  } else {
    if constexpr (OP == kNormAdd) {
      h = from_f32<BF16>(a + b);
      a = to_f32<BF16>(h);
    }
    square += a * a;
    return a * gain;
  }
}

constexpr uint32_t kInfBits = 0x7F800000u;

// Rows of tiny bf16 numbers: where mean(h^2) + eps is below kTiny, squares may lie below fp32's smallest numbers, and the sum is made again
// of h * kLift (2^-133 and more: squares from 2^-74 up; (2^31 columns) * kTiny * kLift^2 = 2^123).  fp16 squares are 2^-48 and more.
constexpr float kTiny = 0x1p-100f, kLift = 0x1p96f;
template <bool BF16, RowOp OP>
__device__ __forceinline__ bool tiny_squares(uint32_t top_bits, float square, int64_t cols, float eps) {
  return BF16 && OP != kSiluMul && top_bits != 0 && square < (kTiny - eps) * static_cast<float>(cols);
}
// the norm's factor from the sum of the squares of h * lift, over lift
__device__ __forceinline__ float norm_factor(float square, int64_t cols, float eps, float lift) {
  return 1.0f / sqrtf(square / static_cast<float>(cols) + eps * lift * lift);
}

__device__ __forceinline__ float wave_sum_f(float v) {
  v += dpp_move<kDppSwap1>(v);
  v += dpp_move<kDppSwap2>(v);
  v += dpp_move<kDppHalfMirror>(v);
  v += dpp_move<kDppMirror>(v);
  const int b = __builtin_bit_cast(int, v);
  return (__builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16))) +
         (__builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48)));
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = umax(v, static_cast<uint32_t>(dpp_move_i<kDppSwap1>(static_cast<int>(v))));
  v = umax(v, static_cast<uint32_t>(dpp_move_i<kDppSwap2>(static_cast<int>(v))));
  v = umax(v, static_cast<uint32_t>(dpp_move_i<kDppHalfMirror>(static_cast<int>(v))));
  v = umax(v, static_cast<uint32_t>(dpp_move_i<kDppMirror>(static_cast<int>(v))));
  const uint32_t r0 = __builtin_amdgcn_readlane(v, 0), r1 = __builtin_amdgcn_readlane(v, 16), r2 = __builtin_amdgcn_readlane(v, 32),
                 r3 = __builtin_amdgcn_readlane(v, 48);
  return umax(umax(r0, r1), umax(r2, r3));
}

// top and square over the workgroup (up to 16 waves)
__device__ __forceinline__ void block_reduce(uint32_t &top, float &square, uint32_t *red) {
  top = wave_max_u(top);
  square = wave_sum_f(square);
  const int waves = static_cast<int>(blockDim.x >> 6);
  if (waves == 1) return;
  float *reds = reinterpret_cast<float *>(red + 16);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = top;
    reds[threadIdx.x >> 6] = square;
  }
  __syncthreads();
  top = red[0];
  square = reds[0];
  for (int w = 1; w < waves; ++w) {
    top = umax(top, red[w]);
    square += reds[w];
  }
}

// a further sum of the workgroup's
__device__ __forceinline__ void block_sum(float &v, uint32_t *red) {
  __syncthreads();  // (the sums before are read)
  uint32_t none = 0;
  block_reduce(none, v, red);
}

// Sixteen bytes at the alignment of one element (global memory takes any), eight codes at any.
typedef uint32_t loose4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(1)));

}  // namespace
}  // namespace quik
