// Products with 4-bit weights that have one scale (and zero) per group of a row:
//   y[m, n] = s_row[m] * sum_g s[n, g] * ( sum_{k in g} x[m, k] q[n, k] - z[n, g] * sum_{k in g} x[m, k] ) + bias[n]
// x fp16, bf16 or int8 (then with s_row), q signed 4-bit codes as int4Matmul takes them (two per byte, low nibble = even k), groups of
// G columns (a multiple of 32, the last one may be shorter).
//
// The weights never leave 4 bits in memory; a wave widens them in registers, in front of the matrix instruction:
//   fp16  (w & 0x000F000F) ^ 0x64086408 is the pair 1032 + q, one packed subtraction leaves q; exact
//   bf16  (w & 0x000F000F) ^ 0x43084308 is the pair 136 + q (there is no packed bf16 subtraction): the 136 goes the way of the zeros
//   int8  w & 0xF0F0F0F0 and (w << 4) & 0xF0F0F0F0 are 16 q; the 16 leaves with the scale
// Each group's product is a matrix-core sum of its own (fp32; exact int32 for int8), scaled in fp32: no product of a scale and a code is
// rounded to 16 bits.  sum x of a group comes from the same instruction with a matrix of ones.
#include "common.h"

#include <type_traits>

namespace quik {
namespace {

enum Acts { kF16, kBF16, kI8 };

struct GroupArgs {
  const void *x;
  const uint8_t *w;
  const void *scales, *zeros;
  const float *scale_row;
  const void *bias;
  void *out;
  int64_t M, N, K;
  int32_t G, groups;
  int32_t out_bf16;
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

template <int XT>
using Acc = std::conditional_t<XT == kI8, i32x4, f32x4>;

// one 32-column step: eight k per lane and operand
template <int XT>
__device__ __forceinline__ Acc<XT> mfma32(u32x4 a, u32x4 b, Acc<XT> c) {
  if constexpr (XT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// eight codes -> eight 16-bit values in the order k0 k4 k1 k5 k2 k6 k3 k7
template <int XT>
__device__ __forceinline__ u32x4 widen16(uint32_t w) {
  u32x4 r;
  if constexpr (XT == kF16) {
    const half2v one = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = ((w >> (4 * i)) & 0x000F000Fu) ^ 0x64086408u;
      r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, t) - one);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = ((w >> (4 * i)) & 0x000F000Fu) ^ 0x43084308u;
  }
  return r;
}
// sixteen-bit activations of eight columns in that order
__device__ __forceinline__ u32x4 order16(u32x4 v) {
  u32x4 r;
  r[0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100u);
  r[1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302u);
  r[2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100u);
  r[3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302u);
  return r;
}
// eight codes -> eight bytes of 16 q: k0 k2 k4 k6, k1 k3 k5 k7
__device__ __forceinline__ u32x2 widen8(uint32_t w) { return u32x2{(w << 4) & 0xF0F0F0F0u, w & 0xF0F0F0F0u}; }
__device__ __forceinline__ u32x2 order8(u32x2 v) {
  return u32x2{__builtin_amdgcn_perm(v[1], v[0], 0x06040200u), __builtin_amdgcn_perm(v[1], v[0], 0x07050301u)};
}

// dword s of lane row r <-> dword r of lane row s (four rows of 16 lanes)
__device__ __forceinline__ void transpose4(u32x4 &v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false), b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = u32x4{static_cast<uint32_t>(c[0]), static_cast<uint32_t>(c[1]), static_cast<uint32_t>(d[0]), static_cast<uint32_t>(d[1])};
}

__device__ __forceinline__ float load16(const void *p, int64_t i, bool bf16) {
  const uint16_t v = static_cast<const uint16_t *>(p)[i];
  return bf16 ? to_f32<true>(v) : to_f32<false>(v);
}

// Weight-streaming kernel.  A workgroup takes 16 * FT output columns and 16 * MT token rows (RR < 4: 4 * RR rows, in the result
// registers 0 .. RR - 1); its W waves take the 128-column blocks of K in turn and add their sums through LDS at the end.  Lane
// l of a wave holds 32 codes (16 bytes) of weight row l % 16, columns 32 (l / 16) .. of the block.
// SMALL: groups that are no multiple of 128.  The codes are exchanged between the lane rows so that matrix step s is columns 32 s
// .. 32 s + 31 of the block, which one group holds; otherwise step s is columns 8 s .. 8 s + 7 of each lane row's 32.
template <int XT, int RR, int MT, int FT, int W, bool SMALL, bool ZEROS>
__global__ __launch_bounds__(64 * W) void group4_stream_kernel(GroupArgs p) {
  constexpr bool kSums = ZEROS || XT == kBF16;
  constexpr int kX = XT == kI8 ? 2 : 4;  // 16-byte pieces of activations per lane and block
  extern __shared__ float red[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * FT), m0 = static_cast<int64_t>(blockIdx.y) * (RR < 4 ? 4 * RR : 16 * MT);
  const bool sbf = XT == kI8 ? p.out_bf16 : XT == kBF16;
  const uint8_t *wp[FT];
  int64_t sp[FT];
#pragma unroll
  for (int t = 0; t < FT; ++t) {
    const int64_t n = n0 + 16 * t + col < p.N ? n0 + 16 * t + col : p.N - 1;
    wp[t] = p.w + n * (p.K / 2);
    sp[t] = n * p.groups;
  }
  const uint8_t *xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    int64_t m = m0 + (RR < 4 ? (col >> 2) * RR + ((col & 3) < RR ? (col & 3) : RR - 1) : 16 * t + col);
    m = m < p.M ? m : p.M - 1;
    xp[t] = static_cast<const uint8_t *>(p.x) + m * p.K * (XT == kI8 ? 1 : 2);
  }
  float total[FT][MT][RR];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < RR; ++r) total[f][t][r] = 0.0f;

  const int blocks = static_cast<int>((p.K + 127) >> 7);
  for (int blk = wave; blk < blocks; blk += W) {
    const int64_t k0 = static_cast<int64_t>(blk) * 128, kl = k0 + 32 * kg;
    const bool in = kl < p.K;
    u32x4 w[FT], x[MT][kX];
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      w[f] = *reinterpret_cast<const u32x4 *>(wp[f] + (in ? kl / 2 : 0));
      if constexpr (SMALL) transpose4(w[f]);
    }
    if constexpr (!SMALL) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < kX; ++i) {
          x[t][i] = *reinterpret_cast<const u32x4 *>(xp[t] + (in ? kl * (XT == kI8 ? 1 : 2) + 16 * i : 0));
          if (!in) x[t][i] = u32x4{0, 0, 0, 0};  // (past the end of K)
        }
    }
    constexpr int kParts = SMALL ? 4 : 1;  // sums of their own per block
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int64_t kp = k0 + 32 * part;
      if (SMALL && kp >= p.K) break;
      const int g = static_cast<int>(kp / p.G);
      Acc<XT> acc[FT][MT], sums[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        sums[t] = Acc<XT>{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < FT; ++f) acc[f][t] = Acc<XT>{0, 0, 0, 0};
      }
      if constexpr (XT == kI8) {
        const int one = 0x01010101;
        if constexpr (SMALL) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const u32x2 xo = order8(*reinterpret_cast<const u32x2 *>(xp[t] + kp + 8 * kg));
            const long xa = __builtin_bit_cast(long, xo);
            if constexpr (kSums) sums[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, __builtin_bit_cast(long, u32x2{0x01010101u, 0x01010101u}), sums[t], 0, 0, 0);
#pragma unroll
            for (int f = 0; f < FT; ++f) acc[f][t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, __builtin_bit_cast(long, widen8(w[f][part])), acc[f][t], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            i32x4 xa[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const u32x2 lo = order8(u32x2{x[t][s][0], x[t][s][1]}), hi = order8(u32x2{x[t][s][2], x[t][s][3]});
              xa[t] = i32x4{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]), static_cast<int>(hi[1])};
              if constexpr (kSums) sums[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa[t], i32x4{one, one, one, one}, sums[t], 0, 0, 0);
            }
#pragma unroll
            for (int f = 0; f < FT; ++f) {
              const u32x2 lo = widen8(w[f][2 * s]), hi = widen8(w[f][2 * s + 1]);
              const i32x4 wb = {static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]), static_cast<int>(hi[1])};
#pragma unroll
              for (int t = 0; t < MT; ++t) acc[f][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa[t], wb, acc[f][t], 0, 0, 0);
            }
          }
        }
      } else {
        const uint32_t one = XT == kBF16 ? 0x3F803F80u : 0x3C003C00u;
        constexpr int kSteps = SMALL ? 1 : 4;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          u32x4 xa[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if constexpr (SMALL)
              xa[t] = order16(*reinterpret_cast<const u32x4 *>(xp[t] + (kp + 8 * kg) * 2));
            else
              xa[t] = order16(x[t][s]);
            if constexpr (kSums) sums[t] = mfma32<XT>(xa[t], u32x4{one, one, one, one}, sums[t]);
          }
#pragma unroll
          for (int f = 0; f < FT; ++f) {
            const u32x4 wb = widen16<XT>(w[f][SMALL ? part : s]);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[f][t] = mfma32<XT>(xa[t], wb, acc[f][t]);
          }
        }
      }
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        const float s = load16(p.scales, sp[f] + g, sbf);
        const float z = (XT == kBF16 ? 136.0f : 0.0f) + (ZEROS ? load16(p.zeros, sp[f] + g, sbf) * (XT == kI8 ? 16.0f : 1.0f) : 0.0f);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            float d = static_cast<float>(acc[f][t][r]);
            if constexpr (kSums) d = __builtin_fmaf(-z, static_cast<float>(sums[t][r]), d);
            total[f][t][r] = __builtin_fmaf(s, d, total[f][t][r]);
          }
      }
    }
  }
  // the waves' sums
  constexpr int kRegs = FT * MT * RR;
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < RR; ++r) red[(wave * kRegs + (f * MT + t) * RR + r) * 64 + lane] = total[f][t][r];
  __syncthreads();
  for (int e = threadIdx.x; e < kRegs * 64; e += 64 * W) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += red[i * kRegs * 64 + e];
    const int reg = e >> 6, l = e & 63, r = reg % RR, t = reg / RR % MT, f = reg / (RR * MT);
    const int64_t n = n0 + 16 * f + (l & 15), m = m0 + (RR < 4 ? (l >> 4) * RR + r : 16 * t + 4 * (l >> 4) + r);
    if (n < p.N && m < p.M) {
      if constexpr (XT == kI8) v *= p.scale_row[m] * 0.0625f;
      if (p.bias) v += load16(p.bias, n, sbf);
      static_cast<uint16_t *>(p.out)[m * p.N + n] = sbf ? from_f32<true>(v) : from_f32<false>(v);
    }
  }
}

template <int XT, int RR, int MT, int FT, bool SMALL, bool ZEROS>
int launch_stream(const GroupArgs &p, hipStream_t st) {
  constexpr int W = 8, smem = W * FT * MT * RR * 64 * 4, rows = RR < 4 ? 4 * RR : 16 * MT;
  auto kern = group4_stream_kernel<XT, RR, MT, FT, W, SMALL, ZEROS>;
  if (int rc = prepare(kern, smem)) return rc;
  const dim3 grid(static_cast<unsigned>((p.N + 16 * FT - 1) / (16 * FT)), static_cast<unsigned>((p.M + rows - 1) / rows));
  hipLaunchKernelGGL(kern, grid, dim3(64 * W), smem, st, p);
  return check_launch();
}

template <int XT, bool SMALL, bool ZEROS>
int by_rows(const GroupArgs &p, hipStream_t st) {
  if (p.M <= 4) return launch_stream<XT, 1, 1, 2, SMALL, ZEROS>(p, st);
  if (p.M <= 8) return launch_stream<XT, 2, 1, 2, SMALL, ZEROS>(p, st);
  if (p.M <= 16) return launch_stream<XT, 4, 1, 2, SMALL, ZEROS>(p, st);
  if (p.M <= 32) return launch_stream<XT, 4, 2, 2, SMALL, ZEROS>(p, st);
  return launch_stream<XT, 4, 4, 2, SMALL, ZEROS>(p, st);
}

template <int XT>
int by_groups(const GroupArgs &p, hipStream_t st) {
  const bool small = p.G % 128 != 0 && p.groups > 1;
  if (p.zeros) return small ? by_rows<XT, true, true>(p, st) : by_rows<XT, false, true>(p, st);
  return small ? by_rows<XT, true, false>(p, st) : by_rows<XT, false, false>(p, st);
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int quik_int4_group_matmul(const void *x, int x_bits, const uint8_t *w, const void *scales, const void *zeros,
                                      const float *scale_row, const void *bias, int dtype, int64_t M, int64_t N, int64_t K, int64_t group,
                                      void *out, void *stream) {
  if (x_bits != 8 && x_bits != 16) return QUIK_ERR_BITS;
  if (dtype != QUIK_F16 && dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || group <= 0) return QUIK_ERR_SHAPE;
  if (K % 32 || group % 32) return QUIK_ERR_ALIGN;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return QUIK_ERR_RANGE;
  if ((M + 63) / 64 > 65535) return QUIK_ERR_RANGE;  // (one grid dimension)
  if (M == 0 || N == 0) return QUIK_OK;
  if (!x || !w || !scales || !out || (x_bits == 8 && !scale_row)) return QUIK_ERR_NULL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(scales, 2) || !aligned(zeros, 2) || !aligned(scale_row, 4) || !aligned(bias, 2) ||
      !aligned(out, 2))
    return QUIK_ERR_ALIGN;
  const int64_t g = group < K ? group : (K + 31) / 32 * 32;
  const GroupArgs p{x, w, scales, zeros, x_bits == 8 ? scale_row : nullptr, bias, out, M, N, K, static_cast<int32_t>(g),
                    static_cast<int32_t>((K + g - 1) / g), dtype == QUIK_BF16};
  if (x_bits == 8) return by_groups<kI8>(p, as_stream(stream));
  return dtype == QUIK_BF16 ? by_groups<kBF16>(p, as_stream(stream)) : by_groups<kF16>(p, as_stream(stream));
}
