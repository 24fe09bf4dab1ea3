// Products with 4-bit weights that have one scale (and zero) per group of a row:
//   y[m, n] = s_row[m] * sum_g s[n, g] * ( sum_{k in g} x[m, k] q[n, k] - z[n, g] * sum_{k in g} x[m, k] ) + bias[n]
// x fp16, bf16 or int8 (then with s_row), q signed 4-bit codes as int4Matmul takes them (two per byte, low nibble = even k), groups of
// G columns (a multiple of 32, the last one may be shorter).
//
// The weights never leave 4 bits in memory; a wave widens them in registers, in front of the matrix instruction:
//   fp16  few rows: a nibble in a half of zeros is the subnormal (q + 8) 2^-24 or, four bits up, 2^-20; many rows: a nibble under the bits of
//         1024 is 1032 + q or 1152 + 16 q, and one packed fma leaves q.  All exact.
//   bf16  a nibble under the bits of 128 is 136 + q (there is no packed bf16 subtraction): the 136 goes the way of the zeros
//   int8  w & 0xF0F0F0F0 and (w << 4) & 0xF0F0F0F0 are 16 q; the 16 leaves with the scale
// The product of a block of up to 128 columns of one group (32 in the kernel of few rows where groups are no multiples of 128) is a
// matrix-core sum of its own (fp32; exact int32 for int8), scaled and added to the others in fp32: no product of a scale and a code is rounded
// to 16 bits.  sum x of a block comes from the same instruction with a matrix of ones.
//
// Times are per launch, launches one after the other, three weight matrices in turn, groups of 128 without zeros and K not split where nothing
// else is said.  Up to 16 rows the stream of codes bounds it (group4_decode_kernel: 1 x 8192 -> 28672 fp16 26.5 us, 4.6 TB/s; bf16 with zeros
// 30.9; 16 x 13824 -> 5120 int8 8.6; a copy on this card 5.2 TB/s).  Above, neither the vector nor the matrix unit is full (group4_tile_kernel:
// 2048 x 4096 -> 11008 int8 140 us, 1320 TOP/s, fp16 205, 900 TFLOP/s, bf16 217): of a SIMD's cycles vector instructions take 43 % (int8; fp16 29,
// bf16 35), matrix instructions 25 (37, 35), and the rest is waiting: two waves per SIMD, kept in step by a barrier per 128 columns.  Per
// result and group there are a conversion (int8) and an fma beside the matrix instructions, and the widening, which a matrix instruction hides
// two to three of (measured: 16 cycles alone, 19 with two vector instructions beside it, 39 with eight).  Widening less often is why the
// wide tiles are 128 rows per wave.
#include "common.h"

#include <type_traits>

namespace quik {
namespace {

// activations and the type of everything else: fp16 with fp16, bf16 with bf16, int8 with fp16 or bf16 scales and results
enum Acts { kF16, kBF16, kI8F16, kI8BF16 };
constexpr bool is_i8(int xt) { return xt >= kI8F16; }
constexpr bool is_bf16(int xt) { return xt == kBF16 || xt == kI8BF16; }  // scales and results

struct GroupArgs {
  const void *x;
  const uint8_t *w;
  const void *scales, *zeros;
  const float *scale_row;
  const void *bias;
  void *out;
  int64_t M, N, K;
  int32_t G, groups;
  int32_t width;   // columns per tile of the kernel of few rows
  float *partial;  // K split: sums [splits][M][N rounded up to 4]
  int32_t splits;
  uint32_t group_factor;  // ceil(2^31 / (G / 32)): group of a unit of 32 columns = unit * group_factor >> 31
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

template <int XT>
using Acc = std::conditional_t<is_i8(XT), i32x4, f32x4>;

// one 32-column step: eight k per lane and operand
template <int XT>
__device__ __forceinline__ Acc<XT> mfma32(u32x4 a, u32x4 b, Acc<XT> c) {
  if constexpr (XT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// eight fp16 codes in the order of the columns: a byte of two codes to both halves is (1032 + q, 1152 + 16 q), one packed fma leaves q
__device__ __forceinline__ u32x4 widen_f16(uint32_t w) {
  u32x4 r;
  const half2v factor = {static_cast<_Float16>(1.0f), static_cast<_Float16>(0.0625f)}, less = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-72.0f)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = (__builtin_amdgcn_perm(w, w, 0x0C000C00u + 0x00010001u * i) & 0x00F0000Fu) ^ 0x64806408u;
    r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, t), factor, less));
  }
  return r;
}
// eight codes -> eight bytes of 16 q in the order of the columns
__device__ __forceinline__ u32x2 widen8_in_order(uint32_t w) {
  const uint32_t even = (w << 4) & 0xF0F0F0F0u, odd = w & 0xF0F0F0F0u;
  return u32x2{__builtin_amdgcn_perm(odd, even, 0x05010400u), __builtin_amdgcn_perm(odd, even, 0x07030602u)};
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

__device__ __forceinline__ float from16(uint32_t low, bool bf16) {
  const uint16_t v = static_cast<uint16_t>(low);
  return bf16 ? to_f32<true>(v) : to_f32<false>(v);
}
__device__ __forceinline__ float load16(const void *p, int64_t i, bool bf16) {
  const uint16_t v = static_cast<const uint16_t *>(p)[i];
  return bf16 ? to_f32<true>(v) : to_f32<false>(v);
}

// eight bf16 codes in the order of the columns: a byte of two codes to both halves, then each half its nibble (the odd codes
// from w >> 4)
__device__ __forceinline__ u32x4 widen_bf16(uint32_t w) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (__builtin_amdgcn_perm(w >> 4, w, 0x0C040C00u + 0x00010001u * i) & 0x000F000Fu) ^ 0x43084308u;
  return r;
}
// Sixteen fp16 codes of two words as subnormals: a nibble at the low end of a half is (q + 8) 2^-24, one at bits 4 .. 7 is (q + 8)
// 2^-20, both exact operands of the matrix instruction.  Low nibbles: columns 0 4, 2 6 of each word; high ones: 1 5, 3 7.
__device__ __forceinline__ u32x4 widen_f16_low(uint32_t w0, uint32_t w1) {
  return u32x4{(w0 & 0x000F000Fu) ^ 0x00080008u, ((w0 >> 8) & 0x000F000Fu) ^ 0x00080008u, (w1 & 0x000F000Fu) ^ 0x00080008u,
               ((w1 >> 8) & 0x000F000Fu) ^ 0x00080008u};
}
__device__ __forceinline__ u32x4 widen_f16_high(uint32_t w0, uint32_t w1) {
  return u32x4{(w0 & 0x00F000F0u) ^ 0x00800080u, ((w0 >> 8) & 0x00F000F0u) ^ 0x00800080u, (w1 & 0x00F000F0u) ^ 0x00800080u,
               ((w1 >> 8) & 0x00F000F0u) ^ 0x00800080u};
}
// activations of the same sixteen columns (a: the first eight)
__device__ __forceinline__ u32x4 order_f16(u32x4 a, u32x4 b, uint32_t sel) {
  return u32x4{__builtin_amdgcn_perm(a[2], a[0], sel), __builtin_amdgcn_perm(a[3], a[1], sel), __builtin_amdgcn_perm(b[2], b[0], sel),
               __builtin_amdgcn_perm(b[3], b[1], sel)};
}

// Up to 16 token rows (4 * RR of them in the result registers 0 .. RR - 1).  A workgroup takes tiles of p.width <= 16 * FT output columns, which
// deals all columns evenly to the CUs (the matrix columns behind them repeat the last one's codes, which are not read from memory again); its W
// waves take the 128-column blocks of K in turn and add their sums through LDS at a tile's end.  Codes, activations, scales and
// zeros come to LDS by direct copies, D - 1 blocks ahead and on into the next tile, into a ring of the wave's own (no barrier
// but at a tile's end): a matrix operand wants 16 rows side by side, of which four neighbouring lanes that loaded it to registers
// would touch four lines of memory; as copies they take 64 or 256 bytes of a row.  Pieces of 16 bytes lie in the ring so that eight
// lanes read them from different banks.
template <int XT, int RR, int FT, int W, int D, bool SMALL, bool ZEROS>
__global__ __launch_bounds__(64 * W) void group4_decode_kernel(GroupArgs p) {
  constexpr bool kSums = ZEROS || !is_i8(XT);      // 16-bit codes are widened with an offset
  constexpr int kX = is_i8(XT) ? 2 : 4;           // 16-byte pieces of activations per lane and block
  constexpr int kRowPieces = is_i8(XT) ? 8 : 16;  // of a row
  constexpr int kSize = is_i8(XT) ? 1 : 2;
  constexpr int kCopiesX = is_i8(XT) ? (RR + 1) / 2 : RR;
  constexpr int kCopiesS = SMALL ? FT : (FT + 3) / 4;  // of 64 scales: 64 columns, or (SMALL) 16 columns at 4 groups
  constexpr int kCopies = FT + kCopiesX + kCopiesS * (ZEROS ? 2 : 1);
  constexpr int kAtX = FT * 1024, kAtS = kAtX + kCopiesX * 1024, kAtZ = kAtS + kCopiesS * 256, kStage = kAtS + kCopiesS * 256 * (ZEROS ? 2 : 1);
  constexpr int kRegs = FT * RR;
  extern __shared__ float red[];  // W * kRegs * 64 sums, then the rings
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  constexpr bool sbf = is_bf16(XT);
  const int blocks = static_cast<int>((p.K + 127) >> 7), tiles = static_cast<int>((p.N + p.width - 1) / p.width);
  uint8_t *ring = reinterpret_cast<uint8_t *>(red) + W * kRegs * 256 + wave * (D * kStage);
  const uint32_t ring_at = lds_address(ring);

  // where this lane's copies come from: piece (lane % 4) ^ (row / 2 % 4) of weight row lane / 4, and of an activation row likewise
  const int cw = (lane & 3) ^ ((lane >> 3) & 3), last_w = static_cast<int>(p.K / 32) - 1;
  const int last_x = static_cast<int>(p.K * kSize / 16) - 1;
  int cx[kCopiesX];
  uint32_t from_x[kCopiesX];
#pragma unroll
  for (int i = 0; i < kCopiesX; ++i) {
    const int64_t left = p.M - 1, row = (64 / kRowPieces) * i + lane / kRowPieces;
    cx[i] = (lane % kRowPieces) ^ static_cast<int>(row % kRowPieces);
    from_x[i] = static_cast<uint32_t>((row < left ? row : left) * p.K * kSize);
  }
  uint32_t from_w[FT], from_s[kCopiesS];
  const uint8_t *wbase, *sbase, *zbase;
  auto aim = [&](int tile) {  // at a tile's columns (past its end: the last one)
    const int64_t n0 = static_cast<int64_t>(tile) * p.width, left = (p.N - n0 < p.width ? p.N - n0 : p.width) - 1;
    wbase = p.w + n0 * (p.K / 2);
    sbase = static_cast<const uint8_t *>(p.scales) + n0 * p.groups * 2;
    zbase = static_cast<const uint8_t *>(p.zeros) + n0 * p.groups * 2;
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const int64_t row = 16 * f + (lane >> 2);
      from_w[f] = static_cast<uint32_t>((row < left ? row : left) * (p.K / 2));
    }
#pragma unroll
    for (int i = 0; i < kCopiesS; ++i) {
      int64_t row = SMALL ? 16 * i + col : 64 * i + lane;
      row = row < 16 * FT ? row : 16 * FT - 1;
      from_s[i] = static_cast<uint32_t>((row < left ? row : left) * p.groups * 2);
    }
  };
  auto group_of = [&](int unit) { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(unit)) * p.group_factor) >> 31); };
  auto copy = [&](int stage, int blk) {
    const uint32_t to = ring_at + stage * kStage;
    if (blk * 128 + 128 <= p.K) {
      const uint8_t *wfrom = wbase + blk * 64, *xfrom = static_cast<const uint8_t *>(p.x) + blk * (128 * kSize);
#pragma unroll
      for (int f = 0; f < FT; ++f) dma_load16(wfrom, from_w[f] + cw * 16, to + f * 1024);
#pragma unroll
      for (int i = 0; i < kCopiesX; ++i) dma_load16(xfrom, from_x[i] + cx[i] * 16, to + kAtX + i * 1024);
    } else {  // (pieces past the end of a row come from its last one)
      const int at = blk * 4 + cw;
      const uint32_t w_at = static_cast<uint32_t>(at < last_w ? at : last_w) * 16;
#pragma unroll
      for (int f = 0; f < FT; ++f) dma_load16(wbase, from_w[f] + w_at, to + f * 1024);
#pragma unroll
      for (int i = 0; i < kCopiesX; ++i) {
        const int xa = blk * kRowPieces + cx[i];
        dma_load16(static_cast<const uint8_t *>(p.x), from_x[i] + static_cast<uint32_t>(xa < last_x ? xa : last_x) * 16, to + kAtX + i * 1024);
      }
    }
    if constexpr (SMALL) {
      const int unit = blk * 4 + kg;
      const uint32_t g = 2 * group_of(unit < last_w ? unit : last_w);
#pragma unroll
      for (int i = 0; i < kCopiesS; ++i) {
        dma_load_u16(sbase, from_s[i] + g, to + kAtS + i * 256);
        if constexpr (ZEROS) dma_load_u16(zbase, from_s[i] + g, to + kAtZ + i * 256);
      }
    } else {
      const int g = 2 * group_of(blk * 4);
#pragma unroll
      for (int i = 0; i < kCopiesS; ++i) {
        dma_load_u16(sbase + g, from_s[i], to + kAtS + i * 256);
        if constexpr (ZEROS) dma_load_u16(zbase + g, from_s[i], to + kAtZ + i * 256);
      }
    }
  };
  int ahead_tile = blockIdx.x, ahead_blk = wave;
  auto copy_next = [&](int stage) {
    copy(stage, ahead_blk);
    ahead_blk += W;
    if (ahead_blk >= blocks) {
      ahead_blk = wave;
      if (ahead_tile + static_cast<int>(gridDim.x) < tiles) {  // (past the last tile: its first blocks once more, not used)
        ahead_tile += gridDim.x;
        aim(ahead_tile);
      }
    }
  };
  if (wave < blocks) {
    aim(ahead_tile);
#pragma unroll
    for (int d = 0; d < D - 1; ++d) copy_next(d);
  }
  const int token = (col >> 2) * RR + ((col & 3) < RR ? (col & 3) : RR - 1);
  const int w_slot = (col * 4 + (kg ^ ((col >> 1) & 3))) * 16;
  int stage = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    float total[FT][RR];
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int r = 0; r < RR; ++r) total[f][r] = 0.0f;
    for (int blk = wave; blk < blocks; blk += W) {
      copy_next(stage == 0 ? D - 1 : stage - 1);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(kCopies * (D - 1)));
      asm volatile("" ::: "memory");
      const uint8_t *from = ring + stage * kStage;
      u32x4 w[FT], x[kX];
#pragma unroll
      for (int f = 0; f < FT; ++f) w[f] = *reinterpret_cast<const u32x4 *>(from + f * 1024 + w_slot);
      const uint8_t *xfrom = from + kAtX + token * (kRowPieces * 16);
#pragma unroll
      for (int i = 0; i < kX; ++i) {
        // 16-bit: piece of step i; int8: of the 16 columns of step i, or (SMALL) 8 of step 2 i and 8 of step 2 i + 1
        if constexpr (is_i8(XT) && SMALL) {
          const uint8_t *lo = xfrom + (((4 * i + kg / 2) ^ (token % kRowPieces)) * 16 + (kg & 1) * 8);
          const uint8_t *hi = xfrom + (((4 * i + 2 + kg / 2) ^ (token % kRowPieces)) * 16 + (kg & 1) * 8);
          const u32x2 a = *reinterpret_cast<const u32x2 *>(lo), b = *reinterpret_cast<const u32x2 *>(hi);
          x[i] = u32x4{a[0], a[1], b[0], b[1]};
        } else {
          const int piece = SMALL ? 4 * i + kg : kX * kg + i;
          x[i] = *reinterpret_cast<const u32x4 *>(xfrom + ((piece ^ (token % kRowPieces)) * 16));
        }
      }
      const int k0 = blk * 128;
      if constexpr (SMALL) {
#pragma unroll
        for (int f = 0; f < FT; ++f) transpose4(w[f]);
      } else if (k0 + 128 > p.K) {
        if (k0 + 32 * kg >= p.K) {
#pragma unroll
          for (int i = 0; i < kX; ++i) x[i] = u32x4{0, 0, 0, 0};
        }
      }
      constexpr int kParts = SMALL ? 4 : 1;  // sums of their own per block
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        if (SMALL && k0 + 32 * part >= p.K) break;
        Acc<XT> acc[FT], high[FT], sums = Acc<XT>{0, 0, 0, 0};  // (high: fp16, of the high nibbles)
#pragma unroll
        for (int f = 0; f < FT; ++f) acc[f] = high[f] = Acc<XT>{0, 0, 0, 0};
        if constexpr (is_i8(XT)) {
          if constexpr (SMALL) {
            const u32x2 xo = order8(u32x2{x[part / 2][2 * (part & 1)], x[part / 2][2 * (part & 1) + 1]});
            const long xa = __builtin_bit_cast(long, xo);
            if constexpr (kSums) sums = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, 0x0101010101010101l, sums, 0, 0, 0);
#pragma unroll
            for (int f = 0; f < FT; ++f) acc[f] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, __builtin_bit_cast(long, widen8(w[f][part])), acc[f], 0, 0, 0);
          } else {
            const int one = 0x01010101;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const u32x2 lo = order8(u32x2{x[s][0], x[s][1]}), hi = order8(u32x2{x[s][2], x[s][3]});
              const i32x4 xa = {static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]), static_cast<int>(hi[1])};
              if constexpr (kSums) sums = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa, i32x4{one, one, one, one}, sums, 0, 0, 0);
#pragma unroll
              for (int f = 0; f < FT; ++f) {
                const u32x2 wl = widen8(w[f][2 * s]), wh = widen8(w[f][2 * s + 1]);
                const i32x4 wb = {static_cast<int>(wl[0]), static_cast<int>(wl[1]), static_cast<int>(wh[0]), static_cast<int>(wh[1])};
                acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa, wb, acc[f], 0, 0, 0);
              }
            }
          }
        } else {
          const uint32_t one = XT == kBF16 ? 0x3F803F80u : 0x3C003C00u;
          constexpr int kSteps = SMALL ? 1 : 4;
          if constexpr (XT == kBF16) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
              const u32x4 xa = x[SMALL ? part : s];
              sums = mfma32<XT>(xa, u32x4{one, one, one, one}, sums);
#pragma unroll
              for (int f = 0; f < FT; ++f) acc[f] = mfma32<XT>(xa, widen_bf16(w[f][SMALL ? part : s]), acc[f]);
            }
          } else if constexpr (SMALL) {  // (a word of low and high nibbles each: the other half of the operand is 0)
            const u32x4 xl = order_f16(x[part], u32x4{0, 0, 0, 0}, 0x05040100u), xh = order_f16(x[part], u32x4{0, 0, 0, 0}, 0x07060302u);
            sums = mfma32<XT>(x[part], u32x4{one, one, one, one}, sums);
#pragma unroll
            for (int f = 0; f < FT; ++f) {
              acc[f] = mfma32<XT>(xl, widen_f16_low(w[f][part], 0), acc[f]);
              high[f] = mfma32<XT>(xh, widen_f16_high(w[f][part], 0), high[f]);
            }
          } else {
#pragma unroll
            for (int s = 0; s < 4; s += 2) {
              const u32x4 xl = order_f16(x[s], x[s + 1], 0x05040100u), xh = order_f16(x[s], x[s + 1], 0x07060302u);
              sums = mfma32<XT>(x[s], u32x4{one, one, one, one}, sums);
              sums = mfma32<XT>(x[s + 1], u32x4{one, one, one, one}, sums);
#pragma unroll
              for (int f = 0; f < FT; ++f) {
                acc[f] = mfma32<XT>(xl, widen_f16_low(w[f][s], w[f][s + 1]), acc[f]);
                high[f] = mfma32<XT>(xh, widen_f16_high(w[f][s], w[f][s + 1]), high[f]);
              }
            }
          }
        }
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          const int at = SMALL ? f * 64 + part * 16 + col : f * 16 + col;  // (four bytes each, the value in the low half)
          constexpr float kUnit = XT == kF16 ? 0x1p-24f : is_i8(XT) ? 16.0f : 1.0f;  // what a code of 1 is in the sums
          const float s = load16(from + kAtS, 2 * at, sbf) * (XT == kF16 ? 0x1p24f : 1.0f);
          float z = XT == kBF16 ? 136.0f : XT == kF16 ? 8 * kUnit : 0.0f;
          if constexpr (ZEROS) z += load16(from + kAtZ, 2 * at, sbf) * kUnit;
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            float d = static_cast<float>(acc[f][r]);
            if constexpr (XT == kF16) d = __builtin_fmaf(0.0625f, high[f][r], d);
            if constexpr (kSums) d = __builtin_fmaf(-z, static_cast<float>(sums[r]), d);
            total[f][r] = __builtin_fmaf(s, d, total[f][r]);
          }
        }
      }
      stage = stage == D - 1 ? 0 : stage + 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wait only; this stage is copied to next: its reads are done)
    }
    // the waves' sums
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int r = 0; r < RR; ++r) red[(wave * kRegs + f * RR + r) * 64 + lane] = total[f][r];
    __syncthreads();
    const int64_t n0 = static_cast<int64_t>(tile) * p.width;
    for (int e = threadIdx.x; e < kRegs * 64; e += 64 * W) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += red[i * kRegs * 64 + e];
      const int l = e & 63, r = (e >> 6) % RR, f = (e >> 6) / RR;
      const int64_t n = n0 + 16 * f + (l & 15), m = (l >> 4) * RR + r;
      if (16 * f + (l & 15) < p.width && n < p.N && m < p.M) {
        if constexpr (is_i8(XT)) v *= p.scale_row[m] * 0.0625f;
        if (p.bias) v += load16(p.bias, n, sbf);
        static_cast<uint16_t *>(p.out)[m * p.N + n] = sbf ? from_f32<true>(v) : from_f32<false>(v);
      }
    }
    __syncthreads();  // (the sums are read: the next tile's may be written)
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (no copy is under way when the workgroup's LDS goes to another)
}

template <int XT, int RR, int FT, int W, int D, bool SMALL, bool ZEROS>
constexpr int decode_lds() {
  constexpr int scales = (SMALL ? FT : (FT + 3) / 4) * 256 * (ZEROS ? 2 : 1);
  return W * D * ((FT + (is_i8(XT) ? (RR + 1) / 2 : RR)) * 1024 + scales) + W * FT * RR * 256;
}

template <int XT, int RR, int FT, int W, int D, bool SMALL, bool ZEROS>
int launch_decode(const GroupArgs &p, hipStream_t st) {
  constexpr int smem = decode_lds<XT, RR, FT, W, D, SMALL, ZEROS>();
  static_assert(smem <= kLdsBytes, "");
  auto kern = group4_decode_kernel<XT, RR, FT, W, D, SMALL, ZEROS>;
  if (int rc = prepare(kern, smem)) return rc;
  // as many workgroups as run at a time, two of eight waves per CU at most (1 x 8192 -> 28672 fp16: one 26.8 us, two 26.4, three 26.5; in one
  // matrix tile each two 29.8, three 30.8)
  const int per_cu = kLdsBytes / smem < 16 / W ? kLdsBytes / smem : 16 / W;
  const int64_t tiles = (p.N + p.width - 1) / p.width, slots = static_cast<int64_t>(num_cus()) * per_cu;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tiles < slots ? tiles : slots)), dim3(64 * W), smem, st, p);
  return check_launch();
}

// More than 16 token rows.  WM x WN waves side by side, each with RM x RN result tiles of 16 x 16, on a step of 128 columns; WK such sets of
// waves take 128 columns each of a step of 128 * WK and add their sums at the end.  All operands come to LDS by direct copies, D - 1
// steps ahead, one barrier per step.  PARTS sums of their own per 128 columns: 1 where groups are multiples of 128, 2 of 64, 4.
template <int XT, int RM, int RN, int WM, int WN, int WK, int D, int PARTS, bool ZEROS>
struct TileShape {
  static constexpr int kW = WM * WN * WK, kBM = 16 * RM * WM, kBN = 16 * RN * WN;
  static constexpr int kRowBytes = is_i8(XT) ? 128 : 256;
  static constexpr int kX = WK * kBM * kRowBytes / 1024, kWt = WK * kBN / 16;     // copies of 1 KB per step
  static constexpr int kS = WK * (PARTS == 1 ? (kBN + 63) / 64 : kBN / 16);        // copies of 64 scales
  static constexpr int kAtW = kX * 1024, kAtS = kAtW + kWt * 1024, kAtZ = kAtS + kS * 256, kStage = kAtS + kS * 256 * (ZEROS ? 2 : 1);
  static constexpr int kMyX = (kX + kW - 1) / kW, kMyW = (kWt + kW - 1) / kW, kMyS = (kS + kW - 1) / kW;
  static constexpr int kCopies = kMyX + kMyW + kMyS * (ZEROS ? 2 : 1);
  static constexpr int kReduce = WK > 1 ? WM * WN * WK * RM * RN * 1024 : 0;
  static constexpr bool kSums = ZEROS || XT == kBF16;
  // Sums of the activations: of eight row tiles the waves side by side make one each and take the others' a step later (us at 2048 x 4096 ->
  // 11008, each wave all of them and this: bf16 327, 218, fp16 with zeros 552, 248, int8 with zeros 186, 183); of
  // fewer each wave makes all that it needs (so and shared: 300 x 4544 -> 4541 fp16, groups of 64 with zeros 41.1, 44.1; 64 x 4096 -> 11008
  // bf16 with zeros, K split 21.9, 22.1).
  static constexpr bool kShared = kSums && RM >= 8, kOwnSums = kSums && !kShared;
  // Groups of 32 and the like: what the sums are multiplied by is a matrix product of its own, of 16 columns and 16 rows over the block's four
  // units of 32 columns, in fp32 (300 x 4544 -> 4541, groups of 32 with zeros: int8 56 us, so 46, fp16 49.6, 45.0; groups of 64 lost 1 - 7 %).
  static constexpr bool kUnits = kOwnSums && PARTS == 4;
  static constexpr int kAtSums = D * kStage, kRings = kAtSums + (kShared ? 2 * WK * PARTS * kBM * 4 : 0);  // of two steps
  static constexpr int kLds = kRings > kReduce ? kRings : kReduce;
  static_assert(!kShared || WN >= RM, "");
};

template <int XT, int RM, int RN, int WM, int WN, int WK, int D, int PARTS, bool ZEROS>
__global__ __launch_bounds__(64 * WM * WN * WK) void group4_tile_kernel(GroupArgs p) {
  using S = TileShape<XT, RM, RN, WM, WN, WK, D, PARTS, ZEROS>;
  constexpr bool kShared = S::kShared, kOwnSums = S::kOwnSums, kUnits = S::kUnits;
  constexpr bool kTurn = PARTS > 1;  // matrix step s: columns 32 s .. of the block; else columns 8 s .. of each lane row's 32
  constexpr int kRowPieces = S::kRowBytes / 16, kSize = is_i8(XT) ? 1 : 2;
  extern __shared__ float red[];
  uint8_t *lds = reinterpret_cast<uint8_t *>(red);
  const uint32_t lds_at = lds_address(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);
  constexpr bool sbf = is_bf16(XT);
  const int blocks = static_cast<int>((p.K + 127) >> 7), all_steps = (blocks + WK - 1) / WK;
  // Workgroups go to the eight dies in turn: each die gets a run of tiles, in bands of four row tiles, column by column, so that those
  // that run on a die at a time share both their rows and their weights in its L2 (2048 x 8192 -> 8192 fp16, 128x256 tiles: 278 us row
  // tiles first, 274 in bands).  A tile whose K is split is `splits` workgroups, one after the other.
  constexpr int kBand = 4;
  const int m_tiles = static_cast<int>((p.M + S::kBM - 1) / S::kBM), n_tiles = static_cast<int>((p.N + S::kBN - 1) / S::kBN);
  const int all = static_cast<int>(gridDim.x), die = blockIdx.x & 7, run = all >> 3, rest = all & 7;
  const int unit = die * run + (die < rest ? die : rest) + static_cast<int>(blockIdx.x >> 3), tile = unit / p.splits, split = unit % p.splits;
  const int band = tile / (kBand * n_tiles), in_band = tile - band * kBand * n_tiles;
  const int high = m_tiles - band * kBand < kBand ? m_tiles - band * kBand : kBand;
  const int64_t m0 = static_cast<int64_t>(band * kBand + in_band % high) * S::kBM, n0 = static_cast<int64_t>(in_band / high) * S::kBN;
  const int first = static_cast<int>(static_cast<int64_t>(all_steps) * split / p.splits);
  const int steps = static_cast<int>(static_cast<int64_t>(all_steps) * (split + 1) / p.splits);

  const uint8_t *xbase = static_cast<const uint8_t *>(p.x) + m0 * p.K * kSize, *wbase = p.w + n0 * (p.K / 2);
  const uint8_t *sbase = static_cast<const uint8_t *>(p.scales) + n0 * p.groups * 2, *zbase = static_cast<const uint8_t *>(p.zeros) + n0 * p.groups * 2;
  const int64_t left_m = p.M - 1 - m0, left_n = p.N - 1 - n0;
  const int last_w = static_cast<int>(p.K / 32) - 1, last_x = static_cast<int>(p.K * kSize / 16) - 1;
  // Where a row's 16-byte pieces lie in LDS: at the row's number exclusive-or the piece's; in wide tiles with the piece's two fields (lane row,
  // matrix step) changed over where a lane reads neighbouring pieces in its steps.  A 16-byte read goes by lanes 0 .. 3, 12 .. 15, 20 .. 27 and
  // so on, which are at different banks then (else half as many cycles again per read: 2048 x 4096 -> 11008 int8 144.5 us, so 140.6, fp16 206.9,
  // 204.8, bf16 221.7, 216.8).  Copies in that order cost more than the banks in small tiles (64 x 8192 -> 8192 fp16 33.5 us, 34.1).
  constexpr bool kSwap = !kTurn && RM >= 8;
  auto place_of = [](int piece) { return !kSwap ? piece : is_i8(XT) ? (piece & 1) * 4 + (piece >> 1) : (piece & 3) * 4 + (piece >> 2); };
  auto piece_at = [](int place) { return !kSwap ? place : is_i8(XT) ? (place & 3) * 2 + (place >> 2) : (place & 3) * 4 + (place >> 2); };
  // this wave's copies: which of the step's, the row's offset and the piece of the step that this lane takes
  uint32_t x_row[S::kMyX], w_row[S::kMyW], s_row[S::kMyS];
  int x_piece[S::kMyX], w_piece[S::kMyW], s_unit[S::kMyS];
#pragma unroll
  for (int i = 0; i < S::kMyX; ++i) {
    const int c = (wave + i * S::kW) % S::kX, part = c / (S::kX / WK), row = (c % (S::kX / WK)) * (64 / kRowPieces) + lane / kRowPieces;
    x_piece[i] = part * kRowPieces + piece_at((lane % kRowPieces) ^ (row % kRowPieces));
    x_row[i] = static_cast<uint32_t>((row < left_m ? row : left_m) * p.K * kSize);
  }
#pragma unroll
  for (int i = 0; i < S::kMyW; ++i) {
    const int c = (wave + i * S::kW) % S::kWt, part = c / (S::kWt / WK), row = (c % (S::kWt / WK)) * 16 + (lane >> 2);
    w_piece[i] = part * 4 + ((lane & 3) ^ ((lane >> 3) & 3));
    w_row[i] = static_cast<uint32_t>((row < left_n ? row : left_n) * (p.K / 2));
  }
#pragma unroll
  for (int i = 0; i < S::kMyS; ++i) {
    const int c = (wave + i * S::kW) % S::kS, part = c / (S::kS / WK);
    int row = kTurn ? (c % (S::kS / WK)) * 16 + col : (c % (S::kS / WK)) * 64 + lane;
    row = row < S::kBN ? row : S::kBN - 1;
    s_unit[i] = part * 4 + (kTurn ? kg : 0);
    s_row[i] = static_cast<uint32_t>((row < left_n ? row : left_n) * p.groups * 2);
  }
  auto group_of = [&](int unit) { return static_cast<uint32_t>((static_cast<uint64_t>(static_cast<uint32_t>(unit)) * p.group_factor) >> 31); };
  // Copies `from` .. `until` - 1 of this wave's S::kCopies of a step.
  auto copy = [&](int step, int from, int until) {
    const uint32_t to = lds_at + step % D * S::kStage;
    const int xp0 = step * (WK * kRowPieces), wp0 = step * (WK * 4);
    if ((static_cast<int64_t>(step) + 1) * (128 * WK) <= p.K) {  // (what goes on along K in scalar registers)
      const uint8_t *xfrom = xbase + xp0 * 16, *wfrom = wbase + wp0 * 16;
#pragma unroll
      for (int i = 0; i < S::kMyX; ++i)
        if (i >= from && i < until) dma_load16(xfrom, x_row[i] + x_piece[i] * 16, to + (wave + i * S::kW) % S::kX * 1024);
#pragma unroll
      for (int i = 0; i < S::kMyW; ++i)
        if (S::kMyX + i >= from && S::kMyX + i < until) dma_load16(wfrom, w_row[i] + w_piece[i] * 16, to + S::kAtW + (wave + i * S::kW) % S::kWt * 1024);
    } else {  // pieces past the end of a row come from its last one
#pragma unroll
      for (int i = 0; i < S::kMyX; ++i) {
        const int piece = xp0 + x_piece[i];
        if (i >= from && i < until)
          dma_load16(xbase, x_row[i] + static_cast<uint32_t>(piece < last_x ? piece : last_x) * 16, to + (wave + i * S::kW) % S::kX * 1024);
      }
#pragma unroll
      for (int i = 0; i < S::kMyW; ++i) {
        const int piece = wp0 + w_piece[i];
        if (S::kMyX + i >= from && S::kMyX + i < until)
          dma_load16(wbase, w_row[i] + static_cast<uint32_t>(piece < last_w ? piece : last_w) * 16, to + S::kAtW + (wave + i * S::kW) % S::kWt * 1024);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kMyS; ++i) {
      const int nth = S::kMyX + S::kMyW + (ZEROS ? 2 * i : i), c = (wave + i * S::kW) % S::kS;
      if (nth + (ZEROS ? 1 : 0) < from || nth >= until) continue;
      const int unit = wp0 + (kTurn ? s_unit[i] : c / (S::kS / WK) * 4);
      const uint32_t g = 2 * group_of(unit < last_w ? unit : last_w);
      const uint8_t *sfrom = kTurn ? sbase : sbase + g, *zfrom = kTurn ? zbase : zbase + g;
      const uint32_t at = kTurn ? s_row[i] + g : s_row[i];
      if (nth >= from) dma_load_u16(sfrom, at, to + S::kAtS + c * 256);
      if (ZEROS && nth + 1 >= from && nth + 1 < until) dma_load_u16(zfrom, at, to + S::kAtZ + c * 256);
    }
  };
  f32x4 total[RM][RN];
#pragma unroll
  for (int t = 0; t < RM; ++t)
#pragma unroll
    for (int f = 0; f < RN; ++f) total[t][f] = f32x4{0, 0, 0, 0};
  const int w_slot = (col * 4 + (kg ^ ((col >> 1) & 3))) * 16;
  // activations of row tile t: the 16 bytes of matrix step s (16 bits: 8 columns; int8: 16), or (int8, kTurn) the 8 bytes
  auto x_row_at = [&](const uint8_t *from, int t) { return from + (wk * S::kBM + wm * 16 * RM + 16 * t + col) * S::kRowBytes; };
  auto x_piece_of = [&](const uint8_t *from, int t, int s) {
    const int piece = is_i8(XT) ? 2 * kg + s : kTurn ? 4 * s + kg : 4 * kg + s;
    return *reinterpret_cast<const u32x4 *>(x_row_at(from, t) + ((place_of(piece) ^ (col % kRowPieces)) * 16));
  };
  auto x_half = [&](const uint8_t *from, int t, int s) {
    return *reinterpret_cast<const u32x2 *>(x_row_at(from, t) + (((2 * s + kg / 2) ^ (col % kRowPieces)) * 16 + (kg & 1) * 8));
  };
  // operands of this step are in LDS, for every wave (the copies of D - 2 later steps may be under way)
  auto arrive = [&](int step) {
    if (D > 2 && step + D - 2 < steps) __builtin_amdgcn_s_waitcnt(vmcnt_imm(S::kCopies * (D - 2)));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    if (!kTurn && (static_cast<int64_t>(step) + 1) * (128 * WK) > p.K) {  // pieces past the end of K: zeros
#pragma unroll
      for (int i = 0; i < S::kMyX; ++i) {
        const int c = (wave + i * S::kW) % S::kX;
        if (step * (WK * kRowPieces) + x_piece[i] > last_x)
          *reinterpret_cast<u32x4 *>(lds + step % D * S::kStage + c * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (a wait and a barrier: what was read of LDS is read)
  };
  // Sums of the activations of a part (columns of one group), by a matrix of ones: what the zeros and the offset of widened bf16 codes are
  // multiplied by.
  constexpr float kOffset = XT == kBF16 ? 136.0f : 0.0f, kUnit = is_i8(XT) ? 16.0f : 1.0f;
  float *const sums = reinterpret_cast<float *>(lds + S::kAtSums);
  float less[kShared ? PARTS : 1][RN][4];  // -scale * (offset + zero) of the step before
  auto sums_of = [&](int step, int part) { return sums + (((step & 1) * WK + wk) * PARTS + part) * S::kBM + wm * 16 * RM + col; };
  auto add_ones = [&](auto x, Acc<XT> v) {
    if constexpr (sizeof(x) == 8) return __builtin_amdgcn_mfma_i32_16x16x32_i8(0x0101010101010101l, __builtin_bit_cast(long, x), v, 0, 0, 0);
    else if constexpr (is_i8(XT)) return __builtin_amdgcn_mfma_i32_16x16x64_i8(i32x4{0x01010101, 0x01010101, 0x01010101, 0x01010101}, __builtin_bit_cast(i32x4, x), v, 0, 0, 0);
    else return mfma32<XT>(XT == kBF16 ? u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u} : u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}, __builtin_bit_cast(u32x4, x), v);
  };
  auto sum = [&](const uint8_t *from, int step, int part, int64_t k0) {
    const int own = wn % RM;
    Acc<XT> v = Acc<XT>{0, 0, 0, 0};
    constexpr int kSteps = is_i8(XT) && !kTurn ? 2 : 4;
#pragma unroll
    for (int s = part * kSteps / PARTS; s < (part + 1) * kSteps / PARTS; ++s) {
      if (PARTS == 2 && k0 + 32 * s >= p.K) break;
      if constexpr (is_i8(XT) && kTurn) v = add_ones(x_half(from, own, s), v);
      else v = add_ones(x_piece_of(from, own, s), v);
    }
    if (kg == 0) sums_of(step, part)[16 * own] = static_cast<float>(v[0]);
  };
  auto correct = [&](int step) {
    const int64_t k0 = (static_cast<int64_t>(step) * WK + wk) * 128;
    if (WK > 1 && k0 >= p.K) return;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      if (kTurn && k0 + 128 / PARTS * part >= p.K) break;
#pragma unroll
      for (int t = 0; t < RM; ++t) {
        const float v = sums_of(step, part)[16 * t];
#pragma unroll
        for (int f = 0; f < RN; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) total[t][f][r] = __builtin_fmaf(less[part][f][r], v, total[t][f][r]);
      }
    }
  };
  // The copies of the step D - 1 on: in front of the products, or dealt to the places between them, where all of them first hold a wave longer
  // than they are late then (us, first and dealt: 300 x 4544 -> 4541 fp16, groups of 64 with zeros 46.6, 41.4, int8, groups of 32 with zeros 52.4,
  // 46.1; 2048 x 4096 -> 11008 fp16 206.7, 204.6, bf16 222.4, 217.2, but int8 138.7, 140.9; 64 x 8192 -> 8192 fp16 33.6, 41.9, K split 19.5, 20.8).
  constexpr bool kDealt = PARTS > 1 || RM >= 8;
  constexpr int kSlots = (is_i8(XT) && !kTurn ? 2 : 4) * RN;
  auto multiply = [&](int step) {
    const int64_t k0 = (static_cast<int64_t>(step) * WK + wk) * 128;
    const bool more = step + D - 1 < steps;
    auto slot = [&](int nth) {
      if (kDealt && more) copy(step + D - 1, nth * S::kCopies / kSlots, (nth + 1) * S::kCopies / kSlots);
    };
    if (!kDealt && more) copy(step + D - 1, 0, S::kCopies);
    if (WK > 1 && k0 >= p.K) return;  // (in the last step, which has no copies behind it)
    const uint8_t *from = lds + step % D * S::kStage, *from_s = from + S::kAtS;
    u32x4 w[RN];
#pragma unroll
    for (int f = 0; f < RN; ++f) {
      w[f] = *reinterpret_cast<const u32x4 *>(from + S::kAtW + (wk * (S::kBN / 16) + wn * RN + f) * 1024 + w_slot);
      if constexpr (kTurn) transpose4(w[f]);
    }
    Acc<XT> units[kUnits ? RM : 1];  // (kUnits: first value, of the lane row's 32 columns)
    if constexpr (kUnits) {
#pragma unroll
      for (int t = 0; t < RM; ++t) units[t] = Acc<XT>{0, 0, 0, 0};
    }
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        if (kTurn && k0 + 128 / PARTS * part >= p.K) break;  // (the last step, which has no copies behind it)
        if constexpr (kShared) sum(from, step, part, k0);
        Acc<XT> acc[RM][RN], own[kOwnSums && !kUnits ? RM : 1];
        __builtin_amdgcn_s_setprio(1);  // a wave among its products before one that widens codes for its next
#pragma unroll
        for (int t = 0; t < RM; ++t) {
          if constexpr (kOwnSums && !kUnits) own[t] = Acc<XT>{0, 0, 0, 0};
#pragma unroll
          for (int f = 0; f < RN; ++f) acc[t][f] = Acc<XT>{0, 0, 0, 0};
        }
        if constexpr (is_i8(XT) && kTurn) {
#pragma unroll
          for (int s = part * 4 / PARTS; s < (part + 1) * 4 / PARTS; ++s) {
            if (PARTS == 2 && k0 + 32 * s >= p.K) break;
            long xa[RM];
#pragma unroll
            for (int t = 0; t < RM; ++t) {
              xa[t] = __builtin_bit_cast(long, x_half(from, t, s));
              if constexpr (kUnits) {
                const Acc<XT> v = add_ones(xa[t], Acc<XT>{0, 0, 0, 0});
                units[t][0] = kg == s ? v[0] : units[t][0];
              } else if constexpr (kOwnSums) {
                own[t] = add_ones(xa[t], own[t]);
              }
            }
#pragma unroll
            for (int f = 0; f < RN; ++f) {
              const long wb = __builtin_bit_cast(long, widen8_in_order(w[f][s]));
#pragma unroll
              for (int t = 0; t < RM; ++t) acc[t][f] = __builtin_amdgcn_mfma_i32_16x16x32_i8(wb, xa[t], acc[t][f], 0, 0, 0);
              slot(s * RN + f);
            }
          }
        } else if constexpr (is_i8(XT)) {
          static_assert(!kUnits, "");  // (parts of 32 columns: kTurn)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            i32x4 xa[RM];
#pragma unroll
            for (int t = 0; t < RM; ++t) {
              xa[t] = __builtin_bit_cast(i32x4, x_piece_of(from, t, s));
              if constexpr (kOwnSums) own[t] = add_ones(xa[t], own[t]);
            }
#pragma unroll
            for (int f = 0; f < RN; ++f) {
              const u32x2 wl = widen8_in_order(w[f][2 * s]), wh = widen8_in_order(w[f][2 * s + 1]);
              const i32x4 wb = {static_cast<int>(wl[0]), static_cast<int>(wl[1]), static_cast<int>(wh[0]), static_cast<int>(wh[1])};
#pragma unroll
              for (int t = 0; t < RM; ++t) acc[t][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wb, xa[t], acc[t][f], 0, 0, 0);
              slot(s * RN + f);
            }
          }
        } else {
#pragma unroll
          for (int s = part * 4 / PARTS; s < (part + 1) * 4 / PARTS; ++s) {
            if (PARTS == 2 && k0 + 32 * s >= p.K) break;
            u32x4 xa[RM];
#pragma unroll
            for (int t = 0; t < RM; ++t) {
              xa[t] = x_piece_of(from, t, s);
              if constexpr (kUnits) {
                const Acc<XT> v = add_ones(xa[t], Acc<XT>{0, 0, 0, 0});
                units[t][0] = kg == s ? v[0] : units[t][0];
              } else if constexpr (kOwnSums) {
                own[t] = add_ones(xa[t], own[t]);
              }
            }
#pragma unroll
            for (int f = 0; f < RN; ++f) {
              const u32x4 wb = XT == kBF16 ? widen_bf16(w[f][s]) : widen_f16(w[f][s]);
#pragma unroll
              for (int t = 0; t < RM; ++t) acc[t][f] = mfma32<XT>(wb, xa[t], acc[t][f]);
              slot(s * RN + f);
            }
          }
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int f = 0; f < RN; ++f) {
          // (four bytes each, the value in the low half; kTurn: 16 columns at the block's four units of 32)
          const int at = (kTurn ? (wk * (S::kBN / 16) + wn * RN + f) * 64 + part * (64 / PARTS) : wk * (S::kS / WK) * 64 + (wn * RN + f) * 16) + 4 * kg;
          const u32x4 sw = *reinterpret_cast<const u32x4 *>(from_s + 4 * at);
          float s[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) s[r] = from16(sw[r], sbf);
          float z[4] = {kOffset, kOffset, kOffset, kOffset};
          if constexpr (ZEROS && !kUnits) {
            const u32x4 zw = *reinterpret_cast<const u32x4 *>(from_s + (S::kAtZ - S::kAtS) + 4 * at);
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] += kUnit * from16(zw[r], sbf);
          }
          if constexpr (kShared) {
#pragma unroll
            for (int r = 0; r < 4; ++r) less[part][f][r] = -s[r] * z[r];
          }
#pragma unroll
          for (int t = 0; t < RM; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float d = static_cast<float>(acc[t][f][r]);
              if constexpr (kOwnSums && !kUnits) d = __builtin_fmaf(-z[r], static_cast<float>(own[t][0]), d);
              total[t][f][r] = __builtin_fmaf(s[r], d, total[t][f][r]);
            }
        }
      }
    if constexpr (kUnits) {
#pragma unroll
      for (int f = 0; f < RN; ++f) {
        const int at = (wk * (S::kBN / 16) + wn * RN + f) * 64 + lane;
        float z = kOffset;
        if constexpr (ZEROS) z += kUnit * load16(from_s + (S::kAtZ - S::kAtS), 2 * at, sbf);
        const float less_of = -load16(from_s, 2 * at, sbf) * z;
#pragma unroll
        for (int t = 0; t < RM; ++t) total[t][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(less_of, static_cast<float>(units[t][0]), total[t][f], 0, 0, 0);
      }
    }
  };
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (first + d < steps) copy(first + d, 0, S::kCopies);
  for (int step = first; step < steps; ++step) {
    arrive(step);
    if (kShared && step > first) correct(step - 1);
    multiply(step);
  }
  if constexpr (kShared) {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (a wait and a barrier: the last step's sums are there)
    correct(steps - 1);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wait only)
  typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(2)));  // four columns of a row in one store, at any of them
  float row_scale[RM];
#pragma unroll
  for (int t = 0; t < RM; ++t) {
    const int64_t m = m0 + wm * 16 * RM + 16 * t + col;
    row_scale[t] = is_i8(XT) ? p.scale_row[m < p.M ? m : p.M - 1] * 0.0625f : 1.0f;
  }
  auto store = [&](int t, int f, f32x4 v) {
    const int64_t m = m0 + wm * 16 * RM + 16 * t + col, n = n0 + wn * 16 * RN + 16 * f + 4 * kg;
    if (m >= p.M || n >= p.N) return;
    if (p.splits > 1) {
      *reinterpret_cast<f32x4 *>(p.partial + (split * p.M + m) * ((p.N + 3) & ~int64_t{3}) + n) = v;
      return;
    }
    uint32_t b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (is_i8(XT)) v[r] *= row_scale[t];
      if (p.bias) v[r] += load16(p.bias, n + r < p.N ? n + r : p.N - 1, sbf);
      b[r] = sbf ? from_f32<true>(v[r]) : from_f32<false>(v[r]);
    }
    uint16_t *to = static_cast<uint16_t *>(p.out) + m * p.N + n;
    if (n + 3 < p.N) {
      *reinterpret_cast<loose2 *>(to) = loose2{b[0] | b[1] << 16, b[2] | b[3] << 16};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.N) to[r] = static_cast<uint16_t>(b[r]);
    }
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int t = 0; t < RM; ++t)
#pragma unroll
      for (int f = 0; f < RN; ++f) store(t, f, total[t][f]);
  } else {
    __syncthreads();  // (the last step's operands are read)
    f32x4 *sums = reinterpret_cast<f32x4 *>(red) + (wm * WN + wn) * (WK * RM * RN * 64);
#pragma unroll
    for (int t = 0; t < RM; ++t)
#pragma unroll
      for (int f = 0; f < RN; ++f) sums[(wk * RM * RN + t * RN + f) * 64 + lane] = total[t][f];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < RM * RN; ++e) {
      if (e % WK != wk) continue;
      f32x4 v = sums[e * 64 + lane];
#pragma unroll
      for (int i = 1; i < WK; ++i) v += sums[(i * RM * RN + e) * 64 + lane];
      store(e / RN, e % RN, v);
    }
  }
}

// the sums of a split K in the order of the splits, then what the tiles do with a sum
template <int XT>
__global__ __launch_bounds__(256) void group4_join_kernel(GroupArgs p) {
  const int64_t pitch = (p.N + 3) & ~int64_t{3}, quads = pitch / 4, at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= p.M * quads) return;
  const int64_t m = at / quads, n = at % quads * 4;
  const float *from = p.partial + m * pitch + n;
  f32x4 v = *reinterpret_cast<const f32x4 *>(from);
  for (int i = 1; i < p.splits; ++i) v += *reinterpret_cast<const f32x4 *>(from + i * p.M * pitch);
  const float row = is_i8(XT) ? p.scale_row[m] * 0.0625f : 1.0f;
  for (int r = 0; r < 4 && n + r < p.N; ++r) {
    float y = is_i8(XT) ? v[r] * row : v[r];
    if (p.bias) y += load16(p.bias, n + r, is_bf16(XT));
    static_cast<uint16_t *>(p.out)[m * p.N + n + r] = from_f32<is_bf16(XT)>(y);
  }
}

// (2^31 threads per launch: rows beyond are further launches, which follow each other and share the memory of the parts' sums)
template <int XT, int RM, int RN, int WM, int WN, int WK, int D, int PARTS, bool ZEROS>
int launch_tile(const GroupArgs &p, hipStream_t st) {
  using S = TileShape<XT, RM, RN, WM, WN, WK, D, PARTS, ZEROS>;
  static_assert(S::kLds <= kLdsBytes, "");
  auto kern = group4_tile_kernel<XT, RM, RN, WM, WN, WK, D, PARTS, ZEROS>;
  if (int rc = prepare(kern, S::kLds)) return rc;
  const int64_t across = (p.N + S::kBN - 1) / S::kBN * p.splits, most = INT32_MAX / (S::kW * 64) / across * S::kBM;
  if (most == 0) return QUIK_ERR_RANGE;
  for (int64_t m = 0; m < p.M; m += most) {
    GroupArgs q = p;
    q.M = p.M - m < most ? p.M - m : most;
    q.x = static_cast<const uint8_t *>(p.x) + m * p.K * (is_i8(XT) ? 1 : 2);
    if (is_i8(XT)) q.scale_row = p.scale_row + m;
    q.out = static_cast<uint16_t *>(p.out) + m * p.N;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((q.M + S::kBM - 1) / S::kBM * across)), dim3(64 * S::kW), S::kLds, st, q);
    if (int rc = check_launch()) return rc;
    if (p.splits > 1) {
      hipLaunchKernelGGL((group4_join_kernel<XT>), dim3(static_cast<unsigned>((q.M * ((p.N + 3) / 4) + 255) / 256)), dim3(256), 0, st, q);
      if (int rc = check_launch()) return rc;
    }
  }
  return QUIK_OK;
}

// Columns per workgroup for up to 16 rows: with FT matrix tiles side by side, the rounds that all CUs need, and the columns of a round dealt
// to them evenly.  A round's time goes as the columns that are read, as the matrix tiles that are computed (a quarter of it; half where sums of
// the activations come in), and as the activations' share (of 16 columns: 0.1 for one to four rows, 0.3 up to eight, 1 up to sixteen of 16
// bits, half of it for int8).  us with the rule's matrix tiles and the next best, in turn on one card: 1 x 4096 -> 4096 4.4 (1), 5.1 (2); 1 x 8192
// -> 28672 26.6 (2), 30.0 (1), bf16 with zeros 30.9 (1), 32.1 (2); 1 x 4096 -> 22016 int8 8.7 (2), 10.2 (1); 1 x 5120 -> 13824 9.2 (2), 10.9 (1);
// 16 x 13824 -> 5120 int8 8.6 (2), 11.5 (1); 16 x 5120 -> 13824 11.5 (4), 11.3 (2), 15.3 (1).
struct Columns {
  int matrix_tiles, width;
};
Columns deal_columns(int64_t N, int RR, bool i8, bool bf16, bool zeros) {
  const double share = (RR == 1 ? 0.1 : RR == 2 ? 0.3 : 1.0) * (i8 ? 0.5 : 1.0), products = zeros || (bf16 && !i8) ? 0.5 : 0.25;
  const int64_t cus = num_cus();
  auto width = [&](int ft) {
    const int64_t most = 16 * ft, rounds = ((N + most - 1) / most + cus - 1) / cus;
    return static_cast<int>((N + rounds * cus - 1) / (rounds * cus));
  };
  auto cost = [&](int ft) {
    const int w = width(ft);
    const int64_t rounds = ((N + w - 1) / w + cus - 1) / cus;
    return static_cast<double>(rounds) * ((1.0 - products) * w / 16.0 + products * ft + share);
  };
  const double c1 = cost(1), c2 = cost(2), c4 = RR == 4 ? cost(4) : 1e30;
  const int ft = c4 < c2 && c4 < c1 ? 4 : c2 < c1 ? 2 : 1;
  return Columns{ft, width(ft)};
}

template <int XT, int RR, bool SMALL, bool ZEROS>
int by_columns(GroupArgs p, hipStream_t st) {
  const Columns c = deal_columns(p.N, RR, is_i8(XT), is_bf16(XT), ZEROS);
  p.width = c.width;
  if constexpr (RR == 4)
    if (c.matrix_tiles == 4) return launch_decode<XT, RR, 4, 4, 2, SMALL, ZEROS>(p, st);
  if (c.matrix_tiles == 2) return launch_decode<XT, RR, 2, 8, 2, SMALL, ZEROS>(p, st);
  return launch_decode<XT, RR, 1, 8, 2, SMALL, ZEROS>(p, st);
}

// Tiles of more than 16 rows: rows, columns, columns of K per step, and the time of a step on a CU in us for fp16, bf16 and int8
// activations (measured with groups of 128 and no zeros; others take longer in all of them alike).
struct TilePlan {
  int rows, cols, depth;
  double step[3], round;  // round: what first copies and stores of a workgroup take, where one runs per CU
};
constexpr TilePlan kPlans[3] = {{32, 128, 256, {0.94, 1.37, 0.72}, 0}, {64, 128, 256, {1.35, 1.9, 0.9}, 0}, {128, 256, 128, {1.9, 2.1, 1.2}, 6}};

struct Choice {
  int plan, splits;
};
// The cheapest tiles and K split: rounds of the busiest CU, 4 us around them, and for a split the second launch (3 us) and its sums, written
// and read.  us, as the rule has it and measured: 64 x 13824 -> 5120 int8, 64 rows, K in 6: 18.2, 17.7 (not split: 51.7); 64 x 8192 -> 8192
// fp16, K in 4: 21.2, 19.6 (44); 128 x 13824 -> 5120 int8, K in 3: 26.3, 25.1 (51); 2048 x 4096 -> 11008 int8, 128 rows: 137, 140 (64
// rows: 146.5).
Choice choose(int64_t M, int64_t N, int64_t K, int acts, bool may_split) {
  Choice best{1, 1};
  double least = 1e30;
  const int64_t cus = num_cus();
  for (int i = 0; i < 3; ++i) {
    const TilePlan &t = kPlans[i];
    const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols), steps = (K + t.depth - 1) / t.depth;
    for (int s = 1; s <= (may_split ? 16 : 1) && s <= steps; ++s) {
      const int64_t rounds = (tiles * s + cus - 1) / cus, deep = (steps + s - 1) / s;
      const double us = static_cast<double>(rounds) * (static_cast<double>(deep) * t.step[acts] + t.round) + 4.0 +
                        (s > 1 ? 3.0 + static_cast<double>(s) * static_cast<double>(M) * static_cast<double>(N) * 8e-6 / 5.0 : 0.0);
      if (us < least) {
        least = us;
        best = Choice{i, s};
      }
    }
  }
  return best;
}
int acts_of(int x_bits, int dtype) { return x_bits == 8 ? 2 : dtype == QUIK_BF16 ? 1 : 0; }
int64_t partial_bytes(int64_t M, int64_t N, int splits) { return splits > 1 ? splits * M * ((N + 3) / 4 * 4) * 4 : 0; }
Choice choose_within(int64_t M, int64_t N, int64_t K, int acts, int64_t workspace_bytes) {
  const Choice c = choose(M, N, K, acts, true);
  return workspace_bytes < partial_bytes(M, N, c.splits) ? choose(M, N, K, acts, false) : c;
}

template <int XT, int PARTS, bool ZEROS>
int by_rows(const GroupArgs &p, int64_t workspace_bytes, hipStream_t st) {
  if (p.M <= 4) return by_columns<XT, 1, (PARTS > 1), ZEROS>(p, st);
  if (p.M <= 8) return by_columns<XT, 2, (PARTS > 1), ZEROS>(p, st);
  if (p.M <= 16) return by_columns<XT, 4, (PARTS > 1), ZEROS>(p, st);
  GroupArgs q = p;
  const Choice c = choose_within(p.M, p.N, p.K, is_i8(XT) ? 2 : XT == kBF16 ? 1 : 0, p.partial ? workspace_bytes : 0);
  q.splits = c.splits;
  if (c.plan == 0) return launch_tile<XT, 2, 2, 1, 4, 2, 2, PARTS, ZEROS>(q, st);
  if (c.plan == 1) return launch_tile<XT, 4, 2, 1, 4, 2, 2, PARTS, ZEROS>(q, st);
  constexpr int ahead = TileShape<XT, 8, 2, 1, 8, 1, 3, PARTS, ZEROS>::kLds <= kLdsBytes ? 3 : 2;
  return launch_tile<XT, 8, 2, 1, 8, 1, ahead, PARTS, ZEROS>(q, st);
}

template <int XT>
int by_groups(const GroupArgs &p, int64_t bytes, hipStream_t st) {
  const int parts = p.groups == 1 || p.G % 128 == 0 ? 1 : p.G % 64 == 0 ? 2 : 4;
  if (p.zeros) return parts == 1 ? by_rows<XT, 1, true>(p, bytes, st) : parts == 2 ? by_rows<XT, 2, true>(p, bytes, st) : by_rows<XT, 4, true>(p, bytes, st);
  return parts == 1 ? by_rows<XT, 1, false>(p, bytes, st) : parts == 2 ? by_rows<XT, 2, false>(p, bytes, st) : by_rows<XT, 4, false>(p, bytes, st);
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int64_t quik_int4_group_matmul_workspace_bytes(int x_bits, int dtype, int64_t M, int64_t N, int64_t K) {
  if (M <= 16 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > 1 << 20) return 0;
  return partial_bytes(M, N, choose(M, N, K, acts_of(x_bits, dtype), true).splits);
}

extern "C" int quik_int4_group_matmul_tile(int x_bits, int dtype, int zeros, int64_t M, int64_t N, int64_t K, int64_t workspace_bytes) {
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > 1 << 20) return 0;
  if (M > 16) {
    const TilePlan &t = kPlans[choose_within(M, N, K, acts_of(x_bits, dtype), workspace_bytes).plan];
    return t.rows << 16 | t.cols;
  }
  const int rr = M <= 4 ? 1 : M <= 8 ? 2 : 4;
  return 4 * rr << 16 | deal_columns(N, rr, x_bits == 8, dtype == QUIK_BF16, zeros != 0).width;
}

extern "C" int quik_int4_group_matmul(const void *x, int x_bits, const uint8_t *w, const void *scales, const void *zeros,
                                      const float *scale_row, const void *bias, int dtype, int64_t M, int64_t N, int64_t K, int64_t group,
                                      void *out, void *workspace, int64_t workspace_bytes, void *stream) {
  if (x_bits != 8 && x_bits != 16) return QUIK_ERR_BITS;
  if (dtype != QUIK_F16 && dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0 || group <= 0) return QUIK_ERR_SHAPE;
  if (K % 32 || group % 32) return QUIK_ERR_ALIGN;
  if (M > INT32_MAX || N > INT32_MAX || K > 1 << 20) return QUIK_ERR_RANGE;  // (offsets of a workgroup's rows and the group of a column in 32 bits)
  if (M == 0 || N == 0) return QUIK_OK;
  if (!x || !w || !scales || !out || (x_bits == 8 && !scale_row)) return QUIK_ERR_NULL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(scales, 2) || !aligned(zeros, 2) || !aligned(scale_row, 4) || !aligned(bias, 2) ||
      !aligned(out, 2) || !aligned(workspace, 16))
    return QUIK_ERR_ALIGN;

  const int64_t g = group < K ? group : (K + 31) / 32 * 32;
  const GroupArgs p{x, w, scales, zeros, x_bits == 8 ? scale_row : nullptr, bias, out, M, N, K, static_cast<int32_t>(g),
                    static_cast<int32_t>((K + g - 1) / g), 0, static_cast<float *>(workspace), 1, static_cast<uint32_t>(((int64_t{1} << 31) + g / 32 - 1) / (g / 32))};
  if (x_bits == 8) return dtype == QUIK_BF16 ? by_groups<kI8BF16>(p, workspace_bytes, as_stream(stream)) : by_groups<kI8F16>(p, workspace_bytes, as_stream(stream));
  return dtype == QUIK_BF16 ? by_groups<kBF16>(p, workspace_bytes, as_stream(stream)) : by_groups<kF16>(p, workspace_bytes, as_stream(stream));
}
