// Products of rows in blocks of 32 with 4-bit weights in blocks of 32 (mx_format.h):
//   y[m, n] = row[m] * sum_b 2^(ex[m, b] - 127) 2^(ew[n, b] - 127) sum_{k in b} x[m, k] w[n, k] + bias[n]
// and the first half of a gated feed-forward block on them, with its result in such blocks.
//
// The scaled matrix instructions take a block of 32 codes per lane and its exponent byte, for either operand: 4-bit codes are 16 bytes, as they
// lie in a row, and nothing is widened, scaled or summed apart from them.  8-bit codes lie in two pieces of 16 bytes, columns 16 g .. of the
// first and of the second half of the instruction's columns (g: the lane's group), while the byte of group g is that of columns 32 g ..
// Sums of products of 4-bit codes are exact up to fp32's alignment (off by 2^-24 of the magnitudes' sum per instruction).  Of
// 8-bit ones eight at a time are aligned to the largest sum of two exponents among them and cut off 2^-13 below it, and e4m3's numbers reach over 17
// powers of two: they are taken in two parts, magnitudes from 2 up (bit 6 of the code) and those below, with zeros in each other's place.  Products of the
// first part are multiples of 2^-3 and of exponents up to 8 + 2, of the second multiples of 2^-10 and up to 0 + 2: neither loses anything.
// (In one part sums were off by 1.5e-4 of their size, and the codes behind a gated product by 8e-4 in place of 2e-4.)
// Columns behind the end of K: codes of x are made 0 in registers, the weights and bytes there are the row's last ones.
#include "mx_format.h"

#include <type_traits>

namespace quik {
namespace {

struct MxArgs {
  const uint8_t *x, *xs, *w, *ws;
  const float *row;
  const void *bias;
  void *out;      // 16-bit [M, N], or (gated) codes
  uint8_t *out_scale;  // gated
  int64_t M, N, K;     // N: columns of the result (gated: of either half)
  int32_t bf16, q_bits;
  int32_t width;   // result columns per tile of the kernel of few rows
  float *partial;  // K split: sums [splits][M][N rounded up to 4]
  int32_t splits;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_bytes16 __attribute__((ext_vector_type(4), aligned(1)));

// one byte per lane: it lands in the low byte of the four at LDS address m0 + 4 i (the others are not to be read)
__device__ __forceinline__ void dma_load_u8(const void *sbase, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %2" : : "s"(lds_addr), "v"(voff), "s"(sbase) : "memory", "m0");
}

// An operand of 4-bit codes is 16 bytes; of 8-bit ones 32.
template <int BITS>
struct Operand {
  u32x4 v[BITS / 4];
};
__device__ __forceinline__ i32x8 as_operand(const Operand<4> &o) {
  i32x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = static_cast<int>(o.v[0][i]);
  r[4] = r[5] = r[6] = r[7] = 0;  // (not read)
  return r;
}
__device__ __forceinline__ i32x8 as_operand(const Operand<8> &o) {
  i32x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = static_cast<int>(o.v[0][i]);
    r[4 + i] = static_cast<int>(o.v[1][i]);
  }
  return r;
}
// of four 8-bit codes: those from 2 up, those below, either with zeros of their signs in the others' place; and those from 2 up (turn 0) or below (kBelow)
__device__ __forceinline__ uint32_t large_of(uint32_t v) {
  const uint32_t six = v & 0x40404040u;
  return v & ((six - (six >> 6)) | 0xC0C0C0C0u);
}
__device__ __forceinline__ uint32_t small_of(uint32_t v) {
  const uint32_t six = v & 0x40404040u;
  return v & ~((six - (six >> 6)) | 0x40404040u);
}
__device__ __forceinline__ uint32_t part_of(uint32_t v, uint32_t turn) {
  const uint32_t six = v & 0x40404040u;
  return v & (((six - (six >> 6)) | 0xC0C0C0C0u) ^ turn);
}
constexpr uint32_t kBelow = 0x7F7F7F7Fu;

template <int BITS>
constexpr int kFormat = BITS == 4 ? 4 : 0;
template <int XB>
__device__ __forceinline__ f32x4 mfma16(const Operand<4> &w, const Operand<XB> &x, f32x4 c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(as_operand(w), as_operand(x), c, 4, kFormat<XB>, 0, static_cast<int>(sw), 0, static_cast<int>(sx));
}
template <int XB, int BYTE>
__device__ __forceinline__ f32x16 mfma32(const Operand<4> &w, const Operand<XB> &x, f32x16 c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(as_operand(w), as_operand(x), c, 4, kFormat<XB>, BYTE, static_cast<int>(sw), BYTE, static_cast<int>(sx));
}

__device__ __forceinline__ float from16(uint16_t v, bool bf16) { return bf16 ? to_f32<true>(v) : to_f32<false>(v); }
__device__ __forceinline__ uint16_t to16(float v, bool bf16) { return bf16 ? from_f32<true>(v) : from_f32<false>(v); }
__device__ __forceinline__ float bias_of(const MxArgs &p, int64_t n) { return from16(static_cast<const uint16_t *>(p.bias)[n], p.bf16); }
// the activation of a gated block, of products rounded to the 16-bit type
template <bool BF16>
__device__ __forceinline__ float activate(float gate, float up) {
  gate = round_storage<BF16>(gate);
  up = round_storage<BF16>(up);
  return __float_as_uint(gate) > kFarBits ? gated_far(gate, up) : gated(gate, up);
}

// Where a row's 16-byte pieces lie in LDS: at the piece's number exclusive-or this, so that 16 rows' reads of one piece go to different banks.
template <int PIECES>
__device__ __forceinline__ int turn_of(int row) {
  static_assert(PIECES == 4 || PIECES == 8 || PIECES == 16 || PIECES == 32, "");
  return PIECES >= 16 ? row & 15 : PIECES == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// Up to 32 token rows (TR of them in LDS, by sixteens), on 16x16x128 instructions: the weights are the rows of the result tile, the tokens its columns.  A workgroup
// takes tiles of p.width <= 16 * FT result columns, which deals all of them evenly to the CUs; its W waves take blocks of STEPS * 128 columns of K in
// turn and add their sums through LDS at a tile's end.  Operands and bytes come by direct copies, D - 1 blocks ahead and on into the next tile,
// into a ring of the wave's own (no barrier but at a tile's end).  Up to eight rows of 8-bit codes are sixteen columns: their codes from 2 up, and behind
// them those below, whose sums are added in the end.  Gated: matrix tiles 0 .. FT / 2 - 1 are gates, the others the same columns of up.
// Bound by the weights' stream: 1 x 8192 -> 28672 24.7 us, 5.1 TB/s (a copy's rate), with 8-bit rows 27.3, of which the codes' parting is 1.5; 1 x 13824 -> 5120 8.9 us,
// 4.2 TB/s; 1 x 4096 -> 4096 4.2 us, a launch and three trips to memory one after the other.  Gated 4 x 8192 -> 57344 48.6 us, 5.1 TB/s, 1 x 4096 -> 22016 13.1:
// 344 tiles of 32 columns for 256 CUs (smaller rings, two workgroups per CU, 13.8 .. 15.1).
template <int XB, int TR, int FT, int W, int D, int STEPS, bool TAIL>
struct RingShape {
  static constexpr int kPw = 4 * STEPS, kPx = kPw * (XB / 4), kPlanes = TAIL ? 4 : 1;
  static constexpr int kCW = FT * STEPS, kCX = TR * kPx / 64, kCSW = (16 * FT * STEPS + 63) / 64, kCSX = (TR * STEPS + 63) / 64;
  static constexpr int kCopies = kCW + kCX + kPlanes * (kCSW + kCSX);
  static constexpr int kAtX = kCW * 1024, kAtSW = kAtX + kCX * 1024, kAtSX = kAtSW + kPlanes * kCSW * 256, kStage = kAtSX + kPlanes * kCSX * 256;
  static constexpr int kGroups = (TR + 15) / 16, kRed = W * FT * kGroups * 1024, kLds = kRed + W * D * kStage;
  static_assert(TR * kPx % 64 == 0 && kCopies * (D - 1) < 64, "");
};

template <int XB, int TR, int FT, int W, int D, int STEPS, bool TAIL, bool GATED>
__global__ __launch_bounds__(64 * W) void mx_ring_kernel(MxArgs p) {
  using S = RingShape<XB, TR, FT, W, D, STEPS, TAIL>;
  static_assert(!GATED || FT == 4, "");  // (a block of 32 results)
  constexpr bool kBoth = XB == 8 && TR == 8;
  constexpr int kGroups = S::kGroups;  // of sixteen rows
  extern __shared__ float red[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int nb = static_cast<int>(p.K / kMxBlock), steps = (nb + 3) / 4, blocks = (steps + STEPS - 1) / STEPS;
  const int tiles = static_cast<int>((p.N + p.width - 1) / p.width);
  uint8_t *ring = reinterpret_cast<uint8_t *>(red) + S::kRed + wave * (D * S::kStage);
  const uint32_t ring_at = lds_address(ring);
  const int64_t pitch_w = p.K / 2, pitch_x = p.K * XB / 8;

  uint32_t from_x[S::kCX], from_sx[S::kCSX];
#pragma unroll
  for (int i = 0; i < S::kCX; ++i) {
    const int64_t row = i * (64 / S::kPx) + lane / S::kPx;
    from_x[i] = static_cast<uint32_t>((row < p.M ? row : p.M - 1) * pitch_x);
  }
#pragma unroll
  for (int i = 0; i < S::kCSX; ++i) {
    int64_t row = (i * 64 + lane) / STEPS;
    row = row < p.M ? row : p.M - 1;
    from_sx[i] = static_cast<uint32_t>(row * nb);
  }
  uint32_t from_w[S::kCW], from_sw[S::kCSW];
  const uint8_t *wbase, *wbase_up, *sbase;
  auto aim = [&](int tile) {  // at a tile's columns (past its end: the last one)
    const int64_t n0 = static_cast<int64_t>(tile) * p.width, left = (p.N - n0 < p.width ? p.N - n0 : p.width) - 1;
    wbase = p.w + n0 * pitch_w;
    wbase_up = GATED ? wbase + p.N * pitch_w : wbase;
    sbase = p.ws + n0 * nb;
    constexpr int kRows = GATED ? 8 * FT : 16 * FT;  // of either half
#pragma unroll
    for (int i = 0; i < S::kCW; ++i) {
      const int64_t row = (i * (64 / S::kPw) + lane / S::kPw) % kRows;
      from_w[i] = static_cast<uint32_t>((row < left ? row : left) * pitch_w);
    }
#pragma unroll
    for (int i = 0; i < S::kCSW; ++i) {
      const int at = (i * 64 + lane) / STEPS;
      const int64_t row = at % kRows;
      from_sw[i] = static_cast<uint32_t>(((row < left ? row : left) + (GATED && at >= kRows ? p.N : 0)) * nb);
    }
  };
  auto copy = [&](int stage, int blk) {
    const uint32_t to = ring_at + stage * S::kStage;
    const bool whole = (blk + 1) * STEPS <= steps && (!TAIL || (blk + 1) * STEPS * 4 <= nb);
    // (pieces past the end of a row come from its last one)
    const int w0 = blk * S::kPw, last_w = nb - 1, x0 = blk * S::kPx, last_x = nb * (XB / 4) - 1;
#pragma unroll
    for (int i = 0; i < S::kCW; ++i) {
      const int row = i * (64 / S::kPw) + lane / S::kPw, piece = w0 + ((lane % S::kPw) ^ turn_of<S::kPw>(row));
      const uint8_t *base = GATED && i * (64 / S::kPw) >= 8 * FT ? wbase_up : wbase;
      dma_load16(base, from_w[i] + static_cast<uint32_t>(whole || piece < last_w ? piece : last_w) * 16, to + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < S::kCX; ++i) {
      const int row = i * (64 / S::kPx) + lane / S::kPx, piece = x0 + ((lane % S::kPx) ^ turn_of<S::kPx>(row));
      dma_load16(p.x, from_x[i] + static_cast<uint32_t>(whole || piece < last_x ? piece : last_x) * 16, to + S::kAtX + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < S::kCSW + S::kCSX; ++i) {
      const bool is_x = i >= S::kCSW;
      const int j = is_x ? i - S::kCSW : i, step = blk * STEPS + (j * 64 + lane) % STEPS;
      const uint32_t row = is_x ? from_sx[is_x ? j : 0] : from_sw[is_x ? 0 : j];
      const uint32_t at = to + (is_x ? S::kAtSX : S::kAtSW) + j * 256;
      if constexpr (TAIL) {
#pragma unroll
        for (int plane = 0; plane < 4; ++plane) {
          const int b = 4 * step + plane;
          dma_load_u8(is_x ? p.xs : sbase, row + static_cast<uint32_t>(b < nb ? b : nb - 1), at + plane * (is_x ? S::kCSX : S::kCSW) * 256);
        }
      } else {
        dma_load_u32(is_x ? p.xs : sbase, row + 4u * static_cast<uint32_t>(step < steps ? step : steps - 1), at);
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
  const int token = TR >= 16 ? col : col % TR;
  const uint32_t turn = col < 8 ? 0 : kBelow;
  int stage = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    f32x4 acc[FT][kGroups];
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int g = 0; g < kGroups; ++g) acc[f][g] = f32x4{0, 0, 0, 0};
    for (int blk = wave; blk < blocks; blk += W) {
      copy_next(stage == 0 ? D - 1 : stage - 1);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(S::kCopies * (D - 1)));
      asm volatile("" ::: "memory");
      const uint8_t *from = ring + stage * S::kStage;
      // a row's bytes of all steps; whole planes: of this lane's group
      uint32_t sw[FT][STEPS], sx[kGroups][STEPS];
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int plane = TAIL ? kg : 0;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          sx[g][s] = *reinterpret_cast<const uint32_t *>(from + S::kAtSX + plane * S::kCSX * 256 + ((token + 16 * g) * STEPS + s) * 4);
#pragma unroll
        for (int f = 0; f < FT; ++f)
          sw[f][s] = *reinterpret_cast<const uint32_t *>(from + S::kAtSW + plane * S::kCSW * 256 + ((16 * f + col) * STEPS + s) * 4);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (blk * STEPS + s >= steps) break;
        Operand<XB> x[kGroups], below[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int row = token + 16 * g;
#pragma unroll
          for (int h = 0; h < XB / 4; ++h) {
            const int piece = XB == 4 ? 4 * s + kg : 8 * s + 4 * h + kg;
            x[g].v[h] = *reinterpret_cast<const u32x4 *>(from + S::kAtX + (row * S::kPx + (piece ^ turn_of<S::kPx>(row))) * 16);
            if constexpr (TAIL) {
              const int b = 4 * (blk * STEPS + s) + (XB == 4 ? kg : 2 * h + (kg >> 1));
              if (b >= nb) x[g].v[h] = u32x4{0, 0, 0, 0};
            }
          }
          if constexpr (XB == 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t v = x[g].v[i / 4][i % 4];
              if constexpr (!kBoth) below[g].v[i / 4][i % 4] = small_of(v);
              x[g].v[i / 4][i % 4] = kBoth ? part_of(v, turn) : large_of(v);
            }
          }
        }
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          Operand<4> w;
          w.v[0] = *reinterpret_cast<const u32x4 *>(from + ((16 * f + col) * S::kPw + ((4 * s + kg) ^ turn_of<S::kPw>(col))) * 16);
          const uint32_t by_w = TAIL ? sw[f][s] : sw[f][s] >> (8 * kg);
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            const uint32_t by_x = TAIL ? sx[g][s] : sx[g][s] >> (8 * kg);
            acc[f][g] = mfma16<XB>(w, x[g], acc[f][g], by_w, by_x);
            if constexpr (XB == 8 && !kBoth) acc[f][g] = mfma16<XB>(w, below[g], acc[f][g], by_w, by_x);
          }
        }
      }
      stage = stage == D - 1 ? 0 : stage + 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wait only; this stage is copied to next: its reads are done)
    }
    // the waves' sums: value r of lane l is column 16 f + 4 (l / 16) + r of token 16 g + l % 16
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[(((wave * FT + f) * kGroups + g) * 4 + r) * 64 + lane] = acc[f][g][r];
    __syncthreads();
    const int64_t n0 = static_cast<int64_t>(tile) * p.width;
    auto sum = [&](int m, int n) {
      const int at = (((n >> 4) * kGroups + (m >> 4)) * 4 + (n & 3)) * 64 + ((n >> 2) & 3) * 16 + (m & 15);
      constexpr int kWave = FT * kGroups * 256;
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += kBoth ? red[i * kWave + at] + red[i * kWave + at + 8] : red[i * kWave + at];
      return p.row ? v * p.row[m] : v;
    };
    if constexpr (GATED) {
      for (int e = threadIdx.x; e < p.M * 32; e += 64 * W) {
        const int m = e >> 5, n = e & 31;  // (inner is a multiple of 32: the block is whole)
        const float g = sum(m, n), u = sum(m, 32 + n), v = p.bf16 ? activate<true>(g, u) : activate<false>(g, u);
        uint32_t top = __float_as_uint(v) & 0x7FFFFFFFu;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) top = umax(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
        const int64_t block = m * (p.N / kMxBlock) + n0 / kMxBlock;
        const uint32_t byte = p.q_bits == 4 ? block_byte<4>(top) : block_byte<8>(top);
        const float other = __shfl_xor(v, 1);
        if (n == 0) p.out_scale[block] = static_cast<uint8_t>(byte);
        const float pair[8] = {v, other, 0, 0, 0, 0, 0, 0};
        if (p.q_bits == 8) static_cast<uint8_t *>(p.out)[block * 32 + n] = static_cast<uint8_t>(encode8(pair, byte).x);
        else if (n % 2 == 0) static_cast<uint8_t *>(p.out)[block * 16 + n / 2] = static_cast<uint8_t>(encode4(pair, byte));
      }
    } else {
      for (int e = threadIdx.x; e < p.M * 16 * FT; e += 64 * W) {
        const int m = e / (16 * FT), n = e % (16 * FT);
        if (n >= p.width || n0 + n >= p.N) continue;
        float v = sum(m, n);
        if (p.bias) v += bias_of(p, n0 + n);
        static_cast<uint16_t *>(p.out)[m * p.N + n0 + n] = to16(v, p.bf16);
      }
    }
    __syncthreads();  // (the sums are read: the next tile's may be written)
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (no copy is under way when the workgroup's LDS goes to another)
}

// More token rows than that, on 32x32x64 instructions: WM x WN waves side by side, each with RM x RN result tiles of 32 x 32, on stages of 256 columns: whole lines
// of 128 bytes of the weights' rows (half lines cost as many requests again: 8192 x 8192 -> 8192 on stages of 128 columns 434 us).  LDS holds two
// stages; one or two more are on their way to registers.  (Direct copies to LDS hold the wave that issues them until the CU has taken the ones before, some
// 36 cycles per kilobyte, and its products with it; and they can start only when their place is free: 300 us.)
// A stage is four products of 64 columns.  An operand is read again for the next one behind its last product of this one.  In the middle of the fourth
// there is a barrier: every wave has read all of the stage, and the next one is there; behind it the stage after the next is written over
// this one, and the one behind that is requested.
// Exponent bytes lie apart, eight of a row per stage in a ring of four stages, and come two stages at a time, also through registers: rows of them may start
// at any byte.  Four bytes of a stage, those of this lane's group, are one operand for it.  Bytes behind the end of K are 0 on both sides:
// whatever codes stand there, a product of 2^-254 does not change a sum.
// Gated: a wave's tiles f < RN / 2 are gates, the others the same columns of up.
// 8-bit rows: the codes of the next 64 columns are taken apart behind the products of these, five vector instructions per four codes, in the places where
// the matrix unit is busy.  So a wave has one row of matrix tiles and up to four of them in it (with two rows of two, each wave takes twice as many
// codes apart: 2048 x 8192 -> 28672 782 us, this 637; its products are 75 % of the SIMDs' cycles, at a clock of 1.74 GHz).
// 4 bits: 2048 x 8192 -> 28672 275 us, 3.5 PFLOP/s, the matrix unit busy for 48 % of the cycles, at 1.8 GHz (24576 columns, three full rounds of workgroups, 220:
// 54 %, 1.7 GHz); 64 x 5120 -> 27648 gated 22.0 us, 3.6 TB/s.
template <int XB, int RM, int RN, int WM, int WN>
struct TileShape {
  // Stages on their way to registers: two where the results leave room, with their loads dealt to three quarters of a stage (us, one on its way and
  // this: 300 x 4544 -> 4544 16.2, 14.9, 64 x 5120 -> 27648 23.8, 22.4).
  static constexpr int kPre = RM * RN <= 4 ? 2 : 1;
  static constexpr int kW = WM * WN, kBM = 32 * RM * WM, kBN = 32 * RN * WN, kT = 64 * kW;
  static constexpr int kPx = 2 * XB, kPw = 8;                         // 16-byte pieces of a row in a stage
  static constexpr int kCX = kBM * kPx / 64, kCW = kBN * kPw / 64;    // loads of 1 KB
  static constexpr int kMyX = kCX / kW, kMyW = kCW / kW, kLoads = kMyX + kMyW;
  static_assert(kCX % kW == 0 && kCW % kW == 0, "");
  static constexpr int kAtW = kCX * 1024, kStage = kAtW + kCW * 1024;
  static constexpr int kAtS = 2 * kStage, kRings = kAtS + (kBM + kBN) * 32;
  static constexpr int kPitch = RN * 64 + 16, kOut = kW * 32 * kPitch;  // (a wave's 32 rows on their way out)
  static constexpr int kLds = kRings > kOut ? kRings : kOut;
  static constexpr int kRows = (kBM + kBN + kT - 1) / kT;              // rows of exponent bytes per thread
};

template <int XB, int RM, int RN, int WM, int WN, bool GATED>
__global__ __launch_bounds__(64 * WM * WN) void mx_tile_kernel(MxArgs p) {
  using S = TileShape<XB, RM, RN, WM, WN>;
  static_assert((!GATED || RN % 2 == 0) && (XB == 4 || RM == 1), "");
  constexpr int kCols = GATED ? S::kBN / 2 : S::kBN;  // result columns per tile
  extern __shared__ float red[];
  uint8_t *lds = reinterpret_cast<uint8_t *>(red);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, kg = lane >> 5;
  const int wn = wave % WN, wm = wave / WN;
  const int nb = static_cast<int>(p.K / kMxBlock), all_stages = (nb + 7) / 8;
  // Workgroups go to the eight dies in turn: each die gets a run of tiles, in bands of four row tiles, column by column, so that those
  // that run on a die at a time share both their rows and their weights in its L2.  A tile whose K is split is `splits` workgroups, one after
  // the other.
  constexpr int kBand = 4;
  const int m_tiles = static_cast<int>((p.M + S::kBM - 1) / S::kBM), n_tiles = static_cast<int>((p.N + kCols - 1) / kCols);
  const int all = static_cast<int>(gridDim.x), die = blockIdx.x & 7, run = all >> 3, rest = all & 7;
  const int unit = die * run + (die < rest ? die : rest) + static_cast<int>(blockIdx.x >> 3);
  // (a division is some thirty vector instructions; its result, the same for all lanes, goes back to a scalar register)
  int tile = unit, split = 0, first = 0, stages = all_stages;
  if (p.splits > 1) {
    tile = __builtin_amdgcn_readfirstlane(unit / p.splits), split = unit - tile * p.splits;
    first = __builtin_amdgcn_readfirstlane(all_stages * split / p.splits);  // (at most 2^12 stages)
    stages = __builtin_amdgcn_readfirstlane(all_stages * (split + 1) / p.splits);
  }
  const int band = __builtin_amdgcn_readfirstlane(tile / (kBand * n_tiles)), in_band = tile - band * kBand * n_tiles;
  const int high = m_tiles - band * kBand < kBand ? m_tiles - band * kBand : kBand;
  const int across = __builtin_amdgcn_readfirstlane(high == 4 ? in_band >> 2 : high == 3 ? in_band / 3 : high == 2 ? in_band >> 1 : in_band);
  static_assert(kBand == 4, "");
  const int64_t m0 = static_cast<int64_t>(band * kBand + in_band - across * high) * S::kBM, n0 = static_cast<int64_t>(across) * kCols;

  const int64_t pitch_w = p.K / 2, pitch_x = p.K * XB / 8, left_m = p.M - 1 - m0, left_n = p.N - 1 - n0;
  const uint8_t *xbase = p.x + m0 * pitch_x, *wbase = p.w + n0 * pitch_w;
  // weight row R of the tile: wave R / (32 RN)'s, of its tiles the first half gates, the second up
  auto column_of = [](int R) { return GATED ? R / (32 * RN) * (16 * RN) + R % (16 * RN) : R; };
  auto is_up = [](int R) { return GATED && R % (32 * RN) >= 16 * RN; };
  // this wave's loads: the row's offset and the piece of the stage that this lane takes, and where it goes
  uint32_t x_off[S::kMyX], w_off[S::kMyW];
  auto nth = [&](int i) { return wave + i * S::kW; };
  auto x_row = [&](int i) { return nth(i) * (64 / S::kPx) + lane / S::kPx; };
  auto w_row = [&](int i) { return nth(i) * 8 + (lane >> 3); };
  const int x_piece = lane % S::kPx, w_piece = lane & 7;
#pragma unroll
  for (int i = 0; i < S::kMyX; ++i) x_off[i] = static_cast<uint32_t>((x_row(i) < left_m ? x_row(i) : left_m) * pitch_x);
#pragma unroll
  for (int i = 0; i < S::kMyW; ++i) {
    const int n = column_of(w_row(i));
    w_off[i] = static_cast<uint32_t>((n < left_n ? n : left_n) * pitch_w);
  }
  // (a load's rows are a multiple of 16 behind the first one's: the same turn)
  static_assert(S::kW * (64 / S::kPx) % 16 == 0, "");
  const int x_to = (x_row(0) * S::kPx + (x_piece ^ turn_of<S::kPx>(x_row(0)))) * 16, w_to = S::kAtW + (w_row(0) * 8 + (w_piece ^ turn_of<8>(w_row(0)))) * 16;
  constexpr int kPre = S::kPre;
  u32x4 staged_of[kPre][S::kLoads];
  auto load = [&](u32x4 (&staged)[S::kLoads], int stage, int i) {  // (pieces past the end of a row come from its last one)
    if (i < S::kMyX) {
      const int last = nb * (XB / 4) - 1 - stage * S::kPx, piece = x_piece < last ? x_piece : last;
      staged[i] = *reinterpret_cast<const u32x4 *>(xbase + stage * (S::kPx * 16) + (x_off[i] + static_cast<uint32_t>(piece) * 16));
    } else {
      const int last = nb - 1 - stage * 8, piece = w_piece < last ? w_piece : last;
      const uint8_t *from = is_up(nth(i - S::kMyX) * 8) ? wbase + p.N * pitch_w : wbase;
      staged[i] = *reinterpret_cast<const u32x4 *>(from + stage * 128 + (w_off[i - S::kMyX] + static_cast<uint32_t>(piece) * 16));
    }
  };
  auto write = [&](const u32x4 (&staged)[S::kLoads], int stage, int i) {
    uint8_t *to = lds + ((stage - first) & 1) * S::kStage;
    if (i < S::kMyX) *reinterpret_cast<u32x4 *>(to + x_to + (nth(i) - wave) * 1024) = staged[i];
    else *reinterpret_cast<u32x4 *>(to + w_to + (nth(i - S::kMyX) - wave) * 1024) = staged[i];
  };
  // exponent bytes: rows of x, then of w (a thread without a row of its own takes the last one too)
  const uint8_t *bytes_of[S::kRows];
  auto byte_row = [&](int i) {
    const int row = threadIdx.x + i * S::kT;
    return row < S::kBM + S::kBN ? row : S::kBM + S::kBN - 1;
  };
#pragma unroll
  for (int i = 0; i < S::kRows; ++i) {
    const int row = byte_row(i), R = row < S::kBM ? 0 : row - S::kBM, n = column_of(R);
    bytes_of[i] = row < S::kBM ? p.xs + (m0 + (row < left_m ? row : left_m)) * nb : p.ws + (n0 + (n < left_n ? n : left_n) + (is_up(R) ? p.N : 0)) * nb;
  }
  u32x4 bytes[S::kRows];  // of two stages
  // A pair of stages' bytes; of the last pair the row's last sixteen, of which the first `less` belong to stages before.
  auto load_bytes = [&](int pair) {
    const int at = (first + 2 * pair) * 8, from = at < nb - 16 ? at : nb - 16;
#pragma unroll
    for (int i = 0; i < S::kRows; ++i) bytes[i] = *reinterpret_cast<const mx_bytes16 *>(bytes_of[i] + (nb < 16 ? 0 : from));
    return at - from;
  };
  // (eight bytes of a row, a stage's, at their number exclusive-or (row / 8) % 4: 32 rows' reads of one stage at different banks)
  auto write_bytes = [&](int pair, int less) {
#pragma unroll
    for (int i = 0; i < S::kRows; ++i) {
      // (sixteen bytes less the first `less`, zeros behind; bit by bit: no branch)
      const uint32_t by4 = less & 4 ? ~0u : 0, by8 = less & 8 ? ~0u : 0, some = less >= 16 ? 0 : ~0u;
      auto choose_of = [](uint32_t mask, uint32_t a, uint32_t b) { return (a & mask) | (b & ~mask); };
      u32x4 v = bytes[i];
      v = u32x4{choose_of(by4, v[1], v[0]), choose_of(by4, v[2], v[1]), choose_of(by4, v[3], v[2]), v[3] & ~by4};
      v = u32x4{choose_of(by8, v[2], v[0]), choose_of(by8, v[3], v[1]), v[2] & ~by8, v[3] & ~by8};
      v = u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], less & 3) & some, __builtin_amdgcn_alignbyte(v[2], v[1], less & 3) & some,
                __builtin_amdgcn_alignbyte(v[3], v[2], less & 3) & some, __builtin_amdgcn_alignbyte(0, v[3], less & 3) & some};
      const int row = byte_row(i);
      uint8_t *to = lds + S::kAtS + row * 32;
      *reinterpret_cast<uint2 *>(to + ((2 * pair & 3) ^ ((row >> 3) & 3)) * 8) = make_uint2(v[0], v[1]);
      *reinterpret_cast<uint2 *>(to + (((2 * pair + 1) & 3) ^ ((row >> 3) & 3)) * 8) = make_uint2(v[2], v[3]);
    }
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int t = 0; t < RM; ++t)
#pragma unroll
    for (int f = 0; f < RN; ++f)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][f][r] = 0.0f;

  // operands of 64 columns
  Operand<XB> x[RM];
  Operand<4> w[RN];
  Operand<8> part[XB == 8 ? 2 : 1][2];  // x in its two parts, of this and of the next 64 columns
  uint2 raw[RM + RN];  // the next stage's exponent bytes of their rows
  uint32_t by[RM + RN];
  const int x_at = (wm * RM * 32 + col) * S::kPx * 16, w_at = S::kAtW + (wn * RN * 32 + col) * 128;
  const int x_turn = turn_of<S::kPx>(col), w_turn = turn_of<8>(col);  // (of every tile's rows: they are 32 apart)
  auto read_x = [&](const uint8_t *from, int s, int t) {
#pragma unroll
    for (int i = 0; i < XB / 4; ++i) {
      const int piece = XB == 4 ? 2 * s + kg : 4 * s + 2 * i + kg;
      x[t].v[i] = *reinterpret_cast<const u32x4 *>(from + x_at + t * (32 * S::kPx * 16) + (piece ^ x_turn) * 16);
    }
  };
  auto read_w = [&](const uint8_t *from, int s, int f) {
    w[f].v[0] = *reinterpret_cast<const u32x4 *>(from + w_at + f * 4096 + ((2 * s + kg) ^ w_turn) * 16);
  };
  const int bytes_at = S::kAtS + (wm * RM * 32 + col) * 32, bytes_at_w = S::kAtS + (S::kBM + wn * RN * 32 + col) * 32;
  auto read_bytes = [&](int stage, int n) {
    const int to = (((stage - first) & 3) ^ ((col >> 3) & 3)) * 8;
    raw[n] = *reinterpret_cast<const uint2 *>(lds + (n < RM ? bytes_at + n * 1024 : bytes_at_w + (n - RM) * 1024) + to);
  };
  const uint32_t pick = 0x06040200u + static_cast<uint32_t>(kg) * 0x01010101u;
  // (four codes each)
  auto take_apart = [&](Operand<8> (&to)[2], int from, int end) {
    if constexpr (XB == 8) {
#pragma unroll
      for (int i = from; i < end; ++i) {
        const uint32_t v = x[0].v[i / 4][i % 4];
        to[0].v[i / 4][i % 4] = large_of(v);
        to[1].v[i / 4][i % 4] = small_of(v);
      }
    }
  };
  constexpr int kBefore = RM * (RN / 2);  // products of a stage's last quarter in front of the barrier: those of the first half of the weights' tiles
  // Product i of quarter s, then the reads for the next quarter (of `next`) that wait for it, in this order (left to itself the compiler puts all reads
  // first, behind them all products).
  auto product = [&](auto quarter, int i, const uint8_t *next, bool reads) {
    constexpr int s = decltype(quarter)::value;
    const int f = i / RM, t = i % RM;
    if constexpr (XB == 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        acc[0][f] = mfma32<8, s>(w[f], part[s & 1][h], acc[0][f], by[RM + f], by[0]);
        constexpr int kChunks = 2 * (RN - kBefore);
        const int chunk = 2 * (f - kBefore) + h;
        if (reads && f >= kBefore) take_apart(part[(s + 1) & 1], chunk * 8 / kChunks, (chunk + 1) * 8 / kChunks);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (reads) read_w(next, (s + 1) % 4, f);
    } else {
      acc[t][f] = mfma32<XB, s>(w[f], x[t], acc[t][f], by[RM + f], by[t]);
      if (reads && t == RM - 1) read_w(next, (s + 1) % 4, f);
      if (reads && f == RN - 1) read_x(next, (s + 1) % 4, t);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto quarter = [&](auto which, const uint8_t *next, auto behind) {
    if constexpr (XB == 8) read_x(next, decltype(which)::value + 1, 0);
#pragma unroll
    for (int i = 0; i < RM * RN; ++i) {
      product(which, i, next, true);
      behind(decltype(which)::value * RM * RN + i);
    }
  };
  constexpr std::integral_constant<int, 0> k0{};
  constexpr std::integral_constant<int, 1> k1{};
  constexpr std::integral_constant<int, 2> k2{};
  constexpr std::integral_constant<int, 3> k3{};
  // (past the last stage: that one once more, not used)
  auto there = [&](int stage) { return stage < stages ? stage : stages - 1; };
  int less = 0;
  if (nb >= 16) {
    less = load_bytes(0);
  } else {  // rows of fewer bytes than a load: one pair, byte by byte; the loop's loads, whose bytes are not used, are of x, a row of which has sixteen
#pragma unroll
    for (int i = 0; i < S::kRows; ++i) {
      uint64_t v[2] = {0, 0};
#pragma unroll 1
      for (int e = 0; e < nb; ++e) {
        const uint64_t byte = bytes_of[i][e];
        if (e < 8) v[0] |= byte << (8 * e);
        else v[1] |= byte << (8 * (e - 8));
      }
      bytes[i] = u32x4{static_cast<uint32_t>(v[0]), static_cast<uint32_t>(v[0] >> 32), static_cast<uint32_t>(v[1]), static_cast<uint32_t>(v[1] >> 32)};
      bytes_of[i] = p.x;
    }
  }
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) load(staged_of[0], first, i);
  write_bytes(0, nb < 16 ? first * 8 : less);
  less = load_bytes(1);
#pragma unroll
  for (int d = 0; d < 2; ++d) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      write(staged_of[0], first + d, i);
      load(staged_of[0], there(first + d + 1), i);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < RM + RN; ++n) read_bytes(first, n);
#pragma unroll
  for (int f = 0; f < RN; ++f) read_w(lds, 0, f);
#pragma unroll
  for (int t = 0; t < RM; ++t) read_x(lds, 0, t);
  take_apart(part[0], 0, 8);
  constexpr int kHalf = S::kLoads / 2;
  auto stage_of = [&](int stage, auto odd) {
    constexpr int kOdd = decltype(odd)::value;
    const uint8_t *from = lds + kOdd * S::kStage, *next = lds + (1 - kOdd) * S::kStage;
#pragma unroll
    for (int n = 0; n < RM + RN; ++n) by[n] = __builtin_amdgcn_perm(raw[n].y, raw[n].x, pick);
    // What is requested of the stage behind those under way, in the places of the stage's products: two on their way, in the first three quarters;
    // one, half of it behind its place's writing and half in the first quarter.
    constexpr int kSlots = kPre == 2 ? 3 * RM * RN : RM * RN, kFrom = kPre == 2 ? 0 : kHalf;
    auto request = [&](int i) {
      if (i >= kSlots) return;
#pragma unroll
      for (int k = kFrom + i * (S::kLoads - kFrom) / kSlots; k < kFrom + (i + 1) * (S::kLoads - kFrom) / kSlots; ++k)
        load(staged_of[(kOdd + 1) % kPre], there(stage + 1 + kPre), k);
      __builtin_amdgcn_sched_barrier(0);
    };
    quarter(k0, from, request);
    quarter(k1, from, request);
    quarter(k2, from, request);
#pragma unroll
    for (int i = 0; i < kBefore; ++i) product(k3, i, nullptr, false);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (a wait and a barrier)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < RN / 2; ++f) read_w(next, 0, f);
    if constexpr (XB == 8) read_x(next, 0, 0);
#pragma unroll
    for (int n = 0; n < RM + RN; ++n) read_bytes(stage + 1, n);
    __builtin_amdgcn_sched_barrier(0);
    // The next pair's bytes are requested at once where two stages are on their way, so that a wait for them is none for the loads of the stages between (300 x 8192 ->
    // 4544 21.8, 21.1 us), else at the end of the next stage (2048 x 8192 -> 28672 299, 290).
    if constexpr (kOdd == 0) write_bytes((stage - first) / 2 + 1, less);
    if constexpr (kOdd == 0 && kPre == 2) less = load_bytes((stage - first) / 2 + 2);
    // the rest of the products, and between them what is written and requested
    constexpr int kRest = RM * RN - kBefore;
#pragma unroll
    for (int i = 0; i < kRest; ++i) {
#pragma unroll
      for (int k = i * S::kLoads / kRest; k < (i + 1) * S::kLoads / kRest; ++k) {
        write(staged_of[kOdd % kPre], stage + 2, k);
        if (kPre == 1 && k < kHalf) load(staged_of[0], there(stage + 3), k);
      }
      if (kPre == 1 && kOdd == 1 && i == kRest - 1) less = load_bytes((stage - first + 1) / 2 + 1);
      product(k3, kBefore + i, next, true);
    }
  };
  int stage = first;
  for (; stage + 2 < stages; stage += 2) {
    stage_of(stage, std::false_type{});
    stage_of(stage + 1, std::true_type{});
  }
  const uint8_t *at_last = lds;
  if (stage + 1 < stages) {
    stage_of(stage, std::false_type{});
    at_last = lds + S::kStage;
  }
#pragma unroll
  for (int n = 0; n < RM + RN; ++n) by[n] = __builtin_amdgcn_perm(raw[n].y, raw[n].x, pick);
  quarter(k0, at_last, [](int) {});
  quarter(k1, at_last, [](int) {});
  quarter(k2, at_last, [](int) {});
#pragma unroll
  for (int i = 0; i < RM * RN; ++i) product(k3, i, nullptr, false);
  // value r of a lane: column 8 (r / 4) + 4 kg + r % 4 of token col
  if constexpr (!GATED) {
    if (p.splits == 1) __syncthreads();  // (the last stage is read: results go out through its place)
  }
  // (one code for either type: a choice per number costs a branch per number, 9 us of a 256 x 256 tile's results)
  auto finish = [&](auto type) {
    constexpr bool kBF16 = decltype(type)::value;
    // added without a bias: -0, which leaves every number as it is
    float bias[GATED ? 1 : RN][4][4];
    if constexpr (!GATED) {
#pragma unroll
      for (int f = 0; f < RN; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) bias[f][j][r] = -0.0f;
      if (p.bias) {
#pragma unroll
        for (int f = 0; f < RN; ++f)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int64_t n = n0 + (wn * RN + f) * 32 + 8 * j + 4 * kg + r;
              bias[f][j][r] = to_f32<kBF16>(static_cast<const uint16_t *>(p.bias)[n < p.N ? n : p.N - 1]);
            }
      }
    }
#pragma unroll
    for (int t = 0; t < RM; ++t) {
      const int64_t m = m0 + (wm * RM + t) * 32 + col;
      const float scale = p.row && m < p.M ? p.row[m] : 1.0f;
      if constexpr (GATED) {
#pragma unroll
        for (int f = 0; f < RN / 2; ++f) {
          const int64_t n = n0 + wn * (16 * RN) + 32 * f;
          float v[16];
          uint32_t top = 0;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            v[r] = activate<kBF16>(acc[t][f][r] * scale, acc[t][f + RN / 2][r] * scale);
            top = umax(top, __float_as_uint(v[r]) & 0x7FFFFFFFu);
          }
          top = umax(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
          const uint32_t byte = p.q_bits == 4 ? block_byte<4>(top) : block_byte<8>(top);
          const int64_t block = m * (p.N / kMxBlock) + n / kMxBlock;
          const bool there = m < p.M && n < p.N;  // (inner is a multiple of 32)
          if (there && kg == 0) p.out_scale[block] = static_cast<uint8_t>(byte);
          if (p.q_bits == 4) {  // two bytes of every four are this lane's, the others the lane's 32 on
            uint32_t mine[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float e[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) e[r] = v[8 * i + r];
              mine[i] = encode4(e, byte);
            }
            const uint32_t o0 = static_cast<uint32_t>(__shfl_xor(static_cast<int>(mine[0]), 32)), o1 = static_cast<uint32_t>(__shfl_xor(static_cast<int>(mine[1]), 32));
            const uint32_t lo = kg ? o1 : mine[0], hi = kg ? mine[1] : o0;  // group 0 stores columns 0 .. 15, group 1 the others
            const uint2 both = make_uint2((lo & 0xFFFFu) | hi << 16, lo >> 16 | (hi & 0xFFFF0000u));
            if (there) *reinterpret_cast<loose2 *>(static_cast<uint8_t *>(p.out) + block * 16 + 8 * kg) = loose2{both.x, both.y};
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float e[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) e[r] = v[8 * i + r];
              const uint2 both = encode8(e, byte);
              uint8_t *to = static_cast<uint8_t *>(p.out) + block * 32 + 16 * i + 4 * kg;
              if (there) {
                *reinterpret_cast<mx_loose1 *>(to) = both.x;
                *reinterpret_cast<mx_loose1 *>(to + 8) = both.y;
              }
            }
          }
        }
      } else {
        // 32 rows of the wave's columns through LDS, so that a store takes whole pieces of rows (four columns per lane as they lie in the registers: 29 us
        // of 256 tiles of 256 x 256)
        uint8_t *out = lds + wave * (32 * S::kPitch);
#pragma unroll
        for (int f = 0; f < RN; ++f)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[t][f][4 * j + r] * scale + bias[f][j][r];
            *reinterpret_cast<uint2 *>(out + col * S::kPitch + (f * 32 + 8 * j + 4 * kg) * 2) =
                make_uint2(pack2_from_f32<kBF16>(v[0], v[1]), pack2_from_f32<kBF16>(v[2], v[3]));
          }
        asm volatile("" ::: "memory");  // (one wave's LDS accesses follow each other)
#pragma unroll
        for (int i = 0; i < 2 * RN; ++i) {
          const int piece = i * 64 + lane, row = piece / (4 * RN), at = piece % (4 * RN) * 8;
          const int64_t mm = m0 + (wm * RM + t) * 32 + row, n = n0 + wn * (RN * 32) + at;
          const uint4 w = *reinterpret_cast<const uint4 *>(out + row * S::kPitch + at * 2);
          if (mm >= p.M || n >= p.N) continue;
          uint16_t *to = static_cast<uint16_t *>(p.out) + mm * p.N + n;
          if (n + 7 < p.N) {
            *reinterpret_cast<loose4 *>(to) = loose4{w.x, w.y, w.z, w.w};
          } else {
            const uint32_t h[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int r = 0; r < 7; ++r)
              if (n + r < p.N) to[r] = static_cast<uint16_t>(h[r / 2] >> (16 * (r & 1)));
          }
        }
        asm volatile("" ::: "memory");
      }
    }
  };
  if constexpr (!GATED) {
    if (p.splits > 1) {
#pragma unroll
      for (int t = 0; t < RM; ++t)
#pragma unroll
        for (int f = 0; f < RN; ++f)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + (wm * RM + t) * 32 + col, n = n0 + (wn * RN + f) * 32 + 8 * j + 4 * kg;
            if (m < p.M && n < p.N)
              *reinterpret_cast<f32x4 *>(p.partial + (split * p.M + m) * ((p.N + 3) & ~int64_t{3}) + n) =
                  f32x4{acc[t][f][4 * j], acc[t][f][4 * j + 1], acc[t][f][4 * j + 2], acc[t][f][4 * j + 3]};
          }
      return;
    }
  }
  if (p.bf16) finish(std::true_type{});
  else finish(std::false_type{});
}

// the sums of a split K in the order of the splits, then what the tiles do with a sum
__global__ __launch_bounds__(256) void mx_join_kernel(MxArgs p) {
  const int64_t pitch = (p.N + 3) & ~int64_t{3}, quads = pitch / 4, at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= p.M * quads) return;
  const int64_t m = at / quads, n = at % quads * 4;
  const float *from = p.partial + m * pitch + n;
  const int64_t part = p.M * pitch;
  f32x4 v = *reinterpret_cast<const f32x4 *>(from);
  int i = 1;
  for (; i + 2 < p.splits; i += 3) {  // (three requested together)
    const f32x4 a = *reinterpret_cast<const f32x4 *>(from + i * part), b = *reinterpret_cast<const f32x4 *>(from + (i + 1) * part),
                c = *reinterpret_cast<const f32x4 *>(from + (i + 2) * part);
    v = v + a + b + c;
  }
  for (; i < p.splits; ++i) v += *reinterpret_cast<const f32x4 *>(from + i * part);
  const float row = p.row ? p.row[m] : 1.0f;
  for (int r = 0; r < 4 && n + r < p.N; ++r) {
    float y = p.row ? v[r] * row : v[r];
    if (p.bias) y += bias_of(p, n + r);
    static_cast<uint16_t *>(p.out)[m * p.N + n + r] = to16(y, p.bf16);
  }
}

template <int XB, int TR, int FT, int W, int D, int STEPS, bool TAIL, bool GATED>
int launch_ring(const MxArgs &p, hipStream_t st) {
  using S = RingShape<XB, TR, FT, W, D, STEPS, TAIL>;
  static_assert(S::kLds <= kLdsBytes, "");
  auto kern = mx_ring_kernel<XB, TR, FT, W, D, STEPS, TAIL, GATED>;
  if (int rc = prepare(kern, S::kLds)) return rc;
  const int per_cu = kLdsBytes / S::kLds < 16 / W ? kLdsBytes / S::kLds : 16 / W;
  const int64_t tiles = (p.N + p.width - 1) / p.width, slots = static_cast<int64_t>(num_cus()) * per_cu;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tiles < slots ? tiles : slots)), dim3(64 * W), S::kLds, st, p);
  return check_launch();
}

// (2^31 threads per launch: rows beyond are further launches, which follow each other and share the memory of the parts' sums)
template <int XB, int RM, int RN, int WM, int WN, bool GATED>
int launch_tile(const MxArgs &p, hipStream_t st) {
  using S = TileShape<XB, RM, RN, WM, WN>;
  static_assert(S::kLds <= kLdsBytes, "");
  auto kern = mx_tile_kernel<XB, RM, RN, WM, WN, GATED>;
  if (int rc = prepare(kern, S::kLds)) return rc;
  constexpr int kCols = GATED ? S::kBN / 2 : S::kBN;
  const int64_t across = (p.N + kCols - 1) / kCols * p.splits, most = INT32_MAX / (S::kW * 64) / across * S::kBM;
  if (most == 0) return QUIK_ERR_RANGE;
  for (int64_t m = 0; m < p.M; m += most) {
    MxArgs q = p;
    q.M = p.M - m < most ? p.M - m : most;
    q.x = p.x + m * p.K * XB / 8;
    q.xs = p.xs + m * (p.K / kMxBlock);
    if (p.row) q.row = p.row + m;
    q.out = static_cast<uint8_t *>(p.out) + (GATED ? m * p.N * p.q_bits / 8 : m * p.N * 2);
    if (GATED) q.out_scale = p.out_scale + m * (p.N / kMxBlock);
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((q.M + S::kBM - 1) / S::kBM * across)), dim3(64 * S::kW), S::kLds, st, q);
    if (int rc = check_launch()) return rc;
    if (p.splits > 1) {
      hipLaunchKernelGGL(mx_join_kernel, dim3(static_cast<unsigned>((q.M * ((p.N + 3) / 4) + 255) / 256)), dim3(256), 0, st, q);
      if (int rc = check_launch()) return rc;
    }
  }
  return QUIK_OK;
}

// Result columns per workgroup of the kernel of few rows: the rounds that all CUs need with FT matrix tiles side by side, and the columns of a round
// dealt to them evenly.
int deal_columns(int64_t N, int ft) {
  const int64_t cus = num_cus(), most = 16 * ft, rounds = ((N + most - 1) / most + cus - 1) / cus;
  return static_cast<int>((N + rounds * cus - 1) / (rounds * cus));
}

int tiles_side_by_side(int64_t N) { return N > 16 * num_cus() ? 2 : 1; }
// Two matrix tiles side by side where one would leave a second round of workgroups; then four waves with two blocks under way, not eight with one
// (us: 1 x 8192 -> 28672 24.7, 25.4; 1 x 13824 -> 5120 8.8, 8.9; 16 rows of it 10.2, 10.4), but for up to eight rows of 8 bits, whose waves take their
// codes apart meanwhile (1 x 8192 -> 28672 30.2, 27.3).  Gated the ring of two is the better one (1 x 5120 -> 27648 17.6, 20.5), and with one
// tile (1 x 4096 -> 4096 4.2, 4.6).
template <int XB, bool TAIL>
int few_rows(MxArgs p, hipStream_t st) {
  const int ft = tiles_side_by_side(p.N);
  p.width = deal_columns(p.N, ft);
  if (p.M <= 8) {
    if (ft == 2) return launch_ring<XB, 8, 2, (XB == 8 ? 8 : 4), (XB == 8 ? 2 : 3), 2, TAIL, false>(p, st);
    return launch_ring<XB, 8, 1, 8, 2, 2, TAIL, false>(p, st);
  }
  if (p.M <= 16) {
    if (ft == 2) return launch_ring<XB, 16, 2, 4, 3, 2, TAIL, false>(p, st);
    return launch_ring<XB, 16, 1, 4, 2, 2, TAIL, false>(p, st);
  }
  if (ft == 2) return launch_ring<XB, 32, 2, 4, (XB == 8 ? 2 : 3), 2, TAIL, false>(p, st);
  return launch_ring<XB, 32, 1, 4, 2, 2, TAIL, false>(p, st);
}
constexpr int kFewGated = 16;  // rows of a gated product that the kernel of few rows takes
template <int XB, bool TAIL>
int few_rows_gated(MxArgs p, hipStream_t st) {
  p.width = kMxBlock;
  if (p.M <= 8) return launch_ring<XB, 8, 4, 4, 2, 2, TAIL, true>(p, st);
  return launch_ring<XB, 16, 4, 4, 2, 2, TAIL, true>(p, st);
}

// Tiles of more than 16 rows, for 4- and for 8-bit rows: rows, columns, workgroups that a CU takes at a time, the time of a stage of 256 columns with
// one of them and with all, and what a workgroup takes besides, in us.
struct TilePlan {
  int rows, cols, slots;
  double one, full, round;
};
constexpr TilePlan kPlans[2][4] = {{{32, 128, 3, 0.5, 1.2, 2.0}, {64, 128, 2, 0.58, 0.98, 2.0}, {128, 128, 2, 0.76, 1.5, 2.0}, {256, 256, 1, 1.75, 2.0, 5.0}},
                                   {{32, 128, 2, 0.85, 1.5, 2.0}, {64, 128, 2, 1.08, 1.8, 2.0}, {128, 128, 1, 1.6, 1.65, 2.0}, {128, 256, 1, 2.35, 2.8, 4.0}}};
struct Choice {
  int plan, splits;
  double us;
};
// The cheapest tiles and K split: the rounds of workgroups, no less than the weights from memory (of whose rate each CU has its share), and for a split the
// second launch and its sums, written and read (from the cache that all dies share); a part is four stages at least (64 x 4096 -> 4096, in parts of two 14.5,
// of four 11.1).  us, as the rule has it and measured (the next best measured):
// 64 x 13824 -> 5120, 64 rows, K in 6, 16.8, 16.2 (32 rows, K in 3: 18.5); 64 x 8192 -> 8192, 64 rows, K in 4, 16.4, 15.5 (32 rows, K in 2: 16.8); 32 x 28672 -> 8192, 32 rows, K in
// 4, 33.1, 29.6 (in 3, 192 workgroups: 42.2); 64 x 4096 -> 11008, 32 rows, 12.5, 9.9 (64 rows 13.0); 128 x 5120 -> 13824, 64 rows, 16.1, 17.2 (128 rows 22.2); 300 x 4544 -> 4544,
// 64 rows, 14.9, 13.7 (128 rows 18.1); 300 x 13824 -> 5120, 128 rows, K in 2, 31.9, 31.3 (64 rows 37.6); 777 x 5120 -> 5120, 128 rows, 34.5, 28.8 (64 rows 33.6); 2048 x 8192 ->
// 28672, 256 rows, 270.5, 275 (128 rows 333), 24576 columns 209.5, 220, 8192 x 8192 -> 8192 278.5, 282.  8 bit: 300 x 4544 -> 4544, 64 rows, 23.9, 22.6 (128 rows 29.0); 300 x 13824 ->
// 5120, 128 x 256, K in 4, 49.7, 51.9 (128 x 128 55.7); 777 x 5120 -> 5120, 128 x 256, 53.5, 51.5 (64 rows 58.7); 1024 x 4096 -> 4096, 128 x 128, 30.9, 31.6 (64 rows 36.3); 2048 x
// 8192 -> 28672, 128 x 256, 657.7, 637 (128 x 128 757).
Choice choose(int64_t M, int64_t N, int64_t K, int x_bits, bool may_split) {
  Choice best{1, 1, 1e30};
  const int64_t cus = num_cus(), stages = (K + 255) / 256;
  const double weights = static_cast<double>(N) * static_cast<double>(K) * 0.53125 / 5.0e6;
  for (int i = 0; i < 4; ++i) {
    const TilePlan &t = kPlans[x_bits == 8][i];
    const int64_t tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols);
    for (int s = 1; s <= (may_split ? 16 : 1) && (s == 1 || 4 * s <= stages); ++s) {
      const int64_t groups = tiles * s, rounds = groups / (cus * t.slots), rest = groups % (cus * t.slots), deep = (stages + s - 1) / s;
      double us = static_cast<double>(rounds) * (static_cast<double>(deep) * t.full + t.round);
      if (rest) us += static_cast<double>(deep) * (rest <= cus ? t.one : t.full) + t.round;
      const double share = 1.05 * static_cast<double>(groups) / static_cast<double>(cus), stream = weights / (share < 1.0 ? share : 1.0) + 1.0;
      us = (us > stream ? us : stream) + 2.5 + (s > 1 ? 3.5 + static_cast<double>(s) * static_cast<double>(M) * static_cast<double>(N) * 1.1e-6 : 0.0);
      if (us < best.us) best = Choice{i, s, us};
    }
  }
  return best;
}
// Up to 16 rows take the kernel of few rows, up to 32 where that is quicker: each CU takes the rows of its tiles' columns and all token rows through direct
// copies, 32 bytes per ns of them and 3 us beside.  us, as the rule has it and measured (tiles): 24 x 4096 -> 4096 6.3, 4.9 (8.7), 17 x 13824 -> 5120 14.9, 11.1 (13.6), 24 x 5120 ->
// 13824 13.0, 12.3 (17.3), 32 x 8192 -> 28672 35.6, 36 (27.4), 24 x 28672 -> 8192 33.5, 30.0 (28.6); 8 bit: 24 x 4096 -> 4096 8.3, 6.6 (10.1), 32 x 4096 -> 11008 14.4, 13.9 (15.8), 32 x 13824 ->
// 5120 21.8, 18.8 (16.5).  (Gated, tiles of 32 results: 20 x 4096 -> 22016 19.0, tiles 15.3: up to 16 rows only.)
bool by_ring(int64_t M, int64_t N, int64_t K, int x_bits) {
  if (M <= 16) return true;
  if (M > 32) return false;
  const int ft = tiles_side_by_side(N), width = deal_columns(N, ft);
  const int64_t tiles = (N + width - 1) / width, rounds = (tiles + num_cus() - 1) / num_cus();
  const double bytes = static_cast<double>(rounds * K) * (width * 0.53125 + 32 * (x_bits / 8.0 + 1.0 / 32));
  return 3.0 + bytes / 32e3 < choose(M, N, K, x_bits, true).us;
}
int64_t partial_bytes(int64_t M, int64_t N, int splits) { return splits > 1 ? splits * M * ((N + 3) / 4 * 4) * 4 : 0; }

// the choice of a call with that much memory for the parts' sums
Choice choose_within(int64_t M, int64_t N, int64_t K, int x_bits, int64_t workspace_bytes) {
  const Choice c = choose(M, N, K, x_bits, true);
  return workspace_bytes < partial_bytes(M, N, c.splits) ? choose(M, N, K, x_bits, false) : c;
}
// a gated product's, of `inner` results: K is not split, and tiles of 32 rows are those of 64
int choose_gated(int64_t M, int64_t inner, int64_t K, int x_bits) {
  const int plan = choose(M, 2 * inner, K, x_bits, false).plan;
  return plan == 0 ? 1 : plan;
}

template <int XB>
int many_rows(const MxArgs &p, int64_t workspace_bytes, hipStream_t st) {
  MxArgs q = p;
  const Choice c = choose_within(p.M, p.N, p.K, XB, p.partial ? workspace_bytes : 0);
  q.splits = c.splits;
  if (c.plan == 0) return launch_tile<XB, 1, 1, 1, 4, false>(q, st);
  if constexpr (XB == 8) {
    if (c.plan == 1) return launch_tile<8, 1, 2, 2, 2, false>(q, st);
    if (c.plan == 2) return launch_tile<8, 1, 4, 4, 1, false>(q, st);
    return launch_tile<8, 1, 4, 4, 2, false>(q, st);
  } else {
    if (c.plan == 1) return launch_tile<4, 2, 1, 1, 4, false>(q, st);
    if (c.plan == 2) return launch_tile<4, 2, 2, 2, 2, false>(q, st);
    return launch_tile<4, 4, 2, 2, 4, false>(q, st);
  }
}
template <int XB>
int many_rows_gated(const MxArgs &p, hipStream_t st) {
  MxArgs q = p;
  q.splits = 1;
  const int plan = choose_gated(p.M, p.N, p.K, XB);
  if (plan == 1) return launch_tile<XB, 1, 2, 2, 2, true>(q, st);
  if constexpr (XB == 8) {
    if (plan == 2) return launch_tile<8, 1, 4, 4, 1, true>(q, st);
    return launch_tile<8, 1, 4, 4, 2, true>(q, st);
  } else {
    if (plan == 2) return launch_tile<4, 2, 2, 2, 2, true>(q, st);
    return launch_tile<4, 4, 2, 2, 4, true>(q, st);
  }
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// what both products check
int check_product(const void *x, int x_bits, const uint8_t *xs, const uint8_t *w, const uint8_t *ws, const float *row, int dtype, int64_t M, int64_t N,
                  int64_t K, const void *out) {
  if (x_bits != 4 && x_bits != 8) return QUIK_ERR_BITS;
  if (dtype != QUIK_F16 && dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  if (M < 0 || N < 0 || K <= 0) return QUIK_ERR_SHAPE;
  if (K % kMxBlock) return QUIK_ERR_ALIGN;
  if (M > INT32_MAX || N > INT32_MAX / 2 || K > 1 << 20) return QUIK_ERR_RANGE;  // (offsets of a tile's rows in 32 bits)
  if (M == 0 || N == 0) return QUIK_OK;
  if (!x || !xs || !w || !ws || !out) return QUIK_ERR_NULL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(row, 4)) return QUIK_ERR_ALIGN;
  return QUIK_OK;
}
// exponent bytes by fours, or one by one where rows of them do not start at multiples of four or end inside a step
bool by_fours(const uint8_t *xs, const uint8_t *ws, int64_t K) { return K % 128 == 0 && aligned(xs, 4) && aligned(ws, 4); }
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int64_t quik_mx_matmul_workspace_bytes(int x_bits, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX / 2 || K > 1 << 20 || by_ring(M, N, K, x_bits)) return 0;
  return partial_bytes(M, N, choose(M, N, K, x_bits, true).splits);
}

extern "C" int quik_mx_matmul_tile(int x_bits, int gated, int64_t M, int64_t N, int64_t K, int64_t workspace_bytes) {
  if ((x_bits != 4 && x_bits != 8) || M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX / 2 || K > 1 << 20) return 0;
  if (gated ? M <= kFewGated : by_ring(M, N, K, x_bits)) {
    const int rows = M <= 8 ? 8 : M <= 16 ? 16 : 32;
    return rows << 12 | (gated ? kMxBlock : deal_columns(N, tiles_side_by_side(N)));
  }
  const Choice c = gated ? Choice{choose_gated(M, N, K, x_bits), 1, 0.0} : choose_within(M, N, K, x_bits, workspace_bytes);
  const TilePlan &t = kPlans[x_bits == 8][c.plan];
  return c.splits << 24 | t.rows << 12 | (gated ? t.cols / 2 : t.cols);
}

extern "C" int quik_mx_matmul(const void *x, int x_bits, const uint8_t *x_scale, const uint8_t *w, const uint8_t *w_scale, const float *scale_row,
                              const void *bias, int dtype, int64_t M, int64_t N, int64_t K, void *out, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  if (int rc = check_product(x, x_bits, x_scale, w, w_scale, scale_row, dtype, M, N, K, out)) return rc;
  if (M == 0 || N == 0) return QUIK_OK;
  if (!aligned(bias, 2) || !aligned(out, 2) || !aligned(workspace, 16)) return QUIK_ERR_ALIGN;
  const MxArgs p{static_cast<const uint8_t *>(x), x_scale, w, w_scale, scale_row, bias, out, nullptr, M, N, K, dtype == QUIK_BF16, 0, 0,
                 static_cast<float *>(workspace), 1};
  hipStream_t st = as_stream(stream);
  const bool fours = by_fours(x_scale, w_scale, K);
  if (by_ring(M, N, K, x_bits)) {
    if (x_bits == 4) return fours ? few_rows<4, false>(p, st) : few_rows<4, true>(p, st);
    return fours ? few_rows<8, false>(p, st) : few_rows<8, true>(p, st);
  }
  return x_bits == 4 ? many_rows<4>(p, workspace_bytes, st) : many_rows<8>(p, workspace_bytes, st);
}

extern "C" int quik_mx_gated_matmul(const void *x, int x_bits, const uint8_t *x_scale, const uint8_t *w, const uint8_t *w_scale, const float *scale_row,
                                    int dtype, int64_t M, int64_t inner, int64_t K, int q_bits, void *q, uint8_t *q_scale, void *stream) {
  if (q_bits != 4 && q_bits != 8) return QUIK_ERR_BITS;
  if (int rc = check_product(x, x_bits, x_scale, w, w_scale, scale_row, dtype, M, inner, K, q)) return rc;
  if (inner % kMxBlock) return QUIK_ERR_ALIGN;
  if (inner * (K / kMxBlock) > INT32_MAX) return QUIK_ERR_RANGE;  // (up's exponent bytes lie as far behind the gates')
  if (M == 0 || inner == 0) return QUIK_OK;
  if (!q_scale) return QUIK_ERR_NULL;
  const MxArgs p{static_cast<const uint8_t *>(x), x_scale, w, w_scale, scale_row, nullptr, q, q_scale, M, inner, K, dtype == QUIK_BF16, q_bits, 0, nullptr, 1};
  hipStream_t st = as_stream(stream);
  const bool fours = by_fours(x_scale, w_scale, K);
  if (M <= kFewGated) {
    if (x_bits == 4) return fours ? few_rows_gated<4, false>(p, st) : few_rows_gated<4, true>(p, st);
    return fours ? few_rows_gated<8, false>(p, st) : few_rows_gated<8, true>(p, st);
  }
  return x_bits == 4 ? many_rows_gated<4>(p, st) : many_rows_gated<8>(p, st);
}
