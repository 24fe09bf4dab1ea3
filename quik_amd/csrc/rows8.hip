// Rows of a decoder block in 8 bits: the two places where a block makes the input of its next product itself.
//   rms_norm  h = x + residual, rounded to the 16-bit type (and stored: it is the next residual; no residual: h = x)
//             u = h * gain;  value = u / sqrt(mean(h^2) + eps)
//   silu_mul  u = gate / (1 + exp(-gate)) * up;  value = u
// Output: q = rne(u * (127 / top)) with top = max |u| of the row, and scale = top / 127 (/ sqrt(mean(h^2) + eps)), so that
// value ~ q * scale.  The norm's factor is the same for a whole row and leaves the codes alone: largest magnitude and sum of
// squares come from the same single pass, and a norm's codes do not depend on the order of a sum.  u is exact in fp32 (products of
// 8 or 11 bits, down to its smallest number 2^-149); every other step of the norm is one IEEE operation in fp32.  A row of zeros has codes 0 and scale 0; a row that
// holds a NaN or an infinity, or whose sum of squares passes the range of fp32, has codes 0 and a NaN as its scale.
//
// Bound by memory where there are many rows: 4096 x 8192 bf16 with a residual 40 us (235 MB, 5.9 TB/s), 2048 x 28672 bf16 silu_mul 56 us (294 MB,
// 5.2 TB/s), a copy on this card 5.2.  One row is a chain of launch, one trip to memory, a reduction and a store: 2.4 us for 4096
// columns, 3.4 for 11008.  Hence a workgroup per row that holds it in registers, with nothing read twice.
#include "rows_math.h"

#include <type_traits>

namespace quik {
namespace {

struct RowArgs {
  const uint16_t *a, *b, *gain;  // norm: x, residual, gain; silu_mul: gate, up
  int64_t first, rows, cols, pitch_a, pitch_b;  // first: of this launch's rows
  float eps;
  uint16_t *sum;  // norm with a residual: h [rows, cols]
  int8_t *q;
  void *scale;  // of scale_type
  int scale_type;
};

// what is the same for the row: factor of the codes, scale
template <RowOp OP>
__device__ __forceinline__ void row_scale(uint32_t top_bits, float square, int64_t cols, float eps, float lift, float &pre, float &inv, float &scale) {
  const float top = __uint_as_float(top_bits);
  // (127 / top must not overflow, top / 127 not lose bits: rows of tiny numbers are made larger by a power of two first)
  pre = top < 0x1p-100f ? 0x1p100f : 1.0f;
  const bool bad = top_bits >= kInfBits || !(square < __builtin_inff());
  inv = bad || top_bits == 0 ? 0.0f : 127.0f / (top * pre);
  if constexpr (OP == kSiluMul) scale = top / 127.0f;
  else scale = top * pre / 127.0f * norm_factor(square, cols, eps, lift) * (pre == 1.0f ? lift : lift * 0x1p-100f);
  if (top_bits == 0) scale = 0.0f;  // (a row of zeros at an eps of 0 has no finite factor)
  if (bad) scale = __builtin_nanf("");
}

// (the codes go by the row's largest value, not by what a 16-bit scale rounds to: its half a step of 2^-11 or 2^-8 is in every
// value of the row alike)
__device__ __forceinline__ void store_scale(const RowArgs &p, int64_t row, float scale) {
  if (p.scale_type == QUIK_F32) static_cast<float *>(p.scale)[row] = scale;
  else static_cast<uint16_t *>(p.scale)[row] = p.scale_type == QUIK_BF16 ? from_f32<true>(scale) : from_f32<false>(scale);
}

// q in the low byte: |u * inv| <= 127 (1 + 2^-23), and adding 1.5 * 2^23 rounds to nearest even at 1
__device__ __forceinline__ uint32_t code_bits(float u, float inv) { return __float_as_uint(u * inv + 12582912.0f); }

// One row per workgroup of as many waves as it takes, held in registers: V chunks of eight columns per thread.  WIDE: rows are multiples of
// eight columns at 16-byte addresses; else the last chunk is as many columns as there are left.
template <bool BF16, RowOp OP, bool WIDE, int V>
__global__ __launch_bounds__(1024) void rows8_kernel(RowArgs p) {
  __shared__ uint32_t red[2 * 16];
  const int tid = threadIdx.x, T = static_cast<int>(blockDim.x);
  const int chunks = static_cast<int>((p.cols + 7) / 8), last = WIDE ? 8 : static_cast<int>(p.cols - (chunks - 1) * int64_t{8});
  const int64_t row = p.first + blockIdx.x;
  const uint16_t *a = p.a + row * p.pitch_a;
  const uint16_t *b = OP == kNorm ? nullptr : p.b + row * p.pitch_b;
  using Eight = std::conditional_t<WIDE, uint4, loose4>;
  // A thread reads a column before it writes it: the sum may lie where x or the residual lies.  So no load moves up past a store by itself,
  // and what is read of the row is requested in front of the first store where the registers allow it.  (Where there is no store the compiler
  // does better: all of 2048 x 28672 bf16 silu_mul first takes 66.5 us, half the workgroups per CU, so 54.9.)
  constexpr bool kFirst = OP == kNormAdd && V <= 2;
  alignas(16) uint16_t va[V][8], vb[V][8], vg[V][8];
  auto get = [&](int j) {
    const int c = tid + j * T;
    if (c >= chunks) return;
    if (WIDE || c < chunks - 1 || last == 8) {
      *reinterpret_cast<Eight *>(va[j]) = *reinterpret_cast<const Eight *>(a + c * int64_t{8});
      if constexpr (OP != kNorm) *reinterpret_cast<Eight *>(vb[j]) = *reinterpret_cast<const Eight *>(b + c * int64_t{8});
      if constexpr (OP != kSiluMul) *reinterpret_cast<Eight *>(vg[j]) = *reinterpret_cast<const Eight *>(p.gain + c * int64_t{8});
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // (zeros behind the end: they change neither maximum nor sum)
        const int64_t at = c * int64_t{8} + e;
        va[j][e] = e < last ? a[at] : 0;
        if constexpr (OP != kNorm) vb[j][e] = e < last ? b[at] : 0;
        if constexpr (OP != kSiluMul) vg[j][e] = e < last ? p.gain[at] : 0;
      }
    }
  };
  if constexpr (kFirst) {
#pragma unroll
    for (int j = 0; j < V; ++j) get(j);
  }
  float u[V][8];
  uint32_t top = 0;
  float square = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = tid + j * T;
    if (c < chunks) {
      if constexpr (!kFirst) get(j);
      alignas(16) uint16_t vh[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[j][e] = row_value<BF16, OP, false>(to_f32<BF16>(va[j][e]), OP == kNorm ? 0.0f : to_f32<BF16>(vb[j][e]), OP == kSiluMul ? 0.0f : to_f32<BF16>(vg[j][e]),
                                      vh[e], square);
      }
      if constexpr (OP == kSiluMul) {
        uint32_t low = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) low = umax(low, __float_as_uint(to_f32<BF16>(va[j][e])));
        if (low > kFarBits) {  // (us for 2048 x 28672 bf16: without 54.1, so 54.8, halves for all gates 58.4; 512 x 40000 in the kernel below 39.2, 41.7)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float gate = to_f32<BF16>(va[j][e]);
            if (__float_as_uint(gate) > kFarBits) u[j][e] = gated_far(gate, to_f32<BF16>(vb[j][e]));
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = umax(top, __float_as_uint(u[j][e]) & 0x7FFFFFFFu);
      }
      if constexpr (OP == kNormAdd) {
        uint16_t *s = p.sum + row * p.cols + c * int64_t{8};
        if (WIDE || c < chunks - 1 || last == 8) {
          *reinterpret_cast<Eight *>(s) = *reinterpret_cast<const Eight *>(vh);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < last) s[e] = vh[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[j][e] = 0.0f;
    }
  }
  block_reduce(top, square, red);
  float lift = 1.0f, pre, inv, scale;
  if (tiny_squares<BF16, OP>(top, square, p.cols, p.eps)) {
    const uint16_t *h = OP == kNormAdd ? p.sum + row * p.cols : a;  // (a thread's own columns: what it has written of the sum)
    lift = kLift;
    square = 0.0f;
    for (int64_t at = tid * int64_t{8}; at < p.cols; at += T * int64_t{8})
      for (int64_t c = at; c < at + 8 && c < p.cols; ++c) square += to_f32<BF16>(h[c]) * lift * (to_f32<BF16>(h[c]) * lift);
    block_sum(square, red);
  }
  row_scale<OP>(top, square, p.cols, p.eps, lift, pre, inv, scale);
  if (tid == 0) store_scale(p, row, scale);
  if (pre != 1.0f) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) u[j][e] *= pre;
  }
  if (inv == 0.0f) {  // (NaNs and infinities among the values: codes 0)
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) u[j][e] = 0.0f;
  }
  int8_t *q = p.q + row * p.cols;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = tid + j * T;
    if (c < chunks) {
      uint32_t w[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float *v = &u[j][4 * k];
        const uint32_t lo = __builtin_amdgcn_perm(code_bits(v[1], inv), code_bits(v[0], inv), 0x0C0C0400u);
        const uint32_t hi = __builtin_amdgcn_perm(code_bits(v[3], inv), code_bits(v[2], inv), 0x04000C0Cu);
        w[k] = lo | hi;
      }
      int8_t *to = q + c * int64_t{8};
      if (WIDE) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
      } else if (c < chunks - 1 || last == 8) {
        *reinterpret_cast<loose2 *>(to) = loose2{w[0], w[1]};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < last) to[e] = static_cast<int8_t>(w[e >> 2] >> (8 * (e & 3)));
      }
    }
  }
}

// Rows that no instance of the kernel above holds in registers: the row is read twice, the second time from the caches (with a residual, its
// sum: it may lie where x or the residual lies).
template <bool BF16, RowOp OP>
__global__ __launch_bounds__(1024) void rows8_long_kernel(RowArgs p) {
  __shared__ uint32_t red[2 * 16];
  const int64_t row = p.first + blockIdx.x;
  const uint16_t *a = p.a + row * p.pitch_a;
  const uint16_t *b = OP == kNorm ? nullptr : p.b + row * p.pitch_b;
  uint16_t *sum = OP == kNormAdd ? p.sum + row * p.cols : nullptr;
  uint32_t top = 0;
  float square = 0.0f;
  for (int64_t c = threadIdx.x; c < p.cols; c += 1024) {
    uint16_t h = 0;
    const float u = row_value<BF16, OP, true>(to_f32<BF16>(a[c]), OP == kNorm ? 0.0f : to_f32<BF16>(b[c]), OP == kSiluMul ? 0.0f : to_f32<BF16>(p.gain[c]), h, square);
    top = umax(top, __float_as_uint(u) & 0x7FFFFFFFu);
    if constexpr (OP == kNormAdd) sum[c] = h;
  }
  block_reduce(top, square, red);
  float lift = 1.0f, pre, inv, scale;
  if (tiny_squares<BF16, OP>(top, square, p.cols, p.eps)) {
    const uint16_t *h = OP == kNormAdd ? sum : a;  // (a thread's own columns: what it has written of the sum)
    lift = kLift;
    square = 0.0f;
    for (int64_t c = threadIdx.x; c < p.cols; c += 1024) square += to_f32<BF16>(h[c]) * lift * (to_f32<BF16>(h[c]) * lift);
    block_sum(square, red);
  }
  row_scale<OP>(top, square, p.cols, p.eps, lift, pre, inv, scale);
  if (threadIdx.x == 0) store_scale(p, row, scale);
  for (int64_t c = threadIdx.x; c < p.cols; c += 1024) {  // (a thread's own columns: what it has written of the sum)
    uint16_t h = 0;
    float unused = 0.0f;
    constexpr RowOp kAgain = OP == kNormAdd ? kNorm : OP;
    const float u = row_value<BF16, kAgain, true>(to_f32<BF16>(OP == kNormAdd ? sum[c] : a[c]), OP == kSiluMul ? to_f32<BF16>(b[c]) : 0.0f,
                                            OP == kSiluMul ? 0.0f : to_f32<BF16>(p.gain[c]), h, unused);
    p.q[row * p.cols + c] = inv == 0.0f ? int8_t{0} : static_cast<int8_t>(code_bits(u * pre, inv) & 0xFFu);
  }
}

template <bool BF16, RowOp OP>
int launch_rows(const RowArgs &p, int64_t rows, bool wide, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows));
  // Chunks per thread: one where a row's time is a chain of latencies, more where many rows' memory is what takes the time.  us with one, two
  // and four: 1 x 4096 fp16 with a residual 3.2, 3.4, 3.75; 777 x 5120 fp16 5.9, 5.1, 5.3; 4096 x 8192 bf16 with a residual 43.8, 40.1, 38.6.
  const int64_t chunks = (p.cols + 7) / 8, cus = num_cus();
  const int v = rows > 8 * cus || chunks > 2048 ? 4 : rows > cus || chunks > 1024 ? 2 : 1;
#define QUIK_ROWS(WIDE, V) hipLaunchKernelGGL((rows8_kernel<BF16, OP, WIDE, V>), grid, dim3(static_cast<unsigned>((chunks + 64 * V - 1) / (64 * V) * 64)), 0, st, p)
  if (chunks > 4096) hipLaunchKernelGGL((rows8_long_kernel<BF16, OP>), grid, dim3(1024), 0, st, p);
  else if (wide && v == 1) QUIK_ROWS(true, 1);
  else if (wide && v == 2) QUIK_ROWS(true, 2);
  else if (wide) QUIK_ROWS(true, 4);
  else if (v == 1) QUIK_ROWS(false, 1);
  else if (v == 2) QUIK_ROWS(false, 2);
  else QUIK_ROWS(false, 4);
#undef QUIK_ROWS
  return check_launch();
}

// 2^20 rows per launch (a grid has less than 2^32 threads).  A loop over rows in the kernel costs registers: 2048 x 28672 bf16 silu_mul 55
// -> 61.5 us.
template <bool BF16, RowOp OP>
int launch(RowArgs p, bool wide, hipStream_t st) {
  for (; p.first < p.rows; p.first += 1 << 20)
    if (int rc = launch_rows<BF16, OP>(p, p.rows - p.first < 1 << 20 ? p.rows - p.first : 1 << 20, wide, st)) return rc;
  return QUIK_OK;
}

template <RowOp OP>
int launch_typed(const RowArgs &p, int dtype, bool wide, hipStream_t st) {
  return dtype == QUIK_BF16 ? launch<true, OP>(p, wide, st) : launch<false, OP>(p, wide, st);
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// sizes that both operations check: rows in one grid, offsets of a row's elements in 63 bits
int check_rows(int dtype, int scale_type, int64_t rows, int64_t cols, int64_t pitch_a, int64_t pitch_b) {
  if (dtype != QUIK_F16 && dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  if (scale_type != QUIK_F16 && scale_type != QUIK_BF16 && scale_type != QUIK_F32) return QUIK_ERR_DTYPE;
  if (rows < 0 || cols <= 0 || (rows > 1 && (pitch_a < cols || pitch_b < cols))) return QUIK_ERR_SHAPE;
  if (rows > INT32_MAX || cols > INT32_MAX) return QUIK_ERR_RANGE;
  return QUIK_OK;
}
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int quik_rms_norm_quantize(const void *x, int64_t x_pitch, const void *residual, int64_t residual_pitch, const void *gain,
                                      float eps, int dtype, int64_t rows, int64_t cols, void *sum, int8_t *q, void *scale, int scale_type, void *stream) {
  if (int rc = check_rows(dtype, scale_type, rows, cols, x_pitch, residual ? residual_pitch : cols)) return rc;
  if (!(eps >= 0.0f)) return QUIK_ERR_RANGE;
  if (rows == 0) return QUIK_OK;
  if (!x || !gain || !q || !scale || (residual && !sum)) return QUIK_ERR_NULL;
  if (!aligned(x, 2) || !aligned(residual, 2) || !aligned(gain, 2) || !aligned(sum, 2) || !aligned(scale, scale_type == QUIK_F32 ? 4 : 2)) return QUIK_ERR_ALIGN;
  const RowArgs p{static_cast<const uint16_t *>(x), static_cast<const uint16_t *>(residual), static_cast<const uint16_t *>(gain), 0, rows, cols,
                  x_pitch, residual_pitch, eps, static_cast<uint16_t *>(sum), q, scale, scale_type};
  const bool wide = cols % 8 == 0 && aligned(x, 16) && aligned(gain, 16) && aligned(q, 8) && (rows == 1 || x_pitch % 8 == 0) &&
                    (!residual || (aligned(residual, 16) && aligned(sum, 16) && (rows == 1 || residual_pitch % 8 == 0)));
  return residual ? launch_typed<kNormAdd>(p, dtype, wide, as_stream(stream)) : launch_typed<kNorm>(p, dtype, wide, as_stream(stream));
}

extern "C" int quik_silu_mul_quantize(const void *gate, int64_t gate_pitch, const void *up, int64_t up_pitch, int dtype, int64_t rows,
                                      int64_t cols, int8_t *q, void *scale, int scale_type, void *stream) {
  if (int rc = check_rows(dtype, scale_type, rows, cols, gate_pitch, up_pitch)) return rc;
  if (rows == 0) return QUIK_OK;
  if (!gate || !up || !q || !scale) return QUIK_ERR_NULL;
  if (!aligned(gate, 2) || !aligned(up, 2) || !aligned(scale, scale_type == QUIK_F32 ? 4 : 2)) return QUIK_ERR_ALIGN;
  const RowArgs p{static_cast<const uint16_t *>(gate), static_cast<const uint16_t *>(up), nullptr, 0, rows, cols, gate_pitch, up_pitch, 0.0f,
                  nullptr, q, scale, scale_type};
  const bool wide = cols % 8 == 0 && aligned(gate, 16) && aligned(up, 16) && aligned(q, 8) &&
                    (rows == 1 || (gate_pitch % 8 == 0 && up_pitch % 8 == 0));
  return launch_typed<kSiluMul>(p, dtype, wide, as_stream(stream));
}
