// Rows in blocks of 32 (mx_format.h), made where they arise, and read back:
//   quantize   value = x
//   silu_mul   value = gate / (1 + exp(-gate)) * up
//   rms_norm   h = x + residual, rounded to the 16-bit type (and stored: it is the next residual; no residual: h = x), u = h * gain (exact in
//              fp32); the codes are those of u, and the row's factor 1 / sqrt(mean(h^2) + eps) is an fp32 number beside them, which the product
//              applies to its sums: a block's power of two could not hold it, and so no code depends on the order of a sum
//   dequantize 16-bit numbers of codes, of all rows or of those that a list names (a cache's slots)
//
// All are bound by memory.  A block is four lanes of eight columns, 16 bytes of a 16-bit row each, and its largest magnitude two exchanges between
// neighbouring lanes: there is nothing to wait for but the load, and a norm stores its codes before it knows the row's factor.
// us, bytes per us against a copy's 5.1e6: quantize 2048 x 8192, 4 bits, 9.3, 4.6e6; silu_mul 2048 x 13824, 8 bits, 26.3, 5.4e6; norm with a residual 777 x 5120, 4 bits,
// 7.4, 3.5e6 (one row per workgroup, all at once: loads, then stores), 8192 x 4096 37.3, 5.9e6; dequantize 32768 rows of 8 x 128, 8 bits, 18.6, 5.4e6.
#include "mx_format.h"

namespace quik {
namespace {

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

struct MxRows {
  const uint16_t *a, *b, *gain;  // quantize: a; silu_mul: gate, up; rms_norm: x, residual, gain
  int64_t rows, cols, pitch_a, pitch_b;
  float eps;
  uint16_t *sum;   // rms_norm with a residual: h [rows, cols]
  uint8_t *q;      // [rows, cols / 2] or [rows, cols]
  uint8_t *scale;  // [rows, blocks]
  float *factor;   // rms_norm: [rows]
  Divide by_lanes;  // lanes of a row: four per block
};

enum FlatOp { kPlain, kGated };

// Lanes of all rows one after the other, one each: chunks of several per thread, requested together, take longer (us, four per thread and this: quantize
// 2048 x 8192, 4 bits, 10.7, 9.3 (4.6 TB/s, a copy's are 5.1), 8192 x 4096 19.5, 17.2; two and this: silu_mul 2048 x 13824, 8 bits, 28.6, 26.3 (5.4 TB/s)).
// (rows * lanes < 2^31 per launch)
template <bool BF16, FlatOp OP, int BITS, bool WIDE>
__global__ __launch_bounds__(256) void mx_flat_kernel(MxRows p) {
  const uint32_t at = blockIdx.x * 256u + threadIdx.x, all = static_cast<uint32_t>(p.rows) * p.by_lanes.d, blocks = p.by_lanes.d / 4;
  uint32_t c;
  const uint32_t row = p.by_lanes(at < all ? at : 0, c);
  const int64_t rest = p.cols - static_cast<int64_t>(c) * 8;
  const int left = at >= all ? 0 : rest < 8 ? static_cast<int>(rest) : 8;
  alignas(16) uint16_t va[8] = {}, vb[8] = {};
  if (left > 0) {
    load_eight<WIDE>(p.a + row * p.pitch_a + c * int64_t{8}, left, va);
    if constexpr (OP == kGated) load_eight<WIDE>(p.b + row * p.pitch_b + c * int64_t{8}, left, vb);
  }
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = OP == kGated ? gated(to_f32<BF16>(va[e]), to_f32<BF16>(vb[e])) : to_f32<BF16>(va[e]);
  if constexpr (OP == kGated) {
    uint32_t low = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) low = umax(low, __float_as_uint(to_f32<BF16>(va[e])));
    if (low > kFarBits) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gate = to_f32<BF16>(va[e]);
        if (__float_as_uint(gate) > kFarBits) v[e] = gated_far(gate, to_f32<BF16>(vb[e]));
      }
    }
  }
  store_block<BITS, WIDE>(v, left, p.q + (row * p.cols + c * int64_t{8}) * BITS / 8, p.scale + row * static_cast<int64_t>(blocks) + c / 4, c % 4 == 0);
}

template <bool BF16, bool ADD, int BITS, bool WIDE>
__global__ __launch_bounds__(1024) void mx_norm_kernel(MxRows p) {
  __shared__ uint32_t red[2 * 16];
  const int64_t row = blockIdx.x;
  const uint16_t *a = p.a + row * p.pitch_a;
  const uint16_t *b = ADD ? p.b + row * p.pitch_b : nullptr;
  uint16_t *sum = ADD ? p.sum + row * p.cols : nullptr;
  const uint32_t lanes = p.by_lanes.d, T = blockDim.x;
  float square = 0.0f;
  for (uint32_t c = threadIdx.x; c < lanes; c += T) {
    const int64_t rest = p.cols - static_cast<int64_t>(c) * 8;
    const int left = rest < 8 ? static_cast<int>(rest) : 8;
    alignas(16) uint16_t va[8] = {}, vb[8] = {}, vg[8] = {}, vh[8] = {};
    if (left > 0) {
      load_eight<WIDE>(a + c * int64_t{8}, left, va);
      if constexpr (ADD) load_eight<WIDE>(b + c * int64_t{8}, left, vb);
      load_eight<WIDE>(p.gain + c * int64_t{8}, left, vg);
    }
    float u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      u[e] = row_value<BF16, ADD ? kNormAdd : kNorm, false>(to_f32<BF16>(va[e]), to_f32<BF16>(vb[e]), to_f32<BF16>(vg[e]), vh[e], square);
    if constexpr (ADD)
      if (left > 0) store_eight<WIDE>(sum + c * int64_t{8}, left, vh);
    store_block<BITS, WIDE>(u, left, p.q + (row * p.cols + c * int64_t{8}) * BITS / 8, p.scale + row * static_cast<int64_t>(lanes / 4) + c / 4, c % 4 == 0);
  }
  uint32_t none = 0;
  block_reduce(none, square, red);
  float lift = 1.0f;
  if (tiny_squares<BF16, kNorm>(1, square, p.cols, p.eps)) {
    const uint16_t *h = ADD ? sum : a;  // (a thread's own columns: what it has written of the sum)
    lift = kLift;
    square = 0.0f;
    for (uint32_t c = threadIdx.x; c < lanes; c += T)
      for (int64_t at = c * int64_t{8}; at < c * int64_t{8} + 8 && at < p.cols; ++at) square += to_f32<BF16>(h[at]) * lift * (to_f32<BF16>(h[at]) * lift);
    block_sum(square, red);
  }
  if (threadIdx.x == 0) {
    float f = norm_factor(square, p.cols, p.eps, lift) * lift;
    if (square == 0.0f && p.eps == 0.0f) f = 0.0f;  // (a row of zeros has no finite factor then)
    if (!(square < __builtin_inff())) f = __builtin_nanf("");
    p.factor[row] = f;
  }
}

struct MxRead {
  const uint8_t *q, *scale;
  const int64_t *index;
  const float *factor;
  int64_t source_rows, heads, cols, count;  // count: rows of the result
  uint16_t *out;
  Divide by_lanes, by_heads;  // lanes (eight columns) of a vector
};

// (count * heads * lanes < 2^31 per launch)
template <bool BF16, int BITS, bool WIDE, int V>
__global__ __launch_bounds__(256) void mx_read_kernel(MxRead p) {
  const uint32_t first = blockIdx.x * (256u * V) + threadIdx.x, all = static_cast<uint32_t>(p.count * p.heads) * p.by_lanes.d;
  const int64_t blocks = (p.cols + kMxBlock - 1) / kMxBlock;
  uint2 w[V];
  uint32_t byte[V], vec[V], c[V];
  float factor[V];
  int left[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const uint32_t at = first + 256u * j;
    vec[j] = p.by_lanes(at < all ? at : 0, c[j]);
    const int64_t rest = p.cols - static_cast<int64_t>(c[j]) * 8;
    left[j] = at >= all ? 0 : rest < 8 ? static_cast<int>(rest) : 8;
    uint32_t head;
    const uint32_t row = p.by_heads(vec[j], head);
    const int64_t source = p.index ? p.index[row] : row;
    factor[j] = p.factor && left[j] > 0 ? p.factor[row] : 1.0f;
    w[j] = make_uint2(0, 0);
    byte[j] = 0;
    if (left[j] > 0 && source >= 0 && source < p.source_rows) {
      const int64_t from = source * p.heads + head;
      byte[j] = p.scale[from * blocks + c[j] / 4];
      const uint8_t *q = p.q + (from * p.cols + c[j] * int64_t{8}) * BITS / 8;
      if constexpr (BITS == 4) {
        if constexpr (WIDE) w[j].x = *reinterpret_cast<const uint32_t *>(q);
        else if (left[j] == 8) w[j].x = *reinterpret_cast<const mx_loose1 *>(q);
        else
          for (int e = 0; 2 * e < left[j]; ++e) w[j].x |= static_cast<uint32_t>(q[e]) << (8 * e);
      } else {
        if constexpr (WIDE) {
          w[j] = *reinterpret_cast<const uint2 *>(q);
        } else if (left[j] == 8) {
          const loose2 t = *reinterpret_cast<const loose2 *>(q);
          w[j] = make_uint2(t[0], t[1]);
        } else {
          for (int e = 0; e < left[j]; ++e) (e < 4 ? w[j].x : w[j].y) |= static_cast<uint32_t>(q[e]) << (8 * (e & 3));
        }
      }
    } else {
      factor[j] = 1.0f;  // (a row that is not there: zeros)
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (left[j] <= 0) continue;
    float v[8];
    decode8<BITS>(w[j], byte[j], v);
    alignas(16) uint16_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = from_f32<BF16>(p.factor ? v[e] * factor[j] : v[e]);
    store_eight<WIDE>(p.out + (vec[j] * p.cols + c[j] * int64_t{8}), left[j], h);
  }
}

constexpr int64_t kLanes = INT32_MAX - 4096;  // per launch, with the last workgroup's overhang

int64_t lanes_of(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock * 4; }

template <bool BF16, FlatOp OP, int BITS>
int launch_flat(MxRows p, bool wide, hipStream_t st) {
  const int64_t lanes = lanes_of(p.cols), most = kLanes / lanes, all = p.rows;
  p.by_lanes = divide_by(lanes);
  for (int64_t first = 0; first < all; first += most) {
    p.rows = all - first < most ? all - first : most;
    const dim3 grid(static_cast<unsigned>((p.rows * lanes + 255) / 256));
    if (wide) hipLaunchKernelGGL((mx_flat_kernel<BF16, OP, BITS, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((mx_flat_kernel<BF16, OP, BITS, false>), grid, dim3(256), 0, st, p);
    if (int rc = check_launch()) return rc;
    p.a += most * p.pitch_a;
    if (p.b) p.b += most * p.pitch_b;
    p.q += most * p.cols * BITS / 8;
    p.scale += most * (lanes / 4);
  }
  return QUIK_OK;
}

template <bool BF16, bool ADD, int BITS>
int launch_norm(MxRows p, bool wide, hipStream_t st) {
  const int64_t lanes = lanes_of(p.cols), all = p.rows, most = 1 << 20;
  p.by_lanes = divide_by(lanes);
  // One chunk per thread where so all rows run at once (2048 threads per CU); else two, one after the other (us, one and two: 777 x 5120 8.1, 7.4,
  // 2048 x 8192 20.3, 19.1; 64 x 5120, which fits, 3.8, 4.3); two or four requested together gain nothing: 777 x 5120 8.2, 8.4, 8.9, 300 x 28672 13.5, 15.6, 17.3.
  const int64_t one = (lanes + 63) / 64 * 64, two = ((lanes + 1) / 2 + 63) / 64 * 64;
  const int64_t threads = lanes > 1024 ? 1024 : all > num_cus() * (2048 / one) ? two : one;
  for (int64_t first = 0; first < all; first += most) {
    p.rows = all - first < most ? all - first : most;
    const dim3 grid(static_cast<unsigned>(p.rows)), block(static_cast<unsigned>(threads));
    if (wide) hipLaunchKernelGGL((mx_norm_kernel<BF16, ADD, BITS, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((mx_norm_kernel<BF16, ADD, BITS, false>), grid, block, 0, st, p);
    if (int rc = check_launch()) return rc;
    p.a += most * p.pitch_a;
    if (ADD) {
      p.b += most * p.pitch_b;
      p.sum += most * p.cols;
    }
    p.q += most * p.cols * BITS / 8;
    p.scale += most * (lanes / 4);
    p.factor += most;
  }
  return QUIK_OK;
}

template <bool BF16, int BITS>
int launch_read(MxRead p, bool wide, hipStream_t st) {
  constexpr int V = 4;
  const int64_t lanes = (p.cols + 7) / 8, most = kLanes / (p.heads * lanes), all = p.count;
  if (most == 0) return QUIK_ERR_RANGE;
  p.by_lanes = divide_by(lanes);
  p.by_heads = divide_by(p.heads);
  for (int64_t first = 0; first < all; first += most) {
    p.count = all - first < most ? all - first : most;
    const int64_t total = p.count * p.heads * lanes;
    // Four chunks per thread for the largest calls: us, one and four, 32768 rows of 8 x 128, 8 bits, 19.1, 18.6 (101 MB, 5.4 TB/s of which codes still
    // lie in the cache), 4096 of 40 x 128, 4 bits, 12.4, 12.0; below one spreads the lanes over more CUs, 2048 x 8192, 4 bits, 9.9, 10.4, 777 x 5120 4.7, 5.2.
    const bool few = total <= num_cus() * int64_t{256} * 32;
    const dim3 grid(static_cast<unsigned>((total + 256 * (few ? 1 : V) - 1) / (256 * (few ? 1 : V))));
    if (wide && few) hipLaunchKernelGGL((mx_read_kernel<BF16, BITS, true, 1>), grid, dim3(256), 0, st, p);
    else if (wide) hipLaunchKernelGGL((mx_read_kernel<BF16, BITS, true, V>), grid, dim3(256), 0, st, p);
    else if (few) hipLaunchKernelGGL((mx_read_kernel<BF16, BITS, false, 1>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((mx_read_kernel<BF16, BITS, false, V>), grid, dim3(256), 0, st, p);
    if (int rc = check_launch()) return rc;
    if (p.index) {
      p.index += most;
    } else {
      p.q += most * p.heads * p.cols * BITS / 8;
      p.scale += most * p.heads * ((p.cols + kMxBlock - 1) / kMxBlock);
      p.source_rows -= most;
    }
    if (p.factor) p.factor += most;
    p.out += most * p.heads * p.cols;
  }
  return QUIK_OK;
}

int check_sizes(int dtype, int bits, int64_t rows, int64_t cols, int64_t pitch_a, int64_t pitch_b) {
  if (bits != 4 && bits != 8) return QUIK_ERR_BITS;
  if (dtype != QUIK_F16 && dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  if (rows < 0 || cols <= 0 || (rows > 1 && (pitch_a < cols || pitch_b < cols))) return QUIK_ERR_SHAPE;
  if (bits == 4 && cols % 2) return QUIK_ERR_ALIGN;
  if (rows > INT32_MAX || cols > 1 << 30) return QUIK_ERR_RANGE;
  return QUIK_OK;
}
bool wide_row(const void *p, int64_t rows, int64_t pitch) { return aligned(p, 16) && (rows == 1 || pitch % 8 == 0); }

#define QUIK_BY_TYPE(CALL)                                                                   \
  (dtype == QUIK_BF16 ? (bits == 4 ? CALL(true, 4) : CALL(true, 8)) : (bits == 4 ? CALL(false, 4) : CALL(false, 8)))
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int quik_mx_quantize(const void *x, int64_t x_pitch, int dtype, int64_t rows, int64_t cols, int bits, void *q, uint8_t *scale, void *stream) {
  if (int rc = check_sizes(dtype, bits, rows, cols, x_pitch, cols)) return rc;
  if (rows == 0) return QUIK_OK;
  if (!x || !q || !scale) return QUIK_ERR_NULL;
  if (!aligned(x, 2)) return QUIK_ERR_ALIGN;
  MxRows p{};
  p.a = static_cast<const uint16_t *>(x), p.rows = rows, p.cols = cols, p.pitch_a = x_pitch, p.q = static_cast<uint8_t *>(q), p.scale = scale;
  const bool wide = cols % 8 == 0 && wide_row(x, rows, x_pitch) && aligned(q, 8);
#define QUIK_CALL(BF16, BITS) launch_flat<BF16, kPlain, BITS>(p, wide, as_stream(stream))
  return QUIK_BY_TYPE(QUIK_CALL);
#undef QUIK_CALL
}

extern "C" int quik_mx_silu_mul_quantize(const void *gate, int64_t gate_pitch, const void *up, int64_t up_pitch, int dtype, int64_t rows, int64_t cols,
                                         int bits, void *q, uint8_t *scale, void *stream) {
  if (int rc = check_sizes(dtype, bits, rows, cols, gate_pitch, up_pitch)) return rc;
  if (rows == 0) return QUIK_OK;
  if (!gate || !up || !q || !scale) return QUIK_ERR_NULL;
  if (!aligned(gate, 2) || !aligned(up, 2)) return QUIK_ERR_ALIGN;
  MxRows p{};
  p.a = static_cast<const uint16_t *>(gate), p.b = static_cast<const uint16_t *>(up), p.rows = rows, p.cols = cols, p.pitch_a = gate_pitch;
  p.pitch_b = up_pitch, p.q = static_cast<uint8_t *>(q), p.scale = scale;
  const bool wide = cols % 8 == 0 && wide_row(gate, rows, gate_pitch) && wide_row(up, rows, up_pitch) && aligned(q, 8);
#define QUIK_CALL(BF16, BITS) launch_flat<BF16, kGated, BITS>(p, wide, as_stream(stream))
  return QUIK_BY_TYPE(QUIK_CALL);
#undef QUIK_CALL
}

extern "C" int quik_mx_rms_norm_quantize(const void *x, int64_t x_pitch, const void *residual, int64_t residual_pitch, const void *gain, float eps,
                                         int dtype, int64_t rows, int64_t cols, int bits, void *sum, void *q, uint8_t *scale, float *scale_row,
                                         void *stream) {
  if (int rc = check_sizes(dtype, bits, rows, cols, x_pitch, residual ? residual_pitch : cols)) return rc;
  if (!(eps >= 0.0f)) return QUIK_ERR_RANGE;
  if (rows == 0) return QUIK_OK;
  if (!x || !gain || !q || !scale || !scale_row || (residual && !sum)) return QUIK_ERR_NULL;
  if (!aligned(x, 2) || !aligned(residual, 2) || !aligned(gain, 2) || !aligned(sum, 2) || !aligned(scale_row, 4)) return QUIK_ERR_ALIGN;
  MxRows p{};
  p.a = static_cast<const uint16_t *>(x), p.b = static_cast<const uint16_t *>(residual), p.gain = static_cast<const uint16_t *>(gain);
  p.rows = rows, p.cols = cols, p.pitch_a = x_pitch, p.pitch_b = residual_pitch, p.eps = eps, p.sum = static_cast<uint16_t *>(sum);
  p.q = static_cast<uint8_t *>(q), p.scale = scale, p.factor = scale_row;
  const bool wide = cols % 8 == 0 && wide_row(x, rows, x_pitch) && aligned(gain, 16) && aligned(q, 8) &&
                    (!residual || (wide_row(residual, rows, residual_pitch) && aligned(sum, 16)));
#define QUIK_CALL(BF16, BITS) (residual ? launch_norm<BF16, true, BITS>(p, wide, as_stream(stream)) : launch_norm<BF16, false, BITS>(p, wide, as_stream(stream)))
  return QUIK_BY_TYPE(QUIK_CALL);
#undef QUIK_CALL
}

extern "C" int quik_mx_dequantize(const void *q, int bits, const uint8_t *scale, const int64_t *index, const float *scale_row, int dtype, int64_t rows,
                                  int64_t source_rows, int64_t heads, int64_t cols, void *out, void *stream) {
  if (int rc = check_sizes(dtype, bits, rows, cols, cols, cols)) return rc;
  if (source_rows < 0 || heads < 0) return QUIK_ERR_SHAPE;
  if (heads > 1 << 30) return QUIK_ERR_RANGE;
  if (rows == 0 || heads == 0) return QUIK_OK;
  if (!index && rows != source_rows) return QUIK_ERR_SHAPE;
  if ((source_rows && (!q || !scale)) || !out) return QUIK_ERR_NULL;
  if (!aligned(out, 2) || !aligned(index, 8) || !aligned(scale_row, 4)) return QUIK_ERR_ALIGN;
  MxRead p{};
  p.q = static_cast<const uint8_t *>(q), p.scale = scale, p.index = index, p.factor = scale_row, p.source_rows = source_rows, p.heads = heads;
  p.cols = cols, p.count = rows, p.out = static_cast<uint16_t *>(out);
  const bool wide = cols % 8 == 0 && aligned(q, 8) && aligned(out, 16);
#define QUIK_CALL(BF16, BITS) launch_read<BF16, BITS>(p, wide, as_stream(stream))
  return QUIK_BY_TYPE(QUIK_CALL);
#undef QUIK_CALL
}
