// Heads between a block's first product and its attention, one launch over the columns of q, k and v:
//   n = x / sqrt(mean(x^2) + eps) * gain   per head of q and k, where there is a gain
//   y = n turned by its token's position: y_i = n_i cos_i - n_{i+r} sin_i, y_{i+r} = n_{i+r} cos_i + n_i sin_i for i < r, columns from 2r on as they are
//   q: y in the 16-bit type;  k: y, v: x, in blocks of 32 columns of a head (mx_format.h), into the cache row that the token's slot names
// fp32 from the load to the one rounding: y is not rounded to 16 bits in front of its codes.
//
// Bound by memory: every number is read once and written once.  A head is 4 lanes per block, eight columns each; the columns that turn with a lane's are
// loaded a second time (from the nearest cache) rather than exchanged.  A workgroup keeps its token's cosines and sines in registers and goes through
// the heads; few tokens are dealt to several workgroups each.
// 4096 tokens of 40 + 2 * 40 heads of 128 fp16, keys 8 bit, values 4: 45.4 us for 195 MB, 4.3 TB/s of a copy's 5.1 (by single columns 73.9 us); 64 tokens of
// 64 + 2 * 8 heads bf16 with norms 4.1 us, which is a launch and its loads' way.
#include "mx_format.h"

namespace quik {
namespace {

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

struct HeadArgs {
  const uint16_t *q, *k, *v;
  int64_t pitch_q, pitch_k, pitch_v;  // of tokens
  const float *cos, *sin;             // [positions, half]
  int64_t positions;
  const int64_t *position, *slot;
  const uint16_t *q_gain, *k_gain;
  float eps;
  uint16_t *q_out;
  uint8_t *k_codes, *k_scale, *v_codes, *v_scale;
  int64_t slots;
  int q_heads, kv_heads, size, half, k_bits, v_bits, splits;
};

template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_move<kDppSwap1>(v);
  v += dpp_move<kDppSwap2>(v);
  if constexpr (L >= 8) v += dpp_move<kDppHalfMirror>(v);
  if constexpr (L >= 16) v += dpp_move<kDppMirror>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

template <int BITS, bool WIDE>
__device__ __forceinline__ void put(const float (&v)[8], int left, uint8_t *codes, uint8_t *scale, int64_t vec, int size, int blocks, int c) {
  store_block<BITS, WIDE>(v, left, codes + (vec * size + c * int64_t{8}) * BITS / 8, scale + vec * blocks + c / 4, c % 4 == 0);
}

// L lanes per head, the power of two from four per block up.  WHOLE: every column turns, in chunks of eight that turn with each other, at 16-byte
// addresses; the other instance takes every size, element by element where a column's fellow is concerned.
// FOLD: a token's angles are multiplied with the norms' weights before its heads, for workgroups that go through many (us, as numbers are normed and
// this: 4096 tokens of 64 + 2 * 8 heads of 128, five rounds of heads each, 46.1, 41.3; of 32 + 2 * 32 46.0, 42.1; 300
// tokens, one round, 5.9, 7.1).
template <bool BF16, int L, bool WHOLE, bool FOLD>
__global__ __launch_bounds__(256) void mx_heads_kernel(HeadArgs p) {
  constexpr int kGroups = 256 / L;
  const int64_t token = blockIdx.x / static_cast<uint32_t>(p.splits);
  const int split = static_cast<int>(blockIdx.x % static_cast<uint32_t>(p.splits)), c = threadIdx.x % L, blocks = (p.size + kMxBlock - 1) / kMxBlock;
  const int rest = p.size - 8 * c, left = rest < 0 ? 0 : rest < 8 ? rest : 8, turned = 2 * p.half;
  const int64_t at = p.position[token], slot = p.slot[token];
  const bool known = at >= 0 && at < p.positions, kept = slot >= 0 && slot < p.slots;
  // this lane's columns: the factors of their own and of the number that they turn with, and where that one is
  alignas(16) float own[8], other[8];
  int with[8];
  if constexpr (WHOLE) {
    const bool front = 8 * c < p.half;
    const int j = left > 0 ? (front ? 8 * c : 8 * c - p.half) : 0;
    const int64_t from = (known ? at : 0) * p.half + j;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      if (known) {
        *reinterpret_cast<float4 *>(own + e) = *reinterpret_cast<const float4 *>(p.cos + from + e);
        *reinterpret_cast<float4 *>(other + e) = *reinterpret_cast<const float4 *>(p.sin + from + e);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      other[e] = front ? -other[e] : other[e];
      if (!known) own[e] = __builtin_nanf(""), other[e] = 0.0f;
      if (left <= 0) own[e] = 0.0f, other[e] = 0.0f;  // (behind the head's end, in its last block: zeros whatever the angles are)
    }
    with[0] = front ? j + p.half : j;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * c + e;
      own[e] = known ? 1.0f : __builtin_nanf(""), other[e] = 0.0f, with[e] = e < left ? i : 0;
      if (i < turned && e < left) {
        const int j = i < p.half ? i : i - p.half;
        if (known) {
          own[e] = p.cos[at * p.half + j];
          other[e] = p.sin[at * p.half + j];
          if (i < p.half) other[e] = -other[e];
        }
        with[e] = i < p.half ? i + p.half : j;
      }
    }
  }
  float weight_q[FOLD ? 2 : 1][8], weight_k[FOLD ? 2 : 1][8];
  if constexpr (FOLD) {
    auto weigh = [&](const uint16_t *gain, float (&to)[2][8]) {
      alignas(16) uint16_t g[8] = {}, h[8] = {};
      if (gain && left > 0) {
        load_eight<true>(gain + 8 * c, left, g);
        load_eight<true>(gain + with[0], 8, h);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        to[0][e] = gain ? own[e] * to_f32<BF16>(g[e]) : own[e];
        to[1][e] = gain ? other[e] * to_f32<BF16>(h[e]) : other[e];
      }
    };
    weigh(p.q_gain, weight_q);
    weigh(p.k_gain, weight_k);
  }
  const int all = p.q_heads + 2 * p.kv_heads;
  const int64_t base_q = token * p.pitch_q, base_k = token * p.pitch_k, base_v = token * p.pitch_v;
  for (int item = split * kGroups + threadIdx.x / L; item < all; item += p.splits * kGroups) {
    const bool is_q = item < p.q_heads, is_v = item >= p.q_heads + p.kv_heads;
    const int head = is_q ? item : is_v ? item - p.q_heads - p.kv_heads : item - p.q_heads;
    const uint16_t *from = (is_q ? p.q + base_q : is_v ? p.v + base_v : p.k + base_k) + head * p.size;
    alignas(16) uint16_t x[8] = {}, y[8] = {};
    if (left > 0) {
      load_eight<WHOLE>(from + 8 * c, left, x);
      if (!is_v) {
        if constexpr (WHOLE) {
          load_eight<true>(from + with[0], 8, y);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = from[with[e]];
        }
      }
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<BF16>(x[e]);
    if (!is_v) {
      const uint16_t *gain = is_q ? p.q_gain : p.k_gain;
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = to_f32<BF16>(y[e]);
      if (gain) {  // (the same for all lanes of the head)
        float square = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) square += v[e] * v[e];
        square = group_sum<L>(square);
        float lift = 1.0f;
        if (tiny_squares<BF16, kNorm>(1, square, p.size, p.eps)) {
          lift = kLift;
          square = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) square += v[e] * lift * (v[e] * lift);
          square = group_sum<L>(square);
        }
        float f = norm_factor(square, p.size, p.eps, lift);
        if (square == 0.0f && p.eps == 0.0f) f = 0.0f;  // (a head of zeros)
        if (!(square < __builtin_inff())) f = __builtin_nanf("");
        alignas(16) uint16_t g[8] = {}, h[8] = {};
        if (!FOLD && left > 0) {
          load_eight<WHOLE>(gain + 8 * c, left, g);
          if constexpr (WHOLE) {
            load_eight<true>(gain + with[0], 8, h);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = gain[with[e]];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = v[e] * lift * f * (FOLD ? 1.0f : to_f32<BF16>(g[e]));
          t[e] = t[e] * lift * f * (FOLD ? 1.0f : to_f32<BF16>(h[e]));
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = FOLD ? (is_q ? weight_q[0][e] : weight_k[0][e]) : own[e], b = FOLD ? (is_q ? weight_q[FOLD][e] : weight_k[FOLD][e]) : other[e];
        const float turn = v[e] * a + t[e] * b;
        v[e] = WHOLE || (e < left && (8 * c + e < turned || !known)) ? turn : v[e];  // (a column that stays is not added 0 * t: t may be an infinity)
      }
      if constexpr (!WHOLE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? v[e] : 0.0f;
      }
    }
    if (is_q) {
      alignas(16) uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = pack2_from_f32<BF16>(v[2 * e], v[2 * e + 1]);
      alignas(16) uint16_t out[8];
      *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(h);
      if (left > 0) store_eight<WHOLE>(p.q_out + (token * p.q_heads + head) * p.size + 8 * c, left, out);
    } else {
      uint8_t *codes = is_v ? p.v_codes : p.k_codes, *scale = is_v ? p.v_scale : p.k_scale;
      const int64_t vec = slot * p.kv_heads + head;
      if ((is_v ? p.v_bits : p.k_bits) == 4) put<4, WHOLE>(v, kept ? left : 0, codes, scale, vec, p.size, blocks, c);
      else put<8, WHOLE>(v, kept ? left : 0, codes, scale, vec, p.size, blocks, c);
    }
  }
}

template <bool BF16, int L>
int launch_heads(const HeadArgs &p, int64_t tokens, bool wide, hipStream_t st) {
  HeadArgs a = p;
  constexpr int kGroups = 256 / L;
  const int64_t most = (p.q_heads + 2 * static_cast<int64_t>(p.kv_heads) + kGroups - 1) / kGroups, wanted = (4 * num_cus() + tokens - 1) / tokens;
  // A workgroup per round of heads where all of them run at once; more than that wait for their token's position and angles once more each (us, the heads of a
  // token dealt to four per CU, and one round each: 300 tokens of 64 + 2 * 8 heads of 128 7.8, 5.8; 1024 of 40 + 2 * 40 12.3, 17.0).
  a.splits = static_cast<int>(tokens * most <= 8 * num_cus() || wanted >= most ? most : wanted);
  const int64_t per_launch = (INT32_MAX / 256) / a.splits;
  for (int64_t first = 0; first < tokens; first += per_launch) {
    const int64_t n = tokens - first < per_launch ? tokens - first : per_launch;
    const dim3 grid(static_cast<unsigned>(n * a.splits));
    const bool fold = wide && (p.q_gain || p.k_gain) && most >= 4 * static_cast<int64_t>(a.splits);
    if (fold) hipLaunchKernelGGL((mx_heads_kernel<BF16, L, true, true>), grid, dim3(256), 0, st, a);
    else if (wide) hipLaunchKernelGGL((mx_heads_kernel<BF16, L, true, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mx_heads_kernel<BF16, L, false, false>), grid, dim3(256), 0, st, a);
    if (int rc = check_launch()) return rc;
    a.q += n * p.pitch_q, a.k += n * p.pitch_k, a.v += n * p.pitch_v;
    a.position += n, a.slot += n;
    a.q_out += n * p.q_heads * p.size;
  }
  return QUIK_OK;
}
template <bool BF16>
int by_size(const HeadArgs &p, int64_t tokens, bool wide, hipStream_t st) {
  if (p.size <= 64) return launch_heads<BF16, 8>(p, tokens, wide, st);
  if (p.size <= 128) return launch_heads<BF16, 16>(p, tokens, wide, st);
  if (p.size <= 256) return launch_heads<BF16, 32>(p, tokens, wide, st);
  return launch_heads<BF16, 64>(p, tokens, wide, st);
}
}  // namespace
}  // namespace quik

using namespace quik;

extern "C" int quik_mx_rotate_to_cache(const quik_mx_heads *h, void *stream) {
  if (!h) return QUIK_ERR_NULL;
  if (h->struct_bytes != static_cast<int32_t>(sizeof(quik_mx_heads))) return QUIK_ERR_SHAPE;
  if ((h->k_bits != 4 && h->k_bits != 8) || (h->v_bits != 4 && h->v_bits != 8)) return QUIK_ERR_BITS;
  if (h->dtype != QUIK_F16 && h->dtype != QUIK_BF16) return QUIK_ERR_DTYPE;
  const int64_t D = h->size;
  if (h->tokens < 0 || h->q_heads < 0 || h->kv_heads < 0 || D <= 0 || h->half <= 0 || 2 * h->half > D || h->positions < 0 || h->slots < 0) return QUIK_ERR_SHAPE;
  if (D % 2) return QUIK_ERR_ALIGN;
  if (D > 512 || h->q_heads > 1 << 20 || h->kv_heads > 1 << 20 || h->tokens > INT32_MAX) return QUIK_ERR_RANGE;
  if (h->tokens > 1 && (h->q_pitch < h->q_heads * D || h->k_pitch < h->kv_heads * D || h->v_pitch < h->kv_heads * D)) return QUIK_ERR_SHAPE;
  if (!(h->eps >= 0.0f)) return QUIK_ERR_RANGE;
  if (h->tokens == 0 || h->q_heads + h->kv_heads == 0) return QUIK_OK;
  if ((h->positions && (!h->cos || !h->sin)) || !h->position || !h->slot || (h->q_heads && (!h->q || !h->q_out)) ||
      (h->kv_heads && (!h->k || !h->v || (h->slots && (!h->k_codes || !h->k_scale || !h->v_codes || !h->v_scale)))))
    return QUIK_ERR_NULL;
  if (!aligned(h->q, 2) || !aligned(h->k, 2) || !aligned(h->v, 2) || !aligned(h->q_out, 2) || !aligned(h->cos, 4) || !aligned(h->sin, 4) ||
      !aligned(h->position, 8) || !aligned(h->slot, 8) || !aligned(h->q_gain, 2) || !aligned(h->k_gain, 2))
    return QUIK_ERR_ALIGN;
  HeadArgs p{};
  p.q = static_cast<const uint16_t *>(h->q), p.k = static_cast<const uint16_t *>(h->k), p.v = static_cast<const uint16_t *>(h->v);
  p.pitch_q = h->q_pitch, p.pitch_k = h->k_pitch, p.pitch_v = h->v_pitch;
  p.cos = h->cos, p.sin = h->sin, p.positions = h->positions, p.position = h->position, p.slot = h->slot;
  p.q_gain = static_cast<const uint16_t *>(h->q_gain), p.k_gain = static_cast<const uint16_t *>(h->k_gain), p.eps = h->eps;
  p.q_out = static_cast<uint16_t *>(h->q_out);
  p.k_codes = static_cast<uint8_t *>(h->k_codes), p.k_scale = h->k_scale, p.v_codes = static_cast<uint8_t *>(h->v_codes), p.v_scale = h->v_scale;
  p.slots = h->slots, p.q_heads = static_cast<int>(h->q_heads), p.kv_heads = static_cast<int>(h->kv_heads), p.size = static_cast<int>(D);
  p.half = static_cast<int>(h->half), p.k_bits = h->k_bits, p.v_bits = h->v_bits;
  auto wide_rows = [&](const void *at, int64_t pitch) { return aligned(at, 16) && (h->tokens == 1 || pitch % 8 == 0); };
  const bool wide = 2 * h->half == D && h->half % 8 == 0 && wide_rows(h->q, h->q_pitch) && wide_rows(h->k, h->k_pitch) && wide_rows(h->v, h->v_pitch) &&
                    aligned(h->q_out, 16) && aligned(h->cos, 16) && aligned(h->sin, 16) && aligned(h->q_gain, 16) && aligned(h->k_gain, 16) &&
                    aligned(h->k_codes, 8) && aligned(h->v_codes, 8);
  return h->dtype == QUIK_BF16 ? by_size<true>(p, h->tokens, wide, as_stream(stream)) : by_size<false>(p, h->tokens, wide, as_stream(stream));
}
