// Cache write with the position rotation applied on the way: one pass that norms (optionally) and rotates
// every new token's query and key heads, writes the queries out and the keys, with the values as they are,
// into the block pool.
//
//   y = x w / sqrt(mean(x^2) + eps)                                  (per head, where weights are given)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)             pairs (i, i + R / 2) or (2 i, 2 i + 1), i < R / 2
//
// with cos and sin from the caller's fp32 table, so their angles are as exact as the caller made them; all
// arithmetic is fp32, rounded once to the rows' type.
//
// HBM bound: every element is read once and written once (8,192 tokens of 32 + 8 + 8 heads of 128, normed: 206 MB in 45 us, 4.5
// TB/s, where a device copy moves 5.07). A thread holds 16 elements of one head, the two
// octets that the rotation pairs (8 t .. and R / 2 + 8 t .., or 16 t ..), so both are moved by 16-byte accesses
// and the pairs meet in registers; the D / 16 threads of a head share its sum of squares by lane permutations.

#include "half_types.h"

namespace tq {
namespace {

struct RopeArgs {
  void* q_out;
  int64_t q_out_stride;
  const void* q;
  int64_t q_stride;
  const void* k;
  int64_t k_stride;
  const void* v;
  int64_t v_stride;
  void* pool_layer;
  int64_t block_stride;
  int64_t kv_stride;
  int64_t head_stride;
  const int64_t* slot_mapping;
  const int64_t* positions;
  const float* table;  // [num_positions][rotary]: cos of the rotary / 2 angles, then sin
  int64_t num_positions;
  const void* q_norm;
  const void* k_norm;
  float eps;
  int32_t rotary;
  int32_t heads;
  int32_t kv_heads;
  int32_t block_size;
  int64_t num_tokens;
  int64_t num_slots;
  int32_t* d_error;
};

struct F32 {};

// Eight consecutive elements as floats, and back with one rounding.
template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (__is_same(T, F32)) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
    const f32x4 lo = p[0], hi = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = lo[e];
      x[4 + e] = hi[e];
    }
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = T::load((uint16_t)w[e]);
      x[2 * e + 1] = T::load((uint16_t)(w[e] >> 16));
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
  if constexpr (__is_same(T, F32)) {
    f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + at);
    p[0] = f32x4{x[0], x[1], x[2], x[3]};
    p[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + at) =
        u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
  }
}

// Bits as they are (a value's NaN keeps its payload).
template <typename T>
__device__ __forceinline__ void copy8(void* to, int64_t to_at, const void* from, int64_t from_at) {
  if constexpr (__is_same(T, F32)) {
    const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(from) + from_at);
    u32x4* o = reinterpret_cast<u32x4*>(static_cast<float*>(to) + to_at);
    const u32x4 lo = p[0], hi = p[1];
    o[0] = lo;
    o[1] = hi;
  } else {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(to) + to_at) =
        *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(from) + from_at);
  }
}

// Sum over the D / 16 neighbouring lanes of a head (4 or 8).
template <int D>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp_move<kDppQuadXor1>(v);
  v += dpp_move<kDppQuadXor2>(v);
  if constexpr (D == 128) v += dpp_move<kDppRowHalfMirror>(v);
  return v;
}

template <int D, typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_cache_write_kernel(const RopeArgs a) {
  constexpr int kLanes = D / 16;  // threads of a head
  const uint32_t head_rows = a.heads + 2 * a.kv_heads;
  const uint32_t unit = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;  // below 2^32: 64-bit divisions are slow
  const int64_t n = unit / head_rows;
  if (n >= a.num_tokens) return;  // whole heads: the lanes that trade sums end together
  const int hr = (int)(unit - (uint32_t)n * head_rows), t = threadIdx.x % kLanes;
  const int64_t slot = a.slot_mapping[n], pos = a.positions[n];
  if (pos < 0 || pos >= a.num_positions) {
    if (hr == 0 && t == 0) flag_error(a.d_error, TQ_DEVERR_POSITION);
    return;
  }
  if (slot >= a.num_slots && hr == 0 && t == 0) flag_error(a.d_error, TQ_DEVERR_SLOT);
  const bool cached = slot >= 0 && slot < a.num_slots;
  const int64_t blk = cached ? (uint32_t)slot / (uint32_t)a.block_size : 0;
  const int64_t at = blk * a.block_stride + (slot - blk * a.block_size) * D;
  const int half = a.rotary / 2;
  const bool turned = 16 * t < a.rotary;
  // The thread's octets: the pair's two halves, 16 neighbours where pairs are neighbours or nothing turns.
  const int lo = INTERLEAVED || !turned ? 16 * t : 8 * t, hi = INTERLEAVED || !turned ? 16 * t + 8 : half + 8 * t;

  if (hr >= a.heads + a.kv_heads) {
    if (!cached) return;
    const int h = hr - a.heads - a.kv_heads;
    const int64_t to = at + a.kv_stride + h * a.head_stride, from = n * a.v_stride + (int64_t)h * D;
    copy8<T>(a.pool_layer, to + 16 * t, a.v, from + 16 * t);
    copy8<T>(a.pool_layer, to + 16 * t + 8, a.v, from + 16 * t + 8);
    return;
  }
  const bool is_q = hr < a.heads;
  if (!is_q && !cached) return;
  const int h = is_q ? hr : hr - a.heads;
  const void* src = is_q ? a.q : a.k;
  const int64_t from = (is_q ? n * a.q_stride : n * a.k_stride) + (int64_t)h * D;
  float x[8], y[8];
  load8<T>(src, from + lo, x);
  load8<T>(src, from + hi, y);
  const void* w = is_q ? a.q_norm : a.k_norm;
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
    const float r = 1.f / sqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
    float wx[8], wy[8];
    load8<T>(w, lo, wx);
    load8<T>(w, hi, wy);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = x[e] * r * wx[e];
      y[e] = y[e] * r * wy[e];
    }
  }
  if (turned) {
    const float* cp = a.table + pos * a.rotary + 8 * t;
    float c[8], s[8];
    load8<F32>(cp, 0, c);
    load8<F32>(cp + half, 0, s);
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float xa = x[2 * e], xb = x[2 * e + 1], ya = y[2 * e], yb = y[2 * e + 1];
        x[2 * e] = xa * c[e] - xb * s[e];
        x[2 * e + 1] = xb * c[e] + xa * s[e];
        y[2 * e] = ya * c[4 + e] - yb * s[4 + e];
        y[2 * e + 1] = yb * c[4 + e] + ya * s[4 + e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xa = x[e], yb = y[e];
        x[e] = xa * c[e] - yb * s[e];
        y[e] = yb * c[e] + xa * s[e];
      }
    }
  }
  void* dst = is_q ? a.q_out : a.pool_layer;
  const int64_t to = is_q ? n * a.q_out_stride + (int64_t)h * D : at + h * a.head_stride;
  store8<T>(dst, to + lo, x);
  store8<T>(dst, to + hi, y);
}

template <int D, typename T>
tq_status launch(const RopeArgs& a, bool interleaved, hipStream_t stream) {
  constexpr int kUnits = 256 / (D / 16);  // heads of a workgroup
  const int64_t head_rows = a.heads + 2LL * a.kv_heads;
  if (a.num_tokens > 0xffff0000LL / head_rows) return TQ_ERR_UNSUPPORTED;
  const int64_t grid = (a.num_tokens * head_rows + kUnits - 1) / kUnits;
  if (interleaved)
    hipLaunchKernelGGL((rope_cache_write_kernel<D, T, true>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((rope_cache_write_kernel<D, T, false>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  return check_launch();
}

template <typename T>
tq_status launch(const RopeArgs& a, int32_t head_dim, bool interleaved, hipStream_t stream) {
  return head_dim == 64 ? launch<64, T>(a, interleaved, stream) : launch<128, T>(a, interleaved, stream);
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_rope_cache_write(void* q_out, int64_t q_out_row_stride, const void* q, int64_t q_row_stride,
                                         const void* k, int64_t k_row_stride, const void* v, int64_t v_row_stride,
                                         void* pool, int64_t num_blocks, int32_t num_layers, int32_t num_heads,
                                         int32_t num_kv_heads, int32_t block_size, int32_t head_dim, int32_t layer,
                                         const int64_t* slot_mapping, const int64_t* positions, const float* table,
                                         int64_t num_positions, int32_t rotary_dim, int32_t interleaved,
                                         const void* q_norm, const void* k_norm, float eps, int64_t num_tokens,
                                         int32_t dtype, int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_tokens < 0 || num_blocks < 1 || num_layers < 1 || num_heads < 1 || num_kv_heads < 1 || block_size < 1 ||
      head_dim < 1 || layer < 0 || layer >= num_layers || num_positions < 0 || rotary_dim < 1 ||
      rotary_dim > head_dim || (interleaved != 0 && interleaved != 1) || !(eps >= 0.f))
    return TQ_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128) || block_size > kMaxBlockSize || rotary_dim % 16 != 0 ||
      num_blocks > 0xffffffffLL / block_size || num_heads > 1 << 20 || num_kv_heads > 1 << 20 ||
      (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16))
    return TQ_ERR_UNSUPPORTED;
  if (num_tokens == 0) return TQ_OK;
  const int64_t q_width = (int64_t)num_heads * head_dim, kv_width = (int64_t)num_kv_heads * head_dim;
  if (q_out == nullptr || q == nullptr || k == nullptr || v == nullptr || pool == nullptr || slot_mapping == nullptr ||
      positions == nullptr || table == nullptr || q_out_row_stride < q_width || q_row_stride < q_width ||
      k_row_stride < kv_width || v_row_stride < kv_width)
    return TQ_ERR_INVALID_ARGUMENT;
  // 16-byte accesses.
  const int64_t per16 = dtype == TQ_F32 ? 4 : 8;
  if (((uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)pool | (uintptr_t)table |
       (uintptr_t)q_norm | (uintptr_t)k_norm) % 16 != 0 ||
      q_out_row_stride % per16 != 0 || q_row_stride % per16 != 0 || k_row_stride % per16 != 0 ||
      v_row_stride % per16 != 0)
    return TQ_ERR_INVALID_ARGUMENT;

  const PoolGeom g = pool_geom(num_layers, num_kv_heads, block_size, head_dim, layer);
  RopeArgs a;
  a.q_out = q_out;
  a.q_out_stride = q_out_row_stride;
  a.q = q;
  a.q_stride = q_row_stride;
  a.k = k;
  a.k_stride = k_row_stride;
  a.v = v;
  a.v_stride = v_row_stride;
  a.pool_layer = static_cast<char*>(pool) + g.layer_offset * (dtype == TQ_F32 ? 4 : 2);
  a.block_stride = g.block_stride;
  a.kv_stride = g.kv_stride;
  a.head_stride = g.head_stride;
  a.slot_mapping = slot_mapping;
  a.positions = positions;
  a.table = table;
  a.num_positions = num_positions;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.rotary = rotary_dim;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.block_size = block_size;
  a.num_tokens = num_tokens;
  a.num_slots = num_blocks * block_size;
  a.d_error = d_error;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TQ_F32) return launch<F32>(a, head_dim, interleaved != 0, st);
  return dtype == TQ_BF16 ? launch<Bf16>(a, head_dim, interleaved != 0, st)
                          : launch<Fp16>(a, head_dim, interleaved != 0, st);
}
