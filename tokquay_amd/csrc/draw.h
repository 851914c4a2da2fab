// What the kernels that draw tokens from rows of logits share: exponentials and their sums in fp64, reductions of a wave.
#pragma once

#include "half_types.h"

namespace tq {
namespace {

// 2^t for t <= 0: 2^k 2^f with k the nearest integer (read off the low bits of t + 1.5 2^52), the second factor by the polynomial
// that meets 2^f at 0 and at the 8 Chebyshev points of [-1/2, 1/2]; off by at most 2.2e-12, and 1 for 0, so that equal logits
// have equal, whole weights. Below -1000, and for NaN: 2^-1000, which no sum of theirs notices.
__device__ __forceinline__ double exp2_neg(double t) {
  t = __builtin_fmax(t, -1000.0);
  const double shifted = t + 0x1.8p52;
  const double f = t - (shifted - 0x1.8p52);
  double r = 1.3250805512080399e-06;
  r = __builtin_fma(r, f, 1.5303700711214572e-05);
  r = __builtin_fma(r, f, 1.5403475186561525e-04);
  r = __builtin_fma(r, f, 1.333347847368613e-03);
  r = __builtin_fma(r, f, 9.618129135236088e-03);
  r = __builtin_fma(r, f, 5.550410906325866e-02);
  r = __builtin_fma(r, f, 2.4022650695888503e-01);
  r = __builtin_fma(r, f, 6.931471805568324e-01);
  r = __builtin_fma(r, f, 1.0);
  u32x2 bits = __builtin_bit_cast(u32x2, r);
  bits[1] += __builtin_bit_cast(u32x2, shifted)[0] << 20;
  return __builtin_bit_cast(double, bits);
}

template <typename T>
__device__ __forceinline__ float logit_at(const void* row, int64_t j) {
  if constexpr (__is_same(T, float))
    return static_cast<const float*>(row)[j];
  else
    return T::load(static_cast<const uint16_t*>(row)[j]);
}

// The value an argmax_key stands for (NaN: every NaN).
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// Reductions of a wave, through DPP in rows of 16 lanes and lanes 0, 16, 32, 48 (a 64-bit shuffle through LDS takes five times as
// long, and they lie on the path of a small call). Every lane gets the result; all orders of the lanes give the same.
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_move64(uint64_t v) {
  const uint32_t lo = __float_as_uint(dpp_move<CTRL>(__uint_as_float((uint32_t)v)));
  const uint32_t hi = __float_as_uint(dpp_move<CTRL>(__uint_as_float((uint32_t)(v >> 32))));
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}
template <typename F>
__device__ __forceinline__ uint64_t wave_reduce(uint64_t v, F&& join) {
  v = join(v, dpp_move64<kDppQuadXor1>(v));
  v = join(v, dpp_move64<kDppQuadXor2>(v));
  v = join(v, dpp_move64<kDppRowHalfMirror>(v));
  v = join(v, dpp_move64<kDppRowMirror>(v));
  return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ double wave_sum(double v) {
  return __builtin_bit_cast(double, wave_reduce(__builtin_bit_cast(uint64_t, v), [](uint64_t a, uint64_t b) {
                              return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b));
                            }));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  return wave_reduce(v, [](uint64_t a, uint64_t b) { return max_u64(a, b); });
}
__device__ __forceinline__ float wave_maximum(float v) {  // NaN, if any is
  v = __builtin_elementwise_maximum(v, dpp_move<kDppQuadXor1>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppQuadXor2>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppRowHalfMirror>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppRowMirror>(v));
  auto lane = [&](int l) { return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); };
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(lane(0), lane(16)),
                                       __builtin_elementwise_maximum(lane(32), lane(48)));
}

template <typename T>
constexpr int kVec = __is_same(T, float) ? 4 : 8;  // logits in 16 bytes

// Thread t's column i of a chunk: pieces of VEC columns t, t + N, .. (of N threads), or (RUNS) PER columns in a row.
template <int VEC, int N, int PER, bool RUNS>
__device__ __forceinline__ int column_of(int i) {
  return RUNS ? (int)threadIdx.x * PER + i : (i / VEC * N + (int)threadIdx.x) * VEC + i % VEC;
}

// Those columns of a row of T as floats, columns past n as -inf. Rows start at any element.
template <typename T, int VEC, int N, int PER, bool RUNS>
__device__ __forceinline__ void columns(const void* row, int base, int n, float (&x)[PER]) {
  constexpr int kSize = __is_same(T, float) ? 4 : 2;
#pragma unroll
  for (int v = 0; v < PER; v += VEC) {
    const int at = column_of<VEC, N, PER, RUNS>(v);
    if (at + VEC <= n) {
      u32x4 w[VEC * kSize / 16];
      __builtin_memcpy(w, static_cast<const char*>(row) + (int64_t)(base + at) * kSize, VEC * kSize);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if constexpr (__is_same(T, float))
          x[v + e] = __uint_as_float(w[e / 4][e % 4]);
        else
          x[v + e] = T::load((uint16_t)(w[e / 8][e % 8 / 2] >> (16 * (e & 1))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[v + e] = at + e < n ? logit_at<T>(row, base + at + e) : -INFINITY;
    }
  }
}

constexpr double kLog2e = 1.4426950408889634;

// The sequence that a row belongs to: the last one with cu[b] <= row (empty sequences hold no row), among 64 parts at a time.
// Its temperature, asked for before the logits, arrives before them. (Counted through all 1,024 sequences of 5 rows, 50,257 bf16
// logits each, the call took 328 us instead of 259.) Where cu falls somewhere this may be another one, still below num_seqs; every
// count grows with the row, so if it is b for two rows it is for those between them.
__device__ __forceinline__ int64_t owner_of(const int32_t* cu, int num_seqs, int row) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t b = 0, n = num_seqs;
  while (n > 1) {
    const int64_t step = (n + kWave - 1) / kWave, at = b + lane * step;
    const int k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane * step < n && cu[at] <= row));
    const int64_t skip = max(k - 1, 0) * step;
    b += skip;
    n = min(step, n - skip);
  }
  return b;
}

struct Stat {  // of one row's chunk
  double sum;      // of exp((logit - max) / T); 0 at T = 0
  uint64_t key;    // argmax_key of its largest logit (the column: where T = 0 or the maximum is not finite)
};

template <int N>
struct StatShared {
  float top[N / kWave];
  double sum[N / kWave];
  int col;
};

// What is kept of a row's chunk of N * PER columns, n of them there, by the workgroup of N threads that holds it (columns). The sum only
// where it is asked for and the row has a temperature.
template <typename T, int PER, int N>
__device__ __forceinline__ void chunk_stat(const float (&x)[PER], float temp, bool sums, int base, int n, Stat* to,
                                           StatShared<N>& sh) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = __builtin_elementwise_maximum(top, x[i]);  // NaN, if any is
  top = wave_maximum(top);
  if (lane == 0) sh.top[wave] = top;
  if (threadIdx.x == 0) sh.col = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < N / kWave; ++v) top = __builtin_elementwise_maximum(top, sh.top[v]);
  double sum = 0.0;
  int col = 0;
  if (temp > 0.f && top > -INFINITY && top < INFINITY) {  // uniform
    if (sums) {
      const double c = kLog2e / (double)temp, t0 = (double)top;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += exp2_neg(((double)x[i] - t0) * c);
      sum = wave_sum(sum);
    }
    if (lane == 0) sh.sum[wave] = sum;
  } else {  // no distribution, or none needed: the first column that holds the maximum
    int mine = 0x7fffffff;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i) {
      const int at = column_of<kVec<T>, N, PER, false>(i);
      if (at < n && (top != top ? x[i] != x[i] : x[i] == top)) mine = at;
    }
    // One lane of the workgroup, if no others hold the maximum (the atomics of all lanes go one by one: 64 greedy rows of 50,257 bf16
    // logits 9.0 us instead of 4.6).
    if (mine != 0x7fffffff) atomicMin(&sh.col, mine);
    if (lane == 0) sh.sum[wave] = 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = sh.sum[0];
#pragma unroll
    for (int v = 1; v < N / kWave; ++v) sum += sh.sum[v];
    if (sh.col != 0x7fffffff) col = sh.col;
    *to = Stat{sum, argmax_key(top, base + col)};
  }
}

}  // namespace
}  // namespace tq
