// Tokens drawn from rows of logits with temperature, top-k, top-p and min-p, from given random numbers.
//
// A row's columns are ranked by logit, the largest first, equal ones by column. With w_j = exp((x_j - max) / T):
//
//   top-k leaves the first k ranks; top-p of these every rank before which less than p of their weight lies (one at least);
//   min-p of these the columns with w_j >= min_p; the token is the lowest of the columns that are left with
//   w_0 + .. + w_j > u (sum of w), in the order of columns.
//
// Ranks are found by value: with d the distance of a column's ordered key (argmax_key) from the row's largest, the first
// ranks are those with d below some d*, and the first columns of those with d = d*. d* is found by counting (and weighing) columns in
// 2,048 intervals of d, then in the intervals of the one that it lies in. Weights are counted there in fixed point, so that the order of
// the additions changes nothing.
#include "draw.h"

namespace tq {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2 * kThreads;

struct SampleArgs {
  int64_t* tokens;
  const void* logits;
  int64_t logits_stride;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;  // this and the next two: or null
  const float* top_p;
  const float* min_p;
  const int32_t* cu;  // or null: a setting a row
  int32_t* d_error;
  int32_t num_rows;
  int32_t num_seqs;
  int32_t vocab;
  int32_t mass_bits;  // weights are counted in units of 2^-mass_bits
};

struct Shared {
  uint32_t n[kBins];
  uint64_t m[kBins];
  uint64_t part[kWaves];
  double sum[kWaves], goal;
  float top[kWaves];
  int col, found, pick[kWaves][2];
  uint64_t before_n, before_m, bin_n;
  double tile[512];
};

__device__ __forceinline__ uint32_t ordered(float v) { return (uint32_t)(argmax_key(v, 0) >> 32); }

// The sequence of a row, -1: none.
__device__ __forceinline__ int owner_of(const SampleArgs& a, int row) {
  if (row < a.cu[0] || row >= a.cu[a.num_seqs]) return -1;
  int lo = 0, hi = a.num_seqs;  // cu[lo] <= row < cu[hi], where cu does not fall
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (a.cu[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(const SampleArgs a) {
  __shared__ Shared sh;
  constexpr int V = kVec<T>, kTile = kThreads * V;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  int set = row;
  if (a.cu != nullptr) {
    set = owner_of(a, row);
    if (set < 0) return;
  }
  const char* at = static_cast<const char*>(a.logits) + row * a.logits_stride * (__is_same(T, float) ? 4 : 2);
  const int vocab = a.vocab, tiles = (vocab + kTile - 1) / kTile;
  const float temp = a.temperature[set];
  int64_t* token = a.tokens + row;
  float x[V];
  auto load = [&](int tile) { columns<T, V, kThreads, V, true>(at, tile * kTile, min(kTile, vocab - tile * kTile), x); };
  auto column = [&](int tile, int e) { return tile * kTile + tid * V + e; };

  // The largest logit.
  float top = -INFINITY;
  for (int t = 0; t < tiles; ++t) {
    load(t);
#pragma unroll
    for (int e = 0; e < V; ++e) top = __builtin_elementwise_maximum(top, x[e]);
  }
  top = wave_maximum(top);
  if (lane == 0) sh.top[wave] = top;
  if (tid == 0) sh.col = 0x7fffffff;
  __syncthreads();
  for (int v = 0; v < kWaves; ++v) top = __builtin_elementwise_maximum(top, sh.top[v]);
  if (!(temp > 0.f) || !(top > -INFINITY && top < INFINITY)) {
    if (temp > 0.f && tid == 0) flag_error(a.d_error, TQ_DEVERR_VALUE);
    int mine = 0x7fffffff;
    for (int t = tiles - 1; t >= 0; --t) {
      load(t);
#pragma unroll
      for (int e = V - 1; e >= 0; --e)
        if (column(t, e) < vocab && (top != top ? x[e] != x[e] : x[e] == top)) mine = column(t, e);
    }
    atomicMin(&sh.col, mine);
    __syncthreads();
    if (tid == 0) *token = sh.col;
    return;
  }

  const double c = kLog2e / (double)temp, t0 = (double)top;
  auto weight = [&](float v) {
    const double t = ((double)v - t0) * c;
    return t >= -1000.0 ? exp2_neg(t) : 0.0;
  };
  const double unit = __builtin_ldexp(1.0, a.mass_bits);
  auto fixed = [&](double w) {  // w below 2^(52 - mass_bits)
    return __builtin_bit_cast(uint64_t, __builtin_fma(w, unit, 0x1p52)) & 0xfffffffffffffull;
  };
  const uint32_t key = ordered(top);
  auto distance = [&](float v) { return key - ordered(v); };

  // The d where the count of columns, or their mass, up to it first reaches `goal`; the count and mass before it and the count at it.
  struct Cut {
    uint32_t d;
    uint64_t n, m, ties;
  };
  auto find = [&](bool by_mass, double goal) {
    uint64_t lo = 0, n0 = 0, m0 = 0;
    int shift = 14;
    for (;;) {
      for (int i = tid; i < kBins; i += kThreads) {
        sh.n[i] = 0;
        sh.m[i] = 0;
      }
      if (tid == 0) sh.found = -1;
      __syncthreads();
      for (int t = 0; t < tiles; ++t) {
        load(t);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint64_t d = distance(x[e]);
          const uint64_t b = (d - lo) >> shift;
          if (column(t, e) < vocab && d >= lo && b < kBins) {
            atomicAdd(&sh.n[b], 1u);
            atomicAdd((unsigned long long*)&sh.m[b], (unsigned long long)fixed(weight(x[e])));
          }
        }
      }
      __syncthreads();
      const uint64_t na = sh.n[2 * tid], nb = sh.n[2 * tid + 1], ma = sh.m[2 * tid], mb = sh.m[2 * tid + 1];
      uint64_t n = n0 + scan<kThreads>(na + nb, sh.part), m = m0 + scan<kThreads>(ma + mb, sh.part);
      auto reaches = [&](uint64_t n, uint64_t m) { return by_mass ? (double)m >= goal : (double)n >= goal; };
      const uint64_t n1 = n - na - nb, m1 = m - ma - mb;  // before this thread's
      if (reaches(n, m) && (tid == 0 || !reaches(n1, m1))) {
        const bool first = reaches(n1 + na, m1 + ma);
        sh.found = 2 * tid + (first ? 0 : 1);
        sh.before_n = first ? n1 : n1 + na;
        sh.before_m = first ? m1 : m1 + ma;
        sh.bin_n = first ? na : nb;
      }
      if (tid == kThreads - 1) {
        sh.part[0] = n;
        sh.part[1] = m;
      }
      __syncthreads();
      const int found = sh.found;
      if (found < 0) {
        n0 = sh.part[0];
        m0 = sh.part[1];
        lo += (uint64_t)kBins << shift;
        shift = 21;
        if (lo >> 32 != 0) return Cut{0xffffffffu, n0, m0, 0};  // everything
      } else {
        n0 = sh.before_n;
        m0 = sh.before_m;
        lo += (uint64_t)found << shift;
        if (shift == 0) return Cut{(uint32_t)lo, n0, m0, sh.bin_n};
        shift = shift == 14 ? 3 : shift == 21 ? 10 : 0;
      }
      __syncthreads();
    }
  };
  auto weight_at = [&](uint32_t d) {  // of a column at distance d: an ordered key back to its value
    return weight(key_value((uint64_t)(key - d) << 32));
  };

  // Columns with d < cut.d and the first `ties` of those with d = cut.d are kept.
  Cut cut = {0xffffffffu, 0, 0, 0};
  uint64_t ties = 0;
  bool some = false;  // whether `ties` is less than there are
  const int k = a.top_k != nullptr ? a.top_k[set] : 0;
  const float p = a.top_p != nullptr ? a.top_p[set] : 1.f;
  if (k > 0 && k < vocab) {
    cut = find(false, (double)k);
    ties = k - cut.n;
    some = ties < cut.ties;
    __syncthreads();
  }
  if (p < 1.f) {
    uint64_t mass = 0;
    if (k > 0 && k < vocab) {
      mass = cut.m + ties * fixed(weight_at(cut.d));
    } else {
      for (int t = 0; t < tiles; ++t) {
        load(t);
#pragma unroll
        for (int e = 0; e < V; ++e) mass += column(t, e) < vocab ? fixed(weight(x[e])) : 0;
      }
      mass = scan<kThreads>(mass, sh.part);
      if (tid == kThreads - 1) sh.before_m = mass;
      __syncthreads();
      mass = sh.before_m;
      __syncthreads();
    }
    const double goal = (double)mass * (p > 0.f ? (double)p : 0.0);
    const Cut nucleus = find(true, goal);
    const double each = (double)fixed(weight_at(nucleus.d)), need = __builtin_ceil((goal - (double)nucleus.m) / each);
    uint64_t want = need >= 1.0 && need < (double)nucleus.ties ? (uint64_t)need : need < 1.0 ? 1 : nucleus.ties;
    if (k > 0 && k < vocab && nucleus.d == cut.d && want > ties) want = ties;
    cut = nucleus;
    ties = want;
    some = ties < cut.ties;
    __syncthreads();
  }
  // The column of the last tie that is kept.
  int last = vocab;
  if (some) {
    uint64_t before = 0;
    for (int t = 0; t < tiles; ++t) {
      load(t);
      uint64_t mine = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) mine += column(t, e) < vocab && distance(x[e]) == cut.d;
      const uint64_t upto = before + scan<kThreads>(mine, sh.part);
      if (upto >= ties && upto - mine < ties) {
        uint64_t left = ties - (upto - mine);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (column(t, e) < vocab && distance(x[e]) == cut.d && left-- == 1) sh.col = column(t, e);
      }
      if (tid == kThreads - 1) sh.before_n = upto;
      __syncthreads();
      before = sh.before_n;
      __syncthreads();
      if (before >= ties) break;
    }
    last = sh.col;
  }
  const float low = a.min_p != nullptr ? a.min_p[set] : 0.f;
  const double least = low > 0.f ? __builtin_fmin((double)low, 1.0) : 0.0;
  auto kept = [&](int tile, int e) {
    const uint32_t d = distance(x[e]);
    if (column(tile, e) >= vocab || d > cut.d || (d == cut.d && column(tile, e) > last)) return 0.0;
    const double w = weight(x[e]);
    return w >= least ? w : 0.0;
  };
  // The draw: the tile, then the column.
  for (int t = 0; t < tiles; ++t) {
    load(t);
    double w = 0.0;
#pragma unroll
    for (int e = 0; e < V; ++e) w += kept(t, e);
    w = wave_sum(w);
    if (lane == 0) sh.sum[wave] = w;
    __syncthreads();
    if (tid == 0) {
      w = 0.0;
      for (int v = 0; v < kWaves; ++v) w += sh.sum[v];
      sh.tile[t] = w;
    }
    __syncthreads();
  }
  const double mine = tid < tiles ? sh.tile[tid] : 0.0;
  const double upto = scan<kThreads>(mine, sh.sum);
  if (tid == kThreads - 1) sh.goal = (double)a.uniforms[row] * upto;
  __syncthreads();
  const double goal = sh.goal;
  const int chosen = pick<kThreads>(mine > 0.0 && upto > goal, mine > 0.0, sh.pick);
  if (tid == chosen) sh.goal = goal - (upto - mine);
  __syncthreads();
  const double rest = sh.goal;
  load(chosen);
  double w[V], run = 0.0;
#pragma unroll
  for (int e = 0; e < V; ++e) run += w[e] = kept(chosen, e);
  const double sum = scan<kThreads>(run, sh.sum);
  if (tid == pick<kThreads>(run > 0.0 && sum > rest, run > 0.0, sh.pick)) {
    double cum = sum - run;
    int col = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      cum += w[e];
      if (!done && w[e] > 0.0) {
        col = column(chosen, e);
        done = cum > rest;
      }
    }
    *token = col;
  }
}

constexpr int kMaxVocab = 1 << 21;

}  // namespace
}  // namespace tq

extern "C" tq_status tq_sample_tokens(int64_t* tokens, const void* logits, int64_t logits_row_stride,
                                      const float* uniforms, const float* temperature, const int32_t* top_k,
                                      const float* top_p, const float* min_p, const int32_t* cu_seqlens_q,
                                      int32_t num_seqs, int32_t num_rows, int32_t vocab, int32_t dtype, int32_t* d_error,
                                      void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || vocab < 1) return TQ_ERR_INVALID_ARGUMENT;
  if ((dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) || vocab > kMaxVocab) return TQ_ERR_UNSUPPORTED;
  if (num_rows == 0 || num_seqs == 0) return TQ_OK;
  if (tokens == nullptr || logits == nullptr || uniforms == nullptr || temperature == nullptr ||
      (cu_seqlens_q == nullptr && num_seqs < num_rows) || (num_rows > 1 && logits_row_stride < vocab))
    return TQ_ERR_INVALID_ARGUMENT;
  SampleArgs a;
  a.tokens = tokens;
  a.logits = logits;
  a.logits_stride = logits_row_stride;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.cu = cu_seqlens_q;
  a.d_error = d_error;
  a.num_rows = num_rows;
  a.num_seqs = num_seqs;
  a.vocab = vocab;
  int bits = 0;
  while (1 << bits < vocab) ++bits;
  a.mass_bits = bits > 12 ? 63 - bits : 51;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)num_rows), block(kThreads);
  if (dtype == TQ_F32)
    hipLaunchKernelGGL(sample_rows_kernel<float>, grid, block, 0, st, a);
  else if (dtype == TQ_BF16)
    hipLaunchKernelGGL(sample_rows_kernel<Bf16>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(sample_rows_kernel<Fp16>, grid, block, 0, st, a);
  return check_launch();
}
